"""Refusals of the paged-cache operators: the C ABI and the Python front end turn a bad call into an error before any GPU work."""
import ctypes

import pytest
import torch

from ringattention_b200 import _lib
from ringattention_b200 import build as lib_build


@pytest.fixture(scope="module")
def lib():
    lib_build.build()
    return _lib.load()


def paged(**kw):
    p = _lib.Ring_paged_params()
    base = dict(k_cache=0x1000, v_cache=0x2000, k_page_stride=2 * 16 * 64, k_head_stride=16 * 64, k_place_stride=64,
                v_page_stride=2 * 16 * 64, v_head_stride=16 * 64, v_place_stride=64, num_pages=8, page_size=16, kv_heads=2, dim=64,
                page_table=0x3000, table_stride=4, max_pages=4, batch=2, kv_lens=0x4000, tokens=2, q=0x5000, q_token_stride=4 * 64,
                q_head_stride=64, heads=4, out=0x6000, out_token_stride=4 * 64, out_head_stride=64, lse=0x7000, softmax_scale=0.125,
                causal=1, k_new=0x8000, v_new=0x9000, k_new_token_stride=128, k_new_head_stride=64, v_new_token_stride=128,
                v_new_head_stride=64, weights=0xa000, weights_batch_stride=128, weights_head_stride=64, weights_len=64,
                workspace=0x10000, workspace_bytes=1 << 40)
    base.update(kw)
    for k, v in base.items():
        setattr(p, k, v)
    return p


def evict(**kw):
    p = _lib.Ring_evict_params()
    base = dict(k_cache=0x1000, v_cache=0x2000, k_page_stride=2 * 16 * 64, k_head_stride=16 * 64, k_place_stride=64,
                v_page_stride=2 * 16 * 64, v_head_stride=16 * 64, v_place_stride=64, num_pages=8, page_size=16, kv_heads=2, dim=64,
                page_table=0x3000, table_stride=4, max_pages=4, batch=2, kv_lens=0x4000, dst_table=0x3100, dst_stride=2, dst_pages=2,
                budget=32, first=2, recent=8, weights=0xa000, weights_batch_stride=128, weights_head_stride=64, weights_len=64,
                new_weights=0xb000, new_weights_batch_stride=64, new_weights_head_stride=32, new_weights_len=32, kept=0xc000,
                new_lens=0xd000)
    base.update(kw)
    for k, v in base.items():
        setattr(p, k, v)
    return p


CACHE = [
    (dict(dim=96), "dim must be 64 or 128"), (dict(page_size=12), "power of two"), (dict(page_size=4), "power of two"),
    (dict(page_size=0), "power of two"), (dict(num_pages=0), "num_pages"), (dict(kv_heads=0), "kv_heads"),
    (dict(max_pages=0), "max_pages"), (dict(max_pages=1 << 27, table_stride=1 << 27), "2^30"), (dict(batch=0), "batch"),
    (dict(batch=65536), "batch"), (dict(batch=40000, tokens=40000), "65535"), (dict(page_table=None), "page_table"),
    (dict(kv_lens=None), "kv_lens"), (dict(table_stride=3), "table_stride"), (dict(k_cache=None), "k_cache"),
    (dict(k_cache=0x1008), "16-byte aligned"), (dict(k_place_stride=60), "multiples of 8"), (dict(v_head_stride=4), "multiples of 8"),
    (dict(k_page_stride=-64), "negative"), (dict(k_head_stride=0), "strides of 0"), (dict(k_place_stride=0), "strides of 0"),
]


@pytest.mark.parametrize("kw,needle", CACHE)
@pytest.mark.parametrize("fn", ["ring_paged_append", "ring_paged_attention_fwd", "ring_paged_weights", "ring_paged_evict"])
def test_every_call_refuses_a_bad_cache(lib, fn, kw, needle):
    if fn == "ring_paged_evict":
        p = evict(**{k: v for k, v in kw.items() if k != "tokens"})
    else:
        p = paged(**kw)
    assert getattr(lib, fn)(ctypes.byref(p)) == _lib.RING_ERR_INVALID_ARGUMENT
    assert needle in lib.ring_last_error_string().decode()


@pytest.mark.parametrize("fn,kw,needle", [
    ("ring_paged_append", dict(tokens=-1), "tokens"), ("ring_paged_append", dict(tokens=3), "multiple of batch"),
    ("ring_paged_append", dict(k_new=None), "k_new"), ("ring_paged_append", dict(v_cache=None), "v_cache"),
    ("ring_paged_append", dict(v_new=0x9004), "aligned"), ("ring_paged_append", dict(k_new_token_stride=60), "multiples of 8"),
    ("ring_paged_append", dict(weights_len=63), "weights_len"), ("ring_paged_append", dict(k_head_stride=0), "strides of 0"),
    ("ring_paged_attention_fwd", dict(tokens=3), "multiple of batch"), ("ring_paged_attention_fwd", dict(heads=3), "multiple of kv_heads"),
    ("ring_paged_attention_fwd", dict(heads=0), "multiple of kv_heads"), ("ring_paged_attention_fwd", dict(max_new=-1), "max_new"),
    ("ring_paged_attention_fwd", dict(softmax_scale=0.0), "softmax_scale"),
    ("ring_paged_attention_fwd", dict(softmax_scale=float("nan")), "softmax_scale"),
    ("ring_paged_attention_fwd", dict(softmax_scale=float("inf")), "softmax_scale"),
    ("ring_paged_attention_fwd", dict(window=-1), "window"), ("ring_paged_attention_fwd", dict(sinks=-1), "sinks"),
    ("ring_paged_attention_fwd", dict(window=8, causal=0), "causal"), ("ring_paged_attention_fwd", dict(q=None), "null q"),
    ("ring_paged_attention_fwd", dict(lse=None), "lse"), ("ring_paged_attention_fwd", dict(q=0x5002), "aligned"),
    ("ring_paged_attention_fwd", dict(q_head_stride=20), "multiples of 8"), ("ring_paged_weights", dict(q_head_stride=0), "strides of 0"), ("ring_paged_attention_fwd", dict(out=None), "out"),
    ("ring_paged_attention_fwd", dict(out_token_stride=12), "out strides"), ("ring_paged_attention_fwd", dict(v_cache=None), "v_cache"),
    ("ring_paged_attention_fwd", dict(tokens=1 << 30, heads=4), "2^31"),
    ("ring_paged_weights", dict(weights=None), "null weights"), ("ring_paged_weights", dict(weights_len=10), "weights_len"),
    ("ring_paged_weights", dict(weights_head_stride=-1), "negative"), ("ring_paged_weights", dict(lse=None), "lse"),
    ("ring_paged_weights", dict(window=8, causal=0), "causal"),
])
def test_paged_calls_refuse(lib, fn, kw, needle):
    p = paged(**kw)
    assert getattr(lib, fn)(ctypes.byref(p)) == _lib.RING_ERR_INVALID_ARGUMENT
    assert needle in lib.ring_last_error_string().decode()


@pytest.mark.parametrize("kw,needle", [
    (dict(budget=0), "budget"), (dict(first=-1), "first"), (dict(first=20, recent=13), "at most budget"), (dict(budget=33, new_weights_len=33), "dst_table"),
    (dict(dst_table=None), "dst_table"), (dict(dst_stride=1), "dst_stride"), (dict(dst_table=0x3000), "pages of its own"),
    (dict(new_weights=0xa000), "must not be weights"), (dict(kept=None), "kept"), (dict(new_lens=0x4000), "kv_lens"),
    (dict(weights_len=63), "weights_len"), (dict(new_weights_len=31), "new_weights_len"), (dict(v_place_stride=0), "strides of 0"),
    (dict(v_cache=None), "v_cache"), (dict(recent=(1 << 31) - 1, first=2), "at most budget"),
    (dict(budget=(1 << 30) + 1, dst_pages=1 << 27, dst_stride=1 << 27, new_weights_len=(1 << 31) - 1), "2^30"),
    (dict(new_weights_len=(1 << 31) - 1), "2^30"),
])
def test_evict_refuses(lib, kw, needle):
    p = evict(**kw)
    assert lib.ring_paged_evict(ctypes.byref(p)) == _lib.RING_ERR_INVALID_ARGUMENT
    assert needle in lib.ring_last_error_string().decode()


@pytest.mark.parametrize("fn,kw,needle", [
    ("ring_paged_append", dict(weights_batch_stride=0), "weights overlap"), ("ring_paged_append", dict(weights_head_stride=63), "weights overlap"),
    ("ring_paged_weights", dict(weights_batch_stride=63), "weights overlap"), ("ring_paged_weights", dict(weights_head_stride=0), "weights overlap"),
    ("ring_paged_attention_fwd", dict(out_token_stride=0), "out overlap"), ("ring_paged_attention_fwd", dict(out_head_stride=56), "out overlap"),
    ("ring_paged_evict", dict(new_weights_batch_stride=0), "new_weights overlap"), ("ring_paged_evict", dict(new_weights_head_stride=31), "new_weights overlap"),
])
def test_results_in_one_memory_are_refused(lib, fn, kw, needle):
    p = evict(**kw) if fn == "ring_paged_evict" else paged(**kw)
    assert getattr(lib, fn)(ctypes.byref(p)) == _lib.RING_ERR_INVALID_ARGUMENT
    assert needle in lib.ring_last_error_string().decode()


def test_null_params_and_workspace(lib):
    for fn in ("ring_paged_append", "ring_paged_attention_fwd", "ring_paged_weights", "ring_paged_evict", "ring_paged_attention_workspace",
               "ring_paged_weights_workspace"):
        assert getattr(lib, fn)(None) == _lib.RING_ERR_INVALID_ARGUMENT
    assert lib.ring_paged_attention_workspace(ctypes.byref(paged(dim=32))) == _lib.RING_ERR_INVALID_ARGUMENT


def test_calls_without_tokens_do_nothing(lib):
    p = paged(tokens=0)
    for fn in ("ring_paged_append", "ring_paged_attention_fwd", "ring_paged_weights"):
        assert getattr(lib, fn)(ctypes.byref(p)) == _lib.RING_OK


def test_front_ends_refuse_cpu_tensors():
    import ringattention_b200 as ra
    from ringattention_b200 import torch_ops
    lib_build.build_torch_ext()
    c = torch.zeros((4, 2, 16, 64), dtype=torch.float16)
    t, n = torch.zeros((1, 4), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    q = torch.zeros((1, 4, 64), dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        torch_ops.paged_attention(q, c, c, t, n)
    with pytest.raises(RuntimeError, match="float16 or bfloat16"):
        torch_ops.paged_attention(q, c.float(), c.float(), t, n)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        torch_ops.paged_append(q[:, :2], q[:, :2], c, c, t, n)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        torch_ops.paged_evict(c, c, torch.zeros((1, 2, 64)), t, n, t, 16)
    with pytest.raises(ValueError, match="CUDA tensor"):
        ra.paged_attention_fwd(q, c, c, t, n, q, torch.zeros((1, 4)))
    with pytest.raises(ValueError, match="CUDA tensor"):
        ra.paged_append(q[:, :2], q[:, :2], c, c, t, n)
    with pytest.raises(ValueError, match="CUDA tensor"):
        ra.paged_weights(torch.zeros((1, 2, 64)), q, c, torch.zeros((1, 4)), t, n)
    with pytest.raises(ValueError, match="CUDA tensor"):
        ra.paged_evict(c, c, torch.zeros((1, 2, 64)), t, n, t, 16, n, torch.zeros((1, 2, 16)), torch.zeros((1, 2, 16), dtype=torch.int32))
