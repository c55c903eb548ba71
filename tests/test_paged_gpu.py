"""Paged-cache operators (append, attention, weights, evict) against the plain 64-bit statement of tests/paged_util.py."""
import math

import pytest
import torch

from tests.paged_util import Setup, attention_ref, check_attention, evict_ref, weights_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from ringattention_b200 import build, torch_ops
    build.build_torch_ext()
    torch_ops._load()
    return torch_ops


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    import ringattention_b200 as ra
    yield
    assert ra.device_status() == 0


def attend(ops, s, **kw):
    return ops.paged_attention(s.q, s.k_cache, s.v_cache, s.table, s.kv_lens, cu_seqlens=s.cu, max_new=kw.pop("max_new", s.max_new), **kw)


# lens, news, then what differs from Setup's defaults
CASES = {
    "one_place": ([1], [1], {}),
    "decode_lengths": ([1, 2, 7, 8, 9, 63, 64, 65, 127, 128, 129, 200], [1] * 12, dict(ragged=False, page=8)),
    "decode_d128_g4": ([1000, 333, 5], [1, 1, 1], dict(dim=128, kv_heads=2, group=4, dtype="bf16", ragged=False)),
    "decode_nhd_g8": ([517, 1200], [1, 1], dict(dim=128, kv_heads=1, group=8, layout="NHD", page=64)),
    "decode_g16": ([700], [1], dict(kv_heads=2, group=16, page=32)),
    "decode_g40": ([300], [1], dict(kv_heads=1, group=40, dim=128, page=256)),
    "idle_slots": ([0, 40, 0, 300], [1, 1, 1, 1], dict(ragged=False)),
    "nothing_new_for_some": ([50, 40, 0, 130], [0, 3, 0, 2], dict(group=3)),
    "more_new_than_places": ([3, 2], [5, 4], {}),
    "few_tokens_g5": ([100, 256, 61], [4, 1, 7], dict(group=5, dtype="bf16", dim=128)),
    "prompt_g1": ([130, 257], [130, 257], dict(group=1, kv_heads=3, page=64)),
    "chunk_g4_d128": ([700, 300, 129], [150, 64, 129], dict(group=4, dim=128, dtype="bf16", page=128)),
    "chunk_g7": ([515, 40], [131, 40], dict(group=7, kv_heads=1, layout="NHD", page=32, dim=128)),
    "chunk_g40": ([300, 90], [30, 11], dict(kv_heads=1, group=40, dtype="bf16")),
    "chunk_g130": ([200], [3], dict(kv_heads=1, group=130, page=32)),
    "long_chunk": ([5000, 1300], [700, 33], dict(kv_heads=1, group=2, page=64, dtype="bf16")),
    "one_head_one_page": ([300], [100], dict(kv_heads=1, group=1, page=512, spare_pages=0, extra_cols=0, dtype="bf16")),
    "many_sequences_one_long": ([740] + [(13 * i) % 60 for i in range(44)], [700] + [(13 * i) % 60 % 7 for i in range(44)],
                                dict(kv_heads=1, group=2, page=16)),
    "page_above_tile": ([900, 513], [70, 200], dict(group=2, page=512, dim=128)),
}


@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("mask", ["causal", "full", "window", "window_sinks"])
def test_attention(ops, name, mask):
    lens, news, kw = CASES[name]
    s = Setup(lens, news, seed=len(name), **kw)
    m = {"causal": {}, "full": dict(causal=False), "window": dict(window=33), "window_sinks": dict(window=64, sinks=5)}[mask]
    got = attend(ops, s, **m)
    check_attention(s, got, attention_ref(s, **m), what=f"{name} {mask}")


@pytest.mark.parametrize("name", ["decode_d128_g4", "few_tokens_g5", "chunk_g4_d128", "prompt_g1"])
def test_attention_fp32_out_scale_and_hint(ops, name):
    lens, news, kw = CASES[name]
    s = Setup(lens, news, seed=3, **kw)
    got = attend(ops, s, fp32_out=True, softmax_scale=0.2)
    assert got[0].dtype == torch.float32
    want = attention_ref(s, scale=0.2)
    check_attention(s, got, want, out_type=torch.float32, what=name)
    for hint in (1, 0, 10_000):  # a wrong hint chooses another kernel, not another result
        check_attention(s, attend(ops, s, fp32_out=True, softmax_scale=0.2, max_new=hint), want, out_type=torch.float32, what=f"{name} {hint}")


@pytest.mark.parametrize("name", ["decode_d128_g4", "few_tokens_g5", "chunk_g7"])
def test_attention_extreme_masks(ops, name):
    """Windows and first tokens beyond any sequence are no mask; a window of one place and no first tokens is the token itself."""
    lens, news, kw = CASES[name]
    s = Setup(lens, news, seed=13, **kw)
    want = attention_ref(s)
    for m in (dict(window=(1 << 31) - 1), dict(window=1, sinks=(1 << 31) - 1), dict(window=1 << 30, sinks=7)):
        check_attention(s, attend(ops, s, **m), want, what=str(m))
        lse = want[1].float().cuda()
        w, tol = weights_ref(s, lse)
        got = s.weights.clone()
        ops.paged_weights_(got, s.q, s.k_cache, lse, s.table, s.kv_lens, cu_seqlens=s.cu, max_new=s.max_new, **m)
        assert bool(((got.cpu().double() - w).abs() <= tol).all())
    check_attention(s, attend(ops, s, window=1), attention_ref(s, window=1))


@pytest.mark.parametrize("name", ["decode_d128_g4", "chunk_g4_d128"])
def test_keys_and_values_laid_out_differently(ops, name):
    lens, news, kw = CASES[name]
    s = Setup(lens, news, seed=14, **kw)
    v = torch.empty((s.pages, s.page, s.kv_heads, s.dim), dtype=s.dtype, device="cuda").transpose(1, 2)
    v.copy_(s.v_cache)
    got = ops.paged_attention(s.q, s.k_cache, v, s.table, s.kv_lens, cu_seqlens=s.cu, max_new=s.max_new)
    check_attention(s, got, attention_ref(s))


@pytest.mark.parametrize("name", ["decode_d128_g4", "chunk_g4_d128"])
def test_attention_large_scores_and_growing_maximum(ops, name):
    lens, news, kw = CASES[name]
    s = Setup(lens, news, seed=4, gain=3.0, **kw)
    # the last places hold the largest keys, so the running maximum keeps growing
    s.k_cache.mul_(torch.linspace(0.1, 2.0, s.pages, device="cuda").to(s.dtype)[:, None, None, None])
    check_attention(s, attend(ops, s), attention_ref(s), what=name)


@pytest.mark.parametrize("name", ["decode_d128_g4", "few_tokens_g5", "chunk_g4_d128", "chunk_g7", "page_above_tile"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_unseen_places_may_hold_anything(ops, name, bad):
    """Behind the length, in pages nobody names, in front of every window: no value there reaches a result."""
    lens, news, kw = CASES[name]
    s = Setup(lens, news, seed=5, **kw)
    m = dict(window=40, sinks=3)
    want = attention_ref(s, **m)
    for b in range(s.batch):
        first = s.lens[b] - s.news[b] - 40 + 1
        for i in range(s.table.shape[1]):
            pg = int(s.table[b, i])
            if pg < 0:
                continue
            for c in (s.k_cache, s.v_cache):
                for slot in range(s.page):
                    j = i * s.page + slot
                    if j >= s.lens[b] or (j < first and j >= 3):
                        c[pg, :, slot] = bad
    for pg in s.free:
        s.k_cache[pg] = bad
        s.v_cache[pg] = bad
    check_attention(s, attend(ops, s, **m), want, what=name)


@pytest.mark.parametrize("name", ["decode_lengths", "few_tokens_g5", "chunk_g4_d128", "chunk_g7", "page_above_tile"])
@pytest.mark.parametrize("wrong", [-1, 1 << 30, -(1 << 31)])
def test_pages_that_do_not_exist_hold_no_places(ops, name, wrong):
    lens, news, kw = CASES[name]
    s = Setup(lens, news, seed=6, **kw)
    s.table[0, 0] = wrong
    if s.table.shape[1] > 3:
        s.table[-1, 2] = wrong
        s.table[0, 3] = s.pages
    got = attend(ops, s)
    check_attention(s, got, attention_ref(s), what=name)
    w, tol = weights_ref(s, got[1])
    ops.paged_weights_(s.weights, s.q, s.k_cache, got[1], s.table, s.kv_lens, cu_seqlens=s.cu, max_new=s.max_new)
    assert bool(((s.weights.cpu().double() - w).abs() <= tol).all())


@pytest.mark.parametrize("new", [1, 40])
def test_places_behind_the_table_do_not_exist(ops, new):
    s = Setup([40, 40], [new, new], extra_cols=0, ragged=False, page=8)
    s.kv_lens[0] = (1 << 31) - 1
    s.kv_lens[1] = -5
    got = attend(ops, s)
    s.lens = [s.table.shape[1] * s.page, 0]
    check_attention(s, got, attention_ref(s, causal=False) if new > 1 else attention_ref(s))
    # new tokens whose places do not exist go nowhere, those in front of them to their own
    s.kv_lens[0] = 45
    k, v, w = s.k_cache.clone(), s.v_cache.clone(), s.weights.clone()
    for i in range(new):
        j = 45 - new + i
        if j < 40:
            pg = int(s.table[0, j // 8])
            k[pg, :, j % 8], v[pg, :, j % 8], w[0, :, j] = s.k_new[i], s.v_new[i], 0.0
    ops.paged_append(s.k_new, s.v_new, s.k_cache, s.v_cache, s.table, s.kv_lens, weights=s.weights)
    assert torch.equal(k, s.k_cache) and torch.equal(v, s.v_cache) and torch.equal(w, s.weights)
    got = attend(ops, s, window=30, sinks=2)
    p = torch.arange(new)[:, None] + 45 - new
    j = torch.arange(40)[None]
    see = (j <= p) & ((j > p - 30) | (j < 2))
    for h in range(4):
        x = s.q[:new, h].cpu().double() @ s.rows(s.k_cache, 0, h // 2)[0].T / 8.0
        want = torch.softmax(x.masked_fill(~see, -math.inf), dim=1) @ s.rows(s.v_cache, 0, h // 2)[0]
        # fp16: P and out by half a step each, scores as in check_attention, all below 2^-9 of the largest |v|
        assert float((got[0][:new, h].cpu().double() - want).abs().max()) <= 2.0 ** -9 * float(s.v_cache.abs().max())


def test_two_threads_share_a_stream(ops):
    """Calls from two host threads on one stream: every call has scratch of its own."""
    import threading
    s, t = Setup([700], [1], dim=128, group=4, ragged=False), Setup([900, 300], [200, 90], dim=128, group=4, seed=2)
    want = [attend(ops, s), attend(ops, t)]
    stream, bad = torch.cuda.current_stream(), []

    def work(x, w):
        try:
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got = attend(ops, x)
                    if not (torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])):
                        bad.append("differs")
        except Exception as e:  # an exception ends the thread, not the test
            bad.append(repr(e))

    threads = [threading.Thread(target=work, args=a) for a in ((s, want[0]), (t, want[1]))]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not bad


def test_first_call_of_a_host_thread(ops):
    """A new thread's first CUDA call of any kind is one of these (no context is current in it yet)."""
    import threading
    from ringattention_b200 import torch_ops
    s = Setup([900, 300], [200, 90], dim=128, group=4, seed=2)
    out, lse = attend(ops, s)
    w = s.weights.clone()
    ops.paged_weights_(w, s.q, s.k_cache, lse, s.table, s.kv_lens, cu_seqlens=s.cu, max_new=s.max_new)
    q = torch.randn((1, 2, 256, 128), device="cuda").half()
    whole = torch_ops.block_forward(q, q, q)
    torch.cuda.synchronize()
    got = {}

    def run(name, f):
        try:
            got[name] = f()
        except Exception as e:
            got[name] = e

    calls = {"attention": lambda: attend(ops, s), "block": lambda: torch_ops.block_forward(q, q, q),
             "weights": lambda: ops.paged_weights_(s.weights, s.q, s.k_cache, lse, s.table, s.kv_lens, cu_seqlens=s.cu, max_new=s.max_new)}
    for name, f in calls.items():
        th = threading.Thread(target=run, args=(name, f))
        th.start()
        th.join()
    torch.cuda.synchronize()
    assert not [v for v in got.values() if isinstance(v, Exception)], got
    assert torch.equal(got["attention"][0], out) and torch.equal(got["block"][0], whole[0]) and torch.equal(s.weights, w)


def test_strided_operands(ops):
    """q, k, v as slices of one projection, the cache as a slice of a larger one, tables with columns to spare."""
    s = Setup([70, 20], [3, 2], group=2, kv_heads=2, dim=64)
    qkv = torch.zeros((s.tokens, 4 + 2 + 2, 64 + 8), dtype=s.dtype, device="cuda")
    qkv[:, :4, :64], qkv[:, 4:6, :64], qkv[:, 6:, :64] = s.q, s.k_new, s.v_new
    q, k, v = qkv[:, :4, :64], qkv[:, 4:6, :64], qkv[:, 6:, :64]
    both = torch.zeros((s.pages, 2, s.kv_heads, s.page, 64), dtype=s.dtype, device="cuda")
    both[:, 0], both[:, 1] = s.k_cache, s.v_cache
    table = torch.full((2, 32), 77, dtype=torch.int32, device="cuda")
    table[:, :s.table.shape[1]] = s.table
    view = table[:, :s.table.shape[1]]
    ops.paged_append(k, v, both[:, 0], both[:, 1], view, s.kv_lens, cu_seqlens=s.cu)
    ops.paged_append(s.k_new, s.v_new, s.k_cache, s.v_cache, s.table, s.kv_lens, cu_seqlens=s.cu)
    assert torch.equal(both[:, 0], s.k_cache) and torch.equal(both[:, 1], s.v_cache)
    got = ops.paged_attention(q, both[:, 0], both[:, 1], view, s.kv_lens, cu_seqlens=s.cu, max_new=3)
    check_attention(s, got, attention_ref(s))


@pytest.mark.parametrize("name", ["decode_d128_g4", "chunk_g4_d128"])
def test_rows_outside_the_sequences_stay_and_reruns_are_equal(ops, name):
    import ringattention_b200 as ra
    lens, news, kw = CASES[name]
    s = Setup(lens, news, seed=8, **{**kw, "ragged": True})
    pad = 5
    q = torch.cat([s.q, torch.full_like(s.q[:pad], math.nan)])
    results = []
    for _ in range(3):
        out = torch.full(q.shape, 7.0, dtype=s.dtype, device="cuda")
        lse = torch.full(q.shape[:2], 7.0, device="cuda")
        ra.paged_attention_fwd(q, s.k_cache, s.v_cache, s.table, s.kv_lens, out, lse, cu_seqlens=s.cu, max_new=s.max_new)
        results.append((out, lse))
    out, lse = results[0]
    assert bool((out[s.tokens:] == 7).all()) and bool((lse[s.tokens:] == 7).all())
    check_attention(s, (out[:s.tokens], lse[:s.tokens]), attention_ref(s), what=name)
    for o, l in results[1:]:
        assert torch.equal(o, out) and torch.equal(l, lse)


def test_partials_of_two_caches_join(ops):
    """Two ranks that each hold a part of a sequence's places: fp32 partials and lse_merge_ give the whole."""
    s = Setup([300, 150], [1, 1], dim=128, group=4, page=16, ragged=False)
    whole = attention_ref(s, causal=False)
    cut = 8  # pages of the first part
    a = ops.paged_attention(s.q, s.k_cache, s.v_cache, s.table[:, :cut].contiguous(), s.kv_lens.clamp(max=cut * 16), causal=False, fp32_out=True)
    b = ops.paged_attention(s.q, s.k_cache, s.v_cache, s.table[:, cut:].contiguous(), (s.kv_lens - cut * 16).clamp(min=0), causal=False, fp32_out=True)
    ops.lse_merge_(a[0], a[1], b[0], b[1])
    check_attention(s, a, whole, out_type=torch.float32)


@pytest.mark.parametrize("dim,kv_heads,dtype", [(64, 1, "fp16"), (64, 5, "bf16"), (128, 3, "fp16"), (128, 20, "bf16")])
@pytest.mark.parametrize("ragged", [False, True])
def test_append(ops, dim, kv_heads, dtype, ragged):
    lens, news = ([33, 7, 0, 100], [2, 2, 2, 2]) if not ragged else ([33, 7, 0, 100, 5], [33, 0, 3, 17, 9])
    s = Setup(lens, news, dim=dim, kv_heads=kv_heads, group=1, dtype=dtype, ragged=ragged, page=8, layout="NHD" if dim == 64 else "HND")
    s.table[0, 1] = -1
    k, v, w = s.k_cache.clone(), s.v_cache.clone(), s.weights.clone()
    for b in range(s.batch):
        for i in range(s.news[b]):
            j = s.lens[b] - s.news[b] + i
            if j < 0 or int(s.table[b, j // 8]) < 0:
                continue
            pg = int(s.table[b, j // 8])
            k[pg, :, j % 8], v[pg, :, j % 8], w[b, :, j] = s.k_new[s.cu_list[b] + i], s.v_new[s.cu_list[b] + i], 0.0
    pad = torch.cat([s.k_new, s.k_new[:3]]) if ragged else s.k_new  # rows behind the last sequence go nowhere
    padv = torch.cat([s.v_new, s.v_new[:3]]) if ragged else s.v_new
    ops.paged_append(pad, padv, s.k_cache, s.v_cache, s.table, s.kv_lens, cu_seqlens=s.cu, weights=s.weights)
    assert torch.equal(k, s.k_cache) and torch.equal(v, s.v_cache) and torch.equal(w, s.weights)


def test_append_many_sequences(ops):
    """More sequences than one step of the search over cu_seqlens covers, empty ones among them."""
    news = [(7 * i) % 4 for i in range(1500)]
    s = Setup([n + 1 for n in news], news, kv_heads=1, group=1, page=8, extra_cols=0)
    seq = torch.repeat_interleave(torch.arange(1500), torch.tensor(news))
    idx = torch.arange(s.tokens) - torch.tensor(s.cu_list)[seq]
    k = s.k_cache.clone()
    pg = s.table.cpu()[seq, 0].long().cuda()
    k[pg, :, (idx + 1).cuda()] = s.k_new
    ops.paged_append(s.k_new, s.v_new, s.k_cache, s.v_cache, s.table, s.kv_lens, cu_seqlens=s.cu)
    assert torch.equal(k, s.k_cache)
    check = ops.paged_attention(s.q, s.k_cache, s.v_cache, s.table, s.kv_lens, cu_seqlens=s.cu, max_new=3)
    check_attention(s, check, attention_ref(s))


@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("mask", ["causal", "full", "window_sinks"])
def test_weights(ops, name, mask):
    lens, news, kw = CASES[name]
    s = Setup(lens, news, seed=20 + len(name), **kw)
    m = {"causal": {}, "full": dict(causal=False), "window_sinks": dict(window=64, sinks=5)}[mask]
    lse = attention_ref(s, **m)[1].float().cuda()
    want, tol = weights_ref(s, lse, **m)
    first = s.weights.clone()
    ops.paged_weights_(s.weights, s.q, s.k_cache, lse, s.table, s.kv_lens, cu_seqlens=s.cu, max_new=s.max_new, **m)
    err = (s.weights.cpu().double() - want).abs()
    assert bool((err <= tol).all()), f"{name} {mask}: {(err / tol).max():.2f} times the bound"
    again = first
    ops.paged_weights_(again, s.q, s.k_cache, lse, s.table, s.kv_lens, cu_seqlens=s.cu, max_new=s.max_new, **m)
    assert torch.equal(again, s.weights)  # the same bits again


@pytest.mark.parametrize("name", ["decode_d128_g4", "few_tokens_g5", "chunk_g4_d128", "nothing_new_for_some"])
@pytest.mark.parametrize("hint", [1, 3, 0])
def test_weights_hint(ops, name, hint):
    lens, news, kw = CASES[name]
    s = Setup(lens, news, seed=31, **kw)
    lse = attention_ref(s)[1].float().cuda()
    want, tol = weights_ref(s, lse)
    ops.paged_weights_(s.weights, s.q, s.k_cache, lse, s.table, s.kv_lens, cu_seqlens=s.cu, max_new=hint)
    assert bool(((s.weights.cpu().double() - want).abs() <= tol).all())


@pytest.mark.parametrize("name", ["few_tokens_g5", "chunk_g4_d128", "chunk_g7"])
def test_weights_ignore_unseen_places(ops, name):
    lens, news, kw = CASES[name]
    s = Setup(lens, news, seed=9, **kw)
    lse = attention_ref(s)[1].float().cuda()
    want, tol = weights_ref(s, lse)
    for b in range(s.batch):
        pg, slot = int(s.table[b, s.lens[b] // s.page]) if s.lens[b] % s.page else -1, s.lens[b] % s.page
        if pg >= 0:
            s.k_cache[pg, :, slot:] = math.nan
    for pg in s.free:
        s.k_cache[pg] = math.nan
    q = torch.cat([s.q, torch.full_like(s.q[:9], math.nan)])  # rows behind the last sequence
    lse = torch.cat([lse, torch.full_like(lse[:9], math.nan)])
    ops.paged_weights_(s.weights, q, s.k_cache, lse, s.table, s.kv_lens, cu_seqlens=s.cu, max_new=s.max_new)
    assert bool(((s.weights.cpu().double() - want).abs() <= tol).all())


EVICT = [  # lens, budget, first, recent
    ([100], 64, 4, 16), ([64, 65, 0, 1, 130], 64, 0, 0), ([500, 63], 100, 1, 99), ([5000, 4097, 9000], 4096, 4, 1000),
    ([300], 299, 0, 0), ([300, 200], 1, 0, 0), ([300], 17, 0, 17), ([70000], 33000, 4, 2048),
]


@pytest.mark.parametrize("kind", ["heavy", "ties", "odd"])
@pytest.mark.parametrize("lens,budget,first,recent", EVICT)
def test_evict(ops, lens, budget, first, recent, kind):
    dim = 128 if len(lens) % 2 else 64
    s = Setup(lens, [0] * len(lens), dim=dim, kv_heads=2, page=32, spare_pages=len(lens) * -(-budget // 32) + 2,
              layout="NHD" if len(lens) > 2 else "HND", seed=budget)
    g = torch.Generator().manual_seed(7)
    w = torch.rand(s.weights.shape, generator=g)
    if kind == "heavy":
        w = 0.001 / (1.0001 - w)
    elif kind == "ties":
        w = (w * 4).floor() / 4
    else:  # values that an accumulated weight should not have: ordered all the same
        w = torch.where(w < 0.1, torch.full_like(w, math.nan), torch.where(w < 0.2, torch.full_like(w, math.inf), w - 0.5))
        w = torch.where((w > 0.4) & (w < 0.45), torch.full_like(w, -0.0), torch.where(w > 0.45, torch.zeros_like(w), w))
    s.weights = w.cuda()
    cols = -(-budget // 32)
    dst = torch.tensor(s.free[:len(lens) * cols], dtype=torch.int32).reshape(len(lens), cols)
    k, v = s.k_cache.clone(), s.v_cache.clone()
    new_lens, new_w, kept = ops.paged_evict(s.k_cache, s.v_cache, s.weights, s.table, s.kv_lens, dst.cuda(), budget, first=first, recent=recent)
    want = evict_ref(lens, w, budget, first, recent)
    assert new_lens.tolist() == [min(n, budget) for n in lens]
    table = s.table.cpu().long()
    for b in range(len(lens)):
        for h in range(2):
            m = min(lens[b], budget)
            assert kept[b, h, :m].tolist() == want[b][h] and bool((kept[b, h, m:] == -1).all())
            idx = torch.tensor(want[b][h], dtype=torch.long)
            assert torch.equal(new_w[b, h, :m].cpu().view(torch.int32), w[b, h, idx].view(torch.int32)) and bool((new_w[b, h, m:] == 0).all())
            at = torch.arange(m)
            src, to = table[b, idx // 32].cuda(), dst.long()[b, at // 32].cuda()
            k[to, h, (at % 32).cuda()] = k[src, h, (idx % 32).cuda()]
            v[to, h, (at % 32).cuda()] = v[src, h, (idx % 32).cuda()]
    assert torch.equal(k, s.k_cache) and torch.equal(v, s.v_cache)  # the new places, and nothing else


def test_evict_pages_that_do_not_exist(ops):
    s = Setup([100, 90], [0, 0], page=16, spare_pages=10)
    dst = torch.tensor(s.free[:8], dtype=torch.int32).reshape(2, 4)
    dst[0, 1], dst[1, 2] = -1, s.pages
    s.table[0, 0] = 1 << 30
    k = s.k_cache.clone()
    new_lens, _, kept = ops.paged_evict(s.k_cache, s.v_cache, s.weights, s.table, s.kv_lens, dst.cuda(), 64, first=16, recent=16)
    assert new_lens.tolist() == [64, 64]
    t = s.table.cpu().tolist()
    for b in range(2):
        for h in range(2):
            for j, i in enumerate(kept[b, h].tolist()):
                src, to = t[b][i // 16], int(dst[b, j // 16])
                if 0 <= src < s.pages and 0 <= to < s.pages:
                    k[to, h, j % 16] = k[src, h, i % 16]
    assert torch.equal(k, s.k_cache)


def test_places_beyond_32_bit_offsets(ops):
    """A cache of more than 2^31 elements, the sequences in its last pages."""
    s = Setup([200, 90], [2, 3], dim=128, kv_heads=8, group=2, page=128, seed=12)
    pages = (1 << 31) // (8 * 128 * 128) + 64
    big = torch.empty((pages, 8, 128, 128), dtype=s.dtype, device="cuda")
    big[pages - s.pages:] = s.k_cache
    table = torch.where(s.table >= 0, s.table + (pages - s.pages), s.table)
    s.v_cache = s.k_cache
    got = ops.paged_attention(s.q, big, big, table, s.kv_lens, cu_seqlens=s.cu, max_new=3)
    check_attention(s, got, attention_ref(s), what="rows")
    got = ops.paged_attention(s.q, big, big, table, s.kv_lens, cu_seqlens=s.cu, max_new=0)
    check_attention(s, got, attention_ref(s), what="no hint")
    w, tol = weights_ref(s, got[1])
    ops.paged_weights_(s.weights, s.q, big, got[1], table, s.kv_lens, cu_seqlens=s.cu, max_new=3)
    assert bool(((s.weights.cpu().double() - w).abs() <= tol).all())
    new = big.new_ones((s.tokens, 8, 128))
    ops.paged_append(new, new, big, big, table, s.kv_lens, cu_seqlens=s.cu)
    pg = int(table[0, 199 // 128])
    assert bool((big[pg, :, 199 % 128] == 1).all()) and not bool((big[pg, :, 197 % 128] == 1).all())


def test_a_run_of_them_together(ops):
    """Prompt, decoding steps, eviction, more steps: the cache, the weights and the answers follow a plain 64-bit model."""
    from tests.paged_util import visible
    torch.manual_seed(5)
    H, G, D, page, budget = 2, 2, 64, 16, 48
    pages = 40
    kc = torch.zeros((pages, H, page, D), dtype=torch.bfloat16, device="cuda")
    vc = torch.zeros_like(kc)
    width = 8
    tables = [torch.arange(i * 16, i * 16 + 16, dtype=torch.int32).reshape(2, 8) for i in range(2)]
    table, spare = tables[0].cuda(), tables[1].cuda()
    weights = torch.zeros((2, H, width * page), device="cuda")
    model = [[([], [], []) for _ in range(H)] for _ in range(2)]  # rows of k, of v, weights
    lens = [0, 0]
    for step, news in enumerate([(37, 50), (1, 1), (1, 1), "evict", (1, 1), (3, 2), "evict", (1, 0), (1, 1)]):
        if news == "evict":
            dst = spare[:, :-(-budget // page)]
            new_lens, new_w, kept = ops.paged_evict(kc, vc, weights, table, kv_lens, dst, budget, first=2, recent=8)
            want = evict_ref(lens, weights.cpu(), budget, 2, 8)
            for b in range(2):
                for h in range(H):
                    assert kept[b, h, :len(want[b][h])].tolist() == want[b][h]
                    model[b][h] = tuple([x[i] for i in want[b][h]] for x in model[b][h])
            lens = [min(n, budget) for n in lens]
            assert new_lens.tolist() == lens
            weights = torch.zeros_like(weights)
            weights[:, :, :new_w.shape[2]] = new_w
            table, spare = spare, table
            continue
        cu = [0, news[0], news[0] + news[1]]
        lens = [a + n for a, n in zip(lens, news)]
        kv_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        cut = torch.tensor(cu, dtype=torch.int32, device="cuda")
        q = torch.randn((cu[2], H * G, D)).bfloat16()
        k, v = torch.randn((cu[2], H, D)).bfloat16(), torch.randn((cu[2], H, D)).bfloat16()
        args = dict(cu_seqlens=cut, max_new=max(news))
        ops.paged_append(k.cuda(), v.cuda(), kc, vc, table, kv_lens, cu_seqlens=cut, weights=weights)
        out, lse = ops.paged_attention(q.cuda(), kc, vc, table, kv_lens, **args)
        ops.paged_weights_(weights, q.cuda(), kc, lse, table, kv_lens, **args)
        for b in range(2):
            for h in range(H):
                mk, mv, mw = model[b][h]
                for t in range(cu[b], cu[b + 1]):
                    mk.append(k[t, h].double()), mv.append(v[t, h].double()), mw.append(0.0)
                if cu[b] == cu[b + 1]:
                    continue
                K, V = torch.stack(mk), torch.stack(mv)
                see = visible(len(mk), news[b], True, 0, 0)
                for g in range(G):
                    x = (q[cu[b]:cu[b + 1], h * G + g].double() @ K.T * D ** -0.5).masked_fill(~see, -math.inf)
                    p = torch.softmax(x, dim=1)
                    got = out[cu[b]:cu[b + 1], h * G + g].cpu().double()
                    # two roundings to bf16 (P, out), each at most 2^-8 of sum p |v|, and 2^-12 for the 32-bit arithmetic
                    assert bool(((got - p @ V).abs() <= (2.0 ** -7 + 2.0 ** -12) * (p @ V.abs()) + 1e-6).all()), (step, b, h)
                    for j, add in enumerate(p.sum(dim=0).tolist()):
                        mw[j] += add
                got_w = weights[b, h, :lens[b]].cpu().double()
                # scores of 64 products within 2^-24 * 67 * sum |q k| < 2^-24 * 67 * 20, twice, and the 32-bit sums
                assert bool(((got_w - torch.tensor(mw)).abs() <= 5e-4 * torch.tensor(mw) + 1e-6).all()), (step, b, h)


def test_graph_capture_replay_and_overlapping_calls(ops):
    """Captured calls follow the lengths and tables their tensors hold at replay; calls on two streams do not meet."""
    s = Setup([100, 257], [1, 1], dim=128, group=4, dtype="bf16", ragged=False)
    t = Setup([400, 300], [90, 120], dim=128, group=4, dtype="bf16", seed=2)
    attend(ops, s), attend(ops, t)
    torch.cuda.synchronize()
    graphs = []
    for x in (s, t):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.paged_append(x.k_new, x.v_new, x.k_cache, x.v_cache, x.table, x.kv_lens, cu_seqlens=x.cu, weights=x.weights)
            out = attend(ops, x)
            ops.paged_weights_(x.weights, x.q, x.k_cache, out[1], x.table, x.kv_lens, cu_seqlens=x.cu, max_new=x.max_new)
        graphs.append((g, out))
    for lens in ([100, 257], [64, 130], [1, 2]):
        s.lens = lens
        s.kv_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        for _ in range(3):
            for (g, _), st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        for x, (_, out) in zip((s, t), graphs):
            check_attention(x, out, attention_ref(x), what=str(lens))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(attend(ops, (s, t)[i % 2]))
    torch.cuda.synchronize()
    for i in range(6):
        check_attention((s, t)[i % 2], outs[i], attention_ref((s, t)[i % 2]))


def test_plain_api_matches_front_end(ops):
    """The C-ABI functions of the package on a stream of the caller's, with its own workspace and strided outputs."""
    import ringattention_b200 as ra
    s = Setup([300, 77], [5, 40], dim=64, group=2, dtype="bf16")
    want = attend(ops, s)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    hold = torch.zeros((s.tokens, s.kv_heads * s.group, 2, s.dim), dtype=s.dtype, device="cuda")
    lse = torch.empty((s.tokens, s.kv_heads * s.group), device="cuda")
    n = ra.paged_attention_workspace(s.q, s.k_cache, s.table, cu_seqlens=s.cu, max_new=s.max_new)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for extra in (dict(), dict(workspace=ws)):
        hold.zero_()
        lse.zero_()
        torch.cuda.synchronize()
        ra.paged_attention_fwd(s.q, s.k_cache, s.v_cache, s.table, s.kv_lens, hold[:, :, 1], lse, cu_seqlens=s.cu, max_new=s.max_new,
                               stream=st, **extra)
        st.synchronize()
        assert torch.equal(hold[:, :, 1], want[0]) and torch.equal(lse, want[1]) and not bool(hold[:, :, 0].any())
    w1, w2 = s.weights.clone(), s.weights.clone()
    ops.paged_weights_(w1, s.q, s.k_cache, lse, s.table, s.kv_lens, cu_seqlens=s.cu, max_new=s.max_new)
    torch.cuda.synchronize()
    n = ra.paged_weights_workspace(s.q, s.k_cache, s.table, cu_seqlens=s.cu, max_new=s.max_new)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    ra.paged_weights(w2, s.q, s.k_cache, lse, s.table, s.kv_lens, cu_seqlens=s.cu, max_new=s.max_new, stream=st, workspace=ws)
    st.synchronize()
    assert torch.equal(w1, w2)
    k1, k2 = s.k_cache.clone(), s.k_cache.clone()
    v1, v2 = s.v_cache.clone(), s.v_cache.clone()
    ops.paged_append(s.k_new, s.v_new, k1, v1, s.table, s.kv_lens, cu_seqlens=s.cu)
    ra.paged_append(s.k_new, s.v_new, k2, v2, s.table, s.kv_lens, cu_seqlens=s.cu)
    assert torch.equal(k1, k2) and torch.equal(v1, v2)
    dst = torch.tensor(s.free[:2], dtype=torch.int32, device="cuda").reshape(2, 1)
    a = ops.paged_evict(k1, v1, w1, s.table, s.kv_lens, dst, 16, first=1, recent=3)
    b = [torch.empty_like(x) for x in a]
    ra.paged_evict(k2, v2, w1, s.table, s.kv_lens, dst, 16, b[0], b[1], b[2], first=1, recent=3)
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and torch.equal(k1, k2) and torch.equal(v1, v2)


def test_no_tokens_and_launch_counts(ops):
    import ringattention_b200 as ra
    s = Setup([20, 30], [0, 0])
    n = ra.kernel_launch_count()
    out, lse = attend(ops, s)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    ops.paged_append(s.k_new, s.v_new, s.k_cache, s.v_cache, s.table, s.kv_lens, cu_seqlens=s.cu)
    ops.paged_weights_(s.weights, s.q, s.k_cache, lse, s.table, s.kv_lens, cu_seqlens=s.cu)
    assert ra.kernel_launch_count() == n
