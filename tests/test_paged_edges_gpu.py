"""Paged-cache operators where a kernel's form, a mask or a limit changes: against the 64-bit statement of tests/paged_util.py, or
exactly where the definition gives an exact value."""
import math

import pytest
import torch

from tests.paged_util import Setup, attention_ref, check_attention, visible, weights_ref

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
    return ops.paged_attention(s.q, s.k_cache, s.v_cache, s.table, s.kv_lens, cu_seqlens=s.cu, max_new=s.max_new, **kw)


def weigh(ops, s, weights, lse, q=None, **kw):
    ops.paged_weights_(weights, s.q if q is None else q, s.k_cache, lse, s.table, s.kv_lens, cu_seqlens=s.cu, max_new=s.max_new, **kw)
    return weights


# lens, news, what differs from Setup's defaults: the first two with few query rows, the others with many
TRACKED = {
    "rows_g4_d128": ([700, 300], [6, 3], dict(group=4, dim=128, dtype="bf16")),
    "rows_g1_d64": ([700, 300], [20, 3], dict(group=1)),
    "chunk_g1_d64": ([700, 300], [150, 90], dict(group=1, dtype="bf16")),
    "chunk_g4_d128": ([700, 300], [150, 90], dict(group=4, dim=128, dtype="bf16", page=64)),
    "chunk_g7_d128": ([515, 40], [131, 40], dict(group=7, kv_heads=1, layout="NHD", page=32, dim=128)),
    "chunk_g40_d64": ([700], [30], dict(kv_heads=1, group=40, page=128)),
    "chunk_cut_units": ([9000], [2000], dict(kv_heads=1, group=1, page=64)),
}


@pytest.mark.parametrize("name", TRACKED)
@pytest.mark.parametrize("sinks", [0, 5])
def test_weights_of_places_nobody_sees_stay_zero(ops, name, sinks):
    """Left of every window the definition adds 0, and eviction ranks equal weights by place: not even 2^-126 may be added there."""
    lens, news, kw = TRACKED[name]
    s = Setup(lens, news, seed=40 + sinks, **kw)
    s.weights.zero_()
    m = dict(window=33, sinks=sinks)
    lse = attention_ref(s, **m)[1].float().cuda()
    want, tol = weights_ref(s, lse, **m)
    got = weigh(ops, s, s.weights.clone(), lse, **m).cpu()
    seen = torch.zeros(got.shape, dtype=torch.bool)
    for b in range(s.batch):
        seen[b, :, :lens[b]] = visible(lens[b], news[b], True, 33, sinks).any(dim=0)
    assert bool((~seen[:, :, :max(lens)]).any())
    assert bool((got[~seen].view(torch.int32) == 0).all()), got[~seen].max().item()
    assert bool(((got.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("name", TRACKED)
def test_rows_without_lse_add_nothing(ops, name):
    """A window of one place: token i gives its weight to its own place alone, and none at all if its lse is -inf."""
    lens, news, kw = TRACKED[name]
    s = Setup(lens, news, seed=43, **kw)
    s.weights.zero_()
    lse = attention_ref(s, window=1)[1].float().cuda()
    off = torch.arange(s.tokens) % 3 == 1
    lse[off.cuda()] = -math.inf
    got = weigh(ops, s, s.weights.clone(), lse, window=1).cpu()
    for b in range(s.batch):
        w = got[b, :, lens[b] - news[b]:lens[b]]
        skip = off[s.cu_list[b]:s.cu_list[b + 1]]
        assert bool((w[:, skip].view(torch.int32) == 0).all())
        # each of the group's heads gives its only place exp(s - lse) = 1: s is off by 2 (dim + 3) half steps of its terms' sizes
        # (2 * 131 * 2^-24 * 20 = 3.2e-4 at most), lse and its product with log2 e by 2^-22 of at most 20
        assert bool(((w[:, ~skip] / s.group - 1).abs() <= 1e-3).all())


@pytest.mark.parametrize("name", ["rows_g1_d64", "chunk_g1_d64", "chunk_g4_d128", "chunk_g7_d128"])
@pytest.mark.parametrize("where", ["q", "lse", "q and lse"])
def test_weights_keep_a_nan_row_visible(ops, name, where):
    """A NaN query row, or a NaN lse, makes every place that its token sees NaN, and no other, whichever column of a tile it is."""
    lens, news, kw = TRACKED[name]
    s = Setup(lens, news, seed=44, **kw)
    lse = attention_ref(s)[1].float().cuda()
    heads = s.kv_heads * s.group
    for i in range(8):
        tok, head = min(9 + i, news[0] - 1), (3 * i) % heads
        q, l = s.q.clone(), lse.clone()
        if "q" in where:
            q[tok, head, i] = math.nan
        if "lse" in where:
            l[tok, head] = math.nan
        got = weigh(ops, s, s.weights.clone(), l, q=q).cpu()
        want = torch.zeros(got.shape, dtype=torch.bool)
        want[0, head // s.group, :lens[0] - news[0] + tok + 1] = True
        assert torch.equal(torch.isnan(got), want), (tok, head)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("back", [1, 5, 127, 128, 129, 300])
def test_windows_of_lengths_near_the_end_of_32_bits(ops, new, dim, back):
    """A length far behind what the table's pages hold: the window lies where no places are, and only the first tokens are seen."""
    s = Setup([40, 40], [new, new], dim=dim, extra_cols=0, ragged=False, page=8, seed=back)
    s.kv_lens[0] = (1 << 31) - back
    for sinks in (0, 2):
        m = dict(window=30, sinks=sinks)
        out, lse = (x.cpu() for x in attend(ops, s, **m))
        got = weigh(ops, s, s.weights.clone(), lse.cuda(), **m).cpu()
        t = Setup([sinks, 40], [new, new], dim=dim, ragged=False, page=8)
        t.q, t.k_cache, t.v_cache, t.table, t.weights, t.pages = s.q, s.k_cache, s.v_cache, s.table, s.weights, s.pages
        # sequence 0 as one of `sinks` places that all its tokens see, sequence 1 with its own mask
        far, near = attention_ref(t, causal=False), attention_ref(t, **m)
        want = [torch.cat([f[:new], n[new:]]) for f, n in zip(far, near)]
        check_attention(t, (out, lse), want, what=f"{sinks}")
        wf, tf = weights_ref(t, lse, causal=False)
        wn, tn = weights_ref(t, lse, **m)
        err = torch.cat([(got.double() - wf).abs()[:1] / tf[:1], (got.double() - wn).abs()[1:] / tn[1:]])
        assert bool((err <= 1).all()), f"{sinks}: {err.max():.2f} times the bound"
        if sinks == 0:
            assert torch.equal(got[0], s.weights[0].cpu())
