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


# The forms change at 9, 17 and 33 query rows a K/V head: (group, new tokens of the longest) on both sides of each, and between
FORM_ROWS = {8: (8, 1), 9: (3, 3), 16: (4, 4), 17: (1, 17), 24: (8, 3), 31: (1, 31), 32: (4, 8), 33: (3, 11)}


@pytest.mark.parametrize("rows", FORM_ROWS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_both_sides_of_every_choice_of_form(ops, rows, dim, dtype):
    """Units cut into few and into many partials, units of fewer rows, pages that do not exist, windows; attention and weights."""
    group, new = FORM_ROWS[rows]
    s = Setup([2900, 500, 64, 0], [new, max(new - 1, 1), 1, 0], dim=dim, dtype=dtype, group=group, page=16, seed=rows)
    s.table[0, 3], s.table[1, 30] = -1, s.pages
    for m in (dict(), dict(causal=False), dict(window=1200, sinks=40)):
        want = attention_ref(s, **m)
        got = attend(ops, s, **m)
        check_attention(s, got, want, what=str(m))
        lse = want[1].float().cuda()
        w, tol = weights_ref(s, lse, **m)
        once, again = weigh(ops, s, s.weights.clone(), lse, **m), weigh(ops, s, s.weights.clone(), lse, **m)
        assert bool(((once.cpu().double() - w).abs() <= tol).all()), str(m)
        repeat = attend(ops, s, **m)
        assert torch.equal(once, again) and torch.equal(got[0], repeat[0]) and torch.equal(got[1], repeat[1])


@pytest.mark.parametrize("rows", [16, 24, 32])
@pytest.mark.parametrize("dim,dtype", [(64, "fp16"), (64, "bf16"), (128, "bf16")])
def test_one_long_sequence_in_every_share(ops, rows, dim, dtype):
    group, new = FORM_ROWS[rows]
    s = Setup([40000], [new], dim=dim, dtype=dtype, group=group, kv_heads=1, page=64, layout="NHD", seed=rows)
    want = attention_ref(s)
    got = attend(ops, s)
    check_attention(s, got, want)
    w, tol = weights_ref(s, got[1])
    assert bool(((weigh(ops, s, s.weights.clone(), got[1]).cpu().double() - w).abs() <= tol).all())


@pytest.mark.parametrize("name", TRACKED)
def test_weights_with_a_window_and_no_first_tokens(ops, name):
    lens, news, kw = TRACKED[name]
    s = Setup(lens, news, seed=47, **kw)
    for window in (1, 64, 300):
        lse = attention_ref(s, window=window)[1].float().cuda()
        want, tol = weights_ref(s, lse, window=window)
        got = weigh(ops, s, s.weights.clone(), lse, window=window)
        assert bool(((got.cpu().double() - want).abs() <= tol).all()), window


@pytest.mark.parametrize("group,dim", [(4, 128), (1, 64), (7, 128)])
def test_query_strides_on_the_tensor_map_forms(ops, group, dim):
    """q as a slice of a wider projection, of a transposed one, and the head dimension padded: the same bits as contiguous rows."""
    s = Setup([700, 300], [150, 64], group=group, dim=dim, dtype="bf16", page=64, seed=48)
    heads = s.kv_heads * group
    want = attend(ops, s)
    w = weigh(ops, s, s.weights.clone(), want[1])
    wide = torch.full((s.tokens, heads + 5, dim), math.nan, dtype=s.dtype, device="cuda")
    turned = torch.full((heads, s.tokens + 3, dim), math.nan, dtype=s.dtype, device="cuda")
    padded = torch.full((s.tokens, heads, dim + 8), math.nan, dtype=s.dtype, device="cuda")
    for q in (wide[:, 2:2 + heads], turned[:, 1:1 + s.tokens].transpose(0, 1), padded[:, :, :dim]):
        q.copy_(s.q)
        got = ops.paged_attention(q, s.k_cache, s.v_cache, s.table, s.kv_lens, cu_seqlens=s.cu, max_new=s.max_new)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert torch.equal(weigh(ops, s, s.weights.clone(), want[1], q=q), w)


def test_overlapping_graphs_leave_what_eager_calls_leave(ops):
    """Append, attention and weights captured, replayed on two streams at once: cache, weights, out and lse are those of eager calls."""
    sets = [Setup([100, 257], [1, 1], dim=128, group=4, dtype="bf16", ragged=False), Setup([400, 300], [90, 120], dim=128, group=4, dtype="bf16", seed=2),
            Setup([600], [40], group=1, seed=3)]

    def step(x):
        ops.paged_append(x.k_new, x.v_new, x.k_cache, x.v_cache, x.table, x.kv_lens, cu_seqlens=x.cu, weights=x.weights)
        got = attend(ops, x)
        weigh(ops, x, x.weights, got[1])
        return got

    def contents(x):
        return [x.k_cache, x.v_cache, x.weights]

    first = [[c.clone() for c in contents(x)] for x in sets]

    def reset():
        for x, f in zip(sets, first):
            for c, old in zip(contents(x), f):
                c.copy_(old)
        torch.cuda.synchronize()

    for x in sets:
        step(x)
    torch.cuda.synchronize()
    graphs = []
    for x in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(x)
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in sets]
    for lens in ([100, 257], [64, 130], [1, 2]):
        sets[0].kv_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        reset()
        want = []
        for x in sets:
            for _ in range(3):
                got = step(x)
            want.append([c.clone() for c in contents(x) + list(got)])
        reset()
        for _ in range(3):
            for (g, _), st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        for x, (_, out), ref in zip(sets, graphs, want):
            for c, r in zip(contents(x) + list(out), ref):
                assert torch.equal(c, r), str(lens)


@pytest.mark.parametrize("dtype,dim", [("fp16", 64), ("bf16", 128)])
def test_rows_of_a_ring_forward_become_the_cache(ops, dtype, dim):
    """A prompt goes through the ring on two virtual ranks, its K and V into pages; a chunk's attention gives the same rows, and a token
    then answers over the cache."""
    from ringattention_b200 import RingContext
    s = Setup([512, 512], [512, 512], dim=dim, dtype=dtype, group=1, kv_heads=3, page=32, ragged=False, seed=49)
    b, h, n = 2, 3, 512
    q, k, v = (x.reshape(b, n, h, dim).transpose(1, 2).contiguous() for x in (s.q, s.k_new, s.v_new))
    ctx = RingContext.create_local(2)
    half = n // 2
    shards = [[x[:, :, r * half:(r + 1) * half].contiguous() for r in range(2)] for x in (q, k, v)]
    ctx.set_local_shards(shards[1], shards[2])
    parts = [ops.ring_forward(ctx, shards[0][r], shards[1][r], shards[2][r], causal=True, mype=r) for r in range(2)]
    ctx.synchronize()
    torch.cuda.synchronize()
    # the shards' rows go to the cache shard after shard, the lengths growing with them
    for r in range(2):
        lens = torch.full((2,), (r + 1) * half, dtype=torch.int32, device="cuda")
        kr, vr = (torch.cat([x[i].transpose(0, 1) for i in range(b)]) for x in (shards[1][r], shards[2][r]))
        ops.paged_append(kr, vr, s.k_cache, s.v_cache, s.table, lens)
    want = attention_ref(s)
    ring = [torch.cat([p[i] for p in parts], dim=2) for i in range(2)]
    ring = ring[0].transpose(1, 2).reshape(b * n, h, dim), ring[1].transpose(1, 2).reshape(b * n, h)
    check_attention(s, ring, want, out_type=torch.float32, what="ring")
    check_attention(s, attend(ops, s), want, what="paged")
    # one more token each, in a page of its own behind the prompt's
    t = Setup([513, 513], [1, 1], dim=dim, dtype=dtype, group=1, kv_heads=3, page=32, ragged=False, seed=50, extra_cols=0, spare_pages=s.pages)
    t.k_cache[:s.pages], t.v_cache[:s.pages] = s.k_cache, s.v_cache
    t.table[:, :16] = s.table[:, :16]
    t.table[:, 16] = torch.tensor([s.pages, s.pages + 1])
    ops.paged_append(t.k_new, t.v_new, t.k_cache, t.v_cache, t.table, t.kv_lens)
    check_attention(t, attend(ops, t), attention_ref(t), what="next token")
    ctx.destroy()
