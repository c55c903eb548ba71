"""Plain 64-bit statement of the paged-cache operators, and the tolerances their tests use."""
import math

import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


class Setup:
    """A cache with sequences in it, on `device`, made from a seed; new tokens included in the lengths."""

    def __init__(self, lens, news, *, dtype="fp16", dim=64, kv_heads=2, group=2, page=16, layout="HND", seed=0, device="cuda",
                 ragged=True, spare_pages=3, extra_cols=1, gain=1.0):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.dim, self.kv_heads, self.group, self.page = TYPES[dtype], dim, kv_heads, group, page
        self.lens, self.news, self.batch = list(lens), list(news), len(lens)
        need = [-(-n // page) for n in lens]
        width = max(max(need), 1) + extra_cols
        self.pages = sum(need) + spare_pages
        order = torch.randperm(self.pages, generator=g)
        table = torch.full((self.batch, width), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = order[at:at + n]
            at += n
        self.free = order[at:].tolist()
        shape = (self.pages, kv_heads, page, dim) if layout == "HND" else (self.pages, page, kv_heads, dim)

        def cache():
            x = (torch.randn(shape, generator=g) * gain).to(self.dtype).to(device)
            return x if layout == "HND" else x.transpose(1, 2)

        self.k_cache, self.v_cache = cache(), cache()
        self.table = table.to(device)
        self.kv_lens = torch.tensor(lens, dtype=torch.int32, device=device)
        self.cu_list = [0]
        for n in news:
            self.cu_list.append(self.cu_list[-1] + n)
        self.tokens = self.cu_list[-1]
        self.cu = torch.tensor(self.cu_list, dtype=torch.int32, device=device) if ragged else None
        self.max_new = max(news) if news else 0
        self.q = (torch.randn((self.tokens, kv_heads * group, dim), generator=g) * gain).to(self.dtype).to(device)
        self.k_new = (torch.randn((self.tokens, kv_heads, dim), generator=g) * gain).to(self.dtype).to(device)
        self.v_new = (torch.randn((self.tokens, kv_heads, dim), generator=g) * gain).to(self.dtype).to(device)
        self.weights = torch.rand((self.batch, kv_heads, width * page), generator=g).to(device)

    def rows(self, cache, b, head):
        """(rows [places, dim] float64 on the CPU, page-exists mask) of one head of one sequence; rows without a page are 0."""
        n = min(max(self.lens[b], 0), self.table.shape[1] * self.page)
        x = torch.zeros((n, self.dim), dtype=torch.float64)
        ok = torch.zeros(n, dtype=torch.bool)
        c, t = cache.cpu(), self.table.cpu()
        for i in range(-(-n // self.page)):
            lo, hi = i * self.page, min((i + 1) * self.page, n)
            if 0 <= int(t[b, i]) < self.pages:
                x[lo:hi] = c[int(t[b, i]), head, :hi - lo].double()
                ok[lo:hi] = True
        return x, ok


def visible(n_places, n_new, causal, window, sinks):
    """[n_new, n_places] truth values."""
    p = torch.arange(n_new)[:, None] + (n_places - n_new)
    j = torch.arange(n_places)[None, :]
    see = torch.ones((n_new, n_places), dtype=torch.bool)
    if causal:
        see &= j <= p
    if window:
        see &= (j > p - window) | (j < sinks)
    return see


def attention_ref(s, scale=None, causal=True, window=0, sinks=0):
    """(out, lse, sum p |v|, bound of a score's error, bound of what small probabilities lose), in 64 bits."""
    scale = s.dim ** -0.5 if scale is None else scale
    heads = s.kv_heads * s.group
    out = torch.zeros((s.tokens, heads, s.dim), dtype=torch.float64)
    lse = torch.full((s.tokens, heads), -math.inf, dtype=torch.float64)
    absout, delta, low = torch.zeros_like(out), torch.zeros_like(lse), torch.zeros_like(out)
    q = s.q.cpu().double()
    for b in range(s.batch):
        lo, hi = s.cu_list[b], s.cu_list[b + 1]
        for h in range(heads):
            k, ok = s.rows(s.k_cache, b, h // s.group)
            v, _ = s.rows(s.v_cache, b, h // s.group)
            see = visible(k.shape[0], hi - lo, causal, window, sinks) & ok[None]
            if hi == lo or not see.any():
                continue
            some = see.any(dim=0)
            k, v = torch.where(some[:, None], k, torch.zeros_like(k)), torch.where(some[:, None], v, torch.zeros_like(v))
            x = (q[lo:hi, h] @ k.T * scale).masked_fill(~see, -math.inf)
            l = torch.logsumexp(x, dim=1)
            p = torch.where(see, torch.exp(x - l.clamp(min=-1e300)[:, None]), torch.zeros_like(x))
            out[lo:hi, h], lse[lo:hi, h] = p @ v, l
            absout[lo:hi, h] = p @ v.abs()
            if s.dtype == torch.float16:  # a probability below the normal range (its largest is held as 1) is off by up to 2^-25
                top = torch.where(see.any(dim=1), torch.exp(x.amax(dim=1) - l), torch.zeros_like(l))
                low[lo:hi, h] = 2.0 ** -25 * top[:, None] * (see.double() @ v.abs())
            # a score is a sum of D products in 32 bits: its error is at most (D + 3) half steps of the sum of their sizes
            size = ((q[lo:hi, h].abs() @ k.abs().T) * scale).masked_fill(~see, 0.0).amax(dim=1)
            delta[lo:hi, h] = (s.dim + 3) * 2.0 ** -24 * size
    return out, lse, absout, delta, low


def check_attention(s, got, want, out_type=None, what=""):
    """Every element of out and lse against its bound.

    out: P is rounded to the inputs' type (half a step of each p: at most half_step * sum p |v|), the scores are off by delta (each
    p by a factor of at most e^(2 delta)), exponentials and 32-bit sums by 2^-19 in all, the output by half a step of its own type
    (fp16 below its normal range: 2^-25 in absolute terms).
    """
    (out, lse), (ro, rl, ra, delta, low) = got, want
    out_type = out_type or s.dtype
    out, lse = out.cpu().double(), lse.cpu().double()
    empty = torch.isinf(rl)
    assert torch.equal(torch.isneginf(lse), empty), f"{what}: rows without a visible place differ"
    assert not torch.isnan(out).any(), f"{what}: NaN"
    assert bool((out[empty] == 0).all()), f"{what}: a row without a visible place must be 0"
    tol = HALF_STEP[s.dtype] * ra + HALF_STEP[out_type] * (ro.abs() + HALF_STEP[s.dtype] * ra) + (2 * delta[..., None] + 2.0 ** -19) * ra + low + 2.0 ** -25
    worst = ((out - ro).abs() / tol.clamp(min=1e-300)).max().item() if out.numel() else 0.0
    assert worst <= 1.0, f"{what}: out is {worst:.2f} times its bound off"
    fin = ~empty
    tol_l = delta + 2.0 ** -19 + 2.0 ** -22 * rl.abs()
    if fin.any():
        worst = ((lse - rl).abs()[fin] / tol_l[fin]).max().item()
        assert worst <= 1.0, f"{what}: lse is {worst:.2f} times its bound off"


def weights_ref(s, lse, scale=None, causal=True, window=0, sinks=0):
    """The weights after the call, and the bound of each."""
    scale = s.dim ** -0.5 if scale is None else scale
    w = s.weights.cpu().double()
    tol = 2.0 ** -23 * w.abs()
    q, lse = s.q.cpu().double(), lse.cpu().double()
    for b in range(s.batch):
        lo, hi = s.cu_list[b], s.cu_list[b + 1]
        if hi == lo:
            continue
        for h in range(s.kv_heads * s.group):
            k, ok = s.rows(s.k_cache, b, h // s.group)
            n = k.shape[0]
            see = visible(n, hi - lo, causal, window, sinks) & ok[None] & ~torch.isinf(lse[lo:hi, h])[:, None]
            k = torch.where(see.any(dim=0)[:, None], k, torch.zeros_like(k))
            l = torch.where(torch.isinf(lse[lo:hi, h]), torch.zeros_like(lse[lo:hi, h]), lse[lo:hi, h])[:, None]
            x = q[lo:hi, h] @ k.T * scale
            p = torch.where(see, torch.exp(x - l), torch.zeros_like(x))
            size = (q[lo:hi, h].abs() @ k.abs().T) * scale
            add = p.sum(dim=0)
            w[b, h // s.group, :n] += add
            # scores off by (dim + 3) half steps of their terms' sizes, lse and its product with log2 e by 2^-23 of it; the sum
            # of all rows in 32 bits by a half step per row
            tol[b, h // s.group, :n] += (p * (2 * (s.dim + 3) * 2.0 ** -24 * size + 2.0 ** -22 * l.abs() + 2.0 ** -20)).sum(dim=0)
            tol[b, h // s.group, :n] += add * (hi - lo) * s.group * 2.0 ** -24
    return w, tol + 2.0 ** -23 * w.abs() + 1e-30


def evict_ref(lens, weights, budget, first, recent):
    """kept places per sequence and head, ascending, as lists."""
    kept = []
    for b, n in enumerate(lens):
        per_head = []
        for h in range(weights.shape[1]):
            if n <= budget:
                per_head.append(list(range(n)))
                continue
            w = weights[b, h].tolist()
            mid = sorted(range(first, n - recent), key=lambda j: (-math.inf if w[j] != w[j] else -w[j], 0 if w[j] != w[j] else 1, j))
            mid = sorted(mid[:budget - first - recent])
            per_head.append(list(range(first)) + mid + list(range(n - recent, n)))
        kept.append(per_head)
    return kept
