"""What is measured of the paged-cache operators: append, attention, accumulated attention weights, eviction.

The operators serve a sequence after its prompt.  K and V live in pages of `page` places ([pages, kv_heads, page, dim], or
with the heads inside the place); page_table[b, i] names the page that holds places [i*page, (i+1)*page) of sequence b;
kv_lens[b] counts its places, the last n_b of which are the new tokens of this step, packed one after the other in q / k / v
([tokens, heads, dim], cu_seqlens where the sequences bring different numbers).
"""
import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------------------ cases
def _case(op, name=None, **kw):
    c = {"op": op, "dtype": "bf16", "batch": 1, "kv_heads": 8, "group": 4, "dim": 128, "page": 16, "layout": "HND",
         "len_lo": 1024, "len_hi": 1024, "new_lo": 1, "new_hi": 1, "window": 0, "sinks": 0, "idle": 0,
         "budget": 0, "first": 0, "recent": 0, "weights": False}
    c.update(kw)
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # one decoding step's new rows for a batch: as small as a call gets, latency counts; a tracked cache (weights cleared)
        _case("append", "append b32 one token", batch=32, len_lo=130, len_hi=4096, weights=True),
        # the rows of prompts that a ring forward has just computed, ragged, taken into the cache with heads inside the place
        _case("append", "append 4 prompts 16 heads", dtype="fp16", batch=4, kv_heads=16, group=1, page=64, layout="NHD",
              len_lo=2049, len_hi=8192, new_lo=2049, new_hi=8192),
        # one user, one token, a short conversation: nothing but latency
        _case("attention", "decode b1 short", dtype="fp16", batch=1, kv_heads=4, group=4, dim=64, len_lo=1000, len_hi=1000),
        # a serving batch of conversations of very different lengths, some slots idle
        _case("attention", "decode b32 ragged", batch=32, len_lo=300, len_hi=8192, idle=2),
        # two very long documents read by one token each: the cache is all there is to read
        _case("attention", "decode b2 131072", dtype="fp16", batch=2, kv_heads=2, group=8, page=64, layout="NHD",
              len_lo=131072, len_hi=131072),
        # a verification step of a few drafted tokens within a window, the first tokens kept in sight
        _case("attention", "few tokens window sinks", batch=16, group=3, dim=64, page=32, len_lo=2000, len_hi=16384,
              new_lo=2, new_hi=5, window=1024, sinks=4),
        # follow-up questions behind their conversations, every head with K/V of its own, odd lengths
        _case("attention", "chunk b4 16 heads", dtype="fp16", batch=4, kv_heads=16, group=1, page=64, len_lo=1500, len_hi=6001,
              new_lo=130, new_hi=515),
        # a piece of a long prompt behind what the earlier pieces left: the largest call, bound by arithmetic
        _case("attention", "chunk 2048 of 32768", batch=1, page=128, len_lo=32768, len_hi=32768, new_lo=2048, new_hi=2048),
        # the weights that one decoded token per sequence adds to a tracked cache
        _case("weights", "weights b16 decode", batch=16, len_lo=500, len_hi=8192),
        # the weights that a piece of a prompt adds
        _case("weights", "weights chunk 1024 of 8192", dtype="fp16", batch=1, page=64, len_lo=8192, len_hi=8192, new_lo=1024,
              new_hi=1024),
        # one conversation over its budget by a little
        _case("evict", "evict b1 to 1024", dtype="fp16", batch=1, kv_heads=4, dim=64, len_lo=1100, len_hi=1100, budget=1024,
              first=4, recent=256),
        # a batch halved
        _case("evict", "evict b16 8192 to 4096", batch=16, len_lo=4000, len_hi=8192, budget=4096, first=4, recent=1024),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "attention", "attention", "weights", "weights", "evict", "evict"])
    c = _case(op, dtype=rng.choice(["fp16", "bf16"]), kv_heads=rng.choice([1, 2, 4, 8, 16]), dim=rng.choice([64, 128]),
              page=rng.choice([8, 16, 32, 64, 128, 256]), layout=rng.choice(["HND", "NHD"]), batch=_log(rng, 1, 64))
    c["group"] = rng.choice([g for g in (1, 2, 3, 4, 5, 6, 7, 8, 16) if g * c["kv_heads"] <= 64])
    # places in all: about what the largest listed decode case holds; the longest sequence up to 131072
    most = max(64, min(131072, 2_000_000 // (c["batch"] * c["kv_heads"] * (c["dim"] // 64))))
    c["len_hi"] = _log(rng, 33, most)
    c["len_lo"] = rng.choice([c["len_hi"], _log(rng, 1, c["len_hi"])])
    if op in ("attention", "weights", "append"):
        kind = rng.choice(["one", "few", "chunk", "chunk"])
        heads = c["kv_heads"] * c["group"]
        if kind == "few":
            c["new_lo"], c["new_hi"] = 1, rng.randint(2, 9)
        elif kind == "chunk":
            pairs = 500_000_000 // (heads * c["batch"])  # below the largest listed case, batch x heads x new x places
            c["new_hi"] = _log(rng, 9, max(16, min(4096, pairs // c["len_hi"])))
            c["new_lo"] = rng.choice([c["new_hi"], _log(rng, 1, c["new_hi"])])
        c["len_hi"] = max(c["len_hi"], c["new_hi"])
        c["idle"] = rng.choice([0, 0, 1]) if c["batch"] > 1 else 0
    if op in ("attention", "weights") and rng.random() < 0.35:
        c["window"], c["sinks"] = _log(rng, 32, 8192), rng.choice([0, 1, 4, 64, 130])
    if op == "append":
        c["weights"] = rng.random() < 0.5
    if op == "evict":
        c["group"] = 1
        c["budget"] = max(16, int(c["len_hi"] * rng.uniform(0.3, 1.0)))
        c["first"], c["recent"] = rng.choice([0, 1, 4]), int(c["budget"] * rng.uniform(0.0, 0.7))
    return c


def _spread(lo, hi, n):
    """n whole numbers from hi down to lo in an order without a pattern, the same for everybody."""
    return [hi if i == 0 else lo + int((hi - lo) * ((i * 0.6180339887498949) % 1.0)) for i in range(n)]


def _shape(c):
    """(places, new tokens) of every sequence."""
    b = c["batch"]
    lens, new = _spread(c["len_lo"], c["len_hi"], b), _spread(c["new_lo"], c["new_hi"], b)
    lens = [max(a, n) for a, n in zip(lens, new)]
    for i in range(b - c["idle"], b):  # idle slots of a batch: no places; their token, if every slot has one, sees nothing
        lens[i] = 0
        if c["new_lo"] != c["new_hi"]:
            new[i] = 0
    return lens, new


# ------------------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dt, page, h, d, b = TYPES[c["dtype"]], c["page"], c["kv_heads"], c["dim"], c["batch"]
    lens, new = _shape(c)
    need = [-(-n // page) for n in lens]
    width = max(max(need), 1)
    dst_width = -(-c["budget"] // page) if c["op"] == "evict" else 0
    pages = sum(need) + b * dst_width + 2
    order = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)

    def cache():
        shape = (pages, h, page, d) if c["layout"] == "HND" else (pages, page, h, d)
        x = torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32).to(dt)
        return x if c["layout"] == "HND" else x.transpose(1, 2)

    table = torch.full((b, width), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    s = {"case": c, "k_cache": cache(), "v_cache": cache(), "table": table, "width": width, "max_new": max(new),
         "kv_lens": torch.tensor(lens, dtype=torch.int32, device=DEVICE), "cu": None}
    total = sum(new)
    if c["new_lo"] != c["new_hi"]:
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        s["cu"] = torch.tensor(cu, dtype=torch.int32, device=DEVICE)
    s["total"] = total
    if c["op"] == "append":
        s["k"] = torch.randn((total, h, d), generator=g, device=DEVICE).to(dt)
        s["v"] = torch.randn((total, h, d), generator=g, device=DEVICE).to(dt)
        s["weights"] = torch.rand((b, h, width * page), generator=g, device=DEVICE) if c["weights"] else None
    if c["op"] in ("attention", "weights"):
        s["q"] = torch.randn((total, h * c["group"], d), generator=g, device=DEVICE).to(dt)
    if c["op"] == "weights":
        s["lse"] = _plain_attention(s)[1]  # what the attention of the same step has returned
        s["weights"] = torch.rand((b, h, width * page), generator=g, device=DEVICE)
    if c["op"] == "evict":
        s["dst"] = order[at:at + b * dst_width].reshape(b, dst_width).contiguous()
        # heavy-tailed, as accumulated weights are; many places have received nothing at all (ties)
        w = torch.rand((b, h, width * page), generator=g, device=DEVICE)
        s["weights"] = torch.where(w < 0.2, torch.zeros_like(w), 0.01 / (1.0001 - w))
    return s


# ------------------------------------------------------------------------------------------------------------ plain forms
def _tokens(s):
    """(sequence, index within it) of every packed token, as device tensors."""
    c, total = s["case"], s["total"]
    t = torch.arange(total, device=DEVICE)
    if s["cu"] is None:
        n = s["max_new"]
        return t // n, t % n
    seq = torch.searchsorted(s["cu"].long(), t, right=True) - 1
    return seq, t - s["cu"].long()[seq]


def _counts(s):
    if s["cu"] is None:
        return torch.full_like(s["kv_lens"], s["max_new"]).long()
    return (s["cu"][1:] - s["cu"][:-1]).long()


def _gather(cache, table):
    """[batch, heads, places, dim] in 32 bits."""
    x = cache[table.clamp(min=0).long()]  # [b, width, h, page, d]
    b, w, h, p, d = x.shape
    return x.transpose(1, 2).reshape(b, h, w * p, d).float()


def _scores(s):
    """Scaled scores [batch, kv_heads, group * new, places], -inf where not visible, and (seq, index) of the tokens."""
    c = s["case"]
    b, h, gr, d, n = c["batch"], c["kv_heads"], c["group"], c["dim"], s["max_new"]
    seq, idx = _tokens(s)
    q = torch.zeros((b, n, h, gr, d), device=DEVICE)
    q[seq, idx] = s["q"].float().reshape(-1, h, gr, d)
    q = q.permute(0, 2, 3, 1, 4).reshape(b, h, gr * n, d)
    x = torch.matmul(q, _gather(s["k_cache"], s["table"]).transpose(-1, -2)).mul_(d ** -0.5)
    lens = s["kv_lens"].long()
    pos = (lens - _counts(s))[:, None] + torch.arange(n, device=DEVICE)[None, :]  # place of token i
    j = torch.arange(x.shape[-1], device=DEVICE)
    hidden = (j[None, None, :] > pos[:, :, None]) | (j[None, None, :] >= lens[:, None, None])
    if c["window"]:
        hidden |= (j[None, None, :] <= pos[:, :, None] - c["window"]) & (j[None, None, :] >= c["sinks"])
    x.reshape(b, h * gr, n, -1).masked_fill_(hidden[:, None], -math.inf)
    return x, seq, idx


def _plain_attention(s):
    c = s["case"]
    b, h, gr, d, n = c["batch"], c["kv_heads"], c["group"], c["dim"], s["max_new"]
    x, seq, idx = _scores(s)
    top = x.amax(dim=-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    x.sub_(top).exp_()
    total = x.sum(dim=-1, keepdim=True)
    some = total > 0
    out = torch.matmul(x, _gather(s["v_cache"], s["table"]))
    out = torch.where(some, out / total, torch.zeros_like(out))
    lse = torch.where(some, top + torch.log(total), torch.full_like(top, -math.inf))
    out = out.reshape(b, h, gr, n, d).permute(0, 3, 1, 2, 4)[seq, idx].reshape(-1, h * gr, d)
    lse = lse.reshape(b, h, gr, n).permute(0, 3, 1, 2)[seq, idx].reshape(-1, h * gr)
    return out.to(s["q"].dtype), lse


def _plain_weights(s):
    c = s["case"]
    b, h, gr, n = c["batch"], c["kv_heads"], c["group"], s["max_new"]
    x, seq, idx = _scores(s)
    lse = torch.zeros((b, n, h, gr), device=DEVICE)
    lse[seq, idx] = s["lse"].reshape(-1, h, gr)
    real = torch.zeros((b, n), dtype=torch.bool, device=DEVICE)
    real[seq, idx] = True
    lse = lse.permute(0, 2, 3, 1)
    lse = torch.where(torch.isinf(lse) | ~real[:, None, None], torch.full_like(lse, math.inf), lse).reshape(b, h, gr * n, 1)
    s["weights"] += x.sub_(lse).exp_().sum(dim=2)
    return s["weights"]


def _plain_append(s):
    c = s["case"]
    seq, idx = _tokens(s)
    place = (s["kv_lens"].long() - _counts(s))[seq] + idx
    fine = place >= 0  # (an idle slot's token has no place: its row goes nowhere)
    place = place.clamp(min=0)
    page, slot = s["table"].long()[seq, place // c["page"]], place % c["page"]
    fine &= page >= 0
    page = page.clamp(min=0)
    if c["idle"]:
        # the rows without a place are written over the first row of all, with its own value
        first = fine.long().argmax()
        src = torch.where(fine, torch.arange(s["total"], device=DEVICE), first)
        page, slot, seq, place, k, v = page[src], slot[src], seq[src], place[src], s["k"][src], s["v"][src]
    else:
        k, v = s["k"], s["v"]
    s["k_cache"][page, :, slot] = k
    s["v_cache"][page, :, slot] = v
    if s["weights"] is None:
        return s["k_cache"], s["v_cache"]
    s["weights"][seq, :, place] = 0.0
    return s["k_cache"], s["v_cache"], s["weights"]


def _plain_evict(s):
    c = s["case"]
    budget, page, h = c["budget"], c["page"], c["kv_heads"]
    w, lens = s["weights"], s["kv_lens"].long()
    j = torch.arange(w.shape[-1], device=DEVICE)
    stays = (j < c["first"]) | (j[None, :] >= lens[:, None] - c["recent"])
    key = torch.where(stays[:, None], torch.full_like(w, math.inf), w)
    key = torch.where((j[None, :] >= lens[:, None])[:, None], torch.full_like(w, -math.inf), key)
    best = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :budget]
    if best.shape[-1] < budget:
        best = torch.nn.functional.pad(best, (0, budget - best.shape[-1]), value=w.shape[-1])
    none = best >= lens[:, None, None]
    kept = torch.sort(torch.where(none, torch.full_like(best, 1 << 30), best), dim=-1).values
    none = kept == 1 << 30
    kept = kept.masked_fill(none, 0)
    m = torch.arange(budget, device=DEVICE)
    heads = torch.arange(h, device=DEVICE)[None, :, None]
    batch = torch.arange(c["batch"], device=DEVICE)[:, None, None]
    src = s["table"].long().clamp(min=0)[batch, kept // page]
    dst = s["dst"].long()[:, m // page][:, None].expand_as(kept)
    for cache in (s["k_cache"], s["v_cache"]):
        rows = torch.where(none[..., None], cache[dst, heads, m % page], cache[src, heads, kept % page])
        cache[dst, heads, (m % page).expand_as(kept)] = rows
    new_w = torch.zeros((c["batch"], h, s["dst"].shape[1] * page), device=DEVICE)
    new_w[..., :budget] = torch.gather(w, 2, kept).masked_fill(none, 0.0)
    return lens.clamp(max=budget).to(torch.int32), new_w, kept.masked_fill(none, -1).to(torch.int32), s["k_cache"], s["v_cache"]


# ------------------------------------------------------------------------------------------------------------ one pass
def run(s):
    c = s["case"]
    if not own:
        return {"append": _plain_append, "attention": _plain_attention, "weights": _plain_weights, "evict": _plain_evict}[c["op"]](s)
    from ringattention_b200 import torch_ops
    if c["op"] == "append":
        torch_ops.paged_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["kv_lens"], cu_seqlens=s["cu"],
                               weights=s["weights"])
        return (s["k_cache"], s["v_cache"]) if s["weights"] is None else (s["k_cache"], s["v_cache"], s["weights"])
    if c["op"] == "attention":
        return torch_ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["kv_lens"], cu_seqlens=s["cu"],
                                         max_new=s["max_new"], window=c["window"], sinks=c["sinks"])
    if c["op"] == "weights":
        torch_ops.paged_weights_(s["weights"], s["q"], s["k_cache"], s["lse"], s["table"], s["kv_lens"], cu_seqlens=s["cu"],
                                 max_new=s["max_new"], window=c["window"], sinks=c["sinks"])
        return s["weights"]
    lens, weights, kept = torch_ops.paged_evict(s["k_cache"], s["v_cache"], s["weights"], s["table"], s["kv_lens"], s["dst"],
                                                c["budget"], first=c["first"], recent=c["recent"])
    return lens, weights, kept, s["k_cache"], s["v_cache"]


# ------------------------------------------------------------------------------------------------------------ work
def _visible(c, n_places, n_new):
    """(visible pairs, places that some token sees) of one sequence."""
    pairs = seen = 0
    low = n_places
    for i in range(n_new):
        p = n_places - n_new + i
        if p < 0:
            continue
        lo = max(0, p - c["window"] + 1) if c["window"] else 0
        pairs += p + 1 - lo + min(c["sinks"], lo)
        low = min(low, lo)
    if pairs:
        seen = n_places - low + min(c["sinks"], low)
    return pairs, seen


def work(case):
    c = case
    lens, new = _shape(c)
    h, d, total = c["kv_heads"], c["dim"], sum(new)
    if c["op"] == "append":
        rows = sum(n for a, n in zip(lens, new) if a)
        return {"bytes": 8 * rows * h * d + (4 * rows * h if c["weights"] else 0), "flops": 0}
    if c["op"] == "evict":
        kept = sum(min(a, c["budget"]) for a in lens)
        width = -(-c["budget"] // c["page"]) * c["page"]
        return {"bytes": 8 * kept * h * d + 4 * sum(lens) * h + 4 * c["batch"] * h * (width + c["budget"]), "flops": 0}
    vis = [_visible(c, a, n) for a, n in zip(lens, new)]
    pairs, seen = sum(v[0] for v in vis), sum(v[1] for v in vis)
    q_bytes = 2 * total * h * c["group"] * d
    if c["op"] == "attention":
        return {"bytes": 4 * seen * h * d + 2 * q_bytes + 4 * total * h * c["group"], "flops": 4 * d * pairs * h * c["group"]}
    return {"bytes": 2 * seen * h * d + 8 * seen * h + q_bytes + 4 * total * h * c["group"], "flops": 2 * d * pairs * h * c["group"]}


# ------------------------------------------------------------------------------------------------------------ 64 bits
def _rows64(cache, table_row, n, page, head):
    """The first n places of one head of one sequence, [n, dim] in 64 bits."""
    ids = table_row[:-(-n // page)].tolist()
    return torch.cat([cache[i, head] for i in ids]).double()[:n]


def _probabilities(s, i, head, at, n, n_places):
    """exp(score) pieces of the tokens [at, at + n) of sequence i with one kv head: (P, lse), rows token-major then group."""
    c = s["case"]
    gr, d = c["group"], c["dim"]
    k = _rows64(s["k_cache"], s["table"][i], n_places, c["page"], head)
    q = s["q"][at:at + n, head * gr:(head + 1) * gr].double().reshape(n * gr, d)
    x = (q @ k.T) / math.sqrt(d)
    p = (torch.arange(n, device=DEVICE) + (n_places - n)).repeat_interleave(gr)
    j = torch.arange(n_places, device=DEVICE)
    see = j[None] <= p[:, None]
    if c["window"]:
        see &= (j[None] > p[:, None] - c["window"]) | (j[None] < c["sinks"])
    x = torch.where(see, x, torch.full_like(x, -math.inf))
    return x, torch.logsumexp(x, dim=1)


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    lens, new = _shape(c)
    h, gr, d, page = c["kv_heads"], c["group"], c["dim"], c["page"]
    if c["op"] == "append":
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        w = None if s["weights"] is None else s["weights"].double()
        seq_of, place_of, token = [], [], []
        at = 0
        for i in range(c["batch"]):
            for t in range(new[i]):
                if lens[i]:
                    seq_of.append(i), place_of.append(lens[i] - new[i] + t), token.append(at + t)
            at += new[i]
        si, pi, ti = (torch.tensor(x, device=DEVICE) for x in (seq_of, place_of, token))
        pg = s["table"].long()[si, torch.div(pi, page, rounding_mode="floor")]
        for head in range(h):
            kc[pg, head, pi % page] = s["k"][ti, head].double()
            vc[pg, head, pi % page] = s["v"][ti, head].double()
            if w is not None:
                w[si, head, pi] = 0
        return (kc, vc) if w is None else (kc, vc, w)
    if c["op"] == "evict":
        budget = c["budget"]
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        new_w = torch.zeros((c["batch"], h, s["dst"].shape[1] * page), dtype=torch.float64, device=DEVICE)
        kept = torch.full((c["batch"], h, budget), -1, dtype=torch.int32, device=DEVICE)
        for i in range(c["batch"]):
            n, m = lens[i], min(lens[i], budget)
            if not n:
                continue
            for head in range(h):
                if n <= budget:
                    keep = torch.arange(n, device=DEVICE)
                else:
                    free = torch.arange(c["first"], n - c["recent"], device=DEVICE)
                    heavy = torch.argsort(-s["weights"][i, head, free].double(), stable=True)[:budget - c["first"] - c["recent"]]
                    keep = torch.cat([torch.arange(c["first"], device=DEVICE), torch.sort(free[heavy]).values,
                                      torch.arange(n - c["recent"], n, device=DEVICE)])
                to = torch.arange(m, device=DEVICE)
                a, z = s["table"][i].long()[keep // page], s["dst"][i].long()[to // page]
                kc[z, head, to % page] = s["k_cache"][a, head, keep % page].double()
                vc[z, head, to % page] = s["v_cache"][a, head, keep % page].double()
                new_w[i, head, :m] = s["weights"][i, head, keep].double()
                kept[i, head, :m] = keep.to(torch.int32)
        return torch.tensor([min(a, budget) for a in lens], dtype=torch.int32, device=DEVICE), new_w, kept, kc, vc
    if c["op"] == "attention":
        out = torch.zeros((s["total"], h * gr, d), dtype=torch.float64, device=DEVICE)
        lse = torch.full((s["total"], h * gr), -math.inf, dtype=torch.float64, device=DEVICE)
    else:
        w = s["weights"].double()
    at = 0
    for i in range(c["batch"]):
        for head in range(h if lens[i] and new[i] else 0):
            x, l = _probabilities(s, i, head, at, new[i], lens[i])
            mine = slice(head * gr, (head + 1) * gr)
            if c["op"] == "attention":
                v = _rows64(s["v_cache"], s["table"][i], lens[i], page, head)
                out[at:at + new[i], mine] = (torch.exp(x - l[:, None]) @ v).reshape(new[i], gr, d)
                lse[at:at + new[i], mine] = l.reshape(new[i], gr)
            else:
                given = s["lse"][at:at + new[i], mine].double().reshape(-1, 1)
                w[i, head, :lens[i]] += torch.exp(x - given).sum(dim=0)
        at += new[i]
    return (out, lse) if c["op"] == "attention" else w
