"""torch.Tensor front end: the operator the reference's include/attention_api.cuh:1-30 prepares for
(torch/extension.h plus the CHECK_INPUT argument checks) but never declares.

The functions here take and return torch tensors; argument checking (CUDA device, contiguity, dtype, shape)
happens in C++ (csrc/torch_ext.cpp) with the reference's CHECK_INPUT macro, the work happens in the C-ABI
library.  The extension is compiled by ``python -m ringattention_b200.build --torch``; importing this module
without it raises, there is no fallback.  Forward only, as in the reference.
"""
from __future__ import annotations

import importlib
from typing import Optional, Sequence, Tuple

_ext = None


def _load():
    global _ext
    if _ext is None:
        import torch  # noqa: F401  (the extension resolves libtorch symbols from the loaded torch)
        try:
            _ext = importlib.import_module("ringattention_b200._torch_ext")
        except ImportError as e:
            raise ImportError("ringattention_b200._torch_ext is not built: run "
                              "`python -m ringattention_b200.build --torch`") from e
    return _ext


def block_forward(q, k, v, softmax_scale: Optional[float] = None, causal: bool = False, q_off: int = 0, k_off: int = 0) -> Tuple:
    """One Q shard [B,H,Sq,D] against one K/V shard [B,H,Sk,D] (fp16 or bf16): returns (out fp32, lse fp32).

    The flash inner loop over one source shard and the final normalisation (csrc/ring_attention.cu:536-609,
    621-664).  softmax_scale None means 1/sqrt(D); q_off / k_off place the shards in the global sequence for the
    causal mask.  Asynchronous on the current torch stream.
    """
    return tuple(_load().block_forward(q, k, v, float(softmax_scale or 0.0), bool(causal), int(q_off), int(k_off)))


def ring_forward(ctx, q, k, v, seqlens: Optional[Sequence[int]] = None, softmax_scale: Optional[float] = None,
                 causal: bool = False, mype: Optional[int] = None) -> Tuple:
    """Ring-attention forward of this rank through a RingContext: returns (out fp32, lse fp32).

    set_params_fprop + run_ring_fwd of the reference (csrc/ring_attention.cu:361-395, 669-704) on tensors.
    seqlens are the rows of every rank's shard (default: all equal to this rank's); mype defaults to ctx.rank
    (virtual-rank contexts pass it explicitly).  Asynchronous on the current torch stream.
    """
    rank = ctx.rank if mype is None else int(mype)
    lens = [int(q.shape[2])] * ctx.world if seqlens is None else [int(s) for s in seqlens]
    return tuple(_load().ring_forward(int(ctx._h.value), q, k, v, lens, rank, float(softmax_scale or 0.0), bool(causal)))


def lse_merge_(o_acc, lse_acc, o_part, lse_part) -> None:
    """Merges the partial (o_part, lse_part) into (o_acc, lse_acc) in place (csrc/ring_attention.cu:439-443, 621-633)."""
    _load().lse_merge_(o_acc, lse_acc, o_part, lse_part)


# ---- paged K/V cache: conventions as in include/ring_attention_b200.h; asynchronous on the current stream of the tensors' device ----

def paged_append(k, v, k_cache, v_cache, page_table, kv_lens, cu_seqlens=None, weights=None) -> None:
    """Writes the new tokens' rows k, v [tokens, kv_heads, dim] to their places in k_cache, v_cache [pages, kv_heads, page_size, dim].

    page_table [batch, max_pages] and kv_lens [batch] are int32; kv_lens counts the new tokens already.  cu_seqlens [batch + 1]
    int32 when the sequences bring different numbers of tokens.  weights [batch, kv_heads, places]: set to 0 at the new places.
    """
    _load().paged_append(k, v, k_cache, v_cache, page_table, kv_lens, cu_seqlens, weights)


def paged_attention(q, k_cache, v_cache, page_table, kv_lens, cu_seqlens=None, max_new: int = 0, softmax_scale: Optional[float] = None,
                    causal: bool = True, window: int = 0, sinks: int = 0, fp32_out: bool = False) -> Tuple:
    """Attention of the new tokens q [tokens, heads, dim] over the paged cache: returns (out, lse [tokens, heads] fp32).

    A token at place p sees the places <= p (or, causal=False, all of its sequence); with window > 0 only those > p - window,
    and the first `sinks`.  out has q's type, or fp32 with fp32_out: the partials of several caches then join with
    lse_merge_.  max_new bounds the new tokens of one sequence when cu_seqlens is given.  softmax_scale None: 1/sqrt(dim).
    """
    return _load().paged_attention(q, k_cache, v_cache, page_table, kv_lens, cu_seqlens, max_new, softmax_scale, causal, window, sinks,
                                   fp32_out)


def paged_weights_(weights, q, k_cache, lse, page_table, kv_lens, cu_seqlens=None, max_new: int = 0,
                   softmax_scale: Optional[float] = None, causal: bool = True, window: int = 0, sinks: int = 0) -> None:
    """weights [batch, kv_heads, places] += the attention every cached place received from the new tokens, given the lse that
    paged_attention returned for the same arguments."""
    _load().paged_weights_(weights, q, k_cache, lse, page_table, kv_lens, cu_seqlens, max_new, softmax_scale, causal, window, sinks)


def paged_evict(k_cache, v_cache, weights, page_table, kv_lens, dst_table, budget: int, first: int = 0, recent: int = 0) -> Tuple:
    """Keeps the first `first`, the last `recent` and the heaviest other places of every sequence and K/V head, `budget` in all, and
    copies their rows to the pages dst_table names (other pages than the sources).

    Returns (new_lens [batch] int32, new_weights [batch, kv_heads, dst places] fp32, kept [batch, kv_heads, budget] int32,
    ascending, -1 behind the last).
    """
    return _load().paged_evict(k_cache, v_cache, weights, page_table, kv_lens, dst_table, budget, first, recent)
