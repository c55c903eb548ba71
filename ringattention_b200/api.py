"""Python host side of the B200 ring-attention forward.

Mirrors the operator interface of the reference for this path, over the C ABI of
include/ring_attention_b200.h:
  * ring_attention(q, k, v, out, npes, mype, seqlen, dim, max_seq) -- same name, argument order
    and meaning as csrc/ring_attention.cu:706 of the reference (synchronous, single head);
  * Ring_fwd_params / set_params_fprop -- csrc/ring.h:5-19 and csrc/ring_attention.cu:361-395;
  * RingContext -- what nvshmem_init + the symmetric buffers provide there
    (csrc/ring_attention.cu:754-761, 391-393): communicator, side stream, receive buffers.
torch is used only for device memory, streams and the rendezvous; every computation goes through
the CUDA library, and a missing library is an error, never a fallback.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Sequence

from . import _lib
from ._lib import Ring_fwd_params, check

__all__ = [
    "ring_attention", "ring_attention_scaled", "set_params_fprop", "Ring_fwd_params", "RingContext",
    "attention_block_fwd", "lse_merge", "device_status", "device_status_reset", "kernel_launch_count",
    "attention_chunked_fwd_static", "static_status",
    "paged_append", "paged_attention_fwd", "paged_attention_workspace", "paged_weights", "paged_weights_workspace", "paged_evict",
]


def _ptr(x, what: str = "tensor", dtypes=None) -> int:
    """Device address of a torch tensor (checked like the reference's CHECK_INPUT,
    include/attention_api.cuh:12-18) or a raw integer address."""
    if x is None:
        return 0
    if isinstance(x, int):
        return x
    if hasattr(x, "data_ptr"):
        if not x.is_cuda:
            raise ValueError(f"{what} must be a CUDA tensor")
        if not x.is_contiguous():
            raise ValueError(f"{what} must be contiguous")
        if dtypes is not None and x.dtype not in dtypes:
            raise ValueError(f"{what} has dtype {x.dtype}, expected one of {dtypes}")
        return x.data_ptr()
    raise TypeError(f"{what}: expected a CUDA tensor or an integer device address")


def _half_types():
    import torch
    return (torch.float16, torch.bfloat16)


def _stream_handle(stream) -> int:
    if stream is None:
        import torch
        return torch.cuda.current_stream().cuda_stream
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


def _int_array(values: Sequence[int]):
    return (ctypes.c_int * len(values))(*[int(v) for v in values])


def ring_attention(q, k, v, out, npes: int, mype: int, seqlen: Sequence[int], dim: int, max_seq: int) -> None:
    """The reference's entry point (csrc/ring_attention.cu:706): q, k, v [seqlen[mype], dim] fp16 on the
    device, out [seqlen[mype], dim] fp32, single head, non-causal, synchronous.  Softmax scale 1/sqrt(dim)."""
    lib = _lib.load()
    arr = _int_array(seqlen)
    check(lib.ring_attention(_ptr(q, "q"), _ptr(k, "k"), _ptr(v, "v"), _ptr(out, "out"), int(npes), int(mype),
                             arr, int(dim), int(max_seq)), "ring_attention")


def ring_attention_scaled(q, k, v, out, npes, mype, seqlen, dim, max_seq, softmax_scale: float) -> None:
    """ring_attention with an explicit natural-base scale (1.0 reproduces csrc/self_attention.py:22-26)."""
    lib = _lib.load()
    arr = _int_array(seqlen)
    check(lib.ring_attention_scaled(_ptr(q, "q"), _ptr(k, "k"), _ptr(v, "v"), _ptr(out, "out"), int(npes), int(mype),
                                    arr, int(dim), int(max_seq), float(softmax_scale)), "ring_attention_scaled")


def set_params_fprop(q, k, v, out, npes: int, mype: int, seqlen: Sequence[int], dim: int, max_seq: int = 0,
                     *, batch: int = 1, heads: int = 1, lse=None, causal: bool = False,
                     softmax_scale: Optional[float] = None, stream=None) -> Ring_fwd_params:
    """Fill a Ring_fwd_params like the reference's set_params_fprop (csrc/ring_attention.cu:361-395);
    keyword arguments cover the extension fields.  The returned struct keeps the seqlen table alive."""
    import torch
    p = Ring_fwd_params()
    arr = _int_array(seqlen)
    p._keep = arr  # ctypes does not own the pointee otherwise
    p.mype, p.npes = int(mype), int(npes)
    p.seqlen = None
    p.h_seqlen = ctypes.cast(arr, ctypes.POINTER(ctypes.c_int))
    p.dim = int(dim)
    p.softmax_scale = float(softmax_scale) if softmax_scale is not None else 1.0 / math.sqrt(dim)
    p.q_ptr, p.k_ptr, p.v_ptr = (_ptr(x, n, _half_types() if hasattr(x, "dtype") else None)
                                 for x, n in ((q, "q"), (k, "k"), (v, "v")))
    p.out_ptr = _ptr(out, "out", (torch.float32,) if hasattr(out, "dtype") else None)
    p.k_buffer = p.v_buffer = None
    p.batch, p.heads = int(batch), int(heads)
    p.lse_ptr = _ptr(lse, "lse", (torch.float32,) if hasattr(lse, "dtype") else None) or None
    p.causal = int(bool(causal))
    p.is_bf16 = int(hasattr(q, "dtype") and q.dtype == torch.bfloat16)
    p.stream = _stream_handle(stream)
    return p


class RingContext:
    """Owns the communicator, the exchange stream, events, the receive double buffer and the workspace."""

    def __init__(self, handle: int, rank: int, world: int, local: bool):
        self._h = ctypes.c_void_p(handle)
        self.rank, self.world, self.local = rank, world, local
        self._keep = None

    # ---- construction -------------------------------------------------------------------------------
    @staticmethod
    def unique_id() -> bytes:
        buf = ctypes.create_string_buffer(_lib.RING_UNIQUE_ID_BYTES)
        check(_lib.load().ring_get_unique_id(buf), "ring_get_unique_id")
        return buf.raw

    @classmethod
    def create(cls, rank: int = 0, world: int = 1, unique_id: Optional[bytes] = None) -> "RingContext":
        h = ctypes.c_void_p()
        uid = ctypes.create_string_buffer(unique_id, _lib.RING_UNIQUE_ID_BYTES) if unique_id else None
        check(_lib.load().ring_ctx_create(ctypes.byref(h), int(rank), int(world), uid), "ring_ctx_create")
        return cls(h.value, rank, world, False)

    @classmethod
    def from_torch_distributed(cls, group=None) -> "RingContext":
        """One process per GPU: rank 0 makes the id, torch.distributed carries it to the others."""
        import torch.distributed as dist
        rank, world = dist.get_rank(group), dist.get_world_size(group)
        if world == 1:
            return cls.create(0, 1, None)
        box = [cls.unique_id() if rank == 0 else None]
        dist.broadcast_object_list(box, src=dist.get_global_rank(group, 0) if group is not None else 0, group=group)
        return cls.create(rank, world, box[0])

    @classmethod
    def create_local(cls, world: int) -> "RingContext":
        """`world` virtual ranks on the current GPU; the exchange is a device-to-device copy."""
        h = ctypes.c_void_p()
        check(_lib.load().ring_ctx_create_local(ctypes.byref(h), int(world)), "ring_ctx_create_local")
        return cls(h.value, 0, world, True)

    def set_local_shards(self, k_shards, v_shards) -> None:
        n = self.world
        ks = (ctypes.c_void_p * n)(*[_ptr(x, "k shard") for x in k_shards])
        vs = (ctypes.c_void_p * n)(*[_ptr(x, "v shard") for x in v_shards])
        self._keep = (list(k_shards), list(v_shards))
        check(_lib.load().ring_ctx_set_local_shards(self._h, ks, vs), "ring_ctx_set_local_shards")

    # ---- options --------------------------------------------------------------------------------------
    def set_option(self, option: int, value: int) -> None:
        check(_lib.load().ring_ctx_set_option(self._h, int(option), int(value)), "ring_ctx_set_option")

    def get_option(self, option: int) -> int:
        v = ctypes.c_int(0)
        check(_lib.load().ring_ctx_get_option(self._h, int(option), ctypes.byref(v)), "ring_ctx_get_option")
        return v.value

    def set_default(self) -> None:
        """Make this the context the plain ring_attention() call uses."""
        check(_lib.load().ring_set_default_ctx(self._h), "ring_set_default_ctx")

    # ---- the forward ------------------------------------------------------------------------------------
    def forward_params(self, params: Ring_fwd_params) -> None:
        check(_lib.load().ring_attention_fwd(self._h, ctypes.byref(params)), "ring_attention_fwd")

    def forward(self, q, k, v, out, lse=None, *, causal: bool = False, softmax_scale: Optional[float] = None,
                stream=None, rank: Optional[int] = None, seqlens: Optional[Sequence[int]] = None) -> None:
        """q, k, v: [B, H, S_local, D] fp16/bf16 shards of this rank; out [B, H, S_local, D] fp32;
        lse [B, H, S_local] fp32 or None.  Asynchronous on `stream` (default: torch's current stream)."""
        B, H, S, D = q.shape
        if tuple(k.shape) != (B, H, S, D) or tuple(v.shape) != (B, H, S, D) or tuple(out.shape) != (B, H, S, D):
            raise ValueError("q, k, v, out must all be [B, H, S_local, D]")
        if lse is not None and tuple(lse.shape) != (B, H, S):
            raise ValueError("lse must be [B, H, S_local]")
        mype = self.rank if rank is None else int(rank)
        # seqlens: rows held by every rank when the shards differ in length (the reference's seqlen[], csrc/ring.h:9)
        table = [S] * self.world if seqlens is None else [int(x) for x in seqlens]
        if len(table) != self.world or table[mype] != S:
            raise ValueError("seqlens must list every rank's rows and agree with this rank's tensors")
        p = set_params_fprop(q, k, v, out, self.world, mype, table, D, max(table), batch=B, heads=H, lse=lse,
                             causal=causal, softmax_scale=softmax_scale, stream=stream)
        self.forward_params(p)

    def forward_host(self, q, k, v, out, lse=None, *, chunks: int = 4, causal: bool = False,
                     softmax_scale: Optional[float] = None, stream=None, rank: Optional[int] = None) -> None:
        """Same forward with HOST tensors (pinned CPU torch tensors [B, H, S_local, D]): copies in, computes and
        copies out in `chunks` overlapping groups of (batch, head) slabs.  Asynchronous on `stream`; when the
        stream reaches the end of the call, `out` / `lse` hold the results."""
        import torch
        B, H, S, D = q.shape
        for x, n in ((q, "q"), (k, "k"), (v, "v"), (out, "out")):
            if x.is_cuda or not x.is_contiguous() or not x.is_pinned():
                raise ValueError(f"{n} must be a contiguous pinned host tensor")
            if tuple(x.shape) != (B, H, S, D):
                raise ValueError("q, k, v, out must all be [B, H, S_local, D]")
        if q.dtype not in _half_types() or out.dtype != torch.float32:
            raise ValueError("q, k, v must be fp16/bf16 and out fp32")
        if lse is not None and (lse.is_cuda or not lse.is_pinned() or tuple(lse.shape) != (B, H, S)):
            raise ValueError("lse must be a pinned host tensor [B, H, S_local]")
        mype = self.rank if rank is None else int(rank)
        p = set_params_fprop(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), self.world, mype, [S] * self.world,
                             D, S, batch=B, heads=H, lse=None if lse is None else lse.data_ptr(), causal=causal,
                             softmax_scale=softmax_scale, stream=stream)
        p.is_bf16 = int(q.dtype == torch.bfloat16)
        check(_lib.load().ring_attention_fwd_host(self._h, ctypes.byref(p), int(chunks)), "ring_attention_fwd_host")

    def synchronize(self, timeout_ms: Optional[int] = None) -> None:
        """Waits for everything the context enqueued.  With timeout_ms the wait is polled from the host and raises
        RingError (code RING_ERR_HOST_TIMEOUT) when the deadline passes; the context stays usable."""
        if timeout_ms is None:
            check(_lib.load().ring_ctx_synchronize(self._h), "ring_ctx_synchronize")
        else:
            check(_lib.load().ring_ctx_synchronize_timeout(self._h, int(timeout_ms)), "ring_ctx_synchronize_timeout")

    def timings(self):
        """(compute_ms, comm_ms, exposed_ms) lists of the last forward, one entry per ring step."""
        n = self.world
        a, b, c = ((ctypes.c_float * n)() for _ in range(3))
        check(_lib.load().ring_ctx_get_timings(self._h, a, b, c, n), "ring_ctx_get_timings")
        return list(a), list(b), list(c)

    def exchange_timings(self):
        """(wait_ms, copy_ms) lists of the last forward's exchanges, one entry per ring step: time spent waiting
        for the go-ahead, and the transfer itself."""
        n = self.world
        a, b = ((ctypes.c_float * n)() for _ in range(2))
        check(_lib.load().ring_ctx_get_exchange_timings(self._h, a, b, n), "ring_ctx_get_exchange_timings")
        return list(a), list(b)

    def abort(self) -> None:
        """After synchronize(timeout_ms=...) raised RING_ERR_HOST_TIMEOUT: release every queued wait of this context
        from the host, abort its communicator and mark it dead; destroy() then returns without waiting for the device."""
        check(_lib.load().ring_ctx_abort(self._h), "ring_ctx_abort")

    def destroy(self) -> None:
        if self._h:
            _lib.load().ring_ctx_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.destroy()
        except Exception:
            pass


def attention_block_fwd(q, k, v, o, lse, *, softmax_scale: Optional[float] = None, causal: bool = False,
                        q_off: int = 0, k_off: int = 0, merge: bool = False, stream=None) -> None:
    """One Q shard [B,H,Sq,D] against one K/V shard [B,H,Sk,D] -> o [B,H,Sq,D] fp32, lse [B,H,Sq] fp32."""
    import torch
    B, H, Sq, D = q.shape
    Sk = k.shape[2]
    if tuple(k.shape) != (B, H, Sk, D) or tuple(v.shape) != (B, H, Sk, D):
        raise ValueError("k, v must be [B, H, Sk, D]")
    if tuple(o.shape) != (B, H, Sq, D) or tuple(lse.shape) != (B, H, Sq):
        raise ValueError("o must be [B, H, Sq, D] and lse [B, H, Sq]")
    scale = float(softmax_scale) if softmax_scale is not None else 1.0 / math.sqrt(D)
    check(_lib.load().ring_attention_block_fwd(
        _ptr(q, "q", _half_types()), _ptr(k, "k", _half_types()), _ptr(v, "v", _half_types()),
        _ptr(o, "o", (torch.float32,)), _ptr(lse, "lse", (torch.float32,)), B, H, Sq, Sk, D, scale,
        int(bool(causal)), int(q_off), int(k_off), int(bool(merge)), int(q.dtype == torch.bfloat16),
        _stream_handle(stream)), "ring_attention_block_fwd")


def lse_merge(o_acc, lse_acc, o_part, lse_part, *, stream=None) -> None:
    """(o_acc, lse_acc) <- merge with (o_part, lse_part); tensors [..., D] fp32 and [...] fp32."""
    import torch
    D = o_acc.shape[-1]
    rows = lse_acc.numel()
    if o_acc.numel() != rows * D or o_part.numel() != rows * D or lse_part.numel() != rows:
        raise ValueError("shape mismatch between the partials")
    f32 = (torch.float32,)
    check(_lib.load().ring_lse_merge(_ptr(o_acc, "o_acc", f32), _ptr(lse_acc, "lse_acc", f32),
                                     _ptr(o_part, "o_part", f32), _ptr(lse_part, "lse_part", f32),
                                     rows, D, _stream_handle(stream)), "ring_lse_merge")


def device_status() -> int:
    s = ctypes.c_int(0)
    check(_lib.load().ring_device_status(ctypes.byref(s)), "ring_device_status")
    return s.value


def device_status_reset() -> None:
    check(_lib.load().ring_device_status_reset(), "ring_device_status_reset")


def kernel_launch_count() -> int:
    return int(_lib.load().ring_kernel_launch_count())


def attention_chunked_fwd_static(q, k, v, o, lse, kv_chunk: int, *, softmax_scale: Optional[float] = None,
                                 causal: bool = False, stream=None) -> None:
    """Attention of q [B,H,Sq,D] against k/v [B,H,Sk,D], `kv_chunk` key rows at a time, for hosts that do
    not let this library allocate device memory (a runtime that owns the whole GPU, a fixed memory budget).
    Nothing is allocated: the partial of each chunk lives in a fixed ~16 MiB array inside the library, so
    B*H*Sq <= 65536 rows and B*H*Sq*D <= 4 Mi floats, and calls that overlap on the GPU would race on it.
    The first call on a device also does the one-time set-up; make it before any stream capture."""
    import torch
    B, H, Sq, D = q.shape
    Sk = k.shape[2]
    if tuple(k.shape) != (B, H, Sk, D) or tuple(v.shape) != (B, H, Sk, D):
        raise ValueError("k, v must be [B, H, Sk, D]")
    if tuple(o.shape) != (B, H, Sq, D) or tuple(lse.shape) != (B, H, Sq):
        raise ValueError("o must be [B, H, Sq, D] and lse [B, H, Sq]")
    scale = float(softmax_scale) if softmax_scale is not None else 1.0 / math.sqrt(D)
    check(_lib.load().ring_attention_chunked_fwd_static(
        _ptr(q, "q", _half_types()), _ptr(k, "k", _half_types()), _ptr(v, "v", _half_types()),
        _ptr(o, "o", (torch.float32,)), _ptr(lse, "lse", (torch.float32,)), B, H, Sq, Sk, D, scale,
        int(bool(causal)), int(kv_chunk), int(q.dtype == torch.bfloat16), _stream_handle(stream)),
        "ring_attention_chunked_fwd_static")


def static_status(stream=None) -> int:
    """Status word of the no-allocation path: waits for `stream`, then returns 0 or the code of the bounded wait that
    ran out inside the last attention_chunked_fwd_static() on this device (its outputs are then invalid)."""
    s = ctypes.c_int(0)
    check(_lib.load().ring_static_status(ctypes.byref(s), _stream_handle(stream)), "ring_static_status")
    return s.value


# ---- paged K/V cache ------------------------------------------------------------------------------------------------
# The conventions (pages, places, lengths, masks) are those of the C ABI, include/ring_attention_b200.h.  Tensors may have any
# strides there that are multiples of 8 elements with the last dimension contiguous.  Every call runs on the device of its
# tensors, on `stream` (default: torch's current stream of that device), and returns without waiting.

def _strided(x, what: str, ndim: int, dtypes, device=None):
    """(address, strides) of a CUDA tensor whose last dimension is contiguous; strides of one-element dimensions count as 0."""
    if not hasattr(x, "data_ptr"):
        raise TypeError(f"{what}: expected a CUDA tensor")
    if not x.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor")
    if x.dim() != ndim:
        raise ValueError(f"{what} must have {ndim} dimensions, got {x.dim()}")
    if x.dtype not in dtypes:
        raise ValueError(f"{what} has dtype {x.dtype}, expected one of {tuple(dtypes)}")
    if device is not None and x.device != device:
        raise ValueError(f"{what} is on {x.device}, expected {device}")
    if x.shape[-1] > 1 and x.stride(-1) != 1:
        raise ValueError(f"the last dimension of {what} must be contiguous")
    return x.data_ptr(), [0 if n == 1 else s for n, s in zip(x.shape[:-1], x.stride()[:-1])]


def _distinct(x, what: str) -> None:
    if any(n > 1 and s == 0 for n, s in zip(x.shape, x.stride())):
        raise ValueError(f"{what} is written to and must not be an expanded tensor")


def _fill_cache(p, k_cache, v_cache, page_table, kv_lens) -> None:
    import torch
    half, dev = _half_types(), k_cache.device
    p.k_cache, (p.k_page_stride, p.k_head_stride, p.k_place_stride) = _strided(k_cache, "k_cache", 4, half)
    p.num_pages, p.kv_heads, p.page_size, p.dim = k_cache.shape
    if v_cache is not None:
        p.v_cache, (p.v_page_stride, p.v_head_stride, p.v_place_stride) = _strided(v_cache, "v_cache", 4, (k_cache.dtype,), dev)
        if v_cache.shape != k_cache.shape:
            raise ValueError("k_cache and v_cache must both be [pages, kv_heads, page_size, dim]")
    p.page_table, (p.table_stride,) = _strided(page_table, "page_table", 2, (torch.int32,), dev)
    p.batch, p.max_pages = page_table.shape
    p.kv_lens, _ = _strided(kv_lens, "kv_lens", 1, (torch.int32,), dev)
    if kv_lens.shape[0] != p.batch:
        raise ValueError("kv_lens must have one entry per row of page_table")


def _fill_tokens(p, tokens: int, cu_seqlens, max_new: int, device) -> None:
    import torch
    p.tokens, p.max_new = int(tokens), int(max_new)
    if cu_seqlens is not None:
        p.cu_seqlens, _ = _strided(cu_seqlens, "cu_seqlens", 1, (torch.int32,), device)
        if cu_seqlens.shape[0] != p.batch + 1:
            raise ValueError("cu_seqlens must have batch + 1 entries")


def _fill_queries(p, q, k_cache, lse, softmax_scale, causal, window, sinks) -> None:
    import torch
    p.q, (p.q_token_stride, p.q_head_stride) = _strided(q, "q", 3, (k_cache.dtype,), k_cache.device)
    p.heads = q.shape[1]
    if q.shape[2] != p.dim:
        raise ValueError("q must be [tokens, heads, dim] with the cache's dim")
    if tuple(lse.shape) != tuple(q.shape[:2]) or not lse.is_contiguous():
        raise ValueError("lse must be a contiguous [tokens, heads]")
    p.lse, _ = _strided(lse, "lse", 2, (torch.float32,), k_cache.device)
    p.softmax_scale = float(softmax_scale) if softmax_scale is not None else 1.0 / math.sqrt(p.dim)
    p.causal, p.window, p.sinks = int(bool(causal)), int(window), int(sinks)
    p.is_bf16 = int(q.dtype == torch.bfloat16)


def _fill_weights(p, weights, device) -> None:
    import torch
    p.weights, (p.weights_batch_stride, p.weights_head_stride) = _strided(weights, "weights", 3, (torch.float32,), device)
    if tuple(weights.shape[:2]) != (p.batch, p.kv_heads):
        raise ValueError("weights must be [batch, kv_heads, places]")
    p.weights_len = weights.shape[2]


def _on(device, stream):
    """(context, handle): the device made current, the stream the call goes to."""
    import torch
    ctx = torch.cuda.device(device)
    if stream is None:
        return ctx, torch.cuda.current_stream(device).cuda_stream
    return ctx, _stream_handle(stream)


def _workspace(p, size, workspace, device, where: str):
    """The caller's scratch, or one from torch's allocator for the stream the call goes to, so that the allocator orders the
    memory's next user behind this call."""
    import torch
    if workspace is None:
        n = size(ctypes.byref(p))
        if n < 0:
            check(int(n), where)
        with torch.cuda.stream(torch.cuda.ExternalStream(p.stream, device) if p.stream else torch.cuda.default_stream(device)):
            workspace = torch.empty(int(n), dtype=torch.uint8, device=device)
    p.workspace, _ = _strided(workspace, "workspace", 1, (torch.uint8,), device)
    p.workspace_bytes = workspace.numel()
    return workspace


def paged_append(k, v, k_cache, v_cache, page_table, kv_lens, *, cu_seqlens=None, weights=None, stream=None) -> None:
    """Write the new tokens' rows k, v [tokens, kv_heads, dim] to their places in the pages.

    k_cache, v_cache [pages, kv_heads, page_size, dim]; page_table [batch, max_pages], kv_lens [batch] int32, the lengths
    WITH the new tokens; cu_seqlens [batch + 1] int32 if the sequences bring different numbers of tokens.  weights (see
    paged_weights) start at 0 at the new places."""
    p = _lib.Ring_paged_params()
    _fill_cache(p, k_cache, v_cache, page_table, kv_lens)
    dev = k_cache.device
    p.k_new, (p.k_new_token_stride, p.k_new_head_stride) = _strided(k, "k", 3, (k_cache.dtype,), dev)
    p.v_new, (p.v_new_token_stride, p.v_new_head_stride) = _strided(v, "v", 3, (k_cache.dtype,), dev)
    if tuple(k.shape) != (k.shape[0], p.kv_heads, p.dim) or v.shape != k.shape:
        raise ValueError("k and v must both be [tokens, kv_heads, dim]")
    for x, n in ((k_cache, "k_cache"), (v_cache, "v_cache"), (weights, "weights")):
        if x is not None:
            _distinct(x, n)
    _fill_tokens(p, k.shape[0], cu_seqlens, 0, dev)
    if weights is not None:
        _fill_weights(p, weights, dev)
    ctx, p.stream = _on(dev, stream)
    with ctx:
        check(_lib.load().ring_paged_append(ctypes.byref(p)), "ring_paged_append")


def _workspace_bytes(name: str, q, k_cache, page_table, cu_seqlens, max_new) -> int:
    import torch
    p = _lib.Ring_paged_params()
    p.kv_heads, p.dim, p.heads, p.softmax_scale = k_cache.shape[1], k_cache.shape[3], q.shape[1], 1.0
    p.batch, p.max_pages = page_table.shape
    _fill_tokens(p, q.shape[0], cu_seqlens, max_new, k_cache.device)
    with torch.cuda.device(k_cache.device):
        n = getattr(_lib.load(), name)(ctypes.byref(p))
    if n < 0:
        check(int(n), name)
    return int(n)


def paged_attention_workspace(q, k_cache, page_table, *, cu_seqlens=None, max_new: int = 0) -> int:
    """Bytes of scratch paged_attention_fwd needs for tensors of these shapes (independent of what they hold)."""
    return _workspace_bytes("ring_paged_attention_workspace", q, k_cache, page_table, cu_seqlens, max_new)


def paged_weights_workspace(q, k_cache, page_table, *, cu_seqlens=None, max_new: int = 0) -> int:
    """Bytes of scratch paged_weights needs for tensors of these shapes; 0: none."""
    return _workspace_bytes("ring_paged_weights_workspace", q, k_cache, page_table, cu_seqlens, max_new)


def paged_attention_fwd(q, k_cache, v_cache, page_table, kv_lens, out, lse, *, cu_seqlens=None, max_new: int = 0,
                        softmax_scale: Optional[float] = None, causal: bool = True, window: int = 0, sinks: int = 0,
                        workspace=None, stream=None) -> None:
    """Attention of the new tokens q [tokens, heads, dim] over the paged cache (append their rows first).

    heads is a multiple of the cache's kv_heads.  A token at place p of its sequence sees the places <= p (causal) or all of
    kv_lens (causal=False); with window > 0 only those > p - window, and the first `sinks`.  out [tokens, heads, dim] in q's
    type or fp32 (then lse_merge joins the partials of several caches), lse [tokens, heads] fp32.  max_new: an upper
    bound on the new tokens of one sequence when cu_seqlens is given (helps to choose the kernel).
    workspace: a uint8 tensor of paged_attention_workspace() bytes of the caller's, for this call alone while it runs;
    by default one comes from torch's allocator."""
    import torch
    p = _lib.Ring_paged_params()
    _fill_cache(p, k_cache, v_cache, page_table, kv_lens)
    dev = k_cache.device
    _fill_queries(p, q, k_cache, lse, softmax_scale, causal, window, sinks)
    _fill_tokens(p, q.shape[0], cu_seqlens, max_new, dev)
    if out.shape != q.shape:
        raise ValueError("out must have q's shape")
    p.out, (p.out_token_stride, p.out_head_stride) = _strided(out, "out", 3, (q.dtype, torch.float32), dev)
    _distinct(out, "out")
    p.out_fp32 = int(out.dtype == torch.float32)
    ctx, p.stream = _on(dev, stream)
    with ctx:
        lib = _lib.load()
        keep = _workspace(p, lib.ring_paged_attention_workspace, workspace, dev, "ring_paged_attention_fwd")
        check(lib.ring_paged_attention_fwd(ctypes.byref(p)), "ring_paged_attention_fwd")
        del keep  # until here


def paged_weights(weights, q, k_cache, lse, page_table, kv_lens, *, cu_seqlens=None, max_new: int = 0,
                  softmax_scale: Optional[float] = None, causal: bool = True, window: int = 0, sinks: int = 0, workspace=None, stream=None) -> None:
    """weights [batch, kv_heads, places] fp32 += the attention that every cached place received from the new tokens: exp(s - lse)
    summed over the tokens that see it and the query heads of its K/V head, with the lse of paged_attention_fwd for the same
    arguments.  places >= max_pages * page_size.  workspace as for paged_attention_fwd, of paged_weights_workspace() bytes."""
    p = _lib.Ring_paged_params()
    _fill_cache(p, k_cache, None, page_table, kv_lens)
    _fill_queries(p, q, k_cache, lse, softmax_scale, causal, window, sinks)
    _fill_tokens(p, q.shape[0], cu_seqlens, max_new, k_cache.device)
    _fill_weights(p, weights, k_cache.device)
    _distinct(weights, "weights")
    ctx, p.stream = _on(k_cache.device, stream)
    with ctx:
        lib = _lib.load()
        keep = _workspace(p, lib.ring_paged_weights_workspace, workspace, k_cache.device, "ring_paged_weights")
        check(lib.ring_paged_weights(ctypes.byref(p)), "ring_paged_weights")
        del keep  # until here


def paged_evict(k_cache, v_cache, weights, page_table, kv_lens, dst_table, budget: int, new_lens, new_weights, kept, *,
                first: int = 0, recent: int = 0, stream=None) -> None:
    """Keep at most `budget` places of every sequence and K/V head -- the first `first`, the last `recent` and the heaviest of the
    others by weights [batch, kv_heads, places] (ties: the lowest place) -- and copy their rows, in order, to the pages
    dst_table [batch, pages] int32 names, which must not hold places of the sources.  new_lens [batch] int32,
    new_weights [batch, kv_heads, >= budget] fp32 (0 behind the kept) and kept [batch, kv_heads, budget] int32 (-1 behind) are
    written."""
    import torch
    p = _lib.Ring_evict_params()
    _fill_cache(p, k_cache, v_cache, page_table, kv_lens)
    dev = k_cache.device
    _fill_weights(p, weights, dev)
    for x, n in ((k_cache, "k_cache"), (v_cache, "v_cache"), (new_weights, "new_weights")):
        _distinct(x, n)
    p.dst_table, (p.dst_stride,) = _strided(dst_table, "dst_table", 2, (torch.int32,), dev)
    if dst_table.shape[0] != p.batch:
        raise ValueError("dst_table must have one row per row of page_table")
    p.dst_pages = dst_table.shape[1]
    p.budget, p.first, p.recent = int(budget), int(first), int(recent)
    p.new_weights, (p.new_weights_batch_stride, p.new_weights_head_stride) = _strided(new_weights, "new_weights", 3, (torch.float32,), dev)
    if tuple(new_weights.shape[:2]) != (p.batch, p.kv_heads):
        raise ValueError("new_weights must be [batch, kv_heads, places]")
    p.new_weights_len = new_weights.shape[2]
    if tuple(kept.shape) != (p.batch, p.kv_heads, p.budget) or not kept.is_contiguous():
        raise ValueError("kept must be a contiguous [batch, kv_heads, budget]")
    p.kept, _ = _strided(kept, "kept", 3, (torch.int32,), dev)
    p.new_lens, _ = _strided(new_lens, "new_lens", 1, (torch.int32,), dev)
    if new_lens.shape[0] != p.batch:
        raise ValueError("new_lens must have one entry per sequence")
    ctx, p.stream = _on(dev, stream)
    with ctx:
        check(_lib.load().ring_paged_evict(ctypes.byref(p)), "ring_paged_evict")
