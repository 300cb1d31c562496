"""Python face of the engine: same entry points as the reference's ``directkv/kernel/__init__.py``
(``smpv2_fwd`` :225-257, ``smpv2_init_tma`` :260-279, ``smpv2_fwd_graph`` :282-314 and the
``directkv_*`` aliases the non-smpv2 backend asks for, directkv/directkv_backend.py:83-93), plus
the ragged, page-tabled decode call the B200 engine is built around.

Everything here only checks tensors, turns them into pointers and calls the C ABI; there is no
torch compute and no fallback.
"""

from __future__ import annotations

import ctypes as C
import math
import struct
from typing import Optional, Sequence

import torch

from . import _lib
from ._lib import DKV_NEW_GIVEN, DKV_NEW_NONE, DKV_NEW_PROJECT, PARTIAL_STRIDE, DecodeArgs, LayerDesc, get_context

HEAD_DIM = 128


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _chk(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def _check_cuda_bf16(t: torch.Tensor, name: str) -> None:
    _chk(t.is_cuda, f"{name} must be a CUDA tensor")
    _chk(t.is_contiguous(), f"{name} must be contiguous")
    _chk(t.dtype == torch.bfloat16, f"{name} must be bfloat16")


def _check_kv(t: torch.Tensor, name: str) -> None:
    """KV storage: pinned host memory (the reference's only mode) or device memory (HBM-resident mode)."""
    _chk(t.is_contiguous(), f"{name} must be contiguous")
    _chk(t.dtype == torch.bfloat16, f"{name} must be bfloat16")
    if not t.is_cuda:
        _chk(t.is_pinned(), f"{name} must be a CPU tensor in pinned memory (or a CUDA tensor)")


def _check_cos_sin(cos_sin: Optional[torch.Tensor]) -> None:
    if cos_sin is None:
        return
    _chk(cos_sin.is_cuda, "cos_sin must be a CUDA tensor")
    _chk(cos_sin.dtype == torch.float32, "cos_sin must be float32")
    _chk(cos_sin.dim() == 2, "cos_sin must be 2D [max_pos, head_dim]")
    _chk(cos_sin.size(1) == HEAD_DIM, f"cos_sin.size(1) must equal head_dim={HEAD_DIM}, got {cos_sin.size(1)}")
    _chk(cos_sin.is_contiguous(), "cos_sin must be contiguous")


# ---------------------------------------------------------------------------
# Layer registration and the ragged decode call
# ---------------------------------------------------------------------------
def register_layer(
    layer_id: int,
    k_pool: torch.Tensor,            # [n_slots, NH_kv, 128] bf16 pinned-CPU or CUDA (any leading dims that flatten to slots)
    v_pool: torch.Tensor,
    wk: Optional[torch.Tensor] = None,   # [NH_kv, 128, H] bf16 CUDA
    wv: Optional[torch.Tensor] = None,
    cos_sin: Optional[torch.Tensor] = None,  # [max_pos, 128] fp32 CUDA
    page_size: int = 1,
    row_stride: int = 0,
    device: Optional[int] = None,
) -> None:
    """Builds and caches the TMA descriptors of one layer's KV pool and projection weights.

    Takes the place of ``smpv2_init_tma`` (directkv/kernel/smpv2_extension.cu:363-423).  The
    pool is used IN PLACE: nothing is copied, so what the engine stores for new tokens is
    visible to every later reader of the pool tensor.
    """
    _check_kv(k_pool, "k_pool")
    _check_kv(v_pool, "v_pool")
    _chk(k_pool.shape == v_pool.shape, "k_pool and v_pool must have the same shape")
    _chk(k_pool.dim() >= 3 and k_pool.size(-1) == HEAD_DIM, f"pool must be [..., NH_kv, {HEAD_DIM}]")
    nh_kv = k_pool.size(-2)
    n_slots = k_pool.numel() // (nh_kv * HEAD_DIM)
    hidden = 0
    if wk is not None:
        _check_cuda_bf16(wk, "Wk")
        _check_cuda_bf16(wv, "Wv")
        _chk(wk.dim() == 3 and wk.shape == wv.shape, "Wk/Wv must be 3D [NH, D, H] and equal in shape")
        _chk(wk.size(0) == nh_kv and wk.size(1) == HEAD_DIM, "Wk must be [NH_kv, 128, H] for this pool")
        hidden = wk.size(2)
    _check_cos_sin(cos_sin)
    ctx = get_context(device)
    d = LayerDesc(
        k_pool=_ptr(k_pool), v_pool=_ptr(v_pool), n_slots=n_slots, nh_kv=nh_kv, page_size=page_size,
        row_stride=row_stride, wk=_ptr(wk), wv=_ptr(wv), hidden=hidden, cos_sin=_ptr(cos_sin),
        max_pos=0 if cos_sin is None else cos_sin.size(0),
    )
    _lib.check(_lib.load().dkv_layer_register(ctx.handle, int(layer_id), C.byref(d)))
    ctx._keepalive[int(layer_id)] = (k_pool, v_pool, wk, wv, cos_sin)


def unregister_layer(layer_id: int, device: Optional[int] = None) -> None:
    ctx = get_context(device)
    _lib.check(_lib.load().dkv_layer_unregister(ctx.handle, int(layer_id)))
    ctx._keepalive.pop(int(layer_id), None)


def decode(
    layer_id: int,
    q: torch.Tensor,                      # [B, NH_q*128] or [B, NH_q, 128] bf16 CUDA
    seq_lens: torch.Tensor,               # [B] int32 CUDA, lengths INCLUDING the token decoded now
    softmax_scale: float,
    page_table: Optional[torch.Tensor] = None,   # [rows, max_pages] int32 CUDA; None = contiguous rows
    row_map: Optional[torch.Tensor] = None,      # [B] int32 CUDA
    x: Optional[torch.Tensor] = None,            # [B, H] bf16 CUDA -> project the new token's K/V
    k_new: Optional[torch.Tensor] = None,        # [B, NH_kv, 128] bf16 CUDA (already rotated)
    v_new: Optional[torch.Tensor] = None,
    save_kv_cache: bool = True,
    out: Optional[torch.Tensor] = None,
    lse_out: Optional[torch.Tensor] = None,
    partial_out: Optional[torch.Tensor] = None,  # [B, NH_q, 132] fp32: unnormalised (O, m, l)
    normalized: bool = True,
    pos_offset: Optional[torch.Tensor] = None,   # [B] int32 CUDA: added to seq_len-1 for the RoPE position
    exchange=None,                               # handle of a connected peer-memory exchange (sharding.PartialExchange)
    kv_source_layer: int = 0,                    # attend a copy of the past rows registered as this layer (0: off)
    src_page_table: Optional[torch.Tensor] = None,   # addressing of the copy (its page size) ...
    src_row_map: Optional[torch.Tensor] = None,      # ... or its rows
) -> Optional[torch.Tensor]:
    """One decode step of one registered layer for a ragged batch.  Returns O with q's shape.

    With ``exchange`` the call is this rank's part of a sequence-split decode: partial records go to
    every rank's exchange buffer over NVLink and ``out`` is the merged result of all ranks.
    """
    _check_cuda_bf16(q, "q")
    b = q.size(0)
    nh_q = q.numel() // (b * HEAD_DIM) if b else 0
    _chk(seq_lens.is_cuda and seq_lens.dtype == torch.int32 and seq_lens.is_contiguous(), "seq_lens must be int32 CUDA")
    _chk(seq_lens.numel() == b, "seq_lens must have one entry per request")
    if page_table is not None:
        _chk(page_table.is_cuda and page_table.dtype == torch.int32 and page_table.dim() == 2
             and page_table.stride(1) == 1, "page_table must be 2D int32 CUDA with unit inner stride")
    if row_map is not None:
        _chk(row_map.is_cuda and row_map.dtype == torch.int32 and row_map.numel() == b, "row_map must be [B] int32 CUDA")
    mode = DKV_NEW_NONE
    if x is not None:
        _check_cuda_bf16(x, "x")
        _chk(x.dim() == 2 and x.size(0) == b, "x must be [B, H]")
        mode = DKV_NEW_PROJECT
    elif k_new is not None:
        _check_cuda_bf16(k_new, "k_new")
        _check_cuda_bf16(v_new, "v_new")
        mode = DKV_NEW_GIVEN
    if normalized and out is None:
        out = torch.empty_like(q)
    if out is not None:
        _check_cuda_bf16(out, "out")
    if lse_out is not None:
        _chk(lse_out.is_cuda and lse_out.dtype == torch.float32 and lse_out.numel() == b * nh_q, "lse_out must be [B, NH_q] fp32 CUDA")
    if partial_out is not None:
        _chk(partial_out.is_cuda and partial_out.dtype == torch.float32 and partial_out.is_contiguous()
             and partial_out.numel() == b * nh_q * PARTIAL_STRIDE, "partial_out must be [B, NH_q, 132] fp32 CUDA")
    if pos_offset is not None:
        _chk(pos_offset.is_cuda and pos_offset.dtype == torch.int32 and pos_offset.numel() == b, "pos_offset must be [B] int32 CUDA")
    if src_page_table is not None:
        _chk(kv_source_layer != 0 and src_page_table.is_cuda and src_page_table.dtype == torch.int32
             and src_page_table.dim() == 2 and src_page_table.stride(1) == 1,
             "src_page_table needs kv_source_layer and must be 2D int32 CUDA with unit inner stride")
    if src_row_map is not None:
        _chk(kv_source_layer != 0 and src_row_map.is_cuda and src_row_map.dtype == torch.int32 and src_row_map.numel() == b,
             "src_row_map needs kv_source_layer and must be [B] int32 CUDA")
    if b == 0:
        return out
    a = DecodeArgs(
        layer_id=int(layer_id), batch=b, nh_q=nh_q, q=_ptr(q), q_stride=nh_q * HEAD_DIM,
        out=_ptr(out), out_stride=nh_q * HEAD_DIM, seq_lens=_ptr(seq_lens),
        page_table=_ptr(page_table), pt_stride=0 if page_table is None else page_table.stride(0),
        row_map=_ptr(row_map), new_mode=mode, x=_ptr(x), k_new=_ptr(k_new), v_new=_ptr(v_new),
        save_kv_cache=1 if save_kv_cache else 0, softmax_scale=float(softmax_scale),
        lse_out=_ptr(lse_out), partial_out=_ptr(partial_out), pos_offset=_ptr(pos_offset),
        kv_source_layer=int(kv_source_layer), src_page_table=_ptr(src_page_table),
        src_pt_stride=0 if src_page_table is None else src_page_table.stride(0), src_row_map=_ptr(src_row_map),
        pt_rows=0 if page_table is None else page_table.size(0),
    )
    ctx = get_context(q.device.index)
    if exchange is not None:
        _lib.check(_lib.load().dkv_decode_exchange(ctx.handle, exchange, C.byref(a), _ptr(out), _ptr(lse_out), _stream()))
    else:
        _lib.check(_lib.load().dkv_decode(ctx.handle, C.byref(a), _stream()))
    return out


def extend(
    layer_id: int,
    X: torch.Tensor,                  # [B, S_new, H] bf16 CUDA
    Q: torch.Tensor,                  # [B, S_new, NH_q, 128] bf16 CUDA
    softmax_scale: float,
    is_causal: bool,
    seqlen_past: int,
    q_pos_start: int = -1,
    row_map: Optional[torch.Tensor] = None,   # [B] int32 CUDA: pool row of each request
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Extend / chunked prefill on the rows of a registered layer (no descriptor rebuild).

    The kernel call of ``forward_extend`` (directkv/directkv_backend.py:681-697): the new rows'
    K/V are projected, rotated and stored at ``[row, seqlen_past + i]`` of the pool in place.
    """
    _check_cuda_bf16(X, "X")
    _check_cuda_bf16(Q, "Q")
    _chk(X.dim() == 3 and Q.dim() == 4 and Q.size(3) == HEAD_DIM, "X must be [B,S_new,H] and Q [B,S_new,NH_q,128]")
    B, S_new, _ = X.shape
    _chk(Q.size(0) == B and Q.size(1) == S_new, "Q must match X in batch and S_new")
    if row_map is not None:
        _chk(row_map.is_cuda and row_map.dtype == torch.int32 and row_map.numel() == B, "row_map must be [B] int32 CUDA")
    if out is None:
        out = torch.empty_like(Q)
    _check_cuda_bf16(out, "out")
    ctx = get_context(X.device.index)
    _lib.check(_lib.load().dkv_extend(
        ctx.handle, int(layer_id), _ptr(X), _ptr(Q), _ptr(out), B, S_new, Q.size(2), float(softmax_scale),
        1 if is_causal else 0, int(seqlen_past), int(q_pos_start), _ptr(row_map), _stream()))
    return out


def extend_attend(
    layer_id: int,
    Q: torch.Tensor,                  # [B, S_new, NH_q, 128] bf16 CUDA
    softmax_scale: float,
    is_causal: bool,
    seqlen_past: int,
    row_map: Optional[torch.Tensor] = None,      # [B] int32 CUDA: pool row / page-table row of each request
    page_table: Optional[torch.Tensor] = None,   # [rows, max_pages] int32 CUDA (page size of the registered layer)
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Attention of new rows that are already stored in the pool (``dkv_extend_attend``): the engine's form of
    ``_sdpa_extend_manual`` (directkv/directkv_backend.py:861-891) on the tensor-core extend kernel."""
    _check_cuda_bf16(Q, "Q")
    _chk(Q.dim() == 4 and Q.size(3) == HEAD_DIM, "Q must be [B,S_new,NH_q,128]")
    B, S_new = Q.size(0), Q.size(1)
    if row_map is not None:
        _chk(row_map.is_cuda and row_map.dtype == torch.int32 and row_map.numel() == B, "row_map must be [B] int32 CUDA")
    pt_stride = 0
    if page_table is not None:
        _chk(page_table.is_cuda and page_table.dtype == torch.int32 and page_table.dim() == 2 and page_table.stride(1) == 1,
             "page_table must be a 2-D int32 CUDA tensor with unit inner stride")
        pt_stride = page_table.stride(0)
    if out is None:
        out = torch.empty_like(Q)
    _check_cuda_bf16(out, "out")
    ctx = get_context(Q.device.index)
    _lib.check(_lib.load().dkv_extend_attend(
        ctx.handle, int(layer_id), _ptr(Q), _ptr(out), B, S_new, Q.size(2), float(softmax_scale),
        1 if is_causal else 0, int(seqlen_past), _ptr(row_map), _ptr(page_table), int(pt_stride), _stream()))
    return out


def extend_ragged(
    layer_id: int,
    X: Optional[torch.Tensor],        # [T, H] bf16 CUDA, or None when the new rows are stored already
    Q: torch.Tensor,                  # [T, NH_q, 128] bf16 CUDA: the requests' rows one after the other
    s_new: Sequence[int],             # new rows per request (host)
    past: Sequence[int],              # stored rows per request (host)
    rows: Sequence[int],              # pool row / page-table row per request (host)
    softmax_scale: float,
    is_causal: bool = True,
    page_table: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Extend of a ragged batch in one launch sequence (``dkv_extend_ragged``); the reference calls its kernel
    once per request (directkv/directkv_backend.py:681-697)."""
    import ctypes as C

    _check_cuda_bf16(Q, "Q")
    _chk(Q.dim() == 3 and Q.size(2) == HEAD_DIM, "Q must be [T,NH_q,128]")
    B = len(s_new)
    _chk(len(past) == B and len(rows) == B and B > 0, "s_new, past and rows must have one entry per request")
    _chk(int(sum(int(n) for n in s_new)) == Q.size(0), "sum(s_new) must equal the rows of Q")
    if X is not None:
        _check_cuda_bf16(X, "X")
        _chk(X.dim() == 2 and X.size(0) == Q.size(0), "X must be [T,H]")
    pt_stride = 0
    if page_table is not None:
        _chk(page_table.is_cuda and page_table.dtype == torch.int32 and page_table.dim() == 2 and page_table.stride(1) == 1,
             "page_table must be a 2-D int32 CUDA tensor with unit inner stride")
        pt_stride = page_table.stride(0)
    if out is None:
        out = torch.empty_like(Q)
    _check_cuda_bf16(out, "out")
    arr = C.c_int32 * B
    a_new, a_past, a_rows = arr(*[int(v) for v in s_new]), arr(*[int(v) for v in past]), arr(*[int(v) for v in rows])
    ctx = get_context(Q.device.index)
    _lib.check(_lib.load().dkv_extend_ragged(
        ctx.handle, int(layer_id), _ptr(X), _ptr(Q), _ptr(out), B, C.cast(a_new, C.c_void_p), C.cast(a_past, C.c_void_p),
        C.cast(a_rows, C.c_void_p), Q.size(1), float(softmax_scale), 1 if is_causal else 0, _ptr(page_table),
        int(pt_stride), _stream()))
    return out


def decode_noalloc(
    k_pool: torch.Tensor,        # [n_slots, NH_kv, 128] bf16, pinned CPU or CUDA
    v_pool: torch.Tensor,
    q: torch.Tensor,             # [B, NH_q, 128] or [B, NH_q*128] bf16 CUDA
    out: torch.Tensor,           # same shape as q, pre-allocated by the caller
    seq_lens: torch.Tensor,      # [B] int32 CUDA; every attended token is already in the pool
    page_table: torch.Tensor,    # [B, max_pages] int32 CUDA
    page_size: int,
    softmax_scale: float,
    lse_out: Optional[torch.Tensor] = None,
    sync_and_check: bool = False,
    status_out: Optional[torch.Tensor] = None,   # [1] int32 CUDA of the caller's: failure bits are OR-ed into it
) -> torch.Tensor:
    """Attention-only decode that allocates no device memory (``dkv_decode_noalloc``).

    For callers that cannot allocate when they call in: graph-capture regions, serving loops with
    a frozen memory plan, hosts that forbid ``cudaMalloc`` from plugins.  The caller passes every
    tensor, output included; scratch is a fixed 4 MiB array inside the library, shared by all
    calls, so calls that overlap on the GPU race and sizes beyond the array are rejected with
    ``RuntimeError``.  The first call on a device does a one-time set-up and should happen
    before any stream capture.  Needs no registered layer and no context.
    """
    _check_kv(k_pool, "k_pool")
    _check_kv(v_pool, "v_pool")
    _check_cuda_bf16(q, "q")
    _check_cuda_bf16(out, "out")
    _chk(out.shape == q.shape, "out must have q's shape")
    _chk(k_pool.dim() >= 3 and k_pool.size(-1) == HEAD_DIM and k_pool.shape == v_pool.shape, "pools must be [..., NH_kv, 128]")
    b = q.size(0)
    nh_q = q.numel() // (b * HEAD_DIM)
    nh_kv = k_pool.size(-2)
    _chk(seq_lens.is_cuda and seq_lens.dtype == torch.int32 and seq_lens.numel() == b, "seq_lens must be [B] int32 CUDA")
    _chk(page_table.is_cuda and page_table.dtype == torch.int32 and page_table.dim() == 2 and page_table.stride(1) == 1,
         "page_table must be 2D int32 CUDA with unit inner stride")
    if status_out is not None:
        _chk(status_out.is_cuda and status_out.dtype == torch.int32 and status_out.numel() >= 1,
             "status_out must be an int32 CUDA tensor")
    err = C.create_string_buffer(512)
    a = _lib.NoAllocArgs(
        k_pool=_ptr(k_pool), v_pool=_ptr(v_pool), n_slots=k_pool.numel() // (nh_kv * HEAD_DIM), nh_kv=nh_kv,
        page_size=int(page_size), batch=b, nh_q=nh_q, q=_ptr(q), q_stride=nh_q * HEAD_DIM, out=_ptr(out),
        out_stride=nh_q * HEAD_DIM, seq_lens=_ptr(seq_lens), page_table=_ptr(page_table),
        pt_stride=page_table.stride(0), softmax_scale=float(softmax_scale), lse_out=_ptr(lse_out),
        sync_and_check=1 if sync_and_check else 0, err_buf=C.cast(err, C.c_char_p), err_buf_len=512,
        status_out=_ptr(status_out),
    )
    with torch.cuda.device(q.device):
        rc = _lib.load().dkv_decode_noalloc(C.byref(a), _stream())
    if rc != _lib.DKV_OK:
        raise RuntimeError(f"directkv_b200 error {rc}: {err.value.decode()}")
    return out


def merge_partials(parts: torch.Tensor, out: Optional[torch.Tensor] = None,
                   lse_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Combines ``parts [R, rows, 132]`` (one unnormalised partial set per rank) into ``[rows, 128]`` bf16."""
    _chk(parts.is_cuda and parts.dtype == torch.float32 and parts.is_contiguous() and parts.dim() == 3
         and parts.size(2) == PARTIAL_STRIDE, "parts must be [R, rows, 132] fp32 CUDA contiguous")
    r, rows = parts.size(0), parts.size(1)
    if out is None:
        out = torch.empty(rows, HEAD_DIM, dtype=torch.bfloat16, device=parts.device)
    ctx = get_context(parts.device.index)
    _lib.check(_lib.load().dkv_merge_partials(ctx.handle, _ptr(parts), r, rows, _ptr(out), _ptr(lse_out), _stream()))
    return out


def stream_copy(dst: torch.Tensor, src: torch.Tensor) -> None:
    """SM-issued copy of ``src`` (pinned host or device) into ``dst`` (device): host-link probe."""
    nbytes = src.numel() * src.element_size()
    _chk(dst.is_cuda and dst.numel() * dst.element_size() >= nbytes, "dst must be a CUDA tensor at least as large as src")
    ctx = get_context(dst.device.index)
    _lib.check(_lib.load().dkv_stream_copy(ctx.handle, _ptr(dst), _ptr(src), nbytes, _stream()))


# ---------------------------------------------------------------------------
# A paged cache held in 4 bits, and what a decode step over it needs beside the attention
# ---------------------------------------------------------------------------
# These calls are short on the GPU, so the host side is kept short too: arguments are packed straight into the C structs' bytes, and a
# contiguous tensor is recognised by one question.
KV4_BLOCK = 16          # consecutive dimensions that share a scale
_BF16, _I32, _I64, _F32 = torch.bfloat16, torch.int32, torch.int64, torch.float32
_pack_decode_kv4 = struct.Struct("@iiiPqPqPPqiiPfP").pack     # _lib.DecodeKv4Args
_pack_qk_norm = struct.Struct("@qiiPqPqPqPqPPiiiiPiPif").pack  # _lib.QkNormArgs
_pack_pages = struct.Struct("@PqiiPPPiiPiP").pack              # _lib.PagesArgs


def _call(dev: int):
    """Handle of the device's context and the raw handle of torch's current stream there."""
    ctx = _lib._contexts.get(dev) or get_context(dev)
    return ctx.handle, torch._C._cuda_getCurrentRawStream(dev)


def _elsewhere(name: str) -> None:
    raise RuntimeError(f"{name} must be a CUDA tensor on the same device as the other tensors")


def _int32_1d(t: torch.Tensor, n: int, name: str) -> None:
    if t.dtype is not _I32 or t.shape != (n,) or not t.is_contiguous():
        raise RuntimeError(f"{name} must be a contiguous int32 tensor of {n} entries")


def _heads_stride(t: torch.Tensor, name: str) -> int:
    """Elements from token to token of ``[..., NH, 128]`` whose heads lie next to each other (a slice of a fused
    projection's output is fine)."""
    shape = t.shape
    if t.dtype is _BF16 and len(shape) in (3, 4) and shape[-1] == HEAD_DIM:
        row = shape[-2] * HEAD_DIM
        if t.is_contiguous():
            return row
        st = t.stride()
        if st[-1] == 1 and (st[-2] == HEAD_DIM or shape[-2] == 1):
            if len(shape) == 3:
                return st[0] if shape[0] > 1 else row
            if shape[0] == 1 or shape[1] == 1 or st[0] == shape[1] * st[1]:
                return st[1] if shape[1] > 1 else (st[0] if shape[0] > 1 else row)
            raise RuntimeError(f"{name} must have evenly spaced tokens")
    raise RuntimeError(f"{name} must be bfloat16 [..., NH, {HEAD_DIM}], 3D or 4D, with the heads of a token next to each other")


def _check_page_table(t: torch.Tensor) -> None:
    if t.dtype is not _I32 or t.dim() != 2 or not (t.is_contiguous() or t.stride(1) == 1):
        raise RuntimeError("page_table must be 2D int32 with unit inner stride")


class KV4Pool:
    """One layer's K and V pool in 4 bits (the format stands in include/directkv_b200.h at ``dkv_kv4_pool``).

    ``k_codes`` / ``v_codes`` are uint8 ``[n_slots, NH_kv, 64]``, ``k_scales`` / ``v_scales`` uint8 ``[n_slots, NH_kv, 8]`` (e4m3
    bytes), in device memory or page-locked host memory.  Token ``t`` of a request lies at slot
    ``page_table[row, t // page_size] * page_size + t % page_size``.  ``k_scale`` / ``v_scale`` are powers of two that
    the stored values are multiplied by; values above 2688 times the scale are cut off.
    """

    __slots__ = ("k_codes", "k_scales", "v_codes", "v_scales", "page_size", "k_scale", "v_scale", "n_slots", "nh_kv", "_descs")

    def __init__(self, k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor, v_scales: torch.Tensor,
                 page_size: int = 1, k_scale: float = 1.0, v_scale: float = 1.0):
        _chk(k_codes.dim() == 3, "k_codes must be 3D [n_slots, NH_kv, 64]")
        n_slots, nh = k_codes.size(0), k_codes.size(1)
        for t, width, name in ((k_codes, HEAD_DIM // 2, "k_codes"), (v_codes, HEAD_DIM // 2, "v_codes"),
                               (k_scales, HEAD_DIM // KV4_BLOCK, "k_scales"), (v_scales, HEAD_DIM // KV4_BLOCK, "v_scales")):
            _chk(t.dtype == torch.uint8 and t.is_contiguous() and tuple(t.shape) == (n_slots, nh, width),
                 f"{name} must be contiguous uint8 [{n_slots}, {nh}, {width}]")
            _chk(t.device == k_codes.device, f"{name} must be on the device of k_codes")
            _chk(t.is_cuda or t.is_pinned() or not torch.cuda.is_available(), f"{name} must be in pinned memory (or a CUDA tensor)")
        _chk(page_size >= 1 and page_size & (page_size - 1) == 0, f"page_size ({page_size}) must be a power of two")
        _chk(n_slots > 0 and n_slots % page_size == 0, f"the number of slots ({n_slots}) must be a positive multiple of page_size ({page_size})")
        for s, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
            _chk(2.0 ** -24 <= s <= 2.0 ** 24 and math.frexp(s)[0] == 0.5, f"{name} must be a power of two from 2^-24 to 2^24")
        self.k_codes, self.k_scales, self.v_codes, self.v_scales = k_codes, k_scales, v_codes, v_scales
        self.page_size, self.k_scale, self.v_scale = int(page_size), float(k_scale), float(v_scale)
        self.n_slots, self.nh_kv = n_slots, nh
        self._descs = {}
        if k_codes.is_cuda:
            self._resolve(k_codes.get_device())
        elif torch.cuda.is_available():
            self._resolve(torch.cuda.current_device())

    @classmethod
    def empty(cls, n_slots: int, nh_kv: int, page_size: int = 1, device="cuda", k_scale: float = 1.0, v_scale: float = 1.0) -> "KV4Pool":
        """A pool of zeros; ``device="cpu"`` puts it in page-locked host memory (beside the current GPU where the
        machine has more than one memory node)."""
        from .sglang_compat import pinned_zeros

        def make(width):
            if torch.device(device).type == "cpu":
                return pinned_zeros((n_slots, nh_kv, width), torch.uint8)
            return torch.zeros(n_slots, nh_kv, width, dtype=torch.uint8, device=device)

        c, s = HEAD_DIM // 2, HEAD_DIM // KV4_BLOCK
        return cls(make(c), make(s), make(c), make(s), page_size, k_scale, v_scale)

    def nbytes(self) -> int:
        return 2 * self.n_slots * self.nh_kv * (HEAD_DIM // 2 + HEAD_DIM // KV4_BLOCK)

    def _resolve(self, dev: int):
        """The C struct for one device, checked and resolved by the library on first use (never under stream capture: it
        makes room for the attention's workspace)."""
        if self.k_codes.is_cuda and self.k_codes.get_device() != dev:
            raise RuntimeError("the pool must be on the device of the other tensors")
        d = _lib.Kv4PoolDesc(_ptr(self.k_codes), _ptr(self.k_scales), _ptr(self.v_codes), _ptr(self.v_scales), self.n_slots,
                             self.nh_kv, self.page_size, self.k_scale, self.v_scale, 0)
        _lib.check(_lib.load().dkv_kv4_pool_resolve((_lib._contexts.get(dev) or get_context(dev)).handle, C.byref(d)))
        self._descs[dev] = ref = C.byref(d)
        return ref


def _check_slots(slots: torch.Tensor) -> int:
    if (slots.dtype is not _I32 and slots.dtype is not _I64) or slots.dim() != 1 or not slots.is_contiguous():
        raise RuntimeError("slots must be a contiguous 1D int32 or int64 tensor")
    return slots.numel()


def store_kv4(pool: KV4Pool, slots: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> None:
    """Quantises row ``i`` of ``k`` / ``v`` ``[n, NH_kv, 128]`` (bf16, tokens may be strided) into slot ``slots[i]``.

    A slot of -1 stands for no token (``assign_pages`` gives it to the padding of a batch): its row is passed over.  Other slots
    outside the pool are not written and reported in the status word, and so are infinities (stored as the largest value)
    and not-a-numbers (stored as zero).  Slots must be distinct, save for a padding slot that nobody attends.
    """
    n = _check_slots(slots)
    want = (n, pool.nh_kv, HEAD_DIM)
    if k.shape != want or v.shape != want:
        raise RuntimeError(f"k and v must be [{n}, {pool.nh_kv}, {HEAD_DIM}]")
    ks, vs = _heads_stride(k, "k"), _heads_stride(v, "v")
    dev = k.get_device()
    if dev < 0 or v.get_device() != dev or slots.get_device() != dev:
        _elsewhere("k, v and slots each")
    if n == 0:
        return
    handle, stream = _call(dev)
    rc = _lib.load().dkv_kv4_store(handle, pool._descs.get(dev) or pool._resolve(dev), slots.data_ptr(), slots.dtype is _I64, k.data_ptr(), ks,
                                   v.data_ptr(), vs, n, stream)
    if rc:
        _lib.check(rc)


def load_kv4(pool: KV4Pool, slots: torch.Tensor, k_out: Optional[torch.Tensor] = None, v_out: Optional[torch.Tensor] = None):
    """The values of ``slots`` as bf16 ``(k, v)``, each ``[n, NH_kv, 128]``; exact.  A slot outside the pool gives zeros and
    is reported in the status word, but for -1 (no token)."""
    n = _check_slots(slots)
    dev = slots.get_device()
    if dev < 0:
        _elsewhere("slots")
    shape = (n, pool.nh_kv, HEAD_DIM)
    if k_out is None and v_out is None:
        k_out = slots.new_empty_strided(shape, (pool.nh_kv * HEAD_DIM, HEAD_DIM, 1), dtype=_BF16)
        v_out = torch.empty_like(k_out)
    if k_out is None:
        k_out = torch.empty(shape, dtype=_BF16, device=slots.device)
    elif k_out.dtype is not _BF16 or k_out.shape != shape or not k_out.is_contiguous() or k_out.get_device() != dev:
        raise RuntimeError(f"k_out must be contiguous bfloat16 [{n}, {pool.nh_kv}, {HEAD_DIM}] on the device of slots")
    if v_out is None:
        v_out = torch.empty_like(k_out)
    elif v_out.dtype is not _BF16 or v_out.shape != shape or not v_out.is_contiguous() or v_out.get_device() != dev:
        raise RuntimeError(f"v_out must be contiguous bfloat16 [{n}, {pool.nh_kv}, {HEAD_DIM}] on the device of slots")
    if n:
        handle, stream = _call(dev)
        rc = _lib.load().dkv_kv4_load(handle, pool._descs.get(dev) or pool._resolve(dev), slots.data_ptr(), slots.dtype is _I64,
                                      k_out.data_ptr(), v_out.data_ptr(), n, stream)
        if rc:
            _lib.check(rc)
    return k_out, v_out


def decode_kv4(
    q: torch.Tensor,                  # [B, NH_q, 128], [B, n_q, NH_q, 128] or [B, NH_q*128] bf16 CUDA (tokens may be strided)
    pool: KV4Pool,
    seq_lens: torch.Tensor,           # [B] int32 CUDA: stored tokens, the query tokens' own included
    softmax_scale: float,
    page_table: torch.Tensor,         # [rows, max_pages] int32 CUDA
    row_map: Optional[torch.Tensor] = None,   # [B] int32 CUDA
    out: Optional[torch.Tensor] = None,
    lse_out: Optional[torch.Tensor] = None,   # [B, NH_q] or [B, n_q, NH_q] fp32
) -> torch.Tensor:
    """Decode attention over a 4-bit pool whose tokens are all stored (``store_kv4``).  Returns O with q's shape.

    With ``n_q`` query tokens per request, token ``j`` attends the first ``seq_lens - n_q + 1 + j`` stored tokens (drafted
    tokens under verification, a short chunk of a prompt).  A row that attends nothing is zero, its LSE -inf.
    """
    shape = q.shape
    nd = len(shape)
    if nd == 3:
        b, nh_q, _ = shape
        n_q = 1
        qs = _heads_stride(q, "q")
    elif nd == 2:
        if shape[1] % HEAD_DIM or shape[1] == 0:
            raise RuntimeError(f"q must be [B, NH_q*{HEAD_DIM}]")
        b, nh_q, n_q = shape[0], shape[1] // HEAD_DIM, 1
        qs = _heads_stride(q.view(b, nh_q, HEAD_DIM), "q")
    else:
        qs = _heads_stride(q, "q")
        b, n_q, nh_q, _ = shape
    if nh_q == 0 or nh_q % pool.nh_kv:
        raise RuntimeError(f"q has {nh_q} heads, not a multiple of the pool's {pool.nh_kv}")
    if b > 4096 or not 1 <= n_q <= 1024:
        raise RuntimeError(f"{b} requests of {n_q} query tokens: at most 4096 of 1 to 1024")
    _int32_1d(seq_lens, b, "seq_lens")
    _check_page_table(page_table)
    rows, max_pages = page_table.shape
    dev = q.get_device()
    row_ptr = lse_ptr = 0
    if row_map is not None:
        _int32_1d(row_map, b, "row_map")
        if row_map.get_device() != dev:
            _elsewhere("row_map")
        if rows == 0 < b:                                     # (to the library 0 rows mean an unknown number)
            raise RuntimeError(f"page_table has no rows for {b} requests")
        row_ptr = row_map.data_ptr()
    elif rows < b:
        raise RuntimeError(f"page_table has {rows} rows for {b} requests")
    if lse_out is not None:
        if lse_out.dtype is not _F32 or lse_out.numel() != b * n_q * nh_q or not lse_out.is_contiguous() or lse_out.get_device() != dev:
            raise RuntimeError("lse_out must be contiguous fp32 CUDA with one entry per query row")
        lse_ptr = lse_out.data_ptr()
    if dev < 0 or seq_lens.get_device() != dev or page_table.get_device() != dev:
        _elsewhere("q, seq_lens and page_table each")
    row = nh_q * HEAD_DIM
    if out is None:
        out = torch.empty_like(q)                             # (contiguous for a slice of a fused projection, too)
        os = row
    else:
        if out.shape != shape or out.get_device() != dev:
            raise RuntimeError("out must have q's shape and device")
        os = _heads_stride(out.view(b, nh_q, HEAD_DIM) if nd == 2 else out, "out")
    if b == 0:
        return out
    handle, stream = _call(dev)
    a = _pack_decode_kv4(b, n_q, nh_q, q.data_ptr(), qs, out.data_ptr(), os, seq_lens.data_ptr(), page_table.data_ptr(),
                         page_table.stride(0), rows, max_pages, row_ptr, softmax_scale, lse_ptr)
    rc = _lib.load().dkv_decode_kv4(handle, pool._descs.get(dev) or pool._resolve(dev), a, stream)
    if rc:
        _lib.check(rc)
    return out


def _norm_side(x, y, w, n: int, dev: int, name: str):
    """Output and struct fields of the queries or the keys."""
    shape, st = x.shape, x.stride()
    if len(shape) != 3 or shape[0] != n:
        raise RuntimeError(f"{name} must be [{n}, NH, {HEAD_DIM}]")
    nh = shape[1]
    row = nh * HEAD_DIM
    if x.dtype is not _BF16 or shape[2] != HEAD_DIM or st[2] != 1 or (st[1] != HEAD_DIM and nh > 1):
        _heads_stride(x, name)                                # raises
    if y is None:
        y, ys = torch.empty_like(x), row                      # (contiguous for a slice of a fused projection, too)
    else:
        if y.shape != shape or y.get_device() != dev:
            raise RuntimeError(f"{name}_out must have the shape of {name} and its device")
        ys = _heads_stride(y, f"{name}_out")
    per_head = f32 = w_ptr = 0
    if w is not None:
        f32, w_shape = w.dtype is _F32, w.shape
        per_head = len(w_shape) == 2
        if not (f32 or w.dtype is _BF16) or w_shape != ((nh, HEAD_DIM) if per_head else (HEAD_DIM,)) or not w.is_contiguous() or w.get_device() != dev:
            raise RuntimeError(f"{name}_weight must be contiguous bfloat16 or float32 [{HEAD_DIM}] or [{nh}, {HEAD_DIM}], a CUDA tensor on the device of {name}")
        w_ptr = w.data_ptr()
    if dev < 0 or x.get_device() != dev:
        _elsewhere(name)
    return y, nh, x.data_ptr(), st[0] if n > 1 else row, y.data_ptr(), ys, w_ptr, f32, per_head


def qk_norm_rope(
    q: Optional[torch.Tensor],        # [T, NH_q, 128] bf16 CUDA (tokens may be strided: a slice of a fused projection)
    k: Optional[torch.Tensor],        # [T, NH_kv, 128]
    positions: Optional[torch.Tensor],     # [T] int32 or int64 CUDA
    cos_sin: Optional[torch.Tensor],       # [max_pos, 128] fp32 CUDA = [cos | sin]; None: no rotation
    q_weight: Optional[torch.Tensor] = None,   # [128] or [NH, 128], bf16 or fp32; None: no norm
    k_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    q_out: Optional[torch.Tensor] = None,      # may be q itself (in place)
    k_out: Optional[torch.Tensor] = None,
):
    """RMS norm of every query and key head and the Neox rotation at the tokens' positions, in one pass.

    Returns ``(q_out, k_out)``; the norm of q or k is left out where it has no weight.  Computed in fp32 and rounded
    once.  A position outside the table leaves its token unrotated and is reported in the status word.
    """
    lead = q if q is not None else k
    if lead is None:
        raise RuntimeError("q or k must be given")
    n, dev = lead.shape[0], lead.get_device()
    qy, hq, qp, qs, qo, qos, qw, qf, qh = _norm_side(q, q_out, q_weight, n, dev, "q") if q is not None else (None, 0, 0, 0, 0, 0, 0, 0, 0)
    ky, hk, kp, ks, ko, kos, kw, kf, kh = _norm_side(k, k_out, k_weight, n, dev, "k") if k is not None else (None, 0, 0, 0, 0, 0, 0, 0, 0)
    max_pos = pos_ptr = pos64 = cs_ptr = 0
    if cos_sin is not None:
        if cos_sin.dtype is not _F32 or cos_sin.dim() != 2 or cos_sin.shape[1] != HEAD_DIM or not cos_sin.is_contiguous() or cos_sin.shape[0] == 0:
            raise RuntimeError(f"cos_sin must be contiguous float32 [max_pos, {HEAD_DIM}]")
        pos64 = positions is not None and positions.dtype is _I64
        if positions is None or not (pos64 or positions.dtype is _I32) or positions.shape != (n,) or not positions.is_contiguous():
            raise RuntimeError(f"positions must be a contiguous int32 or int64 tensor of {n} entries")
        if cos_sin.get_device() != dev or positions.get_device() != dev:
            _elsewhere("cos_sin and positions each")
        max_pos, pos_ptr, cs_ptr = cos_sin.shape[0], positions.data_ptr(), cos_sin.data_ptr()
    if not eps >= 0.0:
        raise RuntimeError("eps must not be negative")
    if n:
        handle, stream = _call(dev)
        a = _pack_qk_norm(n, hq, hk, qp, qs, kp, ks, qo, qos, ko, kos, qw, kw, qf, kf, qh, kh, pos_ptr, pos64, cs_ptr, max_pos, eps)
        rc = _lib.load().dkv_qk_norm_rope(handle, a, stream)
        if rc:
            _lib.check(rc)
    return qy, ky


def _pages_refuse(page_table, lens, more, more_name, free_pages, n_free, page_size, rows) -> None:
    """Says what is wrong with the arguments of assign_pages or release_pages."""
    b = lens.numel()
    _int32_1d(lens, b, "lens")
    _int32_1d(more, b, more_name)
    _check_page_table(page_table)
    if page_table.shape[0] > 1 and page_table.stride(0) < page_table.shape[1]:
        raise RuntimeError("the rows of page_table must not overlap")
    if free_pages.dtype is not _I32 or free_pages.dim() != 1 or not free_pages.is_contiguous():
        raise RuntimeError("free_pages must be a contiguous 1D int32 tensor")
    _int32_1d(n_free, 1, "n_free")
    if b > 4096:
        raise RuntimeError(f"{b} requests: at most 4096 per call")
    if page_size < 1 or page_size & (page_size - 1):
        raise RuntimeError(f"page_size ({page_size}) must be a power of two")
    if rows is not None:
        _int32_1d(rows, b, "rows")
    _elsewhere(f"page_table, lens, {more_name}, free_pages, n_free and rows each")


def _pages_args(page_table, lens, more, more_name, free_pages, n_free, page_size, rows):
    n_rows, max_pages = page_table.shape if page_table.dim() == 2 else (0, 0)
    b, stride, dev = lens.numel(), page_table.stride(0), page_table.get_device()
    # One pass over what is right; what is wrong is told apart in _pages_refuse.
    if not (page_table.dtype is _I32 and lens.dtype is _I32 and more.dtype is _I32 and free_pages.dtype is _I32 and n_free.dtype is _I32
            and page_table.dim() == 2 and lens.dim() == 1 and free_pages.dim() == 1 and n_free.dim() == 1 and n_free.numel() == 1
            and more.shape == lens.shape and b <= 4096 and (n_rows <= 1 or stride >= max_pages)
            and (page_table.is_contiguous() or page_table.stride(1) == 1) and lens.is_contiguous() and more.is_contiguous() and free_pages.is_contiguous()
            and page_size >= 1 and page_size & (page_size - 1) == 0
            and lens.get_device() == dev >= 0 and more.get_device() == dev and free_pages.get_device() == dev and n_free.get_device() == dev
            and (rows is None or (rows.dtype is _I32 and rows.shape == lens.shape and rows.is_contiguous() and rows.get_device() == dev))):
        _pages_refuse(page_table, lens, more, more_name, free_pages, n_free, page_size, rows)
    return dev, b, _pack_pages(page_table.data_ptr(), stride, n_rows, max_pages, 0 if rows is None else rows.data_ptr(), lens.data_ptr(),
                               more.data_ptr(), b, page_size, free_pages.data_ptr(), free_pages.numel(), n_free.data_ptr())


def assign_pages(
    page_table: torch.Tensor,         # [rows, max_pages] int32 CUDA, updated
    lens: torch.Tensor,               # [B] int32 CUDA: tokens stored so far
    new_lens: torch.Tensor,           # [B] int32 CUDA: tokens to come
    free_pages: torch.Tensor,         # [N] int32 CUDA: a stack of page numbers, free_pages[:n_free] are free
    n_free: torch.Tensor,             # [1] int32 CUDA, updated
    page_size: int,
    n_tokens: int,                    # room for the new tokens: their sum, or an upper bound of it
    rows: Optional[torch.Tensor] = None,       # [B] int32 CUDA: row of the table of each request; None: row b
    slots: Optional[torch.Tensor] = None,      # outputs (int32 CUDA), allocated where not given
    positions: Optional[torch.Tensor] = None,
    seq_lens: Optional[torch.Tensor] = None,   # may be ``lens`` itself
    cu_new: Optional[torch.Tensor] = None,
):
    """Gives every request pages for its new tokens, on the GPU: no host copy of the lengths, capturable in a CUDA graph.

    Returns ``(slots [n_tokens], positions [n_tokens], seq_lens [B], cu_new [B + 1])``: slot and position of each new token
    packed in request order, the lengths with the new tokens, and the packed offsets.  Behind the last token a slot becomes -1,
    which ``store_kv4`` and ``load_kv4`` pass over, and a position 0 (given tensors: entries that are negative there are
    left as they were).  The call takes effect as a whole or not at all: when the pages run out, a length does not fit the
    table or ``n_tokens``, or two requests with new tokens have one row, everything is left as it was, the slots are -1 and
    the status word says why.  A page number that gives no slot (a held page that was never entered in the table) is reported
    there, too; its tokens have slot -1.
    """
    dev, b, a = _pages_args(page_table, lens, new_lens, "new_lens", free_pages, n_free, page_size, rows)
    if not 0 <= n_tokens < 2 ** 31:
        raise RuntimeError(f"n_tokens ({n_tokens}) must be 0..2^31-1")
    fresh = (slots is None) + 2 * (positions is None)
    if slots is None and positions is None and seq_lens is None and cu_new is None:
        pad = -n_tokens & 3                                   # positions 16-byte aligned as well
        room = lens.new_empty_strided((2 * n_tokens + pad + 2 * b + 1,), (1,))
        if pad:
            slots, _, positions, seq_lens, cu_new = room.split_with_sizes((n_tokens, pad, n_tokens, b, b + 1))
        else:
            slots, positions, seq_lens, cu_new = room.split_with_sizes((n_tokens, n_tokens, b, b + 1))
    else:
        outs = []
        for t, n, name in ((slots, n_tokens, "slots"), (positions, n_tokens, "positions"), (seq_lens, b, "seq_lens"), (cu_new, b + 1, "cu_new")):
            if t is None:
                t = lens.new_empty(n)
            else:
                _int32_1d(t, n, name)
                if t.get_device() != dev:
                    _elsewhere(name)
            outs.append(t)
        slots, positions, seq_lens, cu_new = outs
    handle, stream = _call(dev)
    rc = _lib.load().dkv_assign_pages_fresh(handle, a, slots.data_ptr(), positions.data_ptr(), n_tokens, seq_lens.data_ptr(), cu_new.data_ptr(), fresh, stream)
    if rc:
        _lib.check(rc)
    return slots, positions, seq_lens, cu_new


def release_pages(
    page_table: torch.Tensor,
    lens: torch.Tensor,               # [B] int32 CUDA: tokens stored
    keep_lens: torch.Tensor,          # [B] int32 CUDA: tokens that stay (0: all of the request's pages are freed)
    free_pages: torch.Tensor,
    n_free: torch.Tensor,
    page_size: int,
    rows: Optional[torch.Tensor] = None,
) -> None:
    """Puts the pages behind the tokens that stay back on the stack of free pages, on the GPU.

    A release of exactly what the last ``assign_pages`` gave restores the stack.  The table's entries are left; nothing reads
    them once the lengths are shorter.  As a whole or not at all, like ``assign_pages``; two requests that give pages of one
    row back are refused.
    """
    dev, b, a = _pages_args(page_table, lens, keep_lens, "keep_lens", free_pages, n_free, page_size, rows)
    if b == 0:
        return
    handle, stream = _call(dev)
    rc = _lib.load().dkv_release_pages(handle, a, stream)
    if rc:
        _lib.check(rc)


# ---------------------------------------------------------------------------
# Reference-shaped entry points
# ---------------------------------------------------------------------------
def smpv2_fwd(
    X: torch.Tensor,                  # [B, S_new, hidden_dim]      GPU bf16
    Wk: torch.Tensor,                 # [NH, head_dim, hidden_dim]  GPU bf16
    Wv: torch.Tensor,
    Q: torch.Tensor,                  # [B, S_new, NH_q, head_dim]  GPU bf16
    K_cpu: torch.Tensor,              # [B, S_total, NH, head_dim]  CPU-pinned bf16 (or CUDA: HBM mode)
    V_cpu: torch.Tensor,
    cos_sin: Optional[torch.Tensor],  # [max_pos, head_dim] GPU fp32, or None
    softmax_scale: float,
    is_causal: bool,
    seqlen_past: int,
    q_pos_start: int,
) -> torch.Tensor:
    """Fused forward: X->K,V projection + Neox RoPE + attention (directkv/kernel/__init__.py:225-257).

    Same arguments and result as the reference.  Unlike the reference, ``seqlen_past`` and
    ``S_new`` may be any positive sizes and the projection contracts the full hidden size.
    """
    _chk(X.dim() == 3, f"X must be 3D [B, S_new, H], got {X.dim()}D")
    _chk(Wk.dim() == 3, "Wk must be 3D [NH, D, H]")
    _chk(Wv.dim() == 3, "Wv must be 3D [NH, D, H]")
    _chk(Q.dim() == 4, "Q must be 4D [B, S_new, NH, D]")
    _chk(K_cpu.dim() == 4, "K_cpu must be 4D [B, S_total, NH, D]")
    _chk(V_cpu.dim() == 4, "V_cpu must be 4D [B, S_total, NH, D]")
    for t, n in ((X, "X"), (Wk, "Wk"), (Wv, "Wv"), (Q, "Q")):
        _check_cuda_bf16(t, n)
    _check_kv(K_cpu, "K_cpu")
    _check_kv(V_cpu, "V_cpu")
    _chk(Q.size(3) == HEAD_DIM, f"head_dim must be {HEAD_DIM}, got {Q.size(3)}")
    _chk(Q.size(2) % Wk.size(0) == 0,
         f"Q.size(2) (NH_q={Q.size(2)}) must be a multiple of Wk.size(0) (NH_kv={Wk.size(0)})")
    _check_cos_sin(cos_sin)
    B, S_new, H = X.shape
    nh_kv, nh_q = Wk.size(0), Q.size(2)
    S_total = K_cpu.size(1)
    _chk(Wk.size(1) == HEAD_DIM and Wk.size(2) == H and Wv.shape == Wk.shape, "Wk/Wv must be [NH, 128, H]")
    _chk(Q.size(0) == B and Q.size(1) == S_new, "Q must match X in batch and S_new")
    _chk(K_cpu.size(0) == B and K_cpu.size(2) == nh_kv and K_cpu.size(3) == HEAD_DIM and V_cpu.shape == K_cpu.shape,
         "K_cpu/V_cpu must be [B, S_total, NH_kv, 128]")
    O = torch.empty(B, S_new, nh_q, HEAD_DIM, dtype=torch.bfloat16, device=X.device)
    ctx = get_context(X.device.index)
    _lib.check(_lib.load().dkv_smpv2_fwd(
        ctx.handle, _ptr(X), _ptr(Wk), _ptr(Wv), _ptr(Q), _ptr(K_cpu), _ptr(V_cpu), _ptr(cos_sin),
        0 if cos_sin is None else cos_sin.size(0), B, S_new, H, nh_q, nh_kv, S_total,
        float(softmax_scale), 1 if is_causal else 0, int(seqlen_past), int(q_pos_start), _ptr(O), _stream()))
    return O


def smpv2_init_tma(
    layer_id: int,
    X_max: torch.Tensor,     # [max_bs, S_new_max, H]          GPU bf16
    Wk: torch.Tensor,        # [NH, D, H]                      GPU bf16
    Wv: torch.Tensor,
    Q_max: torch.Tensor,     # [max_bs, S_new_max, NH, D]      GPU bf16
    K_max: torch.Tensor,     # [n_pool, S_total_max, NH, D]    CPU-pinned bf16
    V_max: torch.Tensor,
    cos_sin: Optional[torch.Tensor] = None,
) -> None:
    """Per-layer set-up before graph capture (directkv/kernel/__init__.py:260-279).

    Registers the layer (descriptors for K_max/V_max rows and the weights) and pre-sizes
    scratch for ``max_bs * S_new_max`` query rows so that ``smpv2_fwd_graph`` allocates nothing.
    ``cos_sin`` is an addition: the reference passes the table on every call instead.
    """
    for t, n in ((X_max, "X_max"), (Wk, "Wk"), (Wv, "Wv"), (Q_max, "Q_max")):
        _check_cuda_bf16(t, n)
    _check_kv(K_max, "K_max")
    _check_kv(V_max, "V_max")
    _chk(K_max.dim() == 4 and X_max.dim() == 3 and Q_max.dim() == 4, "bad tensor ranks")
    register_layer(layer_id, K_max, V_max, Wk, Wv, cos_sin, page_size=1, row_stride=K_max.size(1),
                   device=X_max.device.index)
    ctx = get_context(X_max.device.index)
    ctx.reserve(X_max.size(0) * X_max.size(1), Q_max.size(2), Wk.size(0), X_max.size(2))


def smpv2_fwd_graph(
    layer_id: int,
    X_pad: torch.Tensor,         # [bs, S_new, H]        GPU bf16
    Q_pad: torch.Tensor,         # [bs, S_new, NH, D]    GPU bf16
    O_out: torch.Tensor,         # [bs, S_new, NH, D]    GPU bf16 (pre-allocated output)
    n_past_dev: torch.Tensor,    # [1] int32 GPU: number of past 64-token blocks for this step
    n_blks_dev: torch.Tensor,    # [1] int32 GPU (kept for signature compatibility; = n_past + S_new/64)
    cos_sin: Optional[torch.Tensor],
    softmax_scale: float,
    is_causal: bool,
    S_total_max: int,
    seqlen_past_max: int,
    req_pool_indices: Optional[torch.Tensor] = None,  # [bs] int32 GPU: batch_pos -> pool row
) -> torch.Tensor:
    """Graph-safe forward (directkv/kernel/__init__.py:282-314): loop bounds come from device memory."""
    for t, n in ((X_pad, "X_pad"), (Q_pad, "Q_pad"), (O_out, "O_out")):
        _check_cuda_bf16(t, n)
    _chk(n_past_dev.is_cuda and n_past_dev.dtype == torch.int32, "n_past_dev must be int32")
    _chk(n_blks_dev.is_cuda and n_blks_dev.dtype == torch.int32, "n_blks_dev must be int32")
    if req_pool_indices is not None:
        _chk(req_pool_indices.is_cuda and req_pool_indices.dtype == torch.int32, "req_pool_indices must be int32")
    B, S_new, _ = X_pad.shape
    ctx = get_context(X_pad.device.index)
    kept = ctx._keepalive.get(int(layer_id))
    if kept is not None and cos_sin is not None and (kept[4] is None or kept[4].data_ptr() != cos_sin.data_ptr()):
        # The reference passes the table per call; re-register (host-only work) when it changed.
        _check_cos_sin(cos_sin)
        register_layer(layer_id, kept[0], kept[1], kept[2], kept[3], cos_sin, page_size=1,
                       row_stride=kept[0].size(1), device=X_pad.device.index)
    _lib.check(_lib.load().dkv_smpv2_fwd_graph(
        ctx.handle, int(layer_id), _ptr(X_pad), _ptr(Q_pad), _ptr(O_out), _ptr(n_past_dev), B, S_new,
        Q_pad.size(2), float(softmax_scale), 1 if is_causal else 0, _ptr(req_pool_indices), _stream()))
    return O_out


# The plain ``directkv`` backend imports these names (directkv/directkv_backend.py:83-93).
directkv_fwd = smpv2_fwd
directkv_init_tma = smpv2_init_tma
directkv_fwd_graph = smpv2_fwd_graph
