"""Paged K/V cache: new tokens into it, and attention over it (Python side of the C ABI).

The prefill entry points (:func:`usagi_b200.block_sparse_attn_fwd`) answer one pass over a prompt.
These continue it token by token: :func:`paged_kv_append` puts the keys and values of new tokens
into the cache, rotated to their positions, and :func:`paged_attn_fwd` is the attention of the new
tokens over everything held, with the same window + global-blocks rows as
:func:`usagi_b200.block_sparse_attn_fwd_window`; :func:`shared_prefix_attn_fwd` is the same for a
batch whose sequences begin with the same pages.  Serving only: there is no backward pass here, as
there is none for the prefill.

The cache is plain tensors that the caller owns:

* ``k_pages``, ``v_pages``: fp16 or bf16 ``[n_pages, Hkv, page_size, 128]``, page_size a power of two
  from 16 to 1024.  Any strides that are multiples of 8 with a contiguous last dimension: a
  ``[n_pages, page_size, Hkv, 128]`` cache is passed as ``pages.transpose(1, 2)``.
* ``block_table``: int ``[B, max_pages]``, the pages of each sequence in order.  Entries behind a
  sequence's length are not read and may be anything.
* ``seq_lens``: int ``[B]``, tokens of each sequence, the new ones of this call included.
* ``q_lens``: int ``[B]`` or None, how many of the Tq rows of each sequence are live (None: all).
  Row t < q_lens[b] is the token at position ``seq_lens[b] - q_lens[b] + t``; the rows behind them are
  padding.

A page table entry, a length or a row count out of range is found on the device, never used as an
address, and raised by :func:`usagi_b200.check_errors` (code ``E_PAGE``).
"""
from __future__ import annotations

import ctypes
import struct
import threading
from functools import lru_cache
from typing import Optional, Tuple

import torch

from . import _lib
from .api import HEAD_DIM, BsattnError, _workspace

__all__ = ["paged_kv_append", "paged_attn_fwd", "shared_prefix_attn_fwd", "rope_inv_freq"]

# A decode step is a few microseconds of GPU time, so the host side is kept short: the call record
# is packed in one go, and the current device and stream are asked for without wrapper objects.
_PACK = _lib.PAGED_CALL.pack
_STRIDES9 = struct.Struct("@9q").pack
_HALF = (torch.float16, torch.bfloat16)
_PAGE_SIZES = frozenset(1 << i for i in range(4, 11))
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


def rope_inv_freq(rot_dim: int = HEAD_DIM, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """``base ** (-2 i / rot_dim)`` for i < rot_dim / 2 in 64 bits, for :func:`paged_kv_append`."""
    i = torch.arange(rot_dim // 2, dtype=torch.float64)
    return (float(base) ** (-2.0 * i / rot_dim)).to(device)


def _index(t: torch.Tensor, name: str, dev, shape) -> torch.Tensor:
    """``t`` as int32 on ``dev`` with a contiguous last dimension."""
    if t.shape != shape:
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype is not torch.int32 or t.device != dev:
        t = t.to(device=dev, dtype=torch.int32)
    if not t.is_contiguous() and t.stride(-1) != 1:
        t = t.contiguous()
    return t


def _rows(t: torch.Tensor, name: str, dev, dtype, shape):
    """A [B, H, T, 128] input as the kernels read it in place (16-byte rows and strides), with its
    strides and address."""
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    if t.dtype is not dtype or t.device != dev:
        raise TypeError(f"{name} must be {dtype} on {dev} like the pages, got {t.dtype} on "
                        f"{t.device}")
    s0, s1, s2, s3 = t.stride()
    at = t.data_ptr()
    if s3 != 1 or (s0 | s1 | s2) & 7 or at & 15:
        t = t.contiguous()
        if t.data_ptr() & 15:
            t = t.clone()
        s0, s1, s2, s3 = t.stride()
        at = t.data_ptr()
    return t, s0, s1, s2, at


def _cache(k_pages, v_pages, block_table, seq_lens, q_lens, B):
    """Checks of the cache arguments: (device, dtype, Hkv, max_pages, page_size, first fields of the
    call record, tensors to keep until the launch)."""
    shape = k_pages.shape
    if len(shape) != 4 or shape[3] != HEAD_DIM or v_pages.shape != shape:
        raise ValueError(f"k_pages and v_pages must be [n_pages, Hkv, page_size, {HEAD_DIM}] of one "
                         f"shape, got {tuple(shape)}, {tuple(v_pages.shape)}")
    dev, dtype = k_pages.device, k_pages.dtype
    if dtype not in _HALF or v_pages.dtype is not dtype:
        raise TypeError("k_pages and v_pages must both be float16 or both bfloat16, got "
                        f"{dtype}, {v_pages.dtype}")
    if not k_pages.is_cuda or v_pages.device != dev:
        raise ValueError("the paged cache needs CUDA tensors on one device (there is no CPU path)")
    n_pages, Hkv, page_size, _ = shape
    if n_pages == 0 or Hkv == 0:
        raise ValueError(f"the cache has no pages or no heads: {tuple(shape)}")
    if page_size not in _PAGE_SIZES:
        raise ValueError(f"page_size must be a power of two from 16 to 1024, got {page_size}")
    k0, k1, k2, k3 = k_pages.stride()
    v0, v1, v2, v3 = v_pages.stride()
    kp, vp = k_pages.data_ptr(), v_pages.data_ptr()
    if k3 != 1 or v3 != 1 or (k0 | k1 | k2 | v0 | v1 | v2) & 7 or (kp | vp) & 15:
        raise ValueError("k_pages and v_pages must be 16-byte aligned, with a contiguous last "
                         "dimension and strides that are multiples of 8")
    tshape = block_table.shape
    if len(tshape) != 2 or tshape[1] == 0:
        raise ValueError(f"block_table must be [B, max_pages], got {tuple(tshape)}")
    max_pages = tshape[1]
    table = _index(block_table, "block_table", dev, (B, max_pages))
    sl = _index(seq_lens, "seq_lens", dev, (B,))
    ql, qp = None, 0
    if q_lens is not None:
        ql = _index(q_lens, "q_lens", dev, (B,))
        qp = ql.data_ptr()
    head = (kp, vp, k0, k1, k2, v0, v1, v2, table.data_ptr(), table.stride(0), sl.data_ptr(), qp,
            max_pages, n_pages, page_size, B)
    return dev, dtype, Hkv, max_pages, page_size, head, (table, sl, ql)


@lru_cache(maxsize=4096)
def _scratch_bytes(device_index, B, Hq, Hkv, Tq, max_pages, page_size, prefix_len) -> int:
    """``bsattn_paged_scratch_bytes`` on the current device: a function of the sizes alone."""
    need = ctypes.c_size_t(0)
    rc = _lib.load().bsattn_paged_scratch_bytes(B, Hq, Hkv, Tq, max_pages, page_size, prefix_len,
                                                ctypes.byref(need))
    if rc != 0:
        raise BsattnError(rc, "bsattn_paged_scratch_bytes")
    return need.value


def paged_kv_append(k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                    seq_lens: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                    q: Optional[torch.Tensor] = None, q_lens: Optional[torch.Tensor] = None,
                    inv_freq: Optional[torch.Tensor] = None, interleaved: bool = False,
                    q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Put the keys and values of new tokens into the cache (``bsattn_paged_append``).

    k, v: ``[B, Hkv, Tq, 128]``, q: ``[B, Hq, Tq, 128]`` or None, all of the pages' dtype and with any
    strides (the slices of a fused projection are read in place).  With ``inv_freq`` (float64
    ``[rot_dim / 2]``, rot_dim a multiple of 16 up to 128; see :func:`rope_inv_freq`) the first
    rot_dim values of every row of k and q are turned by position * inv_freq[i], pairs
    (x_i, x_{i + rot_dim/2}) or, ``interleaved``, (x_2i, x_{2i+1}); angles are formed in 64 bits.  Only
    the slots of live rows are written.  Returns the rotated q, contiguous, with zeros in padding
    rows (``q_out`` when given; it may be q itself if that is contiguous), or None without q.
    """
    shape = k.shape
    if len(shape) != 4:
        raise ValueError(f"k must be [B, Hkv, Tq, {HEAD_DIM}], got {tuple(shape)}")
    B, _, Tq, _ = shape
    dev, dtype, Hkv, _, _, head, keep = _cache(k_pages, v_pages, block_table, seq_lens, q_lens, B)
    rows = (B, Hkv, Tq, HEAD_DIM)
    k, k0, k1, k2, kp = _rows(k, "k", dev, dtype, rows)
    v, v0, v1, v2, vp = _rows(v, "v", dev, dtype, rows)
    Hq = q0 = q1 = q2 = 0
    qp = qo = None
    if q is not None:
        Hq = q.shape[1] if q.dim() == 4 else 0
        if Hq == 0:
            raise ValueError(f"q must be [{B}, Hq, {Tq}, {HEAD_DIM}], got {tuple(q.shape)}")
        rows = (B, Hq, Tq, HEAD_DIM)
        q, q0, q1, q2, qp = _rows(q, "q", dev, dtype, rows)
        if q_out is None:
            q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        elif q_out.shape != rows or q_out.dtype is not dtype or q_out.device != dev \
                or not q_out.is_contiguous() or q_out.data_ptr() & 15:
            raise ValueError("q_out has the wrong shape, dtype, device, layout or alignment")
        qo = q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out needs q")
    rot, inv = 0, None
    if inv_freq is not None:
        if inv_freq.dim() != 1 or inv_freq.dtype is not torch.float64 or inv_freq.device != dev:
            raise TypeError("inv_freq must be float64 [rot_dim / 2] on the device of the pages")
        rot = 2 * inv_freq.shape[0]
        if rot % 16 or not 0 < rot <= HEAD_DIM:
            raise ValueError(f"rot_dim must be a multiple of 16 up to {HEAD_DIM}, got {rot}")
        inv_freq = inv_freq.contiguous()
        inv = inv_freq.data_ptr()
    if B == 0 or Tq == 0:
        return q_out
    flags = _lib.IN_BF16 if dtype is torch.bfloat16 else 0

    def launch():
        stream = _raw_stream(dev.index)
        ws = _workspace(dev, stream)
        return _lib.load().bsattn_paged_append(
            _PACK(*head, Hq, Hkv, Tq, flags, ws.data_ptr(), 4 * ws.numel(), stream), qp, kp, vp,
            _STRIDES9(q0, q1, q2, k0, k1, k2, v0, v1, v2), qo, inv, rot, 1 if interleaved else 0)

    rc = _on(dev, launch)
    if rc != 0:
        raise BsattnError(rc, "bsattn_paged_append")
    return q_out


def _on(dev, launch) -> int:
    """``launch()`` with ``dev`` current."""
    if _current_device() == dev.index:
        return launch()
    with torch.cuda.device(dev):
        return launch()


def paged_attn_fwd(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                   block_table: torch.Tensor, seq_lens: torch.Tensor, *,
                   q_lens: Optional[torch.Tensor] = None, window: Optional[int] = None,
                   global_blocks: int = 0, scale: Optional[float] = None,
                   out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None,
                   lse_out: Optional[torch.Tensor] = None, return_lse: bool = True
                   ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Attention of the new tokens over the paged cache (``bsattn_paged_fwd``).

    q: ``[B, Hq, Tq, 128]`` of the pages' dtype, Hq a multiple of Hkv; Tq = 1 is the usual decode
    step, more rows check drafted tokens or process a chunk of a prompt.  The new tokens' keys are
    in the cache already (:func:`paged_kv_append`); each row sees the keys up to its own position.
    ``window`` (in blocks of 128) keeps, for a row in block i, the blocks > i - window and the first
    ``global_blocks``: the rows of :func:`usagi_b200.block_sparse_attn_fwd_window`.  Returns
    ``(o, lse)`` like the prefill calls: o ``[B, Hq, Tq, 128]`` in ``out_dtype`` (default: q's),
    lse fp32 ``[B, Hq, Tq]`` (None if ``return_lse=False``); rows without a key, padding among them,
    get o = 0, lse = -inf.
    """
    if window is not None and window < 1:
        raise ValueError(f"window must be at least 1 block, got {window}")
    if global_blocks < 0 or (global_blocks and window is None):
        raise ValueError("global_blocks must not be negative and needs a window")
    return _attn(q, k_pages, v_pages, block_table, seq_lens, q_lens, window or 0, global_blocks, 0,
                 scale, out_dtype, out, lse_out, return_lse)


def shared_prefix_attn_fwd(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                           block_table: torch.Tensor, seq_lens: torch.Tensor, *, prefix_len: int,
                           q_lens: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                           out_dtype: Optional[torch.dtype] = None,
                           out: Optional[torch.Tensor] = None,
                           lse_out: Optional[torch.Tensor] = None, return_lse: bool = True
                           ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """:func:`paged_attn_fwd` for a batch whose sequences all begin with the same ``prefix_len``
    tokens (a system prompt, a document): whole pages, at the front of every row of ``block_table``,
    read through the row of sequence 0 and once for the whole batch.  Same arguments and same
    result; a sequence may also be shorter than the prefix.
    """
    page = k_pages.shape[2] if k_pages.dim() == 4 else 1
    if prefix_len < 0 or prefix_len % page:
        raise ValueError(f"prefix_len must be whole pages (multiples of {page}), got {prefix_len}")
    if block_table.dim() == 2 and prefix_len > block_table.shape[1] * page:
        raise ValueError("prefix_len is more than block_table holds")
    return _attn(q, k_pages, v_pages, block_table, seq_lens, q_lens, 0, 0, int(prefix_len), scale,
                 out_dtype, out, lse_out, return_lse)


def _attn(q, k_pages, v_pages, block_table, seq_lens, q_lens, window, global_blocks, prefix_len,
          scale, out_dtype, out, lse_out, return_lse):
    shape = q.shape
    if len(shape) != 4 or shape[3] != HEAD_DIM:
        raise ValueError(f"q must be [B, Hq, Tq, {HEAD_DIM}], got {tuple(shape)}")
    B, Hq, Tq, _ = shape
    dev, dtype, Hkv, max_pages, page_size, head, keep = _cache(k_pages, v_pages, block_table,
                                                               seq_lens, q_lens, B)
    if q.dtype is not dtype or q.device != dev:
        raise TypeError(f"q must be {dtype} on {dev} like the pages, got {q.dtype} on {q.device}")
    if Hq == 0 or Hq % Hkv:
        raise ValueError(f"Hq must be a multiple of Hkv, got {Hq} and {Hkv}")
    if out_dtype is None:
        out_dtype = dtype
    elif out_dtype not in _HALF:
        raise TypeError(f"out_dtype must be float16 or bfloat16, got {out_dtype}")
    q = q.contiguous()
    if q.data_ptr() & 15:
        q = q.clone()
    if out is None:
        out = torch.empty_like(q) if out_dtype is dtype else torch.empty_like(q, dtype=out_dtype)
    elif out.shape != shape or out.dtype is not out_dtype or out.device != dev \
            or not out.is_contiguous() or out.data_ptr() & 15:
        raise ValueError("out has the wrong shape, dtype, device, layout or alignment")
    lse, lp = None, None
    if return_lse:
        lse = lse_out
        if lse is None:
            lse = q.new_empty((B, Hq, Tq), dtype=torch.float32)
        elif lse.shape != (B, Hq, Tq) or lse.dtype is not torch.float32 or lse.device != dev \
                or not lse.is_contiguous():
            raise ValueError("lse_out has the wrong shape, dtype, device or layout")
        lp = lse.data_ptr()
    if B == 0 or Tq == 0:
        return out, lse
    flags = (_lib.IN_BF16 if dtype is torch.bfloat16 else 0) | \
        (_lib.OUT_BF16 if out_dtype is torch.bfloat16 else 0)

    def launch():
        stream = _raw_stream(dev.index)
        ws = _workspace(dev, stream)
        need = _scratch_bytes(dev.index, B, Hq, Hkv, Tq, max_pages, page_size, prefix_len)
        scratch, counters = _room(dev, stream, need)
        return _lib.load().bsattn_paged_fwd(
            _PACK(*head, Hq, Hkv, Tq, flags, ws.data_ptr(), 4 * ws.numel(), stream), q.data_ptr(),
            out.data_ptr(), lp, window, global_blocks, prefix_len,
            0.0 if scale is None else scale, scratch.data_ptr(), need, counters.data_ptr())

    rc = _on(dev, launch)
    if rc != 0:
        raise BsattnError(rc, "bsattn_paged_fwd")
    return out, lse


_room_lock = threading.Lock()
_rooms: dict = {}
_KEPT = 32 << 20  # bytes of scratch that a stream keeps


def _room(dev, stream, need):
    """(scratch, counters) of a call.  The calls of one CUDA stream follow one another, so a stream
    keeps its own; a captured call gets new ones, which belong to the graph (the counters zeroed by
    it), since graphs captured on one stream may be replayed at the same time."""
    if torch.cuda.is_current_stream_capturing():
        return (torch.empty(need, dtype=torch.uint8, device=dev),
                torch.zeros(_lib.load().bsattn_paged_counters(), dtype=torch.int32, device=dev))
    key = (dev.index, stream)
    room = _rooms.get(key)
    if room is None or room[0].numel() < min(need, _KEPT):
        with _room_lock:
            room = _rooms.get(key)
            if room is None or room[0].numel() < min(need, _KEPT):
                counters = room[1] if room is not None else torch.zeros(
                    _lib.load().bsattn_paged_counters(), dtype=torch.int32, device=dev)
                room = _rooms[key] = (torch.empty(min(max(need, 4 << 20), _KEPT),
                                                  dtype=torch.uint8, device=dev), counters)
    if need > _KEPT:
        return torch.empty(need, dtype=torch.uint8, device=dev), room[1]
    return room
