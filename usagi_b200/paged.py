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
  from 16 to 1024.  16-byte aligned, with a contiguous last dimension and strides that are multiples of 8
  (those of dimensions of one entry do not count): a ``[n_pages, page_size, Hkv, 128]`` cache is passed
  as ``pages.transpose(1, 2)``.
* ``block_table``: int ``[B, max_pages]``, the pages of each sequence in order.  Entries behind a
  sequence's length are not read and may be anything, and so may, with a window, the entries of pages
  that no row of the call sees, and all entries of a sequence without live rows (behind a shared prefix
  those of its own pages).
  A table that is no wider than the sequences need is best (``block_table[:, :n]`` is read in place):
  the room it has sizes the scratch, and decides for more than 8 rows of a K/V head whether a short
  cache is read by the kernel that starts 3 us sooner.
* ``seq_lens``: int ``[B]``, tokens of each sequence, the new ones of this call included.
* ``q_lens``: int ``[B]`` or None, how many of the Tq rows of each sequence are live (None: all).
  Row t < q_lens[b] is the token at position ``seq_lens[b] - q_lens[b] + t``; the rows behind them are
  padding.

Like those of any call, the tensors of these must stay as they are until the call has run on its stream.

Scores and sums are held in 32 bits; softmax weights are rounded to the pages' type before they meet V.
For bf16 that is coarser than the prefill calls, which take fp16 weights and a V converted to fp16.

Slots that hold no token may hold anything.  Values that are held must be finite: those that one row
of a call sees reach the others as well, with weight 0, and 0 times NaN is NaN.

A page table entry, a length or a row count out of range is found on the device, never used as an
address, and raised by :func:`usagi_b200.check_errors` (code ``E_PAGE``).  Such an entry's tokens are
not written; of a sequence whose length or count is out of range none are, and its rotated q is zero.
"""
from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import threading
from typing import Optional, Tuple

import torch

from . import _lib
from .api import HEAD_DIM, BsattnError, _workspace, _workspaces
from .build import BINDING_PATH

__all__ = ["paged_kv_append", "paged_attn_fwd", "shared_prefix_attn_fwd", "rope_inv_freq"]

_lock = threading.Lock()
_binding = None


def _load():
    """The binding (csrc/paged_binding.cpp), which checks the arguments and calls the C ABI; raises if
    it or the kernel library is missing."""
    global _binding
    with _lock:
        if _binding is None:
            lib = _lib.load()
            if not BINDING_PATH.exists():
                raise RuntimeError(f"{BINDING_PATH} is missing; build it with "
                                   "`python -m usagi_b200.build`")
            loader = importlib.machinery.ExtensionFileLoader("_paged_binding", str(BINDING_PATH))
            spec = importlib.util.spec_from_loader("_paged_binding", loader)
            module = importlib.util.module_from_spec(spec)
            loader.exec_module(module)
            address = [ctypes.cast(f, ctypes.c_void_p).value for f in (
                lib.bsattn_paged_append, lib.bsattn_paged_fwd, lib.bsattn_paged_scratch_bytes,
                lib.bsattn_paged_counters)]
            module.init(*address, _workspaces, _workspace, BsattnError)
            _binding = module
        return _binding


def rope_inv_freq(rot_dim: int = HEAD_DIM, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """``base ** (-2 i / rot_dim)`` for i < rot_dim / 2 in 64 bits, for :func:`paged_kv_append`."""
    i = torch.arange(rot_dim // 2, dtype=torch.float64)
    return (float(base) ** (-2.0 * i / rot_dim)).to(device)


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
    rows (``q_out`` when given; it may be q itself if that is contiguous), or None without q.  Sequences
    must not share a page that new tokens go to.
    """
    return (_binding or _load()).append(k_pages, v_pages, block_table, seq_lens, k, v, q, q_lens,
                                        inv_freq, interleaved, q_out)


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
    ``global_blocks`` (both up to 2^24): the rows of :func:`usagi_b200.block_sparse_attn_fwd_window`.  Returns
    ``(o, lse)`` like the prefill calls: o ``[B, Hq, Tq, 128]`` in ``out_dtype`` (default: q's),
    lse fp32 ``[B, Hq, Tq]`` (None if ``return_lse=False``); rows without a key, padding among them,
    get o = 0, lse = -inf.  ``scale`` is positive (None: 1/sqrt(128)).
    """
    if window is not None and window < 1:
        raise ValueError(f"window must be at least 1 block, got {window}")
    if global_blocks < 0 or (global_blocks and window is None):
        raise ValueError("global_blocks must not be negative and needs a window")
    return (_binding or _load()).attn(q, k_pages, v_pages, block_table, seq_lens, q_lens,
                                      window or 0, global_blocks, 0, scale, out_dtype, out, lse_out,
                                      return_lse)


def shared_prefix_attn_fwd(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                           block_table: torch.Tensor, seq_lens: torch.Tensor, *, prefix_len: int,
                           q_lens: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                           out_dtype: Optional[torch.dtype] = None,
                           out: Optional[torch.Tensor] = None,
                           lse_out: Optional[torch.Tensor] = None, return_lse: bool = True
                           ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """:func:`paged_attn_fwd` for a batch whose sequences all begin with the same ``prefix_len``
    tokens (a system prompt, a document): whole pages, all held, the same ones at the front of every row
    of ``block_table`` (also in the rows of shorter sequences).  Where it pays they are read once for the whole batch, through the row of sequence
    0, with the rows of all sequences stacked on the tensor cores.  Same arguments and same result as
    :func:`paged_attn_fwd` without a window; a sequence may also be shorter than the prefix.
    """
    return (_binding or _load()).attn(q, k_pages, v_pages, block_table, seq_lens, q_lens, 0, 0,
                                      prefix_len, scale, out_dtype, out, lse_out, return_lse)
