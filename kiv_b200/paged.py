"""Paged caches of batches of unequal lengths, and the turn of queries and keys in front of a cache.

``TieredKVCache`` / ``ColdKVStore`` hold one batch of equal lengths in dense
buffers.  A serving engine batches requests of unequal lengths and keeps their
recent tokens in pages; these are the calls one attention layer of its step
makes, on pages of the same ``[.., Hkv, page_size, D]`` layout as the cold tier:

* ``qk_norm_rope``  norms of the query and key rows of each head and their
  position rotation, in one pass (also in front of ``TieredKVCache.update``);
* ``paged_append``  the new tokens' keys, turned on the way, and values into
  their pages;
* ``paged_attend``  attention of every sequence's new tokens over its pages.

``PagedKVCache`` keeps the pages of a model's layers and hands them out.

``block_table`` (int32 ``[batch, width]``), ``seq_lens`` (int32 ``[batch]``, new
tokens included) and ``q_starts`` (int32 ``[batch + 1]``, first row of each
sequence's new tokens among the packed rows) are device tensors that the
kernels read, so a call captured in a CUDA graph serves other lengths and pages
on replay.  Rows behind ``q_starts[-1]`` (a padded batch) are neither read nor
written.  ``errors`` (int64, optional) collects ``ERRBIT_*`` bits of
``kiv_b200._native``: page numbers, lengths and positions that the kernels
could not follow -- they never read or write out of bounds.

Every call runs on the current stream of its tensors' device, allocates its
scratch from that stream's pool and raises ``KIVNativeError`` on refused
arguments.  There is no CPU implementation.
"""

from __future__ import annotations

import torch

from . import _native as nat
from . import ops


def _rows(x: torch.Tensor, what: str) -> torch.Tensor:
    """Rows as the kernels read them: on a GPU, last dim contiguous, 16-byte aligned."""
    if not x.is_cuda:
        raise nat.KIVNativeError(f"{what} must be on a CUDA device (got {x.device}); the B200 kernels are the only "
                                 "implementation")
    nat.dtype_code(x.dtype)
    mult = 16 // x.element_size()
    if x.numel() and (x.stride(-1) != 1 or x.data_ptr() % 16 or any(s % mult for s, n in zip(x.stride()[:-1], x.shape) if n > 1)):
        x = x.contiguous()
    return x


def rotary_table(inv_freq: torch.Tensor, length: int, scaling: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """cos and sin, float32 ``[length, len(inv_freq)]``, of positions 0 .. length - 1.  The angles are formed in 64
    bits: at position p one in 32 bits is off by up to p * 2^-24."""
    angle = torch.outer(torch.arange(length, dtype=torch.float64, device=inv_freq.device), inv_freq.double())
    return (angle.cos() * scaling).float(), (angle.sin() * scaling).float()


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor | None, cos: torch.Tensor | None = None, sin: torch.Tensor | None = None,
                 *, positions: torch.Tensor | None = None, pair_axes: torch.Tensor | None = None, interleaved: bool = False,
                 eps: float | None = None, q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                 weight_offset: float = 0.0, out: tuple[torch.Tensor, torch.Tensor | None] | None = None,
                 errors: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Norm (``eps`` given) and rotation of ``q [B, Hq, Q, D]`` and ``k [B, Hkv, Q, D]``; returns both.

    Norm: ``x * rsqrt(mean(x^2) + eps) * (weight_offset + weight)``.  Rotation: pair j of the first ``2 * cos.shape[1]``
    elements -- ``(j, j + half)``, or ``(2j, 2j + 1)`` with ``interleaved`` -- by ``cos / sin[row, j]`` (float32 or the
    rows' dtype).  The row is the token's position (``positions [B, Q]``); with several axes (``positions [A, B, Q]``:
    time, height, width) that of axis ``pair_axes[j]`` (int32); without ``positions`` it is ``b * Q + t``, for tables
    already gathered per token.  A row whose position is outside the table comes out as NaN.
    Computed in float32 and rounded once.  ``out`` may be ``(q, k)`` themselves.
    """
    q = _rows(q, "q")
    if k is not None:
        k = _rows(k, "k")
    q_out, k_out = out if out is not None else (torch.empty_like(q), None if k is None else torch.empty_like(k))
    ops.call(ops.kiv().qk_norm_rope, q, k, cos, sin, positions, pair_axes, interleaved, eps, q_weight, k_weight,
             weight_offset, q_out, k_out, errors)
    return q_out, k_out


def paged_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                 seq_lens: torch.Tensor, q_starts: torch.Tensor, *, cos: torch.Tensor | None = None,
                 sin: torch.Tensor | None = None, positions: torch.Tensor | None = None,
                 pair_axes: torch.Tensor | None = None, interleaved: bool = False, eps: float | None = None,
                 k_weight: torch.Tensor | None = None, weight_offset: float = 0.0,
                 errors: torch.Tensor | None = None) -> None:
    """Write the new rows ``k, v [tokens, Hkv, D]`` to the pages ``[num_pages, Hkv, page_size, D]``.

    New token i of the n of sequence b goes to place ``seq_lens[b] - n + i``.  Keys are normed and rotated on the way as
    in ``qk_norm_rope`` (``positions [tokens]`` or ``[A, tokens]``; without them by their place).  A token without a valid
    page, or with a position outside the table, is not written.
    """
    k, v = _rows(k, "k"), _rows(v, "v")
    ops.call(ops.kiv().paged_append, k, v, k_pages, v_pages, block_table, seq_lens, q_starts, cos, sin, positions,
             pair_axes, interleaved, eps, k_weight, weight_offset, errors)


def paged_attend(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                 seq_lens: torch.Tensor, q_starts: torch.Tensor, scaling: float, *, causal: bool = True, window: int = 0,
                 softcap: float = 0.0, max_query_len: int = 0, out: torch.Tensor | None = None, return_lse: bool = False,
                 errors: torch.Tensor | None = None):
    """Attention of the new tokens' queries ``q [tokens, Hq, D]`` over their sequences' keys; ``out [tokens, Hq, D]``.

    ``causal``: new token i of the n of sequence b sees keys ``j <= seq_lens[b] - n + i``, with ``window`` only the last
    ``window`` of them; otherwise all.  ``softcap``: scores ``c * tanh(s / c)``.  ``max_query_len``: the largest n, where
    the host knows it (chooses kernels, never changes which keys count).  With ``return_lse`` also the float32
    log-sum-exp of the scores ``[tokens, Hq]``; a row that sees no key gets 0 and -inf.  Keys without a valid page read
    as rows of zeros.  Rows of ``out`` and ``lse`` behind ``q_starts[-1]`` are left as they are.
    """
    q = _rows(q, "q")
    if out is None:
        out = torch.empty_like(q)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device) if return_lse else None
    ops.call(ops.kiv().paged_attend, q, k_pages, v_pages, block_table, seq_lens, q_starts, scaling, causal, window, softcap,
             max_query_len, out, lse, errors)
    return (out, lse) if return_lse else out
