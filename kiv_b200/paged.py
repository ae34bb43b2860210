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
could not follow -- they never read or write out of bounds -- and
``ERRBIT_WAIT_TIMEOUT``, a wait inside a kernel that gave up after about a
second, which leaves rows of ``paged_attend`` wrong.  Without ``errors`` none of
these is told (``PagedKVCache`` keeps one).

Every call runs on the current stream of its tensors' device, allocates its
scratch from that stream's pool and raises ``KIVNativeError`` on refused
arguments.  There is no CPU implementation, no backward and no forward
derivative: inputs that require gradients are refused outside
``torch.no_grad()``, inputs with a forward-mode tangent everywhere.
"""

from __future__ import annotations

from array import array

import torch
from torch.autograd import forward_ad

from . import _native as nat
from . import ops


_ops: dict = {}


def _run(name: str, rows: torch.Tensor, *args) -> None:
    """One operator on the GPU of ``rows`` (the operator copies rows that are not 16-byte aligned)."""
    if not rows.is_cuda:
        raise nat.KIVNativeError(f"{name} needs tensors on a CUDA device (got {rows.device}); the B200 kernels are the only "
                                 "implementation")
    op = _ops.get(name)
    if op is None:
        op = _ops[name] = getattr(ops.kiv(), name).default
    try:
        op(rows, *args)
    except RuntimeError as e:
        if "kiv" in str(e):
            raise nat.KIVNativeError(str(e)) from e
        raise


def needs_derivative(*tensors: torch.Tensor | None) -> bool:
    """Whether a gradient or a forward-mode tangent of an input would have to come through the call."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    if getattr(forward_ad, "_current_level", 0) >= 0:           # inside a dual level, where there can be tangents
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                return True
    return False


def _refuse_gradients(name: str, *tensors: torch.Tensor | None) -> None:
    """There is no derivative: an input that needs one is refused, it would be missing without a word."""
    if needs_derivative(*tensors):
        raise nat.KIVNativeError(f"{name} has no backward and no forward derivative: call it under torch.no_grad(), on "
                                 "detached tensors and on tensors without a tangent")


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
    _refuse_gradients("qk_norm_rope", q, k, cos, sin, q_weight, k_weight)
    if out is None:                                  # outputs like the inputs, with a contiguous last dim
        q = q if q.stride(-1) == 1 else q.contiguous()
        k = k if k is None or k.stride(-1) == 1 else k.contiguous()
    q_out, k_out = out if out is not None else (torch.empty_like(q), None if k is None else torch.empty_like(k))
    _run("qk_norm_rope", q, k, cos, sin, positions, pair_axes, interleaved, eps, q_weight, k_weight,
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
    _refuse_gradients("paged_append", k, v, k_pages, v_pages, cos, sin, k_weight)
    _run("paged_append", k, v, k_pages, v_pages, block_table, seq_lens, q_starts, cos, sin, positions,
             pair_axes, interleaved, eps, k_weight, weight_offset, errors)


def paged_attend(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                 seq_lens: torch.Tensor, q_starts: torch.Tensor, scaling: float, *, causal: bool = True, window: int = 0,
                 softcap: float = 0.0, max_query_len: int = 0, out: torch.Tensor | None = None, return_lse: bool = False,
                 errors: torch.Tensor | None = None):
    """Attention of the new tokens' queries ``q [tokens, Hq, D]`` over their sequences' keys; ``out [tokens, Hq, D]``.

    ``causal``: new token i of the n of sequence b sees keys ``j <= seq_lens[b] - n + i``, with ``window`` only the last
    ``window`` of them; otherwise all.  ``softcap``: scores ``c * tanh(s / c)``.  ``max_query_len``: the largest n, where
    the host knows it (chooses tilings, and so the order of fp32 sums, never which keys count or how exactly).  With
    ``return_lse`` also the float32 log-sum-exp of the scores ``[tokens, Hq]``; a row that sees no key gets 0 and -inf.
    Keys without a valid page read as rows of zeros.  Rows of ``out`` and ``lse`` behind ``q_starts[-1]`` are left as they
    are.  Statistics and sums are float32; with 16-bit rows the softmax weights are rounded to the rows' dtype before they
    meet the values, and kept with at least twice its bits where the tcgen05 kernels do not take the call: a page size that
    is no multiple of 8, a head dimension other than 64, 96, 128 and 256, more than 128 query heads per key head.
    """
    _refuse_gradients("paged_attend", q, k_pages, v_pages)
    if out is None:
        q = q if q.stride(-1) == 1 else q.contiguous()
        out = torch.empty_like(q)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device) if return_lse else None
    _run("paged_attend", q, k_pages, v_pages, block_table, seq_lens, q_starts, scaling, causal, window, softcap,
             max_query_len, out, lse, errors)
    return (out, lse) if return_lse else out


class _PageBook:
    """Which pages each sequence holds, and which cells of the block table a step changes (host only).

    Slot i of the table remembers whose row it holds and how much of it is written: while a sequence keeps its slot, a step
    costs the pages that are new, whatever it holds already.
    """

    def __init__(self, num_pages: int, page_size: int, max_batch: int, width: int) -> None:
        self.page_size, self.max_batch, self.width = page_size, max_batch, width
        self.unused = list(range(num_pages - 1, -1, -1))
        self.held: dict = {}
        self.lengths: dict = {}
        self._slots: list = [(None, 0)] * max_batch             # (a sequence's list of pages, entries written)

    def step(self, new: list[tuple]) -> tuple[list[int], list[int], list[tuple], array]:
        """Row starts, lengths, and the changed cells: runs (first, count) of ``[max_batch, width]`` laid flat, and the pages
        of all of them."""
        if len(new) > self.max_batch:
            raise ValueError(f"{len(new)} sequences exceed max_batch {self.max_batch}")
        if len({s for s, _ in new}) != len(new):
            raise ValueError("a sequence appears twice in one step")
        need = []
        for seq, n in new:
            if n < 0:
                raise ValueError("negative token count")
            pages = -(-(self.lengths.get(seq, 0) + n) // self.page_size)
            if pages > self.width:
                raise nat.KIVNativeError(f"sequence {seq!r} needs {pages} pages, a sequence holds at most {self.width}")
            need.append(pages - len(self.held.get(seq, ())))
        if sum(need) > len(self.unused):
            raise nat.KIVNativeError(f"out of pages: the step needs {sum(need)}, {len(self.unused)} are free")
        starts, lens, runs, pages = [0], [], [], array("i")
        for i, (seq, n) in enumerate(new):
            held = self.held.setdefault(seq, array("i"))
            held.extend(self.unused.pop() for _ in range(need[i]))
            self.lengths[seq] = self.lengths.get(seq, 0) + n
            lens.append(self.lengths[seq])
            starts.append(starts[-1] + n)
            owner, written = self._slots[i]
            keep = written if owner is held else 0
            end = max(written, len(held))                       # a longer row before it: no page from there on
            if keep < end:
                runs.append((i * self.width + keep, end - keep))
                pages.extend(held[keep:])
                pages.extend([-1] * (end - len(held)))
                self._slots[i] = (held, len(held))
        return starts, lens, runs, pages

    def free(self, seq) -> None:
        self.unused.extend(reversed(self.held.pop(seq, ())))
        self.lengths.pop(seq, None)


class PagedKVCache:
    """Pages of a model's KV layers for a batch of sequences of unequal lengths.

    The pages of a layer are ``k[layer]``, ``v[layer]`` ``[num_pages, Hkv,
    page_size, D]``; all layers share one block table.  A serving step:

        cache.step([(seq, new_tokens), ...])        # reserves pages, uploads table and lengths
        for layer in ...:
            cache.append(layer, k, v, cos=..., sin=...)
            out = cache.attend(layer, q, scaling)   # packed rows, in the step's order

    ``step`` is host work (it raises before it changes anything when the pages
    run out); ``append`` and ``attend`` read its device arrays, which stay where
    they are, so a captured ``append`` / ``attend`` serves later steps of the
    same number of sequences and at most the captured number of rows.  To
    capture before their tokens are there, begin a step of the sequences with 0
    new tokens each and pass rows of the later number: nothing is written while
    capturing, and the replay after the next ``step`` finds its tokens.
    ``errors`` collects the kernels' bits.
    """

    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, *, layers: int = 1,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device | str = "cuda", max_batch: int = 64,
                 max_pages_per_seq: int | None = None) -> None:
        if min(num_pages, page_size, num_kv_heads, head_dim, layers, max_batch) < 1:
            raise ValueError("PagedKVCache sizes must be positive")
        device = torch.device(device)
        if device.type != "cuda":
            raise nat.KIVNativeError(f"PagedKVCache runs on CUDA devices only (got {device}); the B200 kernels are the "
                                     "only implementation")
        nat.dtype_code(dtype)
        self.page_size, self.num_pages, self.max_batch = page_size, num_pages, max_batch
        width = min(num_pages, max_pages_per_seq or num_pages)
        # zeros: a stale row never reaches a result, whatever it holds, but NaN in a dump would mislead
        self.k = torch.zeros(layers, num_pages, num_kv_heads, page_size, head_dim, dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.device = self.k.device
        self._table = torch.full((max_batch, width), -1, dtype=torch.int32, device=device)
        self._lens = torch.zeros(max_batch, dtype=torch.int32, device=device)
        self._starts = torch.zeros(max_batch + 1, dtype=torch.int32, device=device)
        self.errors = torch.zeros(1, dtype=torch.int64, device=device)
        self._book = _PageBook(num_pages, page_size, max_batch, width)
        self._batch = self._tokens = self._most = 0

    # ------------------------------------------------------------------ host
    @property
    def free_pages(self) -> int:
        return len(self._book.unused)

    def length(self, seq) -> int:
        """Tokens of a sequence, those of the current step included (0: unknown)."""
        return self._book.lengths.get(seq, 0)

    def step(self, new: list[tuple]) -> int:
        """Begin a step: ``new`` lists ``(sequence, new tokens)`` in the order of the packed rows; unknown sequences
        start empty.  Reserves their pages and uploads lengths, row starts and what changed of the table: host work per
        sequence and new page, not per page held.  Returns the number of rows."""
        starts, lens, runs, pages = self._book.step(new)
        if runs:
            page = torch.frombuffer(pages, dtype=torch.int32)
            at = torch.cat([torch.arange(first, first + count) for first, count in runs])
            self._table.view(-1).index_copy_(0, *(x.pin_memory().to(self.device, non_blocking=True) for x in (at, page)))
        self._upload(self._lens[:len(new)], torch.tensor(lens, dtype=torch.int32))
        self._upload(self._starts[:len(new) + 1], torch.tensor(starts, dtype=torch.int32))
        self._batch, self._tokens, self._most = len(new), starts[-1], max([n for _, n in new], default=0)
        return self._tokens

    def _upload(self, dst: torch.Tensor, src: torch.Tensor) -> None:
        if src.numel():
            dst.copy_(src.pin_memory(), non_blocking=True)     # a fresh pinned buffer: the allocator keeps it until the copy is done

    def free(self, seq) -> None:
        """Give a sequence's pages back (a step that is still running may read them: free after it)."""
        self._book.free(seq)

    # ---------------------------------------------------------------- device
    def arrays(self) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """``(block_table, seq_lens, q_starts)`` of the current step."""
        return self._table[:self._batch], self._lens[:self._batch], self._starts[:self._batch + 1]

    def _check(self, rows: torch.Tensor) -> None:
        if rows.shape[0] < self._tokens:
            raise nat.KIVNativeError(f"the step has {self._tokens} rows, got {rows.shape[0]}")

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, **turn) -> None:
        """Write the step's new rows of a layer (``paged_append``; ``turn``: its keyword arguments)."""
        self._check(k)
        paged_append(k, v, self.k[layer], self.v[layer], *self.arrays(), errors=self.errors, **turn)

    def attend(self, layer: int, q: torch.Tensor, scaling: float, **kw):
        """Attention of the step's new tokens over a layer's pages (``paged_attend``)."""
        self._check(q)
        return paged_attend(q, self.k[layer], self.v[layer], *self.arrays(), scaling, max_query_len=self._most,
                            errors=self.errors, **kw)
