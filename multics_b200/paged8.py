"""Key/value caches held in 8 bits, in pages: several sessions served at once
from one pool.

The reference keeps bf16 rolling caches per session and lists their rows in a
page table (``multics/models/kernels/hier_paged_attention.py:232-249``).  Here
a pool of 64-token pages holds int8 or e4m3 codes with one power-of-two scale
per page and head (:class:`Paged8Cache`), half the bytes of bf16, and the
tables are built on the GPU:

* :func:`page_step` - block tables, slots and positions of one step from the
  requests' lengths (tokens appended, dropped, requests ended);
* :func:`paged8_append` - the new keys and values into their pages;
* :func:`paged8_attention` - attention of the new rows over the pages, causal
  by blocks of latent frames and windowed like the action branch's masks
  (``multics/models/blocks.py:300-305,366-371``).

None of them reads back from the device, so a step can be captured into a CUDA
graph (whose caches, like its tensors, the caller keeps).  What a kernel finds wrong in device tables (a page outside the pool, a
length outside the table) it skips and records in the cache's status word
(:meth:`Paged8Cache.check`).
"""

from __future__ import annotations

import contextlib
import ctypes
import math
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import check, dev_err, is_current, raw_stream

__all__ = ["PAGE_TOKENS", "Paged8Cache", "PageStep", "page_step", "paged8_append",
           "paged8_attention"]

PAGE_TOKENS = 64
HEAD_DIM = 128
_I32, _BF16 = torch.int32, torch.bfloat16
_FORMATS = {torch.int8: 0, torch.float8_e4m3fn: 1}
_STATUS = {}  # (device, stream): words that no cache has yet
_KEPT = []  # words that captured graphs write to
_SPLIT = torch.unsafe_split_with_sizes  # (integers: no versions to share)

_CACHE_BITS = ((1, "row starts leave the rows or descend"),
               (2, "a length leaves the block table"),
               (4, "a block table entry leaves the page pool"),
               (8, "a NaN or an infinity was given to the cache"))
_STEP_BITS = ((1, "too few free pages"), (2, "more new tokens than rows"),
              (4, "a length leaves the block table"),
              (8, "an addition is below -length or above the step's most"),
              (16, "the free count leaves the free list"))


def _status_word(dev):
    """A zero status word of its own for a cache: one of 256 zeroed together on
    the current stream, or beside the graph that is being captured (no replay
    clears it, and it is kept for replays after the cache is gone)."""
    if dev.type != "cuda":
        key = dev, 0
    elif not is_current(dev):
        with torch.cuda.device(dev):
            return _status_word(dev)
    elif torch.cuda.is_current_stream_capturing():
        key = dev, "captured"
    else:
        key = dev, raw_stream(dev.index)
    try:
        return _STATUS[key].pop()
    except (KeyError, IndexError):
        if key[1] == "captured":
            zeros = _lib.calls().words_beside_capture(dev.index, 256)
            _KEPT.append(zeros)
        else:
            with torch.inference_mode(False):  # (made in that mode, cleared outside)
                zeros = torch.zeros(256, dtype=_I32, device=dev)
        words = list(zeros.unsafe_split_with_sizes((1,) * 256))
        word = words.pop()
        _STATUS[key] = words
        return word


def _vector(name, t, n, dev):
    if (t.dtype is not _I32 or t.dim() != 1 or t.shape[0] != n or t.device != dev
            or not t.is_contiguous()):
        raise ValueError(f"{name} must be contiguous int32 [{n}] on {dev}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")


def _table(t, dev):
    """(requests, width, row stride) of a block table."""
    if t.dtype is not _I32 or t.dim() != 2 or t.device != dev:
        raise ValueError(f"table must be int32 [requests, width] on {dev}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")
    n, width = t.shape
    stride, inner = t.stride()
    if n and width and (inner != 1 or stride < width):
        raise ValueError("table must be row-major")
    return n, width, stride if stride > width else width


def _cuda(what, dev):
    if dev.type != "cuda":
        raise NotImplementedError(f"{what} requires CUDA tensors")


def _raise_bits(what, bits, table):
    if bits:
        raise ValueError(f"{what}: " + "; ".join(msg for bit, msg in table if bits & bit))


def token_rows(name, x, width):
    """``x`` ``[T, width]`` or ``[1, T, width]`` bf16 as 16-byte aligned rows."""
    if x.dim() == 3 and x.shape[0] == 1:
        x = x[0]
    if x.dim() != 2 or x.shape[1] != width:
        raise ValueError(f"{name} must be [T, {width}], got {tuple(x.shape)}")
    if x.dtype is not _BF16:
        raise NotImplementedError(f"{name} must be bf16; got {x.dtype}")
    stride, inner = x.stride()
    if inner != 1 or stride % 8 or stride < width or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    return x


class Paged8Cache:
    """A pool of ``num_pages`` pages of 64 tokens of ``num_heads`` key heads.

    ``k`` ``[pages, heads, 2, 64, 64]`` (dimension half, token, dimension) and
    ``v`` ``[pages, heads, 128, 64]`` (dimension, token) hold the codes (int8 or
    float8_e4m3fn), ``k_scale`` / ``v_scale`` float32 ``[pages, heads]`` their
    power-of-two scales.  int8 has the finer steps for values of like size,
    e4m3 for values spread over many magnitudes.  The cache holds finite
    numbers: a NaN is held as 0 and an infinity as the largest value of its
    block, and :meth:`check` reports it."""

    def __init__(self, num_pages: int, num_heads: int, *, dtype=torch.int8, device="cuda",
                 head_dim: int = HEAD_DIM):
        if head_dim != HEAD_DIM:
            raise NotImplementedError(f"the 8-bit cache needs head_dim {HEAD_DIM}; got {head_dim}")
        if dtype not in _FORMATS:
            raise ValueError(f"dtype must be torch.int8 or torch.float8_e4m3fn, got {dtype}")
        if num_pages < 1 or num_heads < 1:
            raise ValueError(f"invalid num_pages={num_pages} or num_heads={num_heads}")
        dev = torch.device(device)
        shape = (num_pages, num_heads)
        k = torch.zeros(*shape, 2, PAGE_TOKENS, 64, dtype=torch.int8, device=dev).view(dtype)
        self._set(k, torch.zeros(*shape, HEAD_DIM, PAGE_TOKENS, dtype=torch.int8, device=dev).view(dtype),
                  torch.ones(shape, device=dev), torch.ones(shape, device=dev), _status_word(k.device))

    def _set(self, k, v, k_scale, v_scale, status):
        self.k, self.v, self.k_scale, self.v_scale, self.status = k, v, k_scale, v_scale, status
        self.num_pages, self.num_heads = k.shape[0], k.shape[1]
        self.dtype, self.device, self.format = k.dtype, k.device, _FORMATS[k.dtype]

    @classmethod
    def from_tensors(cls, k, v, k_scale, v_scale, status=None) -> "Paged8Cache":
        """A cache over tensors in the layout above (finite codes, power-of-two
        scales, in ``[2^-126, 2^126]``).  ``status`` (int32 ``[1]``, zero): a word
        to record faults in, where caches are to share one."""
        if _lib.calls().layout(k, v, k_scale, v_scale) is None:
            cls._refuse(k, v, k_scale, v_scale)
        dev = k.device
        if status is None:
            status = _status_word(dev)
        else:
            _vector("status", status, 1, dev)
        self = cls.__new__(cls)
        self._set(k, v, k_scale, v_scale, status)
        return self

    @staticmethod
    def _refuse(k, v, k_scale, v_scale):
        """Raise ValueError for what is wrong with a cache's tensors."""
        if k.dtype not in _FORMATS or v.dtype != k.dtype:
            raise ValueError(f"codes must both be int8 or float8_e4m3fn, got {k.dtype}, {v.dtype}")
        shape = k.shape
        if len(shape) != 5 or shape[2:] != (2, PAGE_TOKENS, 64):
            raise ValueError(f"k must be [pages, heads, 2, 64, 64], got {tuple(shape)}")
        pool = shape[:2]
        if 0 in pool:
            raise ValueError(f"k {tuple(shape)} has no pages or no heads")
        if v.shape != (*pool, HEAD_DIM, PAGE_TOKENS):
            raise ValueError(f"v must be [pages, heads, 128, 64] like k {tuple(k.shape)}, got "
                             f"{tuple(v.shape)}")
        if (k_scale.dtype is not torch.float32 or v_scale.dtype is not torch.float32
                or k_scale.shape != pool or v_scale.shape != pool):
            raise ValueError(f"k_scale and v_scale must be float32 {tuple(pool)}, got "
                             f"{k_scale.dtype} {tuple(k_scale.shape)}, {v_scale.dtype} "
                             f"{tuple(v_scale.shape)}")
        raise ValueError(f"codes and scales must be contiguous on {k.device}")

    def check(self):
        """Raise ValueError for what the kernels recorded since the last check
        (one host read)."""
        if self.device.type == "cuda":  # (read and cleared at once: nothing recorded meanwhile is lost)
            with contextlib.nullcontext() if is_current(self.device) else torch.cuda.device(self.device):
                taken = torch.empty_like(self.status)
                check(_lib.lib().hier_status_take(self.status.data_ptr(), taken.data_ptr(),
                                                  raw_stream(self.device.index)))
            bits = int(taken.item())
        else:
            bits = int(self.status.item())
            self.status &= ~bits
        _raise_bits("8-bit cache", bits, _CACHE_BITS)

    def dequantized(self):
        """The pool's keys and values as bf16 ``[pages, heads, 64, 128]`` (exact)."""
        k = self.k.float() * self.k_scale[..., None, None, None]
        v = self.v.float() * self.v_scale[..., None, None]
        return (k.permute(0, 1, 3, 2, 4).flatten(3).bfloat16(), v.transpose(2, 3).bfloat16())


class PageStep(NamedTuple):
    """What :func:`page_step` built: the requests' new ``lengths``, the
    ``free_count`` left, ``q_start`` ``[n + 1]`` of their rows, and per row its
    ``slots`` entry (page * 64 + token of the page: the row of a 64-token paged
    pool) and ``positions`` entry, -1 behind the last request.  int32 on the
    device."""

    lengths: torch.Tensor
    free_count: torch.Tensor
    q_start: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor
    status: torch.Tensor

    def check(self):
        """Raise ValueError when the step could not be taken (one host read)."""
        _raise_bits("page step refused", int(self.status.item()), _STEP_BITS)


def page_step(lengths, add, table, free_pages, free_count, rows: int, *,
              most_new: Optional[int] = None, in_place: bool = False) -> PageStep:
    """One step of a paged cache's bookkeeping, on the GPU: request ``b`` goes
    from ``lengths[b]`` to ``lengths[b] + add[b]`` tokens (``add < 0`` drops its
    last tokens, ``-lengths[b]`` ends it).

    ``table`` int32 ``[n, width]`` (row-major, updated) lists each request's
    pages; ``free_pages`` int32 (updated) is a stack of ``free_count`` (int32
    ``[1]``) free pages: pages given up are put on its end, pages needed are
    taken from there, both in request order (as they are listed: entries below a
    request's length are its pages until it gives them up here).  ``rows`` is the number of rows of
    the step's token tensors; the new tokens fill them request by request.  A
    step that cannot be taken whole (too few pages or rows, a length outside the
    table, an addition above ``most_new``) changes nothing and maps no row;
    :meth:`PageStep.check` reports it.  ``in_place`` writes the new lengths and
    count over the old ones (a captured step)."""
    done = _lib.calls().page_step(lengths, add, table, free_pages, free_count, rows, most_new, in_place)
    if done is not None:
        if done.__class__ is int:
            check(done)
        new_len, new_count, q_start, status, slots, positions = done
        return PageStep(new_len, new_count, q_start, slots, positions, status)
    dev = table.device
    n, width, stride = _table(table, dev)
    _vector("lengths", lengths, n, dev)
    _vector("add", add, n, dev)
    _vector("free_pages", free_pages, free_pages.shape[0] if free_pages.dim() else 0, dev)
    _vector("free_count", free_count, 1, dev)
    rows = int(rows)
    if rows < 0 or rows >= 1 << 31:
        raise ValueError(f"rows must be in [0, 2^31), got {rows}")
    if most_new is not None and most_new < 0:
        raise ValueError(f"most_new must not be negative, got {most_new}")
    _cuda("page_step", dev)
    if not is_current(dev):
        with torch.cuda.device(dev):
            return page_step(lengths, add, table, free_pages, free_count, rows, most_new=most_new,
                             in_place=in_place)
    if in_place:
        q_start, status, slots, positions = _SPLIT(
            lengths.new_empty(n + 2 + 2 * rows), (n + 1, 1, rows, rows))
        new_len, new_count = lengths, free_count
    else:
        new_len, new_count, q_start, status, slots, positions = _SPLIT(
            lengths.new_empty(2 * n + 3 + 2 * rows), (n, 1, n + 1, 1, rows, rows))
    rc = _lib.calls().hier_page_step(
        lengths.data_ptr(), add.data_ptr(), n, table.data_ptr(), stride, width,
        free_pages.data_ptr(), free_pages.shape[0], free_count.data_ptr(), rows,
        -1 if most_new is None else int(most_new), new_len.data_ptr(), new_count.data_ptr(),
        q_start.data_ptr(), slots.data_ptr(), positions.data_ptr(), status.data_ptr(),
        raw_stream(dev.index))
    if rc:
        check(rc)
    return PageStep(new_len, new_count, q_start, slots, positions, status)


def _requests(cache, table, lengths, q_start):
    n, width, stride = _table(table, cache.device)
    _vector("lengths", lengths, n, cache.device)
    _vector("q_start", q_start, n + 1, cache.device)
    return n, width, stride


def _workspace_floats(*sizes):
    floats = ctypes.c_int64()
    check(_lib.lib().hier_paged8_attn_workspace(*sizes, ctypes.byref(floats)))
    return floats.value


def paged8_append(cache: Paged8Cache, k, v, table, lengths, q_start):
    """Write the new rows ``k``, ``v`` (bf16 ``[T, heads * 128]``) of every
    request into its pages: rows ``q_start[b] .. q_start[b + 1] - 1`` are the
    last of request ``b``'s ``lengths[b]`` tokens.  A page written to must
    belong to one request (pages that several requests list are for reading).
    When a page's scale grows, the codes it held are re-encoded."""
    rc = _lib.calls().append(cache.k, cache.v, cache.k_scale, cache.v_scale, cache.status, cache.format,
                             k, v, table, lengths, q_start)
    if rc is not None:
        if rc:
            check(rc)
        return
    width_k = cache.num_heads * HEAD_DIM
    k, v = token_rows("k", k, width_k), token_rows("v", v, width_k)
    if k.shape != v.shape:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} disagree")
    n, width, stride = _requests(cache, table, lengths, q_start)
    dev = cache.device
    _cuda("paged8_append", dev)
    if k.device != dev or v.device != dev:
        raise ValueError(f"k, v must be on {dev}")
    if not is_current(dev):
        with torch.cuda.device(dev):
            return paged8_append(cache, k, v, table, lengths, q_start)
    rc = _lib.calls().hier_paged8_append(
        k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), k.shape[0], cache.num_heads,
        cache.format, cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(),
        cache.v_scale.data_ptr(), cache.num_pages, table.data_ptr(), stride, width,
        lengths.data_ptr(), q_start.data_ptr(), n, cache.status.data_ptr(), raw_stream(dev.index))
    if rc:
        check(rc)


def paged8_attention(q, cache: Paged8Cache, table, lengths, q_start, num_heads: int, *,
                     tokens_per_frame: int = 1, block_frames: int = 1, window: int = -1,
                     softmax_scale: Optional[float] = None, max_rows: Optional[int] = None,
                     out=None, return_lse: bool = False):
    """Attention of the rows ``q`` (bf16 ``[T, num_heads * 128]``) over an
    8-bit cache; ``num_heads`` is a multiple of the cache's heads, consecutive
    query heads sharing a key head.

    Row ``i`` of request ``b`` is at position ``p = lengths[b] - rows + i`` (the
    rows are the last tokens held; append first).  In frames of
    ``tokens_per_frame`` tokens, token ``j`` is seen when its block of
    ``block_frames`` frames is not after ``p``'s (``block_frames=0``: always, as
    in a cross-attention) and, with a ``window``, when it is less than
    ``window`` frames back: ``cached_frame_mask`` over token positions.
    Rows that see nothing are 0.  Rows of no request (before the first, behind
    the last, or those of a request whose row starts are refused) are zeros, or
    left as they were in a given ``out``, which may be ``q`` itself.  ``max_rows``: the most rows any request has, where the caller
    knows it; it chooses kernels, not results.
    Returns ``[T, num_heads * 128]`` bf16, with ``return_lse`` also the float32
    ``[T, num_heads]`` log2-sum-exp of the scaled scores (-inf for rows that see
    nothing and rows of no request)."""
    if cache.device.type == "cuda":
        done = _lib.calls().attention(
            cache.k, cache.v, cache.k_scale, cache.v_scale, cache.status, cache.format, q, table, lengths,
            q_start, num_heads, tokens_per_frame, block_frames, window, softmax_scale, max_rows, out,
            return_lse, dev_err(cache.device))
        if done is not None:
            if done.__class__ is int:
                check(done)
            return done
    if num_heads < 1 or num_heads % cache.num_heads:
        raise ValueError(f"{num_heads} query heads are not a multiple of the cache's "
                         f"{cache.num_heads}")
    if tokens_per_frame < 1 or block_frames < 0 or window == 0 or window < -1:
        raise ValueError(f"invalid tokens_per_frame={tokens_per_frame}, "
                         f"block_frames={block_frames} or window={window}")
    if max(tokens_per_frame, block_frames, window) > 1 << 30:
        raise ValueError("tokens_per_frame, block_frames and window must be below 2^30")
    if max_rows is not None and max_rows < 0:
        raise ValueError(f"max_rows must not be negative, got {max_rows}")
    scale = 1.0 / math.sqrt(HEAD_DIM) if softmax_scale is None else float(softmax_scale)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"softmax_scale must be positive and finite, got {softmax_scale}")
    dim = num_heads * HEAD_DIM
    q = token_rows("q", q, dim)
    n, width, stride = _requests(cache, table, lengths, q_start)
    dev, T = cache.device, q.shape[0]
    if out is not None and (out.dtype is not _BF16 or out.shape != q.shape or out.device != dev
                            or out.stride(1) != 1 or (T > 1 and out.stride(0) < dim)):
        raise ValueError(f"out must be bf16 {tuple(q.shape)} rows on {dev}")
    _cuda("paged8_attention", dev)
    if q.device != dev:
        raise ValueError(f"q must be on {dev}")
    if not is_current(dev):
        with torch.cuda.device(dev):
            return paged8_attention(q, cache, table, lengths, q_start, num_heads,
                                    tokens_per_frame=tokens_per_frame, block_frames=block_frames,
                                    window=window, softmax_scale=scale, max_rows=max_rows, out=out,
                                    return_lse=return_lse)
    most = 0 if max_rows is None else int(max_rows)
    lse = ws = None
    if out is None:
        o = q.new_empty((T, dim))
    elif out.data_ptr() % 16 or out.stride(0) % 8:  # rows the kernels cannot store to
        o = out.clone(memory_format=torch.contiguous_format)
    else:
        o = out
    if return_lse:
        lse = cache.k_scale.new_empty((T, num_heads))
    floats = _workspace_floats(T, num_heads, cache.num_heads, n, width, most)
    if floats:
        ws = cache.k_scale.new_empty(floats)
    rc = _lib.calls().hier_paged8_attn(
        q.data_ptr(), q.stride(0), T, num_heads, cache.num_heads, HEAD_DIM, cache.format,
        cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(),
        cache.v_scale.data_ptr(), cache.num_pages, table.data_ptr(), stride, width,
        lengths.data_ptr(), q_start.data_ptr(), n, int(tokens_per_frame), int(block_frames),
        int(window), scale, most, o.data_ptr(), o.stride(0),
        None if lse is None else lse.data_ptr(), 1 if out is None else 2 if return_lse else 0,
        None if ws is None else ws.data_ptr(), cache.status.data_ptr(),
        dev_err(dev).data_ptr(), raw_stream(dev.index))
    if rc:
        check(rc)
    if out is not None and o is not out:
        out.copy_(o)
        o = out
    return (o, lse) if return_lse else o
