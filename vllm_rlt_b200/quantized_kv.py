"""A paged key/value cache in 8 bits, and a step's pages and slots on the GPU.

`QuantizedKV` is one layer's cache: e4m3 codes `[pages, block, kv_heads, dim]` and a float32 scale for each page and head.  A step over it:

    slots = step_slots(lengths, counts, tables, block, rows, held=held, free_pages=free_pages, free_count=free_count)
    quantized_kv_write(cache, k, v, tables, slots.lengths, slots.cu)
    out = quantized_attention(q, cache, tables, slots.lengths, slots.cu, max_new)

The rows of a step are packed: rows cu[s] .. cu[s + 1] - 1 are sequence s's last ones, at positions lengths[s] - n_s .. lengths[s] - 1, and
everything is read on the device, so a step of a fixed number of rows can be captured in a CUDA graph and replayed with other lengths.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import _capi

CODE_DTYPE = torch.float8_e4m3fn


@dataclass(frozen=True)
class QuantizedKV:
    """One layer's keys and values in 8 bits: a value is its code times the scale of its page and head.

    key / value: float8_e4m3fn `[pages, block, kv_heads, dim]` of one layout, pages and tokens with any stride, the `[kv_heads, dim]` tail
    contiguous; dim at most 256.  key_scale / value_scale: float32 `[pages, kv_heads]` of one layout, heads side by side.  Scales that
    `quantized_kv_write` makes are powers of two, 2^-100 .. 2^100.  Others may be read too: a value scale beyond that range counts as its nearer
    end, zero as zero, and a negative or NaN one makes the rows that see its page NaN in its head."""

    key: torch.Tensor
    value: torch.Tensor
    key_scale: torch.Tensor
    value_scale: torch.Tensor

    @classmethod
    def allocate(cls, pages: int, block: int, kv_heads: int, dim: int, device="cuda") -> "QuantizedKV":
        """An empty cache, keys and values in one allocation (a page of both is then one copy)."""
        codes = torch.zeros(2, pages, block, kv_heads, dim, dtype=CODE_DTYPE, device=device)
        scales = torch.zeros(2, pages, kv_heads, dtype=torch.float32, device=device)
        return cls(codes[0], codes[1], scales[0], scales[1])

    def check(self) -> None:
        key, value, ks, vs = self.key, self.value, self.key_scale, self.value_scale
        shape, stride, scale_stride = key.shape, key.stride(), ks.stride()
        if len(shape) != 4 or value.shape != shape or value.stride() != stride or key.dtype != CODE_DTYPE or value.dtype != CODE_DTYPE:
            raise ValueError("key and value must be float8_e4m3fn [pages, block, kv_heads, dim] of one layout")
        pages, block, heads, dim = shape
        if (dim > 1 and stride[3] != 1) or (heads > 1 and stride[2] != dim):
            raise ValueError("the [kv_heads, dim] tail of the cache must be contiguous")
        if not 0 < dim <= 256 or block == 0 or heads == 0:
            raise ValueError("a cache needs tokens, heads, and a dim of 1 .. 256")
        if ks.dtype != torch.float32 or vs.dtype != torch.float32 or ks.shape != (pages, heads) or vs.shape != ks.shape \
                or vs.stride() != scale_stride or (heads > 1 and scale_stride[1] != 1):
            raise ValueError("scales must be float32 [pages, kv_heads] of one layout with unit inner stride")


@dataclass(frozen=True)
class StepSlots:
    """A step's rows (device tensors).  Rows behind the last request's have row_seq -1, write_blocks -1 and zeros."""

    cu: torch.Tensor              # int32 [n + 1]  rows cu[s] .. cu[s + 1] - 1 are request s's
    lengths: torch.Tensor         # int32 [n]      tokens of the request with the step's
    positions: torch.Tensor       # int32 [rows]
    row_seq: torch.Tensor         # int32 [rows]   request of the row
    write_blocks: torch.Tensor    # int64 [rows]   page and offset the row is stored at (`kv_write`, `rope_kv_write`)
    write_offsets: torch.Tensor   # int64 [rows]
    active_rows: torch.Tensor     # int32 []       cu[n]
    status: torch.Tensor          # int32 []       0, or 1: refused, and nothing changed


def _check_words(n: int, **tensors) -> None:
    for name, t in tensors.items():
        if t.dtype != torch.int32 or t.shape != (n,) or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous int32 [{n}]")


# A decoding step makes these calls once a layer, and their kernels take less time than a call of Python's slower ways would: addresses go to
# the library as integers, and the device is switched only where it is another.
def _device_of(*tensors) -> int:
    """The index of the device that all tensors are on."""
    index = tensors[0].get_device()
    if index < 0 or any(t.get_device() != index for t in tensors):
        _capi.require_cuda(*tensors)                 # says what is wrong
    return index


def _run(what: str, index: int, *args) -> None:
    entry = getattr(_capi.load(), "rlt_" + what)
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch.cuda.current_device() == index:
        code = entry(*args, stream)
    else:
        with torch.cuda.device(index):
            code = entry(*args, stream)
    if code:
        _capi.check(code, what)


def _check_stack(tables, held, free_pages, free_count) -> None:
    _check_words(tables.shape[0], held=held)
    _check_words(1, free_count=free_count)
    if free_pages.dtype != torch.int32 or free_pages.dim() != 1 or not free_pages.is_contiguous():
        raise ValueError("free_pages must be contiguous int32 [pages]")


def _check_tables(tables) -> None:
    if tables.dtype != torch.int32 or tables.dim() != 2 or not tables.is_contiguous():
        raise ValueError("tables must be contiguous int32 [requests, pages]")


def step_slots(lengths, counts, tables, block: int, rows: int, *, held=None, free_pages=None, free_count=None) -> StepSlots:
    """Slots of a step that stores `counts[s]` more tokens of request s behind the `lengths[s]` it has, in up to `rows` rows.

    lengths / counts: int32 `[n]`, n at most 8192 (a count below zero is zero).  tables: int32 `[n, pages]`.  With `held` (int32 `[n]`, pages
    that each request holds) missing pages are claimed first, from the end of the stack `free_pages` (int32 `[m]`, of which the first
    free_count[0] are free), in the order of the requests: tables, held and free_count are updated in place.  Without it the tables have to
    name every page already.  A step that does not fit (rows, free pages, a table's width), or a length or number of held or free pages that cannot
    be, is refused as a whole: status 1, no rows, nothing changed.  A number of held pages may be larger than a request needs: a request
    that was rolled back keeps its pages."""
    _check_tables(tables)
    n, width = tables.shape
    _check_words(n, lengths=lengths, counts=counts)
    if (held is None) != (free_pages is None) or (held is None) != (free_count is None):
        raise ValueError("held, free_pages and free_count come together")
    if held is not None:
        _check_stack(tables, held, free_pages, free_count)
    if block < 1 or rows < 0:
        raise ValueError("block must be positive, rows not negative")
    if held is None:
        index, stack = _device_of(lengths, counts, tables), (None, None, 0, None)
    else:
        index = _device_of(lengths, counts, tables, held, free_pages, free_count)
        stack = held.data_ptr(), free_pages.data_ptr(), free_pages.numel(), free_count.data_ptr()
    device = tables.device
    words = torch.empty(2 * n + 3 + 2 * rows, dtype=torch.int32, device=device)
    cu, new_lengths, positions, row_seq, last = words.split_with_sizes((n + 1, n, rows, rows, 2))
    places = torch.empty((2, rows), dtype=torch.int64, device=device)
    at, place_at = words.data_ptr(), places.data_ptr()
    end = at + 4 * (2 * n + 1 + 2 * rows)
    _run("step_slots", index, lengths.data_ptr(), counts.data_ptr(), n, tables.data_ptr(), width, block, *stack, rows, at, at + 4 * (n + 1),
         at + 4 * (2 * n + 1), at + 4 * (2 * n + 1 + rows), place_at, place_at + 8 * rows, end, end + 4)
    return StepSlots(cu, new_lengths, positions, row_seq, places[0], places[1], last[0], last[1])


def return_pages(lengths, tables, block: int, *, held, free_pages, free_count):
    """Request s keeps the pages of its first `lengths[s]` tokens (0: none) and gives the others back to the stack, so that what was claimed
    last is claimed next; held, free_pages and free_count are updated in place, the tables stay.  A page is one request's: holders are not
    counted, and a page that stands in two requests' tables would be given back by each.  Returns an int32 status on the device: 0, or
    1 where the stack has no room (pages given back twice) or a number of held pages cannot be; then nothing has changed."""
    _check_tables(tables)
    n, width = tables.shape
    _check_words(n, lengths=lengths)
    _check_stack(tables, held, free_pages, free_count)
    if block < 1:
        raise ValueError("block must be positive")
    index = _device_of(lengths, tables, held, free_pages, free_count)
    status = torch.empty((), dtype=torch.int32, device=tables.device)
    _run("return_pages", index, lengths.data_ptr(), n, tables.data_ptr(), width, block, held.data_ptr(), free_pages.data_ptr(), free_pages.numel(),
         free_count.data_ptr(), status.data_ptr())
    return status


def _check_step(tables, lengths, cu) -> None:
    _check_tables(tables)
    n = tables.shape[0]
    _check_words(n, lengths=lengths)
    _check_words(n + 1, cu=cu)


def _row_stride(t) -> int:
    """Elements between the rows of a [rows, heads, dim] tensor with a contiguous tail, which may be a slice of wider rows."""
    (rows, heads, dim), (row, head, element) = t.shape, t.stride()
    if (dim > 1 and element != 1) or (heads > 1 and head != dim):
        raise ValueError("the [heads, dim] tail of rows must be contiguous")
    return row if rows > 1 else heads * dim


def _cache_args(cache: QuantizedKV) -> tuple:
    """Addresses, strides and pages of a cache; a dimension of one has the stride of a dense layout."""
    key, scale = cache.key, cache.key_scale
    (pages, block, kv_heads, dim), (page_stride, token_stride, _, _) = key.shape, key.stride()
    token = token_stride if block > 1 else kv_heads * dim
    return (key.data_ptr(), cache.value.data_ptr(), scale.data_ptr(), cache.value_scale.data_ptr(), page_stride if pages > 1 else block * token, token,
            scale.stride()[0] if pages > 1 else kv_heads, pages, block)


def quantized_kv_write(cache: QuantizedKV, k, v, tables, lengths, cu) -> None:
    """Store a step's keys and values, `[rows, kv_heads, dim]` in float32, float16 or bfloat16 (rows may be slices of wider ones).

    In every page that gets rows, and for every head, the scale becomes the smallest power of two (2^-100 .. 2^100) that brings the new rows'
    largest element within the codes' 448, or stays the page's own where that is larger; where it grows, the tokens in front of the new rows
    are rounded again.  A page whose offset 0 is written starts anew: what it held behind the new rows means nothing any more.  Codes are
    rounded to the nearest, ties to even; elements that are not finite are stored as NaN and have no part in a scale.

    So what a page holds depends on every row that was written to it, those that were rejected later among them: a scale that grew for one
    stays, and the tokens in front were rounded for it.  Steps that speculate store other codes than steps of one token, and a prompt in one call
    others than in several; tokens chosen over such a cache may differ by that.

    A page that is written belongs to one sequence of the call.  Rows at negative positions, behind the last sequence, behind the end of
    their table row or in a page that does not exist are not stored."""
    cache.check()
    _check_step(tables, lengths, cu)
    pages, block, kv_heads, dim = cache.key.shape
    if k.dim() != 3 or k.shape[1:] != (kv_heads, dim) or v.shape != k.shape or k.dtype not in _capi.DTYPE_CODES or v.dtype != k.dtype:
        raise ValueError("k and v must be [rows, kv_heads, dim] of the cache's heads, in float32, float16 or bfloat16")
    rows = k.shape[0]
    k_stride, v_stride = _row_stride(k), _row_stride(v)
    index = _device_of(k, v, cache.key, cache.value, cache.key_scale, cache.value_scale, tables, lengths, cu)
    if rows == 0 or pages == 0:
        return
    sequences, width = tables.shape
    _run("quantized_kv_write", index, *_cache_args(cache), kv_heads, dim, k.data_ptr(), k_stride, v.data_ptr(), v_stride, _capi.DTYPE_CODES[k.dtype],
         tables.data_ptr(), lengths.data_ptr(), cu.data_ptr(), sequences, width, rows)


def quantized_attention(q, cache: QuantizedKV, tables, lengths, cu, max_new: int, *, scale: float | None = None, window: int = 0, out=None):
    """Causal attention of a step's rows, `[rows, heads, dim]` in float32, float16 or bfloat16, over an 8-bit cache, in q's type.

    Row i of the n_s rows of sequence s sees lengths[s] - n_s + i + 1 keys, with `window` the last so many of them; a row that sees none gives
    zeros, a length that its table cannot address is cut to what it can, and rows behind the last sequence are left as they are in `out`
    (undefined where `out` is not given; it may not share memory with q).  scale: 1 / sqrt(dim) unless given.  max_new: the longest portion of
    the step.  It, the shapes and the numbers of rows and sequences decide on the kernels: in portions of up to 16 rows, a row's bits are its own,
    whatever else is in the call; in a step of long portions in bfloat16 without a window (64 rows and more on average), those of 64 rows and more
    (128 where no heads share keys) are scored over an expansion of their pages, with weights rounded to bfloat16.  Otherwise weights have 11 bits
    where 16-bit queries meet 64- or 128-wide heads in pages of whole 16-token tiles, fp32's elsewhere.  A call's scratch goes by the tables'
    width: up to 2 GB for the parts of long contexts, and up to 4 GB for expanded pages (where they would take more, nothing is expanded).

    Heads are whole groups over the cache's.  Slots that no token was stored in may hold anything."""
    cache.check()
    _check_step(tables, lengths, cu)
    pages, block, kv_heads, dim = cache.key.shape
    if q.dim() != 3 or q.shape[2] != dim or q.dtype not in _capi.DTYPE_CODES or q.shape[1] == 0 or q.shape[1] % kv_heads:
        raise ValueError("q must be [rows, heads, dim] in float32, float16 or bfloat16, with whole groups of heads over the cache's")
    if isinstance(window, bool) or not isinstance(window, int) or window < 0 or max_new < 0:
        raise ValueError("window and max_new must be integers that are not negative")
    index = _device_of(q, cache.key, cache.value, cache.key_scale, cache.value_scale, tables, lengths, cu)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != q.shape or out.dtype != q.dtype or out.data_ptr() == q.data_ptr() != 0:
        raise ValueError("out must have q's shape and dtype, and memory of its own")
    else:
        _device_of(q, out)
    rows, heads, _ = q.shape
    sequences, width = tables.shape
    q_stride, out_stride = _row_stride(q), _row_stride(out)
    if rows == 0 or sequences == 0:
        return out
    if width == 0:
        raise ValueError("tables need at least one page per sequence")
    window, dtype, max_new = min(window, 2 ** 31 - 1), _capi.DTYPE_CODES[q.dtype], min(int(max_new), rows)
    nbytes = _capi.load().rlt_quantized_attention_workspace_bytes(rows, sequences, max_new, heads, kv_heads, dim, block, width, window, dtype)
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None   # a call's own: graphs and streams share none
    _run("quantized_attention", index, q.data_ptr(), q_stride, out.data_ptr(), out_stride, *_cache_args(cache), heads, kv_heads, dim, dtype,
         tables.data_ptr(), lengths.data_ptr(), cu.data_ptr(), sequences, width, rows, max_new,
         float(1.0 / math.sqrt(dim) if scale is None else scale), window, None if workspace is None else workspace.data_ptr(), nbytes)
    return out
