"""Paged cache of keys and values held in 8 bits: the access layer of the `bitsknn_cache_*` entry points.

These calls run once per layer and decode step, where a microsecond on the host counts: every argument is looked at
once, tensors' devices are compared as integers, sizes go to the allocation one by one (a torch.Size costs it
another 1.5 us), and nothing is kept between calls.
"""
import torch
from torch import bfloat16, empty, empty_like, float16, float32, int32, int64, uint8

from . import BF16, F16, F32, BatchStruct, BitsKnnError, CacheStruct, last_error, lib

_CODES = {bfloat16: BF16, float16: F16, float32: F32}
_current_device = torch.cuda.current_device
_raw_stream = torch._C._cuda_getCurrentRawStream  # torch.cuda.current_stream(device).cuda_stream without the object


def _run(fn, *args):
    status = fn(*args)
    if status != 0:
        raise BitsKnnError(status, last_error())


def _current(index, *tensors):
    """The tensors must be CUDA tensors of the current device (`index`): the library has no CPU path and launches on
    the current device."""
    if index < 0 or index != _current_device():
        raise ValueError("the tensors must be CUDA tensors of the current device (the library has no CPU path), "
                         f"not of device {index}")
    for t in tensors:
        if t.get_device() != index:
            raise ValueError(f"all tensors must be on CUDA device {index} (the library has no CPU path), not {t.device}")


def _token_stride(name, shape, stride):
    """Elements between the tokens of a (tokens, heads, dim) tensor whose vectors lie one after the other."""
    tokens, heads, dim = shape
    if stride[2] != 1 or (heads > 1 and stride[1] != dim):
        raise ValueError(f"{name} must be contiguous in its last two dimensions")
    if tokens < 2:
        return heads * dim
    if stride[0] < heads * dim:  # 0 (an expanded tensor) would mean dense to the library
        raise ValueError(f"the tokens of {name} must not overlap")
    return stride[0]


def _dense(t, dtype, name):
    if t.dtype is not dtype or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor")


class Cache:
    """Keys and values as e4m3 codes in pages: uint8 (pages, heads, page_rows, dim) CUDA tensors and float32
    (pages, heads) scales.  Holds the tensors; pages may lie apart (stride of the first dimension)."""

    def __init__(self, keys, values, key_scales, value_scales):
        if keys.dim() != 4 or values.shape != keys.shape:
            raise ValueError("keys and values must be (pages, heads, page_rows, dim) tensors of the same shape")
        if keys.dtype is not uint8 or values.dtype is not uint8:
            raise ValueError("keys and values must be uint8 (e4m3 codes)")
        pages, heads, rows, dim = keys.shape
        # strides of dimensions of one entry are never used, and differ between views of the same memory
        for t in (keys, values):
            for size, have, want in zip(t.shape[1:], t.stride()[1:], (rows * dim, dim, 1)):
                if have != want and size > 1:
                    raise ValueError("a page must be contiguous")
        if pages > 1 and values.stride(0) != keys.stride(0):
            raise ValueError("the pages of keys and values must lie equally far apart")
        stride = keys.stride(0) if pages > 1 else heads * rows * dim
        if stride < heads * rows * dim:
            raise ValueError("pages must not overlap")
        for t, name in ((key_scales, "key_scales"), (value_scales, "value_scales")):
            _dense(t, float32, name)
            if t.shape != (pages, heads):
                raise ValueError(f"{name} must be (pages, heads)")
        self.index = keys.get_device()
        if self.index < 0 or any(t.get_device() != self.index for t in (values, key_scales, value_scales)):
            raise ValueError("the cache's tensors must be CUDA tensors of one device (the library has no CPU path)")
        self.keys, self.values, self.key_scales, self.value_scales = keys, values, key_scales, value_scales
        self.pages, self.heads, self.page_rows, self.dim = pages, heads, rows, dim
        self.device = keys.device
        self.struct = CacheStruct(keys.data_ptr(), values.data_ptr(), key_scales.data_ptr(), value_scales.data_ptr(),
                                  pages, stride, heads, rows, dim)

    @classmethod
    def empty(cls, pages, heads, page_rows, dim, device="cuda"):
        """A cache without content; its pages are to be appended to from their first row."""
        shape = (pages, heads, page_rows, dim)
        codes = [torch.zeros(shape, dtype=uint8, device=device) for _ in range(2)]
        scales = [torch.zeros(shape[:2], dtype=float32, device=device) for _ in range(2)]
        return cls(*codes, *scales)


def _batch(cache, queries, shape, lengths, table, starts, *more):
    """bitsknn_cache_batch_t of a call; all its tensors (`more`: further ones) have to be on the current device."""
    if len(shape) != 3 or shape[2] != cache.dim:
        raise ValueError(f"queries of shape {tuple(shape)} do not fit the cache")
    if lengths.dtype is not int32 or table.dtype is not int32:
        raise ValueError("lengths and table must be torch.int32")
    requests, pages = table.shape
    ld, inner = table.stride()
    if lengths.shape != (requests,) or (inner != 1 and pages > 1) or not lengths.is_contiguous():
        raise ValueError("table must be (requests, pages) and lengths (requests,), contiguous in the last dimension")
    first = None
    if starts is not None:
        _dense(starts, int32, "starts")
        if starts.shape != (requests + 1,):
            raise ValueError("starts must be (requests + 1,)")
        first = starts.data_ptr()
    _current(cache.index, queries, lengths, table, *(() if starts is None else (starts,)), *more)
    return BatchStruct(table.data_ptr(), ld if requests > 1 else pages, pages, lengths.data_ptr(), first, requests,
                       shape[0])


def _code(t, name):
    code = _CODES.get(t.dtype)
    if code is None:
        raise ValueError(f"{name} must be float32, float16 or bfloat16")
    return code


def cache_plan(lengths, new, free_pages, table, page_rows, max_tokens, out=None):
    """Places for `new` tokens of every request: writes the new pages into `table` and returns
    (starts, new_lengths, slots, counts); counts = (tokens, pages taken, tokens without a place)."""
    index = lengths.get_device()
    _current(index, new, free_pages, table)
    requests, pages = table.shape
    ld, inner = table.stride()
    for t, name in ((lengths, "lengths"), (new, "new"), (free_pages, "free_pages")):
        _dense(t, int32, name)
    if table.dtype is not int32 or (inner != 1 and pages > 1):
        raise ValueError("table must be torch.int32, contiguous in its last dimension")
    if lengths.shape != (requests,) or new.shape != (requests,) or free_pages.dim() != 1:
        raise ValueError("lengths and new must be (requests,), table (requests, pages)")
    if out is None:
        out = (lengths.new_empty(requests + 1), empty_like(lengths),
               empty(max_tokens, dtype=int64, device=lengths.device), lengths.new_empty(3))
    else:
        for t, dtype, size, name in zip(out, (int32, int32, int64, int32), (requests + 1, requests, max_tokens, 3),
                                        ("starts", "new_lengths", "slots", "counts")):
            _dense(t, dtype, name)
            if t.numel() < size:
                raise ValueError(f"{name} must have {size} elements")
        _current(index, *out)
    starts, new_lengths, slots, counts = out
    _run(lib().bitsknn_cache_plan, lengths.data_ptr(), new.data_ptr(), requests, page_rows, free_pages.data_ptr(),
         free_pages.numel(), table.data_ptr(), ld if requests > 1 else pages, pages, starts.data_ptr(),
         new_lengths.data_ptr(), slots.data_ptr(), max_tokens, counts.data_ptr(), _raw_stream(index))
    return out


def cache_append(cache, keys, values, slots):
    """Quantises (tokens, heads, dim) keys and values into the cache at `slots` (int64, from cache_plan)."""
    shape = keys.shape
    if values.shape != shape or len(shape) != 3 or shape[1] != cache.heads or shape[2] != cache.dim:
        raise ValueError(f"keys {tuple(shape)} and values {tuple(values.shape)} do not fit the cache")
    _dense(slots, int64, "slots")
    tokens = shape[0]
    if values.dtype is not keys.dtype or slots.numel() < tokens:
        raise ValueError("keys and values must agree in type, and every token needs a slot")
    _current(cache.index, keys, values, slots)
    _run(lib().bitsknn_cache_append, cache.struct, keys.data_ptr(), values.data_ptr(), _code(keys, "keys"),
         _token_stride("keys", shape, keys.stride()), _token_stride("values", shape, values.stride()), slots.data_ptr(),
         tokens, _raw_stream(cache.index))


def cache_distance(cache, queries, lengths, table, n, starts=None, out=None):
    """(tokens * heads, n) float32 distances for `select`: minus the largest inner product over a head's queries.  Rows of
    tokens behind the last request are left as they were, which is undefined where the call allocates `out`."""
    shape = queries.shape
    batch = _batch(cache, queries, shape, lengths, table, starts)
    rows = shape[0] * cache.heads
    if out is None:
        out = empty(rows, n, dtype=float32, device=cache.device)
        ld = n
    else:
        _current(cache.index, out)
        if out.dim() != 2 or out.dtype is not float32 or out.shape[0] < rows or out.shape[1] < n:
            raise ValueError("out must be float32 and have tokens * heads rows of n distances")
        if out.shape[1] > 1 and out.stride(1) != 1:
            raise ValueError("out must be contiguous in its last dimension")
        ld = out.stride(0) if out.shape[0] > 1 else out.shape[1]
    _run(lib().bitsknn_cache_distance, cache.struct, batch, queries.data_ptr(), _code(queries, "queries"),
         _token_stride("queries", shape, queries.stride()), shape[1], out.data_ptr(), ld, n, _raw_stream(cache.index))
    return out


def cache_attend_workspace_bytes(cache, query_heads):
    return int(lib().bitsknn_cache_attend_workspace_bytes(cache.struct, query_heads))


def _attend_buffers(cache, queries, shape, out, lse, workspace):
    """(out, elements between its tokens, lse, workspace)"""
    stride = 0
    if out is None:
        out = empty_like(queries) if queries.is_contiguous() else empty(*shape, dtype=queries.dtype, device=cache.device)
    else:
        _current(cache.index, out)
        if out.shape != shape or out.dtype is not queries.dtype:
            raise ValueError("out must have the queries' shape and type")
        stride = _token_stride("out", shape, out.stride())
    if lse is None:
        lse = empty(shape[0], shape[1], dtype=float32, device=cache.device)
    else:
        _current(cache.index, lse)
        _dense(lse, float32, "lse")
        if lse.shape != shape[:2]:
            raise ValueError("lse must be (tokens, query_heads)")
    if workspace is None:
        workspace = empty(cache_attend_workspace_bytes(cache, shape[1]), dtype=uint8, device=cache.device)
    else:
        _dense(workspace, uint8, "workspace")
        if workspace.get_device() != cache.index:
            raise ValueError("workspace must be on the cache's device")
    return out, stride, lse, workspace


def cache_attend(cache, queries, lengths, table, scale, starts=None, out=None, lse=None, workspace=None):
    """Attention of (tokens, query_heads, dim) queries over everything cached: (out, lse).  Rows of tokens behind the last
    request are left as they were, which is undefined where the call allocates `out` and `lse`.  With one token for each
    request leave `starts` out: few short requests then take one launch."""
    shape = queries.shape
    batch = _batch(cache, queries, shape, lengths, table, starts)
    out, out_stride, lse, workspace = _attend_buffers(cache, queries, shape, out, lse, workspace)
    _run(lib().bitsknn_cache_attend, cache.struct, batch, queries.data_ptr(), _code(queries, "queries"),
         _token_stride("queries", shape, queries.stride()), shape[1], scale, out.data_ptr(), out_stride, lse.data_ptr(),
         workspace.data_ptr(), workspace.numel(), _raw_stream(cache.index))
    return out, lse


def cache_attend_selected(cache, queries, idx, lengths, table, scale, starts=None, out=None, lse=None, workspace=None):
    """Attention over listed positions: idx (tokens * heads, k) int32, as `select` returns them.  (out, lse), as from
    cache_attend."""
    shape = queries.shape
    batch = _batch(cache, queries, shape, lengths, table, starts, idx)
    rows, k = idx.shape
    ld, inner = idx.stride()
    if rows != shape[0] * cache.heads:
        raise ValueError("idx must be (tokens * heads, k)")
    if idx.dtype is not int32 or (k > 1 and inner != 1):
        raise ValueError("idx must be torch.int32, contiguous in its last dimension")
    out, out_stride, lse, workspace = _attend_buffers(cache, queries, shape, out, lse, workspace)
    _run(lib().bitsknn_cache_attend_selected, cache.struct, batch, queries.data_ptr(), _code(queries, "queries"),
         _token_stride("queries", shape, queries.stride()), shape[1], idx.data_ptr(), ld if rows > 1 else k, k, scale,
         out.data_ptr(), out_stride, lse.data_ptr(), workspace.data_ptr(), workspace.numel(), _raw_stream(cache.index))
    return out, lse
