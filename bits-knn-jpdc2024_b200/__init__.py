"""Python access to the bitsknn C ABI (libbitsknn.so), for the tests and the benchmark.

The product is the C-ABI library (include/bitsknn.h) and the C++ host layer above it; this
module only passes torch tensors' device pointers through ctypes.  There is no fallback: if
the library has not been built, importing `lib()` raises.

The directory name is not a Python identifier; load it with `load_package()` from
`__graft_entry__.py` or `importlib` (tests/conftest.py does this).
"""
import ctypes
import pathlib

_PKG = pathlib.Path(__file__).resolve().parent
LIB_PATH = _PKG / "lib" / "libbitsknn.so"

OK = 0
ERR_INVALID_ARGUMENT = 1
ERR_UNSUPPORTED_K = 2
ERR_UNSUPPORTED_DIM = 3
ERR_WORKSPACE = 4
ERR_CUDA = 5
ERR_DEVICE_TIMEOUT = 6
ERR_UNSUPPORTED_MODE = 7
ERR_COMM = 8
SHARDED_ID_BYTES = 128

F32, F16, BF16 = 0, 1, 2  # enum bitsknn_dtype
L2_EXACT, L2_PARTIAL, L2_TF32, L2_BF16 = 0, 1, 2, 3
STATIC_SCRATCH_BYTES = 8 << 20  # BITSKNN_STATIC_SCRATCH_BYTES

# every symbol include/bitsknn.h declares, with its ctypes signature
_i64 = ctypes.c_int64
_int = ctypes.c_int
_ptr = ctypes.c_void_p
_sz = ctypes.c_size_t


class _CacheStruct(ctypes.Structure):
    """bitsknn_cache_t"""
    _fields_ = [("d_keys", _ptr), ("d_values", _ptr), ("d_key_scales", _ptr), ("d_value_scales", _ptr), ("pages", _i64),
                ("page_stride", _i64), ("heads", ctypes.c_int32), ("page_rows", ctypes.c_int32), ("dim", ctypes.c_int32)]


class _BatchStruct(ctypes.Structure):
    """bitsknn_cache_batch_t"""
    _fields_ = [("d_table", _ptr), ("table_ld", _i64), ("table_pages", _i64), ("d_lengths", _ptr), ("d_starts", _ptr),
                ("requests", _i64), ("tokens", _i64)]


_cache_p = ctypes.POINTER(_CacheStruct)
_batch_p = ctypes.POINTER(_BatchStruct)
SIGNATURES = {
    "bitsknn_version": (_int, []),
    "bitsknn_last_error_string": (ctypes.c_char_p, []),
    "bitsknn_device_status": (_int, [_ptr]),
    "bitsknn_selftest_bounded_wait": (_int, [_ptr]),
    "bitsknn_set_tuning": (_int, [ctypes.c_char_p, _int]),
    "bitsknn_get_tuning": (_int, [ctypes.c_char_p, ctypes.POINTER(_int)]),
    "bitsknn_tuning_key": (ctypes.c_char_p, [_int]),
    "bitsknn_kernel_ms": (_int, [ctypes.c_char_p, ctypes.POINTER(ctypes.c_float)]),
    "bitsknn_select": (_int, [_ptr, _i64, _ptr, _i64, _ptr, _i64, _i64, _int, _ptr, _ptr, _ptr]),
    "bitsknn_select_ablation": (_int, [_ptr, _i64, _i64, _i64, _int, _int, _ptr, _ptr, _ptr]),
    "bitsknn_select_auto_splits": (_int, [_i64, _i64, _int]),
    "bitsknn_select_split_workspace_bytes": (_sz, [_i64, _int, _int]),
    "bitsknn_select_split": (_int, [_ptr, _i64, _ptr, _i64, _i64, _int, _int, _ptr, _sz, _ptr, _ptr, _ptr]),
    "bitsknn_select_split_static": (_int, [_ptr, _i64, _ptr, _i64, _i64, _int, _int, _ptr, _ptr, _ptr]),
    "bitsknn_merge": (_int, [_ptr, _ptr, _i64, _i64, _i64, _int, _int, _ptr, _ptr, _ptr]),
    "bitsknn_merge_lists": (_int, [_ptr, _ptr, _i64, _i64, _i64, _int, _int, _int, _ptr, _ptr, _ptr]),
    "bitsknn_refine": (_int, [_ptr, _ptr, _i64, _i64, _int, _ptr, _i64, _int, ctypes.c_int32, _int, _ptr, _ptr, _ptr]),
    "bitsknn_sharded_unique_id": (_int, [_ptr]),
    "bitsknn_sharded_create": (_int, [ctypes.POINTER(_ptr), _ptr, _int, _int]),
    "bitsknn_sharded_init": (_int, [ctypes.POINTER(_ptr), _ptr, _int, _int]),
    "bitsknn_sharded_destroy": (_int, [_ptr]),
    "bitsknn_sharded_workspace_bytes": (_sz, [_ptr, _i64, _int]),
    "bitsknn_sharded_search_select": (_int, [_ptr, _ptr, _i64, _i64, _i64, _int, ctypes.c_int32, _ptr, _ptr, _ptr, _sz,
                                             _ptr]),
    "bitsknn_sharded_submit_select": (_int, [_ptr, _ptr, _i64, _i64, _i64, _int, ctypes.c_int32, _ptr, _ptr, _ptr, _sz,
                                             _ptr]),
    "bitsknn_sharded_search_fused": (_int, [_ptr, _ptr, _ptr, _i64, _i64, _int, _int, _int, ctypes.c_int32, _ptr, _ptr,
                                            _ptr, _sz, _ptr, _sz, _ptr]),
    "bitsknn_sharded_drain": (_int, [_ptr, _ptr]),
    "bitsknn_l2_workspace_bytes": (_sz, [_i64, _i64, _int, _int]),
    "bitsknn_transpose": (_int, [_ptr, _i64, _i64, _ptr, _ptr]),
    "bitsknn_l2": (_int, [_ptr, _ptr, _i64, _i64, _int, _int, _ptr, _i64, _ptr, _sz, _ptr]),
    "bitsknn_fused_workspace_bytes": (_sz, [_i64, _i64, _int, _int, _int]),
    "bitsknn_cache_plan": (_int, [_ptr, _ptr, _i64, _int, _ptr, _i64, _ptr, _i64, _i64, _ptr, _ptr, _ptr, _i64, _ptr,
                                  _ptr]),
    "bitsknn_cache_append": (_int, [_cache_p, _ptr, _ptr, _int, _i64, _i64, _ptr, _i64, _ptr]),
    "bitsknn_cache_distance": (_int, [_cache_p, _batch_p, _ptr, _int, _i64, _int, _ptr, _i64, _i64, _ptr]),
    "bitsknn_cache_attend_workspace_bytes": (_sz, [_cache_p, _int]),
    "bitsknn_cache_attend": (_int, [_cache_p, _batch_p, _ptr, _int, _i64, _int, ctypes.c_float, _ptr, _i64, _ptr, _ptr,
                                    _sz, _ptr]),
    "bitsknn_cache_attend_selected": (_int, [_cache_p, _batch_p, _ptr, _int, _i64, _int, _ptr, _i64, _int,
                                             ctypes.c_float, _ptr, _i64, _ptr, _ptr, _sz, _ptr]),
    "bitsknn_fused": (_int, [_ptr, _ptr, _i64, _i64, _int, _int, _int, ctypes.c_int32, _ptr, _ptr, _ptr, _sz, _ptr]),
}

_LIB = None


class BitsKnnError(RuntimeError):
    """A non-zero status from the C ABI; `.status` holds the code."""

    def __init__(self, status, message):
        super().__init__(f"bitsknn status {status}: {message}")
        self.status = status
        self.message = message


def lib():
    """The loaded C-ABI library.  Raises if it has not been built (no CPU fallback exists)."""
    global _LIB
    if _LIB is None:
        if not LIB_PATH.exists():
            raise RuntimeError(f"{LIB_PATH} is missing: build it with bits-knn-jpdc2024_b200/build.py "
                               "(the k-NN kernels have no CPU fallback)")
        handle = ctypes.CDLL(str(LIB_PATH))
        for name, (restype, argtypes) in SIGNATURES.items():
            fn = getattr(handle, name)  # AttributeError if the header and the library diverge
            fn.restype = restype
            fn.argtypes = argtypes
        _LIB = handle
    return _LIB


def last_error():
    return lib().bitsknn_last_error_string().decode()


def _check(status):
    if status != OK:
        raise BitsKnnError(status, last_error())


def _p(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream():
    import torch
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def set_tuning(key, value):
    _check(lib().bitsknn_set_tuning(key.encode(), int(value)))


def get_tuning(key):
    out = ctypes.c_int(0)
    _check(lib().bitsknn_get_tuning(key.encode(), ctypes.byref(out)))
    return out.value


def tuning_keys():
    keys = []
    while True:
        key = lib().bitsknn_tuning_key(len(keys))
        if key is None:
            return keys
        keys.append(key.decode())


def kernel_ms(name):
    """Device time of the last timed launch of that kernel (knob "profile.kernel_events" = 1)."""
    out = ctypes.c_float(0)
    _check(lib().bitsknn_kernel_ms(name.encode(), ctypes.byref(out)))
    return out.value


def device_status():
    _check(lib().bitsknn_device_status(_stream()))


def selftest_bounded_wait():
    _check(lib().bitsknn_selftest_bounded_wait(_stream()))


def _device_check(t, dtype, name):
    import torch
    if t is None:
        return
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (the library has no CPU path)")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")


def select(dist, k, labels=None, label_offsets=None, n=None, out=None):
    """k smallest (distance, index) pairs of every row of a (q, ld) float32 CUDA matrix."""
    import torch
    _device_check(dist, torch.float32, "dist")
    _device_check(labels, torch.int32, "labels")
    _device_check(label_offsets, torch.int32, "label_offsets")
    q = dist.shape[0]
    ld = dist.stride(0) if q > 1 else dist.shape[1]
    n = dist.shape[1] if n is None else n
    if out is None:
        out = (torch.empty((q, k), dtype=torch.float32, device=dist.device),
               torch.empty((q, k), dtype=torch.int32, device=dist.device))
    ldl = 0 if labels is None else (labels.stride(0) if q > 1 else labels.shape[1])
    _check(lib().bitsknn_select(_p(dist), ld, _p(labels), ldl, _p(label_offsets), q, n, k,
                                _p(out[0]), _p(out[1]), _stream()))
    return out


ABLATION_NO_BUFFER, ABLATION_SHARED_LIST = 0, 1


def select_ablation(dist, k, variant, out=None):
    """The selection without its radius filter / with its list in shared memory (ablations)."""
    import torch
    _device_check(dist, torch.float32, "dist")
    q, n = dist.shape
    ld = dist.stride(0) if q > 1 else n
    if out is None:
        out = (torch.empty((q, k), dtype=torch.float32, device=dist.device),
               torch.empty((q, k), dtype=torch.int32, device=dist.device))
    _check(lib().bitsknn_select_ablation(_p(dist), ld, q, n, k, variant, _p(out[0]), _p(out[1]), _stream()))
    return out


def select_auto_splits(q, n, k):
    return int(lib().bitsknn_select_auto_splits(q, n, k))


def select_split_workspace_bytes(q, k, splits):
    return int(lib().bitsknn_select_split_workspace_bytes(q, k, splits))


def select_split(dist, k, splits=0, label_offsets=None, workspace=None, out=None):
    import torch
    _device_check(dist, torch.float32, "dist")
    q, n = dist.shape
    ld = dist.stride(0) if q > 1 else n
    if workspace is None:
        workspace = torch.empty(max(select_split_workspace_bytes(q, k, splits), 8), dtype=torch.uint8,
                                device=dist.device)
    if out is None:
        out = (torch.empty((q, k), dtype=torch.float32, device=dist.device),
               torch.empty((q, k), dtype=torch.int32, device=dist.device))
    _check(lib().bitsknn_select_split(_p(dist), ld, _p(label_offsets), q, n, k, splits, _p(workspace),
                                      workspace.numel(), _p(out[0]), _p(out[1]), _stream()))
    return out


def select_split_static(dist, k, splits, label_offsets=None, out=None):
    """Split-row selection whose candidate scratch is the library's built-in device array."""
    import torch
    _device_check(dist, torch.float32, "dist")
    q, n = dist.shape
    ld = dist.stride(0) if q > 1 else n
    if out is None:
        raise ValueError("pass the output tensors: this entry point is for callers that do not allocate")
    _check(lib().bitsknn_select_split_static(_p(dist), ld, _p(label_offsets), q, n, k, splits, _p(out[0]), _p(out[1]),
                                             _stream()))
    return out


def merge(cand_dist, cand_idx, out=None, sorted_lists=False):
    """cand_* of shape (lists, q, k), contiguous -> the k smallest pairs per query."""
    import torch
    _device_check(cand_dist, torch.float32, "cand_dist")
    _device_check(cand_idx, torch.int32, "cand_idx")
    lists, q, k = cand_dist.shape
    assert cand_dist.is_contiguous() and cand_idx.is_contiguous()
    if out is None:
        out = (torch.empty((q, k), dtype=torch.float32, device=cand_dist.device),
               torch.empty((q, k), dtype=torch.int32, device=cand_dist.device))
    _check(lib().bitsknn_merge_lists(_p(cand_dist), _p(cand_idx), q * k, k, q, lists, k, 1 if sorted_lists else 0,
                                     _p(out[0]), _p(out[1]), _stream()))
    return out


def merge_strided(cand_dist, cand_idx, list_stride, query_stride, q, lists, k, out=None, sorted_lists=False):
    """Merge with explicit element strides: pair j of list l of query i at
    [l * list_stride + i * query_stride + j] from the first element of each tensor."""
    import torch
    _device_check(cand_dist, torch.float32, "cand_dist")
    _device_check(cand_idx, torch.int32, "cand_idx")
    if out is None:
        out = (torch.empty((q, k), dtype=torch.float32, device=cand_dist.device),
               torch.empty((q, k), dtype=torch.int32, device=cand_dist.device))
    _check(lib().bitsknn_merge_lists(_p(cand_dist), _p(cand_idx), list_stride, query_stride, q, lists, k,
                                     1 if sorted_lists else 0, _p(out[0]), _p(out[1]), _stream()))
    return out


def refine(points, queries, cand_idx, k, index_base=0, out=None):
    """Exact FP32 re-ranking of (q, candidates) int32 candidate indices -> the k nearest by it."""
    import torch
    _device_check(points, torch.float32, "points")
    _device_check(queries, torch.float32, "queries")
    _device_check(cand_idx, torch.int32, "cand_idx")
    assert points.is_contiguous() and queries.is_contiguous()
    n, dim = points.shape
    q, cands = cand_idx.shape
    if out is None:
        out = (torch.empty((q, k), dtype=torch.float32, device=points.device),
               torch.empty((q, k), dtype=torch.int32, device=points.device))
    _check(lib().bitsknn_refine(_p(points), _p(queries), n, q, dim, _p(cand_idx), cand_idx.stride(0) if q > 1 else cands,
                                cands, index_base, k, _p(out[0]), _p(out[1]), _stream()))
    return out


def l2_workspace_bytes(n, q, dim, mode):
    return int(lib().bitsknn_l2_workspace_bytes(n, q, dim, mode))


def l2(points, queries, mode=L2_EXACT, out=None, workspace=None):
    """(q, n) squared-L2 matrix of row-major (n, dim) points and (q, dim) queries."""
    import torch
    _device_check(points, torch.float32, "points")
    _device_check(queries, torch.float32, "queries")
    assert points.is_contiguous() and queries.is_contiguous()
    n, dim = points.shape
    q = queries.shape[0]
    if out is None:
        out = torch.empty((q, n), dtype=torch.float32, device=points.device)
    need = l2_workspace_bytes(n, q, dim, mode)
    if workspace is None and need > 0:
        workspace = torch.empty(need, dtype=torch.uint8, device=points.device)
    _check(lib().bitsknn_l2(_p(points), _p(queries), n, q, dim, mode, _p(out), out.stride(0) if q > 1 else n,
                            _p(workspace), 0 if workspace is None else workspace.numel(), _stream()))
    return out


def transpose(src, out=None):
    """(rows, cols) float32 CUDA matrix -> its (cols, rows) transpose, on the device."""
    import torch
    _device_check(src, torch.float32, "src")
    assert src.is_contiguous()
    rows, cols = src.shape
    if out is None:
        out = torch.empty((cols, rows), dtype=torch.float32, device=src.device)
    _check(lib().bitsknn_transpose(_p(src), rows, cols, _p(out), _stream()))
    return out


def fused_workspace_bytes(n, q, dim, k, mode):
    return int(lib().bitsknn_fused_workspace_bytes(n, q, dim, k, mode))


def fused(points, queries, k, mode=L2_PARTIAL, index_base=0, out=None, workspace=None):
    """Brute-force k-NN without materialising the distance matrix."""
    import torch
    _device_check(points, torch.float32, "points")
    _device_check(queries, torch.float32, "queries")
    assert points.is_contiguous() and queries.is_contiguous()
    n, dim = points.shape
    q = queries.shape[0]
    if out is None:
        out = (torch.empty((q, k), dtype=torch.float32, device=points.device),
               torch.empty((q, k), dtype=torch.int32, device=points.device))
    need = fused_workspace_bytes(n, q, dim, k, mode)
    if workspace is None and need > 0:
        workspace = torch.empty(need, dtype=torch.uint8, device=points.device)
    _check(lib().bitsknn_fused(_p(points), _p(queries), n, q, dim, k, mode, index_base, _p(out[0]), _p(out[1]),
                               _p(workspace), 0 if workspace is None else workspace.numel(), _stream()))
    return out


# ---- search in a paged cache of keys and values held in 8 bits ---------------------------------
class Cache:
    """Keys and values as e4m3 codes in pages: uint8 (pages, heads, page_rows, dim) CUDA tensors and float32
    (pages, heads) scales.  Holds the tensors; pages may lie apart (stride of the first dimension)."""

    def __init__(self, keys, values, key_scales, value_scales):
        import torch
        for t, name in ((keys, "keys"), (values, "values")):
            _device_check(t, torch.uint8, name)
        for t, name in ((key_scales, "key_scales"), (value_scales, "value_scales")):
            _device_check(t, torch.float32, name)
        if keys.dim() != 4 or values.shape != keys.shape or values.stride() != keys.stride():
            raise ValueError("keys and values must be (pages, heads, page_rows, dim) tensors of the same strides")
        pages, heads, rows, dim = keys.shape
        if keys.stride()[1:] != (rows * dim, dim, 1):
            raise ValueError("a page must be contiguous")
        if any(tuple(s.shape) != (pages, heads) or not s.is_contiguous() for s in (key_scales, value_scales)):
            raise ValueError("scales must be contiguous (pages, heads) tensors")
        if any(t.device != keys.device for t in (values, key_scales, value_scales)):
            raise ValueError("the cache's tensors must be on one device")
        self.keys, self.values, self.key_scales, self.value_scales = keys, values, key_scales, value_scales
        self.pages, self.heads, self.page_rows, self.dim = pages, heads, rows, dim
        self.device = keys.device
        stride = keys.stride(0) if pages > 1 else heads * rows * dim
        self.struct = _CacheStruct(keys.data_ptr(), values.data_ptr(), key_scales.data_ptr(), value_scales.data_ptr(),
                                   pages, stride, heads, rows, dim)

    @classmethod
    def empty(cls, pages, heads, page_rows, dim, device="cuda"):
        """A cache without content; its pages are to be appended to from their first row."""
        import torch
        shape = (pages, heads, page_rows, dim)
        codes = [torch.zeros(shape, dtype=torch.uint8, device=device) for _ in range(2)]
        scales = [torch.zeros(shape[:2], dtype=torch.float32, device=device) for _ in range(2)]
        return cls(*codes, *scales)

    def batch(self, queries, lengths, table, starts):
        """(bitsknn_cache_batch_t, dtype code, elements between tokens) of a call's arguments.  These wrappers run once
        per layer and step: they look at every argument once and keep nothing between calls."""
        import torch
        if queries.dim() != 3 or queries.shape[2] != self.dim:
            raise ValueError(f"queries have shape {tuple(queries.shape)}, which does not fit the cache")
        code, stride = _vectors(queries, "queries")
        if lengths.dtype is not torch.int32 or table.dtype is not torch.int32:
            raise ValueError("lengths and table must be torch.int32")
        tokens, (requests, pages), (ld, inner) = queries.shape[0], table.shape, table.stride()
        if lengths.shape != (requests,) or (inner != 1 and pages > 1) or (requests > 1 and lengths.stride(0) != 1):
            raise ValueError("table must be (requests, pages) and lengths (requests,), contiguous in the last dimension")
        if starts is not None and (starts.dtype is not torch.int32 or starts.shape != (requests + 1,)
                                   or (requests > 0 and starts.stride(0) != 1)):
            raise ValueError("starts must be a contiguous (requests + 1,) torch.int32 tensor")
        _on_device(self.device, queries, lengths, table, starts)
        return _BatchStruct(table.data_ptr(), ld if requests > 1 else pages, pages, lengths.data_ptr(),
                            None if starts is None else starts.data_ptr(), requests, tokens), code, stride


def _on_device(device, *tensors):
    import torch
    if device.index != torch.cuda.current_device():
        raise ValueError(f"the tensors are on {device}, which is not the current device")
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"tensors on {device} and {t.device} (the library has no CPU path)")


def _vectors(t, name):
    """(dtype code, elements between tokens) of a (tokens, heads, dim) tensor of vectors."""
    import torch
    dtype = t.dtype
    code = BF16 if dtype is torch.bfloat16 else F16 if dtype is torch.float16 else F32 if dtype is torch.float32 else None
    if code is None:
        raise ValueError(f"{name} must be float32, float16 or bfloat16")
    tokens, heads, dim = t.shape
    outer, middle, inner = t.stride()
    if inner != 1 or (heads > 1 and middle != dim):
        raise ValueError(f"{name} must be contiguous in its last two dimensions")
    return code, outer if tokens > 1 else heads * dim


def cache_plan(lengths, new, free_pages, table, page_rows, max_tokens, out=None):
    """Places for `new` tokens of every request: writes the new pages into `table` and returns
    (starts, new_lengths, slots, counts); counts = (tokens, pages taken, tokens without a place)."""
    import torch
    int32, device = torch.int32, lengths.device
    for t, name in ((lengths, "lengths"), (new, "new"), (free_pages, "free_pages"), (table, "table")):
        if not t.is_cuda or t.dtype is not int32:
            raise ValueError(f"{name} must be a torch.int32 CUDA tensor (the library has no CPU path)")
        if t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"{name} must be contiguous in its last dimension")
    _on_device(device, new, free_pages, table)
    requests, pages = table.shape
    if lengths.shape != (requests,) or new.shape != (requests,) or free_pages.dim() != 1:
        raise ValueError("lengths and new must be (requests,), table (requests, pages)")
    if out is None:
        out = (torch.empty(requests + 1, dtype=int32, device=device), torch.empty(requests, dtype=int32, device=device),
               torch.empty(max_tokens, dtype=torch.int64, device=device), torch.empty(3, dtype=int32, device=device))
    _check(lib().bitsknn_cache_plan(lengths.data_ptr(), new.data_ptr(), requests, page_rows, free_pages.data_ptr(),
                                    free_pages.shape[0], table.data_ptr(), table.stride(0) if requests > 1 else pages, pages,
                                    out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), max_tokens,
                                    out[3].data_ptr(), _stream()))
    return out


def cache_append(cache, keys, values, slots):
    """Quantises (tokens, heads, dim) keys and values into the cache at `slots` (int64, from cache_plan)."""
    import torch
    shape = keys.shape
    if values.shape != shape or len(shape) != 3 or shape[1] != cache.heads or shape[2] != cache.dim:
        raise ValueError(f"keys {tuple(shape)} and values {tuple(values.shape)} do not fit the cache")
    code, key_stride = _vectors(keys, "keys")
    value_code, value_stride = _vectors(values, "values")
    tokens = shape[0]
    if value_code != code or slots.dtype is not torch.int64 or slots.dim() != 1 or slots.shape[0] < tokens:
        raise ValueError("keys and values must agree in type, and every token needs an int64 slot")
    if tokens > 1 and slots.stride(0) != 1:
        raise ValueError("slots must be contiguous in its last dimension")
    _on_device(cache.device, keys, values, slots)
    _check(lib().bitsknn_cache_append(cache.struct, keys.data_ptr(), values.data_ptr(), code, key_stride, value_stride,
                                      slots.data_ptr(), tokens, _stream()))


def cache_distance(cache, queries, lengths, table, n, starts=None, out=None):
    """(tokens * heads, n) float32 distances for `select`: minus the largest inner product over a head's queries."""
    import torch
    batch, code, stride = cache.batch(queries, lengths, table, starts)
    rows = queries.shape[0] * cache.heads
    if out is None:
        out = torch.empty((rows, n), dtype=torch.float32, device=cache.device)
    else:
        _device_check(out, torch.float32, "out")
        _on_device(cache.device, out)
        if out.dim() != 2 or out.shape[0] < rows or out.shape[1] < n:
            raise ValueError("out must have tokens * heads rows of n distances")
    _check(lib().bitsknn_cache_distance(cache.struct, batch, queries.data_ptr(), code, stride, queries.shape[1],
                                        out.data_ptr(), out.stride(0) if out.shape[0] > 1 else out.shape[1], n, _stream()))
    return out


def cache_attend_workspace_bytes(cache, query_heads):
    return int(lib().bitsknn_cache_attend_workspace_bytes(cache.struct, query_heads))


def _attend_buffers(cache, queries, out, lse, workspace):
    import torch
    shape, device = queries.shape, cache.device
    stride = 0
    if out is None:
        out = torch.empty(shape, dtype=queries.dtype, device=device)
    elif out.shape != shape or out.dtype is not queries.dtype:
        raise ValueError("out must have the queries' shape and type")
    else:
        _on_device(device, out)
        stride = _vectors(out, "out")[1]
    if lse is None:
        lse = torch.empty(shape[:2], dtype=torch.float32, device=device)
    elif lse.shape != shape[:2] or lse.dtype is not torch.float32 or not lse.is_contiguous():
        raise ValueError("lse must be a contiguous (tokens, query_heads) float32 tensor")
    else:
        _on_device(device, lse)
    if workspace is None:
        workspace = torch.empty(cache_attend_workspace_bytes(cache, shape[1]), dtype=torch.uint8, device=device)
    elif workspace.dtype is not torch.uint8 or workspace.device != device or not workspace.is_contiguous():
        raise ValueError("workspace must be a contiguous uint8 tensor on the cache's device")
    return out, stride, lse, workspace


def cache_attend(cache, queries, lengths, table, scale, starts=None, out=None, lse=None, workspace=None):
    """Attention of (tokens, query_heads, dim) queries over everything cached: (out, lse)."""
    batch, code, stride = cache.batch(queries, lengths, table, starts)
    out, out_stride, lse, workspace = _attend_buffers(cache, queries, out, lse, workspace)
    _check(lib().bitsknn_cache_attend(cache.struct, batch, queries.data_ptr(), code, stride, queries.shape[1], scale,
                                      out.data_ptr(), out_stride, lse.data_ptr(), workspace.data_ptr(),
                                      workspace.numel(), _stream()))
    return out, lse


def cache_attend_selected(cache, queries, idx, lengths, table, scale, starts=None, out=None, lse=None, workspace=None):
    """Attention over listed positions: idx (tokens * heads, k) int32, as `select` returns them.  (out, lse)."""
    import torch
    batch, code, stride = cache.batch(queries, lengths, table, starts)
    if idx.dim() != 2 or idx.shape[0] != queries.shape[0] * cache.heads:
        raise ValueError("idx must be (tokens * heads, k)")
    rows, k = idx.shape
    if idx.dtype is not torch.int32 or (k > 1 and idx.stride(1) != 1):
        raise ValueError("idx must be torch.int32, contiguous in its last dimension")
    _on_device(cache.device, idx)
    out, out_stride, lse, workspace = _attend_buffers(cache, queries, out, lse, workspace)
    _check(lib().bitsknn_cache_attend_selected(cache.struct, batch, queries.data_ptr(), code, stride, queries.shape[1],
                                               idx.data_ptr(), idx.stride(0) if rows > 1 else k, k, scale, out.data_ptr(),
                                               out_stride, lse.data_ptr(), workspace.data_ptr(), workspace.numel(),
                                               _stream()))
    return out, lse


# ---- database-sharded search (one handle per GPU; NCCL inside the library) --------------------
def sharded_unique_id():
    """An NCCL unique id (bytes) made on the calling rank; distribute it to the other ranks."""
    buf = ctypes.create_string_buffer(SHARDED_ID_BYTES)
    _check(lib().bitsknn_sharded_unique_id(buf))
    return buf.raw


def sharded_create(unique_id, rank, world):
    """Handle with its own communicator (collective over the ranks; the rank's device is current)."""
    handle = ctypes.c_void_p()
    buf = None if unique_id is None else ctypes.create_string_buffer(bytes(unique_id), SHARDED_ID_BYTES)
    _check(lib().bitsknn_sharded_create(ctypes.byref(handle), buf, rank, world))
    return handle


def sharded_destroy(handle):
    _check(lib().bitsknn_sharded_destroy(handle))


def sharded_workspace_bytes(handle, q, k):
    return int(lib().bitsknn_sharded_workspace_bytes(handle, q, k))


def _sharded_out(q, k, device, out):
    import torch
    if out is None:
        out = (torch.empty((q, k), dtype=torch.float32, device=device),
               torch.empty((q, k), dtype=torch.int32, device=device))
    return out


def sharded_select(handle, dist, k, shard_begin, workspace, out=None, wait=True):
    """One sharded selection; `wait=False` is the submit form (finish with `sharded_drain`)."""
    import torch
    _device_check(dist, torch.float32, "dist")
    q, n = dist.shape
    ld = dist.stride(0) if q > 1 else n
    out = _sharded_out(q, k, dist.device, out)
    fn = lib().bitsknn_sharded_search_select if wait else lib().bitsknn_sharded_submit_select
    _check(fn(handle, _p(dist), ld, q, n, k, shard_begin, _p(out[0]), _p(out[1]), _p(workspace),
              0 if workspace is None else workspace.numel(), _stream()))
    return out


def sharded_fused(handle, points, queries, k, shard_begin, workspace, mode=L2_PARTIAL, fused_workspace=None, out=None):
    import torch
    _device_check(points, torch.float32, "points")
    _device_check(queries, torch.float32, "queries")
    assert points.is_contiguous() and queries.is_contiguous()
    n, dim = points.shape
    q = queries.shape[0]
    out = _sharded_out(q, k, points.device, out)
    need = fused_workspace_bytes(n, q, dim, k, mode)
    if fused_workspace is None and need > 0:
        fused_workspace = torch.empty(need, dtype=torch.uint8, device=points.device)
    _check(lib().bitsknn_sharded_search_fused(handle, _p(points), _p(queries), n, q, dim, k, mode, shard_begin,
                                              _p(out[0]), _p(out[1]), _p(fused_workspace),
                                              0 if fused_workspace is None else fused_workspace.numel(), _p(workspace),
                                              0 if workspace is None else workspace.numel(), _stream()))
    return out


def sharded_drain(handle):
    _check(lib().bitsknn_sharded_drain(handle, _stream()))
