"""What the paged-cache entry points refuse, checked without a device: every refusal comes before the first CUDA call."""
import ctypes

import pytest

FAKE = 4096


def cache_struct(bk, **over):
    fields = dict(d_keys=FAKE, d_values=FAKE, d_key_scales=FAKE, d_value_scales=FAKE, pages=4, page_stride=0, heads=2,
                  page_rows=16, dim=64)
    fields.update(over)
    return bk.CacheStruct(*(fields[name] for name, _ in bk.CacheStruct._fields_))


def batch_struct(bk, **over):
    fields = dict(d_table=FAKE, table_ld=4, table_pages=4, d_lengths=FAKE, d_starts=None, requests=3, tokens=3)
    fields.update(over)
    return bk.BatchStruct(*(fields[name] for name, _ in bk.BatchStruct._fields_))


def attend(bk, cache=None, batch=None, queries=FAKE, dtype=None, stride=0, query_heads=4, out=FAKE, out_stride=0,
           workspace=FAKE, size=1 << 40, lse=None):
    return bk.lib().bitsknn_cache_attend(cache or cache_struct(bk), batch or batch_struct(bk), queries,
                                         bk.BF16 if dtype is None else dtype, stride, query_heads, 0.1, out, out_stride,
                                         lse, workspace, size, None)


@pytest.mark.parametrize("over, status", [
    (dict(d_keys=None), "ERR_INVALID_ARGUMENT"),
    (dict(d_value_scales=None), "ERR_INVALID_ARGUMENT"),
    (dict(dim=80), "ERR_UNSUPPORTED_DIM"),
    (dict(dim=0), "ERR_UNSUPPORTED_DIM"),
    (dict(page_rows=24), "ERR_INVALID_ARGUMENT"),
    (dict(page_rows=8), "ERR_INVALID_ARGUMENT"),
    (dict(page_rows=512), "ERR_INVALID_ARGUMENT"),
    (dict(pages=0), "ERR_INVALID_ARGUMENT"),
    (dict(heads=0), "ERR_INVALID_ARGUMENT"),
    (dict(page_stride=2047), "ERR_INVALID_ARGUMENT"),
    (dict(page_stride=2 * 16 * 64 + 8), "ERR_INVALID_ARGUMENT"),
    (dict(d_keys=FAKE + 8), "ERR_INVALID_ARGUMENT"),
    (dict(d_key_scales=FAKE + 2), "ERR_INVALID_ARGUMENT"),
])
def test_caches_that_are_refused(bk, over, status):
    cache = cache_struct(bk, **over)
    want = getattr(bk, status)
    assert attend(bk, cache=cache) == want
    lib = bk.lib()
    assert lib.bitsknn_cache_append(cache, FAKE, FAKE, bk.F32, 0, 0, FAKE, 1, None) == want
    assert lib.bitsknn_cache_distance(cache, batch_struct(bk), FAKE, bk.F16, 0, 4, FAKE, 64, 64, None) == want
    assert lib.bitsknn_cache_attend_workspace_bytes(cache, 4) == 0
    assert bk.last_error()


@pytest.mark.parametrize("over", [
    dict(d_table=None), dict(d_lengths=None), dict(table_ld=3), dict(table_pages=-1), dict(tokens=5), dict(requests=-1),
    dict(tokens=1 << 31, d_starts=FAKE)])
def test_batches_that_are_refused(bk, over):
    batch = batch_struct(bk, **over)
    assert attend(bk, batch=batch) == bk.ERR_INVALID_ARGUMENT
    assert bk.lib().bitsknn_cache_distance(cache_struct(bk), batch, FAKE, bk.F16, 0, 4, FAKE, 64, 64,
                                           None) == bk.ERR_INVALID_ARGUMENT


def test_queries_that_are_refused(bk):
    assert attend(bk, dtype=bk.F32) == bk.ERR_UNSUPPORTED_MODE
    assert attend(bk, dtype=7) == bk.ERR_UNSUPPORTED_MODE
    assert attend(bk, query_heads=3) == bk.ERR_INVALID_ARGUMENT       # not a multiple of the cache's heads
    assert attend(bk, query_heads=0) == bk.ERR_INVALID_ARGUMENT
    assert attend(bk, queries=None) == bk.ERR_INVALID_ARGUMENT
    assert attend(bk, queries=FAKE + 4) == bk.ERR_INVALID_ARGUMENT
    assert attend(bk, stride=4 * 64 - 8) == bk.ERR_INVALID_ARGUMENT
    assert attend(bk, stride=4 * 64 + 4) == bk.ERR_INVALID_ARGUMENT
    assert attend(bk, out=None) == bk.ERR_INVALID_ARGUMENT
    assert attend(bk, out=FAKE + 1) == bk.ERR_INVALID_ARGUMENT
    assert attend(bk, out_stride=100) == bk.ERR_INVALID_ARGUMENT
    assert attend(bk, lse=FAKE + 2) == bk.ERR_INVALID_ARGUMENT


def test_workspaces_that_are_refused(bk):
    size = bk.lib().bitsknn_cache_attend_workspace_bytes(cache_struct(bk), 4)
    assert size > 0
    assert attend(bk, workspace=None) == bk.ERR_WORKSPACE
    assert attend(bk, workspace=FAKE + 64) == bk.ERR_INVALID_ARGUMENT
    assert attend(bk, size=1000) == bk.ERR_WORKSPACE
    assert "smaller than" in bk.last_error()


def test_selected_lists_that_are_refused(bk):
    fn = bk.lib().bitsknn_cache_attend_selected

    def call(idx=FAKE, ld=8, k=8):
        return fn(cache_struct(bk), batch_struct(bk), FAKE, bk.F16, 0, 4, idx, ld, k, 0.1, FAKE, 0, None, FAKE, 100, None)

    assert call(k=0) == bk.ERR_UNSUPPORTED_K
    assert "Unsupported k value: 0" in bk.last_error()
    assert call(k=(1 << 30) + 1, ld=1 << 31) == bk.ERR_UNSUPPORTED_K
    assert call(ld=7) == bk.ERR_INVALID_ARGUMENT
    assert call(idx=None) == bk.ERR_INVALID_ARGUMENT
    assert call(idx=FAKE + 2) == bk.ERR_INVALID_ARGUMENT
    assert call() == bk.ERR_WORKSPACE


def test_distance_matrices_that_are_refused(bk):
    def call(dist=FAKE, ld=64, n=64):
        return bk.lib().bitsknn_cache_distance(cache_struct(bk), batch_struct(bk), FAKE, bk.F16, 0, 4, dist, ld, n, None)

    assert call(dist=None) == bk.ERR_INVALID_ARGUMENT
    assert call(dist=FAKE + 2) == bk.ERR_INVALID_ARGUMENT
    assert call(ld=63) == bk.ERR_INVALID_ARGUMENT
    assert call(n=-1) == bk.ERR_INVALID_ARGUMENT


def test_appends_that_are_refused(bk):
    def call(keys=FAKE, dtype=bk.F16, key_stride=0, value_stride=0, slots=FAKE, tokens=2):
        return bk.lib().bitsknn_cache_append(cache_struct(bk), keys, FAKE, dtype, key_stride, value_stride, slots, tokens,
                                             None)

    assert call(keys=None) == bk.ERR_INVALID_ARGUMENT
    assert call(keys=FAKE + 8) == bk.ERR_INVALID_ARGUMENT
    assert call(dtype=3) == bk.ERR_UNSUPPORTED_MODE
    assert call(key_stride=127) == bk.ERR_INVALID_ARGUMENT
    assert call(value_stride=132) == bk.ERR_INVALID_ARGUMENT          # halves: rows would not be 16-byte aligned
    assert call(slots=None) == bk.ERR_INVALID_ARGUMENT
    assert call(tokens=-1) == bk.ERR_INVALID_ARGUMENT
    assert call(keys=None, slots=None, tokens=0) == bk.OK


def test_plans_that_are_refused(bk):
    p = [ctypes.c_void_p(FAKE * (i + 1)) for i in range(8)]

    def call(lengths=p[0], new=p[1], requests=3, page_rows=16, free=p[2], table=p[3], ld=4, starts=p[4], out=p[5],
             slots=p[6], tokens=8, counts=p[7]):
        return bk.lib().bitsknn_cache_plan(lengths, new, requests, page_rows, free, 5, table, ld, 4, starts, out, slots,
                                           tokens, counts, None)

    for name in ("lengths", "new", "free", "table", "starts", "out", "slots", "counts"):
        assert call(**{name: None}) == bk.ERR_INVALID_ARGUMENT, name
    assert call(page_rows=20) == bk.ERR_INVALID_ARGUMENT
    assert call(ld=3) == bk.ERR_INVALID_ARGUMENT
    assert call(requests=-1) == bk.ERR_INVALID_ARGUMENT
    assert call(tokens=-1) == bk.ERR_INVALID_ARGUMENT
    assert call(out=p[0]) == bk.ERR_INVALID_ARGUMENT                   # lengths are read while the new ones are written
    assert call(out=p[1]) == bk.ERR_INVALID_ARGUMENT


def test_python_layer_refuses_tensors_that_do_not_fit(bk):
    import torch
    codes = torch.zeros((2, 1, 16, 32), dtype=torch.uint8)
    with pytest.raises(ValueError, match="CUDA tensor"):
        bk.Cache(codes, codes, torch.zeros(2, 1), torch.zeros(2, 1))
    with pytest.raises(ValueError, match="CUDA tensor"):
        bk.cache_plan(torch.zeros(1, dtype=torch.int32), None, None, None, 16, 1)


def test_python_layer_refuses_rows_that_overlap(bk):
    """An expanded tensor has stride 0, which the library would take for dense rows."""
    import torch
    from importlib import import_module
    token_stride = import_module(bk.__name__ + ".cache")._token_stride
    wide = torch.zeros((5, 4, 32))
    assert token_stride("out", wide.shape, wide.stride()) == 128
    assert token_stride("out", (1, 4, 32), (0, 32, 1)) == 128
    for x in (wide[:1].expand(5, 4, 32), wide.as_strided((5, 4, 32), (64, 32, 1))):
        with pytest.raises(ValueError, match="overlap"):
            token_stride("out", x.shape, x.stride())
    codes = torch.zeros((1, 1, 16, 32), dtype=torch.uint8).expand(3, 1, 16, 32)
    with pytest.raises(ValueError, match="overlap"):
        bk.Cache(codes, codes, torch.zeros(3, 1), torch.zeros(3, 1))


def test_more_rows_than_are_numbered_are_refused(bk):
    most = 1 << 30
    assert attend(bk, batch=batch_struct(bk, tokens=most + 1, d_starts=FAKE)) == bk.ERR_INVALID_ARGUMENT
    assert attend(bk, batch=batch_struct(bk, tokens=most + 1, requests=most + 1)) == bk.ERR_INVALID_ARGUMENT
    assert bk.lib().bitsknn_cache_append(cache_struct(bk), FAKE, FAKE, bk.F16, 0, 0, FAKE, most + 1,
                                         None) == bk.ERR_INVALID_ARGUMENT
    assert "token count" in bk.last_error()
    p = [ctypes.c_void_p(FAKE * (i + 1)) for i in range(8)]
    assert bk.lib().bitsknn_cache_plan(p[0], p[1], most + 1, 16, p[2], 5, p[3], 4, 4, p[4], p[5], p[6], 8, p[7],
                                       None) == bk.ERR_INVALID_ARGUMENT


def test_strides_of_dimensions_of_one_entry_do_not_matter(bk):
    """Views of the same memory as (pages, 1, rows, dim) differ in the stride of the head; both fit (and fail for their device)."""
    import torch
    flat = torch.zeros((3, 16, 1, 32), dtype=torch.uint8)
    views = (flat.transpose(1, 2), flat.view(3, 1, 16, 32))
    assert views[0].stride() != views[1].stride()
    scales = torch.zeros(3, 1)
    for keys in views:
        for values in views:
            with pytest.raises(ValueError, match="CUDA tensor"):
                bk.Cache(keys, values, scales, scales)
    one = torch.zeros((1, 2, 16, 32), dtype=torch.uint8)           # one page: the distance to the next does not matter
    other = torch.zeros((3, 2, 16, 32), dtype=torch.uint8)[::2][:1]
    assert one.stride() != other.stride()
    with pytest.raises(ValueError, match="CUDA tensor"):
        bk.Cache(one, other, torch.zeros(1, 2), torch.zeros(1, 2))
    two = torch.zeros((3, 16, 2, 32), dtype=torch.uint8).transpose(1, 2)
    with pytest.raises(ValueError, match="contiguous"):
        bk.Cache(two, two, torch.zeros(3, 2), torch.zeros(3, 2))
    wide = torch.zeros((3, 1, 32, 32), dtype=torch.uint8)[:, :, :16]
    with pytest.raises(ValueError, match="equally far apart"):
        bk.Cache(wide, views[1], scales, scales)


MIB = 1 << 20


def test_outputs_that_lie_where_the_call_reads_are_refused(bk):
    """3 tokens x 4 heads x 64 halves: rows of 512 bytes; 12 lengths of output per row."""
    far = dict(queries=64 * MIB, out=65 * MIB, lse=66 * MIB, workspace=4096 * MIB)

    def refused(batch=None, **over):
        status = attend(bk, batch=batch, **{**far, **over})
        return status == bk.ERR_INVALID_ARGUMENT and "overlaps" in bk.last_error()

    q = far["queries"]
    assert refused(out=q) and refused(out=q + 2) and refused(out=q + 1534) and refused(out=q - 1534)
    assert refused(lse=q) and refused(lse=q + 1532) and refused(lse=q - 44)
    assert refused(lse=far["out"]) and refused(workspace=q) and refused(workspace=far["out"] - 256)
    assert refused(stride=512, out_stride=512, out=q + 768)            # turns in wider rows, by half a row only
    assert refused(stride=512, out=q + 1024)                           # the second row of the queries
    lib, cache, batch = bk.lib(), cache_struct(bk), batch_struct(bk)
    assert lib.bitsknn_cache_distance(cache, batch, q, bk.F16, 0, 4, q + 1024, 64, 64, None) == bk.ERR_INVALID_ARGUMENT
    assert "d_dist overlaps d_queries" in bk.last_error()
    assert lib.bitsknn_cache_attend_selected(cache, batch, q, bk.F16, 0, 4, far["out"] + 512, 8, 8, 0.1, far["out"], 0, None,
                                             far["workspace"], 1 << 40, None) == bk.ERR_INVALID_ARGUMENT
    assert "d_out overlaps d_idx" in bk.last_error()


def test_outputs_of_a_plan_that_lie_on_other_arrays_are_refused(bk):
    names = ("lengths", "new", "free", "table", "starts", "out", "slots", "counts")
    at = {name: MIB * (i + 1) for i, name in enumerate(names)}

    def refused(**over):
        p = {**at, **over}
        status = bk.lib().bitsknn_cache_plan(p["lengths"], p["new"], 3, 16, p["free"], 5, p["table"], 6, 4, p["starts"],
                                             p["out"], p["slots"], 8, p["counts"], None)
        return status == bk.ERR_INVALID_ARGUMENT and "overlaps" in bk.last_error()

    assert refused(out=at["lengths"]) and refused(out=at["lengths"] + 8) and refused(out=at["new"])
    assert refused(starts=at["lengths"]) and refused(starts=at["new"] + 4) and refused(starts=at["free"] + 16)
    assert refused(counts=at["free"]) and refused(slots=at["lengths"] - 56) and refused(slots=at["starts"])
    assert refused(counts=at["table"] + 24 * 2 + 12) and refused(lengths=at["table"])
