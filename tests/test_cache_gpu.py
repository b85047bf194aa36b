"""The paged 8-bit cache operators against plain implementations in 64 bits.

Tolerances.  u = 2^-24 is the rounding unit of FP32.  A product of a code (4 significant bits) and a query half
(at most 11) is exact in FP32; sums of `dim` of them are off by at most dim * 2u * sum |q k| whatever the order, also
with sums that truncate.  Scales are powers of two here unless said otherwise, so they add nothing.
  distance:  dim * 2u * sum |q k|, plus the rounding of queries 2^-28 below their vector's largest entry to halves of
             2^-24 spacing after scaling to 2^14: at most 2^-39 * max |q| * sum |k|;
  logits:    the same times the scale, D; a weight is then off by the factor e^D - 1 <= 2 D, by 2^-20 from the
             exponential and the rounding of its argument, whose size is below 2^6 here (2^6 * u * ln 2 < 2^-18), and by
             2^-11 from its rounding to a half (half a step); sums of n terms by n * 2u (relative to the sums of the
             absolute values).  Numerator and denominator: |error| <= (2^-11 + 2 * (2 D + 2^-17 + n * 2u)) * sum p |v| / sum p,
             and the rounding of the output, half a step of its type;
  lse:       D + 2^-17 + n * 2u, and 2^-22 of its own size.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


# ---- plain implementations ---------------------------------------------------------------------------------
def decode_table():
    out = np.empty(256)
    for c in range(256):
        e, f = (c >> 3) & 15, c & 7
        size = math.ldexp(f, -9) if e == 0 else math.ldexp(8 + f, e - 10)
        out[c] = math.nan if e == 15 and f == 7 else size
        if c & 128:
            out[c] = -out[c]
    return out


DECODE = decode_table()


def round_e4m3(x):
    """Codes of the nearest e4m3 numbers, ties to even, saturating; NaN -> 0x7f."""
    size = np.minimum(np.abs(np.asarray(x, np.float64)), 448.0)
    quantum = np.ldexp(1.0, np.maximum(np.frexp(np.maximum(np.nan_to_num(size), 2.0 ** -80))[1] - 1, -6) - 3)
    steps = np.nan_to_num(np.rint(size / quantum))                  # 0 ... 16, in units of the quantum
    exponent = np.rint(np.log2(quantum)).astype(int) + 3           # -6 and up
    code = np.where(exponent == -6, steps, (exponent + 6) * 8 + steps).astype(int)
    code = np.where(np.isnan(x), 0x7f, np.minimum(code, 0x7e) | np.where(np.signbit(x), 128, 0))
    return code.astype(np.uint8)


def scale_of(amax):
    e = -60
    while e < 60 and amax > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def plain_append(codes, scales, new, slots, page_rows):
    """One token after the other, in runs of ascending rows of a page; codes (pages, heads, rows, dim) uint8."""
    i = 0
    while i < len(slots):
        s = int(slots[i])
        if s < 0 or s // page_rows >= codes.shape[0]:
            i += 1
            continue
        j = i + 1
        while j < len(slots) and slots[j] // page_rows == s // page_rows and slots[j] > slots[j - 1]:
            j += 1
        page, rows = s // page_rows, [int(x) % page_rows for x in slots[i:j]]
        for h in range(codes.shape[1]):
            x = new[i:j, h].astype(np.float64)
            finite = np.abs(x[np.isfinite(x)])
            fresh = scale_of(finite.max() if finite.size else 0.0)
            if rows[0] > 0:
                fresh = max(fresh, float(scales[page, h]))
                if fresh > scales[page, h]:
                    old = DECODE[codes[page, h, :rows[0]]]
                    codes[page, h, :rows[0]] = round_e4m3(old * (float(scales[page, h]) / fresh))
            scales[page, h] = fresh
            codes[page, h, rows] = round_e4m3(x / fresh)
        i = j


class Plain:
    """A random cache and batch on the host in 64 bits, and the same on the device."""

    def __init__(self, bk, lengths, news, heads, group, dim, page_rows, dtype, seed, spread=0.5, page_pad=0):
        rng = np.random.default_rng(seed)
        self.bk, self.heads, self.group, self.dim, self.rows = bk, heads, group, dim, page_rows
        self.lengths, self.news = list(lengths), list(news)
        need = [-(-n // page_rows) for n in lengths]
        pages = sum(need) + 3
        order = rng.permutation(pages)
        self.table = np.full((len(lengths), max(need + [1]) + 1), -1, np.int32)
        at = 0
        for r, n in enumerate(need):
            self.table[r, :n] = order[at:at + n]
            at += n
        shape = (pages, heads, page_rows, dim)
        # rows nobody may look at (behind a request's end, pages of no request) hold NaN codes
        self.codes = {w: np.full(shape, 0x7f, np.uint8) for w in "kv"}
        self.scales = {w: np.full(shape[:2], 2.0 ** 30, np.float32) for w in "kv"}
        for r, n in enumerate(lengths):
            for p in range(need[r]):
                used = min(page_rows, n - p * page_rows)
                for w in "kv":
                    x = rng.standard_normal((heads, used, dim)) * np.exp(spread * rng.standard_normal((heads, used, 1)))
                    page = self.table[r, p]
                    for h in range(heads):
                        s = scale_of(np.abs(x[h]).max())
                        self.scales[w][page, h] = s
                        self.codes[w][page, h, :used] = round_e4m3(x[h] / s)
        self.tokens = sum(news)
        self.dtype = dtype
        q = rng.standard_normal((self.tokens, heads * group, dim))
        self.queries = torch.from_numpy(q).to(dtype)
        self.page_pad = page_pad

    def value(self, w, r, h, j):
        page = self.table[r, j // self.rows]
        return DECODE[self.codes[w][page, h, j % self.rows]] * float(self.scales[w][page, h])

    def matrix(self, w, r, h, n):
        pages = self.table[r, :-(-n // self.rows)]
        there = (pages >= 0) & (pages < len(self.codes[w]))
        safe = np.where(there, pages, 0)
        x = DECODE[self.codes[w][safe, h]] * self.scales[w][safe, h].astype(np.float64)[:, None, None]
        x[~there] = np.nan
        return x.reshape(-1, self.dim)[:n], np.repeat(there, self.rows)[:n]

    def token_rows(self):
        """(packed token, request, visible positions)"""
        at = 0
        limit = self.table.shape[1] * self.rows
        for r, (n, m) in enumerate(zip(self.lengths, self.news)):
            for i in range(m):
                yield at + i, r, min(max(n - m + i + 1, 0), limit)
            at += m

    def upload(self):
        bk, shape = self.bk, self.codes["k"].shape
        parts = {}
        for w in "kv":
            flat = torch.zeros((shape[0], int(np.prod(shape[1:])) + self.page_pad), dtype=torch.uint8, device="cuda")
            flat.fill_(0x7f)
            flat[:, :int(np.prod(shape[1:]))] = torch.from_numpy(self.codes[w].reshape(shape[0], -1)).cuda()
            stride = (flat.stride(0), shape[2] * shape[3], shape[3], 1)
            parts[w] = flat.as_strided(shape, stride)
        self.cache = bk.Cache(parts["k"], parts["v"], torch.from_numpy(self.scales["k"]).cuda(),
                              torch.from_numpy(self.scales["v"]).cuda())
        self.d_table = torch.from_numpy(self.table).cuda()
        self.d_lengths = torch.tensor(self.lengths, dtype=torch.int32, device="cuda")
        starts = np.concatenate([[0], np.cumsum(self.news)])
        single = all(m == 1 for m in self.news)
        self.d_starts = None if single else torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.d_queries = self.queries.cuda()
        return self

    def plain_distance(self, n):
        want = np.full((self.tokens * self.heads, n), np.inf)
        tol = np.zeros_like(want)
        q = self.queries.double().numpy()
        for t, r, vis in self.token_rows():
            vis = min(vis, n)
            for h in range(self.heads):
                k, there = self.matrix("k", r, h, vis)
                qs = q[t, h * self.group:(h + 1) * self.group]
                s = np.nan_to_num(k) @ qs.T
                row = t * self.heads + h
                want[row, :vis] = np.where(there, -s.max(axis=1) if vis else 0, np.inf)
                size = (np.abs(np.nan_to_num(k)) @ np.abs(qs).T).max(axis=1) if vis else 0
                tol[row, :vis] = self.dim * 2 * U * size + 2.0 ** -39 * np.abs(qs).max() * np.abs(np.nan_to_num(k)).sum(axis=1)
        return want, tol

    def plain_attend(self, scale, lists=None):
        out = np.zeros((self.tokens, self.heads * self.group, self.dim))
        lse = np.full(out.shape[:2], -np.inf)
        tol, lse_tol = np.zeros_like(out), np.zeros_like(lse)
        q = self.queries.double().numpy()
        for t, r, vis in self.token_rows():
            for h in range(self.heads):
                k, there = self.matrix("k", r, h, vis)
                v, _ = self.matrix("v", r, h, vis)
                use = np.flatnonzero(there)
                if lists is not None:
                    use = np.array([j for j in lists[t * self.heads + h] if 0 <= j < vis and there[j]], dtype=int)
                if len(use) == 0:
                    continue
                k, v = k[use], v[use]
                for g in range(h * self.group, (h + 1) * self.group):
                    s = scale * (k @ q[t, g])
                    d = abs(scale) * self.dim * 2 * U * (np.abs(k) @ np.abs(q[t, g])).max()
                    p = np.exp(s - s.max())
                    n = len(use)
                    out[t, g] = (p @ v) / p.sum()
                    lse[t, g] = s.max() + np.log(p.sum())
                    near = 2 * (2 * d + 2.0 ** -17 + n * 2 * U)
                    tol[t, g] = (2.0 ** -11 + near) * (p @ np.abs(v)) / p.sum()
                    lse_tol[t, g] = d + 2.0 ** -17 + n * 2 * U + 2.0 ** -22 * abs(lse[t, g])
        tol += HALF_STEP[self.dtype] * (np.abs(out) + tol) + 2.0 ** -25
        return out, lse, tol, lse_tol


def check(got, want, tol, what):
    got = got.double().cpu().numpy().reshape(want.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN in different places"
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf]), f"{what}: infinities differ"
    fine = ~inf & ~np.isnan(want)
    off = np.abs(got[fine] - want[fine]) - tol[fine]
    assert off.size == 0 or off.max() <= 0, f"{what}: beyond the tolerance by {off.max():.3g}"


SHAPES = [
    # lengths, new tokens, heads, group, dim, page_rows, dtype
    ([1], [1], 1, 1, 32, 16, torch.float16),
    ([17, 0, 64, 33], [1, 1, 1, 1], 2, 4, 64, 16, torch.bfloat16),
    ([130, 5, 1], [1, 1, 1], 3, 7, 128, 64, torch.bfloat16),
    ([100, 61], [1, 1], 1, 16, 96, 32, torch.float16),
    ([70, 258], [1, 1], 2, 2, 192, 128, torch.bfloat16),
    ([300], [1], 1, 8, 256, 256, torch.float16),
    ([40, 80], [1, 1], 1, 33, 64, 16, torch.bfloat16),              # more query heads than a block has columns
    ([50, 7, 0, 129], [5, 7, 0, 3], 2, 4, 128, 16, torch.bfloat16),  # several tokens, one request without
    ([200, 90], [37, 90], 1, 5, 64, 32, torch.float16),
    ([66, 3], [20, 5], 2, 3, 256, 64, torch.bfloat16),              # lengths below the new tokens: rows that see nothing
    ([97], [33], 1, 12, 32, 16, torch.float16),
    ([300, 20, 171], [150, 1, 171], 2, 4, 128, 64, torch.float16),
    ([260], [200], 2, 3, 64, 16, torch.bfloat16),
    ([140, 33], [70, 33], 1, 9, 192, 32, torch.float16),
]


def shapes(f):
    return pytest.mark.parametrize("lengths, news, heads, group, dim, page_rows, dtype", SHAPES)(f)


# ---- plan -------------------------------------------------------------------------------------------------
def plain_plan(lengths, new, free, table, page_rows, max_tokens):
    table = table.copy()
    starts, slots, taken, unplaced = [0], [], 0, 0
    for r, (n, m) in enumerate(zip(lengths, new)):
        n, m = max(n, 0), max(m, 0)
        starts.append(starts[-1] + m)
        have, need = -(-n // page_rows), -(-(n + m) // page_rows)
        for c in range(have, need):
            if c < table.shape[1]:
                table[r, c] = free[taken + c - have] if taken + c - have < len(free) else -1
        for pos in range(n, n + m):
            c = pos // page_rows
            page = table[r, c] if c < table.shape[1] else -1
            slots.append(int(page) * page_rows + pos % page_rows if page >= 0 else -1)
            unplaced += c >= have and (c >= table.shape[1] or taken + c - have >= len(free))
            unplaced += c < have and c >= table.shape[1]
        taken += need - have
    total = starts[-1]
    slots = (slots + [-1] * max_tokens)[:max_tokens]
    return (np.array(starts), np.array([max(n, 0) + max(m, 0) for n, m in zip(lengths, new)]), np.array(slots, np.int64),
            np.array([total, taken, unplaced]), table)


@pytest.mark.parametrize("requests, ctx, new, page_rows, free, width, slack", [
    (1, 0, 1, 16, 100, 4, 0),
    (3, 40, 1, 16, 100, 8, 2),
    (7, 100, 60, 32, 1000, 12, 5),
    (600, 300, 9, 16, 10000, 40, 700),
    (2048, 50, 3, 64, 5000, 4, 0),       # exactly one pass over the requests
    (2049, 50, 3, 64, 5000, 4, 1),       # one request in the second pass
    (5000, 20, 2, 128, 9000, 3, 100),
    (50, 100, 40, 16, 60, 12, 0),        # the free list runs out
    (50, 100, 40, 16, 0, 12, 0),         # there is none
    (50, 100, 40, 16, 900, 6, 0),        # table rows run out
    (40, 50, 30, 16, 900, 12, -200),     # fewer slots than tokens
    (3, 0, 0, 16, 5, 2, 4),              # nothing new
    (2, 100, 20000, 256, 900, 100, 3),
])
def test_plan(bk, cuda, requests, ctx, new, page_rows, free, width, slack):
    rng = np.random.default_rng(requests * 31 + new)
    lengths = rng.integers(0, ctx + 1, requests).astype(np.int32)
    added = rng.integers(-1 if new > 3 else 0, new + 1, requests).astype(np.int32)
    pool = rng.permutation(free + requests * width).astype(np.int32)
    table = np.full((requests, width), -7, np.int32)
    at = 0
    for r in range(requests):
        have = min(-(-int(lengths[r]) // page_rows), width)
        table[r, :have] = pool[at:at + have]
        at += have
    free_pages = pool[at:at + free].copy()
    tokens = int(np.maximum(added, 0).sum())
    max_tokens = max(tokens + slack, 0)
    want = plain_plan(lengths, added, free_pages, table, page_rows, max_tokens)
    wide = torch.full((requests, width + 3), -9, dtype=torch.int32, device="cuda")
    d_table = wide[:, :width]
    d_table.copy_(torch.from_numpy(table))
    got = bk.cache_plan(torch.from_numpy(lengths).cuda(), torch.from_numpy(added).cuda(),
                        torch.from_numpy(free_pages).cuda(), d_table, page_rows, max_tokens)
    for name, g, w in zip(("starts", "lengths", "slots", "counts"), got, want):
        assert np.array_equal(g.cpu().numpy(), w), name
    assert np.array_equal(d_table.cpu().numpy(), want[4])
    assert bool((wide[:, width:] == -9).all())


def test_plan_without_requests(bk, cuda):
    empty = torch.empty(0, dtype=torch.int32, device="cuda")
    starts, lengths, slots, counts = bk.cache_plan(empty, empty, empty, torch.empty((0, 2), dtype=torch.int32, device="cuda"),
                                                   16, 5)
    assert starts.tolist() == [0] and slots.tolist() == [-1] * 5 and counts.tolist() == [0, 0, 0]


# ---- append -----------------------------------------------------------------------------------------------
def append_both(bk, codes, scales, news, slots, dtype, page_rows, strided=False):
    """Runs both; returns nothing, asserts equality bit for bit."""
    dev = {w: torch.from_numpy(codes[w].copy()).cuda() for w in "kv"}
    dsc = {w: torch.from_numpy(scales[w].copy()).cuda() for w in "kv"}
    tensors = [torch.from_numpy(news[w]).to(dtype) for w in "kv"]
    dn = []
    for t in tensors:
        if strided:   # rows of a wider array, as keys and values of a joint projection are
            wide = torch.zeros((t.shape[0], t.shape[1] + 2, t.shape[2]), dtype=dtype, device="cuda")
            wide[:, 1:-1] = t.cuda()
            dn.append(wide[:, 1:-1])
        else:
            dn.append(t.cuda())
    cache = bk.Cache(dev["k"], dev["v"], dsc["k"], dsc["v"])
    bk.cache_append(cache, dn[0], dn[1], torch.tensor(slots, dtype=torch.int64, device="cuda"))
    for w, t in zip("kv", tensors):
        c, s = codes[w].copy(), scales[w].copy()
        plain_append(c, s, t.double().numpy(), np.asarray(slots), page_rows)
        assert np.array_equal(dsc[w].cpu().numpy(), s), f"scales of {w}"
        assert np.array_equal(dev[w].cpu().numpy(), c), f"codes of {w}"


def random_cache(rng, pages, heads, rows, dim):
    codes = {w: rng.integers(0, 256, (pages, heads, rows, dim)).astype(np.uint8) for w in "kv"}
    for w in "kv":
        codes[w][(codes[w] & 0x7f) == 0x7f] = 0x7f      # NaN has one code: its sign does not survive a re-rounding
    scales = {w: (2.0 ** rng.integers(-8, 3, (pages, heads))).astype(np.float32) for w in "kv"}
    return codes, scales


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads, dim, page_rows, runs", [
    (1, 32, 16, [(3, 0, 1)]),
    (2, 64, 16, [(0, 5, 4), (2, 0, 16), (5, 15, 1), (1, 1, 15)]),        # (page, first row, rows)
    (3, 128, 32, [(4, 0, 32), (0, 31, 1), (1, 3, 20)]),
    (2, 96, 64, [(1, 0, 64), (2, 0, 64), (3, 0, 11), (0, 60, 4)]),
    (1, 192, 128, [(0, 0, 128), (1, 7, 121)]),
    (1, 256, 256, [(0, 0, 256), (2, 255, 1), (1, 100, 100)]),
])
def test_append(bk, cuda, dtype, heads, dim, page_rows, runs):
    rng = np.random.default_rng(dim + heads)
    codes, scales = random_cache(rng, 7, heads, page_rows, dim)
    slots = [p * page_rows + f + i for p, f, n in runs for i in range(n)]
    news = {w: rng.standard_normal((len(slots), heads, dim)) * np.exp(2 * rng.standard_normal((len(slots), heads, 1)))
            for w in "kv"}
    append_both(bk, codes, scales, news, slots, dtype, page_rows)
    append_both(bk, codes, scales, news, slots, dtype, page_rows, strided=True)


def test_append_skips_slots_outside_the_cache(bk, cuda):
    rng = np.random.default_rng(5)
    codes, scales = random_cache(rng, 4, 2, 16, 64)
    slots = [-1, 3, 4, -1, 5, 4 * 16, 1 << 40, 17, -5, 2 * 16, 2 * 16 + 1]
    news = {w: rng.standard_normal((len(slots), 2, 64)) * 3 for w in "kv"}
    append_both(bk, codes, scales, news, slots, torch.float32, 16)


def test_append_rows_that_do_not_ascend(bk, cuda):
    rng = np.random.default_rng(6)
    codes, scales = random_cache(rng, 3, 1, 16, 32)
    # the same row twice, a step back, a page begun again: like appends one after the other
    slots = [20, 21, 21, 19, 22, 16, 17, 40, 40, 40, 33]
    news = {w: rng.standard_normal((len(slots), 1, 32)) * np.exp(2 * rng.standard_normal((len(slots), 1, 1))) for w in "kv"}
    append_both(bk, codes, scales, news, slots, torch.float32, 16)


def test_append_many_windows(bk, cuda):
    """More tokens than blocks: windows hold many runs, pages reach across their borders."""
    rng = np.random.default_rng(7)
    pages, heads, rows, dim = 700, 1, 16, 32
    codes, scales = random_cache(rng, pages, heads, rows, dim)
    slots = []
    for p in rng.permutation(pages):
        first = int(rng.integers(0, rows))
        slots += [int(p) * rows + i for i in range(first, first + int(rng.integers(1, rows - first + 1)))]
        slots += [-1] * int(rng.integers(0, 3))
    slots += [slots[-4] if slots[-4] >= 0 else 0] * 40             # one row again and again, over several windows
    news = {w: rng.standard_normal((len(slots), heads, dim)) for w in "kv"}
    append_both(bk, codes, scales, news, slots, torch.bfloat16, rows)


def test_append_special_numbers(bk, cuda):
    rng = np.random.default_rng(8)
    codes, scales = random_cache(rng, 6, 2, 16, 64)
    slots = [0, 1, 16, 17, 32, 33, 48, 49, 64, 65, 80]
    news = {w: rng.standard_normal((len(slots), 2, 64)) for w in "kv"}
    for w in "kv":
        x = news[w]
        x[0, 0, 3], x[1, 1, 5], x[1, 0, 7] = np.nan, np.inf, -np.inf
        x[2:4] = 0.0
        x[2, 0, 0] = -0.0
        x[4:6] = np.inf
        x[6:8] *= 1e38                                              # beyond 448 * 2^60: saturates
        x[8:10] *= 1e-30                                            # below 2^-60
        x[10] = 448.0                                               # exactly the largest number
        x[10, 1] = 464.0
    append_both(bk, codes, scales, news, slots, torch.float32, 16)
    append_both(bk, codes, scales, news, slots, torch.bfloat16, 16)


# ---- distance ---------------------------------------------------------------------------------------------
@shapes
def test_distance(bk, cuda, lengths, news, heads, group, dim, page_rows, dtype):
    p = Plain(bk, lengths, news, heads, group, dim, page_rows, dtype, seed=dim + group).upload()
    for n in sorted({max(lengths), max(1, max(lengths) // 2), max(lengths) + 37}):
        want, tol = p.plain_distance(n)
        wide = torch.full((p.tokens * heads + 2, n + 3), -5.0, device="cuda")
        got = bk.cache_distance(p.cache, p.d_queries, p.d_lengths, p.d_table, n, starts=p.d_starts, out=wide)
        check(got[:p.tokens * heads, :n], want, tol, f"n={n}")
        assert bool((wide[:, n:] == -5).all()) and bool((wide[p.tokens * heads:] == -5).all())


def test_distance_feeds_the_selection(bk, cuda):
    p = Plain(bk, [700, 30], [1, 1], 2, 4, 128, 16, torch.bfloat16, seed=3).upload()
    dist = bk.cache_distance(p.cache, p.d_queries, p.d_lengths, p.d_table, 704)
    got_d, got_i = bk.select(dist, 64)
    order = torch.argsort(dist, dim=1, stable=True)[:, :64]
    assert torch.equal(got_i.long(), order) and torch.equal(got_d, dist.gather(1, order))


# ---- attention ----------------------------------------------------------------------------------------------
@shapes
def test_attend(bk, cuda, lengths, news, heads, group, dim, page_rows, dtype):
    p = Plain(bk, lengths, news, heads, group, dim, page_rows, dtype, seed=dim * group).upload()
    scale = 1 / math.sqrt(dim)
    want, lse, tol, lse_tol = p.plain_attend(scale)
    out, got_lse = bk.cache_attend(p.cache, p.d_queries, p.d_lengths, p.d_table, scale, starts=p.d_starts)
    check(out, want, tol, "out")
    check(got_lse, lse, lse_tol, "lse")
    again, _ = bk.cache_attend(p.cache, p.d_queries, p.d_lengths, p.d_table, scale, starts=p.d_starts)
    assert torch.equal(out, again)


@pytest.mark.parametrize("lengths, news, heads, group, dim, page_rows", [
    ([20011], [1], 1, 8, 128, 64),              # one long request over many blocks
    ([9000, 1, 40, 3000], [1, 1, 1, 1], 2, 4, 64, 16),
    ([3000], [64], 1, 4, 128, 32),
    ([2500], [3], 1, 2, 256, 128),
    ([37] * 300, [1] * 300, 2, 3, 64, 16),      # more requests than threads
    ([5 + r % 70 for r in range(150)], [r % 4 for r in range(150)], 1, 4, 128, 16),
])
def test_attend_over_many_blocks(bk, cuda, lengths, news, heads, group, dim, page_rows):
    p = Plain(bk, lengths, news, heads, group, dim, page_rows, torch.float16, seed=len(lengths)).upload()
    want, lse, tol, lse_tol = p.plain_attend(0.2)
    out, got_lse = bk.cache_attend(p.cache, p.d_queries, p.d_lengths, p.d_table, 0.2, starts=p.d_starts)
    check(out, want, tol, "out")
    check(got_lse, lse, lse_tol, "lse")


def test_attend_strides_and_rows_behind_the_last_request(bk, cuda):
    p = Plain(bk, [50, 33], [4, 2], 2, 4, 64, 16, torch.bfloat16, seed=1, page_pad=48).upload()
    want, _, tol, _ = p.plain_attend(0.1)
    tokens, qh = 6, 8
    queries = torch.full((tokens + 3, qh + 2, 64), math.nan, dtype=torch.bfloat16, device="cuda")
    queries[:tokens, :qh] = p.d_queries
    out = torch.full((tokens + 3, qh + 1, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((tokens + 3, qh), 7.0, device="cuda")
    bk.cache_attend(p.cache, queries[:, :qh], p.d_lengths, p.d_table, 0.1, starts=p.d_starts, out=out[:, :qh], lse=lse)
    check(out[:tokens, :qh], want, tol, "out")
    assert bool((out[tokens:] == 7).all()) and bool((out[:, qh:] == 7).all()) and bool((lse[tokens:] == 7).all())
    dist = torch.full(((tokens + 3) * 2, 64), 7.0, device="cuda")
    bk.cache_distance(p.cache, queries[:, :qh], p.d_lengths, p.d_table, 64, starts=p.d_starts, out=dist)
    check(dist[:tokens * 2], *p.plain_distance(64), "distance")
    assert bool((dist[tokens * 2:] == 7).all())


def test_attend_absent_pages(bk, cuda):
    p = Plain(bk, [100, 40], [1, 3], 1, 4, 64, 16, torch.float16, seed=2)
    p.table[0, 2], p.table[0, 4], p.table[1, :3] = -1, 10 ** 6, -3
    p.upload()
    want, lse, tol, lse_tol = p.plain_attend(0.1)
    out, got_lse = bk.cache_attend(p.cache, p.d_queries, p.d_lengths, p.d_table, 0.1, starts=p.d_starts)
    check(out, want, tol, "out")
    check(got_lse, lse, lse_tol, "lse")
    check(bk.cache_distance(p.cache, p.d_queries, p.d_lengths, p.d_table, 100, starts=p.d_starts), *p.plain_distance(100),
          "distance")


def test_lengths_beyond_the_table_are_cut(bk, cuda):
    p = Plain(bk, [48], [1], 1, 2, 64, 16, torch.float16, seed=4)
    p.table = np.ascontiguousarray(p.table[:, :2])
    p.upload()
    want, _, tol, _ = p.plain_attend(0.1)
    check(bk.cache_attend(p.cache, p.d_queries, p.d_lengths, p.d_table, 0.1)[0], want, tol, "out")


@pytest.mark.parametrize("dim, group, count", [(64, 4, 30), (128, 4, 200), (256, 1, 9), (128, 1, 130)])
def test_nan_is_seen_only_where_it_is_visible(bk, cuda, dim, group, count):
    p = Plain(bk, [count + 40], [count], 1, group, dim, 32, torch.bfloat16, seed=dim)
    # a NaN in a key spoils the whole row, one in a value its own dimension, for tokens that see it
    for w, pos, d in (("k", count + 20, 3), ("v", 45, 5), ("v", count + 30, 6)):
        p.codes[w][p.table[0, pos // 32], 0, pos % 32, d] = 0xff
    p.upload()
    with np.errstate(invalid="ignore"):
        want, lse, tol, lse_tol = p.plain_attend(0.1)
    out, got_lse = bk.cache_attend(p.cache, p.d_queries, p.d_lengths, p.d_table, 0.1, starts=p.d_starts)
    assert np.isnan(want).any()
    check(out, want, np.nan_to_num(tol), "out")
    check(got_lse, lse, np.nan_to_num(lse_tol), "lse")


def test_scales_far_apart(bk, cuda):
    """Value scales 2^80 apart within a row, key scales that make the softmax sharp, scales that are no powers of two."""
    p = Plain(bk, [400], [2], 1, 4, 64, 16, torch.float16, seed=9)
    rng = np.random.default_rng(1)
    pages = p.table[0, :25]
    p.scales["v"][pages, 0] = (2.0 ** rng.integers(-40, 40, 25)).astype(np.float32)
    p.scales["k"][pages, 0] *= 1.37
    p.upload()
    want, lse, tol, lse_tol = p.plain_attend(0.5)
    tol = tol * 1.01 + 4 * U * np.abs(want)                         # 1.37 ks: one more rounding of the logit's factor
    out, got_lse = bk.cache_attend(p.cache, p.d_queries, p.d_lengths, p.d_table, 0.5, starts=p.d_starts)
    fits = np.abs(want) < 60000                                     # larger ones are infinite as halves
    got = out.double().cpu().numpy()
    assert (np.abs(got - want)[fits] <= tol[fits]).all()
    assert np.isinf(got[np.abs(want) > 66000]).all()
    check(got_lse, lse, lse_tol * 1.01 + 2.0 ** -20, "lse")


def test_queries_of_extreme_sizes(bk, cuda):
    p = Plain(bk, [60, 60, 60], [1, 1, 1], 1, 2, 64, 16, torch.bfloat16, seed=10)
    p.queries[0] *= 1e-30
    p.queries[1] *= 2.0 ** 20                                       # a softmax of one entry
    p.queries[2] = 0.0
    p.upload()
    want, _, tol, _ = p.plain_attend(0.125)
    out, _ = bk.cache_attend(p.cache, p.d_queries, p.d_lengths, p.d_table, 0.125)
    check(out[[0, 2]], want[[0, 2]], tol[[0, 2]], "out")
    # at 2^20 the logits' own error is large; the gap to the second best is larger still
    check(out[1:2], want[1:2], np.maximum(tol[1:2], 0) * 0 + 2.0 ** -7 * np.abs(want[1:2]) + 1e-6, "sharp")
    check(bk.cache_distance(p.cache, p.d_queries, p.d_lengths, p.d_table, 60), *p.plain_distance(60), "distance")


def test_infinite_queries_spoil_their_own_rows_only(bk, cuda):
    p = Plain(bk, [60], [4], 1, 2, 64, 16, torch.bfloat16, seed=11)
    clean, _, tol, _ = p.plain_attend(0.1)
    p.queries[1, 0, 3], p.queries[2, 1, 4] = math.inf, math.nan
    p.upload()
    out, lse = bk.cache_attend(p.cache, p.d_queries, p.d_lengths, p.d_table, 0.1, starts=p.d_starts)
    assert bool(out[1, 0].isnan().all()) and bool(out[2, 1].isnan().all()) and bool(lse[2, 1].isnan())
    for t, g in ((0, 0), (0, 1), (1, 1), (2, 0), (3, 0), (3, 1)):
        check(out[t, g], clean[t, g], tol[t, g], "other rows")


# ---- attention over lists -----------------------------------------------------------------------------------
@pytest.mark.parametrize("k", [1, 16, 65, 200])
@shapes
def test_attend_selected(bk, cuda, lengths, news, heads, group, dim, page_rows, dtype, k):
    p = Plain(bk, lengths, news, heads, group, dim, page_rows, dtype, seed=dim + k).upload()
    rng = np.random.default_rng(k)
    lists = np.full((p.tokens * heads, k), 0x7fffffff, np.int32)
    for t, r, vis in p.token_rows():
        for h in range(heads):
            pick = rng.permutation(max(lengths) + 9)[:k]            # some beyond what the token sees
            lists[t * heads + h, :len(pick)] = pick
    lists[0, 0] = -2
    if k > 2:
        lists[:, 2] = lists[:, 1]                                   # twice: counts twice
    want, lse, tol, lse_tol = p.plain_attend(0.15, lists)
    wide = torch.full((p.tokens * heads, k + 5), 0, dtype=torch.int32, device="cuda")
    wide[:, :k] = torch.from_numpy(lists)
    out, got_lse = bk.cache_attend_selected(p.cache, p.d_queries, wide[:, :k], p.d_lengths, p.d_table, 0.15,
                                            starts=p.d_starts)
    check(out, want, tol, "out")
    check(got_lse, lse, lse_tol, "lse")


def test_attend_selected_long_lists_and_empty_rows(bk, cuda):
    p = Plain(bk, [5000, 0, 100], [1, 1, 1], 2, 4, 128, 64, torch.bfloat16, seed=12).upload()
    rng = np.random.default_rng(3)
    lists = np.stack([rng.permutation(5000)[:2048] for _ in range(6)]).astype(np.int32)
    lists[1] = 0x7fffffff
    want, lse, tol, lse_tol = p.plain_attend(0.1, lists)
    out, got_lse = bk.cache_attend_selected(p.cache, p.d_queries, torch.from_numpy(lists).cuda(), p.d_lengths, p.d_table, 0.1)
    check(out, want, tol, "out")
    check(got_lse, lse, lse_tol, "lse")
    assert bool((out[0, 4:] == 0).all()) and bool((out[1] == 0).all())


# ---- together ------------------------------------------------------------------------------------------------
def decode_steps(bk, use_graph, stream=None):
    """Prompt, then three decode steps of plan -> append -> distance -> select -> attend over the list and over all."""
    rng = np.random.default_rng(21)
    heads, group, dim, rows, requests, k = 2, 4, 64, 16, 3, 32
    cache = bk.Cache.empty(40, heads, rows, dim)
    table = torch.full((requests, 12), -1, dtype=torch.int32, device="cuda")
    free = torch.from_numpy(rng.permutation(40).astype(np.int32)).cuda()
    lengths = torch.zeros(requests, dtype=torch.int32, device="cuda")
    prompt = torch.tensor([70, 0, 31], dtype=torch.int32, device="cuda")
    total = 101

    def draw(*shape):
        return torch.from_numpy(rng.standard_normal(shape)).to(torch.bfloat16).cuda()

    results = []
    starts, after, slots, counts = bk.cache_plan(lengths, prompt, free, table, rows, total + 4)
    kv = [draw(total + 4, heads, dim) for _ in range(2)]
    bk.cache_append(cache, kv[0], kv[1], slots)
    out, _ = bk.cache_attend(cache, draw(total, heads * group, dim), after, table, 0.1, starts=starts)
    results.append(out)
    lengths.copy_(after)
    free = free[int(counts[1]):].clone()
    one = torch.ones(requests, dtype=torch.int32, device="cuda")
    workspace = torch.empty(bk.cache_attend_workspace_bytes(cache, heads * group), dtype=torch.uint8, device="cuda")
    keys, values = draw(requests, heads, dim), draw(requests, heads, dim)
    queries = draw(requests, heads * group, dim)

    def step():
        _, new_lengths, new_slots, taken = bk.cache_plan(lengths, one, free, table, rows, requests)
        bk.cache_append(cache, keys, values, new_slots)
        dist = bk.cache_distance(cache, queries, new_lengths, table, 128)
        _, idx = bk.select(dist, k)
        near, _ = bk.cache_attend_selected(cache, queries, idx, new_lengths, table, 0.1, workspace=workspace)
        full, _ = bk.cache_attend(cache, queries, new_lengths, table, 0.1, workspace=workspace)
        every, _ = bk.cache_attend_selected(cache, queries, bk.select(dist, 128)[1], new_lengths, table, 0.1,
                                            workspace=workspace)
        lengths.copy_(new_lengths)
        free.copy_(torch.roll(free, -1))     # at most one page is begun in these steps' order of events
        return near, full, every, taken

    graph = None
    for i in range(3):
        for t in (keys, values, queries):
            t.copy_(draw(*t.shape))
        if use_graph and i == 1:
            graph = torch.cuda.CUDAGraph()
            state = [t.clone() for t in (lengths, free, table, cache.keys, cache.values, cache.key_scales, cache.value_scales)]
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                captured = step()
            for t, s in zip((lengths, free, table, cache.keys, cache.values, cache.key_scales, cache.value_scales), state):
                t.copy_(s)
        if graph is not None:
            graph.replay()
            got = captured
        else:
            got = step()
        results += [t.clone() for t in got]
    torch.cuda.synchronize()
    return results


def test_decode_steps_together(bk, cuda):
    eager = decode_steps(bk, False)
    for i in range(3):
        near, full, every, _ = eager[1 + 4 * i:5 + 4 * i]
        # the list of all positions gives what the dense form gives, up to the roundings of both (FP32 sums in another order,
        # 2^-11 of the weights, the output's half step)
        assert bool(((every - full).float().abs() <= 2.0 ** -6 * full.float().abs().amax(dim=2, keepdim=True)).all())
        assert not torch.equal(near, full)


def test_decode_steps_in_a_graph_and_on_another_stream(bk, cuda):
    eager = decode_steps(bk, False)
    graph = decode_steps(bk, True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = decode_steps(bk, False)
    torch.cuda.current_stream().wait_stream(side)
    for a, b, c in zip(eager, graph, other):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_python_layer_refuses(bk, cuda):
    p = Plain(bk, [20], [1], 1, 2, 64, 16, torch.bfloat16, seed=0).upload()
    with pytest.raises(ValueError, match="not fit the cache"):
        bk.cache_attend(p.cache, torch.zeros((1, 2, 32), dtype=torch.bfloat16, device="cuda"), p.d_lengths, p.d_table, 1.0)
    with pytest.raises(bk.BitsKnnError) as err:
        bk.cache_attend(p.cache, torch.zeros((1, 2, 64), device="cuda"), p.d_lengths, p.d_table, 1.0)
    assert err.value.status == bk.ERR_UNSUPPORTED_MODE
    with pytest.raises(ValueError, match="requests"):
        bk.cache_attend(p.cache, p.d_queries, p.d_lengths, p.d_table[:, :0].expand(3, 0), 1.0)
    with pytest.raises(ValueError):
        bk.cache_attend_selected(p.cache, p.d_queries, torch.zeros((5, 4), dtype=torch.int32, device="cuda"), p.d_lengths,
                                 p.d_table, 1.0)
    with pytest.raises(ValueError, match="contiguous"):
        bk.cache_append(p.cache, torch.zeros((2, 1, 128), dtype=torch.float16, device="cuda")[:, :, ::2],
                        torch.zeros((2, 1, 64), dtype=torch.float16, device="cuda"),
                        torch.zeros(2, dtype=torch.int64, device="cuda"))


# ---- many query columns: the tensor-memory kernel ------------------------------------------------------------
@pytest.mark.parametrize("lengths, news, heads, group, dim, page_rows, dtype", [
    ([64], [64], 1, 1, 128, 16, torch.bfloat16),
    ([128], [128], 1, 2, 128, 64, torch.float16),                       # two full query tiles
    ([300], [200], 1, 4, 64, 16, torch.bfloat16),
    ([517], [100], 2, 3, 32, 32, torch.float16),
    ([450], [129], 1, 2, 96, 128, torch.bfloat16),
    ([333], [70], 1, 5, 192, 16, torch.float16),
    ([290], [131], 1, 1, 256, 256, torch.bfloat16),
    ([1000, 3, 0, 260], [90, 3, 0, 200], 2, 4, 128, 32, torch.bfloat16),  # ragged: few rows and none beside many
    ([100], [150], 1, 3, 128, 16, torch.float16),                       # rows that see nothing
    ([129, 4000], [65, 64], 1, 8, 64, 16, torch.bfloat16),
    ([3000], [300], 1, 2, 128, 64, torch.float16),                      # parts of several blocks
    ([2000], [64], 1, 16, 256, 32, torch.bfloat16),
])
def test_attend_many_columns(bk, cuda, lengths, news, heads, group, dim, page_rows, dtype):
    p = Plain(bk, lengths, news, heads, group, dim, page_rows, dtype, seed=dim + heads).upload()
    scale = 1 / math.sqrt(dim)
    want, lse, tol, lse_tol = p.plain_attend(scale)
    out, got_lse = bk.cache_attend(p.cache, p.d_queries, p.d_lengths, p.d_table, scale, starts=p.d_starts)
    bk.device_status()
    check(out, want, tol, "out")
    check(got_lse, lse, lse_tol, "lse")
    again, _ = bk.cache_attend(p.cache, p.d_queries, p.d_lengths, p.d_table, scale, starts=p.d_starts)
    assert torch.equal(out, again)


def test_attend_many_columns_special(bk, cuda):
    """Absent pages, a negative scale, infinite queries, odd strides, one call after the other."""
    p = Plain(bk, [400, 90], [100, 80], 1, 4, 128, 16, torch.bfloat16, seed=31, page_pad=32)
    p.table[0, 3], p.table[0, 20], p.table[1, 0] = -1, 10 ** 7, -5
    p.upload()
    want, lse, tol, lse_tol = p.plain_attend(-0.05)
    wide = torch.full((182, 5, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    out, got_lse = bk.cache_attend(p.cache, p.d_queries, p.d_lengths, p.d_table, -0.05, starts=p.d_starts, out=wide[:180, :4])
    check(out, want, tol, "out")
    check(got_lse, lse, lse_tol, "lse")
    assert bool((wide[180:] == 7).all()) and bool((wide[:, 4] == 7).all())
    odd = torch.full((180 * 4 * 128 + 1,), 7.0, dtype=torch.bfloat16, device="cuda")[1:].view(180, 4, 128)   # 2-byte aligned
    bk.cache_attend(p.cache, p.d_queries, p.d_lengths, p.d_table, -0.05, starts=p.d_starts, out=odd)
    assert torch.equal(odd, out)
    clean = out.clone()
    p.d_queries[5, 2, 7], p.d_queries[150, 0, 0] = math.inf, math.nan
    out, _ = bk.cache_attend(p.cache, p.d_queries, p.d_lengths, p.d_table, -0.05, starts=p.d_starts)
    bad = out.isnan().all(dim=2)
    assert bad.sum() == 2 and bool(bad[5, 2]) and bool(bad[150, 0])
    assert torch.equal(out[~bad], clean[~bad])
    bk.device_status()


def test_attend_sharp_rows_move_the_reference(bk, cuda):
    """Keys that grow along the cache: the running maximum rises tile after tile, and what was summed is scaled."""
    p = Plain(bk, [1500], [64], 1, 4, 128, 64, torch.float16, seed=33, spread=0.0)
    for r, page in enumerate(p.table[0, :24]):
        p.scales["k"][page, 0] *= 2.0 ** (r / 4 // 1)
    p.upload()
    want, lse, tol, lse_tol = p.plain_attend(0.02)
    out, got_lse = bk.cache_attend(p.cache, p.d_queries, p.d_lengths, p.d_table, 0.02, starts=p.d_starts)
    check(out, want, tol, "out")
    check(got_lse, lse, lse_tol, "lse")
    one = bk.cache_attend(p.cache, p.d_queries[-1:], p.d_lengths, p.d_table, 0.02)[0]
    check(one, want[-1:], tol[-1:], "decode")


def test_many_columns_beyond_the_table_are_cut(bk, cuda):
    p = Plain(bk, [200], [70], 1, 4, 64, 32, torch.float16, seed=41)
    p.table = np.ascontiguousarray(p.table[:, :5])                  # 160 positions
    p.upload()
    want, lse, tol, lse_tol = p.plain_attend(0.1)
    out, got_lse = bk.cache_attend(p.cache, p.d_queries, p.d_lengths, p.d_table, 0.1, starts=p.d_starts)
    check(out, want, tol, "out")
    check(got_lse, lse, lse_tol, "lse")


def test_rows_behind_the_last_request_are_left_alone(bk, cuda):
    """Padded batches: packed arrays longer than the requests' tokens, in every kernel that writes rows."""
    for lengths, news, group in (([60, 40], [3, 2], 4), ([90, 300], [40, 60], 4)):
        p = Plain(bk, lengths, news, 2, group, 64, 16, torch.bfloat16, seed=42).upload()
        tokens, pad = p.tokens, 7
        lists = np.stack([np.random.default_rng(i).permutation(max(lengths))[:20] for i in range(tokens * 2)]).astype(np.int32)
        queries = torch.cat([p.d_queries, torch.full((pad, 2 * group, 64), math.nan, dtype=torch.bfloat16, device="cuda")])
        wide_lists = torch.cat([torch.from_numpy(lists).cuda(), torch.zeros((pad * 2, 20), dtype=torch.int32, device="cuda")])
        for which in ("all", "list"):
            out = torch.full(queries.shape, 7.0, dtype=torch.bfloat16, device="cuda")
            lse = torch.full(queries.shape[:2], 7.0, device="cuda")
            args = (p.d_lengths, p.d_table, 0.1)
            if which == "all":
                bk.cache_attend(p.cache, queries, *args, starts=p.d_starts, out=out, lse=lse)
                want, want_lse, tol, lse_tol = p.plain_attend(0.1)
            else:
                bk.cache_attend_selected(p.cache, queries, wide_lists, *args, starts=p.d_starts, out=out, lse=lse)
                want, want_lse, tol, lse_tol = p.plain_attend(0.1, lists)
            check(out[:tokens], want, tol, which)
            check(lse[:tokens], want_lse, lse_tol, which)
            assert bool((out[tokens:] == 7).all()) and bool((lse[tokens:] == 7).all())


def test_offsets_beyond_32_bits(bk, cuda):
    """Pages 2^31 codes apart: the last one begins behind 2^32 bytes."""
    heads, rows, dim, group = 1, 64, 64, 4
    stride = (1 << 31) + 64
    flat = {w: torch.empty(2 * stride + heads * rows * dim, dtype=torch.uint8, device="cuda") for w in "kv"}
    shape = (3, heads, rows, dim)
    views = {w: flat[w].as_strided(shape, (stride, rows * dim, dim, 1)) for w in "kv"}
    scales = {w: torch.ones((3, heads), device="cuda") for w in "kv"}
    cache = bk.Cache(views["k"], views["v"], scales["k"], scales["v"])
    order, count = [2, 0, 1], 170
    table = torch.tensor([order], dtype=torch.int32, device="cuda")
    rng = np.random.default_rng(51)
    kv = {w: torch.from_numpy(rng.standard_normal((count, heads, dim))).to(torch.float32).cuda() for w in "kv"}
    slots = torch.tensor([order[i // rows] * rows + i % rows for i in range(count)], dtype=torch.int64, device="cuda")
    bk.cache_append(cache, kv["k"], kv["v"], slots)
    # the same requests in a small cache
    small = bk.Cache.empty(3, heads, rows, dim)
    bk.cache_append(small, kv["k"], kv["v"], slots)
    for i in range(3):
        used = min(rows, count - order.index(i) * rows)
        for w, t in (("k", small.keys), ("v", small.values)):
            assert torch.equal(views[w][i, :, :used], t[i, :, :used])
    lengths = torch.tensor([count], dtype=torch.int32, device="cuda")
    for tokens in (1, 3, 90):
        q = torch.from_numpy(rng.standard_normal((tokens, group, dim))).to(torch.bfloat16).cuda()
        starts = torch.tensor([0, tokens], dtype=torch.int32, device="cuda")
        lists = torch.from_numpy(np.stack([rng.permutation(count) for _ in range(tokens)]).astype(np.int32)).cuda()
        for f in (lambda c: bk.cache_attend(c, q, lengths, table, 0.1, starts=starts),
                  lambda c: bk.cache_attend_selected(c, q, lists, lengths, table, 0.1, starts=starts),
                  lambda c: (bk.cache_distance(c, q, lengths, table, count, starts=starts),)):
            for x, y in zip(f(cache), f(small)):
                assert torch.equal(x, y)


def test_calls_on_two_streams_with_workspaces_of_their_own(bk, cuda):
    p = Plain(bk, [3000, 500], [1, 1], 2, 4, 128, 16, torch.bfloat16, seed=61).upload()
    many = Plain(bk, [400], [90], 2, 4, 128, 16, torch.bfloat16, seed=62).upload()
    want = bk.cache_attend(p.cache, p.d_queries, p.d_lengths, p.d_table, 0.1)[0]
    want_many = bk.cache_attend(many.cache, many.d_queries, many.d_lengths, many.d_table, 0.1, starts=many.d_starts)[0]
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for _ in range(20):
        for side, q, w in ((sides[0], p, want), (sides[1], many, want_many)):
            with torch.cuda.stream(side):
                results.append((bk.cache_attend(q.cache, q.d_queries, q.d_lengths, q.d_table, 0.1, starts=q.d_starts)[0], w))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in results)


def test_plan_of_lengths_near_the_end_of_int32(bk, cuda):
    """Positions that pass 2^31 have no page in any table: their tokens get no place, and nothing is read for them."""
    top = (1 << 31) - 1
    lengths, new = [top, top - 5, 30], [1, 40, 5]
    table = torch.full((3, 4), -7, dtype=torch.int32, device="cuda")
    table[2, :2] = torch.tensor([8, 9], dtype=torch.int32)
    i32 = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (lengths, new, [3, 4, 5, 6, 7])]
    starts, after, slots, counts = bk.cache_plan(i32[0], i32[1], i32[2], table, 16, 50)
    assert starts.tolist() == [0, 1, 41, 46]
    assert after.tolist() == [top, top, 35]
    # 2^31 - 1 positions fill 2^27 pages but for one row; 2^31 - 6 all but six: 34 more tokens ask for 3 pages
    want = [-1] * 41 + [9 * 16 + 14, 9 * 16 + 15, 6 * 16, 6 * 16 + 1, 6 * 16 + 2] + [-1] * 4
    assert slots.tolist() == want
    assert table.tolist() == [[-7] * 4, [-7] * 4, [8, 9, 6, -7]]
    assert counts.tolist() == [46, 4, 41]


def test_append_of_a_batch_with_long_padding(bk, cuda):
    """A page whose tokens lie thousands of skipped slots apart, and padding behind the last one."""
    heads, rows, dim = 2, 16, 64
    rng = np.random.default_rng(71)
    order = [(0, 5), (300, 6), (2900, 3), (3100, 9), (9000, 40)]      # token, slot: page 0 four times, then page 2
    tokens = 12000
    slots = torch.full((tokens,), -1, dtype=torch.int64)
    for token, slot in order:
        slots[token] = slot
    slots = slots.cuda()
    new = [torch.from_numpy(rng.standard_normal((tokens, heads, dim))).to(torch.bfloat16) for _ in range(2)]
    for x in new:
        x[2900] *= 50                                                   # the page's scale grows
    new = [x.cuda() for x in new]
    got, want = (bk.Cache.empty(3, heads, rows, dim) for _ in range(2))
    bk.cache_append(got, *new, slots)
    for token, _ in order:                                              # 5, 6 ascend but act alike one by one
        one = slice(token, token + 1)
        bk.cache_append(want, new[0][one], new[1][one], slots[one])
    assert int((want.key_scales > 0).sum()) == 4
    for name in ("key_scales", "value_scales"):
        assert torch.equal(getattr(got, name), getattr(want, name))
    for name in ("keys", "values"):
        a, b = (getattr(c, name)[0, :, [3, 9]] for c in (got, want))
        assert torch.equal(a, b)
        assert torch.equal(getattr(got, name)[2], getattr(want, name)[2])


def test_items_with_few_rows_between_items_with_many(bk, cuda):
    """Blocks that alternate between two query tiles and one, with NaN values that only later tokens see."""
    news, lengths = [], []
    for i in range(60):
        news += [50, 9, 8, 10, 9, 11, 10, 9, 8, 9]
        lengths += [60 + i % 7, 20, 9, 40, 70, 66, 12, 130, 30, 64]
    p = Plain(bk, lengths, news, 1, 4, 64, 16, torch.float16, seed=81)
    p.upload()
    # the last position's value of every third request is NaN: its last token alone sees it
    for r in range(0, len(lengths), 3):
        last = lengths[r] - 1
        p.cache.values[int(p.d_table[r, last // 16]), 0, last % 16, 5] = 0x7f
    out, _ = bk.cache_attend(p.cache, p.d_queries, p.d_lengths, p.d_table, 0.1, starts=p.d_starts)
    token = 0
    want = torch.zeros(out.shape, dtype=torch.bool)
    for r, m in enumerate(news):
        token += m
        if r % 3 == 0:
            want[token - 1, :, 5] = True
    assert torch.equal(torch.isnan(out).cpu(), want)
    for _ in range(20):
        again, _ = bk.cache_attend(p.cache, p.d_queries, p.d_lengths, p.d_table, 0.1, starts=p.d_starts)
        assert torch.equal(again.view(torch.int16), out.view(torch.int16))


@pytest.mark.parametrize("rows, dim, dtype", [(16, 128, torch.float16), (32, 128, torch.bfloat16),
                                              (64, 128, torch.float16), (16, 256, torch.float32),
                                              (16, 96, torch.bfloat16), (32, 32, torch.float32)])
def test_append_does_not_depend_on_how_tokens_are_batched(bk, cuda, rows, dim, dtype):
    """Many pages in one call, teams of warps and of blocks, against the same tokens page by page."""
    heads, pages = 3, 40
    rng = np.random.default_rng(rows + dim)
    order = rng.permutation(pages)[:30]
    slots = np.concatenate([p * rows + np.arange(rows) for p in order[:-1]] + [order[-1] * rows + np.arange(5)])
    new = [torch.from_numpy(rng.standard_normal((len(slots), heads, dim)) * np.exp(rng.standard_normal((len(slots), 1, 1))))
           .to(dtype).cuda() for _ in range(2)]
    slots = torch.from_numpy(slots).cuda()
    got, want = (bk.Cache.empty(pages, heads, rows, dim) for _ in range(2))
    bk.cache_append(got, *new, slots)
    for i in range(30):
        one = slice(i * rows, min((i + 1) * rows, len(slots)))
        bk.cache_append(want, new[0][one], new[1][one], slots[one])
    for name in ("keys", "values", "key_scales", "value_scales"):
        assert torch.equal(getattr(got, name), getattr(want, name)), name


# ---- value scales far apart ------------------------------------------------------------------------------------
# A weight is rounded to a half (2^-11 of itself) or to two BF16 numbers (less).  Where halves are subnormal they are off
# by at most 2^-25, half their spacing, with 2^7 or more for the largest p vs so far; the positions that get halves have a
# scale of at least 2^-4 of the largest one so far, so that is 2^-32 * 2^4 = 2^-28 of the largest p.  Below the smallest
# float, 2^-126, weights are zero: 2^-133 of the largest p vs.  Nothing else depends on the other positions' scales.
def plain_attend_by_dimension(p, scale, lists=None):
    """plain_attend with a tolerance that is made of each dimension's own values."""
    out, lse, _, lse_tol = p.plain_attend(scale, lists)
    tol = np.zeros_like(out)
    q = p.queries.double().numpy()
    for t, r, vis in p.token_rows():
        for h in range(p.heads):
            k, there = p.matrix("k", r, h, vis)
            v, _ = p.matrix("v", r, h, vis)
            use = np.flatnonzero(there)
            if lists is not None:
                use = np.array([j for j in lists[t * p.heads + h] if 0 <= j < vis and there[j]], dtype=int)
            if len(use) == 0:
                continue
            k, v = k[use], v[use]
            most = 448 * np.repeat(p.scales["v"][p.table[r], h], p.rows)[:vis][use].max()
            for g in range(h * p.group, (h + 1) * p.group):
                s = scale * (k @ q[t, g])
                d = abs(scale) * p.dim * 2 * U * (np.abs(k) @ np.abs(q[t, g])).max()
                w = np.exp(s - s.max())
                near = 2 * (2 * d + 2.0 ** -17 + len(use) * 2 * U)
                tol[t, g] = ((2.0 ** -11 + near) * (w @ np.abs(v)) + 2.0 ** -28 * np.abs(v).sum(axis=0)
                             + 2.0 ** -133 * len(use) * most) / w.sum()
    least = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}[p.dtype]    # half a step of the smallest numbers
    return out, lse, tol + HALF_STEP[p.dtype] * (np.abs(out) + tol) + least, lse_tol


def pages_apart(bk, lengths, news, heads, group, dim, page_rows, dtype, high, large, low, seed):
    """Pages `high` of every request hold one dimension alone, at 2^large; the scales of the others are 2^low times theirs."""
    p = Plain(bk, lengths, news, heads, group, dim, page_rows, dtype, seed)
    rng = np.random.default_rng(seed + 1)
    for r, n in enumerate(lengths):
        for c in range(-(-n // page_rows)):
            page = p.table[r, c]
            if c in high:
                used = min(page_rows, n - c * page_rows)
                p.codes["v"][page, :, :used] = 0
                p.codes["v"][page, :, :used, 3] = round_e4m3(rng.uniform(1, 2, (heads, used)))
                p.scales["v"][page] = 2.0 ** large
            else:
                p.scales["v"][page] *= 2.0 ** low
    return p.upload()


@pytest.mark.parametrize("dtype, large, low", [
    (torch.bfloat16, 26, 0), (torch.float16, 13, -15), (torch.bfloat16, 40, 0), (torch.bfloat16, 60, -30)])
@pytest.mark.parametrize("lengths, news, heads, group, dim, page_rows, high", [
    ([200], [1], 1, 4, 128, 16, {2}),                              # a cluster of blocks
    ([300, 77], [1, 1], 2, 8, 64, 32, {0, 4}),                     # first: all others lie below what was seen
    ([6000, 250], [1, 1], 1, 4, 128, 64, {5, 40}),                 # parts of several blocks
    ([120, 60], [3, 5], 1, 4, 32, 16, {1, 3}),                     # several tokens, the last ones see more
    ([150, 90], [2, 3], 1, 8, 96, 16, {2, 7}),
    ([420] * 70, [1] * 70, 8, 4, 64, 64, {1}),                     # warps with many subtiles
    ([300] * 100, [3] * 100, 4, 2, 128, 64, {0, 3}),
    ([260] * 60, [1] * 60, 8, 9, 256, 256, {0}),
    ([90], [2], 1, 16, 192, 16, {0, 3}),                           # more than one block of columns
    ([300], [1], 1, 16, 256, 32, {1}),
    ([400], [64], 1, 4, 128, 16, {3, 9}),                          # tensor memory: groups of a tile apart
    ([700, 300], [90, 120], 2, 4, 64, 64, {0, 6}),                 # whole tiles
    ([500], [150], 1, 3, 32, 128, {1}),
    ([450], [70], 1, 8, 96, 16, {0, 11, 27}),
    ([333], [70], 1, 5, 192, 16, {4}),
    ([3000], [131], 1, 2, 256, 32, {70}),                          # late, parts of several blocks
])
def test_weights_of_pages_with_small_scales(bk, cuda, lengths, news, heads, group, dim, page_rows, high, dtype, large, low):
    p = pages_apart(bk, lengths, news, heads, group, dim, page_rows, dtype, high, large, low, seed=dim + group)
    want, lse, tol, lse_tol = plain_attend_by_dimension(p, 0.1)
    calls = [p.d_starts]
    if p.d_starts is None:                                          # one token each: with starts, too
        calls.append(torch.arange(len(news) + 1, dtype=torch.int32, device="cuda"))
    for starts in calls:
        out, got_lse = bk.cache_attend(p.cache, p.d_queries, p.d_lengths, p.d_table, 0.1, starts=starts)
        check(out, want, tol, "out")
        check(got_lse, lse, lse_tol, "lse")
    bk.device_status()


@pytest.mark.parametrize("dtype, large, low", [(torch.bfloat16, 33, 0), (torch.float16, 13, -15), (torch.bfloat16, 60, -30)])
@pytest.mark.parametrize("lengths, news, heads, group, dim, page_rows, high, k", [
    ([200], [1], 1, 4, 128, 16, {2}, 64),
    ([5000, 3000], [1, 1], 2, 4, 128, 64, {5, 40}, 2000),
    ([300, 90], [2, 3], 1, 20, 64, 32, {0, 2}, 90),
    ([400], [2], 1, 9, 256, 16, {3, 9}, 200),
])
def test_weights_of_listed_positions_with_small_scales(bk, cuda, lengths, news, heads, group, dim, page_rows, high, k, dtype,
                                                       large, low):
    p = pages_apart(bk, lengths, news, heads, group, dim, page_rows, dtype, high, large, low, seed=dim + k)
    rng = np.random.default_rng(k)
    lists = np.stack([rng.permutation(max(lengths) + 5)[:k] for _ in range(p.tokens * heads)]).astype(np.int32)
    want, lse, tol, lse_tol = plain_attend_by_dimension(p, 0.1, lists)
    out, got_lse = bk.cache_attend_selected(p.cache, p.d_queries, torch.from_numpy(lists).cuda(), p.d_lengths, p.d_table, 0.1,
                                            starts=p.d_starts)
    check(out, want, tol, "out")
    check(got_lse, lse, lse_tol, "lse")


@pytest.mark.parametrize("dim, group, count", [(64, 4, 7), (128, 4, 100), (256, 1, 90)])
def test_nan_among_scales_far_apart(bk, cuda, dim, group, count):
    p = pages_apart(bk, [count + 70], [count], 1, group, dim, 16, torch.bfloat16, {1, 5}, 40, 0, seed=dim)
    for w, pos, d in (("v", 40, 5), ("v", count + 66, 6), ("k", count + 68, 1)):
        p.codes[w][p.table[0, pos // 16], 0, pos % 16, d] = 0x7f
    p.upload()
    with np.errstate(invalid="ignore"):
        want, lse, tol, lse_tol = plain_attend_by_dimension(p, 0.1)
    assert 0 < np.isnan(want[:, :, 6]).sum() < want[:, :, 6].size
    out, got_lse = bk.cache_attend(p.cache, p.d_queries, p.d_lengths, p.d_table, 0.1, starts=p.d_starts)
    check(out, want, np.nan_to_num(tol), "out")
    check(got_lse, lse, np.nan_to_num(lse_tol), "lse")


@pytest.mark.parametrize("lengths, news, group, dim, page_rows", [
    ([300, 90], [2, 3], 4, 64, 16),                                # warps
    ([90, 40], [1, 1], 8, 128, 32),
    ([300, 90], [200, 80], 4, 64, 16),                             # tensor memory
    ([4000, 90, 700], [150, 80, 90], 2, 128, 32),                  # shares of several blocks
    ([500, 200], [450, 180], 1, 256, 64),
])
def test_rows_that_see_absent_pages_alone_are_empty_whatever_their_query(bk, cuda, lengths, news, group, dim, page_rows):
    p = Plain(bk, lengths, news, 1, group, dim, page_rows, torch.bfloat16, seed=dim + 7)
    hidden = -(-(lengths[0] - news[0] // 2) // page_rows)          # about half of the first request's tokens see none but these
    p.table[0, :hidden] = -1
    p.table[1, :] = 10 ** 6
    p.upload()
    want, lse, tol, lse_tol = p.plain_attend(0.1)
    empty = np.isinf(lse)
    assert empty.any()
    bad = torch.tensor([math.nan, math.inf, -math.inf], dtype=torch.bfloat16, device="cuda")
    spoiled = p.d_queries.clone()
    for n, (t, g) in enumerate(zip(*np.nonzero(empty))):
        spoiled[t, g, n % dim] = bad[n % 3]
    out, got_lse = bk.cache_attend(p.cache, spoiled, p.d_lengths, p.d_table, 0.1, starts=p.d_starts)
    check(out, want, tol, "out")
    check(got_lse, lse, lse_tol, "lse")
    lists = torch.arange(max(lengths), dtype=torch.int32, device="cuda").repeat(p.tokens, 1)
    out, got_lse = bk.cache_attend_selected(p.cache, spoiled, lists, p.d_lengths, p.d_table, 0.1, starts=p.d_starts)
    check(out, want, tol, "selected out")
    check(got_lse, lse, lse_tol, "selected lse")
    dist = bk.cache_distance(p.cache, spoiled, p.d_lengths, p.d_table, max(lengths), starts=p.d_starts)
    none = torch.from_numpy(empty.all(axis=1)).cuda()
    assert bool((dist[none] == math.inf).all())
    bk.device_status()


@pytest.mark.parametrize("lengths, news, group", [([300, 90], [1, 1], 4), ([400, 60], [90, 60], 4)])
def test_outputs_may_take_turns_with_queries_but_not_lie_on_them(bk, cuda, lengths, news, group):
    p = Plain(bk, lengths, news, 2, group, 64, 16, torch.bfloat16, seed=91).upload()
    heads = 2 * group
    rows = torch.full((p.tokens, 2 * heads + 1, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    rows[:, 1:heads + 1] = p.d_queries
    queries, out = rows[:, 1:heads + 1], rows[:, heads + 1:]
    want, _, tol, _ = p.plain_attend(0.1)
    bk.cache_attend(p.cache, queries, p.d_lengths, p.d_table, 0.1, starts=p.d_starts, out=out)
    check(out, want, tol, "out")
    assert torch.equal(queries, p.d_queries) and bool((rows[:, 0] == 7).all())
    with pytest.raises(bk.BitsKnnError, match="d_out overlaps d_queries"):
        bk.cache_attend(p.cache, queries, p.d_lengths, p.d_table, 0.1, starts=p.d_starts, out=queries)
    with pytest.raises(bk.BitsKnnError, match="d_out overlaps d_queries"):
        bk.cache_attend(p.cache, queries, p.d_lengths, p.d_table, 0.1, starts=p.d_starts, out=rows[:, :heads])
    assert torch.equal(queries, p.d_queries)


def test_what_a_workspace_held_does_not_matter(bk, cuda):
    """One workspace of the least size for kernels, row lengths and column counts in turn, filled with two patterns."""
    few = Plain(bk, [9000, 300], [1, 1], 2, 4, 128, 16, torch.bfloat16, seed=101).upload()      # shares, joins of warps' items
    some = Plain(bk, [1500, 700], [4, 4], 2, 4, 128, 16, torch.bfloat16, seed=102).upload()     # two blocks of columns each
    many = Plain(bk, [900, 100], [150, 90], 2, 4, 128, 16, torch.bfloat16, seed=103).upload()   # tensor memory
    apart = pages_apart(bk, [900, 100], [150, 90], 2, 4, 128, 16, torch.bfloat16, {2, 9}, 30, 0, seed=104)
    size = bk.cache_attend_workspace_bytes(few.cache, 8)
    work = torch.empty(size, dtype=torch.uint8, device="cuda")
    lists = {id(p): torch.arange(700, dtype=torch.int32, device="cuda").repeat(p.tokens * 2, 1) for p in (few, some)}

    def call(p, listed, workspace):
        args = (p.d_lengths, p.d_table, 0.1)
        if listed:
            return bk.cache_attend_selected(p.cache, p.d_queries, lists[id(p)], *args, starts=p.d_starts, workspace=workspace)
        return bk.cache_attend(p.cache, p.d_queries, *args, starts=p.d_starts, workspace=workspace)

    calls = [(few, False), (many, False), (some, True), (apart, False), (some, False), (many, False), (few, True)]
    want = [call(p, listed, torch.zeros(size, dtype=torch.uint8, device="cuda")) for p, listed in calls]
    for fill in (None, 0xff, 0x7f, 0x01):
        for (p, listed), w in zip(calls, want):
            if fill is not None:
                work.fill_(fill)
            got = call(p, listed, work)
            assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1]), (fill, listed)
    bk.device_status()


def test_columns_of_a_matrix_may_be_selected_from(bk, cuda):
    """A matrix of one column has no stride along its rows that could matter."""
    wide = torch.randn((5, 7), device="cuda")
    for dist in (wide[:, 3:4], wide.t()[:, :1]):
        got_d, got_i = bk.select(dist, 1)
        assert torch.equal(got_d, dist) and bool((got_i == 0).all())
    with pytest.raises(ValueError, match="contiguous"):
        bk.select(wide.t()[:, :2], 1)


def test_many_columns_in_a_graph(bk, cuda):
    """Captured and replayed with other queries, lengths and scales than at the capture, next to an eager call."""
    p = pages_apart(bk, [900, 100], [150, 90], 2, 4, 128, 16, torch.bfloat16, {2, 9}, 0, 0, seed=111)
    queries = p.d_queries.clone()
    args = (p.cache, queries, p.d_lengths, p.d_table, 0.1)
    bk.cache_attend(*args, starts=p.d_starts)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = bk.cache_attend(*args, starts=p.d_starts)
    for step, (large, first) in enumerate(((0, 900), (40, 777), (0, 900), (60, 400))):
        queries.copy_(torch.roll(p.d_queries, step, dims=0))
        p.d_lengths.copy_(torch.tensor([first, 100 - step], dtype=torch.int32))
        for page in (2, 9):                                         # only at some steps do the scales lie apart
            p.cache.value_scales[int(p.d_table[0, page])] = 2.0 ** large
        graph.replay()
        eager = bk.cache_attend(*args, starts=p.d_starts)
        assert torch.equal(captured[0], eager[0]) and torch.equal(captured[1], eager[1]), step
        assert bool(captured[0].isfinite().all())
    bk.device_status()


@pytest.mark.parametrize("lengths, news, group, tokens", [
    ([60, 90, 30], [3, 5, 4], 4, 5),                                # warps; the second request is cut, the third is not there
    ([60, 90], [3, 5], 4, 3),                                       # cut between requests
    ([300, 90], [90, 60], 4, 70),                                   # tensor memory
    ([30, 700], [10, 200], 4, 150),
])
def test_arrays_that_end_within_a_request(bk, cuda, lengths, news, group, tokens):
    """Packed arrays shorter than the starts say: the tokens that are there see what they see in the whole batch."""
    p = Plain(bk, lengths, news, 2, group, 64, 16, torch.bfloat16, seed=121).upload()
    want, lse, tol, lse_tol = p.plain_attend(0.1)
    queries = p.d_queries[:tokens]
    out, got_lse = bk.cache_attend(p.cache, queries, p.d_lengths, p.d_table, 0.1, starts=p.d_starts)
    check(out, want[:tokens], tol[:tokens], "out")
    check(got_lse, lse[:tokens], lse_tol[:tokens], "lse")
    n = max(lengths)
    want_d, tol_d = p.plain_distance(n)
    check(bk.cache_distance(p.cache, queries, p.d_lengths, p.d_table, n, starts=p.d_starts), want_d[:tokens * 2],
          tol_d[:tokens * 2], "distance")
    lists = torch.arange(n, dtype=torch.int32, device="cuda").repeat(tokens * 2, 1)
    out, got_lse = bk.cache_attend_selected(p.cache, queries, lists, p.d_lengths, p.d_table, 0.1, starts=p.d_starts)
    check(out, want[:tokens], tol[:tokens], "selected out")
    check(got_lse, lse[:tokens], lse_tol[:tokens], "selected lse")
    bk.device_status()
