"""Cases of the paged 8-bit cache operators: what is timed, in a plain form and through the library.

Five operators over a cache of keys and values held as e4m3 codes in pages, with one power-of-two scale per page
and head: `plan` (block tables and slot maps from request lengths), `append` (quantising write), `distance`
(negative inner products as the matrix the top-k selection takes), `attend` (attention over the whole cache) and
`selected` (attention over listed positions).

Sizes: head dimensions are those of this repository's tests and benchmark (32 ... 256); numbers of requests,
lengths and heads are generic serving sizes.
"""
import importlib.util
import math
import pathlib
import random
import sys

import numpy as np
import torch

own = False

_ROOT = pathlib.Path(__file__).resolve().parents[1]
_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_PAD = 0x7FFFFFFF      # index of an empty list entry, as the selection writes it
_E_MIN, _E_MAX = -60, 60


def _package():
    name = "bits_knn_jpdc2024_b200"
    if name not in sys.modules:
        path = _ROOT / "bits-knn-jpdc2024_b200"
        spec = importlib.util.spec_from_file_location(name, path / "__init__.py",
                                                      submodule_search_locations=[str(path)])
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    return sys.modules[name]


# ---- the cases -------------------------------------------------------------------------------------------------
def listed():
    return [
        # scheduling step of a small server: every request gets one token, a few begin a page
        dict(name="plan_step", op="plan", requests=24, ctx_lo=0, ctx_hi=5000, new_lo=1, new_hi=1, page=16, layout=1),
        # scheduling step of a large server with prompts among the decodes
        dict(name="plan_mixed", op="plan", requests=4096, ctx_lo=0, ctx_hi=9000, new_lo=1, new_hi=400, page=32,
             layout=2),
        # one token of each of a batch of requests enters the cache (a decode step)
        dict(name="append_step", op="append", requests=48, ctx_lo=0, ctx_hi=300, new_lo=1, new_hi=1, page=16,
             heads=8, dim=128, dtype="bf16", layout=3),
        # chunks of prompts enter the cache
        dict(name="append_chunks", op="append", requests=12, ctx_lo=0, ctx_hi=300, new_lo=900, new_hi=4100, page=64,
             heads=8, dim=128, dtype="f16", layout=4),
        # one request looks for its nearest keys: the smallest call
        dict(name="distance_one", op="distance", requests=1, ctx_lo=9001, ctx_hi=9001, new_lo=1, new_hi=1, page=16,
             heads=4, group=8, dim=64, dtype="f16", layout=5),
        # a batch of long requests looks for its nearest keys
        dict(name="distance_batch", op="distance", requests=16, ctx_lo=2000, ctx_hi=60000, new_lo=1, new_hi=1,
             page=64, heads=8, group=4, dim=128, dtype="bf16", layout=6),
        # one short request decodes: latency
        dict(name="attend_one", op="attend", requests=1, ctx_lo=777, ctx_hi=777, new_lo=1, new_hi=1, page=16,
             heads=4, group=8, dim=128, dtype="bf16", layout=7),
        # an ordinary decode step of a ragged batch
        dict(name="attend_batch", op="attend", requests=64, ctx_lo=150, ctx_hi=24000, new_lo=1, new_hi=1, page=16,
             heads=8, group=4, dim=128, dtype="bf16", layout=8),
        # one very long request decodes: the long axis has to be split
        dict(name="attend_long", op="attend", requests=1, ctx_lo=250001, ctx_hi=250001, new_lo=1, new_hi=1, page=64,
             heads=8, group=8, dim=128, dtype="f16", layout=9),
        # chunks of prompts attend to what the cache holds and to themselves: compute-bound
        dict(name="attend_chunk", op="attend", requests=3, ctx_lo=1500, ctx_hi=8000, new_lo=700, new_hi=2100,
             page=32, heads=8, group=4, dim=128, dtype="bf16", layout=10),
        # one request attends to its 64 nearest keys: latency
        dict(name="selected_one", op="selected", requests=1, ctx_lo=5000, ctx_hi=5000, new_lo=1, new_hi=1, page=16,
             heads=8, group=4, dim=64, k=64, dtype="bf16", layout=11),
        # a batch attends to its 2048 nearest keys, the longest list of the selection
        dict(name="selected_batch", op="selected", requests=32, ctx_lo=3000, ctx_hi=50000, new_lo=1, new_hi=1,
             page=64, heads=8, group=4, dim=128, k=2048, dtype="bf16", layout=12),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["plan", "append", "distance", "attend", "attend", "selected"])
        case = dict(op=op, page=rng.choice([16, 32, 64, 128]), layout=rng.randrange(1 << 30))
        if op == "plan":
            case["requests"] = _log_int(rng, 1, 4096)
            case.update(ctx_lo=0, ctx_hi=_log_int(rng, 1, 20000), new_lo=rng.randrange(2), new_hi=_log_int(rng, 1, 400))
            return case
        case["heads"] = rng.choice([1, 2, 4, 5, 8, 16])
        case["dim"] = rng.choice([32, 64, 64, 96, 128, 128, 128, 192, 256])
        if op == "append":
            case["dtype"] = rng.choice(["bf16", "f16", "f32"])
            case["requests"] = _log_int(rng, 1, 200)
            case.update(ctx_lo=0, ctx_hi=_log_int(rng, 1, 500), new_lo=1,
                        new_hi=rng.choice([1, 1, _log_int(rng, 2, 3000)]))
        else:
            case["dtype"] = rng.choice(["bf16", "f16"])
            case["group"] = rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16])
            case["requests"] = _log_int(rng, 1, 80)
            hi = _log_int(rng, 1, 100000)
            case.update(ctx_lo=rng.choice([0, hi // 2, hi]), ctx_hi=hi, new_lo=1, new_hi=1)
            if op == "attend" and rng.random() < 0.5:
                case["new_hi"] = _log_int(rng, 2, 1500)
            elif rng.random() < 0.3:
                case["new_hi"] = _log_int(rng, 2, 8)
            if op == "selected":
                case["k"] = _log_int(rng, 1, 2048)
        # no dearer than the largest listed case of the operator, in bytes and in operations
        top = [work(c) for c in listed() if c["op"] == op]
        here = work(case)
        if all(here[u] <= max(t[u] for t in top) for u in ("bytes", "flops")):
            return case


def _lengths(case):
    """(tokens already cached, new tokens) of every request; made from the case alone."""
    rng = random.Random(case["layout"])

    def one(lo, hi):
        return lo if lo == hi else _log_int(rng, lo + 1, hi + 1) - 1

    ctx = [one(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["requests"])]
    new = [one(case["new_lo"], case["new_hi"]) for _ in range(case["requests"])]
    return ctx, new


def work(case):
    ctx, new = _lengths(case)
    page, tokens = case["page"], sum(new)
    if case["op"] == "plan":
        taken = sum(-(-(c + m) // page) - -(-c // page) for c, m in zip(ctx, new))
        # lengths and counts in; starts, lengths, slots and the new table entries out
        return {"bytes": 16 * len(ctx) + 8 * taken + 8 * tokens, "flops": len(ctx) + tokens}
    heads, dim = case["heads"], case["dim"]
    if case["op"] == "append":
        item = 4 if case["dtype"] == "f32" else 2
        return {"bytes": 2 * tokens * heads * dim * (item + 1) + 8 * tokens, "flops": 4 * tokens * heads * dim}
    group = case["group"]
    visible = sum(m * c + m * (m + 1) // 2 for c, m in zip(ctx, new))          # (token, position) pairs
    cached = sum(c + m for c, m in zip(ctx, new))
    pages = sum(-(-(c + m) // page) for c, m in zip(ctx, new))
    rows_io = tokens * heads * group * dim * 2
    if case["op"] == "distance":
        n = max(c + m for c, m in zip(ctx, new))
        return {"bytes": cached * heads * dim + pages * (4 * heads + 4) + rows_io + 4 * tokens * heads * n,
                "flops": 2 * visible * heads * group * dim}
    if case["op"] == "attend":
        return {"bytes": 2 * cached * heads * dim + pages * (8 * heads + 4) + 2 * rows_io + 4 * tokens * heads * group,
                "flops": 4 * visible * heads * group * dim}
    k = case["k"]
    entries = sum(min(k, c + i + 1) for c, m in zip(ctx, new) for i in range(m))
    # a list's keys and values are read once for its row; several tokens of a request may share them
    touched = sum(min(c + m, sum(min(k, c + i + 1) for i in range(m))) for c, m in zip(ctx, new))
    return {"bytes": 2 * touched * heads * dim + 4 * tokens * heads * k + 2 * rows_io,
            "flops": 4 * entries * heads * group * dim}


# ---- inputs ----------------------------------------------------------------------------------------------------
def _exponent(amax):
    """Smallest e in [-60, 60] with amax <= 448 * 2^e (448 = 0.875 * 2^9 is the largest e4m3 number)."""
    mant, ex = torch.frexp(amax)
    e = ex - 9 + (mant > 0.875).to(ex.dtype)
    return torch.where(amax > 0, e, torch.full_like(e, _E_MIN)).clamp(_E_MIN, _E_MAX)


def _pow2(e):
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _to_codes(x):
    return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)


def _fill_pages(pages, heads, page, dim, gen, spread):
    """Codes and scales of pages full of normal vectors whose sizes differ from token to token."""
    codes = torch.empty((pages, heads, page, dim), dtype=torch.uint8, device="cuda")
    scales = torch.empty((pages, heads), dtype=torch.float32, device="cuda")
    step = max(1, (1 << 26) // (heads * page * dim))
    for a in range(0, pages, step):
        b = min(pages, a + step)
        x = torch.randn((b - a, heads, page, dim), generator=gen, device="cuda")
        x *= torch.exp(spread * torch.randn((b - a, heads, page, 1), generator=gen, device="cuda"))
        e = _exponent(x.abs().amax(dim=(2, 3)))
        scales[a:b] = _pow2(e)
        codes[a:b] = _to_codes(x / scales[a:b, :, None, None])
    return codes, scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)
    ctx, new = _lengths(case)
    page, requests, tokens = case["page"], case["requests"], sum(new)
    st = dict(case=case, ctx=ctx, new=new, tokens=tokens)
    old_pages = [-(-c // page) for c in ctx]
    all_pages = [-(-(c + m) // page) for c, m in zip(ctx, new)]
    total = sum(all_pages)
    pool = total + 8
    order = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
    width = max(all_pages) + 1
    # requests came and grew in turns, so their pages lie scattered
    table = np.full((requests, width), -1, dtype=np.int32)
    host_order = order.cpu().numpy()
    at = 0
    for r in range(requests):
        table[r, :old_pages[r]] = host_order[at:at + old_pages[r]]
        at += old_pages[r]
    free = host_order[at:]
    i32 = dict(dtype=torch.int32, device="cuda")
    if case["op"] == "plan":
        st.update(lengths=torch.tensor(ctx, **i32), counts=torch.tensor(new, **i32),
                  table=torch.from_numpy(table).cuda(), free=torch.from_numpy(free.copy()).cuda(),
                  max_tokens=tokens + 3)
        return st
    f = 0
    for r in range(requests):
        more = all_pages[r] - old_pages[r]
        table[r, old_pages[r]:all_pages[r]] = free[f:f + more]
        f += more
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    heads, dim, dtype = case["heads"], case["dim"], _DTYPES[case["dtype"]]
    if case["op"] == "append":
        st["keys"], st["key_scales"] = _fill_pages(pool, heads, page, dim, gen, 0.3)
        st["values"], st["value_scales"] = _fill_pages(pool, heads, page, dim, gen, 0.3)
        slots = [int(table[r, (ctx[r] + i) // page]) * page + (ctx[r] + i) % page
                 for r in range(requests) for i in range(new[r])]
        st["slots"] = torch.tensor(slots, dtype=torch.int64, device="cuda")
        for name in ("new_keys", "new_values"):
            x = torch.randn((tokens, heads, dim), generator=gen, device="cuda")
            x *= torch.exp(0.4 * torch.randn((tokens, heads, 1), generator=gen, device="cuda"))
            st[name] = x.to(dtype)
        if own:
            st["cache"] = _package().Cache(st["keys"], st["values"], st["key_scales"], st["value_scales"])
        return st
    st["keys"], st["key_scales"] = _fill_pages(pool, heads, page, dim, gen, 0.3)
    if case["op"] != "distance":
        st["values"], st["value_scales"] = _fill_pages(pool, heads, page, dim, gen, 0.5)
    else:
        st["values"], st["value_scales"] = st["keys"], st["key_scales"]
    st["table"] = torch.from_numpy(table).cuda()
    st["lengths"] = torch.tensor([c + m for c, m in zip(ctx, new)], **i32)
    st["starts"] = None if all(m == 1 for m in new) else torch.from_numpy(starts).cuda()
    st["queries"] = torch.randn((tokens, heads * case["group"], dim), generator=gen, device="cuda").to(dtype)
    st["scale"] = 1.0 / math.sqrt(dim)
    st["n"] = max(c + m for c, m in zip(ctx, new))
    if case["op"] == "selected":
        # the lists of a selection over some scores: distinct positions in no order, and where fewer are
        # visible than the list holds, entries that name positions behind the visible ones
        k, rows = case["k"], []
        for c, m in zip(ctx, new):
            for i in range(m):
                vis = c + i + 1
                got = torch.rand((heads, vis), generator=gen, device="cuda").topk(min(k, vis), dim=1).indices
                pad = torch.full((heads, k - got.shape[1]), _PAD, dtype=got.dtype, device="cuda")
                pad[:, :1] = vis
                rows.append(torch.cat([got, pad], dim=1).to(torch.int32))
        st["lists"] = torch.cat(rows, dim=0).contiguous()
    if own:
        bk = _package()
        st["cache"] = bk.Cache(st["keys"], st["values"], st["key_scales"], st["value_scales"])
        size = bk.cache_attend_workspace_bytes(st["cache"], heads * case["group"])
        st["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    return st


# ---- one pass --------------------------------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)[state["case"]["op"]](state)


def _own_plan(st):
    bk = _package()
    starts, lengths, slots, counts = bk.cache_plan(st["lengths"], st["counts"], st["free"], st["table"],
                                                   st["case"]["page"], st["max_tokens"])
    return starts, lengths, slots, counts, st["table"]


def _own_append(st):
    _package().cache_append(st["cache"], st["new_keys"], st["new_values"], st["slots"])
    return _cache_outputs(st)


def _own_distance(st):
    return _package().cache_distance(st["cache"], st["queries"], st["lengths"], st["table"], st["n"],
                                     starts=st["starts"])


def _own_attend(st):
    return _package().cache_attend(st["cache"], st["queries"], st["lengths"], st["table"], st["scale"],
                                   starts=st["starts"], workspace=st["workspace"])


def _own_selected(st):
    return _package().cache_attend_selected(st["cache"], st["queries"], st["lists"], st["lengths"], st["table"],
                                            st["scale"], starts=st["starts"], workspace=st["workspace"])


def _cache_outputs(st):
    # the codes as the numbers they stand for (times the page's scale)
    return (st["keys"].view(torch.float8_e4m3fn), st["values"].view(torch.float8_e4m3fn), st["key_scales"],
            st["value_scales"])


def _plain_plan(st):
    page, table, max_tokens = st["case"]["page"], st["table"], st["max_tokens"]
    lengths, new, free = st["lengths"].long(), st["counts"].long(), st["free"]
    ends = torch.cumsum(new, 0)
    starts = torch.cat([torch.zeros_like(ends[:1]), ends])
    have = (lengths + page - 1) // page
    need = (lengths + new + page - 1) // page
    first = torch.cumsum(need - have, 0) - (need - have)
    column = torch.arange(table.shape[1], device=table.device)
    take = (column >= have[:, None]) & (column < need[:, None])
    source = torch.where(take, first[:, None] + column - have[:, None], 0)
    table.copy_(torch.where(take, free[source], table))
    token = torch.arange(max_tokens, device=table.device)
    owner = torch.bucketize(token, ends, right=True).clamp(max=len(new) - 1)
    position = lengths[owner] + token - starts[owner]
    slot = table[owner, (position // page).clamp(0, table.shape[1] - 1)].long() * page + position % page
    slot = torch.where(token < ends[-1], slot, torch.full_like(slot, -1))
    zero = torch.zeros_like(ends[-1])
    counts = torch.stack([ends[-1], (need - have).sum(), zero])
    return starts.int(), (lengths + new).int(), slot, counts.int(), table


def _plain_append_one(codes, scales, new, slots, page):
    pages, heads = scales.shape
    x = new.float()
    where, offset = slots // page, slots % page
    amax = torch.zeros((pages, heads), device=x.device).index_reduce_(0, where, x.abs().amax(dim=2), "amax")
    first = torch.full((pages,), page, dtype=torch.int64, device=x.device).index_reduce_(0, where, offset, "amin")
    touched = torch.nonzero(first < page)[:, 0]
    old = torch.frexp(scales[touched])[1] - 1
    e = _exponent(amax[touched])
    e = torch.where((first[touched] == 0)[:, None], e, torch.maximum(e, old))
    shrink = _pow2((old - e).clamp(-120, 0))
    held = codes[touched].view(torch.float8_e4m3fn).float()
    kept = torch.arange(page, device=x.device)[None, :] < first[touched][:, None]
    held = torch.where(kept[:, None, :, None], held * shrink[:, :, None, None], held)
    codes[touched] = _to_codes(held)
    scales[touched] = _pow2(e)
    codes[where, :, offset] = _to_codes(x / scales[where][:, :, None])


def _plain_append(st):
    page = st["case"]["page"]
    _plain_append_one(st["keys"], st["key_scales"], st["new_keys"], st["slots"], page)
    _plain_append_one(st["values"], st["value_scales"], st["new_values"], st["slots"], page)
    return _cache_outputs(st)


def _requests(st):
    """(request, first token, new tokens, length) of every request with tokens in this pass."""
    at = 0
    for r, (c, m) in enumerate(zip(st["ctx"], st["new"])):
        if m > 0:
            yield r, at, m, c + m
        at += m


def _rows(st, codes, scales, r, length):
    """(heads, length, dim) float32 vectors of a request."""
    page, (_, heads, _, dim) = st["case"]["page"], codes.shape
    ids = st["table"][r, :-(-length // page)].long()
    x = codes[ids].view(torch.float8_e4m3fn).float() * scales[ids][:, :, None, None]
    return x.permute(1, 0, 2, 3).reshape(heads, -1, dim)[:, :length]


def _grouped(st, at, m):
    """(heads, m * group, dim) float32 queries of m tokens."""
    case = st["case"]
    q = st["queries"][at:at + m].float().view(m, case["heads"], case["group"], case["dim"])
    return q.permute(1, 0, 2, 3).reshape(case["heads"], m * case["group"], case["dim"])


def _plain_distance(st):
    case = st["case"]
    heads, group, n = case["heads"], case["group"], st["n"]
    out = torch.full((st["tokens"], heads, n), math.inf, device="cuda")
    for r, at, m, length in _requests(st):
        k = _rows(st, st["keys"], st["key_scales"], r, length)
        s = (_grouped(st, at, m) @ k.transpose(1, 2)).view(heads, m, group, length).amax(dim=2)
        visible = length - m + 1 + torch.arange(m, device="cuda")
        s = torch.where(torch.arange(length, device="cuda") < visible[:, None], -s, math.inf)
        out[at:at + m, :, :length] = s.permute(1, 0, 2)
    return out.view(st["tokens"] * heads, n)


def _plain_attend(st):
    case = st["case"]
    heads, group, dim = case["heads"], case["group"], case["dim"]
    out = torch.zeros_like(st["queries"])
    lse = torch.full((st["tokens"], heads * group), -math.inf, device="cuda")
    for r, at, m, length in _requests(st):
        k = _rows(st, st["keys"], st["key_scales"], r, length)
        v = _rows(st, st["values"], st["value_scales"], r, length)
        s = (_grouped(st, at, m) @ k.transpose(1, 2)) * st["scale"]
        if m > 1:
            visible = (length - m + 1 + torch.arange(m, device="cuda")).repeat_interleave(group)
            s = s.masked_fill(torch.arange(length, device="cuda") >= visible[:, None], -math.inf)
        top = s.amax(dim=2, keepdim=True)
        p = torch.exp(s - top)
        total = p.sum(dim=2, keepdim=True)
        o = (p @ v) / total
        out[at:at + m] = o.view(heads, m, group, dim).permute(1, 0, 2, 3).reshape(m, heads * group, dim).to(out.dtype)
        lse[at:at + m] = (top + torch.log(total)).view(heads, m, group).permute(1, 0, 2).reshape(m, heads * group)
    return out, lse


def _plain_selected(st):
    case = st["case"]
    heads, group, dim, page = case["heads"], case["group"], case["dim"], case["page"]
    tokens, k = st["tokens"], case["k"]
    owner = torch.tensor([r for r, m in enumerate(st["new"]) for _ in range(m)], device="cuda")
    visible = torch.tensor([c + i + 1 for c, m in zip(st["ctx"], st["new"]) for i in range(m)], device="cuda")
    out = torch.empty_like(st["queries"])
    lse = torch.empty((tokens, heads * group), device="cuda")
    step = max(1, (1 << 27) // (heads * k * dim))
    head = torch.arange(heads, device="cuda")[None, :, None]
    for a in range(0, tokens, step):
        b = min(tokens, a + step)
        idx = st["lists"].view(tokens, heads, k)[a:b].long()
        seen = (idx >= 0) & (idx < visible[a:b, None, None])
        idx = torch.where(seen, idx, 0)
        pages = st["table"][owner[a:b, None, None], idx // page].long()

        def rows(codes, scales):
            return codes[pages, head, idx % page].view(torch.float8_e4m3fn).float() * scales[pages, head][..., None]

        q = st["queries"][a:b].float().view(b - a, heads, group, dim)
        s = (q @ rows(st["keys"], st["key_scales"]).transpose(2, 3)) * st["scale"]
        s = s.masked_fill(~seen[:, :, None, :], -math.inf)
        top = s.amax(dim=3, keepdim=True)
        p = torch.exp(s - top)
        total = p.sum(dim=3, keepdim=True)
        o = (p @ rows(st["values"], st["value_scales"])) / total
        out[a:b] = o.reshape(b - a, heads * group, dim).to(out.dtype)
        lse[a:b] = (top + torch.log(total)).reshape(b - a, heads * group)
    return out, lse


_run_plain = {"plan": _plain_plan, "append": _plain_append, "distance": _plain_distance, "attend": _plain_attend,
              "selected": _plain_selected}
_run_own = {"plan": _own_plan, "append": _own_append, "distance": _own_distance, "attend": _own_attend,
            "selected": _own_selected}


# ---- the definitions in 64 bits, written apart from the plain forms ------------------------------------------
def _decode_table():
    """The 256 numbers of e4m3: sign, 4 exponent bits (bias 7), 3 fraction bits; no infinities."""
    out = np.empty(256)
    for c in range(256):
        exponent, fraction = (c >> 3) & 15, c & 7
        size = math.ldexp(fraction, -9) if exponent == 0 else math.ldexp(8 + fraction, exponent - 10)
        if exponent == 15 and fraction == 7:
            size = math.nan
        out[c] = -size if c & 128 else size
    return out


def _round_e4m3(x):
    """Nearest e4m3 number, ties to even, saturating (numpy, 64 bits)."""
    size = np.minimum(np.abs(x), 448.0)
    exponent = np.frexp(np.maximum(size, 2.0 ** -60))[1] - 1
    quantum = np.ldexp(1.0, np.maximum(exponent, -6) - 3)
    return np.copysign(np.minimum(np.rint(size / quantum) * quantum, 448.0), x)


def _exact_plan(st):
    page = st["case"]["page"]
    table, free = st["table"].cpu().numpy().copy(), st["free"].cpu().numpy()
    starts, slots, taken = [0], [], 0
    for r, (c, m) in enumerate(zip(st["ctx"], st["new"])):
        starts.append(starts[-1] + m)
        for i in range(c, c + m):
            if i % page == 0:
                table[r, i // page] = free[taken]
                taken += 1
            slots.append(int(table[r, i // page]) * page + i % page)
    slots += [-1] * (st["max_tokens"] - len(slots))
    lengths = [c + m for c, m in zip(st["ctx"], st["new"])]
    back = [np.array(starts, np.int32), np.array(lengths, np.int32), np.array(slots, np.int64),
            np.array([starts[-1], taken, 0], np.int32), table]
    return tuple(torch.from_numpy(a) for a in back)


def _exact_append(st):
    page, table = st["case"]["page"], _decode_table()
    where = (st["slots"] // page).cpu().numpy()
    offset = (st["slots"] % page).cpu().numpy()
    order = np.argsort(where, kind="stable")
    cuts = np.flatnonzero(np.diff(where[order])) + 1
    result = []
    for codes, scales, new in (("keys", "key_scales", "new_keys"), ("values", "value_scales", "new_values")):
        held = table[st[codes].cpu().numpy()]
        size = st[scales].cpu().numpy().astype(np.float64)
        x = st[new].cpu().to(torch.float64).numpy()
        for run_ in np.split(order, cuts):
            p, first = where[run_[0]], offset[run_].min()
            rows = x[run_]                                                    # (tokens, heads, dim)
            amax = np.abs(rows).max(axis=(0, 2))
            with np.errstate(divide="ignore"):
                e = np.ceil(np.log2(amax / 448.0))
            e = np.where(448.0 * np.exp2(e - 1) >= amax, e - 1, e)            # log2 rounded up over a border
            e = np.where(448.0 * np.exp2(e) < amax, e + 1, e)
            fresh = np.exp2(np.clip(np.nan_to_num(e, neginf=_E_MIN), _E_MIN, _E_MAX))
            fresh = fresh if first == 0 else np.maximum(fresh, size[p])
            held[p, :, :first] = _round_e4m3(held[p, :, :first] * (size[p] / fresh)[:, None, None])
            size[p] = fresh
            held[p][:, offset[run_]] = _round_e4m3(rows / fresh[None, :, None]).transpose(1, 0, 2)
        result.append((torch.from_numpy(held), torch.from_numpy(size)))
    return result[0][0], result[1][0], result[0][1], result[1][1]


def _exact_rows(st, which, r):
    """(heads, positions, dim) float64 vectors of a request, page by page through a table of the 256 numbers."""
    values = torch.from_numpy(_decode_table()).cuda()
    length = st["ctx"][r] + st["new"][r]
    ids = [int(p) for p in st["table"][r].cpu() if p >= 0]
    ids = torch.tensor(ids, device="cuda")
    x = values[st[which][ids].int()] * st[which[:-1] + "_scales"][ids].double()[:, :, None, None]
    return torch.cat(list(x.unbind(0)), dim=1)[:, :length]


def _exact_distance(st):
    case, rows, at = st["case"], [], 0
    for r, (c, m) in enumerate(zip(st["ctx"], st["new"])):
        if m == 0:
            continue
        k = _exact_rows(st, "keys", r)
        for i in range(at, at + m):
            seen = c + i - at + 1
            q = st["queries"][i].double().view(case["heads"], case["group"], case["dim"])
            best = torch.einsum("hgd,hjd->hgj", q, k[:, :seen]).max(dim=1).values
            rows.append(torch.nn.functional.pad(-best, (0, st["n"] - seen), value=math.inf))
        at += m
    return torch.cat(rows)


def _exact_softmax(q, k, v, scale, hidden=None):
    s = torch.einsum("hgd,hjd->hgj", q, k) * scale
    if hidden is not None:
        s = s.masked_fill(hidden, -math.inf)
    lse = torch.logsumexp(s, dim=2)
    return torch.einsum("hgj,hjd->hgd", torch.exp(s - lse[..., None]), v), lse


def _exact_attend(st):
    case, outs, lses, at = st["case"], [], [], 0
    heads, group, dim = case["heads"], case["group"], case["dim"]
    for r, (c, m) in enumerate(zip(st["ctx"], st["new"])):
        if m == 0:
            continue
        k, v = _exact_rows(st, "keys", r), _exact_rows(st, "values", r)
        step = max(1, (1 << 26) // (heads * group * (c + m)))
        for a in range(0, m, step):
            b = min(m, a + step)
            q = st["queries"][at + a:at + b].double().view(b - a, heads, group, dim)
            q = q.transpose(0, 1).reshape(heads, (b - a) * group, dim)
            token = torch.arange(a, b, device="cuda").repeat_interleave(group)
            hidden = torch.arange(c + b, device="cuda")[None, :] > (c + token)[:, None]
            o, lse = _exact_softmax(q, k[:, :c + b], v[:, :c + b], st["scale"], hidden)
            outs.append(o.view(heads, b - a, group, dim).transpose(0, 1).reshape(b - a, heads * group, dim))
            lses.append(lse.view(heads, b - a, group).transpose(0, 1).reshape(b - a, heads * group))
        at += m
    return torch.cat(outs), torch.cat(lses)


def _exact_selected(st):
    case, outs, lses, at = st["case"], [], [], 0
    heads, group, dim, k = case["heads"], case["group"], case["dim"], case["k"]
    for r, (c, m) in enumerate(zip(st["ctx"], st["new"])):
        if m == 0:
            continue
        keys, values = _exact_rows(st, "keys", r), _exact_rows(st, "values", r)
        for i in range(at, at + m):
            lists = st["lists"].view(-1, heads, k)[i].long()
            q = st["queries"][i].double().view(heads, group, dim)
            for h in range(heads):
                use = lists[h][(lists[h] >= 0) & (lists[h] <= c + i - at)]
                o, lse = _exact_softmax(q[h:h + 1], keys[h:h + 1, use], values[h:h + 1, use], st["scale"])
                outs.append(o[0])
                lses.append(lse[0])
        at += m
    return torch.stack(outs).view(-1, heads * group, dim), torch.stack(lses).view(-1, heads * group)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] in ("distance", "selected") and st["tokens"] * case["heads"] > 20000:
        return None
    return {"plan": _exact_plan, "append": _exact_append, "distance": _exact_distance, "attend": _exact_attend,
            "selected": _exact_selected}[case["op"]](st)
