"""Measured cases of the paged-cache operators: attention of single tokens and of prompt
chunks over a page table (causal, optionally a sliding window with a few first tokens that
stay visible), copies of pages and the compaction of a pool.

The cache is the engine's: pool [layer][page][k | v][kv_head][slot][dim] BF16, a page table
of int32 per row, logical page i of a row holding its positions [i * P, (i + 1) * P). Keys
are cached normalized and rotated, queries come normalized and rotated too, so both have
unit mean square; the softmax scale is dim ** -0.5.
"""
import importlib.util
import os
import sys

import torch

own = False

DEV = "cuda"


def _package():
    """The framework's package (its directory name has a hyphen: imported by path)."""
    name = "yue2_mlx_b200"
    if name not in sys.modules:
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "yue2-mlx_b200")
        spec = importlib.util.spec_from_file_location(name, os.path.join(pkg, "__init__.py"),
                                                      submodule_search_locations=[pkg])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


# ---------------------------------------------------------------------------------------
# Cases

def _decode(name, rows, lo, hi, empty=0, heads=16, kv=8, dim=128, page=256, window=0, sinks=0):
    return dict(name=name, op="decode", rows=rows, lo=lo, hi=hi, empty=empty, heads=heads, kv=kv, dim=dim, page=page,
                window=window, sinks=sinks)


def _prefill(name, rows, n_lo, n_hi, c_lo, c_hi, heads=16, kv=8, dim=128, page=256, window=0, sinks=0):
    return dict(name=name, op="prefill", rows=rows, n_lo=n_lo, n_hi=n_hi, c_lo=c_lo, c_hi=c_hi, heads=heads, kv=kv,
                dim=dim, page=page, window=window, sinks=sinks)


def _copy(name, layers, pages, pairs, tokens, kv=8, dim=128, page=256):
    return dict(name=name, op="copy", layers=layers, pages=pages, pairs=pairs, tokens=tokens, kv=kv, dim=dim, page=page)


def _compact(name, layers, pages, rows, per_row, shared, kv=8, dim=128, page=256):
    return dict(name=name, op="compact", layers=layers, pages=pages, rows=rows, per_row=per_row, shared=shared, kv=kv,
                dim=dim, page=page)


def listed():
    return [
        # One song's step right after its 512-token prompt: one launch's latency.
        _decode("decode-1x513", 1, 513, 513),
        # One song near the end of the context: the whole cache of a layer once.
        _decode("decode-1x24000", 1, 24000, 24000),
        # 64 songs at ragged lengths, 2,048 recent positions and 4 first ones visible.
        _decode("decode-64-window", 64, 600, 24576, window=2048, sinks=4),
        # The small model's head dim, a group of seven, small pages, finished rows (empty).
        _decode("decode-33-dim64", 33, 1, 3001, empty=5, heads=14, kv=2, dim=64, page=16, window=1500, sinks=5),
        # A short prompt on the small model.
        _prefill("prefill-77-dim64", 1, 77, 77, 0, 0, heads=4, kv=2, dim=64, page=16),
        # A 1,024-token chunk of a long prompt over 7,168 cached positions, everything visible.
        _prefill("prefill-1024-at-7168", 1, 1024, 1024, 7168, 7168),
        # A 16,384-token prompt with a sliding window.
        _prefill("prefill-16384-window", 1, 16384, 16384, 0, 0, window=2048, sinks=4),
        # A batch of requests of different lengths, some continuing a cached prefix.
        _prefill("prefill-ragged-24", 24, 1, 900, 0, 1100, window=1000, sinks=3),
        # A fork whose last page is part full: 131 positions of every layer.
        _copy("copy-1-part", 28, 24, 1, 131),
        # One prompt forked for 64 songs: 63 copies of its last page.
        _copy("copy-63", 28, 72, 63, 256),
        # A small pool of small pages, a few holes.
        _compact("compact-small", 2, 64, 4, 9, 2, kv=2, dim=64, page=16),
        # The pool of a batch after songs ended and windows moved on.
        _compact("compact-160", 28, 160, 20, 8, 2),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["decode", "decode", "prefill", "prefill", "copy", "compact"])
    dim = rng.choice([64, 128, 128])
    page = rng.choice([16, 32, 64, 128, 256, 256])
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 2, 3, 4, 7, 8])
    window, sinks = rng.choice([(0, 0), (_log(rng, 17, 4096), rng.randint(0, 64))])
    if op == "decode":
        rows = _log(rng, 1, 64)
        hi = _log(rng, 1, min(24576, 130000 * 8 * 128 // (rows * kv * dim)))
        lo = rng.randint(1, hi)
        return _decode("", rows, lo, hi, rng.choice([0, 0, 3]), kv * group, kv, dim, page, window, sinks)
    if op == "prefill":
        n_hi = _log(rng, 2, 8192)
        c_hi = rng.choice([0, _log(rng, 1, 8192)])
        # At most the work of 16,384 queries over 2,048 keys on 16 heads of 128.
        cost = n_hi * (min(n_hi + c_hi, window + sinks if window else 1 << 20)) * kv * group * dim
        rows = max(1, min(32, int(16384 * 2048 * 16 * 128 // max(cost, 1))))
        while cost > 16384 * 2048 * 16 * 128 and kv * group > 1:
            if group > 1:
                group = max(1, group // 2)
            else:
                kv //= 2
            cost = n_hi * (min(n_hi + c_hi, window + sinks if window else 1 << 20)) * kv * group * dim
        rows = _log(rng, 1, rows)
        return _prefill("", rows, rng.randint(1, n_hi), n_hi, rng.randint(0, c_hi), c_hi, kv * group, kv, dim, page,
                        window, sinks)
    # Pools of the engine's layouts, at most the listed pools' bytes.
    layers = rng.choice([2, 28])
    if op == "copy":
        pairs = _log(rng, 1, 60)
        return _copy("", layers, 2 * pairs + rng.randint(1, 9) if pairs < 30 else pairs + 9, pairs, rng.randint(1, page),
                     kv, dim, page)
    pages = _log(rng, 16, 150)
    rows = _log(rng, 1, 24)
    per_row = max(1, int(pages * rng.uniform(0.2, 0.9)) // rows)
    return _compact("", layers, pages, rows, per_row, rng.randint(0, per_row - 1), kv, dim, page)


def _spread(lo, hi, n):
    return [lo + (hi - lo) * i // max(n - 1, 1) for i in range(n)]


def _lengths(case):
    """Cached positions of every row of a decode case; every `empty`-th row has none."""
    lens = _spread(case["lo"], case["hi"], case["rows"])
    if case["empty"]:
        lens = [0 if i % case["empty"] == case["empty"] - 1 else x for i, x in enumerate(lens)]
    return lens


def _chunks(case):
    """(queries, positions cached before them) of every row of a prefill case."""
    n, c = _spread(case["n_lo"], case["n_hi"], case["rows"]), _spread(case["c_lo"], case["c_hi"], case["rows"])
    return [(n[i], c[i * 7 % case["rows"]]) for i in range(case["rows"])]


def _visible(length, window, sinks):
    """Keys that a query sees at the end of `length` positions (itself included)."""
    if not window or length <= window:
        return length
    return window + min(sinks, length - window)


# ---------------------------------------------------------------------------------------
# Inputs

def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(shape, g):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16)


def prepare(case, seed):
    g = _generator(seed)
    P, kv, dim = case["page"], case["kv"], case["dim"]
    st = dict(case)
    if case["op"] in ("decode", "prefill"):
        if case["op"] == "decode":
            order = torch.randperm(case["rows"], generator=g, device=DEV).tolist()
            lens = [_lengths(case)[i] for i in order]
            queries = [1] * case["rows"]
        else:
            order = torch.randperm(case["rows"], generator=g, device=DEV).tolist()
            chunks = [_chunks(case)[i] for i in order]
            queries = [n for n, _ in chunks]
            lens = [n + c for n, c in chunks]
        per_row = max(1, max((x + P - 1) // P for x in lens))
        pages = per_row * case["rows"] + 1
        # Two layers, the second one read: a layer's cache lies inside a larger pool.
        st["pool"] = _randn((2, pages, 2, kv, P, dim), g)
        st["table"] = torch.randperm(pages, generator=g, device=DEV)[:per_row * case["rows"]].to(torch.int32).view(
            case["rows"], per_row).contiguous()
        st["lengths"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        st["max_length"] = max(lens)
        st["q"] = _randn((sum(queries), case["heads"], dim), g)
        if case["op"] == "prefill":
            offs = [0]
            for n in queries:
                offs.append(offs[-1] + n)
            st["offsets"] = torch.tensor(offs, dtype=torch.int32, device=DEV)
            st["spans"] = list(zip(offs[:-1], offs[1:]))
            st["lens"] = lens
        return st
    st["pool"] = _randn((case["layers"], case["pages"], 2, kv, P, dim), g)
    perm = torch.randperm(case["pages"], generator=g, device=DEV).tolist()
    if case["op"] == "copy":
        n, spare = case["pairs"], case["pages"] - case["pairs"]
        st["dst"] = perm[:n]
        st["src"] = [perm[n + i % spare] for i in range(n)] if spare < n else perm[n:2 * n]
        st["tokens"] = [case["tokens"]] * n
        st["src_d"] = torch.tensor(st["src"], device=DEV)
        st["dst_d"] = torch.tensor(st["dst"], device=DEV)
        return st
    rows, per, sh = case["rows"], case["per_row"], case["shared"]
    # Rows share their first `shared` pages (one prompt); the others are their own, as many
    # as the pool has; a page in four behind each row's first has been freed (-1).
    table = torch.full((rows, per + 1), -1, dtype=torch.int32)
    nxt = sh
    for r in range(rows):
        for i in range(per):
            if i < sh:
                table[r, i] = perm[i]
            elif (r + i) % 4 != 1 and nxt < len(perm):
                table[r, i] = perm[nxt]
                nxt += 1
    st["table"] = table.to(DEV)
    st["counts"] = torch.full((rows,), per, dtype=torch.int32, device=DEV)
    return st


# ---------------------------------------------------------------------------------------
# The operators

def _gather(st, rows):
    """K and V [rows][kv][positions][dim] of the listed rows' page tables, FP32."""
    t = st["table"][rows].long()
    blocks = st["pool"][1][t]  # [rows][pages][2][kv][P][dim]
    r, n, _, kv, P, dim = blocks.shape
    k = blocks[:, :, 0].permute(0, 2, 1, 3, 4).reshape(r, kv, n * P, dim).float()
    v = blocks[:, :, 1].permute(0, 2, 1, 3, 4).reshape(r, kv, n * P, dim).float()
    return k, v


def _softmax_v(s, mask, v):
    """softmax over the visible keys of scores s, times v; zeros where nothing is visible."""
    s = torch.where(mask, s, torch.full_like(s, float("-inf")))
    m = s.amax(-1, keepdim=True)
    p = torch.where(mask, torch.exp(s - torch.where(m > float("-inf"), m, torch.zeros_like(m))), torch.zeros_like(s))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))


def _plain_decode(st):
    k, v = _gather(st, slice(None))
    rows, kv, n, dim = k.shape
    j = torch.arange(n, device=DEV)
    length = st["lengths"].long()[:, None]
    mask = j < length
    if st["window"]:
        mask = mask & ((j < st["sinks"]) | (j >= length - st["window"]))
    mask = mask[:, None, None, :]
    v = torch.where(mask[:, 0, :, :, None], v, torch.zeros((), device=DEV))
    q = st["q"].float().view(rows, kv, -1, dim)
    s = torch.matmul(q, k.transpose(-1, -2)) * dim ** -0.5
    return _softmax_v(s, mask, v).view(rows, -1, dim).to(torch.bfloat16)


def _plain_prefill(st):
    out = torch.empty_like(st["q"])
    dim, kv = st["dim"], st["kv"]
    for r, (a, b) in enumerate(st["spans"]):
        k, v = _gather(st, slice(r, r + 1))
        k, v = k[0, :, :st["lens"][r]], v[0, :, :st["lens"][r]]
        first = st["lens"][r] - (b - a)
        for c in range(a, b, 2048):  # blocks of queries: the score matrix stays in memory's bounds
            d = min(b, c + 2048)
            pos = first + torch.arange(c - a, d - a, device=DEV)[:, None]
            # Only the keys that some query of the block can see.
            end = first + d - a
            j = torch.arange(end, device=DEV)
            if st["window"]:
                lo = max(0, first + c - a - st["window"] + 1)
                if lo > st["sinks"]:
                    j = torch.cat([j[:st["sinks"]], j[lo:]])
            mask = j <= pos
            if st["window"]:
                mask = mask & ((j < st["sinks"]) | (j > pos - st["window"]))
            q = st["q"][c:d].float().view(d - c, kv, -1, dim).permute(1, 2, 0, 3)
            s = torch.matmul(q, k[:, None, j].transpose(-1, -2)) * dim ** -0.5
            o = _softmax_v(s, mask, v[:, None, j])
            out[c:d] = o.permute(2, 0, 1, 3).reshape(d - c, -1, dim).to(torch.bfloat16)
    return out


def _plain_copy(st):
    pool, n = st["pool"], st["tokens"][0]
    pool[:, st["dst_d"], :, :, :n] = pool[:, st["src_d"], :, :, :n]
    return pool


def _plain_compact(st):
    pool, table = st["pool"], st["table"]
    pages = pool.shape[1]
    listed_pages = (torch.arange(table.shape[1], device=DEV) < st["counts"][:, None]) & (table >= 0)
    used = torch.zeros(pages + 1, dtype=torch.bool, device=DEV)
    used[torch.where(listed_pages, table, torch.full_like(table, pages)).long().view(-1)] = True
    used = used[:pages]
    count = used.sum()
    index = torch.arange(pages, device=DEV)
    src = index[used & (index >= count)]
    dst = index[~used & (index < count)]
    pool[:, dst] = pool[:, src]
    remap = torch.where(used, index, torch.full_like(index, -1))
    remap[src] = dst
    new = torch.where(listed_pages, remap[table.clamp(min=0).long()].to(torch.int32), table)
    return pool, new, remap.to(torch.int32), count.to(torch.int32).view(1)


def run(state):
    st, op = state, state["op"]
    if own:
        yar = _package()
        if op == "decode":
            return yar.kv_attn_decode(st["pool"], 1, st["table"], st["lengths"], st["q"], window=st["window"],
                                      sinks=st["sinks"], max_length=st["max_length"])
        if op == "prefill":
            return yar.kv_attn_prefill(st["pool"], 1, st["table"], st["lengths"], st["offsets"], st["q"],
                                       window=st["window"], sinks=st["sinks"])
        if op == "copy":
            yar.kv_copy_pages(st["pool"], st["src"], st["dst"], tokens=st["tokens"])
            return st["pool"]
        new, remap, used = yar.kv_compact(st["pool"], st["table"], st["counts"])
        return st["pool"], new, remap, used
    return {"decode": _plain_decode, "prefill": _plain_prefill, "copy": _plain_copy, "compact": _plain_compact}[op](st)


# ---------------------------------------------------------------------------------------
# What a pass cannot do without

def work(case):
    kv, dim, P = case["kv"], case["dim"], case["page"]
    token = kv * dim * 2 * 2  # one position's K and V of one layer
    if case["op"] == "decode":
        seen = sum(_visible(x, case["window"], case["sinks"]) for x in _lengths(case))
        ends = 2 * case["rows"] * case["heads"] * dim * 2
        return {"bytes": seen * token + ends, "flops": 4 * seen * case["heads"] * dim}
    if case["op"] == "prefill":
        pairs = keys = total = 0
        for n, c in _chunks(case):
            pairs += sum(_visible(p + 1, case["window"], case["sinks"]) for p in range(c, c + n))
            keys += n + c if not case["window"] else min(n + c, n - 1 + case["window"] + case["sinks"])
            total += n
        return {"bytes": keys * token + 2 * total * case["heads"] * dim * 2, "flops": 4 * pairs * case["heads"] * dim}
    if case["op"] == "copy":
        return {"bytes": 2 * case["layers"] * case["pairs"] * case["tokens"] * token, "flops": 0}
    # The expected number of used pages behind the used count, moved once each.
    own_pages = sum((r + i) % 4 != 1 for r in range(case["rows"]) for i in range(case["shared"], case["per_row"]))
    used = min(case["pages"], case["shared"] + own_pages)
    moved = used * (case["pages"] - used) / case["pages"]
    return {"bytes": int(2 * moved * case["layers"] * P * token) + 8 * case["rows"] * case["per_row"], "flops": 0}


# ---------------------------------------------------------------------------------------
# The definition in 64 bits, one row (and one page) at a time

def _exact_rows(st, spans, lens):
    pool, dim, P = st["pool"][1], st["dim"], st["page"]
    group = st["heads"] // st["kv"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    for r, (a, b) in enumerate(spans):
        if lens[r] <= 0:
            continue
        ids = st["table"][r, :(lens[r] + P - 1) // P].long()
        keys = torch.cat([pool[i, 0] for i in ids], dim=1)[:, :lens[r]].double()  # [kv][n][dim]
        vals = torch.cat([pool[i, 1] for i in ids], dim=1)[:, :lens[r]].double()
        for c in range(a, b, 512):
            d = min(b, c + 512)
            first = lens[r] - (b - a) + (c - a)
            at = torch.arange(first, first + d - c, device=DEV).view(-1, 1)
            j = torch.arange(lens[r], device=DEV).view(1, -1)
            hidden = j > at
            if st["window"]:
                hidden |= (j >= st["sinks"]) & (at - j >= st["window"])
            lo, hi = 0, min(lens[r], first + d - c)
            if st["window"] and not st["sinks"]:
                lo = max(0, first - st["window"] + 1)
            for h in range(st["heads"]):
                x = st["q"][c:d, h].double() @ keys[h // group, lo:hi].T / dim ** 0.5
                x = x.masked_fill(hidden[:, lo:hi], float("-inf"))
                out[c:d, h] = torch.softmax(x, -1) @ vals[h // group, lo:hi]
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "decode":
        return _exact_rows(st, [(r, r + 1) for r in range(case["rows"])], st["lengths"].tolist())
    if case["op"] == "prefill":
        return _exact_rows(st, st["spans"], st["lens"])
    pool = st["pool"]
    if case["op"] == "copy":
        old = {s: pool[:, s].clone() for s in set(st["src"])}
        for s, d, n in zip(st["src"], st["dst"], st["tokens"]):
            pool[:, d, :, :, :n] = old[s][:, :, :, :n]
        return pool
    rows = [row[:n] for row, n in zip(st["table"].tolist(), st["counts"].tolist())]
    used = sorted({p for row in rows for p in row if p >= 0})
    holes = sorted(set(range(len(used))) - set(used))
    tail = [p for p in used if p >= len(used)]
    remap = {p: p for p in used}
    for s, d in zip(tail, holes):
        pool[:, d] = pool[:, s]
        remap[s] = d
    new = st["table"].clone().cpu()
    for r, row in enumerate(rows):
        for i, p in enumerate(row):
            if p >= 0:
                new[r, i] = remap[p]
    return (pool, new, torch.tensor([remap.get(p, -1) for p in range(pool.shape[1])], dtype=torch.int32),
            torch.tensor([len(used)], dtype=torch.int32))
