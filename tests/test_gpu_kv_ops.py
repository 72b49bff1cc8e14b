"""The paged-cache operators against a plain implementation in 64 bits.

Attention tolerance, per output value. Let A = sum_j p_j |v_j| (p: the exact weights) and
S = max_j scale sum_d |q_d k_jd|.
* products of BF16 values are exact in FP32; a sum of D of them in FP32, in any order, and its
  scaling are off by at most (D + 2) 2^-24 S, and forming the exponent by 4 x 2^-24 S more, so
  each weight by a factor within exp(+-2 (D + 6) 2^-24 S); the weights' sum too (doubled);
* the exponential itself, and the sums over the keys in FP32 (partial sums of positive terms,
  rescaled per block): 2^-18 covers 2^-22 per exponential and 64 rounded blocks;
* the weights enter the second product as BF16 (off by 2^-8 each at most) in the prompt form,
  as two BF16 parts (2^-16) in the single-token form; some of the prompt form's exponentials
  come from a polynomial (2.6e-6 < 2^-18 off in a weight and in their sum);
* the result is rounded to BF16 once: 2^-8 of it.
"""
import math

import numpy as np
import pytest

from tests.conftest import load_package

pytestmark = pytest.mark.gpu

P_ROUND = {"decode": 2.0 ** -16, "prefill": 2.0 ** -8 + 2.0 ** -17}


@pytest.fixture(scope="module")
def yar():
    return load_package()


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def visible(length, pos, window, sinks):
    """Positions that a query at `pos` sees of `length` cached ones, by the definition."""
    j = np.arange(max(0, min(length, pos + 1)))
    return j[(j < sinks) | (j > pos - window)] if window else j


class Cache:
    """A pool of random values in shuffled pages: every value that no query may see (other
    layers, unlisted pages, slots behind a row's length) is NaN or infinite."""

    def __init__(self, torch, lens, kv=2, dim=64, page=16, seed=0, spread=1.0, window=0, sinks=0, first_pos=None):
        rng = np.random.default_rng(seed)
        self.lens, self.kv, self.dim, self.page = lens, kv, dim, page
        per = max(1, max((x + page - 1) // page for x in lens))
        pages = per * len(lens) + 3
        data = np.full((2, pages, 2, kv, page, dim), np.nan, np.float32)
        data[0] = np.inf
        perm = rng.permutation(pages)
        table = np.full((len(lens), per), -1, np.int64)
        self.k, self.v = [], []
        used = 0
        for r, n in enumerate(lens):
            k = rng.standard_normal((kv, max(n, 0), dim)).astype(np.float32) * spread
            v = rng.standard_normal((kv, max(n, 0), dim)).astype(np.float32)
            k, v = (torch.from_numpy(x).bfloat16().float().numpy() for x in (k, v))
            self.k.append(k.astype(np.float64)), self.v.append(v.astype(np.float64))
            first = n - 1 if first_pos is None else first_pos[r]
            hidden = max(0, first - window + 1) if window else 0  # positions before this one: only sinks are seen
            for i in range((n + page - 1) // page):
                a, b = i * page, min(n, (i + 1) * page)
                if a >= sinks and b <= hidden:
                    continue  # a freed page: -1 in the table
                table[r, i] = perm[used]
                used += 1
                data[1, table[r, i], 0, :, :b - a] = k[:, a:b]
                data[1, table[r, i], 1, :, :b - a] = v[:, a:b]
        self.pool = torch.from_numpy(data).bfloat16().cuda()
        self.table = torch.from_numpy(table.astype(np.int32)).cuda()
        self.lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")

    def attend(self, q, row, pos, scale, window, sinks, round_p):
        """(result, tolerance) [heads][dim] of one query in 64 bits."""
        heads = q.shape[0]
        group = heads // self.kv
        j = visible(self.lens[row], pos, window, sinks)
        out, tol = np.zeros(q.shape), np.zeros(q.shape)
        if j.size == 0:
            return out, tol
        for h in range(heads):
            k, v = self.k[row][h // group][j], self.v[row][h // group][j]
            s = scale * (k @ q[h])
            big = (scale * (np.abs(k) @ np.abs(q[h]))).max()
            p = np.exp(s - s.max())
            p /= p.sum()
            out[h] = p @ v
            a = p @ np.abs(v)
            off = math.expm1(4 * (self.dim + 6) * 2.0 ** -24 * big) + 2.0 ** -18 + round_p
            tol[h] = off * a * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(out[h]) + 1e-30
        return out, tol


def check(torch, got, want, tol):
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all()
    bad = np.abs(got - want) > tol
    assert not bad.any(), (int(bad.sum()), float((np.abs(got - want) / tol).max()))


def queries(torch, n, heads, dim, seed, spread=1.0):
    rng = np.random.default_rng(seed + 1000)
    q = torch.from_numpy((rng.standard_normal((n, heads, dim)) * spread).astype(np.float32)).bfloat16()
    return q.cuda(), q.double().numpy()


DECODE = [
    # lens, kv, group, dim, page, window, sinks
    ([1], 2, 2, 64, 16, 0, 0), ([1, 2, 0, 5], 8, 2, 128, 256, 0, 0), ([15, 16, 17], 1, 1, 64, 16, 0, 0),
    ([63, 64, 65, 127, 128, 129], 2, 2, 128, 64, 0, 0), ([255, 256, 257], 8, 2, 128, 256, 0, 0),
    ([1000, 0, 33, 777], 2, 7, 64, 32, 0, 0), ([513], 8, 2, 128, 256, 0, 0), ([3000], 1, 16, 128, 128, 0, 0),
    ([4100, 1], 4, 3, 128, 16, 0, 0), ([700, 20, 64, 1], 2, 8, 64, 16, 1, 0), ([700, 20, 64, 1], 2, 4, 64, 16, 17, 3),
    ([900, 300, 0, 301, 299], 2, 2, 128, 256, 300, 4), ([2000, 1999], 1, 9, 128, 32, 100, 70),
    ([500], 2, 2, 64, 16, 64, 0), ([600, 601], 2, 2, 128, 4096, 37, 600), ([90] * 40, 2, 1, 64, 64, 50, 1),
    ([9001], 2, 2, 128, 256, 2048, 4),
]


@pytest.mark.parametrize("lens,kv,group,dim,page,window,sinks", DECODE)
def test_decode_matches_the_definition(yar, torch, lens, kv, group, dim, page, window, sinks):
    c = Cache(torch, lens, kv, dim, page, seed=len(lens) + lens[0], window=window, sinks=sinks)
    q, q64 = queries(torch, len(lens), kv * group, dim, lens[0])
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = yar.kv_attn_decode(c.pool, 1, c.table, c.lengths, q, window=window, sinks=sinks, error=err)
    pairs = [c.attend(q64[r], r, n - 1, dim ** -0.5, window, sinks, P_ROUND["decode"]) for r, n in enumerate(lens)]
    check(torch, got, np.stack([p[0] for p in pairs]), np.stack([p[1] for p in pairs]))
    assert err.item() == 0
    # A bound of the lengths changes the split, not the result beyond rounding.
    hint = yar.kv_attn_decode(c.pool, 1, c.table, c.lengths, q, window=window, sinks=sinks, max_length=max(1, max(lens)))
    check(torch, hint, np.stack([p[0] for p in pairs]), np.stack([p[1] for p in pairs]))
    hint = yar.kv_attn_decode(c.pool, 1, c.table, c.lengths, q, window=window, sinks=sinks, max_length=1)
    check(torch, hint, np.stack([p[0] for p in pairs]), np.stack([p[1] for p in pairs]))


@pytest.mark.parametrize("lens,kv,group,dim,page,window,sinks", [
    ([24000], 2, 2, 128, 256, 0, 0), ([6000, 1, 0, 12001], 1, 16, 128, 16, 0, 0), ([9000], 2, 3, 64, 64, 5000, 100)])
def test_long_rows_split_into_parts(yar, torch, lens, kv, group, dim, page, window, sinks):
    """With a workspace (rows split over the whole GPU, joined by a second kernel), with one
    that is too small, and without (a cluster)."""
    c = Cache(torch, lens, kv, dim, page, seed=3, window=window, sinks=sinks)
    q, q64 = queries(torch, len(lens), kv * group, dim, 4)
    pairs = [c.attend(q64[r], r, n - 1, dim ** -0.5, window, sinks, P_ROUND["decode"]) for r, n in enumerate(lens)]
    want, tol = np.stack([p[0] for p in pairs]), np.stack([p[1] for p in pairs])
    size = yar.kv_attn_decode_workspace(kv * group, kv, dim)
    dirty = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    guard = torch.full((size + 64,), 255, dtype=torch.uint8, device="cuda")
    for ws in (None, dirty, guard[:size], dirty[:size - 4]):
        got = yar.kv_attn_decode(c.pool, 1, c.table, c.lengths, q, window=window, sinks=sinks, workspace=ws)
        check(torch, got, want, tol)
    assert (guard[size:] == 255).all()
    got = yar.kv_attn_decode(c.pool, 1, c.table, c.lengths, q, window=window, sinks=sinks,
                             stream=torch.cuda.current_stream().cuda_stream)
    check(torch, got, want, tol)


PREFILL = [
    # queries per row, cached before them, kv, group, dim, page, window, sinks
    ([1], [0], 2, 2, 64, 16, 0, 0), ([77], [0], 2, 2, 64, 16, 0, 0), ([5, 0, 130], [0, 9, 3], 1, 1, 128, 256, 0, 0),
    ([127, 128, 129], [1, 0, 500], 2, 2, 128, 64, 0, 0), ([300], [700], 8, 2, 128, 256, 0, 0),
    ([64, 1, 200], [0, 1000, 63], 2, 3, 64, 32, 0, 0), ([260], [0], 1, 8, 128, 16, 0, 0),
    ([200, 40], [0, 400], 2, 2, 128, 256, 1, 0), ([200, 40], [0, 400], 2, 2, 64, 16, 17, 3),
    ([600], [0], 2, 2, 128, 256, 128, 4), ([150, 257], [900, 1], 2, 1, 128, 32, 100, 70),
    ([333], [1111], 1, 4, 64, 128, 200, 130), ([500], [0], 2, 7, 64, 64, 300, 0), ([520], [2000], 2, 2, 128, 256, 512, 4),
]


@pytest.mark.parametrize("ns,before,kv,group,dim,page,window,sinks", PREFILL)
def test_prefill_matches_the_definition(yar, torch, ns, before, kv, group, dim, page, window, sinks):
    lens = [n + b for n, b in zip(ns, before)]
    c = Cache(torch, lens, kv, dim, page, seed=lens[0], window=window, sinks=sinks, first_pos=before)
    offs = np.concatenate([[0], np.cumsum(ns)])
    q, q64 = queries(torch, int(offs[-1]), kv * group, dim, lens[0])
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = yar.kv_attn_prefill(c.pool, 1, c.table, c.lengths, torch.tensor(offs, dtype=torch.int32, device="cuda"), q,
                              window=window, sinks=sinks, error=err)
    want, tol = np.zeros(q64.shape), np.zeros(q64.shape)
    for r, (n, b) in enumerate(zip(ns, before)):
        for i in range(n):
            t = offs[r] + i
            want[t], tol[t] = c.attend(q64[t], r, b + i, dim ** -0.5, window, sinks, P_ROUND["prefill"])
    check(torch, got, want, tol)
    assert err.item() == 0


MANY = [
    # more pieces of work than a GPU has SMs: blocks take several in turn
    ([1 + 7 * i % 61 for i in range(45)], [13 * i % 300 for i in range(45)], 8, 2, 64, 16, 0, 0),
    ([1 + 7 * i % 61 for i in range(45)], [13 * i % 300 for i in range(45)], 8, 3, 64, 32, 37, 3),
    ([i * 5 % 4 for i in range(150)] + [700, 0, 3], [i * 11 % 90 for i in range(153)], 2, 4, 128, 32, 40, 5),
    ([4000], [100], 8, 2, 64, 64, 200, 70), ([900, 60], [0, 500], 8, 7, 128, 256, 0, 0),
    ([2 + 31 * i % 400 for i in range(20)], [0] * 20, 8, 16, 64, 16, 90, 20),
    ([2560], [6000], 8, 2, 64, 64, 0, 0),  # (halves of the keys, in more than one wave)
]


@pytest.mark.parametrize("ns,before,kv,group,dim,page,window,sinks", MANY)
def test_many_rows_and_long_prompts(yar, torch, ns, before, kv, group, dim, page, window, sinks):
    """First, middle and last query of every row against the definition; the same bits again; and a
    bad page or a value that is not finite in one row leaves the other rows' bits alone."""
    lens = [n + b for n, b in zip(ns, before)]
    c = Cache(torch, lens, kv, dim, page, seed=len(lens), window=window, sinks=sinks, first_pos=before)
    offs = np.concatenate([[0], np.cumsum(ns)])
    q, q64 = queries(torch, int(offs[-1]), kv * group, dim, lens[0])
    d_offs = torch.tensor(offs, dtype=torch.int32, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")

    def run(pool, table):
        err.zero_()
        return yar.kv_attn_prefill(pool, 1, table, c.lengths, d_offs, q, window=window, sinks=sinks, error=err)

    got = run(c.pool, c.table)
    assert err.item() == 0
    for r, n in enumerate(ns):
        for i in sorted({0, n // 2, n - 1} if n else ()):
            t = offs[r] + i
            want, tol = c.attend(q64[t], r, before[r] + i, dim ** -0.5, window, sinks, P_ROUND["prefill"])
            check(torch, got[t], want, tol)
    assert torch.equal(run(c.pool, c.table), got)
    row = len(ns) // 2 if ns[len(ns) // 2] else int(np.argmax(ns))
    mine = torch.zeros(int(offs[-1]), dtype=torch.bool, device="cuda")
    mine[offs[row]:offs[row + 1]] = True
    last = (lens[row] - 1) // page  # the page of the row's last position
    table = c.table.clone()
    table[row, last] = -1
    bad = run(c.pool, table)
    assert err.item() == 1 and torch.equal(bad[~mine], got[~mine]) and torch.isfinite(bad.float()).all()
    assert not torch.equal(bad[mine], got[mine])
    pool = c.pool.clone()
    pool[1, int(c.table[row, last]), 1, 0, (lens[row] - 1) % page, 5] = float("inf")  # seen by its last query only
    far = run(pool, c.table)
    assert err.item() == 0 and torch.equal(far[~mine], got[~mine])
    assert torch.isinf(far[offs[row + 1] - 1, :group, 5].float()).all()
    mine[offs[row + 1] - 1] = False
    assert torch.isfinite(far[mine].float()).all()


def test_rows_aligned_to_16_bytes(yar, torch):
    """q and out rows whose addresses are multiples of 16 bytes, not of 32."""
    for dim, heads in ((64, 4), (128, 6)):
        c = Cache(torch, [150, 30], 2, dim, 16, seed=12)
        offs = torch.tensor([0, 100, 130], dtype=torch.int32, device="cuda")
        q, _ = queries(torch, 130, heads, dim, 3)
        want = yar.kv_attn_prefill(c.pool, 1, c.table, c.lengths, offs, q)
        width = heads * dim
        qs, os_ = (torch.full((131 * (width + 8),), 7.0, device="cuda", dtype=torch.bfloat16) for _ in range(2))
        q2, out = (x[8:].as_strided((130, heads, dim), (width + 8, dim, 1), 8) for x in (qs, os_))
        q2.copy_(q)
        assert out.data_ptr() % 32 == 16
        yar.kv_attn_prefill(c.pool, 1, c.table, c.lengths, offs, q2, out=out)
        assert torch.equal(out, want)
        rest = torch.ones_like(os_, dtype=torch.bool)
        rest.as_strided(out.shape, out.stride(), 8)[:] = False
        assert (os_[rest] == 7).all()
        one = yar.kv_attn_decode(c.pool, 1, c.table, c.lengths, q[:2])
        os_.fill_(7.0)
        yar.kv_attn_decode(c.pool, 1, c.table, c.lengths, q2[:2], out=out[:2])
        assert torch.equal(out[:2], one) and (os_[rest] == 7).all()


def test_large_scores_and_a_given_scale(yar, torch):
    """Scores far from zero (a running maximum that moves, weights that vanish)."""
    for dim, spread, scale in ((128, 6.0, None), (64, 3.0, 0.7)):
        lens = [300, 41]
        c = Cache(torch, lens, 2, dim, 16, seed=3, spread=spread)
        q, q64 = queries(torch, 2, 4, dim, 5, spread)
        s = dim ** -0.5 if scale is None else scale
        got = yar.kv_attn_decode(c.pool, 1, c.table, c.lengths, q, scale=scale)
        pairs = [c.attend(q64[r], r, n - 1, s, 0, 0, P_ROUND["decode"]) for r, n in enumerate(lens)]
        check(torch, got, np.stack([p[0] for p in pairs]), np.stack([p[1] for p in pairs]))
        q, q64 = queries(torch, 60, 4, dim, 6, spread)
        got = yar.kv_attn_prefill(c.pool, 1, c.table, c.lengths, torch.tensor([0, 40, 60], dtype=torch.int32).cuda(), q,
                                  scale=scale)
        pairs = [c.attend(q64[t], 0 if t < 40 else 1, 260 + t if t < 40 else 21 + t - 40, s, 0, 0, P_ROUND["prefill"])
                 for t in range(60)]
        check(torch, got, np.stack([p[0] for p in pairs]), np.stack([p[1] for p in pairs]))


@pytest.mark.parametrize("dim,window,sinks", [(128, 0, 0), (64, 90, 3), (128, 300, 0)])
def test_values_that_are_not_finite_reach_only_the_queries_that_see_them(yar, torch, dim, window, sinks):
    """V rows holding infinities and NaN, keys with NaN: a query that does not see them is as
    without them (bit for bit), one that sees them gets what the sum gives."""
    n, heads = 400, 4
    c = Cache(torch, [n], 2, dim, 64, seed=31)
    q, _ = queries(torch, n, heads, dim, 8)
    offs = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    clean = yar.kv_attn_prefill(c.pool, 1, c.table, c.lengths, offs, q, window=window, sinks=sinks)
    last = yar.kv_attn_decode(c.pool, 1, c.table, c.lengths, q[-1:], window=window, sinks=sinks)
    # Positions all over a key tile, in tiles that most queries see whole and in edge tiles.
    for at in (270, 256, 257, 260, 261, 275, 2, 317, 399):
        page, slot = int(c.table[0, at // 64]), at % 64
        sees = torch.tensor([at in visible(n, i, window, sinks) for i in range(n)], device="cuda")
        assert 0 < sees.sum() < n or at == 2
        for what, value in (("v", float("inf")), ("v", float("nan")), ("k", float("nan")), ("k", float("inf"))):
            pool = c.pool.clone()
            pool[1, page, 0 if what == "k" else 1, 0, slot, 7] = value  # KV head 0: heads 0 and 1
            got = yar.kv_attn_prefill(pool, 1, c.table, c.lengths, offs, q, window=window, sinks=sinks)
            err = (got.float() - clean.float()).abs()
            assert torch.equal(got[:, 2:], clean[:, 2:])
            hidden = err[~sees][:, :2]  # recomputed sums may round differently
            assert torch.isfinite(hidden).all()
            assert (hidden <= 2.0 ** -6 * (clean[~sees][:, :2].float().abs() + 1)).all()
            seen = got[sees][:, :2].float()
            if what == "v":
                assert not torch.isfinite(seen[..., 7]).any()
                rest = torch.ones(dim, dtype=torch.bool)
                rest[7] = False
                assert torch.isfinite(seen[..., rest]).all()
            else:  # NaN scores, or infinite ones: +inf makes its weight NaN, -inf makes it vanish
                plus = torch.ones_like(seen[..., 0], dtype=torch.bool)
                if value == float("inf"):
                    plus = q[sees][:, :2, 7].float() >= 0
                assert torch.isnan(seen[plus]).all()
                assert torch.isfinite(seen[~plus]).all()
            one = yar.kv_attn_decode(pool, 1, c.table, c.lengths, q[-1:], window=window, sinks=sinks)
            assert torch.equal(one[:, 2:], last[:, 2:])
            if not sees[-1]:
                assert torch.equal(one, last)
            elif what == "v" or value != float("inf"):
                assert not torch.isfinite(one[0, :2].float()).all()


def test_strided_tensors_and_rows_behind_the_last(yar, torch):
    c = Cache(torch, [40, 90], 2, 64, 16, seed=8)
    wide = torch.randn(6, 9, 64, device="cuda").bfloat16()
    q = wide[:, 2:6]  # row stride 9 x 64
    out_wide = torch.full((6, 6, 64), 7.0, device="cuda", dtype=torch.bfloat16)
    table = torch.full((2, 11), 1 << 30, dtype=torch.int32, device="cuda")
    table[:, :c.table.shape[1]] = c.table
    tab = table[:, :c.table.shape[1]]
    dense = yar.kv_attn_decode(c.pool, 1, c.table, c.lengths, q[:2].contiguous())
    yar.kv_attn_decode(c.pool, 1, tab, c.lengths, q[:2], out=out_wide[:2, 1:5])
    assert torch.equal(out_wide[:2, 1:5], dense)
    assert (out_wide[2:] == 7).all() and (out_wide[:, 0] == 7).all() and (out_wide[:, 5] == 7).all()
    # Queries 1..4 belong to the two rows; 0 and 5 to none: left as they were.
    offs = torch.tensor([1, 3, 5], dtype=torch.int32, device="cuda")
    dense = yar.kv_attn_prefill(c.pool, 1, c.table, c.lengths, torch.tensor([0, 2, 4], dtype=torch.int32).cuda(),
                                q[1:5].contiguous())
    out_wide.fill_(7.0)
    yar.kv_attn_prefill(c.pool, 1, tab, c.lengths, offs, q, out=out_wide[:, 1:5])
    assert torch.equal(out_wide[1:5, 1:5], dense)
    assert (out_wide[0] == 7).all() and (out_wide[5] == 7).all()
    assert (out_wide[:, 0] == 7).all() and (out_wide[:, 5] == 7).all()


def test_queries_before_the_first_position_see_nothing(yar, torch):
    c = Cache(torch, [3, 0], 2, 64, 16, seed=4)
    q, q64 = queries(torch, 9, 4, 64, 2)
    got = yar.kv_attn_prefill(c.pool, 1, c.table, c.lengths, torch.tensor([0, 5, 9], dtype=torch.int32).cuda(), q)
    assert (got[:2] == 0).all() and (got[5:] == 0).all()
    for i in range(2, 5):
        want, tol = c.attend(q64[i], 0, i - 2, 0.125, 0, 0, P_ROUND["prefill"])
        check(torch, got[i], want, tol)


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 256)])
def test_bad_pages_lengths_and_offsets_are_reported_and_not_followed(yar, torch, dim, page):
    n = 3 * page
    c = Cache(torch, [n, n], 2, dim, page, seed=11)
    q, q64 = queries(torch, 2, 4, dim, 9)
    good = yar.kv_attn_decode(c.pool, 1, c.table, c.lengths, q)
    for bad in (-1, -5, c.pool.shape[1], 2 ** 31 - 1):
        table = c.table.clone()
        table[0, 1] = bad
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = yar.kv_attn_decode(c.pool, 1, table, c.lengths, q, error=err)
        assert err.item() == 1 and torch.equal(got[1], good[1])
        # The bad page's positions count as not visible.
        k, v = c.k[0], c.v[0]
        c.k[0], c.v[0] = (np.concatenate([x[:, :page], x[:, 2 * page:]], axis=1) for x in (k, v))
        c.lens[0] = 2 * page
        want, tol = c.attend(q64[0], 0, 2 * page - 1, dim ** -0.5, 0, 0, P_ROUND["decode"])
        _, tol_pre = c.attend(q64[0], 0, 2 * page - 1, dim ** -0.5, 0, 0, P_ROUND["prefill"])
        c.k[0], c.v[0], c.lens[0] = k, v, n
        check(torch, got[0], want, tol)
        err.zero_()
        offs = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
        pre = yar.kv_attn_prefill(c.pool, 1, table, c.lengths, offs, q, error=err)
        assert err.item() == 1
        check(torch, pre[0], want, tol_pre)
    # A length beyond the table is cut to the table's positions.
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    long = torch.tensor([n + 1, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    assert torch.equal(yar.kv_attn_decode(c.pool, 1, c.table, long, q, error=err), good)
    assert err.item() == 2
    err.zero_()
    pre = yar.kv_attn_prefill(c.pool, 1, c.table, c.lengths, torch.tensor([0, 1, 2], dtype=torch.int32).cuda(), q)
    assert torch.equal(yar.kv_attn_prefill(c.pool, 1, c.table, long, torch.tensor([0, 1, 2], dtype=torch.int32).cuda(),
                                           q, error=err), pre)
    assert err.item() == 2
    # Negative lengths: nothing cached.
    neg = torch.tensor([-3, -2 ** 31], dtype=torch.int32, device="cuda")
    assert (yar.kv_attn_decode(c.pool, 1, c.table, neg, q) == 0).all()
    # Offsets that decrease or pass the queries: those rows are skipped.
    for offs, kept in (([0, 1, 3], [0]), ([1, 0, 2], []), ([-1, 1, 2], [1])):
        err.zero_()
        out = torch.full_like(q, 7.0)
        yar.kv_attn_prefill(c.pool, 1, c.table, c.lengths, torch.tensor(offs, dtype=torch.int32).cuda(), q, out=out,
                            error=err)
        assert err.item() == 4, offs
        if kept:
            for t in range(2):
                assert torch.equal(out[t], pre[t] if t in kept else torch.full_like(out[t], 7.0)), (offs, t)


def test_layers_and_shared_pages(yar, torch):
    """Rows with the same table give the same bits, on either layer."""
    c = Cache(torch, [200], 2, 128, 64, seed=5)
    pool = c.pool.clone()
    pool[0] = pool[1]
    q, _ = queries(torch, 1, 4, 128, 1)
    table, lens = c.table.expand(3, -1).contiguous(), c.lengths.expand(3).contiguous()
    got = yar.kv_attn_decode(pool, 0, table, lens, q.expand(3, -1, -1).contiguous())
    one = yar.kv_attn_decode(pool, 1, c.table, c.lengths, q, max_length=0)
    for r in range(3):
        assert torch.equal(got[r], got[0])
    assert (got[0].float() - one[0].float()).abs().max() <= 2.0 ** -7 * one.float().abs().max()


def test_captured_calls_on_another_stream_replay(yar, torch):
    """Both forms, copies and compaction captured into one graph on a side stream; replayed on
    new inputs in the same buffers, two graphs interleaved."""
    c = Cache(torch, [150, 60], 2, 64, 16, seed=12)
    spare = torch.cat([c.pool, torch.zeros_like(c.pool)], dim=1).contiguous()
    q, _ = queries(torch, 2, 4, 64, 3)
    offs = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    n = c.pool.shape[1]
    src = [int(p) for p in c.table[0].tolist() if p >= 0][:2]
    yar.kv_attn_decode(spare, 1, c.table, c.lengths, q)  # first calls outside of the capture
    yar.kv_attn_prefill(spare, 1, c.table, c.lengths, offs, q)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for window in (0, 20):
        side = torch.cuda.Stream()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            a = yar.kv_attn_decode(spare, 1, c.table, c.lengths, q, window=window, sinks=2)
            b = yar.kv_attn_prefill(spare, 1, c.table, c.lengths, offs, q, window=window, sinks=2)
            yar.kv_copy_pages(spare, src, [n, n + 1])
        graphs.append(g), outs.append((a, b))
    for seed in (1, 2):
        q.copy_(queries(torch, 2, 4, 64, 40 + seed)[0])
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (a, b), window in zip(outs, (0, 20)):
            assert torch.equal(a, yar.kv_attn_decode(spare, 1, c.table, c.lengths, q, window=window, sinks=2))
            assert torch.equal(b, yar.kv_attn_prefill(spare, 1, c.table, c.lengths, offs, q, window=window, sinks=2))
        assert torch.equal(spare[:, n:n + 2].view(torch.int16), spare[:, src].view(torch.int16))


def test_calls_in_a_row_see_each_others_results(yar, torch):
    """Copies, both forms of attention and compaction on each other's results without a pause
    (a call may get ready while the one before it runs): as with a synchronization after each.
    The same captured, behind fills and copies and behind another stream's work."""
    c = Cache(torch, [4 * 64, 4 * 64, 900], 8, 64, 64, seed=44)
    q, _ = queries(torch, 3, 16, 64, 6)
    offs = torch.arange(4, dtype=torch.int32, device="cuda")
    counts = torch.tensor([4, 4, 15], dtype=torch.int32, device="cuda")
    a, b = c.table[0, :4].tolist(), c.table[1, :4].tolist()
    pool, dst = torch.empty_like(c.pool), torch.empty_like(c.table)

    def chain(sync, side=None):
        outs = []

        def step(x=None):
            if x is not None:
                outs.append(x)
            if sync:
                torch.cuda.synchronize()

        pool.copy_(c.pool)
        for n in range(3):
            if side is not None:  # the chain goes on behind another stream's work
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    dst.fill_(n)
                torch.cuda.current_stream().wait_stream(side)
            yar.kv_copy_pages(pool, a, b, tokens=[16 * (n + 1)] * 4), step()
            step(yar.kv_attn_decode(pool, 1, c.table, c.lengths, q))
            step(yar.kv_attn_prefill(pool, 1, c.table, c.lengths, offs, outs[-1]))
            step(yar.kv_attn_decode(pool, 1, c.table, c.lengths, outs[-1], window=100, sinks=3))
            table = yar.kv_compact(pool, c.table, counts, out=dst)[0]
            step()
            step(yar.kv_attn_prefill(pool, 1, table, c.lengths, offs, outs[-1]))
            pool.copy_(c.pool)
        return outs

    # Calls of more blocks than the GPU holds, each on the result of the one before.
    long = Cache(torch, [3000], 8, 64, 64, seed=45)
    q0, _ = queries(torch, 3000, 16, 64, 7)
    ends = torch.tensor([0, 3000], dtype=torch.int32, device="cuda")

    def rounds(sync):
        x = q0
        for n in range(4):
            x = yar.kv_attn_prefill(long.pool, 1, long.table, long.lengths, ends, x, window=300 * n, sinks=2)
            if sync:
                torch.cuda.synchronize()
            x = yar.kv_attn_decode(long.pool, 1, long.table.expand(3000, -1).contiguous(),
                                   long.lengths.expand(3000).contiguous(), x, window=40) + x
            if sync:
                torch.cuda.synchronize()
        return x

    want = rounds(True)
    for _ in range(3):
        assert torch.equal(rounds(False), want)

    want = chain(True)
    for _ in range(5):
        for got in zip(chain(False), want):
            assert torch.equal(*got)
    side = torch.cuda.Stream()
    for other in (None, side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = chain(False, other)
        for _ in range(3):
            for o in outs:
                o.zero_()
            g.replay()
            torch.cuda.synchronize()
            for got in zip(outs, want):
                assert torch.equal(*got)


def test_calls_on_two_streams_at_once(yar, torch):
    c = Cache(torch, [1500, 700, 900], 2, 128, 64, seed=13)
    q, _ = queries(torch, 3, 4, 128, 4)
    want = yar.kv_attn_decode(c.pool, 1, c.table, c.lengths, q)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(20):
        for s, o in zip(streams, outs):
            with torch.cuda.stream(s):
                o.append(yar.kv_attn_decode(c.pool, 1, c.table, c.lengths, q))
    torch.cuda.synchronize()
    for o in outs[0] + outs[1]:
        assert torch.equal(o, want)


def test_prompts_on_two_streams_at_once(yar, torch):
    """More pieces of work than SMs on either stream, and decode calls between them."""
    ns, before = [1 + 9 * i % 130 for i in range(40)], [17 * i % 400 for i in range(40)]
    c = Cache(torch, [n + b for n, b in zip(ns, before)], 8, 64, 16, seed=14)
    offs = torch.tensor(np.concatenate([[0], np.cumsum(ns)]), dtype=torch.int32, device="cuda")
    q, _ = queries(torch, int(offs[-1]), 16, 64, 4)
    one = q[:40].contiguous()
    want = yar.kv_attn_prefill(c.pool, 1, c.table, c.lengths, offs, q), yar.kv_attn_decode(c.pool, 1, c.table, c.lengths, one)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append((yar.kv_attn_prefill(c.pool, 1, c.table, c.lengths, offs, q),
                             yar.kv_attn_decode(c.pool, 1, c.table, c.lengths, one)))
    torch.cuda.synchronize()
    for got in outs:
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_offsets_beyond_32_bits(yar, torch):
    """A pool of 2.7 billion values (5.4 GB), used at its end: attention, copies and compaction."""
    kv, dim, page, pages = 8, 128, 64, 20600
    pool = torch.empty((1, pages, 2, kv, page, dim), dtype=torch.bfloat16, device="cuda")
    assert pool.numel() > 2 ** 31
    c = Cache(torch, [200], kv, dim, page, seed=17)
    small = c.table[0].long()
    far = torch.tensor([pages - 1, pages - 7, pages - 3, pages - 2], device="cuda")
    pool[0, far] = c.pool[1][small]
    table = far.to(torch.int32)[None].contiguous()
    q, _ = queries(torch, 1, 16, dim, 3)
    q9, _ = queries(torch, 9, 16, dim, 4)
    offs = torch.tensor([0, 9], dtype=torch.int32, device="cuda")
    want = yar.kv_attn_decode(c.pool, 1, c.table, c.lengths, q), yar.kv_attn_prefill(c.pool, 1, c.table, c.lengths, offs, q9)
    assert torch.equal(yar.kv_attn_decode(pool, 0, table, c.lengths, q), want[0])
    assert torch.equal(yar.kv_attn_prefill(pool, 0, table, c.lengths, offs, q9), want[1])
    new, remap, used = yar.kv_compact(pool, table, torch.tensor([4], dtype=torch.int32, device="cuda"))
    assert used.item() == 4 and sorted(new[0].tolist()) == [0, 1, 2, 3]
    assert torch.equal(yar.kv_attn_decode(pool, 0, new, c.lengths, q), want[0])
    yar.kv_copy_pages(pool, new[0].tolist(), [pages - 20, pages - 21, pages - 22, pages - 23])
    table = torch.tensor([[pages - 20, pages - 21, pages - 22, pages - 23]], dtype=torch.int32, device="cuda")
    assert torch.equal(yar.kv_attn_prefill(pool, 0, table, c.lengths, offs, q9), want[1])


def test_calls_from_two_threads(yar, torch):
    import threading
    c = Cache(torch, [500, 90], 2, 64, 16, seed=19)
    q, _ = queries(torch, 2, 4, 64, 5)
    offs = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    want = yar.kv_attn_decode(c.pool, 1, c.table, c.lengths, q), yar.kv_attn_prefill(c.pool, 1, c.table, c.lengths, offs, q)
    torch.cuda.synchronize()
    bad = []

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            got = [(yar.kv_attn_decode(c.pool, 1, c.table, c.lengths, q),
                    yar.kv_attn_prefill(c.pool, 1, c.table, c.lengths, offs, q)) for _ in range(50)]
            try:
                yar.kv_attn_decode(c.pool, 7, c.table, c.lengths, q)  # an error of this thread alone
                bad.append("layer")
            except yar.YarError as e:
                bad.extend([] if "layer" in e.message else [e.message])
        s.synchronize()
        bad.extend(1 for a, b in got if not (torch.equal(a, want[0]) and torch.equal(b, want[1])))

    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_host_memory_is_refused(yar, torch):
    c = Cache(torch, [20], 2, 64, 16, seed=1)
    q, _ = queries(torch, 1, 4, 64, 1)
    ok = (c.pool, 1, c.table, c.lengths, q)
    for i, bad in ((4, q.cpu()), (4, q.float()), (4, q[0]), (4, q[..., :32]), (4, q.transpose(1, 2)), (0, c.pool[0]),
                   (0, c.pool.cpu()), (0, c.pool.transpose(0, 1)), (2, c.table.long()), (2, c.table[0]), (2, c.table.cpu()),
                   (3, c.lengths[:0]), (3, c.lengths.long()), (3, c.lengths.cpu()), (4, torch.cat([q, q]))):
        with pytest.raises(ValueError):
            yar.kv_attn_decode(*ok[:i], bad, *ok[i + 1:])
    for out in (q.float(), q.cpu(), torch.cat([q, q]), q.transpose(1, 2)):
        with pytest.raises(ValueError):
            yar.kv_attn_decode(*ok, out=out)
        with pytest.raises(ValueError):
            yar.kv_attn_prefill(*ok[:4], torch.tensor([0, 1], dtype=torch.int32).cuda(), q, out=out)
    with pytest.raises(ValueError):
        yar.kv_attn_prefill(*ok[:4], torch.tensor([0], dtype=torch.int32).cuda(), q)
    with pytest.raises(ValueError):
        yar.kv_attn_decode(*ok, error=torch.zeros(1, device="cuda"))
    with pytest.raises(ValueError):  # (as many bytes as it says, but not in memory)
        yar.kv_attn_decode(*ok, workspace=torch.zeros(1, device="cuda").expand(1 << 20))
    for wrong in (dict(window=1 << 31), dict(window=2.5), dict(sinks=-1 << 40), dict(scale="x")):
        with pytest.raises(ValueError):
            yar.kv_attn_decode(*ok, **wrong)
    host = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    call = yar._KvAttn(yar._kv_pool(c.pool), yar._kv_rows(c.table, c.lengths), 0, 4, host.data_ptr(), 256, q.data_ptr(),
                       256, 0, 0, 0.125, None)
    st = yar.lib.yar_kv_attn_decode(bytes(call), 0, None, 0, None)
    assert st == yar.INVALID_INPUT and b"device memory" in yar.lib.yar_last_error()


@pytest.mark.parametrize("layers,kv,dim,page,pairs", [(1, 1, 64, 16, 1), (3, 2, 128, 64, 5), (2, 8, 128, 256, 3),
                                                       (2, 1, 64, 16, 300)])
def test_copy_pages(yar, torch, layers, kv, dim, page, pairs):
    g = torch.Generator().manual_seed(pairs)
    pages = 2 * pairs + 3
    pool = torch.randint(-32768, 32767, (layers, pages, 2, kv, page, dim), generator=g, dtype=torch.int32)
    pool = pool.to(torch.int16).cuda().view(torch.bfloat16)  # any bits, NaN patterns among them
    perm = torch.randperm(pages, generator=g).tolist()
    dst = perm[:pairs]
    src = [perm[pairs + i // 2] for i in range(pairs)]  # a page may be copied to several places
    tokens = [(i * 7) % (page + 1) for i in range(pairs)]
    for tok in (None, tokens):
        want = pool.view(torch.int16).clone()
        for i, (a, b) in enumerate(zip(src, dst)):
            t = page if tok is None else tok[i]
            want[:, b, :, :, :t] = want[:, a, :, :, :t]
        got = pool.clone()
        yar.kv_copy_pages(got, src, dst, tokens=tok)
        assert torch.equal(got.view(torch.int16), want)
    # Into a pool with another number of pages.
    other = torch.zeros((layers, pairs + 1, 2, kv, page, dim), dtype=torch.bfloat16, device="cuda")
    yar.kv_copy_pages(pool, src, list(range(pairs, 0, -1)), dst_pool=other)
    for i, a in enumerate(src):
        assert torch.equal(other[:, pairs - i].view(torch.int16), pool[:, a].view(torch.int16))
    assert (other[:, 0] == 0).all()


def plan(pages, table, counts):
    """The renamed table, remap, used count and moves by the definition."""
    used = sorted({int(p) for row, n in zip(table, counts) for p in row[:max(0, n)] if 0 <= p < pages})
    u = len(used)
    holes = [p for p in range(u) if p not in set(used)]
    moves = dict(zip([p for p in used if p >= u], holes))
    remap = np.full(pages, -1, np.int32)
    for p in used:
        remap[p] = moves.get(p, p)
    new = table.copy()
    for r, n in enumerate(counts):
        for i in range(max(0, min(n, table.shape[1]))):
            if 0 <= table[r, i] < pages:
                new[r, i] = remap[table[r, i]]
    return new, remap, u, moves


@pytest.mark.parametrize("pages,rows,per_row,kv,dim,page", [(5, 1, 3, 1, 64, 16), (64, 4, 9, 2, 64, 16),
                                                              (33, 5, 7, 8, 128, 64), (2500, 40, 30, 1, 64, 16),
                                                              (70000, 3, 50, 1, 64, 16), (40, 0, 1, 2, 64, 16)])
def test_compaction(yar, torch, pages, rows, per_row, kv, dim, page):
    rng = np.random.default_rng(pages)
    layers = 2 if pages < 10000 else 1
    pool = torch.randint(-32768, 32767, (layers, pages, 2, kv, page, dim), dtype=torch.int32, device="cuda")
    pool = pool.to(torch.int16).view(torch.bfloat16)
    table = rng.choice(pages, size=(rows, per_row), replace=rows * per_row > pages).astype(np.int32)
    table[rng.random(table.shape) < 0.2] = -1  # freed pages
    if rows > 1:
        table[1, :2] = table[0, :2]  # shared pages
    counts = rng.integers(0, per_row + 1, rows).astype(np.int32)
    new, remap, u, moves = plan(pages, table, counts)
    d = lambda x: torch.from_numpy(x).cuda()  # noqa: E731
    for in_place in (False, True):
        got, t, err = pool.clone(), d(table), torch.zeros(1, dtype=torch.int32, device="cuda")
        out, rm, used = yar.kv_compact(got, t, d(counts), out=t if in_place else None, error=err)
        assert err.item() == 0 and used.item() == u
        np.testing.assert_array_equal(rm.cpu().numpy(), remap)
        np.testing.assert_array_equal(out.cpu().numpy(), new)
        want = pool.view(torch.int16).clone()
        for a, b in moves.items():
            want[:, b] = want[:, a]
        assert torch.equal(got.view(torch.int16), want)
        if not in_place:
            assert torch.equal(t, d(table))


def test_compaction_reports_bad_entries_and_leaves_them(yar, torch):
    pool = torch.zeros((1, 8, 2, 1, 16, 64), dtype=torch.bfloat16, device="cuda")
    table = torch.tensor([[7, 8, -2, 2], [6, 2 ** 31 - 1, -1, 9]], dtype=torch.int32, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, remap, used = yar.kv_compact(pool, table, torch.tensor([4, 1], dtype=torch.int32, device="cuda"), error=err)
    assert err.item() == 1 and used.item() == 3
    assert out.tolist() == [[1, 8, -2, 2], [0, 2 ** 31 - 1, -1, 9]]
    assert remap.tolist() == [-1, -1, 2, -1, -1, -1, 0, 1]
    err.zero_()
    out, _, used = yar.kv_compact(pool, table, torch.tensor([-1, 99], dtype=torch.int32, device="cuda"), error=err)
    assert err.item() == 3 and used.item() == 1 and out.tolist()[0] == table.tolist()[0]


def test_forked_rows_attend_alike_and_survive_compaction(yar, torch):
    """A run as a server makes it: a prompt's row forked (full pages shared, the last page
    copied), one fork's window moved on (pages freed), the pool compacted: every attention
    over the renamed table gives the bits from before."""
    c = Cache(torch, [100], 2, 128, 16, seed=21)
    per = c.table.shape[1] + 2
    free = [p for p in range(c.pool.shape[1]) if p not in c.table[0].tolist()]
    pool = torch.cat([c.pool, torch.zeros_like(c.pool)], dim=1).contiguous()
    free += list(range(c.pool.shape[1], pool.shape[1]))
    first = c.table[0].tolist()
    table = torch.full((2, per), -1, dtype=torch.int32)
    table[0, :len(first)] = torch.tensor(first)
    table[1, :len(first)] = torch.tensor(first)
    fresh = free[-1]
    yar.kv_copy_pages(pool, [first[6]], [fresh], tokens=[4])  # 100 = 6 x 16 + 4
    table[1, 6] = fresh
    table = table.cuda()
    lens = torch.tensor([100, 100], dtype=torch.int32, device="cuda")
    q, _ = queries(torch, 1, 4, 128, 1)
    q = q.expand(2, -1, -1).contiguous()
    both = yar.kv_attn_decode(pool, 1, table, lens, q)
    assert torch.equal(both[0], both[1])
    seen = yar.kv_attn_decode(pool, 1, table, lens, q, window=30, sinks=3)
    offs = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    pre = yar.kv_attn_prefill(pool, 1, table, lens, offs, q, window=30, sinks=3)
    # Row 0 ends; row 1 frees what its window hides (positions 3..69: pages 1..3).
    table[0] = -1
    table[1, 1:4] = -1
    counts = torch.tensor([0, 7], dtype=torch.int32, device="cuda")
    new, remap, used = yar.kv_compact(pool, table, counts)
    assert used.item() == 4 and sorted(p for p in new[1].tolist() if p >= 0) == [0, 1, 2, 3]
    small = pool[:, :4].contiguous()
    lens = torch.tensor([0, 100], dtype=torch.int32, device="cuda")
    again = yar.kv_attn_decode(small, 1, new, lens, q, window=30, sinks=3)
    assert torch.equal(again[1], seen[1]) and (again[0] == 0).all()
    offs = torch.tensor([0, 0, 1], dtype=torch.int32, device="cuda")
    assert torch.equal(yar.kv_attn_prefill(small, 1, new, lens, offs, q[:1].contiguous(), window=30, sinks=3)[0], pre[1])
