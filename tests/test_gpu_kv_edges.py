"""The paged-cache operators where calls are not alike: page tables wider than their rows, streams
other than the tensors' own, offsets that are wrong, weights that one key dominates, captured calls
on two streams. Against the definition in 64 bits, with the tolerance derived in
test_gpu_kv_ops.py."""
import numpy as np
import pytest

from tests.conftest import load_package
from tests.test_gpu_kv_ops import P_ROUND, Cache, queries

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def yar():
    return load_package()


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def definition(torch, c, q64, row, first, scale, window, sinks, round_p):
    """(result, tolerance) [n][heads][dim] of a row's queries at positions first, first + 1, ..: what
    Cache.attend gives for one query, for all of them at once."""
    n, heads, dim = q64.shape
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
    group = heads // c.kv
    q, k, v = dev(q64), dev(c.k[row]), dev(c.v[row])
    k, v = (x.repeat_interleave(group, 0) for x in (k, v))  # [heads][positions][dim]
    pos = first + torch.arange(n, device="cuda")[:, None]
    j = torch.arange(c.lens[row], device="cuda")[None]
    seen = j <= pos
    if window:
        seen &= (j < sinks) | (j > pos - window)
    seen = seen[:, None]
    none = ~seen.any(-1, keepdim=True)
    s = torch.einsum("nhd,hjd->nhj", q, k) * scale
    s = torch.where(seen, s, -torch.inf)
    big = torch.where(seen, torch.einsum("nhd,hjd->nhj", q.abs(), k.abs()) * scale, 0.0).amax(-1, keepdim=True)
    p = torch.where(none, 0.0, torch.exp(s - torch.where(none, 0.0, s.amax(-1, keepdim=True))))
    p = p / torch.where(none, 1.0, p.sum(-1, keepdim=True))
    out, a = torch.einsum("nhj,hjd->nhd", p, v), torch.einsum("nhj,hjd->nhd", p, v.abs())
    off = torch.expm1(4 * (dim + 6) * 2.0 ** -24 * big) + 2.0 ** -18 + round_p
    return out, torch.where(none, 0.0, off * a * (1 + 2.0 ** -8) + 2.0 ** -8 * out.abs() + 1e-30)


def check(torch, got, want, tol):
    assert torch.isfinite(got).all()
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3].tolist())


def widened(torch, c, positions):
    """The cache's page table with room for `positions` positions a row: entries that no call may
    read point outside of the pool."""
    rows, per = c.table.shape
    table = torch.full((rows, max(per, positions // c.page)), 1 << 30, dtype=torch.int32, device="cuda")
    table[:, :per] = c.table
    return table


def prompts(yar, torch, ns, before, kv, group, dim, page, positions, window=0, sinks=0, repeats=4):
    """A batch of prompts in a table of `positions` positions a row: every query against the
    definition, and the same bits from a cold L2, from other memory and again."""
    c = Cache(torch, [n + b for n, b in zip(ns, before)], kv, dim, page, seed=ns[0] + dim, window=window, sinks=sinks,
              first_pos=before)
    table = widened(torch, c, positions)
    offs = np.concatenate([[0], np.cumsum(ns)])
    q, q64 = queries(torch, int(offs[-1]), kv * group, dim, ns[0])
    d_offs = torch.tensor(offs, dtype=torch.int32, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    cold = torch.empty(192 << 20, dtype=torch.uint8, device="cuda")  # larger than the L2
    first = None
    for i in range(repeats):
        mine = q.clone()
        cold.fill_(i)
        got = yar.kv_attn_prefill(c.pool, 1, table, c.lengths, d_offs, mine, window=window, sinks=sinks, error=err)
        if first is None:
            first = got
            for r, (n, b) in enumerate(zip(ns, before)):
                if n:
                    want, tol = definition(torch, c, q64[offs[r]:offs[r + 1]], r, b, dim ** -0.5, window, sinks,
                                           P_ROUND["prefill"])
                    check(torch, got[offs[r]:offs[r + 1]], want, tol)
        assert torch.equal(got, first)
    assert err.item() == 0


HEADS = [(2, 1, 64), (2, 2, 64), (2, 4, 64), (2, 8, 64), (2, 16, 64), (2, 3, 64), (2, 1, 128), (2, 2, 128), (2, 4, 128),
         (2, 8, 128), (2, 16, 128), (2, 3, 128), (8, 2, 128)]


@pytest.mark.parametrize("kv,group,dim", HEADS)
@pytest.mark.parametrize("positions", [1024, 4096])
def test_short_prompts_in_wide_tables(yar, torch, kv, group, dim, positions):
    """The split along the keys follows the table's width: most blocks of a cluster have no key
    of such a prompt, or keys that one half of the block's queries does not see."""
    for n in (1, 40, 64, 100, 200, 512):
        prompts(yar, torch, [n], [0], kv, group, dim, 64, positions)


@pytest.mark.parametrize("n,window,sinks", [(640, 0, 0), (1000, 0, 0), (1184, 0, 0), (700, 1000, 4), (1024, 1000, 4),
                                            (1024, 640, 70)])
@pytest.mark.parametrize("page,positions", [(64, 0), (256, 4096)])
def test_first_chunks_of_a_prompt(yar, torch, n, window, sinks, page, positions):
    prompts(yar, torch, [n], [0], 8, 2, 128, page, positions, window, sinks)


@pytest.mark.parametrize("ns,before", [([1, 1300], [0, 0]), ([64, 1], [0, 1400]), ([3, 5, 40], [0, 2000, 0]),
                                       ([0, 1, 130], [0, 0, 1500]), ([127, 128, 129], [1, 0, 1500])])
@pytest.mark.parametrize("kv,group,dim", [(2, 1, 64), (2, 2, 128), (1, 16, 128), (2, 3, 128)])
def test_short_rows_beside_long_ones(yar, torch, ns, before, kv, group, dim):
    for positions in (0, 4096):
        prompts(yar, torch, ns, before, kv, group, dim, 32, positions)
    prompts(yar, torch, ns, before, kv, group, dim, 32, 4096, window=1300, sinks=5)


def memory_of(torch, t):
    """The stream whose memory the allocator made the tensor's storage."""
    at = t.data_ptr()
    for s in torch.cuda.memory_snapshot():
        if s["address"] <= at < s["address"] + s["total_size"]:
            return s["stream"]
    raise AssertionError("not the allocator's memory")


def test_results_on_a_given_stream_are_its_memory(yar, torch):
    """What a call allocates belongs to the stream that writes it; ones that the caller brings are
    used as they are, and without a stream the current one's memory is taken."""
    c = Cache(torch, [700, 90], 2, 64, 16, seed=23)
    q, _ = queries(torch, 2, 4, 64, 6)
    wide = torch.cat([q, q], dim=1)[:, :4]  # (rows that are not contiguous to each other)
    offs = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    counts = torch.tensor([44, 6], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    want = yar.kv_attn_decode(c.pool, 1, c.table, c.lengths, q), yar.kv_attn_prefill(c.pool, 1, c.table, c.lengths, offs, q)
    torch.cuda.synchronize()
    here = memory_of(torch, q)
    for stream, home in ((side.cuda_stream, side.cuda_stream), (None, here), (0, 0),
                         (torch.cuda.current_stream().cuda_stream, here)):
        for x in (q, wide):
            a = yar.kv_attn_decode(c.pool, 1, c.table, c.lengths, x, stream=stream)
            b = yar.kv_attn_prefill(c.pool, 1, c.table, c.lengths, offs, x, stream=stream)
            torch.cuda.synchronize()
            assert torch.equal(a, want[0]) and torch.equal(b, want[1])
            assert memory_of(torch, a) == memory_of(torch, b) == home
        pool = c.pool.clone()
        torch.cuda.synchronize()
        table, remap, used = yar.kv_compact(pool, c.table, counts, stream=stream)
        torch.cuda.synchronize()
        assert used.item() == 50 and {memory_of(torch, t) for t in (table, remap, used)} == {home}
        assert torch.equal(yar.kv_attn_decode(pool, 1, table, c.lengths, q), want[0])
    mine = torch.empty_like(q)
    torch.cuda.synchronize()
    assert yar.kv_attn_decode(c.pool, 1, c.table, c.lengths, q, out=mine, stream=side.cuda_stream) is mine
    side.synchronize()
    assert torch.equal(mine, want[0])


def offsets_case(rows, wrong):
    offs = [3 * i for i in range(rows + 1)]
    for at, value in wrong.items():
        offs[at] = value
    return offs


@pytest.mark.parametrize("offs", [[0, 60, 0, 60], [0, 5, 3, 8, 8, 12], [9, 70, 70, 2, 20, 60], [-4, 10, 12], [0, 99, 5, 20],
                                  offsets_case(150, {3: 200, 4: 3}), offsets_case(300, {140: 1, 141: 2}),
                                  offsets_case(300, {127: -1, 200: 901}), offsets_case(400, {131: 1200, 390: 100})])
@pytest.mark.parametrize("group", [2, 3])
def test_rows_behind_wrong_offsets(yar, torch, offs, group):
    """A row is skipped when its offsets are wrong or it starts before an earlier offset; every other
    row has its result, and no query that belongs to none is written."""
    rows, n = len(offs) - 1, 75 if len(offs) < 10 else 3 * (len(offs) - 1)
    c = Cache(torch, [100] * rows, 2, 64, 32, seed=rows)
    q, q64 = queries(torch, n, 2 * group, 64, rows)
    out = torch.full_like(q, 7.0)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    yar.kv_attn_prefill(c.pool, 1, c.table, c.lengths, torch.tensor(offs, dtype=torch.int32, device="cuda"), q, out=out,
                        error=err)
    assert err.item() == 4
    written = torch.zeros(n, dtype=torch.bool, device="cuda")
    for r, (a, b) in enumerate(zip(offs, offs[1:])):
        if not 0 <= a <= b <= n or a < max(offs[:r + 1]):
            continue
        assert not written[a:b].any()
        written[a:b] = True
        want, tol = definition(torch, c, q64[a:b], r, 100 - (b - a), 64 ** -0.5, 0, 0, P_ROUND["prefill"])
        check(torch, out[a:b], want, tol)
    assert (out[~written] == 7).all()


def test_a_short_row_in_a_very_wide_table(yar, torch):
    """A table of 2^24 pages a row, of which the first 7 are meant, in a tensor that ends with the
    row: the result of a narrow table, in about its time (the table is not walked)."""
    c = Cache(torch, [100], 2, 128, 16, seed=24)
    q, _ = queries(torch, 1, 4, 128, 7)
    table = torch.full((1, 1 << 24), 1 << 30, dtype=torch.int32, device="cuda")
    table[:, :c.table.shape[1]] = c.table

    def call(t):
        return yar.kv_attn_decode(c.pool, 1, t, c.lengths, q, max_length=100)

    def us(t, n=50):
        times = []
        for _ in range(5):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(n):
                call(t)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b) * 1e3 / n)
        return min(times)

    assert torch.equal(call(table), call(c.table))
    narrow, wide = us(c.table), us(table)
    print(f"narrow {narrow:.1f} us, wide {wide:.1f} us")
    assert wide <= 3 * narrow + 10


def test_compaction_into_a_table_beside_the_old_one(yar, torch):
    """Both tables as columns of one tensor, either side first."""
    pool = torch.arange(8, device="cuda").view(1, 8, 1, 1, 1, 1).expand(1, 8, 2, 1, 16, 64).bfloat16().contiguous()
    counts = torch.tensor([3, 2], dtype=torch.int32, device="cuda")
    for old, new in ((slice(0, 3), slice(3, 6)), (slice(3, 6), slice(0, 3)), (slice(0, 3), slice(4, 7))):
        both = torch.full((2, 7), -9, dtype=torch.int32, device="cuda")
        both[:, old] = torch.tensor([[7, 0, 5], [3, 7, 6]], dtype=torch.int32)
        mine = pool.clone()
        out, remap, used = yar.kv_compact(mine, both[:, old], counts, out=both[:, new])
        assert used.item() == 4 and both[:, new].tolist() == [[2, 0, 1], [3, 2, 6]]
        assert both[:, old].tolist() == [[7, 0, 5], [3, 7, 6]]
        assert mine[0, :4, 0, 0, 0, 0].tolist() == [0, 5, 7, 3]
    with pytest.raises(yar.YarError):
        yar.kv_compact(pool, both[:, 0:3], counts, out=both[:, 1:4])


@pytest.mark.parametrize("dim,kv,group,n", [(128, 2, 2, 300), (64, 1, 3, 200), (128, 8, 2, 1500)])
def test_keys_that_carry_the_weight(yar, torch, dim, kv, group, n):
    """Every 50th key is 3 to 7 (in units of log2) above the ones before it, less than makes the
    running maximum follow, so that the dominating weight is not a power of two: the weights' rounding
    does not average out, and the result stays within its tolerance (one rounding of the weights, one
    of the result)."""
    c = Cache(torch, [n], kv, dim, 64, seed=25, spread=0.05)
    rng = np.random.default_rng(26)
    unit = np.sign(rng.standard_normal((kv, dim)))
    level = 0.0
    for j in range(0, n, 50):
        level += 3 + 4 * rng.random()
        # q = unit (plus noise) below, so that this key scores level x ln 2
        k = torch.from_numpy(unit * level * np.log(2) / dim ** 0.5).bfloat16()
        c.k[0][:, j] = k.double().numpy()
        c.pool[1, int(c.table[0, j // 64]), 0, :, j % 64] = k.cuda()
    noise = rng.standard_normal((n, kv * group, dim)) * 0.02
    q = torch.from_numpy(unit.repeat(group, 0)[None] + noise).bfloat16()
    offs = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    for window, sinks in ((0, 0), (90, 3)):
        got = yar.kv_attn_prefill(c.pool, 1, c.table, c.lengths, offs, q.cuda(), window=window, sinks=sinks)
        want, tol = definition(torch, c, q.double().numpy(), 0, 0, dim ** -0.5, window, sinks, P_ROUND["prefill"])
        check(torch, got, want, tol)
        one = yar.kv_attn_decode(c.pool, 1, c.table, c.lengths, q[-1:].cuda(), window=window, sinks=sinks)
        want, tol = definition(torch, c, q[-1:].double().numpy(), 0, n - 1, dim ** -0.5, window, sinks, P_ROUND["decode"])
        check(torch, one, want, tol)


@pytest.mark.parametrize("dim,window,sinks,positions", [(128, 0, 0, 0), (64, 90, 3, 0), (128, 300, 0, 0), (128, 0, 0, 4096),
                                                        (64, 700, 5, 1024)])
def test_queries_that_do_not_see_a_value_keep_their_results(yar, torch, dim, window, sinks, positions):
    """Values that are not finite: in K, what does not see them keeps every bit; in V, what does not see
    them stays within the tolerance of the definition without them (the sums are formed again, key by
    key, beside one), in the heads that share the value's KV head too."""
    n, heads = 400, 4
    c = Cache(torch, [n], 2, dim, 64, seed=31)
    table = widened(torch, c, positions)
    q, q64 = queries(torch, n, heads, dim, 8)
    offs = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    want, tol = definition(torch, c, q64, 0, 0, dim ** -0.5, window, sinks, P_ROUND["prefill"])
    clean = yar.kv_attn_prefill(c.pool, 1, table, c.lengths, offs, q, window=window, sinks=sinks)
    check(torch, clean, want, tol)
    for at in (0, 63, 64, 130, 257, 317, 399):
        pos = torch.arange(n, device="cuda")
        sees = (pos >= at) & ((pos - window < at) | (at < sinks) if window else True)
        for what, value in ((0, float("nan")), (0, float("inf")), (1, float("nan")), (1, float("-inf"))):
            pool = c.pool.clone()
            pool[1, int(c.table[0, at // 64]), what, 0, at % 64, 7] = value
            got = yar.kv_attn_prefill(pool, 1, table, c.lengths, offs, q, window=window, sinks=sinks)
            assert torch.equal(got[:, 2:], clean[:, 2:])
            if what == 0:
                assert torch.equal(got[~sees], clean[~sees])
            else:
                check(torch, got[~sees], want[~sees], tol[~sees])
                assert not torch.isfinite(got[sees][:, :2, 7].float()).any()
                rest = torch.arange(dim, device="cuda") != 7
                check(torch, got[..., rest], want[..., rest], tol[..., rest])


def test_graphs_of_all_calls_on_two_streams(yar, torch):
    """Two graphs, each of copies, both forms of attention and compaction on a pool and buffers of its
    own, replayed at the same time on two streams, on new queries each time; a workspace each."""
    def make(seed, window):
        c = Cache(torch, [6000, 150, 60], 2, 128, 64, seed=seed)
        counts = torch.tensor([94, 3, 1], dtype=torch.int32, device="cuda")
        return dict(c=c, counts=counts, pool=c.pool.clone(), table=torch.empty_like(c.table), window=window,
                    q=queries(torch, 3, 4, 128, seed)[0], offs=torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda"),
                    ws=torch.empty(yar.kv_attn_decode_workspace(4, 2, 128), dtype=torch.uint8, device="cuda"),
                    pages=[int(p) for p in c.table[0, :3]],
                    spare=sorted(set(range(c.pool.shape[1])) - set(c.table.flatten().tolist()))[:3])

    def run(s):
        c, kw = s["c"], dict(window=s["window"], sinks=2)
        s["pool"].copy_(c.pool)
        yar.kv_copy_pages(s["pool"], s["pages"], s["spare"], tokens=[1, 20, 64])
        a = yar.kv_attn_decode(s["pool"], 1, c.table, c.lengths, s["q"], workspace=s["ws"], **kw)
        b = yar.kv_attn_prefill(s["pool"], 1, c.table, c.lengths, s["offs"], a, **kw)
        new, remap, used = yar.kv_compact(s["pool"], c.table, s["counts"], out=s["table"])
        return a, b, yar.kv_attn_decode(s["pool"], 1, new, c.lengths, b, workspace=s["ws"], **kw), remap, used

    sets = [make(41, 0), make(42, 500)]
    for s in sets:
        run(s)  # (first calls outside of the capture)
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in sets]
    for s, stream in zip(sets, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            outs.append(run(s))
        graphs.append(g)
    for seed in range(6):
        for s in sets:
            s["q"].copy_(queries(torch, 3, 4, 128, 60 + seed)[0])
        torch.cuda.synchronize()
        for _ in range(3):
            for g, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    g.replay()
        torch.cuda.synchronize()
        for s, out in zip(sets, outs):
            keep = [x.clone() for x in out]
            for x, want in zip(keep, run(s)):
                assert torch.equal(x, want)
