"""Sliding-window attention of a session, and its rows as lists of cache pages (fork, cut back,
release behind the window, free, compaction), through the C ABI.

Tolerances: a windowed session against the CPU oracle with the same mask, on the pinned widths
with 2 layers: 1.5 times the bounds of the unwindowed model (0.0625 / 0.015, twice the radius
between two valid implementations), since its prefill rounds the attention weights to BF16 once
more (the same size of rounding as the output's own: sqrt(2) of it). Everything that only
moves pages changes no bit.
"""
import dataclasses
import os

import numpy as np
import pytest

from oracle import ar_oracle as ora
from tests.conftest import load_package

pytestmark = pytest.mark.gpu
MAX_ABS, REL = 1.5 * 0.0625, 1.5 * 0.015


def f(b):
    return ora.bf16_from_bits(b)


def rel_l2(a, b):
    return float(np.linalg.norm(a - b) / np.linalg.norm(b))


@pytest.fixture(scope="module")
def yar():
    return load_package()


@pytest.fixture(scope="module")
def wide(yar, synth, tmp_path_factory):
    """Pinned widths, 2 layers, 4096-row vocabulary; BF16 and 8-bit files of the same weights."""
    dims = dataclasses.replace(synth.PINNED, layers=2, vocab=4096, context=4096)
    d = str(tmp_path_factory.mktemp("window"))
    synth.write_converted(d, dims, seed=3, norm_std=0.1, precisions=("bf16", "8bit"))
    oracle = ora.OracleAR(synth.read_safetensors(os.path.join(d, "ar-bf16.safetensors")), dims, bf16=True)
    return yar.ARModel(d, any_dims=True), oracle, d


@pytest.fixture(scope="module")
def tiny(yar, tiny_dir, synth):
    oracle = ora.OracleAR(synth.read_safetensors(os.path.join(tiny_dir, "ar-bf16.safetensors")), synth.TINY, bf16=True)
    return yar.ARModel(tiny_dir, any_dims=True), oracle


def ids(seed, n):
    return np.random.default_rng(seed).integers(0, 4096, n).tolist()


def steps(s, rows, tokens):
    """Logits bits [step][row] of teacher-forced steps (the same token on every row)."""
    out = []
    for t in tokens:
        s.step(rows, [t] * len(rows), phase=None)
        out.append([s.logits(r, None) for r in rows])
    return np.array(out)


def oracle_run(oracle, prompt, forced, window, sinks):
    oracle.window, oracle.sinks = window, sinks
    try:
        logits, cache = oracle.prefill(prompt, len(prompt) + len(forced), None)
        return np.stack([logits] + [oracle.step(t, cache, None) for t in forced])
    finally:
        oracle.window, oracle.sinks = 0, 0


@pytest.mark.parametrize("n,window,sinks,page,chunk,rows", [
    (300, 64, 4, 256, 0, 1), (300, 100, 0, 64, 77, 2), (700, 129, 70, 256, 0, 1), (500, 200, 3, 16, 128, 2),
    (90, 1, 1, 256, 0, 1), (40, 300, 5, 256, 0, 1)])
@pytest.mark.parametrize("persistent", [True, False])
def test_windowed_session_vs_oracle(wide, n, window, sinks, page, chunk, rows, persistent):
    model, oracle, _ = wide
    prompt, forced = ids(n, n), ids(n + 1, 6)
    want = oracle_run(oracle, prompt, forced, window, sinks)
    s = model.session(max_rows=2, max_ctx=1024, page_tokens=page)
    s.set_persistent(persistent)
    s.set_window(window, sinks)
    for r in range(rows):
        s.reset(r, 1024)
        s.prefill(r, prompt, phase=None, chunk=chunk)
    got = [f(s.logits(0, None))] + [f(x[0]) for x in steps(s, list(range(rows)), forced)]
    got = np.stack(got)
    assert np.abs(got - want).max() <= MAX_ABS and rel_l2(got, want) <= REL
    if n > window + sinks:  # and the window matters: the whole context gives other logits
        full = oracle_run(oracle, prompt, forced[:1], 0, 0)
        assert rel_l2(want[:2], full) > 3 * REL


def test_windowed_small_model_vs_oracle(tiny):
    """head_dim 64 (per-operation decode, prefill by the paged kernel)."""
    model, oracle = tiny
    prompt, forced = ids(2, 150), ids(3, 8)
    want = oracle_run(oracle, prompt, forced, 50, 3)
    s = model.session(max_rows=1, max_ctx=192, page_tokens=16)
    s.set_window(50, 3)
    s.reset(0, 192)
    s.prefill(0, prompt, phase=None, chunk=60)
    got = np.stack([f(s.logits(0, None))] + [f(x[0]) for x in steps(s, [0], forced)])
    assert np.abs(got - want).max() <= 1.5 * 2e-2 and rel_l2(got, want) <= 1.5 * 2e-2


@pytest.mark.parametrize("rows,window,sinks,n", [(1, 500, 4, 2900), (2, 1000, 130, 2900), (1, 64, 0, 640)])
def test_windowed_persistent_decode_equals_the_per_operation_path(wide, rows, window, sinks, n):
    """Bit for bit, as without a window, at contexts where most chunks are skipped."""
    model, _, _ = wide
    out = []
    for persistent in (True, False):
        s = model.session(max_rows=2, max_ctx=2976)
        s.set_persistent(persistent)
        s.set_trace(persistent)
        s.set_window(window, sinks)
        for r in range(rows):
            s.reset(r, 2976)
            s.prefill(r, ids(7 + r, n - 900 * r), phase=None)
        out.append(steps(s, list(range(rows)), ids(9, 70)))  # the window's start crosses chunk borders
        if persistent:
            assert np.any(s.trace()), "the persistent decode kernel did not run"
        s.close()
    np.testing.assert_array_equal(out[0], out[1])


def test_a_window_over_the_whole_context_changes_no_bit(wide):
    model, _, _ = wide
    s = model.session(max_rows=1, max_ctx=1024)
    got = []
    for window in (0, 1024):
        s.set_window(0)
        s.reset(0, 1024)
        s.prefill(0, ids(1, 400), phase=None)
        s.set_window(window, 3)
        got.append(steps(s, [0], ids(2, 20)))
    np.testing.assert_array_equal(got[0], got[1])


def test_windowed_quantized_decode(yar, wide):
    """The 8-bit persistent kernel with a window against its per-operation path (BF16 weights)."""
    model = yar.ARModel(wide[2], any_dims=True, precision="8bit")
    got = []
    for persistent in (True, False):
        s = model.session(max_rows=1, max_ctx=1024)
        s.set_persistent(persistent)
        s.set_window(150, 4)
        s.reset(0, 1024)
        s.prefill(0, ids(4, 600), phase=None)
        got.append(f(steps(s, [0], ids(5, 6))[:, 0]))
        s.close()
    assert np.abs(got[0] - got[1]).max() <= 2 * MAX_ABS and rel_l2(got[0], got[1]) <= 2 * REL
    model.close()


def test_generate_with_a_window_follows_the_steps(yar, wide):
    """yar_generate (graph replays) at temperature 0 picks the steps' arg max."""
    model, _, _ = wide
    prompt = ids(6, 500)
    s = model.session(max_rows=1, max_ctx=1024)
    s.set_window(120, 4)
    smp = yar.Sampling(temperature=0.0, top_p=1.0, top_k=1, repetition_penalty=1.0, penalty_window=1, min_tokens=0,
                       max_tokens=24)
    tokens, _, _ = s.generate(prompt, smp, seed=1, phase=None)
    s.reset(0, 1024)
    s.prefill(0, prompt, phase=None)
    for t in tokens:
        assert int(np.argmax(f(s.logits(0, None)))) == t
        s.step([0], [t], phase=None)
    s.set_window(0)
    other, _, _ = s.generate(prompt, smp, seed=1, phase=None)
    assert other != tokens  # the graph of the windowed steps is not reused


@pytest.mark.parametrize("window,sinks", [(0, 0), (150, 4)])
def test_batched_attention_option(yar, wide, window, sinks):
    """Steps of 16+ rows with the attention of the paged operator: ragged rows, an idle one
    among them, against the default kernel (same mask, another order of summation)."""
    model, _, _ = wide
    out = []
    for on in (False, True):
        s = model.session(max_rows=18, max_ctx=512, page_tokens=64)
        s.set_window(window, sinks)
        s.set_batched_attention(on)
        rows = [r for r in range(18) if r != 5]
        for r in rows:
            s.reset(r, 512)
            s.prefill(r, ids(20 + r, 1 + 23 * r), phase=None)
        out.append(f(steps(s, rows, ids(8, 5))))
        s.close()
    assert np.abs(out[0] - out[1]).max() <= 0.0625 and rel_l2(out[0], out[1]) <= 0.015


def test_batched_generation_with_the_option(yar, wide):
    model, _, _ = wide
    smp = yar.Sampling(temperature=1.0, top_p=0.9, top_k=20, repetition_penalty=1.1, penalty_window=20, min_tokens=0,
                       max_tokens=12)
    s = model.session(max_rows=16, max_ctx=256)
    s.set_batched_attention(True)
    prompts = [ids(40 + r, 10 + 9 * r) for r in range(16)]
    a, _, _ = s.generate_batch(prompts, smp, list(range(16)), phase=None)
    b, _, _ = s.generate_batch(prompts, smp, list(range(16)), phase=None)
    assert a == b and all(len(t) == 12 for t in a)


def test_paged_prefill_option(wide):
    model, oracle, _ = wide
    prompt = ids(11, 600)
    want = oracle_run(oracle, prompt, [], 0, 0)[0]
    s = model.session(max_rows=1, max_ctx=1024)
    s.set_prefill_attention_tc(2)
    s.reset(0, 1024)
    s.prefill(0, prompt, phase=None, chunk=250)
    got = f(s.logits(0, None))
    assert np.abs(got - want).max() <= MAX_ABS and rel_l2(got, want) <= REL


# ---- rows as page lists -----------------------------------------------------------------

@pytest.mark.parametrize("n,page", [(300, 256), (256, 64), (37, 16), (129, 64)])
def test_fork_shares_full_pages_and_the_rows_part(wide, n, page):
    model, _, _ = wide
    s = model.session(max_rows=3, max_ctx=512, page_tokens=page)
    per = 512 // page
    s.reset(0, 512)
    s.prefill(0, ids(1, n), phase=None)
    before = s.logits(0, None)
    s.fork(0, 1, 512)
    s.fork(1, 2, n + 20)
    assert s.position(1) == s.position(2) == n
    np.testing.assert_array_equal(s.logits(2, None), before)
    total, unused, _ = s.pages()
    need2 = -(-(n + 20) // page)
    assert total - unused == per + (per - n // page) + (need2 - n // page)
    # Different tokens on the three rows; each equals a row that was prefilled by itself.
    got = []
    for t in (3, 5, 8):
        s.step([0, 1, 2], [t, t + 100, t + 200], phase=None)
        got.append([s.logits(r, None) for r in range(3)])
    kv = [s.kv(r, 1, 0, n + 3) for r in range(3)]
    for r in range(3):
        s2 = model.session(max_rows=3, max_ctx=512, page_tokens=page)
        for q in range(3):
            s2.reset(q, 512)
            s2.prefill(q, ids(1, n), phase=None)
        for i, t in enumerate((3, 5, 8)):
            s2.step([0, 1, 2], [t + 100 * r] * 3, phase=None)
            np.testing.assert_array_equal(s2.logits(r, None), got[i][r])
        for a, b in zip(kv[r], s2.kv(r, 1, 0, n + 3)):
            np.testing.assert_array_equal(a, b)
        s2.close()
    # The parent goes; the children keep what they share.
    s.free(0)
    s.step([1, 2], [9, 9], phase=None)
    np.testing.assert_array_equal(s.kv(1, 0, 0, n)[0], s.kv(2, 0, 0, n)[0])
    s.free(1), s.free(2)
    assert s.pages()[1] == total


def test_fork_refusals_change_nothing(yar, wide):
    model, _, _ = wide
    s = model.session(max_rows=3, max_ctx=512, page_tokens=64, pool_pages=9)
    s.reset(0, 300)  # 5 pages
    s.prefill(0, ids(1, 200), phase=None)
    s.reset(1, 64)
    s.prefill(1, ids(2, 10), phase=None)
    keep = s.kv(1, 0, 0, 10)
    def refused(needle, call, *a):
        with pytest.raises(yar.YarError) as e:
            call(*a)
        assert e.value.status == 2 and needle in e.value.message
    refused("itself", s.fork, 0, 0, 300)
    refused("outside", s.fork, 0, 3, 300)
    refused("outside", s.fork, -1, 1, 300)
    refused("capacity", s.fork, 0, 1, 199)
    refused("capacity", s.fork, 0, 1, 513)
    refused("no cache", s.fork, 2, 1, 64)
    refused("exhausted", s.fork, 0, 1, 512)   # 3 shared, 5 own; 4 can be had
    refused("exhausted", s.reset, 1, 512)
    refused("back", s.truncate, 0, 201)
    refused("back", s.truncate, 0, -1)
    refused("no cache", s.truncate, 2, 0)
    refused("no sliding window", s.release, 0)
    refused("window", s.set_window, -1, 0)
    refused("window", s.set_window, 4, 513)
    assert s.pages()[:2] == (9, 3) and s.position(1) == 10
    for a, b in zip(keep, s.kv(1, 0, 0, 10)):
        np.testing.assert_array_equal(a, b)
    s.fork(0, 1, 320)  # drops row 1's page
    assert s.pages()[1] == 9 - 5 - 2
    for bad in (-1, 100):
        with pytest.raises(yar.YarError):
            model.session(max_rows=1, max_ctx=128, page_tokens=64, pool_pages=bad)


@pytest.mark.parametrize("n,back,page", [(200, 130, 64), (200, 128, 64), (300, 0, 256), (90, 89, 16)])
def test_truncate_goes_back(wide, n, back, page):
    model, _, _ = wide
    s = model.session(max_rows=2, max_ctx=512, page_tokens=page)
    s.reset(0, 512)
    s.prefill(0, ids(1, n), phase=None)
    s.fork(0, 1, 512)
    parent = s.kv(0, 1, 0, n)
    s.truncate(1, back)
    assert s.position(1) == back
    if back == 0:
        s.prefill(1, ids(5, 3), phase=None)
    else:
        steps(s, [1], [7, 8, 9])  # rewrites positions that the parent shares
    for a, b in zip(parent, s.kv(0, 1, 0, n)):
        np.testing.assert_array_equal(a, b)
    # The same row without the detour.
    s2 = model.session(max_rows=2, max_ctx=512, page_tokens=page)
    s2.reset(1, 512)
    if back == 0:
        s2.prefill(1, ids(5, 3), phase=None)
    else:
        s2.prefill(1, ids(1, n), phase=None)
        s2.truncate(1, back)
        steps(s2, [1], [7, 8, 9])
    np.testing.assert_array_equal(s.logits(1, None), s2.logits(1, None))
    for a, b in zip(s.kv(1, 1, 0, back + 3), s2.kv(1, 1, 0, back + 3)):
        np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("page,persistent", [(64, True), (64, False), (16, False)])
def test_release_behind_the_window(yar, wide, page, persistent):
    """Released pages are another row's from then on; the windowed row's results keep every bit."""
    model, _, _ = wide
    window, sinks, n = 130, 20, 600
    def run(release):
        s = model.session(max_rows=2, max_ctx=1024, page_tokens=page, pool_pages=1024 // page + 4)
        s.set_persistent(persistent)
        s.set_window(window, sinks)
        s.reset(0, 1024)
        s.prefill(0, ids(1, n), phase=None)
        got = list(steps(s, [0], ids(2, 3)))
        if release:
            unused = s.pages()[1]
            released = s.release(0)
            pos = s.position(0)
            first = -(-sinks // page)
            want = len([i for i in range(first, 1024 // page) if (i + 1) * page - 1 <= pos - window])
            assert released == want > 0 and s.pages()[1] == unused + released
            assert s.release(0) == 0
            with pytest.raises(yar.YarError):
                s.kv(0, 0, first * page, 1)
            assert s.kv(0, 0, 0, sinks)[0].shape[1] == sinks
            for w, k in ((0, 0), (window + 1, sinks), (window, sinks + 1)):
                with pytest.raises(yar.YarError):
                    s.set_window(w, k)
            with pytest.raises(yar.YarError) as e:
                s.truncate(0, 300)
            assert "released" in e.value.message
            s.reset(1, (4 + released) * page)  # takes the released pages
            s.prefill(1, ids(9, (4 + released) * page), phase=None)
        got += list(steps(s, [0], ids(3, 40)))
        s.prefill(0, ids(4, 50), phase=None)
        got.append([s.logits(0, None)])
        s.close()
        return np.array(got)
    np.testing.assert_array_equal(run(False), run(True))


def test_compaction_keeps_every_bit(wide):
    """Rows forked, freed, released and cut back; the pool compacted between steps."""
    model, _, _ = wide
    def run(compact):
        s = model.session(max_rows=4, max_ctx=512, page_tokens=64)
        s.set_window(140, 10)
        s.reset(3, 200)
        s.prefill(3, ids(5, 100), phase=None)
        s.reset(0, 512)
        s.prefill(0, ids(1, 330), phase=None)
        s.fork(0, 1, 512)
        s.fork(0, 2, 400)
        s.free(3)
        s.release(1)
        got = list(steps(s, [0, 1, 2], ids(2, 3)))
        s.free(0)
        if compact:
            total, unused, high = s.pages()
            used = s.compact()
            assert used == total - unused and s.pages() == (total, unused, used - 1) and high >= used
            assert s.compact() == used
        got += list(steps(s, [1, 2], ids(3, 3)))
        s.reset(0, 300)  # the free pages are found again
        s.prefill(0, ids(6, 299), phase=None)
        s.truncate(2, 310)
        if compact:
            s.compact()
        got += list(steps(s, [0, 1, 2], ids(4, 1)))
        kv = [s.kv(2, layer, 200, 111) for layer in (0, 1)]
        s.close()
        return got, kv
    (a, ka), (b, kb) = run(False), run(True)
    for x, y in zip(a, b):
        np.testing.assert_array_equal(x, y)
    np.testing.assert_array_equal(np.array(ka), np.array(kb))


def test_a_small_pool_refuses_and_serves(yar, wide):
    model, _, _ = wide
    s = model.session(max_rows=4, max_ctx=512, page_tokens=64, pool_pages=5)
    smp = yar.Sampling(temperature=0.0, top_p=1.0, top_k=1, repetition_penalty=1.0, penalty_window=1, min_tokens=0,
                       max_tokens=8)
    with pytest.raises(yar.YarError) as e:
        s.generate(ids(1, 400), smp, seed=1, phase=None)
    assert "exhausted" in e.value.message and s.pages()[1] == 5
    tokens, _, _ = s.generate(ids(1, 200), smp, seed=1, phase=None)
    assert len(tokens) == 8 and s.pages()[1] == 5


def test_one_prompt_forked_for_many_songs_in_a_small_pool(yar, wide):
    """A server's run: one prompt prefilled once, forked for 16 rows that share its pages,
    decoded together on the batched path with a window, pages released behind it, the pool
    compacted: against rows that hold everything themselves."""
    model, _, _ = wide
    prompt, n, rows = ids(1, 450), 450, list(range(16))
    def run(lean):
        pool = 6 + 16 * 4 if lean else 0
        s = model.session(max_rows=16, max_ctx=768, page_tokens=64, pool_pages=pool)
        s.set_window(200, 4)
        s.set_batched_attention(True)
        s.reset(0, n + 130)
        s.prefill(0, prompt, phase=None)
        for r in rows[1:]:
            if lean:
                s.fork(0, r, n + 130)
            else:
                s.reset(r, n + 130)
                s.prefill(r, prompt, phase=None)
        got = []
        for i in range(60):
            s.step(rows, [(37 * r + 11 * i) % 4096 for r in rows], phase=None)
            got.append([s.logits(r, None) for r in rows])
            if lean and i % 20 == 19:
                for r in rows:
                    s.release(r)
                s.compact()
        if lean:
            total, unused, high = s.pages()
            assert high == total - unused - 1
        s.close()
        return np.array(got)
    np.testing.assert_array_equal(run(False), run(True))
