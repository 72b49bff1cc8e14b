"""A session's rows and windows where test_gpu_window_rows.py does not go: first chunks in a window as
long as they are, pages released under the shortest window, pools that are too small. Tolerances as
there."""
import dataclasses

import numpy as np
import pytest

from tests.conftest import load_package
from tests.test_gpu_window_rows import REL, f, ids, rel_l2

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def yar():
    return load_package()


@pytest.fixture(scope="module")
def model(yar, synth, tmp_path_factory):
    """Pinned widths, 2 layers, 4096-row vocabulary."""
    dims = dataclasses.replace(synth.PINNED, layers=2, vocab=4096, context=4096)
    d = str(tmp_path_factory.mktemp("edges"))
    synth.write_converted(d, dims, seed=3, norm_std=0.1)
    return yar.ARModel(d, any_dims=True)


@pytest.mark.parametrize("n,window,sinks,page,max_ctx", [(700, 1000, 4, 256, 4096), (1024, 1024, 0, 64, 1024),
                                                         (900, 2000, 4, 256, 2048), (60, 1000, 4, 64, 4096)])
def test_a_windowed_first_chunk_caches_what_an_unwindowed_one_does(model, n, window, sinks, page, max_ctx):
    """No longer than the window, a prompt sees all of itself: the second layer's keys and values of
    every position against those behind the session's other prefill kernel."""
    got = []
    for w in (0, window):
        s = model.session(max_rows=1, max_ctx=max_ctx, page_tokens=page)
        s.set_window(w, sinks)
        s.reset(0, max_ctx)
        s.prefill(0, ids(n, n), phase=None)
        got.append([f(x) for x in s.kv(0, 1, 0, n)] + [f(s.logits(0, None))])
        s.close()
    for a, b in zip(got[1][:2], got[0][:2]):  # [kv_heads][positions][dim]
        assert max(rel_l2(a[:, i], b[:, i]) for i in range(n)) <= REL
    assert rel_l2(got[1][2], got[0][2]) <= REL


def test_no_way_back_into_a_released_page(yar, model):
    """Under a window of one position a row may go back to the start of a released page, not into
    one: its lost positions would be there again for a wider window."""
    s = model.session(max_rows=1, max_ctx=128, page_tokens=16)
    s.set_window(1)
    s.reset(0, 64)
    s.prefill(0, ids(1, 40), phase=None)
    assert s.release(0) == 2  # positions 0..31
    for n in (5, 17, 31):
        with pytest.raises(yar.YarError) as e:
            s.truncate(0, n)
        assert "released" in e.value.message
    assert s.position(0) == 40
    s.truncate(0, 35)
    for w in (0, 2):
        with pytest.raises(yar.YarError):
            s.set_window(w)  # pages are missing still
    s.truncate(0, 0)  # nothing is left to be seen: every page is the row's own again
    s.set_window(0)
    s.prefill(0, ids(2, 40), phase=None)
    again = s.logits(0, None)
    s.reset(0, 64)
    s.prefill(0, ids(2, 40), phase=None)
    np.testing.assert_array_equal(again, s.logits(0, None))
    s.close()


def sampling(yar, n):
    return yar.Sampling(temperature=1.0, top_p=0.9, top_k=20, repetition_penalty=1.1, penalty_window=20, min_tokens=0,
                        max_tokens=n)


def test_generation_that_the_pool_cannot_hold_changes_nothing(yar, model):
    """Two rows of guidance need more pages than there are: refused before anything runs. What fits
    once both rows' own pages are given back is served."""
    s = model.session(max_rows=3, max_ctx=512, page_tokens=64, pool_pages=9)
    s.reset(0, 128), s.prefill(0, ids(1, 70), phase=None)
    s.reset(1, 320), s.prefill(1, ids(2, 80), phase=None)
    keep, pages = [s.kv(r, 1, 0, 70) for r in (0, 1)], s.pages()
    smp = sampling(yar, 8)
    with pytest.raises(yar.YarError) as e:
        s.generate(ids(3, 300), smp, 1, phase=None, negative=ids(4, 250), cfg_scale=1.5)  # 5 + 5 pages
    assert "exhausted" in e.value.message and s.pages() == pages and (s.position(0), s.position(1)) == (70, 80)
    for a, b in zip(keep, [s.kv(r, 1, 0, 70) for r in (0, 1)]):
        np.testing.assert_array_equal(np.array(a), np.array(b))
    s.step([0, 1], [5, 6], phase=None)
    got = s.generate(ids(3, 300), smp, 1, phase=None, negative=ids(4, 150), cfg_scale=1.5)[0]  # 5 + 3 pages
    assert s.pages()[1] == 9
    with pytest.raises(yar.YarError):
        s.step([1], [6], phase=None)  # the rows were the request's
    s.close()
    s = model.session(max_rows=2, max_ctx=512, page_tokens=64)
    assert got == s.generate(ids(3, 300), smp, 1, phase=None, negative=ids(4, 150), cfg_scale=1.5)[0]
    s.close()


@pytest.mark.parametrize("rows,slots,pool", [(4, 4, 7), (2, 2, 4), (18, 17, 20), (4, 4, 1 + 4)])
def test_queued_requests_wait_for_pages(yar, model, rows, slots, pool):
    """Requests served from a pool that does not hold all slots' at once: each one's tokens as with
    room for all, every page given back, a row of another owner left alone."""
    n = 2 * slots + 1
    prompts = [ids(50 + i, 20 + 37 * i % 180) for i in range(n)]  # 1 to 4 pages each
    smps = [sampling(yar, 10 + i % 30) for i in range(n)]
    seeds = list(range(n))
    full = model.session(max_rows=rows, max_ctx=256, page_tokens=64)
    want = full.generate_requests(prompts, smps, seeds, phase=None, slots=slots)
    full.close()
    s = model.session(max_rows=rows, max_ctx=256, page_tokens=64, pool_pages=pool)
    if rows > slots or pool == 5:
        s.reset(rows - 1, 64), s.prefill(rows - 1, ids(1, 30), phase=None)
        other = s.kv(rows - 1, 1, 0, 30)
    tokens, timing, ended = s.generate_requests(prompts, smps, seeds, phase=None, slots=slots)
    assert tokens == want[0] and ended == want[2]
    left, first = pool - (rows > slots), 0  # the requests that start at once: in order, as far as the pages go
    while first < slots and left >= -(-(len(prompts[first]) + smps[first].max_tokens) // 64):
        left -= -(-(len(prompts[first]) + smps[first].max_tokens) // 64)
        first += 1
    assert timing["refills"] == n - first
    if rows > slots:
        np.testing.assert_array_equal(np.array(other), np.array(s.kv(rows - 1, 1, 0, 30)))
    assert s.pages()[1] == pool - (rows > slots)
    again = s.generate_requests(prompts, smps, seeds, phase=None, slots=slots)[0]
    assert again == tokens
    s.close()


def test_a_request_that_the_pool_can_never_hold_is_refused_first(yar, model):
    s = model.session(max_rows=3, max_ctx=512, page_tokens=64, pool_pages=6)
    s.reset(2, 128), s.prefill(2, ids(1, 100), phase=None)
    s.reset(0, 64), s.prefill(0, ids(2, 40), phase=None)
    pages, smp = s.pages(), sampling(yar, 8)
    for prompts in ([ids(3, 30), ids(4, 40), ids(5, 260)], [ids(3, 300)]):  # the last: 5 pages, 4 can be had
        with pytest.raises(yar.YarError) as e:
            s.generate_requests(prompts, [smp] * len(prompts), list(range(len(prompts))), phase=None, slots=min(2, len(prompts)))
        assert "exhausted" in e.value.message and s.pages() == pages and s.position(0) == 40
    with pytest.raises(yar.YarError):
        s.generate_batch([ids(3, 30), ids(4, 260)], smp, [1, 2], phase=None)
    tokens = s.generate_batch([ids(3, 30), ids(4, 200)], smp, [1, 2], phase=None)[0]
    assert [len(t) for t in tokens] == [8, 8] and s.position(2) == 100
    s.close()


def test_shared_pages_count_once_and_come_back(yar, model):
    """Two rows that share pages, replaced by a request of both rows that needs the whole pool; one
    that a third row shares stays that row's."""
    smp, negative = sampling(yar, 8), ids(4, 150)
    s = model.session(max_rows=3, max_ctx=512, page_tokens=64, pool_pages=6)
    s.reset(0, 256), s.prefill(0, ids(1, 200), phase=None)
    s.fork(0, 1, 256)  # 3 shared pages, 2 more: 1 is left
    assert s.pages()[:2] == (6, 1)
    got = s.generate(ids(3, 170), smp, 1, phase=None, negative=negative, cfg_scale=1.5)[0]  # 3 + 3 pages
    assert len(got) == 8 and s.pages()[1] == 6
    s.reset(0, 256), s.prefill(0, ids(1, 200), phase=None)
    s.fork(0, 2, 200)
    keep = s.kv(2, 1, 0, 200)
    for call in (lambda: s.generate(ids(3, 170), smp, 1, phase=None),  # 3 pages, 2 can be had
                 lambda: s.generate_batch([ids(3, 170)], smp, [1], phase=None)):
        with pytest.raises(yar.YarError) as e:
            call()
        assert "exhausted" in e.value.message and s.position(0) == 200
    assert len(s.generate(ids(3, 100), smp, 1, phase=None)[0]) == 8
    np.testing.assert_array_equal(np.array(keep), np.array(s.kv(2, 1, 0, 200)))
    s.close()
