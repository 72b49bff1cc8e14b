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
