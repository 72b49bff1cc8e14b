"""The paged-cache operators' host side where test_kv_ops.py does not go, without a GPU."""
import glob
import os
import re

import pytest

from tests.conftest import ROOT, load_package

CSRC = os.path.join(ROOT, "yue2-mlx_b200", "csrc")


@pytest.fixture(scope="module")
def yar():
    return load_package()


def test_a_session_tells_the_operators_error_bits_from_its_own():
    """Every bit that a session's other kernels set in its error word, by their sources; the paged
    operators' bits, moved as its calls ask for, meet none of them."""
    ops = open(os.path.join(CSRC, "kv_ops.h")).read()
    bits = [int(x) for x in re.findall(r"kKv(?:Bad\w+|Expired) = (\d+)", ops)]
    shift = int(re.search(r"kKvSessionShift = (\d+)", ops).group(1))
    assert sorted(bits) == [1, 2, 4, 64]
    mine = set()
    for path in glob.glob(os.path.join(CSRC, "*.cu*")):
        text = open(path).read()
        for value in re.findall(r"atomicOr\((?:p\.)?error, ([^)]*)\)", text):
            if "kernels_kv_" in path:
                continue
            mine |= {int(x) for x in re.findall(r"\b\d+\b", value)}
    assert {1, 2, 4, 64} <= mine
    assert not mine & {b << shift for b in bits}
    for name in ("attn", "prefill"):  # the kernels that a session launches: no bit without its move
        text = open(os.path.join(CSRC, f"kernels_kv_{name}.cu")).read()
        assert re.findall(r"atomicOr\(p\.error, kKv\w+(.*?)\);", text) and not re.search(r"atomicOr\(p\.error, kKv\w+\);", text)
    assert "a.error_shift = kKvSessionShift" in open(os.path.join(CSRC, "kernels_attn.cu")).read()
