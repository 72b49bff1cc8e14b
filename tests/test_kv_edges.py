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


PTR = 1 << 20  # 16-byte aligned, never followed


def test_compact_takes_tables_that_do_not_overlap(yar):
    """Tables of 3 rows of 4 entries: refused where an entry of one is an entry of the other, and not
    where rows only lie between each other's (the made-up pointers are refused later then)."""
    pool = yar._KvPool(PTR, 2, 8, 2, 16, 64)
    for stride, new_stride, first in [(8, 8, d) for d in range(-28, 29)] + [(4, 4, d) for d in range(-13, 14)] + \
            [(9, 9, d) for d in (3, 4, 5, 6, 22, 23, -4, -5, -6)] + [(8, 5, d) for d in (19, 20, 21, -13, -14, 30)]:
        old = {r * stride + i for r in range(3) for i in range(4)}
        new = {first + r * new_stride + i for r in range(3) for i in range(4)}
        at = PTR + (1 << 12)
        status = yar.lib.yar_kv_compact(pool, at, stride, 3, 4, PTR, at + 4 * first, new_stride, PTR, PTR, PTR, None, None)
        assert status != yar.OK
        said = "overlaps" in yar.lib.yar_last_error().decode()
        if first == 0 and stride == new_stride:
            assert not said  # the same table
        elif stride == new_stride or min(max(old), max(new)) < max(min(old), min(new)):
            assert said == bool(old & new), (stride, first)
        else:
            assert said  # (strides that differ and cross)
