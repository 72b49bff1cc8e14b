"""Refusals of the paged-cache operators (yar_kv_*), without a GPU: every bad argument is an
error before anything is launched. The pointers are made up: a refused call never follows
them."""
import ctypes

import pytest

from tests.conftest import load_package

PTR = 1 << 20  # 16-byte aligned, never followed


@pytest.fixture(scope="module")
def yar():
    return load_package()


def pool(yar, **kw):
    a = dict(data=PTR, layers=2, pages=8, kv_heads=2, page_tokens=16, head_dim=64)
    a.update(kw)
    return yar._KvPool(*[a[k] for k in ("data", "layers", "pages", "kv_heads", "page_tokens", "head_dim")])


def rows(yar, **kw):
    a = dict(page_table=PTR, table_stride=4, lengths=PTR, rows=3, pages_per_row=4)
    a.update(kw)
    return yar._KvRows(*[a[k] for k in ("page_table", "table_stride", "lengths", "rows", "pages_per_row")])


def refused(yar, status, needle):
    assert status == yar.INVALID_INPUT
    assert yar.lib.yar_last_error_type() == b"ValueError"
    assert needle in yar.lib.yar_last_error().decode()


POOL = [
    (dict(data=None), "data"), (dict(data=PTR + 8), "16-byte"), (dict(layers=0), "layers"), (dict(pages=0), "pages"),
    (dict(kv_heads=0), "kv_heads"), (dict(page_tokens=8), "page_tokens"), (dict(page_tokens=48), "page_tokens"),
    (dict(page_tokens=8192), "page_tokens"), (dict(head_dim=96), "head_dim"), (dict(pages=-3), "pages"),
    (dict(layers=64, pages=1 << 20, kv_heads=8, page_tokens=256), "2**31"),
]
ATTN = [
    (dict(layer=2), "layer"), (dict(layer=-1), "layer"), (dict(heads=3), "multiple"), (dict(heads=0), "multiple"),
    (dict(heads=34), "16 for each"), (dict(window=-1), "window"), (dict(sinks=-2), "window"),
    (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=1e300), "scale"), (dict(q=PTR + 2), "16-byte"), (dict(out=PTR + 4), "16-byte"),
    (dict(q_stride=252), "multiples of 8"), (dict(q_stride=248), "hold"), (dict(out_stride=128), "hold"),
    (dict(q=None), "required"), (dict(out=None), "required"), (dict(error=PTR + 1), "error"),
]
ROWS = [
    (dict(rows=-1), "rows"), (dict(rows=70000), "rows"), (dict(pages_per_row=0), "pages_per_row"),
    (dict(pages_per_row=1 << 27, table_stride=1 << 27), "2**30"), (dict(table_stride=3), "stride"),
    (dict(page_table=None), "page table"), (dict(lengths=None), "lengths"), (dict(page_table=PTR + 1), "page table"),
]


def record(yar, p, r, layer, heads, q, q_stride, out, out_stride, window, sinks, scale, error):
    return ctypes.byref(yar._KvAttn(p or pool(yar), r or rows(yar), layer, heads, q, q_stride, out, out_stride, window,
                                    sinks, scale, error))


def decode(yar, p=None, r=None, layer=0, q=PTR, q_stride=256, heads=4, out=PTR, out_stride=256, window=0, sinks=0,
           scale=0.125, max_length=0, workspace=None, workspace_bytes=0, error=None):
    return yar.lib.yar_kv_attn_decode(record(yar, p, r, layer, heads, q, q_stride, out, out_stride, window, sinks,
                                             scale, error), max_length, workspace, workspace_bytes, None)


def prefill(yar, p=None, r=None, layer=0, offsets=PTR, n=5, q=PTR, q_stride=256, heads=4, out=PTR, out_stride=256,
            window=0, sinks=0, scale=0.125, error=None):
    return yar.lib.yar_kv_attn_prefill(record(yar, p, r, layer, heads, q, q_stride, out, out_stride, window, sinks,
                                              scale, error), offsets, n, None)


def test_the_packed_record_is_the_structure(yar):
    v = list(range(1, 20))
    s = yar._KvAttn(yar._KvPool(*v[:6]), yar._KvRows(*v[6:11]), *v[11:18], 0, 0.5, 77)
    s.window, s.sinks = 18, 19
    assert bytes(s) == yar._kv_attn_bytes(*v[:17], 18, 19, 0.5, 77)


@pytest.mark.parametrize("call", [decode, prefill])
def test_attention_refuses_bad_arguments(yar, call):
    for kw, needle in POOL:
        refused(yar, call(yar, p=pool(yar, **kw)), needle)
    for kw, needle in ROWS:
        refused(yar, call(yar, r=rows(yar, **kw)), needle)
    for kw, needle in ATTN:
        refused(yar, call(yar, **kw), needle)
    assert call(yar, r=rows(yar, rows=0, page_table=None, lengths=None)) == yar.OK  # nothing to do


def test_decode_and_prefill_own_arguments(yar):
    refused(yar, decode(yar, max_length=-1), "max_length")
    refused(yar, decode(yar, workspace=PTR + 2, workspace_bytes=64), "workspace")
    refused(yar, decode(yar, workspace=None, workspace_bytes=64), "workspace")
    refused(yar, decode(yar, workspace=PTR, workspace_bytes=-1), "workspace")
    refused(yar, prefill(yar, n=-1), "n_queries")
    refused(yar, prefill(yar, n=1 << 31), "n_queries")
    refused(yar, prefill(yar, offsets=None), "offsets")
    assert prefill(yar, n=0, q=None, out=None, offsets=None) == yar.OK
    refused(yar, yar.lib.yar_kv_attn_decode(None, 0, None, 0, None), "record")
    refused(yar, yar.lib.yar_kv_attn_prefill(None, PTR, 5, None), "record")


def copy(yar, src, dst, tokens=None, a=None, b=None):
    arr = lambda v: None if v is None else (ctypes.c_int32 * len(v))(*v)  # noqa: E731
    a = a or pool(yar)
    return yar.lib.yar_kv_copy_pages(a, b or a, arr(src), arr(dst), arr(tokens), len(src), None)


def test_copy_refuses_bad_pages(yar):
    for src, dst, tokens, needle in [([8], [0], None, "outside"), ([0], [-1], None, "outside"),
                                     ([0, 1], [2, 2], None, "two copies"), ([0, 1], [1, 2], None, "source"),
                                     ([3], [3], None, "source"), ([0], [1], [17], "tokens"), ([0], [1], [-1], "tokens")]:
        refused(yar, copy(yar, src, dst, tokens), needle)
    refused(yar, copy(yar, [0], [1], None, pool(yar), pool(yar, data=PTR * 64, head_dim=128)), "same layers")
    refused(yar, copy(yar, [0], [1], None, pool(yar), pool(yar, pages=9)), "two page counts")
    refused(yar, copy(yar, [0], [1], None, pool(yar), pool(yar, data=PTR + 64)), "overlap")
    assert copy(yar, [], []) == yar.OK
    for kw, needle in POOL:
        refused(yar, copy(yar, [0], [1], a=pool(yar, **kw)), needle)


def compact(yar, p=None, table=PTR, stride=4, n_rows=3, per_row=4, counts=PTR, new=PTR * 2, new_stride=4,
            remap=PTR, used=PTR, work=PTR, error=None):
    return yar.lib.yar_kv_compact(p or pool(yar), table, stride, n_rows, per_row, counts, new, new_stride, remap, used,
                                  work, error, None)


def test_compact_refuses_bad_arguments(yar):
    for kw, needle in [(dict(table=None), "page table"), (dict(stride=3), "stride"), (dict(new_stride=2), "stride"),
                       (dict(n_rows=-1), "rows"), (dict(counts=None), "counts"), (dict(remap=None), "required"),
                       (dict(used=None), "required"), (dict(work=PTR + 2), "aligned"), (dict(new=None), "page table"),
                       (dict(new=PTR + 16), "overlaps"), (dict(new=PTR, new_stride=5), "overlaps")]:
        refused(yar, compact(yar, **kw), needle)
    refused(yar, compact(yar, p=pool(yar, pages=(1 << 20) + 1, layers=1, kv_heads=1)), "2**20")
