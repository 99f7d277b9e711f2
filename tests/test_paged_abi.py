"""The paged cache's C entry points refuse bad arguments on the host, before any CUDA call."""

from __future__ import annotations

import ctypes
import struct

import pytest

PTR = 1 << 20  # never read: every call below is refused, or has nothing to do


def cache(**change):
    names = ["k", "v", "layers", "pages", "page_size", "kv_heads", "head_dim", "layer_stride", "page_stride",
             "row_stride", "head_stride", "dtype"]
    values = dict(zip(names, [PTR, PTR, 1, 10, 16, 2, 64, 0, 2048, 128, 64, 0]))
    assert set(change) <= set(names)
    return struct.pack("=12q", *{**values, **change}.values())


def query(**change):
    names = ["q", "o", "table", "lens", "q_lens", "seqs", "tokens", "heads", "seq_stride", "token_stride", "head_stride",
             "table_stride", "max_pages", "scale"]
    values = dict(zip(names, [PTR, PTR, PTR, PTR, 0, 2, 3, 4, 768, 256, 64, 8, 8, 0.125]))
    assert set(change) <= set(names)
    return struct.pack("=13qd", *{**values, **change}.values())


@pytest.fixture(scope="module")
def call(built_library):
    from ntilang_b200 import _lib

    def run(name, *args):
        rc = getattr(_lib.lib(), name)(*args)
        return rc, _lib.lib().ntl_last_error().decode() if rc else ""

    return run


INVALID, UNSUPPORTED, ALIGNMENT = 1, 2, 5


@pytest.mark.parametrize("c,q,code,text", [
    (dict(dtype=2), {}, UNSUPPORTED, "data type"), (dict(head_dim=96), {}, UNSUPPORTED, "head_dim"),
    (dict(page_size=12), {}, UNSUPPORTED, "page_size"), (dict(page_size=0), {}, UNSUPPORTED, "page_size"),
    (dict(pages=-1), {}, INVALID, "negative"), (dict(k=0), {}, INVALID, "NULL"), (dict(v=0), {}, INVALID, "NULL"),
    (dict(k=PTR + 8), {}, ALIGNMENT, "aligned"), (dict(row_stride=100), {}, ALIGNMENT, "strides"),
    (dict(kv_heads=3), {}, UNSUPPORTED, "key heads"), (dict(kv_heads=0), {}, UNSUPPORTED, "key heads"),
    (dict(kv_heads=1), dict(heads=129), UNSUPPORTED, "key heads"), ({}, dict(seqs=-1), INVALID, "negative"),
    ({}, dict(scale=0.0), INVALID, "scale"), ({}, dict(scale=float("nan")), INVALID, "scale"),
    ({}, dict(scale=-1.0), INVALID, "scale"), ({}, dict(q=0), INVALID, "NULL"), ({}, dict(lens=0), INVALID, "NULL"),
    ({}, dict(table=0), INVALID, "NULL"), ({}, dict(o=PTR + 2), ALIGNMENT, "aligned"),
    ({}, dict(token_stride=4), ALIGNMENT, "strides"), ({}, dict(max_pages=1 << 40), UNSUPPORTED, "too large"),
])
def test_attention_refusals(call, c, q, code, text):
    for name, args in (("ntl_tree_attention", (PTR, 6)), ("ntl_window_attention", (8, 1))):
        rc, why = call(name, cache(**c), query(**q), *args, PTR, 1 << 40, None)
        assert rc == code and text in why, (name, rc, why)


def test_attention_arguments(call):
    assert call("ntl_window_attention", cache(), query(), 0, 0, PTR, 1 << 40, None)[0] == INVALID
    assert call("ntl_window_attention", cache(), query(), 4, -1, PTR, 1 << 40, None)[0] == INVALID
    rc, why = call("ntl_tree_attention", cache(), query(), None, 0, PTR, 1 << 40, None)
    assert rc == INVALID and "mask" in why
    assert call("ntl_tree_attention", cache(), query(), PTR, -1, PTR, 1 << 40, None)[0] == INVALID
    for nothing in (dict(seqs=0), dict(tokens=0), dict(heads=0)):
        assert call("ntl_tree_attention", cache(), query(**nothing), None, 0, None, 0, None) == (0, "")


def test_cache_refusals(call):
    size = ctypes.c_uint64(0)
    assert call("ntl_cache_workspace_size", 100, 7, ctypes.byref(size)) == (0, "") and size.value >= 4 * 307
    assert call("ntl_cache_workspace_size", -1, 7, ctypes.byref(size))[0] == INVALID
    append = lambda c, new=PTR, out=PTR, tokens=4, stride=64: call(  # noqa: E731
        "ntl_cache_append", c, new, PTR, 0, 512, 128, stride, PTR, 8, 2, 8, PTR + 64, None, tokens, out, None)
    for got, code, text in [
        (append(cache(head_dim=60)), UNSUPPORTED, "head_dim"), (append(cache(page_size=0)), UNSUPPORTED, "page_size"),
        (append(cache(layers=-1)), INVALID, "negative"), (append(cache(k=8)), ALIGNMENT, "aligned"),
        (append(cache(head_stride=4)), ALIGNMENT, "strides"), (append(cache(), new=None), INVALID, "NULL"),
        (append(cache(), new=24), ALIGNMENT, "aligned"), (append(cache(), stride=12), ALIGNMENT, "aligned"),
        (append(cache(), out=None), INVALID, "NULL"), (append(cache(), out=PTR + 64), INVALID, "lens_out"),
        (append(cache(), tokens=-1), INVALID, "token count"),
        (call("ntl_cache_accept", cache(), PTR, 8, 2, 8, PTR, None, -1, PTR, 4, 4, PTR, PTR + 64, None), INVALID,
         "draft count"),
        (call("ntl_cache_accept", cache(), PTR, 8, 2, 8, PTR, None, 3, None, 4, 4, PTR, PTR + 64, None), INVALID,
         "NULL path"),
        (call("ntl_cache_accept", cache(), PTR, 8, 2, 8, PTR, None, 3, PTR, 4, 4, PTR, PTR, None), INVALID, "lens_out"),
        (call("ntl_cache_copy_pages", cache(), None, PTR, 2, None), INVALID, "NULL"),
        (call("ntl_cache_copy_pages", cache(), PTR, PTR, -2, None), INVALID, "page count"),
        (call("ntl_cache_fork", cache(), PTR, 8, 2, 8, PTR, PTR, PTR, PTR, 2, PTR, PTR, 8, None), INVALID, "workspace"),
        (call("ntl_cache_fork", cache(), PTR, 8, 2, 8, PTR, PTR, PTR, PTR, 70000, PTR, PTR, 1 << 30, None), UNSUPPORTED,
         "children"),
        (call("ntl_cache_fork", cache(), PTR, -8, 2, 8, PTR, PTR, PTR, PTR, 2, PTR, PTR, 1 << 30, None), INVALID,
         "table"),
        (call("ntl_cache_reserve", 10, 16, PTR, 8, 2, 8, PTR, PTR, PTR, 2, -3, None, PTR, PTR, 1 << 30, None), INVALID,
         "count"),
        (call("ntl_cache_reserve", 10, 0, PTR, 8, 2, 8, PTR, PTR, PTR, 2, 3, None, PTR, PTR, 1 << 30, None), INVALID,
         "pool"),
        (call("ntl_cache_free", 10, PTR, 8, 2, 8, PTR, None, PTR, 2, None), INVALID, "NULL"),
        (call("ntl_cache_compact", cache(), PTR, 8, PTR, 8, 2, 8, PTR, PTR, None, PTR, 1 << 30, None), INVALID, "live"),
        (call("ntl_cache_compact", cache(), PTR, 8, PTR, 8, 2, 8, PTR, PTR, PTR, PTR, 64, None), INVALID, "workspace"),
        (call("ntl_tree_mask", PTR, 4, 2, 9000, PTR, None), UNSUPPORTED, "8192"),
        (call("ntl_tree_mask", None, 4, 2, 4, PTR, None), INVALID, "NULL"),
    ]:
        assert got[0] == code and text in got[1], (got, text)
    # nothing to do is no error, and needs no GPU
    assert call("ntl_cache_copy_pages", cache(), None, None, 0, None) == (0, "")
    assert call("ntl_cache_fork", cache(), PTR, 8, 2, 8, None, None, None, None, 0, None, None, 0, None) == (0, "")
    assert call("ntl_cache_free", 10, PTR, 8, 2, 8, None, None, None, 0, None) == (0, "")
    assert call("ntl_tree_mask", None, 4, 0, 4, None, None) == (0, "")


@pytest.mark.parametrize("stride", [0, 7])
def test_written_tables_do_not_overlap(call, stride):
    """Rows closer than max_pages (8): refused where they are written."""
    big = 1 << 30
    for got in (call("ntl_cache_fork", cache(), PTR, stride, 2, 8, PTR, PTR, PTR, PTR, 2, PTR, PTR, big, None),
                call("ntl_cache_reserve", 10, 16, PTR, stride, 2, 8, PTR, PTR, PTR, 2, 3, None, PTR, PTR, big, None),
                call("ntl_cache_free", 10, PTR, stride, 2, 8, PTR, PTR, PTR, 2, None),
                call("ntl_cache_compact", cache(), PTR, 8, PTR, stride, 2, 8, PTR, PTR, PTR, PTR, big, None)):
        assert got[0] == INVALID and "overlap" in got[1], got


def test_refusals_before_any_gpu(built_library):
    """CPU tensors and wrong sizes are Python errors, on a machine without a GPU too."""
    torch = pytest.importorskip("torch")
    from ntilang_b200 import paged

    q = torch.zeros(1, 1, 2, 64, dtype=torch.float16)
    k = torch.zeros(4, 16, 1, 64, dtype=torch.float16)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(TypeError, match="CUDA"):
        paged.window_attention(q, k, k, i[None], i, 8)
    with pytest.raises(TypeError, match="CUDA"):
        paged.tree_attention(q, k, k, i[None], i, i[None, None])
    with pytest.raises(TypeError, match="CUDA"):
        paged.tree_mask(i[None])
    with pytest.raises(TypeError, match="CUDA"):
        paged.free(i[None], i, i, i)
    with pytest.raises(ValueError, match="window"):
        paged.window_attention(q, k, k, i[None], i, 0)
