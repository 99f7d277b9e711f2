"""A paged key/value cache and the attention that reads it.

A cache is a pair of 16-bit tensors ``k``, ``v`` [pages, page_size, kv_heads, head_dim] (attention reads
one layer) or [layers, pages, page_size, kv_heads, head_dim] (the cache operators move all layers at
once; a 4-D cache is one layer).  A sequence is a row of ``table`` (int32 page numbers, -1 where
there is no page) and its length in ``lens`` (int32); ``refs`` (int32) counts the sequences that hold
each page.  ``Cache`` keeps the five together.

Tables, lengths and counts stay on the GPU: no call here waits for the device, every call is
launched on ``torch.cuda.current_stream()`` and may be captured in a CUDA graph.  What a table or
list says is checked where it is read: a page, position or sequence out of range is skipped.

    cache = Cache(layers=2, pages=256, page_size=16, kv_heads=8, head_dim=128, seqs=4, max_pages=64)
    cache.reserve(seqs, 100)
    cache.append(k_new, v_new)                                # [layers, seqs, tokens, kv_heads, head_dim]
    o = tree_attention(q, cache.k[0], cache.v[0], cache.table, cache.lens, tree_mask(parents))
    cache.accept(path, counts, drafts)

Kernels: ``csrc/cache_attn.cu`` and ``csrc/cache_pages.cu``, through the C ABI of ``ntl_kernels.h``.
"""

from __future__ import annotations

import ctypes
import math
import struct

import torch

from . import _lib

# ntl_cache_t and ntl_query_t: pointers first, then what the shapes decide.
_CACHE = struct.Struct("=12q")
_QUERY = struct.Struct("=13qd")
_CACHE_TAIL = struct.Struct("=10q")
_QUERY_TAIL = struct.Struct("=8qd")
_TWO = struct.Struct("=2q")
_FIVE = struct.Struct("=5q")
_DTYPES = {torch.float16: 0, torch.bfloat16: 1}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_empty, _empty_like, _uint8 = torch.empty, torch.empty_like, torch.uint8


def _stream(index):
    return _raw_stream(index) if _raw_stream is not None else torch.cuda.current_stream(index).cuda_stream


_functions: dict = {}


def _call(index, name, *args):
    """The entry point ``name`` on device ``index``'s current stream; a non-zero return raises ``KernelError``."""
    fn = _functions.get(name)
    if fn is None:
        fn = _functions[name] = getattr(_lib.lib(), name)
    if index == _current_device():
        code = fn(*args, _stream(index))
    else:
        with torch.cuda.device(index):
            code = fn(*args, _stream(index))
    if code:
        raise _lib.KernelError(name, code, (_lib.lib().ntl_last_error() or b"").decode())


_workspaces: dict = {}


def _workspace(index, size, device):
    """At least ``size`` bytes for a call on device ``index``'s current stream.  Calls on one stream follow each
    other, so they share a buffer; a call that is captured in a graph, which may be replayed on any stream,
    gets its own."""
    if torch.cuda.is_current_stream_capturing():
        return _empty(size, dtype=_uint8, device=device)
    key = (index, _stream(index))
    work = _workspaces.get(key)
    if work is None or work.numel() < size:
        if len(_workspaces) >= 64:
            _workspaces.clear()
        work = _workspaces[key] = _empty(size, dtype=_uint8, device=device)
    return work


# ------------------------------------------------------------------------------ argument checks
#
# Checks look at shapes, strides, dtypes and devices alone, so a call whose arguments have been seen in
# that form before skips them (about 10 us of a call): ``_plan`` keeps what a check returned by that
# form, never by a tensor's address or identity.  Addresses are only checked for alignment, every time.

_plans: dict = {}


def _plan(check, tensors, *values):
    """``check(*tensors, *values)``, or what it returned for arguments of the same form."""
    key = [check, *values]
    try:
        for x in tensors:
            if x is not None:
                key += (x.shape, x.stride(), x.dtype, x.get_device())
            else:
                key.append(None)
        key = tuple(key)
        plan = _plans.get(key)
    except (AttributeError, TypeError, RuntimeError):  # not tensors, or not hashable: the check says so
        return check(*tensors, *values)
    if plan is None:
        plan = check(*tensors, *values)
        if len(_plans) >= 4096:
            _plans.clear()
        _plans[key] = plan
    return plan


def _ints(name, x, index, *shape):
    """An int32 CUDA tensor on device ``index`` whose sizes are ``shape`` (None: any), last dim dense."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if x.dtype is not torch.int32:
        raise ValueError(f"{name}: expected dtype int32, got {x.dtype}")
    if x.dim() != len(shape) or any(want is not None and want != got for want, got in zip(shape, x.shape)):
        want = tuple("any" if n is None else n for n in shape)
        raise ValueError(f"{name}: expected shape {want}, got {tuple(x.shape)}")
    if x.shape[-1] > 1 and x.stride(-1) != 1:
        raise ValueError(f"{name} must be dense along its last dimension")
    if x.get_device() != index:
        raise ValueError("All tensor arguments must be on the same CUDA device")


def _values(name, x):
    """A 16-bit CUDA tensor that the kernels can read 16 bytes at a time along its last dimension."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if x.dtype not in _DTYPES:
        raise ValueError(f"{name}: expected dtype float16 or bfloat16, got {x.dtype}")
    if x.numel() and (x.stride(-1) != 1 or any(s % 8 for s in x.stride()[:-1])):
        raise ValueError(f"{name} must be dense along its last dimension, its other strides multiples of 8")


def _aligned(**tensors):
    for name, x in tensors.items():
        if x.data_ptr() % 16:
            raise ValueError(f"{name} requires a tensor with an inspectable, 16-byte-aligned data pointer")


def _check_cache(k, v, dims, written):
    """(descriptor without its pointers, device index) of a cache; ``dims``: the ranks it may have."""
    _values("k", k)
    _values("v", v)
    shape, stride = k.shape, k.stride()
    if len(shape) not in dims:
        raise ValueError(f"k: expected {' or '.join(map(str, dims))} dimensions, got shape {tuple(shape)}")
    if v.shape != shape or v.stride() != stride or v.dtype is not k.dtype:
        raise ValueError("k and v must have the same shape, strides and dtype")
    index = k.get_device()
    if v.get_device() != index:
        raise ValueError("All tensor arguments must be on the same CUDA device")
    if written and any(n > 1 and s == 0 for n, s in zip(shape, stride)):
        raise ValueError("k and v must not be broadcast: their rows are written")
    if len(shape) == 4:
        shape, stride = (1, *shape), (0, *stride)
    if shape[4] % 8 or not shape[4]:
        raise ValueError(f"k: head_dim {shape[4]} is not a multiple of 8")
    if not shape[2]:
        raise ValueError("k: page_size is 0")
    return _CACHE_TAIL.pack(*shape, *stride[:4], _DTYPES[k.dtype]), index


def _cache(k, v, tail):
    kp, vp = k.data_ptr(), v.data_ptr()
    if (kp | vp) & 15:
        _aligned(k=k, v=v)
    return _TWO.pack(kp, vp) + tail


def _pool_workspace(pages, n):
    out = ctypes.c_uint64(0)
    _lib.call("ntl_cache_workspace_size", pages, n, ctypes.byref(out))
    return out.value


# ------------------------------------------------------------------------------ attention


def _check_attention(q, k, v, table, lens, q_lens, tree, scale):
    cache, index = _check_cache(k, v, (4,), False)
    _values("q", q)
    shape, kv = q.shape, k.shape
    if len(shape) != 4:
        raise ValueError(f"q: expected 4 dimensions [seqs, tokens, heads, head_dim], got shape {tuple(shape)}")
    seqs, tokens, heads, dim = shape
    if q.dtype is not k.dtype:
        raise ValueError(f"q: expected dtype {k.dtype} like the cache, got {q.dtype}")
    if dim != kv[3] or dim not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, the same for q ({dim}) and the cache ({kv[3]})")
    if kv[1] % 8:
        raise ValueError(f"page_size {kv[1]} is not a multiple of 8")
    if not kv[2] or heads % kv[2] or heads // kv[2] > 128:
        raise ValueError(f"{heads} query heads cannot share {kv[2]} key heads (a whole number, up to 128 each)")
    if q.get_device() != index:
        raise ValueError("All tensor arguments must be on the same CUDA device")
    _ints("table", table, index, seqs, None)
    _ints("lens", lens, index, seqs)
    if q_lens is not None:
        _ints("q_lens", q_lens, index, seqs)
    tree_stride = 0
    if tree is not None:
        words = (tokens + 31) // 32
        shared = isinstance(tree, torch.Tensor) and tree.dim() == 3 and tree.shape[0] == 1
        _ints("tree", tree, index, 1 if shared else seqs, tokens, words)
        if tokens > 1 and tree.stride(1) != words:
            raise ValueError("tree must be dense along its last two dimensions")
        tree_stride = 0 if shared else tree.stride(0)
    if scale is None:
        scale = 1.0 / math.sqrt(dim)
    elif not 0 < scale < 1e30:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    size = 0
    query = _QUERY_TAIL.pack(seqs, tokens, heads, *q.stride()[:3], table.stride(0), table.shape[1], scale)
    if q.numel():
        out = ctypes.c_uint64(0)
        with torch.cuda.device(index):
            _lib.call("ntl_cache_attention_workspace", _TWO.pack(16, 16) + cache, _FIVE.pack(16, 16, 16, 16, 0) + query,
                      ctypes.byref(out))
        size = out.value
    return cache, query, index, size, q.is_contiguous(), q.device, tree_stride


def _check_out(out, q, k, v):
    _values("out", out)
    if out.shape != q.shape or out.dtype is not q.dtype or not out.is_contiguous() or out.device != q.device:
        raise ValueError(f"out must be a contiguous {q.dtype} tensor of shape {tuple(q.shape)} on q's device")
    _aligned(out=out)
    begin, end = out.data_ptr(), out.data_ptr() + out.numel() * 2
    for name, x in (("q", q), ("k", k), ("v", v)):
        if x.numel() and out.numel():
            reach = sum((n - 1) * s for n, s in zip(x.shape, x.stride())) + 1
            if x.data_ptr() < end and begin < x.data_ptr() + 2 * reach:
                raise ValueError(f"Tensor arguments {name} and out must have disjoint storage")


def _attend(q, k, v, table, lens, q_lens, scale, out, tree, window, sinks):
    cache, query, index, size, dense, device, tree_stride = _plan(_check_attention, (q, k, v, table, lens, q_lens, tree), scale)
    qp = q.data_ptr()
    if qp & 15:
        _aligned(q=q)
    if out is None:
        out = _empty_like(q) if dense else _empty(q.shape, dtype=q.dtype, device=device)
    else:
        _check_out(out, q, k, v)
    if not size:
        return out
    work = _workspace(index, size, device)
    query = _FIVE.pack(qp, out.data_ptr(), table.data_ptr(), lens.data_ptr(),
                       0 if q_lens is None else q_lens.data_ptr()) + query
    if tree is None:
        _call(index, "ntl_window_attention", _cache(k, v, cache), query, window, sinks, work.data_ptr(), size)
    else:
        _call(index, "ntl_tree_attention", _cache(k, v, cache), query, tree.data_ptr(), tree_stride, work.data_ptr(), size)
    return out


def _check_parents(parents):
    if not isinstance(parents, torch.Tensor) or not parents.is_cuda:
        raise TypeError("parents must be a CUDA tensor")
    index = parents.get_device()
    _ints("parents", parents, index, None, None)
    return index, (parents.shape[0], parents.shape[1], (parents.shape[1] + 31) // 32), parents.device


def tree_mask(parents):
    """Visibility words of draft trees: int32 [seqs, tokens, ceil(tokens / 32)], bit s % 32 of word
    s // 32 set where draft s is draft t itself or an ancestor.  ``parents`` int32 [seqs, tokens] holds
    each draft's parent; what is not an earlier draft (-1) is a root."""
    index, shape, device = _plan(_check_parents, (parents,))
    words = _empty(shape, dtype=torch.int32, device=device)
    _call(index, "ntl_tree_mask", parents.data_ptr(), parents.stride(0), shape[0], shape[1], words.data_ptr())
    return words


def tree_attention(q, k, v, table, lens, tree, *, q_lens=None, scale=None, out=None):
    """Attention of drafted tokens over one layer of a cache that already holds their keys and values.

    ``q`` [seqs, tokens, heads, head_dim] (head_dim 64 or 128, heads a multiple of the cache's): sequence
    b's tokens are the last ``q_lens[b]`` (default: tokens) of its ``lens[b]`` cached ones.  A token sees
    every key before the drafts, and draft s where bit s of its words in ``tree`` ([seqs or 1, tokens,
    ceil(tokens / 32)] int32, see ``tree_mask``) is set; a token that sees nothing, and tokens past
    ``q_lens``, give 0.  ``scale`` defaults to 1 / sqrt(head_dim).  One token with its own bit set is
    single-token decode.  Returns [seqs, tokens, heads, head_dim] in q's dtype (``out`` if given).

    Statistics and sums are fp32; the exponentials are rounded to the cache's type for the product
    with V.  A NaN or infinity in a key row reaches the tokens that see it; in a value row that some token
    of the call sees, it may reach tokens of the same sequence that do not."""
    if tree is None:
        raise TypeError("tree must be a CUDA tensor")
    return _attend(q, k, v, table, lens, q_lens, scale, out, tree, 0, 0)


def window_attention(q, k, v, table, lens, window, sinks=0, *, q_lens=None, scale=None, out=None):
    """Causal attention with a sliding window over one layer of a cache that already holds the new tokens.

    As ``tree_attention``, but the token at position i sees the keys j <= i with j > i - window, or
    j < sinks (the first tokens, which stay visible).  ``tokens`` may be one (decode) or a prompt's
    chunk.  Pages wholly outside what the call sees are not read and may be -1 in ``table``."""
    window, sinks = int(window), int(sinks)
    if window < 1 or sinks < 0:
        raise ValueError(f"window must be at least 1 and sinks at least 0, got {window} and {sinks}")
    return _attend(q, k, v, table, lens, q_lens, scale, out, None, window, sinks)


# ------------------------------------------------------------------------------ cache operators


def _check_append(k, v, k_new, v_new, table, lens, counts):
    cache, index = _check_cache(k, v, (4, 5), True)
    _values("k_new", k_new)
    _values("v_new", v_new)
    layered = k.dim() == 5
    if k_new.dim() != k.dim():
        raise ValueError(f"k_new: expected {k.dim()} dimensions, got shape {tuple(k_new.shape)}")
    seqs, tokens = k_new.shape[-4], k_new.shape[-3]
    want = (*k.shape[:1], seqs, tokens, *k.shape[-2:]) if layered else (seqs, tokens, *k.shape[-2:])
    if k_new.shape != want or k_new.dtype is not k.dtype:
        raise ValueError(f"k_new: expected {k.dtype} of shape {tuple(want)}, got {k_new.dtype} {tuple(k_new.shape)}")
    if v_new.shape != want or v_new.dtype is not k.dtype or v_new.stride() != k_new.stride():
        raise ValueError("k_new and v_new must have the same shape, strides and dtype")
    if k_new.get_device() != index or v_new.get_device() != index:
        raise ValueError("All tensor arguments must be on the same CUDA device")
    _ints("table", table, index, seqs, None)
    _ints("lens", lens, index, seqs)
    if counts is not None:
        _ints("counts", counts, index, seqs)
    stride = k_new.stride() if layered else (0, *k_new.stride())
    return cache, index, stride[:4], (table.stride(0), seqs, table.shape[1]), tokens


def append_tokens(k, v, k_new, v_new, table, lens, counts=None):
    """Write new tokens' rows, ``k_new`` / ``v_new`` [layers, seqs, tokens, kv_heads, head_dim] (4-D without
    layers for a 4-D cache), at positions lens[b] + t, t < counts[b] (default: all); returns the new
    lengths.  A row whose position has no page is dropped: ``reserve`` first."""
    cache, index, strides, sizes, tokens = _plan(_check_append, (k, v, k_new, v_new, table, lens, counts))
    kp, vp = k_new.data_ptr(), v_new.data_ptr()
    if (kp | vp) & 15:
        _aligned(k_new=k_new, v_new=v_new)
    new = _empty_like(lens)
    _call(index, "ntl_cache_append", _cache(k, v, cache), kp, vp, *strides, table.data_ptr(), *sizes, lens.data_ptr(),
          None if counts is None else counts.data_ptr(), tokens, new.data_ptr())
    return new


def _check_accept(k, v, table, lens, path, counts, each, common):
    cache, index = _check_cache(k, v, (4, 5), True)
    _ints("lens", lens, index, None)
    seqs = lens.shape[0]
    _ints("table", table, index, seqs, None)
    _ints("path", path, index, seqs, None)
    _ints("counts", counts, index, seqs)
    if each is not None:
        _ints("drafts", each, index, seqs)
    elif common < 0:
        raise ValueError(f"drafts must be at least 0, got {common}")
    return cache, index, (table.stride(0), seqs, table.shape[1]), (path.stride(0), path.shape[1])


def accept_path(k, v, table, lens, path, counts, drafts):
    """Keep a verified path of each sequence's last ``drafts`` cached tokens (an int, or int32 [seqs]): the
    row of draft path[b, i] moves to draft place i, i < counts[b]; ``path`` int32 [seqs, most] increases along
    i.  Returns the new lengths, lens - drafts + counts."""
    each, common = (drafts, 0) if isinstance(drafts, torch.Tensor) else (None, int(drafts))
    cache, index, sizes, steps = _plan(_check_accept, (k, v, table, lens, path, counts, each), common)
    new = _empty_like(lens)
    _call(index, "ntl_cache_accept", _cache(k, v, cache), table.data_ptr(), *sizes, lens.data_ptr(),
          None if each is None else each.data_ptr(), common, path.data_ptr(), *steps, counts.data_ptr(), new.data_ptr())
    return new


def _check_copy(k, v, src, dst):
    cache, index = _check_cache(k, v, (4, 5), True)
    _ints("src", src, index, None)
    _ints("dst", dst, index, src.shape[0])
    return cache, index, src.shape[0]


def copy_pages(k, v, src, dst):
    """Copy pages ``src[i]`` to ``dst[i]`` (int32), all layers, K and V.  No page may be both read and written."""
    cache, index, n = _plan(_check_copy, (k, v, src, dst))
    _call(index, "ntl_cache_copy_pages", _cache(k, v, cache), src.data_ptr(), dst.data_ptr(), n)


def _check_sequences(table, lens, refs, pages, index):
    if index is None:
        if not isinstance(table, torch.Tensor) or not table.is_cuda:
            raise TypeError("table must be a CUDA tensor")
        index = table.get_device()
    _ints("table", table, index, None, None)
    _ints("lens", lens, index, table.shape[0])
    _ints("refs", refs, index, pages)
    return index, (table.stride(0), *table.shape)


def _check_fork(k, v, table, lens, refs, src, dst):
    cache, index = _check_cache(k, v, (4, 5), True)
    pages = k.shape[-4]
    _, sizes = _check_sequences(table, lens, refs, pages, index)
    _ints("src", src, index, None)
    n = src.shape[0]
    _ints("dst", dst, index, n)
    return cache, index, sizes, n, _pool_workspace(pages, n), k.device


def fork(k, v, table, lens, refs, src, dst):
    """Make sequences ``dst[i]`` (int32, holding nothing, no repeats) copies of ``src[i]``: full pages are shared,
    the part of a page at the end is copied into the lowest free page, in order.  ``dst`` and ``src`` have no
    sequence in common.  Updates table, lens and refs in place; returns int32 [n]: 1, or 0 where no
    page was left and the child holds nothing."""
    cache, index, sizes, n, size, device = _plan(_check_fork, (k, v, table, lens, refs, src, dst))
    granted = _empty(n, dtype=torch.int32, device=device)
    work = _workspace(index, size, device)
    _call(index, "ntl_cache_fork", _cache(k, v, cache), table.data_ptr(), *sizes, lens.data_ptr(), refs.data_ptr(),
          src.data_ptr(), dst.data_ptr(), n, granted.data_ptr(), work.data_ptr(), size)
    return granted


def _check_reserve(table, lens, refs, seqs, each, common, page_size):
    index, sizes = _check_sequences(table, lens, refs, None, None)
    _ints("seqs", seqs, index, None)
    n, pages = seqs.shape[0], refs.shape[0]
    if each is not None:
        _ints("extra", each, index, n)
    elif common < 0:
        raise ValueError(f"extra must be at least 0, got {common}")
    if page_size < 1:
        raise ValueError(f"page_size must be at least 1, got {page_size}")
    return index, sizes, n, pages, _pool_workspace(pages, n), table.device


def reserve(table, lens, refs, seqs, extra, page_size):
    """Map the lowest free pages so that each sequence in ``seqs`` (int32, no repeats) can hold ``extra`` (an int,
    or int32 [n]) more tokens, in order.  Updates table and refs in place; returns int32 [n]: 1, or 0 where
    the pages or the table's width ran out and nothing was mapped."""
    each, common = (extra, 0) if isinstance(extra, torch.Tensor) else (None, int(extra))
    index, sizes, n, pages, size, device = _plan(_check_reserve, (table, lens, refs, seqs, each), common, int(page_size))
    granted = _empty(n, dtype=torch.int32, device=device)
    work = _workspace(index, size, device)
    _call(index, "ntl_cache_reserve", pages, int(page_size), table.data_ptr(), *sizes, lens.data_ptr(), refs.data_ptr(),
          seqs.data_ptr(), n, common, None if each is None else each.data_ptr(), granted.data_ptr(), work.data_ptr(),
          size)
    return granted


def _check_free(table, lens, refs, seqs):
    index, sizes = _check_sequences(table, lens, refs, None, None)
    _ints("seqs", seqs, index, None)
    return index, sizes, refs.shape[0], seqs.shape[0]


def free(table, lens, refs, seqs):
    """Sequences ``seqs`` (int32) give their pages back and hold nothing; table, lens and refs in place."""
    index, sizes, pages, n = _plan(_check_free, (table, lens, refs, seqs))
    _call(index, "ntl_cache_free", pages, table.data_ptr(), *sizes, lens.data_ptr(), refs.data_ptr(), seqs.data_ptr(), n)


def _check_compact(k, v, table, refs, table_out, refs_out):
    cache, index = _check_cache(k, v, (4, 5), True)
    pages = k.shape[-4]
    _ints("table", table, index, None, None)
    _ints("refs", refs, index, pages)
    _ints("table_out", table_out, index, *table.shape)
    _ints("refs_out", refs_out, index, pages)
    return cache, index, table.shape, _pool_workspace(pages, 0), k.device


def compact(k, v, table, refs, *, table_out=None, refs_out=None):
    """Move the live pages (refs > 0) to the lowest numbers: of n, the k-th at or past n goes into the k-th hole
    before n.  ``table_out`` and ``refs_out`` (default: in place) follow.  Returns int32 [1]: n."""
    table_out = table if table_out is None else table_out
    refs_out = refs if refs_out is None else refs_out
    cache, index, shape, size, device = _plan(_check_compact, (k, v, table, refs, table_out, refs_out))
    live = _empty(1, dtype=torch.int32, device=device)
    work = _workspace(index, size, device)
    _call(index, "ntl_cache_compact", _cache(k, v, cache), table.data_ptr(), table.stride(0), table_out.data_ptr(),
          table_out.stride(0), *shape, refs.data_ptr(), refs_out.data_ptr(), live.data_ptr(), work.data_ptr(), size)
    return live


class Cache:
    """The tensors of one paged cache and the operators on them.  Every sequence slot starts empty."""

    def __init__(self, *, layers, pages, page_size, kv_heads, head_dim, seqs, max_pages, dtype=torch.float16,
                 device="cuda"):
        shape = (layers, pages, page_size, kv_heads, head_dim)
        self.k = torch.empty(shape, dtype=dtype, device=device)
        self.v = torch.empty(shape, dtype=dtype, device=device)
        self.table = torch.full((seqs, max_pages), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(seqs, dtype=torch.int32, device=device)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=device)

    def part(self, seqs):
        """A cache over some of the sequences (a slice of the slots): the same pool and its rows of the table; its
        lengths are its own from here on."""
        part = object.__new__(Cache)
        part.k, part.v, part.refs = self.k, self.v, self.refs
        part.table, part.lens = self.table[seqs], self.lens[seqs].clone()
        return part

    def reserve(self, seqs, extra):
        return reserve(self.table, self.lens, self.refs, seqs, extra, self.k.shape[2])

    def append(self, k_new, v_new, counts=None):
        self.lens = append_tokens(self.k, self.v, k_new, v_new, self.table, self.lens, counts)

    def accept(self, path, counts, drafts):
        self.lens = accept_path(self.k, self.v, self.table, self.lens, path, counts, drafts)

    def fork(self, src, dst):
        return fork(self.k, self.v, self.table, self.lens, self.refs, src, dst)

    def free(self, seqs):
        free(self.table, self.lens, self.refs, seqs)

    def copy_pages(self, src, dst):
        copy_pages(self.k, self.v, src, dst)

    def compact(self):
        return compact(self.k, self.v, self.table, self.refs)

    def tree_attention(self, layer, q, tree, **kwargs):
        return tree_attention(q, self.k[layer], self.v[layer], self.table, self.lens, tree, **kwargs)

    def window_attention(self, layer, q, window, sinks=0, **kwargs):
        return window_attention(q, self.k[layer], self.v[layer], self.table, self.lens, window, sinks, **kwargs)


__all__ = ["Cache", "accept_path", "append_tokens", "compact", "copy_pages", "fork", "free", "reserve",
           "tree_attention", "tree_mask", "window_attention"]
