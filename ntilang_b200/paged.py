"""A paged key/value cache and the attention that reads it.

A cache is a pair of 16-bit tensors ``k``, ``v`` [pages, page_size, kv_heads, head_dim] (attention reads
one layer) or [layers, pages, page_size, kv_heads, head_dim] (the cache operators move all layers at
once; a 4-D cache is one layer).  A sequence is a row of ``table`` (int32 page numbers, -1 where
there is no page) and its length in ``lens`` (int32); ``refs`` (int32) counts the sequences that hold
each page.  ``Cache`` keeps the five together.

Tables, lengths and counts stay on the GPU: no call here waits for the device, every call is
launched on ``torch.cuda.current_stream()`` and may be captured in a CUDA graph.  What a table or
list says is checked where it is read: a page, position or sequence out of range is skipped.
No call takes part in autograd: outputs carry no gradient, whatever the inputs require.

    cache = Cache(layers=2, pages=256, page_size=16, kv_heads=8, head_dim=128, seqs=4, max_pages=64)
    cache.reserve(seqs, 100)
    cache.append(k_new, v_new)                                # [layers, seqs, tokens, kv_heads, head_dim]
    o = tree_attention(q, cache.k[0], cache.v[0], cache.table, cache.lens, tree_mask(parents))
    cache.accept(path, counts, drafts)

Kernels: ``csrc/cache_attn.cu`` and ``csrc/cache_pages.cu``.  A call's checks, its output and workspace, and
the call of the C ABI (``ntl_kernels.h``) are in ``csrc/paged_binding.cpp``, built with the library.
"""

from __future__ import annotations

import torch

try:
    from . import _paged
except ImportError as error:
    raise ImportError("ntilang_b200/_paged.so is missing or does not load; build it, with a torch that has CUDA, by: "
                      f"python -m ntilang_b200.build ({error})") from error


# ------------------------------------------------------------------------------ attention


def tree_mask(parents):
    """Visibility words of draft trees: int32 [seqs, tokens, ceil(tokens / 32)], bit s % 32 of word
    s // 32 set where draft s is draft t itself or an ancestor.  ``parents`` int32 [seqs, tokens] holds
    each draft's parent; what is not an earlier draft (-1) is a root.  Up to 8192 tokens."""
    return _paged.tree_mask(parents)


def tree_attention(q, k, v, table, lens, tree, *, q_lens=None, scale=None, out=None):
    """Attention of drafted tokens over one layer of a cache that already holds their keys and values.

    ``q`` [seqs, tokens, heads, head_dim] (head_dim 64 or 128, heads a multiple of the cache's): sequence
    b's tokens are the last ``q_lens[b]`` (default: tokens) of its ``lens[b]`` cached ones.  A token sees
    every key before the drafts, and draft s where bit s of its words in ``tree`` ([seqs or 1, tokens,
    ceil(tokens / 32)] int32, see ``tree_mask``) is set; a token that sees nothing, and tokens past
    ``q_lens``, give 0.  ``scale`` defaults to 1 / sqrt(head_dim).  One token with its own bit set is
    single-token decode.  Returns [seqs, tokens, heads, head_dim] in q's dtype (``out`` if given).

    Statistics and sums are fp32; the exponentials are rounded to the cache's type for the product
    with V.  Key and value rows that no token of the call sees may hold anything.  A NaN or infinity in a key
    row reaches the tokens that see it; in a value row that some token of the call sees, it may reach
    tokens of the same sequence that do not."""
    if tree is None:
        raise TypeError("tree must be a CUDA tensor")
    return _paged.attend(q, k, v, table, lens, q_lens, tree, 0, 0, scale, out)


def window_attention(q, k, v, table, lens, window, sinks=0, *, q_lens=None, scale=None, out=None):
    """Causal attention with a sliding window over one layer of a cache that already holds the new tokens.

    As ``tree_attention``, but the token at position i sees the keys j <= i with j > i - window, or
    j < sinks (the first tokens, which stay visible).  ``tokens`` may be one (decode) or a prompt's
    chunk.  Pages wholly outside what the call sees are not read and may be -1 in ``table``."""
    window, sinks = int(window), int(sinks)
    if window < 1 or sinks < 0:
        raise ValueError(f"window must be at least 1 and sinks at least 0, got {window} and {sinks}")
    return _paged.attend(q, k, v, table, lens, q_lens, None, window, sinks, scale, out)


# ------------------------------------------------------------------------------ cache operators


def append_tokens(k, v, k_new, v_new, table, lens, counts=None):
    """Write new tokens' rows, ``k_new`` / ``v_new`` [layers, seqs, tokens, kv_heads, head_dim] (4-D without
    layers for a 4-D cache), at positions lens[b] + t, t < counts[b] (default: all); returns the new
    lengths.  A row whose position has no page is dropped, and the length grows all the same (attention reads
    such a position as zeros): ``reserve`` first, and look at what it granted."""
    return _paged.append_tokens(k, v, k_new, v_new, table, lens, counts)


def accept_path(k, v, table, lens, path, counts, drafts):
    """Keep a verified path of each sequence's last ``drafts`` cached tokens (an int, or int32 [seqs]): the
    row of draft path[b, i] moves to draft place i, i < counts[b]; ``path`` int32 [seqs, most] increases along
    i.  Returns the new lengths, lens - drafts + counts."""
    return _paged.accept_path(k, v, table, lens, path, counts, drafts)


def copy_pages(k, v, src, dst):
    """Copy pages ``src[i]`` to ``dst[i]`` (int32), all layers, K and V.  No page may be both read and written."""
    _paged.copy_pages(k, v, src, dst)


def fork(k, v, table, lens, refs, src, dst):
    """Make sequences ``dst[i]`` (int32, holding nothing, no repeats, up to 65535) copies of ``src[i]``: full pages
    are shared, the part of a page at the end is copied into the lowest free page, in order.  ``dst`` and ``src``
    have no sequence in common.  Updates table, lens and refs in place; returns int32 [n]: 1, or 0 where no page was
    left, the parent has no page for the tokens at its end, or a number is no sequence: the child holds nothing.
    Pages are not copied when they are written: a sequence that shares pages may append, but not ``accept``
    into a page that was full when it was shared."""
    return _paged.fork(k, v, table, lens, refs, src, dst)


def reserve(table, lens, refs, seqs, extra, page_size):
    """Map the lowest free pages so that each sequence in ``seqs`` (int32, no repeats) can hold ``extra`` (an int,
    or int32 [n]) more tokens, in order.  Updates table and refs in place; returns int32 [n]: 1, or 0 where
    the pages or the table's width ran out and nothing was mapped."""
    return _paged.reserve(table, lens, refs, seqs, extra, page_size)


def free(table, lens, refs, seqs):
    """Sequences ``seqs`` (int32) give their pages back and hold nothing; table, lens and refs in place."""
    _paged.free(table, lens, refs, seqs)


def compact(k, v, table, refs, *, table_out=None, refs_out=None):
    """Move the live pages (refs > 0) to the lowest numbers: of n, the k-th at or past n goes into the k-th hole
    before n.  ``table_out`` and ``refs_out`` (default: in place) follow; ``table`` has every sequence that holds
    pages.  Returns int32 [1]: n."""
    return _paged.compact(k, v, table, refs, table if table_out is None else table_out,
                          refs if refs_out is None else refs_out)


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
        self.whole = None  # of a part: the cache with every sequence of the pool

    def part(self, seqs):
        """A cache over some of the sequences (a slice of the slots): the same pool and its rows of the table; its
        lengths are its own from here on.  Before the whole is used for these sequences again, write them back:
        ``cache.lens[seqs] = part.lens``."""
        if not isinstance(seqs, slice):
            raise TypeError(f"seqs must be a slice of the slots, got {type(seqs).__name__}")
        part = object.__new__(Cache)
        part.k, part.v, part.refs, part.whole = self.k, self.v, self.refs, self.whole or self
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
        """As the function, for every sequence of the pool, of a part too."""
        return compact(self.k, self.v, (self.whole or self).table, self.refs)

    def tree_attention(self, layer, q, tree, **kwargs):
        return tree_attention(q, self.k[layer], self.v[layer], self.table, self.lens, tree, **kwargs)

    def window_attention(self, layer, q, window, sinks=0, **kwargs):
        return window_attention(q, self.k[layer], self.v[layer], self.table, self.lens, window, sinks, **kwargs)


__all__ = ["Cache", "accept_path", "append_tokens", "compact", "copy_pages", "fork", "free", "reserve",
           "tree_attention", "tree_mask", "window_attention"]
