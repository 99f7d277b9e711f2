"""The paged cache and its attention against plain 64-bit implementations.

Bounds of the attention tests.  With u the rounding unit of the type (2^-11 fp16, 2^-8 bf16) and
A = sum_j p_j |v_j| (p the exact probabilities): rounding the output costs u |o|, rounding each
exponential u A, an fp16 exponential below 2^-14 at most 2^-25 of the largest one (n of them, over a sum
of at least 1).  The fp32 score is off by at most d 2^-24 sum |q_i k_i| scale and its exponent's
arithmetic by 2^-21 (|s| + 1), and an error e of the scores moves o by at most 2 e A.
"""

from __future__ import annotations

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def make(torch, *, dtype="float16", dim=128, heads=8, kv_heads=2, page=16, lens=(100,), tokens=1, seed=0, spare=2,
         layers=None):
    """A cache whose unwritten rows and pages hold NaN, and queries."""
    rng = np.random.default_rng(seed)
    kind = getattr(torch, dtype)
    lens = np.asarray(lens)
    most = max(1, int(-(-lens.max() // page)) + 1)
    held = np.arange(most)[None, :] * page < lens[:, None]
    pages = int(held.sum()) + spare
    table = np.full(held.shape, -1)
    table[held] = rng.permutation(pages)[: held.sum()]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    k, v = (torch.full((pages, page, kv_heads, dim), math.nan, dtype=kind, device="cuda") for _ in range(2))
    for b, n in enumerate(lens.tolist()):
        at = np.arange(n)
        where = (torch.from_numpy(table[b, at // page]).cuda(), torch.from_numpy(at % page).cuda())
        for x in (k, v):
            x[where] = torch.randn(n, kv_heads, dim, device="cuda", generator=gen, dtype=kind)
    q = torch.randn(len(lens), tokens, heads, dim, device="cuda", generator=gen, dtype=kind) * 1.5
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    return q, k, v, ints(table), ints(lens)


def window_mask(n, m, window, sinks):
    row, col = np.arange(n - m, n)[:, None], np.arange(n)[None, :]
    return (col <= row) & ((row - col < window) | (col < sinks))


def tree_mask_of(bits, n, m):
    """bits [T, T] bool -> [m, n]: everything before the drafts, then the tree's bits."""
    mask = np.ones((m, n), dtype=bool)
    mask[:, n - m:] = bits[:m, :m]
    return mask


def pack(torch, bits):
    """[B, T, T] bool -> the words tree_attention takes."""
    B, T, _ = bits.shape
    wide = np.zeros((B, T, (T + 31) // 32 * 32), dtype=np.uint64)
    wide[:, :, :T] = bits
    words = (wide.reshape(B, T, -1, 32) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32)
    return torch.from_numpy(words.view(np.int32)).cuda()


def check(torch, out, q, k, v, table, lens, masks, scale=None):
    """Every output against the definition in 64 bits; masks[b] is [n_b, len_b]."""
    dim, page, kv_heads = q.shape[3], k.shape[1], k.shape[2]
    scale = scale or 1 / math.sqrt(dim)
    u = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}[q.dtype]
    assert out.shape == q.shape and out.dtype == q.dtype
    group = q.shape[2] // kv_heads
    for b, mask in enumerate(masks):
        m, n = mask.shape
        assert not out[b, m:].any(), "rows past q_lens are 0"
        if m == 0:
            continue
        seen = np.nonzero(mask.any(axis=0))[0]
        rows = table[b].cpu().numpy()[seen // page] * page + seen % page
        kk = k.reshape(-1, kv_heads, dim)[torch.from_numpy(rows).cuda()].double().repeat_interleave(group, dim=1)
        vv = v.reshape(-1, kv_heads, dim)[torch.from_numpy(rows).cuda()].double().repeat_interleave(group, dim=1)
        hidden = torch.from_numpy(~mask[:, seen]).cuda()
        qq = q[b, :m].double()
        s = torch.einsum("thd,jhd->htj", qq, kk) * scale
        size = torch.einsum("thd,jhd->htj", qq.abs(), kk.abs()) * scale
        err = (dim * 2.0**-24 * size + 2.0**-21 * (s.abs() + 1)).masked_fill(hidden, 0).amax(-1) if len(seen) else 0
        p = torch.softmax(s.masked_fill(hidden, -math.inf), dim=-1).nan_to_num(0.0)
        want = torch.einsum("htj,jhd->thd", p, vv)
        spread = torch.einsum("htj,jhd->thd", p, vv.abs())
        tiny = 2.0**-25 * len(seen) * (vv.abs().max() if len(seen) else 0)
        err = err.T[:, :, None] if len(seen) else 0
        bound = 1.01 * (u * want.abs() + (u + 2 * err) * spread + tiny) + 2.0**-24
        off = (out[b, :m].double() - want).abs()
        assert torch.isfinite(out[b, :m]).all()
        assert (off <= bound).all(), f"sequence {b}: {float((off / bound).max()):.3g} of the bound"


SHAPES = [  # dtype, dim, heads, kv_heads, page
    ("float16", 128, 8, 2, 16), ("bfloat16", 128, 4, 4, 64), ("float16", 64, 6, 2, 24), ("bfloat16", 64, 5, 1, 8),
    ("float16", 128, 16, 1, 128), ("bfloat16", 64, 2, 2, 256), ("float16", 64, 3, 1, 48), ("bfloat16", 128, 96, 1, 32),
    ("float16", 128, 2, 1, 200), ("float16", 64, 128, 1, 16),
    ("float16", 128, 4, 1, 136), ("bfloat16", 64, 6, 2, 184), ("bfloat16", 128, 8, 2, 72), ("float16", 64, 4, 2, 272),
]


@pytest.mark.parametrize("dtype,dim,heads,kv_heads,page", SHAPES)
@pytest.mark.parametrize("tokens,window,sinks", [(1, 50, 4), (1, 100000, 0), (7, 1, 0), (5, 64, 33), (70, 129, 1),
                                                 (300, 77, 130)])
def test_window_shapes(torch_cuda, dtype, dim, heads, kv_heads, page, tokens, window, sinks):
    from ntilang_b200 import paged

    torch = torch_cuda
    lens = [tokens, tokens + 1, tokens + 63, 640 + tokens, 1111 + tokens]
    q, k, v, table, n = make(torch, dtype=dtype, dim=dim, heads=heads, kv_heads=kv_heads, page=page, lens=lens,
                             tokens=tokens, seed=dim + tokens)
    out = paged.window_attention(q, k, v, table, n, window, sinks)
    check(torch, out, q, k, v, table, n, [window_mask(x, tokens, window, sinks) for x in lens])


@pytest.mark.parametrize("dtype,dim,heads,kv_heads,page", SHAPES)
@pytest.mark.parametrize("tokens", [1, 2, 31, 33, 64, 100])
def test_tree_shapes(torch_cuda, dtype, dim, heads, kv_heads, page, tokens):
    """Random masks, rows that see no draft among them, over prefixes from nothing up."""
    from ntilang_b200 import paged

    torch = torch_cuda
    lens = [tokens, tokens + 1, tokens + 64, 500 + tokens, 1300 + tokens]
    q, k, v, table, n = make(torch, dtype=dtype, dim=dim, heads=heads, kv_heads=kv_heads, page=page, lens=lens,
                             tokens=tokens, seed=tokens)
    bits = np.random.default_rng(tokens).random((len(lens), tokens, tokens)) < 0.3
    bits[:, ::3] = False  # with a prefix of nothing, such a row sees nothing
    out = paged.tree_attention(q, k, v, table, n, pack(torch, bits))
    check(torch, out, q, k, v, table, n, [tree_mask_of(bits[b], x, tokens) for b, x in enumerate(lens)])
    assert not out[0, ::3].any()


# Several units, whole and cut, run back to back on one CTA: more units than CTAs, units of one key
# tile and of many, lengths that end inside pages.
@pytest.mark.parametrize("dtype,dim,seqs,kv_heads,group,tokens,longest", [
    ("float16", 128, 4, 296, 1, 1, 128), ("bfloat16", 64, 3, 592, 1, 2, 640), ("float16", 64, 40, 30, 4, 8, 700),
    ("bfloat16", 128, 70, 9, 3, 5, 900), ("float16", 128, 60, 6, 4, 40, 500), ("bfloat16", 64, 33, 8, 2, 100, 700),
    ("float16", 64, 300, 3, 8, 30, 130),
])
@pytest.mark.parametrize("kind", ["tree", "window"])
def test_many_units(torch_cuda, kind, dtype, dim, seqs, kv_heads, group, tokens, longest):
    from ntilang_b200 import paged

    torch = torch_cuda
    rng = np.random.default_rng(seqs)
    lens = rng.integers(tokens, longest + 1, seqs)
    lens[0] = longest
    q, k, v, table, n = make(torch, dtype=dtype, dim=dim, heads=kv_heads * group, kv_heads=kv_heads, lens=lens,
                             tokens=tokens, seed=seqs)
    bits = np.tril(rng.random((1, tokens, tokens)) < 0.5)
    for again in range(3):
        if kind == "tree":
            out = paged.tree_attention(q, k, v, table, n, pack(torch, bits))
            masks = [tree_mask_of(bits[0], x, tokens) for x in lens.tolist()]
        else:
            out = paged.window_attention(q, k, v, table, n, 200, 10)
            masks = [window_mask(x, tokens, 200, 10) for x in lens.tolist()]
        if again == 0:
            check(torch, out, q, k, v, table, n, masks)
            first = out
        assert torch.equal(out, first)


# Short units are not cut between CTAs where the table's width or the window says that they are short: both
# ways on the same keys, with as many units as CTAs, fewer and more.
@pytest.mark.parametrize("dtype,dim,seqs,kv_heads,group,tokens,longest", [
    ("float16", 128, 7, 2, 4, 3, 500), ("bfloat16", 64, 90, 4, 3, 2, 750), ("float16", 64, 5, 2, 8, 20, 400),
    ("bfloat16", 128, 20, 3, 2, 30, 512), ("float16", 128, 3, 4, 4, 130, 480), ("bfloat16", 64, 40, 8, 3, 100, 900),
])
def test_short_units(torch_cuda, dtype, dim, seqs, kv_heads, group, tokens, longest):
    from ntilang_b200 import paged

    torch = torch_cuda
    rng = np.random.default_rng(longest)
    lens = rng.integers(tokens, longest + 1, seqs)
    lens[-1] = longest
    q, k, v, table, n = make(torch, dtype=dtype, dim=dim, heads=kv_heads * group, kv_heads=kv_heads, lens=lens,
                             tokens=tokens, seed=seqs)
    wide = torch.full((seqs, 3000), -1, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table
    bits = np.tril(rng.random((1, tokens, tokens)) < 0.5)
    for t in (table, wide):
        out = paged.tree_attention(q, k, v, t, n, pack(torch, bits))
        check(torch, out, q, k, v, t, n, [tree_mask_of(bits[0], x, tokens) for x in lens.tolist()])
        for window, sinks in ((40, 0), (120, 3), (longest, 0)):
            out = paged.window_attention(q, k, v, t, n, window, sinks)
            check(torch, out, q, k, v, t, n, [window_mask(x, tokens, window, sinks) for x in lens.tolist()])


# Sequences without keys or without new tokens: several units in a row in which a CTA has nothing to do but zeros.
@pytest.mark.parametrize("dtype,dim,kv_heads,group,tokens,longest", [
    ("float16", 128, 8, 1, 8, 35), ("bfloat16", 64, 8, 4, 1, 31), ("float16", 64, 8, 8, 4, 10), ("bfloat16", 128, 8, 5, 2, 270),
    ("float16", 128, 8, 4, 60, 200), ("bfloat16", 64, 16, 16, 8, 90),
])
def test_runs_of_empty_units(torch_cuda, dtype, dim, kv_heads, group, tokens, longest):
    from ntilang_b200 import _lib, paged

    torch = torch_cuda
    for seed in range(12):
        rng = np.random.default_rng(seed)
        lens = rng.integers(0, longest + 1, 60) * (rng.random(60) < 0.6)
        lens[3] = longest
        live = np.minimum(rng.integers(0, tokens + 1, 60) * (rng.random(60) < 0.7), lens).astype(np.int64)
        q, k, v, table, n = make(torch, dtype=dtype, dim=dim, heads=kv_heads * group, kv_heads=kv_heads, lens=lens,
                                 tokens=tokens, seed=seed)
        fresh = torch.tensor(live, dtype=torch.int32, device="cuda")
        bits = np.tril(rng.random((1, tokens, tokens)) < 0.7)
        out = paged.tree_attention(q, k, v, table, n, pack(torch, bits), q_lens=fresh)
        check(torch, out, q, k, v, table, n, [tree_mask_of(bits[0], x, m) for x, m in zip(lens.tolist(), live.tolist())])
        out = paged.window_attention(q, k, v, table, n, 50, 2, q_lens=fresh)
        check(torch, out, q, k, v, table, n, [window_mask(x, m, 50, 2) for x, m in zip(lens.tolist(), live.tolist())])
    assert _lib.device_status() == 0


@pytest.mark.parametrize("tokens", [1, 60])
def test_a_wait_that_gives_up_is_reported(torch_cuda, tokens):
    """With a limit of one poll the kernel's waits give up: it returns, says so, and the next call is right."""
    from ntilang_b200 import _lib, paged

    torch = torch_cuda
    lens = [3000, 2000, 900]
    q, k, v, table, n = make(torch, lens=lens, tokens=tokens, seed=2)
    want = paged.window_attention(q, k, v, table, n, 1 << 20)
    torch.cuda.synchronize()
    _lib.clear_device_status()
    _lib.set_wait_limit(1)
    try:
        paged.window_attention(q, k, v, table, n, 1 << 20)
        torch.cuda.synchronize()
        assert _lib.device_status() != 0
    finally:
        _lib.set_wait_limit(1 << 26)
        _lib.clear_device_status()
    assert _lib.device_status() == 0
    assert torch.equal(paged.window_attention(q, k, v, table, n, 1 << 20), want)
    assert _lib.device_status() == 0


# One shape per kind of CTA, with pieces of one tile (all of a loader's copies are out before another role gives up)
# and of more tiles than the rings hold.
@pytest.mark.parametrize("dtype,dim,heads,kv_heads,page,tokens,lens", [
    ("float16", 128, 8, 2, 16, 1, [300, 5]), ("bfloat16", 128, 8, 8, 64, 1, [40000, 30000]),
    ("float16", 64, 8, 2, 24, 2, [700]), ("bfloat16", 64, 8, 2, 64, 2, [60000, 100]),
    ("bfloat16", 128, 8, 2, 136, 20, [400, 90]), ("float16", 64, 8, 2, 16, 30, [30000]),
    ("float16", 128, 8, 2, 16, 60, [130, 61]), ("bfloat16", 128, 8, 1, 64, 200, [9000, 5000]),
    ("bfloat16", 64, 8, 2, 200, 70, [300]), ("float16", 64, 8, 2, 64, 150, [20000, 170]),
])
def test_calls_after_ones_that_gave_up(torch_cuda, dtype, dim, heads, kv_heads, page, tokens, lens):
    """A CTA that gives up lets its copies and products end before it exits: the call launched right behind it, on the
    same SMs, is right every time."""
    from ntilang_b200 import _lib, paged

    torch = torch_cuda
    q, k, v, table, n = make(torch, dtype=dtype, dim=dim, heads=heads, kv_heads=kv_heads, page=page, lens=lens,
                             tokens=tokens, seed=page)
    want = paged.window_attention(q, k, v, table, n, 1 << 20)
    check(torch, want, q, k, v, table, n, [window_mask(x, tokens, 1 << 20, 0) for x in lens])
    got = []
    try:
        for limit in (1, 2, 20) * 5:
            _lib.set_wait_limit(limit)
            paged.window_attention(q, k, v, table, n, 1 << 20)
            _lib.set_wait_limit(1 << 26)
            got.append(paged.window_attention(q, k, v, table, n, 1 << 20))
        torch.cuda.synchronize()
    finally:
        _lib.set_wait_limit(1 << 26)
        _lib.clear_device_status()
    assert all(torch.equal(x, want) for x in got)


@pytest.mark.parametrize("tokens", [1, 5, 64, 200])
def test_tree_of_parents(torch_cuda, tokens):
    """tree_mask, one tree shared by every sequence, and a chain's equality with causal attention."""
    from ntilang_b200 import paged

    torch = torch_cuda
    rng = np.random.default_rng(tokens)
    parents = np.maximum(-1, np.arange(tokens) - 1 - rng.integers(0, 3, tokens))
    bits = np.zeros((1, tokens, tokens), dtype=bool)
    for t in range(tokens):
        a = t
        while a >= 0:
            bits[0, t, a] = True
            a = parents[a]
    tree = paged.tree_mask(torch.tensor(parents[None], dtype=torch.int32, device="cuda"))
    assert torch.equal(tree, pack(torch, bits))
    lens = [tokens + 3, 900 + tokens]
    q, k, v, table, n = make(torch, lens=lens, tokens=tokens, seed=tokens)
    out = paged.tree_attention(q, k, v, table, n, tree)
    check(torch, out, q, k, v, table, n, [tree_mask_of(bits[0], x, tokens) for x in lens])
    chain = paged.tree_mask(torch.arange(-1, tokens - 1, dtype=torch.int32, device="cuda")[None])
    a = paged.tree_attention(q, k, v, table, n, chain)
    check(torch, a, q, k, v, table, n, [window_mask(x, tokens, 1 << 20, 0) for x in lens])


@pytest.mark.parametrize("tokens", [257, 1030])
def test_tree_mask_of_large_trees(torch_cuda, tokens):
    """Chains and random trees of many words, against parents' rows: a draft sees what its parent sees, and itself."""
    from ntilang_b200 import paged

    torch = torch_cuda
    parents = np.stack([np.arange(tokens) - 1, np.random.default_rng(tokens).integers(-1, np.arange(tokens))])
    bits = np.zeros((2, tokens, tokens), dtype=bool)
    for b in range(2):
        for t in range(tokens):
            if parents[b, t] >= 0:
                bits[b, t] = bits[b, parents[b, t]]
            bits[b, t, t] = True
    tree = paged.tree_mask(torch.tensor(parents, dtype=torch.int32, device="cuda"))
    assert torch.equal(tree, pack(torch, bits))


def test_tree_mask_odd_parents(torch_cuda):
    """A parent that is not an earlier draft makes a root: no walk is endless."""
    from ntilang_b200 import paged

    torch = torch_cuda
    parents = torch.tensor([[0, 5, 1, -7, 3, 5]], dtype=torch.int32, device="cuda")
    want = np.eye(6, dtype=bool)[None].copy()
    want[0, 2, 1] = want[0, 4, 3] = True
    assert torch.equal(paged.tree_mask(parents), pack(torch, want))


@pytest.mark.parametrize("kind", ["tree", "window"])
@pytest.mark.parametrize("tokens,heads", [(3, 4), (40, 8), (90, 16)])
def test_ragged_and_empty_sequences(torch_cuda, kind, tokens, heads):
    """Fewer new tokens than rows, none at all, more than the cache holds, an empty cache."""
    from ntilang_b200 import paged

    torch = torch_cuda
    lens = [0, 1, 2, 700, 700, 65, 900]
    new = [tokens, 0, tokens, 1, tokens, max(1, tokens - 2), 0]
    q, k, v, table, n = make(torch, heads=heads, lens=lens, tokens=tokens, seed=3)
    q_lens = torch.tensor(new, dtype=torch.int32, device="cuda")
    live = [min(a, b) for a, b in zip(lens, new)]
    if kind == "tree":
        bits = np.tril(np.ones((1, tokens, tokens), dtype=bool))
        out = paged.tree_attention(q, k, v, table, n, pack(torch, bits), q_lens=q_lens)
        masks = [tree_mask_of(bits[0], a, b) for a, b in zip(lens, live)]
    else:
        out = paged.window_attention(q, k, v, table, n, 30, 2, q_lens=q_lens)
        masks = [window_mask(a, b, 30, 2) for a, b in zip(lens, live)]
    check(torch, out, q, k, v, table, n, masks)


@pytest.mark.parametrize("tokens", [1, 50])
def test_evicted_pages_are_not_read(torch_cuda, tokens):
    """Pages between the sinks and the window may be gone: -1, out of range, or another's NaN."""
    from ntilang_b200 import paged

    torch = torch_cuda
    lens = [2000, 1500, 900]
    q, k, v, table, n = make(torch, lens=lens, tokens=tokens, heads=16, seed=5)
    want = paged.window_attention(q, k, v, table, n, 200, 5)
    held = set(table.flatten().tolist())
    bad = next(p for p in range(k.shape[0]) if p not in held)
    for gone in (-1, 1 << 30, -(1 << 31), bad):
        t = table.clone()
        for b, x in enumerate(lens):
            t[b, 1: (x - tokens - 199) // 16] = gone
        k[bad] = v[bad] = math.nan
        got = paged.window_attention(q, k, v, t, n, 200, 5)
        assert torch.equal(got, want), gone


@pytest.mark.parametrize("dtype,dim,heads,kv_heads,page", SHAPES)
@pytest.mark.parametrize("tokens", [1, 5, 40, 200])
def test_keys_and_values_that_no_token_sees(torch_cuda, dtype, dim, heads, kv_heads, page, tokens):
    """NaN and infinity in rows of the pages that a call reads: between the sinks and the window, and in drafts that
    no token's mask names."""
    from ntilang_b200 import paged

    torch = torch_cuda
    lens = [2000 + tokens, 640 + tokens, 1111 + tokens, 100 + tokens]
    q, k, v, table, n = make(torch, dtype=dtype, dim=dim, heads=heads, kv_heads=kv_heads, page=page, lens=lens,
                             tokens=tokens, seed=page + tokens)

    def spoil(b, at):
        rows = torch.from_numpy(table[b].cpu().numpy()[at // page]).cuda().long(), torch.from_numpy(at % page).cuda()
        k2[rows] = math.nan
        v2[rows] = torch.tensor([math.nan, math.inf, -math.inf], device="cuda", dtype=v.dtype)[
            torch.arange(len(at), device="cuda") % 3][:, None, None]

    for window, sinks in ((50, 4), (129, 0), (300, 70), (1000, 1), (5, 1 << 30), (5, 1 << 40)):
        want = paged.window_attention(q, k, v, table, n, window, sinks)
        k2, v2 = k.clone(), v.clone()
        for b, x in enumerate(lens):
            spoil(b, np.arange(min(sinks, x), max(min(sinks, x), x - tokens - window + 1)))
        out = paged.window_attention(q, k2, v2, table, n, window, sinks)
        check(torch, out, q, k, v, table, n, [window_mask(x, tokens, window, sinks) for x in lens])
        assert torch.equal(out, want), (window, sinks)
    rng = np.random.default_rng(tokens)
    bits = rng.random((len(lens), tokens, tokens)) < 0.5
    bits[:, :, rng.random(tokens) < 0.4] = False
    bits[0, :, -1] = bits[1, :, 0] = False
    tree = pack(torch, bits)
    want = paged.tree_attention(q, k, v, table, n, tree)
    k2, v2 = k.clone(), v.clone()
    for b, x in enumerate(lens):
        spoil(b, x - tokens + np.nonzero(~bits[b].any(axis=0))[0])
    out = paged.tree_attention(q, k2, v2, table, n, tree)
    check(torch, out, q, k, v, table, n, [tree_mask_of(bits[b], x, tokens) for b, x in enumerate(lens)])
    assert torch.equal(out, want)


@pytest.mark.parametrize("tokens", [1, 70])
def test_strides_and_layouts(torch_cuda, tokens):
    """One layer of a cache, heads before rows, transposed queries, a table inside a wider one."""
    from ntilang_b200 import paged

    torch = torch_cuda
    lens = [40 + tokens, 777 + tokens]
    q, k, v, table, n = make(torch, lens=lens, tokens=tokens, seed=9)
    want = paged.window_attention(q, k, v, table, n, 300, 3)
    stacked_k, stacked_v = torch.stack([torch.zeros_like(k), k]), torch.stack([torch.zeros_like(v), v])
    assert torch.equal(paged.window_attention(q, stacked_k[1], stacked_v[1], table, n, 300, 3), want)
    hk, hv = (x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in (k, v))
    assert torch.equal(paged.window_attention(q, hk, hv, table, n, 300, 3), want)
    hq = q.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    assert torch.equal(paged.window_attention(hq, k, v, table, n, 300, 3), want)
    fused = torch.cat([q, q + 1], dim=2)[:, :, : q.shape[2]]
    assert torch.equal(paged.window_attention(fused, k, v, table, n, 300, 3), want)
    wide = torch.full((table.shape[0], table.shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    wide[:, 2: 2 + table.shape[1]] = table
    out = torch.empty_like(q)
    got = paged.window_attention(q, k, v, wide[:, 2: 2 + table.shape[1]], n, 300, 3, out=out)
    assert got is out and torch.equal(out, want)
    longer = torch.full((table.shape[0], 4000), -1, dtype=torch.int32, device="cuda")
    longer[:, : table.shape[1]] = table
    got = paged.window_attention(q, k, v, longer, n, 300, 3)
    check(torch, got, q, k, v, table, n, [window_mask(x, tokens, 300, 3) for x in lens])


def test_scale(torch_cuda):
    from ntilang_b200 import paged

    torch = torch_cuda
    q, k, v, table, n = make(torch, lens=[333], tokens=4)
    out = paged.window_attention(q, k, v, table, n, 100, 4, scale=0.31)
    check(torch, out, q, k, v, table, n, [window_mask(333, 4, 100, 4)], scale=0.31)


@pytest.mark.parametrize("tokens", [1, 80])
def test_wide_scores(torch_cuda, tokens):
    """Scores that climb and fall by hundreds along the keys: the running maximum moves a lot."""
    from ntilang_b200 import paged

    torch = torch_cuda
    q, k, v, table, n = make(torch, lens=[1500], tokens=tokens, seed=4)
    at = torch.arange(1500, device="cuda")
    wave = (torch.sin(at / 97.0) * 3 + at / 500.0).to(k.dtype)
    rows = (table[0].long()[at // 16], at % 16)
    k[rows] = k[rows] * 0.1 + wave[:, None, None]
    q = q.abs()
    out = paged.window_attention(q, k, v, table, n, 1 << 20)
    check(torch, out, q, k, v, table, n, [window_mask(1500, tokens, 1 << 20, 0)])


def test_infinite_scores_match_softmax(torch_cuda):
    """A key of -inf scores is as if hidden; a NaN key makes the rows that see it NaN and no other."""
    from ntilang_b200 import paged

    torch = torch_cuda
    q, k, v, table, n = make(torch, lens=[200], tokens=3, heads=2, kv_heads=2)
    q = q.abs() + 0.1
    page, row = int(table[0, 3]), 5  # position 53
    k[page, row] = -math.inf
    out = paged.window_attention(q, k, v, table, n, 1000)
    mask = window_mask(200, 3, 1000, 0)
    mask[:, 53] = False
    check(torch, out, q, k, v, table, n, [mask])
    k[page, row] = 0
    last, row = int(table[0, 199 // 16]), 199 % 16
    k[last, row] = math.nan  # the last token's own key
    out = paged.window_attention(q, k, v, table, n, 1000)
    assert torch.isnan(out[0, 2]).all() and torch.isfinite(out[0, :2]).all()


def test_long_cache_offsets(torch_cuda):
    """Pages whose first value lies past 2^32 bytes and 2^31 values."""
    from ntilang_b200 import paged

    torch = torch_cuda
    pages, page, kv_heads, dim = 16500, 64, 16, 128  # 2.16e9 values, 4.3 GB each
    k, v = (torch.empty(pages, page, kv_heads, dim, dtype=torch.float16, device="cuda") for _ in range(2))
    assert k.numel() > 1 << 31
    lens = [600, 130]
    table = torch.full((2, 10), -1, dtype=torch.int32, device="cuda")
    table[0] = torch.arange(pages - 1, pages - 11, -1)
    table[1, :3] = torch.arange(pages - 13, pages - 10)
    for x in (k, v):
        x[pages - 13:] = torch.randn(13, page, kv_heads, dim, device="cuda", dtype=torch.float16)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn(2, 2, 32, dim, device="cuda", dtype=torch.float16)
    out = paged.window_attention(q, k, v, table, n, 1 << 20)
    check(torch, out, q, k, v, table, n, [window_mask(x, 2, 1 << 20, 0) for x in lens])
    paged.copy_pages(k, v, table[1, :1], torch.tensor([3], dtype=torch.int32, device="cuda"))
    assert torch.equal(k[3], k[pages - 13]) and torch.equal(v[3], v[pages - 13])


def test_streams_graphs_and_repeats(torch_cuda):
    """Another stream than the tensors', two streams at once, a replayed graph: the same bits."""
    from ntilang_b200 import paged

    torch = torch_cuda
    q, k, v, table, n = make(torch, lens=[5000, 3000], tokens=2, seed=8)
    want = paged.window_attention(q, k, v, table, n, 4000, 4)
    torch.cuda.synchronize()
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(5):
        for s in side:
            with torch.cuda.stream(s):
                got.append(paged.window_attention(q, k, v, table, n, 4000, 4))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)
    graph = torch.cuda.CUDAGraph()
    parents = torch.tensor([[-1, 0], [-1, -1]], dtype=torch.int32, device="cuda")
    tree = paged.tree_attention(q, k, v, table, n, paged.tree_mask(parents))
    with torch.cuda.graph(graph):
        a = paged.window_attention(q, k, v, table, n, 4000, 4)
        b = paged.tree_attention(q, k, v, table, n, paged.tree_mask(parents))
    a.zero_()
    b.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(a, want) and torch.equal(b, tree)


def test_threads(torch_cuda):
    """Threads with a stream each, whose calls need workspaces of different sizes: every call's own result."""
    import threading

    from ntilang_b200 import paged

    torch = torch_cuda
    work = [make(torch, lens=[4000 // tokens, 3000], tokens=tokens, heads=8, seed=tokens) for tokens in (1, 9, 40, 2)]
    want = [paged.window_attention(*w, 1000, 4) for w in work]
    torch.cuda.synchronize()
    got = [[] for _ in work]

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for n in range(40):
                j = (i + n) % len(work)
                got[i].append((j, paged.window_attention(*work[j], 1000, 4)))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(work))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(len(x) == 40 for x in got)
    for j, out in sum(got, []):
        assert torch.equal(out, want[j])


def test_no_rows(torch_cuda):
    from ntilang_b200 import paged

    torch = torch_cuda
    q, k, v, table, n = make(torch, lens=[10], tokens=1)
    assert paged.window_attention(q[:, :0], k, v, table, n, 4).shape == (1, 0, 8, 128)
    assert paged.window_attention(q[:0], k, v, table[:0], n[:0], 4).shape == (0, 1, 8, 128)
    assert not paged.window_attention(q, k, v, table[:, :0], n, 4).any()
    assert paged.tree_mask(torch.empty(2, 0, dtype=torch.int32, device="cuda")).shape == (2, 0, 0)


def test_refusals(torch_cuda):
    from ntilang_b200 import paged

    torch = torch_cuda
    q, k, v, table, n = make(torch, lens=[10, 20], tokens=2)
    tree = paged.tree_mask(torch.full((2, 2), -1, dtype=torch.int32, device="cuda"))
    good = dict(q=q, k=k, v=v, table=table, lens=n, window=8)

    def window(**change):
        return paged.window_attention(**{**good, **change})

    for change, kind, text in [
        (dict(q=q.cpu()), TypeError, "CUDA"), (dict(q=q.float()), ValueError, "dtype"),
        (dict(q=q.bfloat16()), ValueError, "dtype"), (dict(q=q[..., :64]), ValueError, "head_dim"),
        (dict(q=q[:, :, :3]), ValueError, "share"), (dict(k=k[None], v=v[None]), ValueError, "dimensions"),
        (dict(v=v[:, :, :1]), ValueError, "same shape"), (dict(v=v.permute(1, 0, 2, 3)), ValueError, "same shape"),
        (dict(k=k[:, :12], v=v[:, :12]), ValueError, "page_size"), (dict(table=table.long()), ValueError, "int32"),
        (dict(table=table[:1]), ValueError, "shape"), (dict(lens=n[:1]), ValueError, "shape"),
        (dict(window=0), ValueError, "window"), (dict(sinks=-1), ValueError, "sinks"),
        (dict(scale=0.0), ValueError, "scale"), (dict(scale=math.nan), ValueError, "scale"),
        (dict(q_lens=n[:1]), ValueError, "shape"), (dict(out=q), ValueError, "disjoint"),
        (dict(out=torch.empty_like(q)[:, :1]), ValueError, "out"), (dict(table=table.T), ValueError, "table"),
        (dict(q=q.transpose(2, 3).contiguous().transpose(2, 3)), ValueError, "dense"),
    ]:
        with pytest.raises(kind, match=text):
            window(**change)
    for bad in (tree[:, :1], tree.long(), tree.repeat(1, 1, 2), tree.repeat(3, 1, 1)):
        with pytest.raises(ValueError, match="tree"):
            paged.tree_attention(q, k, v, table, n, bad)
    with pytest.raises(ValueError, match="parents"):
        paged.tree_mask(tree[..., 0].float())
    with pytest.raises(ValueError, match="broadcast"):
        paged.copy_pages(k[:1].expand(4, -1, -1, -1), v[:1].expand(4, -1, -1, -1), n, n)


# ------------------------------------------------------------------------------ cache operators


def pool(torch, *, layers=2, pages=40, page=16, kv_heads=2, dim=64, seed=0, dtype="float16"):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shape = (layers, pages, page, kv_heads, dim)
    return [torch.randn(shape, device="cuda", generator=gen, dtype=getattr(torch, dtype)) for _ in range(2)]


def i32(torch, x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("page,kv_heads,dim,dtype", [(16, 2, 64, "float16"), (8, 3, 128, "bfloat16"), (5, 1, 8, "float16")])
@pytest.mark.parametrize("hnd", [False, True])
def test_append_and_accept(torch_cuda, page, kv_heads, dim, dtype, hnd):
    from ntilang_b200 import paged

    torch = torch_cuda
    k, v = pool(torch, page=page, kv_heads=kv_heads, dim=dim, dtype=dtype, pages=60)
    if hnd:
        k, v = (x.transpose(2, 3).contiguous().transpose(2, 3) for x in (k, v))
    rng = np.random.default_rng(1)
    lens, tokens = [0, 7, 33, 15, 64], 11
    table = rng.permutation(60)[:50].reshape(5, 10) if page > 5 else rng.permutation(60)[:60].reshape(5, 12)
    table[3, 1:] = -1  # no page for most of sequence 3's rows
    table[4, -1] = 1000  # out of range
    counts = [11, 4, 0, 9, 11]
    new = [torch.randn(2, 5, tokens, kv_heads, dim, device="cuda").to(k.dtype) for _ in range(2)]
    want = [x.clone() for x in (k, v)]
    for b, n in enumerate(lens):
        for t in range(counts[b]):
            j, r = divmod(n + t, page)
            if j < table.shape[1] and 0 <= table[b, j] < 60:
                for w, x in zip(want, new):
                    w[:, table[b, j], r] = x[:, b, t]
    got = paged.append_tokens(k, v, *new, i32(torch, table), i32(torch, lens), i32(torch, counts))
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    room = table.shape[1] * page
    full = [min(a + b, room) for a, b in zip(lens, counts)]
    assert got.tolist() == full

    path = np.array([np.sort(rng.permutation(11)[:6]) for _ in range(5)])
    path[1] = np.arange(6)  # nothing moves
    kept = [6, 4, 0, 5, 3]
    for b in range(5):
        prefix, n = full[b] - counts[b], min(kept[b], counts[b])
        for w in want:
            rows = []
            for i in range(n):
                j, r = divmod(prefix + path[b, i], page)
                ok = path[b, i] < counts[b] and j < table.shape[1] and 0 <= table[b, j] < 60
                rows.append(w[:, table[b, j], r].clone() if ok else None)
            for i in range(n):
                j, r = divmod(prefix + i, page)
                if rows[i] is not None and 0 <= table[b, j] < 60:
                    w[:, table[b, j], r] = rows[i]
    done = paged.accept_path(k, v, i32(torch, table), got, i32(torch, path), i32(torch, kept), i32(torch, counts))
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    assert done.tolist() == [a - b + min(c, b) for a, b, c in zip(full, counts, kept)]


def test_accept_long_path_reads_before_it_writes(torch_cuda):
    """More steps than are in flight at once, over page boundaries, sources overlapping destinations."""
    from ntilang_b200 import paged

    torch = torch_cuda
    k, v = pool(torch, layers=3, pages=20, page=8, kv_heads=4, dim=128)
    table, lens, drafts = np.random.default_rng(0).permutation(20)[None], 130, 90
    path = np.concatenate([np.arange(0, 30), np.arange(31, 89, 2)])[None]
    flat = lambda x, at: x[:, i32(torch, table[0, at // 8]).long(), i32(torch, at % 8).long()]  # noqa: E731
    want = [flat(x, 40 + path[0]).clone() for x in (k, v)]
    tail = [flat(x, np.arange(40)).clone() for x in (k, v)]
    n = path.shape[1]
    out = paged.accept_path(k, v, i32(torch, table), i32(torch, [lens]), i32(torch, path), i32(torch, [n]), drafts)
    assert out.tolist() == [40 + n]
    for x, w, t in zip((k, v), want, tail):
        assert torch.equal(flat(x, 40 + np.arange(n)), w) and torch.equal(flat(x, np.arange(40)), t)


def plain_fork(table, lens, refs, src, dst, page):
    """(granted, [(old, new, rows)]) and the three updated in place."""
    granted, copies = [], []
    unused = [p for p in range(len(refs)) if refs[p] <= 0]
    rank = 0
    for s, d in zip(src, dst):
        full, part = divmod(int(lens[s]), page)
        fresh = None
        if part:
            rank += 1
            if rank > len(unused):
                granted.append(0)
                lens[d] = 0
                continue
            fresh = unused[rank - 1]
        granted.append(1)
        table[d] = -1
        table[d, :full] = table[s, :full]
        for p in table[d, :full]:
            if p >= 0:
                refs[p] += 1
        if fresh is not None:
            table[d, full] = fresh
            refs[fresh] = 1
            copies.append((table[s, full], fresh, part))
        lens[d] = lens[s]
    return granted, copies


@pytest.mark.parametrize("pages", [24, 45, 20000])
def test_fork_and_free(torch_cuda, pages):
    """Shared pages, copied parts, children left out when the pool is full; then everything given back."""
    from ntilang_b200 import paged

    torch = torch_cuda
    page = 8
    k, v = pool(torch, pages=pages, page=page, kv_heads=1, dim=64)
    rng = np.random.default_rng(pages)
    seqs, width = 32, 9
    lens = np.zeros(seqs, dtype=np.int64)
    lens[:5] = [0, 8, 37, 64, 41]
    table = np.full((seqs, width), -1)
    ids = rng.permutation(pages)
    used = 0
    for b in range(5):
        n = -(-int(lens[b]) // page)
        table[b, :n] = ids[used: used + n]
        used += n
    table[3, 2] = -1  # a page that a window left behind
    refs = np.zeros(pages, dtype=np.int64)
    for p in table[table >= 0]:
        refs[p] += 1
    src = rng.integers(0, 5, 24)
    dst = 5 + np.arange(24)
    t, n, r = (i32(torch, x) for x in (table, lens, refs))
    before = [x.clone() for x in (k, v)]
    granted = paged.fork(k, v, t, n, r, i32(torch, src), i32(torch, dst))
    want, copies = plain_fork(table, lens, refs, src, dst, page)
    assert granted.tolist() == want
    assert (pages > 40) == all(want)
    for got, x in ((t, table), (n, lens), (r, refs)):
        assert np.array_equal(got.cpu().numpy(), x)
    for x, w in zip((k, v), before):
        for old, new, part in copies:
            w[:, new, :part] = w[:, old, :part]
        assert torch.equal(x, w)
    out = [3, 7, 100, -1, 7, 9]  # out of range and repeated sequences
    paged.free(t, n, r, i32(torch, out))
    for b in (3, 7, 9):
        for p in table[b][table[b] >= 0]:
            refs[p] -= 1
        table[b], lens[b] = -1, 0
    for got, x in ((t, table), (n, lens), (r, refs)):
        assert np.array_equal(got.cpu().numpy(), x)
    paged.free(t, n, r, i32(torch, np.arange(seqs)))
    assert not r.any() and not n.any() and (t == -1).all()


def test_fork_of_pairs_that_cannot_be(torch_cuda):
    """A pair that is refused takes no page from the others: sequences out of range, a child that is its parent, a parent
    without a page for the tokens at its end."""
    from ntilang_b200 import paged

    torch = torch_cuda
    page, pages = 8, 12
    k, v = pool(torch, pages=pages, page=page, kv_heads=1, dim=64)
    table = np.full((12, 3), -1)
    table[0, :2], table[1, :3], table[2, 0], table[3, :2] = [0, 1], [2, 3, 4], 5, [6, 7]
    table[4, :2] = [6, 7]
    table[5, :2] = [6, 900]  # no such page
    lens = np.array([12, 21, 8, 20, 13, 11] + [0] * 6)  # 3: its last page is missing
    refs = np.ones(pages, dtype=np.int64)
    refs[[6, 7]] = [3, 2]
    refs[[8, 10, 11]] = 0  # three free pages
    src = [0, 0, -1, 3, 5, 1, 2, 0, 99, 1, 4]
    dst = [99, 0, 6, 6, 7, 8, 9, 10, 11, -5, 11]
    want_granted = [0, 0, 0, 0, 0, 1, 1, 1, 0, 0, 1]
    before = [x.clone() for x in (k, v)]
    t, n, r = (i32(torch, x) for x in (table, lens, refs))
    got = paged.fork(k, v, t, n, r, i32(torch, src), i32(torch, dst))
    ok = [i for i, x in enumerate(want_granted) if x]
    granted, copies = plain_fork(table, lens, refs, [src[i] for i in ok], [dst[i] for i in ok], page)
    assert all(granted) and [c[1] for c in copies] == [8, 10, 11]
    assert got.tolist() == want_granted
    for x, w in ((t, table), (n, lens), (r, refs)):
        assert np.array_equal(x.cpu().numpy(), w)
    for x, w in zip((k, v), before):
        for old, new, part in copies:
            w[:, new, :part] = w[:, old, :part]
        assert torch.equal(x, w)


def test_reserve(torch_cuda):
    from ntilang_b200 import paged

    torch = torch_cuda
    pages, page, width = 30000, 16, 40
    refs = np.ones(pages, dtype=np.int64)
    unused = np.sort(np.random.default_rng(0).permutation(pages)[:60])
    refs[unused] = 0
    table = np.full((6, width), -1)
    lens = np.array([0, 16, 20, 300, 5, 0])
    table[1, 0], table[2, :2], table[3, 15:19], table[4, 0] = 1, [2, 3], [4, 5, 6, 7], 8
    t, n, r = (i32(torch, x) for x in (table, lens, refs))
    # 0: 7 pages; 1: one; 2 needs none; 3 holds one spare: one more, its evicted pages stay away;
    # 5: wider than the table; 4: more than is left
    got = paged.reserve(t, n, r, i32(torch, [0, 1, 2, 3, 5, 4, 77]), i32(torch, [100, 1, 12, 16, 9999, 630, 1]), page)
    assert got.tolist() == [1, 1, 1, 1, 0, 1, 0]
    table[0, :7], table[1, 1], table[3, 19] = unused[:7], unused[7], unused[8]
    table[4, 1:40] = unused[9:48]
    refs[unused[:48]] = 1
    assert np.array_equal(t.cpu().numpy(), table) and np.array_equal(r.cpu().numpy(), refs)
    got = paged.reserve(t, n, r, i32(torch, [5, 2]), 16 * 20, page)
    assert got.tolist() == [0, 0]  # 20 pages of 12: the next in line waits too
    assert np.array_equal(t.cpu().numpy(), table) and np.array_equal(r.cpu().numpy(), refs)
    got = paged.reserve(t, n, r, i32(torch, [5]), 16 * 12, page)
    assert got.tolist() == [1] and t[5, :12].tolist() == unused[48:].tolist()


def test_reserve_of_nothing_behind_a_shortage(torch_cuda):
    """A sequence that needs no page is served, whatever those before it lacked."""
    from ntilang_b200 import paged

    torch = torch_cuda
    table = [[0, -1, -1], [1, -1, -1], [-1, -1, -1], [-1, -1, -1], [3, -1, -1]]
    t, n, r = i32(torch, table), i32(torch, [8, 3, 0, 0, 8]), i32(torch, [1, 1, 0, 1])
    got = paged.reserve(t, n, r, i32(torch, [0, 1, 2, 3, 4]), i32(torch, [16, 5, 8, 0, 0]), 8)
    assert got.tolist() == [0, 1, 0, 1, 1]
    assert t.tolist() == table and r.tolist() == [1, 1, 0, 1]


def test_reserve_for_a_long_prompt(torch_cuda):
    """Thousands of pages for one sequence, from a pool with holes, beside a few for others."""
    from ntilang_b200 import paged

    torch = torch_cuda
    pages, page, width = 20000, 16, 9000
    refs = (np.random.default_rng(1).random(pages) < 0.4).astype(np.int64)
    free = np.nonzero(refs == 0)[0]
    table = np.full((3, width), -1)
    t, r = i32(torch, table), i32(torch, refs)
    got = paged.reserve(t, i32(torch, [0, 0, 0]), r, i32(torch, [2, 0, 1]), i32(torch, [40, 131072, 1]), page)
    assert got.tolist() == [1, 1, 1]
    table[2, :3], table[0, :8192], table[1, 0] = free[:3], free[3:8195], free[8195]
    refs[free[:8196]] = 1
    assert np.array_equal(t.cpu().numpy(), table) and np.array_equal(r.cpu().numpy(), refs)


def test_reserve_of_more_than_31_bits(torch_cuda):
    """Needs whose sum passes 2^31 and 2^32 are a shortage like any other: those before it are served, the others not."""
    from ntilang_b200 import paged

    torch = torch_cuda
    seqs, width, page = 2200, 1 << 20, 16
    t = torch.full((seqs, width), -1, dtype=torch.int32, device="cuda")
    n, r = torch.zeros(seqs, dtype=torch.int32, device="cuda"), torch.zeros(40, dtype=torch.int32, device="cuda")
    r[7] = 1
    extra = torch.full((seqs,), width * page, dtype=torch.int32, device="cuda")
    extra[:2], extra[2100] = i32(torch, [30, 5]), 0
    for order in (torch.arange(seqs), torch.cat([torch.arange(2, seqs), torch.arange(2)])):
        got = paged.reserve(t, n, r, order.int().cuda(), extra[order.cuda()], page).cpu()
        want = torch.zeros(seqs, dtype=torch.int32)
        want[order == 2100] = 1
        if order[0] == 0:
            want[:2] = 1
            assert t[:2, :3].tolist() == [[0, 1, -1], [2, -1, -1]] and int(r.sum()) == 4
            paged.free(t, n, r, i32(torch, [0, 1]))
        assert torch.equal(got, want)
        assert int(r.sum()) == 1 and int(t.max()) == -1


@pytest.mark.parametrize("pages,share", [(1, 1.0), (37, 0.5), (37, 0.0), (64, 1.0), (9001, 0.3)])
@pytest.mark.parametrize("in_place", [True, False])
def test_compact(torch_cuda, pages, share, in_place):
    from ntilang_b200 import paged

    torch = torch_cuda
    k, v = pool(torch, layers=2, pages=pages, page=8, kv_heads=1, dim=64)
    rng = np.random.default_rng(pages)
    live = np.sort(rng.permutation(pages)[: int(pages * share)])
    refs = np.zeros(pages, dtype=np.int64)
    refs[live] = rng.integers(1, 4, len(live))
    table = np.full((7, -(-pages // 7) + 2), -1)
    table.reshape(-1)[rng.permutation(table.size)[: len(live)]] = rng.permutation(live)
    table[6, -1] = 1 << 20  # not a page
    n = len(live)
    new = np.arange(pages)
    new[[p for p in live if p >= n]] = [p for p in range(n) if refs[p] == 0]
    want_refs = np.zeros_like(refs)
    want_refs[new[live]] = refs[live]
    want_table = np.where((table >= 0) & (table < pages), new[np.clip(table, 0, pages - 1)], -1)
    want = [x.clone() for x in (k, v)]
    for w in want:
        for p in live[live >= n]:
            w[:, new[p]] = w[:, p]
    t, r = i32(torch, table), i32(torch, refs)
    t_out, r_out = (t, r) if in_place else (torch.empty_like(t), torch.empty_like(r))
    got = paged.compact(k, v, t, r, **({} if in_place else dict(table_out=t_out, refs_out=r_out)))
    assert got.tolist() == [n]
    assert np.array_equal(t_out.cpu().numpy(), want_table) and np.array_equal(r_out.cpu().numpy(), want_refs)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    if not in_place:
        assert np.array_equal(t.cpu().numpy(), table) and np.array_equal(r.cpu().numpy(), refs)


def test_part_of_a_cache(torch_cuda):
    """Closing up the pool through a part, or through the whole while a part is in use, moves every sequence's pages
    with its table; a part is a slice of the slots."""
    from ntilang_b200 import paged

    torch = torch_cuda
    for whole in (False, True):
        c = paged.Cache(layers=1, pages=24, page_size=8, kv_heads=1, head_dim=64, seqs=4, max_pages=5)
        gen = torch.Generator(device="cuda").manual_seed(3)
        rnd = lambda *s: torch.randn(*s, device="cuda", generator=gen, dtype=torch.float16)  # noqa: E731
        for b in (1, 3, 2, 0):  # sequence 0's pages are the ones that move
            assert c.reserve(i32(torch, [b]), 30).tolist() == [1]
        c.append(rnd(1, 4, 30, 1, 64), rnd(1, 4, 30, 1, 64), i32(torch, [30, 17, 25, 9]))
        c.free(i32(torch, [1]))
        part = c.part(slice(2, 4))
        q = rnd(4, 1, 2, 64)
        want = c.window_attention(0, q, 1 << 20)
        live = int((c if whole else part).compact())
        assert live == int((c.refs > 0).sum()) and int(c.table.max()) == live - 1
        assert torch.equal(c.window_attention(0, q, 1 << 20), want)
        assert torch.equal(part.window_attention(0, q[2:], 1 << 20), want[2:])
        for seqs in ([2, 3], 2, i32(torch, [2, 3])):
            with pytest.raises(TypeError, match="slice"):
                c.part(seqs)


def test_copy_pages(torch_cuda):
    from ntilang_b200 import paged

    torch = torch_cuda
    k, v = pool(torch, pages=12, page=6, kv_heads=3, dim=40)
    want = [x.clone() for x in (k, v)]
    for w in want:
        w[:, [7, 8]] = w[:, [1, 2]]
    paged.copy_pages(k, v, i32(torch, [1, 2, 50, 3, -1]), i32(torch, [7, 8, 9, -4, 3]))
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    paged.copy_pages(k[0], v[0], i32(torch, [0]), i32(torch, [11]))
    assert torch.equal(k[0, 11], k[0, 0]) and torch.equal(k[1], want[0][1])


def test_cache_refusals(torch_cuda):
    from ntilang_b200 import paged

    torch = torch_cuda
    c = paged.Cache(layers=2, pages=8, page_size=16, kv_heads=2, head_dim=64, seqs=3, max_pages=4)
    rows = torch.zeros(2, 3, 5, 2, 64, dtype=torch.float16, device="cuda")
    one = i32(torch, [0])
    for call, kind, text in [
        (lambda: c.append(rows[0], rows[0]), ValueError, "dimensions"),
        (lambda: c.append(rows.float(), rows.float()), ValueError, "dtype"),
        (lambda: c.append(rows[:1], rows[:1]), ValueError, "k_new"),
        (lambda: c.append(rows, rows[:, :, :, :, :32]), ValueError, "same shape"),
        (lambda: c.append(rows[:, :2], rows[:, :2]), ValueError, "table"),
        (lambda: c.append(rows, rows, c.lens[:2]), ValueError, "counts"),
        (lambda: c.accept(one[None], one, 5), ValueError, "path"),
        (lambda: c.accept(c.table, c.lens, -1), ValueError, "drafts"),
        (lambda: c.fork(one, i32(torch, [1, 2])), ValueError, "dst"),
        (lambda: c.fork(one.long(), one.long()), ValueError, "int32"),
        (lambda: c.reserve(one, -1), ValueError, "extra"),
        (lambda: c.free(one.cpu()), TypeError, "CUDA"),
        (lambda: paged.compact(c.k, c.v, c.table, c.refs[:4]), ValueError, "refs"),
        (lambda: paged.compact(c.k, c.v, c.table, c.refs, table_out=c.table[:1]), ValueError, "table_out"),
    ]:
        with pytest.raises(kind, match=text):
            call()


def test_tables_that_are_written_are_not_broadcast(torch_cuda):
    from ntilang_b200 import paged

    torch = torch_cuda
    k, v = pool(torch, pages=8, page=8, kv_heads=1, dim=64)
    one = torch.full((1, 4), -1, dtype=torch.int32, device="cuda")
    n, r, seqs = i32(torch, [0, 0, 0]), i32(torch, [0] * 8), i32(torch, [0, 1])
    lapping = torch.full((12,), -1, dtype=torch.int32, device="cuda").as_strided((3, 4), (2, 1))
    for table in (one.expand(3, 4), lapping):
        for call in (lambda: paged.reserve(table, n, r, seqs, 3, 8), lambda: paged.free(table, n, r, seqs),
                     lambda: paged.fork(k, v, table, n, r, seqs[:1], seqs[1:]), lambda: paged.compact(k, v, table, r),
                     lambda: paged.compact(k, v, one.repeat(3, 1), r, table_out=table)):
            with pytest.raises(ValueError, match="broadcast"):
                call()
    # Reading is another matter: three sequences over the same pages.
    one[0, :2] = i32(torch, [5, 2])
    q = torch.randn(3, 2, 2, 64, device="cuda", dtype=torch.float16)
    lens = i32(torch, [16, 9, 3])
    want = paged.window_attention(q, k[0], v[0], one.repeat(3, 1), lens, 5, 1)
    assert torch.equal(paged.window_attention(q, k[0], v[0], one.expand(3, 4), lens, 5, 1), want)
    out = torch.empty(3, 4, dtype=torch.int32, device="cuda")
    paged.compact(k, v, one.expand(3, 4), i32(torch, [0, 0, 1, 0, 0, 1, 0, 0]), table_out=out,
                  refs_out=torch.empty_like(r))
    assert out.tolist() == [[1, 0, -1, -1]] * 3


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_broadcast_queries_and_heads(torch_cuda, dtype):
    """Expanded tensors (stride 0): one sequence's queries for all, one key head's rows for several."""
    from ntilang_b200 import paged

    torch = torch_cuda
    for tokens in (1, 5, 70):
        q, k, v, table, n = make(torch, dtype=dtype, lens=[300 + tokens, 77 + tokens], tokens=tokens, heads=4, kv_heads=1)
        for x in (q[:1].expand(2, -1, -1, -1), q[:, :, :1].expand(-1, -1, 4, -1), q[:, :1].expand(-1, tokens, -1, -1)):
            assert torch.equal(paged.window_attention(x, k, v, table, n, 100, 2),
                               paged.window_attention(x.contiguous(), k, v, table, n, 100, 2))
        wide = [x.expand(-1, -1, 2, -1) for x in (k, v)]
        assert torch.equal(paged.window_attention(q, *wide, table, n, 100, 2),
                           paged.window_attention(q, *(x.contiguous() for x in wide), table, n, 100, 2))


def test_a_serving_round(torch_cuda):
    """Prompt, fork, drafts, verification and windowed decode, against dense tensors kept beside."""
    from ntilang_b200 import paged

    torch = torch_cuda
    L, H, KV, D = 2, 8, 2, 64
    c = paged.Cache(layers=L, pages=64, page_size=16, kv_heads=KV, head_dim=D, seqs=4, max_pages=16)
    gen = torch.Generator(device="cuda").manual_seed(0)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=gen, dtype=torch.float16)  # noqa: E731
    first = i32(torch, [0, 1])
    assert c.reserve(first, 100).tolist() == [1, 1]
    new = rnd(2, L, 4, 50, KV, D)
    c.append(new[0], new[1], i32(torch, [50, 37, 0, 0]))
    assert c.fork(first, i32(torch, [2, 3])).tolist() == [1, 1]
    dense = [[new[:, :, b % 2, : (50, 37)[b % 2]]] for b in range(4)]
    assert c.reserve(i32(torch, [0, 1, 2, 3]), 20).tolist() == [1] * 4
    drafts = rnd(2, L, 4, 7, KV, D)
    parents = i32(torch, [[-1, 0, 0, 1, 1, 2, 3]] * 4)
    c.append(drafts[0], drafts[1])
    q = rnd(4, 7, H, D)
    bits = paged.tree_mask(parents)
    mask = np.zeros((7, 7), dtype=bool)
    for t in range(7):
        for s in range(7):
            mask[t, s] = int(bits[0, t, 0]) >> s & 1
    lens = c.lens.tolist()
    assert lens == [57, 44, 57, 44]
    for layer in range(L):
        out = c.tree_attention(layer, q, bits)
        check(torch, out, q, c.k[layer], c.v[layer], c.table, c.lens, [tree_mask_of(mask, n, 7) for n in lens])
    path, counts = i32(torch, [[0, 1, 3, 6], [0, 2, 5, 5], [0, 1, 4, 4], [0, 0, 0, 0]]), i32(torch, [4, 3, 3, 1])
    c.accept(path, counts, 7)
    assert c.lens.tolist() == [54, 40, 53, 38]
    for b in range(4):
        keep = path[b, : counts[b]].long()
        dense[b] = torch.cat([*dense[b], drafts[:, :, b][:, :, keep]], dim=2)
        n = int(c.lens[b])
        at = torch.arange(n, device="cuda")
        rows = c.table[b].long()[at // 16], at % 16
        assert torch.equal(c.k[:, rows[0], rows[1]], dense[b][0]) and torch.equal(c.v[:, rows[0], rows[1]], dense[b][1])
    one = rnd(4, 1, H, D)
    out = c.window_attention(1, one, 20, 4)
    check(torch, out, one, c.k[1], c.v[1], c.table, c.lens, [window_mask(n, 1, 20, 4) for n in c.lens.tolist()])
    c.free(first)
    live = int(c.compact())
    assert live == int((c.refs > 0).sum()) and int(c.table.max()) < live
    again = c.window_attention(1, one, 20, 4)
    assert torch.equal(again[2:], out[2:]) and not again[:2].any()


def test_speculative_decoding_example(torch_cuda):
    """The example runs the operators together and checks its text against plain decoding itself."""
    import importlib.util
    from pathlib import Path

    path = Path(__file__).resolve().parents[1] / "examples" / "speculative_decode.py"
    spec = importlib.util.spec_from_file_location("speculative_decode", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    assert mod.main(seqs=3, prompt_len=45, steps=30) <= 31
