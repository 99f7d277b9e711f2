"""Cases for the paged key/value cache and the attention that reads it.

Three operators, each in a plain form (elementary torch operations in 32 bits, rounded once) and
through ``ntilang_b200.paged``:

* ``tree``: attention of a tree of drafted tokens over the cache (one drafted token is decode);
* ``window``: causal attention with a sliding window and a few first tokens that stay visible;
* ``pages``: upkeep of the cache — append and accept a verified path, fork and free, compact.

A cache is ``k``/``v`` [layers, pages, page_size, kv_heads, head_dim] (attention takes one layer of
it), ``table`` int32 [sequences, max_pages] (-1: no page) and ``lens`` int32 [sequences].
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # One user, 16 drafted tokens over a short context: latency.
        dict(name="tree-1x16", op="tree", batch=1, tokens=16, heads=32, kv_heads=8, dim=128, page=16, lo=1000, hi=1000,
             dtype="fp16"),
        # A small server's verification step: ragged contexts, an odd tree.
        dict(name="tree-16x27", op="tree", batch=16, tokens=27, heads=32, kv_heads=8, dim=128, page=32, lo=500,
             hi=9000, dtype="bf16"),
        # Many users with short drafts, multi-head attention (no shared heads).
        dict(name="tree-64x8-mha", op="tree", batch=64, tokens=8, heads=16, kv_heads=16, dim=64, page=64, lo=1024,
             hi=8192, dtype="bf16"),
        # Long contexts and wide trees: 256 query rows for every key that is read.
        dict(name="tree-4x64-long", op="tree", batch=4, tokens=64, heads=32, kv_heads=8, dim=128, page=64, lo=32768,
             hi=65536, dtype="fp16"),
        # One user, one token: latency of a windowed decode step.
        dict(name="window-1x1", op="window", batch=1, tokens=1, heads=32, kv_heads=8, dim=128, page=16, lo=5000,
             hi=5000, window=1024, sinks=4, evict=True, dtype="fp16"),
        # A server's decode step: long conversations, pages outside the window given back.
        dict(name="window-64x1", op="window", batch=64, tokens=1, heads=32, kv_heads=8, dim=128, page=16, lo=2000,
             hi=32768, window=4096, sinks=4, evict=True, dtype="bf16"),
        # Odd everything: three query heads to a key head, ragged chunks, a window inside a page.
        dict(name="window-3x37-odd", op="window", batch=3, tokens=37, heads=24, kv_heads=8, dim=64, page=24, lo=40,
             hi=3000, window=100, sinks=17, evict=False, ragged=True, dtype="fp16"),
        # A prompt chunk over the cache.
        dict(name="window-prompt", op="window", batch=1, tokens=4096, heads=32, kv_heads=8, dim=128, page=64, lo=8192,
             hi=8192, window=2048, sinks=4, evict=False, dtype="bf16"),
        # The end of a verification step: the drafts' rows go in, the accepted ones close up.
        dict(name="pages-step", op="pages", kind="step", layers=4, batch=16, tokens=27, kv_heads=8, dim=128, page=16,
             lo=200, hi=3000, dtype="bf16"),
        # A prompt's rows going into the cache, all layers at once.
        dict(name="pages-prompt", op="pages", kind="step", layers=16, batch=2, tokens=2048, kv_heads=8, dim=128,
             page=64, lo=64, hi=100, dtype="fp16"),
        # A beam search step: 48 children replace the last ones, sharing their parents' full pages.
        dict(name="pages-fork", op="pages", kind="fork", layers=16, parents=8, children=48, kv_heads=8, dim=128,
             page=32, lo=500, hi=6000, dtype="fp16"),
        # A pool that half emptied, closed up before it is shrunk.
        dict(name="pages-compact", op="pages", kind="compact", layers=8, pages=4096, live=0.5, batch=16, kv_heads=8,
             dim=128, page=32, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (16, 16, 64), (24, 8, 64), (32, 4, 128), (8, 1, 128), (12, 4, 64)])
    page = rng.choice([8, 16, 24, 32, 64, 128, 256])
    dtype = rng.choice(["fp16", "bf16"])
    op = rng.choice(["tree", "tree", "window", "window", "pages"])
    base = dict(heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)
    if op == "tree":
        batch, tokens = _log(rng, 1, 64), _log(rng, 1, 64)
        hi = _log(rng, tokens + 8, min(65536, 262144 // batch))
        return dict(base, op="tree", batch=batch, tokens=tokens, lo=max(tokens, int(hi * rng.uniform(0.2, 1.0))), hi=hi)
    if op == "window":
        if rng.random() < 0.5:
            batch, tokens = _log(rng, 1, 64), rng.randint(1, 4)
            hi = _log(rng, 16, min(32768, 1 << 20 >> (batch.bit_length() - 1)))
        else:
            batch, tokens = rng.randint(1, 4), _log(rng, 16, 2048)
            hi = _log(rng, tokens, min(16384, (1 << 24) // (batch * tokens)))
        return dict(base, op="window", batch=batch, tokens=tokens, lo=max(tokens, int(hi * rng.uniform(0.2, 1.0))),
                    hi=hi, window=_log(rng, 8, 8192), sinks=rng.choice([0, 1, 4, 33]), evict=rng.random() < 0.5,
                    ragged=rng.random() < 0.5)
    kind = rng.choice(["step", "fork", "compact"])
    base = dict(kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, op="pages", kind=kind, layers=rng.randint(1, 16))
    if kind == "step":
        return dict(base, batch=_log(rng, 1, 32), tokens=_log(rng, 1, 64), lo=_log(rng, 16, 500), hi=_log(rng, 500, 4000))
    if kind == "fork":
        return dict(base, parents=_log(rng, 1, 16), children=_log(rng, 1, 64), lo=_log(rng, 16, 500),
                    hi=_log(rng, 500, 4000))
    return dict(base, pages=_log(rng, 64, 512), live=round(rng.uniform(0.1, 0.9), 3), batch=_log(rng, 1, 32))


# ------------------------------------------------------------------------------ sizes of a case


def _spread(lo, hi, n):
    """n lengths from lo to hi, evenly over their logarithm."""
    if n == 1:
        return np.array([hi], dtype=np.int64)
    return np.round(np.exp(np.linspace(math.log(lo), math.log(hi), n))).astype(np.int64)


def _tokens(case):
    """New tokens of each sequence: all of them, or a ragged share."""
    n, t = case["batch"], case["tokens"]
    if not case.get("ragged"):
        return np.full(n, t, dtype=np.int64)
    return np.maximum(1, t - (np.arange(n, dtype=np.int64) * 5) % t)


def _first_key(case, lens, new):
    """First position inside the window of each sequence's first new token."""
    return np.maximum(0, lens - new - case["window"] + 1)


def _path(case):
    """Accepted drafts of each sequence: (path [batch, most], counts [batch])."""
    n, t = case["batch"], case["tokens"]
    most = (t + 1) // 2
    path = np.minimum(2 * np.arange(most)[None, :] + (np.arange(n)[:, None] % 2), t - 1)
    counts = 1 + np.arange(n) % most
    return path, np.minimum(counts, np.maximum(1, t // 2))


def work(case):
    size = case["kv_heads"] * case["dim"] * 2  # one token's keys or values, in bytes
    if case["op"] == "pages":
        rows = 0
        if case["kind"] == "step":
            path, counts = _path(case)
            moved = (path != np.arange(path.shape[1])) & (np.arange(path.shape[1]) < counts[:, None])
            rows = case["batch"] * case["tokens"] + int(moved.sum())
        elif case["kind"] == "fork":
            lens = _spread(case["lo"], case["hi"], case["parents"])[np.arange(case["children"]) % case["parents"]]
            rows = int((lens % case["page"]).sum())
        else:
            rows = _movers(case)[1] * case["page"]
        return {"bytes": max(1, 4 * rows * size * case["layers"]), "flops": 0}
    lens, new = _spread(case["lo"], case["hi"], case["batch"]), _tokens(case)
    qo = 4 * case["batch"] * case["tokens"] * case["heads"] * case["dim"]
    if case["op"] == "tree":
        pairs = int(((lens - new) * new + new).sum())
        return {"bytes": int(lens.sum()) * 2 * size + qo, "flops": 4 * case["dim"] * case["heads"] * pairs}
    keys, pairs = 0, 0
    for n, m in zip(lens.tolist(), new.tolist()):
        pos = np.arange(n - m, n)
        first = np.maximum(0, pos - case["window"] + 1)
        pairs += int((pos + 1 - first + np.minimum(first, case["sinks"])).sum())
        keys += int(n - first[0] + min(first[0], case["sinks"]))
    return {"bytes": keys * 2 * size + qo, "flops": 4 * case["dim"] * case["heads"] * pairs}


def _movers(case):
    """(live pages, live pages that lie past them) of a pool to compact."""
    live = max(1, int(case["pages"] * case["live"]))
    return live, int(live * (1 - live / case["pages"]))


# ------------------------------------------------------------------------------ inputs


def _gpu(x, dtype=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(x)).to(dtype).cuda()


def _normal(seed, shape, dtype, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=gen, device="cuda", dtype=dtype)
    return x.mul_(scale) if scale != 1.0 else x


def _table(rng, held, pages):
    """Page numbers in no order for the True places of ``held``."""
    table = np.full(held.shape, -1, dtype=np.int64)
    table[held] = rng.permutation(pages)[: int(held.sum())]
    return table


def prepare(case, seed):
    rng = np.random.RandomState(seed % (1 << 32))
    dtype, page = DTYPES[case["dtype"]], case["page"]
    if case["op"] == "pages":
        return _prepare_pages(case, seed, rng, dtype, page)
    batch, tokens = case["batch"], case["tokens"]
    order = rng.permutation(batch)
    lens, new = _spread(case["lo"], case["hi"], batch)[order], _tokens(case)[order]
    most = int(-(-lens.max() // page)) + 1
    at = np.arange(most) * page
    held = at[None, :] < lens[:, None]
    if case["op"] == "window" and case["evict"]:
        first = _first_key(case, lens, new)
        held &= (at[None, :] + page > first[:, None]) | (at[None, :] < case["sinks"])
    pages = int(held.sum()) + 3
    shape = (pages, page, case["kv_heads"], case["dim"])
    s = {"case": case, "k": _normal(seed, shape, dtype), "v": _normal(seed + 1, shape, dtype),
         "table": _gpu(_table(rng, held, pages)), "lens": _gpu(lens),
         "q": _normal(seed + 2, (batch, tokens, case["heads"], case["dim"]), dtype, 1.5),
         "new": _gpu(new) if case.get("ragged") else None}
    if case["op"] == "tree":
        back = 1 + rng.randint(0, 3, size=(batch, tokens))
        s["parents"] = _gpu(np.maximum(-1, np.arange(tokens)[None, :] - back))
    return s


def _prepare_pages(case, seed, rng, dtype, page):
    layers, heads, dim = case["layers"], case["kv_heads"], case["dim"]
    s = {"case": case}
    if case["kind"] == "step":
        batch, tokens = case["batch"], case["tokens"]
        lens = _spread(case["lo"], case["hi"], batch)
        held = np.arange(-(-(int(lens.max()) + tokens) // page))[None, :] * page < (lens + tokens)[:, None]
        pages = int(held.sum()) + 1
        path, counts = _path(case)
        new = (layers, batch, tokens, heads, dim)
        s |= {"table": _gpu(_table(rng, held, pages)), "lens": _gpu(lens), "path": _gpu(path), "counts": _gpu(counts),
              "k_new": _normal(seed + 2, new, dtype), "v_new": _normal(seed + 3, new, dtype)}
    elif case["kind"] == "fork":
        parents, children = case["parents"], case["children"]
        lens = np.concatenate([_spread(case["lo"], case["hi"], parents), np.zeros(children, dtype=np.int64)])
        held = np.arange(-(-int(lens.max()) // page) + 1)[None, :] * page < lens[:, None]
        pages = int(held.sum()) + children + 5
        table = _table(rng, held, pages)
        refs = np.bincount(table[held], minlength=pages)
        s |= {"table": _gpu(table), "lens": _gpu(lens), "refs": _gpu(refs),
              "src": _gpu(np.arange(children) % parents), "dst": _gpu(parents + np.arange(children))}
    else:
        pages, batch = case["pages"], case["batch"]
        live, movers = _movers(case)
        at = np.concatenate([rng.permutation(live)[: live - movers], live + rng.permutation(pages - live)[:movers]])
        table = np.full((batch, -(-live // batch) + 1), -1, dtype=np.int64)
        table.reshape(-1)[rng.permutation(table.size)[:live]] = rng.permutation(at)
        refs = np.zeros(pages, dtype=np.int64)
        refs[at] = 1
        s |= {"table": _gpu(table), "refs": _gpu(refs)}
        s |= {"table_out": torch.empty_like(s["table"]), "refs_out": torch.empty_like(s["refs"])}
    shape = (layers, pages, page, heads, dim)
    return s | {"k": _normal(seed, shape, dtype), "v": _normal(seed + 1, shape, dtype)}


# ------------------------------------------------------------------------------ a pass


def run(s):
    case = s["case"]
    if case["op"] == "pages":
        return _run_pages(s, case)
    if own:
        from ntilang_b200 import paged

        if case["op"] == "tree":
            return paged.tree_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], paged.tree_mask(s["parents"]))
        return paged.window_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], case["window"], case["sinks"],
                                      q_lens=s["new"])
    q, lens, tokens = s["q"], s["lens"].long(), case["tokens"]
    new = torch.full_like(lens, tokens) if s["new"] is None else s["new"].long()
    at = torch.arange(s["table"].shape[1] * case["page"], device="cuda")
    index = torch.arange(tokens, device="cuda")
    if case["op"] == "tree":
        draft = at[None, :] - (lens - new)[:, None]  # which draft a position holds
        seen = _ancestors(s["parents"]).gather(2, draft.clamp(0, tokens - 1)[:, None, :].expand(-1, tokens, -1))
        visible = (draft < 0)[:, None, :] | (seen & (draft < new[:, None])[:, None, :])
    else:
        pos = (lens - new)[:, None] + index[None, :]
        ahead = pos[:, :, None] - at[None, None, :]
        visible = (ahead >= 0) & ((ahead < case["window"]) | (at < case["sinks"])[None, None, :])
    visible = visible & (index[None, :] < new[:, None])[:, :, None]
    return _attention(q, s["k"], s["v"], s["table"], visible)


def _ancestors(parents):
    """[batch, T, T]: whether s is t or an ancestor of t.  I + A + A^2 + ... = (I - A)^-1 of the parent matrix A."""
    n = parents.shape[1]
    step = (parents[:, :, None] == torch.arange(n, device=parents.device)).float()
    eye = torch.eye(n, device=parents.device).expand_as(step)
    return torch.linalg.solve_triangular(eye - step, eye, upper=False, unitriangular=True) > 0.5


def _attention(q, k, v, table, visible):
    batch, tokens, heads, dim = q.shape
    kv_heads = k.shape[2]
    page = table.clamp(min=0).long()
    usable = visible.any(dim=1)[:, :, None, None]
    keys = k[page].reshape(batch, -1, kv_heads, dim)
    values = v[page].reshape(batch, -1, kv_heads, dim)
    keys = torch.where(usable, keys, 0).float().permute(0, 2, 3, 1)
    values = torch.where(usable, values, 0).float().permute(0, 2, 1, 3)
    rows = q.float().reshape(batch, tokens, kv_heads, heads // kv_heads, dim).permute(0, 2, 3, 1, 4)
    rows = rows.reshape(batch, kv_heads, -1, dim)
    score = torch.matmul(rows, keys).mul_(1.0 / math.sqrt(dim)).reshape(batch, heads, tokens, -1)
    score = score.masked_fill_(~visible[:, None], float("-inf"))
    top = score.amax(dim=-1, keepdim=True).clamp_(min=-3e38)
    score = score.sub_(top).exp_()
    total = score.sum(dim=-1, keepdim=True)
    o = torch.matmul(score.reshape(batch, kv_heads, -1, score.shape[-1]), values).reshape(batch, heads, tokens, dim)
    o = torch.where(total > 0, o / total, 0)
    return o.permute(0, 2, 1, 3).to(q.dtype).contiguous()


def _run_pages(s, case):
    k, v, table, page = s["k"], s["v"], s["table"], case["page"]
    if own:
        from ntilang_b200 import paged

        if case["kind"] == "step":
            full = paged.append_tokens(k, v, s["k_new"], s["v_new"], table, s["lens"])
            lens = paged.accept_path(k, v, table, full, s["path"], s["counts"], case["tokens"])
            return {"k": k, "v": v, "lens": lens}
        if case["kind"] == "fork":
            paged.free(table, s["lens"], s["refs"], s["dst"])
            granted = paged.fork(k, v, table, s["lens"], s["refs"], s["src"], s["dst"])
            return {"k": k, "v": v, "table": table, "lens": s["lens"], "refs": s["refs"], "granted": granted}
        live = paged.compact(k, v, table, s["refs"], table_out=s["table_out"], refs_out=s["refs_out"])
        return {"k": k, "v": v, "table": s["table_out"], "refs": s["refs_out"], "live": live}
    if case["kind"] == "step":
        at = s["lens"][:, None].long() + torch.arange(case["tokens"], device="cuda")
        pages = table.gather(1, at // page).long()
        k[:, pages, at % page] = s["k_new"]
        v[:, pages, at % page] = s["v_new"]
        step = torch.arange(s["path"].shape[1], device="cuda")
        moved = (step[None, :] < s["counts"][:, None]) & (step[None, :] != s["path"])
        old, new = s["lens"][:, None].long() + s["path"], s["lens"][:, None].long() + step[None, :]
        old_page, new_page = table.gather(1, old // page).long()[moved], table.gather(1, new // page).long()[moved]
        k[:, new_page, (new % page)[moved]] = k[:, old_page, (old % page)[moved]]
        v[:, new_page, (new % page)[moved]] = v[:, old_page, (old % page)[moved]]
        return {"k": k, "v": v, "lens": s["lens"] + s["counts"]}
    refs = s["refs"]
    if case["kind"] == "fork":
        lens, src, dst = s["lens"], s["src"].long(), s["dst"].long()
        held = table[dst]
        refs.sub_(torch.bincount(held[held >= 0].long(), minlength=refs.numel()).int())
        size = lens[src].long()
        full, part = size // page, size % page
        rank = (part > 0).cumsum(0) - 1
        unused = torch.nonzero(refs == 0)[:, 0]
        granted = (part == 0) | (rank < unused.numel())
        column = torch.arange(table.shape[1], device="cuda")
        rows = torch.where((column < full[:, None]) & granted[:, None], table[src], -1)
        refs.add_(torch.bincount(rows[rows >= 0].long(), minlength=refs.numel()).int())
        copied = (part > 0) & granted
        old, new = table[src[copied], full[copied]].long(), unused[rank[copied]]
        rows[copied, full[copied]] = new.int()
        refs[new] = 1
        table[dst] = rows
        lens[dst] = torch.where(granted, size, 0).int()
        inside = (torch.arange(page, device="cuda") < part[copied][:, None])[None, :, :, None, None]
        k[:, new] = torch.where(inside, k[:, old], k[:, new])
        v[:, new] = torch.where(inside, v[:, old], v[:, new])
        return {"k": k, "v": v, "table": table, "lens": lens, "refs": refs, "granted": granted.int()}
    live, index = refs > 0, torch.arange(refs.numel(), device="cuda")
    count = live.sum()
    holes, movers = torch.nonzero(~live & (index < count))[:, 0], torch.nonzero(live & (index >= count))[:, 0]
    index[movers] = holes
    k[:, holes] = k[:, movers]
    v[:, holes] = v[:, movers]
    refs_out = torch.zeros_like(refs)
    refs_out[index[live]] = refs[live]
    table_out = torch.where(table >= 0, index[table.clamp(min=0).long()].int(), -1)
    return {"k": k, "v": v, "table": table_out, "refs": refs_out, "live": count.int().reshape(1)}


# ------------------------------------------------------------------------------ definitions in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "pages":
        return _exact_pages(s, case)
    page, dim, group = case["page"], case["dim"], case["heads"] // case["kv_heads"]
    table, lens = s["table"].cpu().numpy(), s["lens"].cpu().numpy()
    new = np.full(case["batch"], case["tokens"]) if s["new"] is None else s["new"].cpu().numpy()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        n, m = int(lens[b]), int(new[b])
        if case["op"] == "tree":
            parents = s["parents"][b].cpu().numpy()
            mask = np.ones((m, n), dtype=bool)
            mask[:, n - m:] = False
            for t in range(m):
                a = t
                while a >= 0:
                    mask[t, n - m + a] = True
                    a = int(parents[a])
        else:
            row, col = np.arange(n - m, n)[:, None], np.arange(n)[None, :]
            mask = (col <= row) & ((row - col < case["window"]) | (col < case["sinks"]))
        keys = np.nonzero(mask.any(axis=0))[0]
        where = torch.from_numpy(table[b, keys // page].astype(np.int64) * page + keys % page).cuda()
        hidden = torch.from_numpy(~mask[:, keys]).cuda()
        for h in range(case["kv_heads"]):
            kk = s["k"].reshape(-1, case["kv_heads"], dim)[where, h].double()
            vv = s["v"].reshape(-1, case["kv_heads"], dim)[where, h].double()
            for g in range(group):
                score = s["q"][b, :m, h * group + g].double() @ kk.T / math.sqrt(dim)
                out[b, :m, h * group + g] = torch.softmax(score.masked_fill(hidden, -math.inf), dim=1) @ vv
    return out


def _exact_pages(s, case):
    """Page by page and row by row, as the operators are described; moved values are exact in any type."""
    k, v, page = s["k"], s["v"], case["page"]
    table = s["table"].cpu().numpy()
    if case["kind"] == "step":
        lens, counts, path = (s[n].cpu().numpy() for n in ("lens", "counts", "path"))
        for b in range(case["batch"]):
            rows = s["k_new"][:, b], s["v_new"][:, b]
            n = int(counts[b])
            taken = np.concatenate([path[b, :n], np.arange(n, case["tokens"])])
            at = int(lens[b]) + np.arange(case["tokens"])
            where = torch.from_numpy(table[b, at // page].astype(np.int64) * page + at % page).cuda()
            for cache, x in zip((k, v), rows):
                cache.reshape(cache.shape[0], -1, *cache.shape[3:])[:, where] = x[:, torch.from_numpy(taken).cuda()]
        return {"k": k.double(), "v": v.double(), "lens": None}
    refs = s["refs"].cpu().numpy()
    if case["kind"] == "fork":
        lens, src = s["lens"].cpu().numpy(), s["src"].cpu().numpy()
        unused = iter(np.nonzero(refs == 0)[0].tolist())
        for parent in src.tolist():
            n = int(lens[parent])
            if n % page:
                old, fresh = int(table[parent, n // page]), next(unused)
                k[:, fresh, : n % page] = k[:, old, : n % page]
                v[:, fresh, : n % page] = v[:, old, : n % page]
    else:
        count = int((refs > 0).sum())
        holes = [p for p in range(count) if refs[p] == 0]
        movers = [p for p in range(count, len(refs)) if refs[p] > 0]
        for hole, mover in zip(holes, movers):
            k[:, hole] = k[:, mover]
            v[:, hole] = v[:, mover]
    return {"k": k.double(), "v": v.double(), "table": None, "refs": None}
