"""Speculative decoding over a paged cache, with one attention layer for a model.

A toy model (embedding, one attention layer with a residual, output head, random weights) and a
cheaper draft (the embedding and output head alone).  Each step drafts a tree of tokens, writes their keys
and values into the cache, verifies the whole tree with one ``tree_attention`` call, keeps the accepted path
and takes the model's own next token after it.  Greedy verification changes speed, not output: the
example checks that plain one-token decoding gives the same text.

    python examples/speculative_decode.py            # needs a B200
"""

from __future__ import annotations

import sys
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

from ntilang_b200 import paged  # noqa: E402

HEADS, KV_HEADS, DIM, VOCAB, PAGE = 8, 2, 64, 512, 16
# Draft tree: three guesses for the next token, two more after the first, one after the second.
PARENTS = [-1, -1, -1, 0, 0, 1]


class Model:
    def __init__(self, seed=0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        width = HEADS * DIM
        init = lambda *s: torch.randn(*s, generator=gen, device="cuda") / s[0] ** 0.5  # noqa: E731
        self.embed = torch.randn(VOCAB, width, generator=gen, device="cuda")
        self.wq, self.wo = init(width, width), init(width, width)
        self.wk, self.wv = init(width, KV_HEADS * DIM), init(width, KV_HEADS * DIM)
        self.head = init(width, VOCAB)

    def project(self, tokens):
        """(hidden, q, k, v) of tokens [seqs, n]; k and v as one cache layer."""
        x = self.embed[tokens]
        heads = lambda w, n: (x @ w).reshape(*tokens.shape, n, DIM).half()  # noqa: E731
        return x, heads(self.wq, HEADS), heads(self.wk, KV_HEADS)[None], heads(self.wv, KV_HEADS)[None]

    def logits(self, hidden, attended):
        return (hidden + attended.float().flatten(2) @ self.wo) @ self.head

    def guess(self, tokens, n):
        """The draft: n likely successors of each token by the embedding alone."""
        return (self.embed[tokens] @ self.head).topk(n, dim=-1).indices


def prefill(model, cache, prompt):
    """Write the prompt's rows; the next token of each sequence."""
    seqs, n = prompt.shape
    slots = torch.arange(seqs, dtype=torch.int32, device="cuda")
    assert bool(cache.reserve(slots, n).all())
    hidden, q, k, v = model.project(prompt)
    cache.append(k, v)
    out = cache.window_attention(0, q, window=1 << 20)
    return model.logits(hidden, out)[:, -1].argmax(-1)


def decode(model, cache, token, steps):
    """Plain decoding: one token at a time."""
    slots = torch.arange(token.shape[0], dtype=torch.int32, device="cuda")
    text = [token]
    for _ in range(steps):
        assert bool(cache.reserve(slots, 1).all())
        hidden, q, k, v = model.project(token[:, None])
        cache.append(k, v)
        out = cache.window_attention(0, q, window=1 << 20)
        token = model.logits(hidden, out)[:, 0].argmax(-1)
        text.append(token)
    return torch.stack(text, 1)


def speculate(model, cache, token, steps):
    """The same text with a tree of drafts verified per step; returns (text, verification steps)."""
    seqs, root = token.shape[0], 1 + len(PARENTS)  # the tree's draft 0 is the token already decided
    slots = torch.arange(seqs, dtype=torch.int32, device="cuda")
    parents = [-1] + [p + 1 for p in PARENTS]
    tree = paged.tree_mask(torch.tensor([parents], dtype=torch.int32, device="cuda"))
    text = [[t] for t in token.tolist()]
    rounds = 0
    while min(map(len, text)) <= steps:
        rounds += 1
        first = model.guess(token, 3)
        second = torch.stack([*model.guess(first[:, 0], 2).unbind(1), model.guess(first[:, 1], 1)[:, 0]], 1)
        drafts = torch.cat([token[:, None], first, second], 1)
        assert bool(cache.reserve(slots, root).all())
        hidden, q, k, v = model.project(drafts)
        cache.append(k, v)
        out = cache.tree_attention(0, q, tree)
        choice = model.logits(hidden, out).argmax(-1)
        # Follow the model's own choice from the root as long as it was drafted.
        want, drafted = choice.tolist(), drafts.tolist()
        paths, nexts = [], []
        for b in range(seqs):
            path = [0]
            while True:
                step = [d for d in range(root) if parents[d] == path[-1] and drafted[b][d] == want[b][path[-1]]]
                if not step:
                    break
                path.append(step[0])
            text[b] += [drafted[b][d] for d in path[1:]] + [want[b][path[-1]]]
            nexts.append(want[b][path[-1]])
            paths.append(path + [path[-1]] * (root - len(path)))
        counts = torch.tensor([len(set(p)) for p in paths], dtype=torch.int32, device="cuda")
        cache.accept(torch.tensor(paths, dtype=torch.int32, device="cuda"), counts, root)
        token = torch.tensor(nexts, device="cuda")
    return torch.tensor([t[: steps + 1] for t in text], device="cuda"), rounds


def main(seqs=4, prompt_len=100, steps=60):
    model = Model()
    prompt = torch.randint(0, VOCAB, (seqs, prompt_len), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    # Plain decoding in the first half of the slots, speculation in the second, from one prompt: the forked
    # half shares its full pages.
    longest = prompt_len + 8 * steps
    cache = paged.Cache(layers=1, pages=2 * seqs * (longest // PAGE + 1), page_size=PAGE, kv_heads=KV_HEADS, head_dim=DIM,
                        seqs=2 * seqs, max_pages=longest // PAGE + 1)
    slots = torch.arange(2 * seqs, dtype=torch.int32, device="cuda")
    plain = cache.part(slice(0, seqs))
    first = prefill(model, plain, prompt)
    cache.lens[:seqs] = plain.lens
    assert bool(cache.fork(slots[:seqs], slots[seqs:]).all())
    fast = cache.part(slice(seqs, 2 * seqs))
    want = decode(model, plain, first, steps)
    got, rounds = speculate(model, fast, first, steps)
    assert torch.equal(want, got), "speculation must not change the text"
    cache.free(slots)
    assert int(cache.refs.max()) == 0
    print(f"{seqs} x {steps} tokens in {rounds} verification steps, same text as {steps} plain ones")
    return rounds


if __name__ == "__main__":
    main()
