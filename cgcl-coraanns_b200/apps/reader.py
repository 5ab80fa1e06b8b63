"""Search, then read: the index answers a query and a small 4-bit decoder reads what it found.

    python cgcl-coraanns_b200/apps/reader.py [--tokens 16] [--layers 2]

Passages are token sequences; their embeddings (and the query's) are synthetic. The search engine
finds the query's nearest passages; their tokens and the question are the prompt of a decoder with
random weights, which fills its 4-bit cache with one call per layer (`Cache4.append`, many tokens),
attends over it (`Cache4.attend`, many queries), and then decodes token by token (the same calls,
one token; projections by `matvec` on 4-bit weights). The same decoder on the dense values that
the 4-bit weights and the cache stand for, in plain torch, runs beside it as a check.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import coraanns_b200 as cb  # noqa: E402
from coraanns_b200 import builder, lowbit  # noqa: E402

DIM, HEADS, KV_HEADS, HEAD, INNER, VOCAB, PAGE = 512, 8, 2, 64, 1024, 2000, 16


def rotation(positions, head=HEAD):
    half = head // 2
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half) / half)
    return angle.cos().float().cuda(), angle.sin().float().cuda()


class Layer:
    """Weights of one layer in 4 bits, and its cache."""

    def __init__(self, gen, pages):
        def weight(n, k):
            return lowbit.Weight4.quantize(torch.randn(n, k, generator=gen, device="cuda") * k ** -0.5)
        self.qkv = weight((HEADS + 2 * KV_HEADS) * HEAD, DIM)
        self.out, self.up, self.down = weight(DIM, HEADS * HEAD), weight(INNER, DIM), weight(DIM, INNER)
        self.cache = lowbit.Cache4(pages, KV_HEADS, HEAD, page_size=PAGE)


def norm(x):
    return (x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6)).to(x.dtype)


def forward(layers, embed, head, tokens, past, table, rope):
    """Logits of the last of `tokens` (one sequence), the cache holding `past` tokens before them."""
    n = tokens.shape[0]
    x = embed[tokens]
    positions = torch.arange(past, past + n, dtype=torch.int32, device="cuda")
    slots = table[0, positions.long() // PAGE].long() * PAGE + positions % PAGE
    lens = torch.tensor([past + n], dtype=torch.int32, device="cuda")
    start = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    for layer in layers:
        qkv = lowbit.matvec(norm(x), layer.qkv).view(n, -1, HEAD)
        q, k, v = qkv[:, :HEADS], qkv[:, HEADS:HEADS + KV_HEADS], qkv[:, HEADS + KV_HEADS:]
        q = layer.cache.append(k, v, slots, q=q, rope=rope, positions=positions).q
        o = layer.cache.attend(q, table, lens, q_start=start, max_queries=n)
        x = x + lowbit.matvec(o.flatten(1), layer.out)
        x = x + lowbit.matvec(torch.nn.functional.silu(lowbit.matvec(norm(x), layer.up)), layer.down)
    return lowbit.matvec(norm(x[-1:]), head)[0]


def dense_weight(w):
    """What a 4-bit weight stands for, fp32."""
    shift = 4 * torch.tensor(lowbit.NIBBLE_OF, device="cuda")
    c = (w.codes.view(torch.int32)[..., None] >> shift) & 15
    c = c.view(w.rows, -1, 4, 4, 8).transpose(2, 3).reshape(w.rows, -1, w.group)
    meta = w.meta.float()
    return (meta[..., :1] * c + meta[..., 1:]).flatten(1)[:, :w.cols]


def dense_cache(cache, table, tokens):
    """The keys and values of a sequence's first `tokens` cached tokens, fp32 (heads, tokens, dim)."""
    P, D, G = cache.page_size, cache.head_dim, cache.group
    blocks, n, m = cache.pool[table[0].long()], P * D // 2, P * (D // G) * 4
    out = []
    for c, s in ((blocks[..., :n], blocks[..., 2 * n:2 * n + m]), (blocks[..., n:2 * n], blocks[..., 2 * n + m:])):
        codes = torch.stack((c & 15, c >> 4), -1).flatten(-2).unflatten(-1, (P, D // G, G))
        f = s.contiguous().view(torch.float16).float().unflatten(-1, (P, D // G, 2))
        out.append((f[..., :1] * codes + f[..., 1:]).flatten(-2).transpose(0, 1).flatten(1, 2)[:, :tokens])
    return out


def check_logits(layers, embed, head, tokens, table, rope):
    """Logits of the last token in plain torch, from the cached keys and values and dense weights."""
    n = tokens.shape[0]
    x = embed[tokens].float()
    cos, sin = rope[0][:n, None], rope[1][:n, None]
    seen = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
    nrm = lambda t: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6)  # noqa: E731
    for layer in layers:
        q = (nrm(x) @ dense_weight(layer.qkv).T)[:, :HEADS * HEAD].view(n, HEADS, HEAD)
        a, b = q[..., :HEAD // 2], q[..., HEAD // 2:]
        q = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        k, v = (t.repeat_interleave(HEADS // KV_HEADS, 0) for t in dense_cache(layer.cache, table, n))
        s = (torch.einsum("nhd,hld->hnl", q, k) * HEAD ** -0.5).masked_fill(~seen, float("-inf"))
        o = torch.einsum("hnl,hld->nhd", s.softmax(-1), v).flatten(1)
        x = x + o @ dense_weight(layer.out).T
        x = x + torch.nn.functional.silu(nrm(x) @ dense_weight(layer.up).T) @ dense_weight(layer.down).T
    return nrm(x[-1]) @ dense_weight(head).T


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--passages", type=int, default=4000)
    ap.add_argument("--tokens", type=int, default=16, help="tokens to decode")
    ap.add_argument("--layers", type=int, default=2)
    a = ap.parse_args(argv)

    # the index: passages in clusters, searched with the query's embedding
    rng = np.random.default_rng(0)
    nlist, dim = 16, 96
    centres = rng.normal(size=(nlist, dim)).astype(np.float32)
    label = rng.integers(0, nlist, a.passages)
    base = (centres[label] + 0.3 * rng.normal(size=(a.passages, dim))).astype(np.float32)
    sd = builder.build_index(base, centres, label)
    text = rng.integers(0, VOCAB, (a.passages, 60))
    query = base[[17]] + 0.02 * rng.normal(size=(1, dim)).astype(np.float32)
    with cb.HybridIndex(0) as index:
        index.load_search_data(sd)
        index.prepare_workspace(1, 5, 8)
        index.reset_buffer(query)
        _, ids = index.search(query, 5, 8)
    prompt = np.concatenate([text[i] for i in ids[0]] + [rng.integers(0, VOCAB, 13)])

    # the reader
    gen = torch.Generator(device="cuda").manual_seed(1)
    total = len(prompt) + a.tokens
    pages = -(-total // PAGE)
    embed = torch.randn(VOCAB, DIM, generator=gen, device="cuda").to(torch.bfloat16)
    head = lowbit.Weight4.quantize(torch.randn(VOCAB, DIM, generator=gen, device="cuda") * DIM ** -0.5)
    layers = [Layer(gen, pages) for _ in range(a.layers)]
    table = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)[None]
    rope = rotation(total)
    tokens = torch.from_numpy(prompt).cuda()
    logits = forward(layers, embed, head, tokens, 0, table, rope)
    for _ in range(a.tokens):
        tokens = torch.cat((tokens, logits.argmax()[None]))
        logits = forward(layers, embed, head, tokens[-1:], len(tokens) - 1, table, rope)
    for layer in layers:
        layer.cache.check()
    want = check_logits(layers, embed, head, tokens, table, rope)
    off = float((logits.float() - want).norm() / want.norm())
    print(f"passages {ids[0].tolist()}; prompt of {len(prompt)} tokens, {a.tokens} decoded: "
          f"{tokens[len(prompt):].tolist()}")
    print(f"last logits against plain torch on the same 4-bit values: relative difference {off:.4f}")
    return ids[0].tolist(), off


if __name__ == "__main__":
    main()
