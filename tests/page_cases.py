"""Batches over a paged cache and the plain forms, in 64 bits and token by token, of attention over chosen pages."""
import math

import torch

BF16, F32 = torch.bfloat16, torch.float32
HALF_STEP = {BF16: 2.0 ** -8, F32: 2.0 ** -24}              # one rounding, relative to the value


def gen(seed):
    return torch.Generator().manual_seed(seed)


class Batch:
    """``requests`` = [(history, new)]; pages in no order in a pool with spare ones; ``pad`` rows behind the last request."""

    def __init__(self, requests, page, seed=0, spare=3, extra_width=0, pad=0):
        g = gen(seed)
        held = [-(-(h + n) // page) for h, n in requests]
        self.requests, self.page, self.pad = requests, page, pad
        self.num_pages = sum(held) + spare
        self.width = max(max(held), 1) + extra_width
        order = torch.randperm(self.num_pages, generator=g).tolist()
        self.table = torch.full((len(requests), self.width), -1, dtype=torch.int32)
        for r, n in enumerate(held):
            for j in range(n):
                self.table[r, j] = order.pop()
        self.new = [n for _, n in requests]
        self.live = sum(self.new)
        self.T = self.live + pad
        self.cu = torch.tensor([0] + self.new).cumsum(0).to(torch.int32)
        self.where = [(r, h + i) for r, (h, n) in enumerate(requests) for i in range(n)]      # (request, position) per token
        self.positions = torch.tensor([p for _, p in self.where] + [0] * pad, dtype=torch.int32)
        self.slots = torch.tensor([int(self.table[r, p // page]) * page + p % page for r, p in self.where] + [-1] * pad, dtype=torch.int32)


def angles(positions, rot, theta=1e4):
    a = torch.arange(positions, dtype=torch.float64)[:, None] * theta ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot)
    return torch.cat([a.cos(), a.sin()], 1).float()


def finished(x, weight, eps, row, interleaved):
    """One head's [D] (64-bit): normed, then turned by the table's row [rot]."""
    if weight is not None:
        x = x / (x.square().mean() + eps).sqrt() * weight.double()
    if row is None:
        return x
    half = row.numel() // 2
    c, s = row[:half].double(), row[half:].double()
    y = x.clone()
    a = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    b = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    y[a], y[b] = x[a] * c - x[b] * s, x[b] * c + x[a] * s
    return y


def plain_scores(q, means, b, H, pages):
    """(64-bit scores [T, G, pages], the sums of the products' sizes that their errors go by)."""
    _, G, D = means.shape
    out = torch.full((b.T, G, pages), -math.inf, dtype=torch.float64)
    size = torch.zeros_like(out)
    for t, (r, p) in enumerate(b.where):
        for j in range(min(p // b.page, pages)):
            page = int(b.table[r, j])
            if 0 <= page < means.shape[0]:
                m = means[page].double()
                x = q[t].double().reshape(G, H // G, D)
                out[t, :, j] = torch.einsum("ghd,gd->gh", x, m).amax(1)      # (a NaN stays one)
                size[t, :, j] = torch.einsum("ghd,gd->gh", x.abs(), m.abs()).amax(1)
    return out, size


def plain_choice(scores, positions, page, top, first, recent):
    T, G, N = scores.shape
    out = torch.full((T, G, top), -1, dtype=torch.int32)
    for t in range(T):
        p = int(positions[t])
        own = -1 if p < 0 else min(p // page, N - 1)
        for g in range(G):
            forced = [j for j in range(own + 1) if j < first or j > own - recent]
            rest = [j for j in range(own + 1) if j not in forced]

            def key(j):
                s = float(scores[t, g, j])
                return (1, 0.0, j) if math.isnan(s) else (0, -s, j)
            picks = sorted(forced + sorted(rest, key=key)[:max(0, top - len(forced))])
            out[t, g, :len(picks)] = torch.tensor(picks, dtype=torch.int32)
    return out


def plain_attention(q, cache, b, chosen, H, scale):
    """(64-bit [T, H * D] of the live tokens, the sums of weight * |v|, the largest |q| |k| of a token's scores)."""
    num_pages, _, G, P, D = cache.shape
    out = torch.zeros(b.live, H, D, dtype=torch.float64)
    size, qk = torch.zeros_like(out), torch.zeros(b.live, H, 1, dtype=torch.float64)
    for t, (r, p) in enumerate(b.where):
        for g in range(G):
            ks, vs = [], []
            for j in chosen[t, g].tolist():
                if 0 <= j < b.width and 0 <= int(b.table[r, j]) < num_pages:
                    n = max(0, min(P, p - j * P + 1))
                    ks.append(cache[int(b.table[r, j]), 0, g, :n].double())
                    vs.append(cache[int(b.table[r, j]), 1, g, :n].double())
            k, v = (torch.cat(x) if x else torch.zeros(0, D, dtype=torch.float64) for x in (ks, vs))
            if not len(k):
                continue
            x = q[t].double().reshape(G, H // G, D)[g]
            w = torch.softmax(scale * x @ k.T, 1)
            h = slice(g * (H // G), (g + 1) * (H // G))
            out[t, h], size[t, h] = w @ v, w @ v.abs()
            qk[t, h, 0] = scale * (x.abs() @ k.abs().T).amax(1)
    return out.reshape(b.live, H * D), size.reshape(b.live, H * D), qk.expand(-1, -1, D).reshape(b.live, H * D)


def attention_bound(dtype, D, want, size, qk):
    """Scores are sums of D products in 32 bits (each step off by 2^-22 at most, also where a tensor core cuts off instead of rounding): a
    weight is off by twice that score error, relatively; exponentials by 2^-20; in bfloat16 the weights are rounded once, the result once.
    Sums of weights times values: 2^-16 relatively (a thousand steps and more of 2^-24, and joined parts)."""
    weights = 2 * D * 2.0 ** -22 * qk + 2.0 ** -20 + 2.0 ** -16
    if dtype == BF16:
        weights = weights + HALF_STEP[BF16]
    return weights * size * 1.01 + HALF_STEP[dtype] * want.abs() + 1e-30
