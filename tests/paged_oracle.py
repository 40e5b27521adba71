"""Plain 64-bit implementations of the paged-cache operators, written from their definitions for the tests."""
import math

import numpy as np
import torch


def tables(lens, page, pages, width, seed, device="cpu"):
    """A table whose rows list distinct pages of a shuffled pool, as many as ``lens`` needs."""
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g).tolist()
    rows = []
    for n in lens:
        held = [order.pop() for _ in range(-(-n // page))]
        rows.append(held + [-1] * (width - len(held)))
    return torch.tensor(rows, dtype=torch.int32, device=device).view(len(lens), width)


def attention(q, k, v, table, lens, scale=None):
    """fp64 ``(out, largest sum of |q k| scale, largest |v|)`` per row and head."""
    q, k, v = (t.double().cpu() for t in (q, k, v))
    table, lens = table.cpu().tolist(), lens.cpu().tolist()
    rows, heads, hd = q.shape
    page, group = k.shape[2], heads // k.shape[1]
    scale = hd ** -0.5 if scale is None else scale
    out, size, top = torch.zeros(rows, heads, hd, dtype=torch.float64), torch.zeros(rows, heads, 1), torch.zeros(rows, heads, 1)
    size, top = size.double(), top.double()
    for r in range(rows):
        n = lens[r]
        if n == 0:
            continue
        at = [(table[r][j // page], j % page) for j in range(n)]
        ids, off = torch.tensor([a for a, _ in at]), torch.tensor([b for _, b in at])
        for h in range(heads):
            keys, values = k[ids, h // group, off], v[ids, h // group, off]
            s = keys @ q[r, h] * scale
            out[r, h] = torch.softmax(s, 0) @ values
            size[r, h] = (keys.abs() @ q[r, h].abs()).max() * abs(scale)
            top[r, h] = values.abs().max()
    return out, size, top


def attention_bound(out, size, top, hd, longest, dtype):
    """How far a kernel with fp32 sums may be off.  A score is a sum of hd products (hd + 4 roundings of its absolute sum, the scale
    and the change of base among them) and the exponential's argument is rounded at its size again; an error d in all scores moves
    weights by 2 d relative to each other.  Sums over the keys add a rounding each, in numerator and denominator, and a few for every
    join of parts.  In bf16 the weights enter the product with 16 bits, and the result is rounded to 8."""
    u = 2.0 ** -24
    d = (hd + 12) * u * size + 8 * u
    part = 4 * d + 2 * (longest + 64) * u
    if dtype == torch.bfloat16:
        return top * (part + 2.0 ** -15) + out.abs() * 2.0 ** -8
    return top * part + out.abs() * u


def rotate(x, positions, rotary, base):
    """fp64 half-split rotation of ``x [tokens, heads, hd]``."""
    x = x.double().cpu().clone()
    half = rotary // 2
    for t, p in enumerate(positions):
        if p < 0:
            continue
        for d in range(half):
            ang = p * base ** (-2.0 * d / rotary)
            c, s = math.cos(ang), math.sin(ang)
            a, b = x[t, :, d].clone(), x[t, :, half + d].clone()
            x[t, :, d], x[t, :, half + d] = a * c - b * s, b * c + a * s
    return x


def beam(logits, scores, finished, eos):
    """Brute force over all continuations: ``(scores, parents, tokens, finished)`` as lists, totals in fp64."""
    b, w = scores.shape
    x = logits.double().cpu().numpy().reshape(b, w, -1)
    start = scores.double().cpu().numpy()
    vocab = x.shape[2]
    out = [[], [], [], []]
    for i in range(b):
        every = []
        for j in range(w):
            row = x[i, j]
            done = finished is not None and bool(finished[i, j])
            lone = np.full(vocab, -np.inf)
            if np.isfinite(start[i, j]):
                if done:
                    lone[eos] = start[i, j]
                elif not np.isnan(row).any() and np.max(row) < np.inf and np.max(row) > -np.inf:
                    top = np.max(row)
                    lone = start[i, j] + (row - top - math.log(float(np.sum(np.exp(row - top)))))
                    lone[np.isnan(lone)] = -np.inf
            # within a beam the logits decide, so that a total that is rounded the same keeps their order
            order = np.lexsort((np.arange(vocab), -np.where(np.isnan(row), -np.inf, row) if lone.max() > -np.inf and not done else np.zeros(vocab), -lone))
            every += [(-lone[t], j, k, int(t), done) for k, t in enumerate(order[:w])]
        every.sort(key=lambda e: e[:3])
        best = every[:w]
        out[0].append([-e[0] for e in best])
        out[1].append([i * w + e[1] for e in best])
        out[2].append([e[3] for e in best])
        out[3].append([bool(e[4] or e[3] == eos) for e in best])
    return out
