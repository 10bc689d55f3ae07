"""The cache operators from their definitions, in 64 bits on the CPU.

Plain loops and searches, sharing no code with the package: MX4 rounding by
looking for the nearest value, attention sequence by sequence, eviction by
sorting tokens.
"""

from __future__ import annotations

import math

import numpy as np
import torch

E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def mx4_encode(x):
    """Rows ``[..., head_dim]`` -> (codes ``[..., head_dim // 2]``, scale bytes ``[..., head_dim // 32]``)."""
    x = np.asarray(torch.as_tensor(x).double())
    blocks = x.reshape(-1, 32)
    codes = np.zeros(blocks.shape, dtype=np.uint8)
    scales = np.zeros(blocks.shape[0], dtype=np.uint8)
    grid = np.array(E2M1)
    for i, row in enumerate(blocks):
        if not np.isfinite(row).all():
            scales[i] = 255
            continue
        top = np.abs(row).max()
        e = -127 if top == 0 else max(-127, math.frexp(top)[1] - 1 - 2)
        scales[i] = e + 127
        far = np.abs(np.abs(row)[:, None] / math.ldexp(1.0, e) - grid)
        best = far.min(1)
        for j in range(32):
            near = [c for c in range(8) if far[j, c] == best[j]]
            code = near[0] if len(near) == 1 or near[0] % 2 == 0 else near[1]
            codes[i, j] = code + (8 if math.copysign(1.0, row[j]) < 0 else 0)
    codes = codes.reshape(x.shape)
    packed = (codes[..., 0::2] | (codes[..., 1::2] << 4)).astype(np.uint8)
    return torch.from_numpy(packed), torch.from_numpy(scales.reshape(*x.shape[:-1], x.shape[-1] // 32))


def mx4_decode(codes, scales):
    """(codes, scale bytes) -> values ``[..., head_dim]`` in 64 bits."""
    c = codes.cpu().long()
    both = torch.stack([c % 16, c // 16], -1).flatten(-2)
    table = torch.tensor(E2M1 + [-v for v in E2M1], dtype=torch.float64)
    s = scales.cpu().double()
    factor = torch.where(s == 255, math.nan, torch.pow(2.0, s - 127))
    return table[both] * factor.repeat_interleave(32, -1)


def gather(cache, table_row, n):
    """The first n rows of a sequence: ``[n, heads, ...]``."""
    ps = cache.shape[1]
    t = torch.arange(n)
    return cache[table_row[t // ps].long(), t % ps]


def attention(q, k_values, v_values, block_table, seq_lens, scale):
    """Outputs ``[batch, heads, d]``, per-token weights (a list of ``[kv heads, n]``) and error terms, all in 64 bits.

    The error terms of each (sequence, query head): the sum of weight * |v| per
    output element, the sum of |v|, and the largest sum of |q k| over a token.
    """
    q = q.double().cpu()
    batch, hq, d = q.shape
    hkv = k_values.shape[2]
    g = hq // hkv
    out = torch.zeros(batch, hq, d, dtype=torch.float64)
    heavy = torch.zeros(batch, hq, d, dtype=torch.float64)
    plain = torch.zeros(batch, hq, d, dtype=torch.float64)
    dots = torch.zeros(batch, hq, dtype=torch.float64)
    weights = []
    for b in range(batch):
        n = int(seq_lens[b])
        if n == 0:
            weights.append(torch.zeros(hkv, 0, dtype=torch.float64))
            continue
        k, v = gather(k_values, block_table[b], n).double(), gather(v_values, block_table[b], n).double()
        w = torch.zeros(hkv, n, dtype=torch.float64)
        for h in range(hq):
            p = torch.softmax(k[:, h // g] @ q[b, h] * scale, 0)
            out[b, h] = p @ v[:, h // g]
            heavy[b, h] = p @ v[:, h // g].abs()
            plain[b, h] = v[:, h // g].abs().sum(0)
            dots[b, h] = (k[:, h // g].abs() @ q[b, h].abs()).max() * abs(scale)
            w[h // g] += p
        weights.append(w)
    return out, weights, {"heavy": heavy, "plain": plain, "dots": dots}


def evict(weights, positions, block_table, seq_lens, keep, recent):
    """(new lengths, moves): per (sequence, kv head) the list of (source slot, target slot)."""
    hkv = weights.shape[2]
    new_lens, moves = [], {}
    for b in range(len(seq_lens)):
        n_all = int(seq_lens[b])
        n = min(int(keep[b]) if isinstance(keep, (list, torch.Tensor)) else keep, n_all)
        new_lens.append(n)
        if n == 0 or n == n_all:
            continue
        w_rows, p_rows = gather(weights, block_table[b], n_all), gather(positions, block_table[b], n_all)
        for h in range(hkv):
            w, p = w_rows[:, h].tolist(), p_rows[:, h].tolist()
            border = max(p) - recent

            def rank(t):
                if p[t] > border:
                    return (0, 0.0, t)
                return (1, 0.0, t) if math.isnan(w[t]) else (2, -w[t], t)

            kept = set(sorted(range(n_all), key=rank)[:n])
            sources = [t for t in range(n, n_all) if t in kept]
            targets = [t for t in range(n) if t not in kept]
            moves[b, h] = list(zip(sources, targets))
    return new_lens, moves
