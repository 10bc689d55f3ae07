"""Cases, tolerances and comparisons of the cache operators' tests."""

from __future__ import annotations

import math
import random

import torch

from oracle import cache as oracle
from tests.helpers import shuffled_table

MX4, E4M3, E5M2 = "mx4", "e4m3", "e5m2"
FP8 = {E4M3: torch.float8_e4m3fn, E5M2: torch.float8_e5m2}
QTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def encode(x, kv, dtype):
    """Values -> (cache, its scale argument, the values it stands for) on the CPU."""
    if kv == MX4:
        codes, scales = oracle.mx4_encode(x.to(dtype))
        return codes, scales, oracle.mx4_decode(codes, scales)
    if kv in FP8:
        scale = float(x.abs().max()) / 200.0
        codes = (x / scale).to(FP8[kv])
        return codes, scale, codes.double() * torch.tensor(scale, dtype=torch.float32).double()
    cache = x.to(dtype)
    return cache, None, cache.double()


def head_major(t):
    """The same tensor with the rows of a kv head next to each other within a page."""
    b = t.view(torch.uint8) if t.element_size() == 1 else t
    return b.transpose(1, 2).contiguous().transpose(1, 2).view(t.dtype) if t.element_size() == 1 else (
        b.transpose(1, 2).contiguous().transpose(1, 2))


class Case:
    """Caches, tables and queries of one decode, on the CPU and (``gpu()``) on the GPU."""

    def __init__(self, lens, hq, hkv, d, ps, q="fp16", kv=None, seed=0, extra_cols=1, stretch=1.0, layout="head"):
        kv = kv or q
        self.dtype, self.kv, self.lens, self.ps = QTYPES[q], kv, list(lens), ps
        self.table, pages = shuffled_table(self.lens, ps, spare_pages=3, extra_cols=extra_cols, seed=seed + 5)
        g = torch.Generator().manual_seed(seed)
        k = torch.randn(pages, ps, hkv, d, generator=g) * stretch
        v = torch.randn(pages, ps, hkv, d, generator=g)
        self.k, self.ks, self.k_values = encode(k, kv, self.dtype)
        self.v, self.vs, self.v_values = encode(v, kv, self.dtype)
        if layout == "head":
            self.k, self.v = head_major(self.k), head_major(self.v)
            if kv == MX4:
                self.ks, self.vs = head_major(self.ks), head_major(self.vs)
        self.q = torch.randn(len(self.lens), hq, d, generator=g).to(self.dtype)
        self.seq_lens = torch.tensor(self.lens, dtype=torch.int32)
        self.weights = torch.rand(pages, ps, hkv, generator=g)
        self.scale = 1.0 / math.sqrt(d)
        self.hkv, self.g, self.d, self.pages = hkv, hq // hkv, d, pages

    def gpu(self):
        """(q, k, v, table, lens, {k_scale, v_scale}) on the GPU, strides kept."""
        up = lambda t: cuda_like(t) if isinstance(t, torch.Tensor) else t  # noqa: E731
        return (up(self.q), up(self.k), up(self.v), up(self.table), up(self.seq_lens),
                {"k_scale": up(self.ks), "v_scale": up(self.vs)})

    def expected(self):
        return oracle.attention(self.q, self.k_values, self.v_values, self.table, self.lens, self.scale)


def cuda_like(t):
    """A copy on the GPU with the same strides."""
    out = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device="cuda")
    if t.element_size() == 1 and t.dtype != torch.uint8:
        out.view(torch.uint8).copy_(t.view(torch.uint8))
    else:
        out.copy_(t)
    return out


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def score_error(case, err):
    """Bound of a score's error in natural units, per (sequence, query head).

    Products of 16-bit values are exact in 32 bits (22 significant bits at most); D of
    them are added with a rounding each, and the scale (a rounding of its own, of
    log2 e times it, and fp8's factor) multiplies the sum: D + 4 roundings of 2^-24 of the sum of
    |q k|.
    """
    return err["dots"] * (case.d + 4) * 2.0**-24


def check_output(case, out, expected, err):
    """|out - exact| within the roundings that the operator makes.

    A weight is rounded to q's type (u of it, or 2^-25 of the largest where fp16 has no more
    bits) and so is the output; the normaliser sums rounded weights (u again).
    A score's error e changes every weight by at most expm1(2 e) relative to the others; 16 roundings
    of 2^-24 cover exponentials, sums and merges of a few splits, and one per token the long sums.
    """
    u = half_step(case.dtype)
    n = torch.tensor(case.lens, dtype=torch.float64).view(-1, 1, 1)
    e = torch.expm1(2 * score_error(case, err)).unsqueeze(-1)
    bound = u * expected.abs() + (2 * u + e + (16 + n) * 2.0**-24) * err["heavy"]
    if case.dtype == torch.float16:
        bound = bound + 2.0**-25 * (err["plain"] + n * err["heavy"]) + 2.0**-24
    got = out.double().cpu()
    assert torch.isfinite(got).all()
    worst = ((got - expected).abs() - bound).max() if got.numel() else 0.0
    assert worst <= 0, f"off by {float((got - expected).abs().max()):.3g}, over its bound by {float(worst):.3g}"


def check_weights(case, before, after, weights, err):
    """Every token's sum within its roundings; every other slot as it was.

    A weight is 2^(x - lse): e of the score and of the normaliser (which is a sum of weights that
    are off by as much), 2^-24 of |x| and of |lse| (scores in base 2 up to a few hundred: 2^-24 * 1024),
    the exponentials and logarithms a few roundings; the sums over the group and into the slot
    one rounding each.  The normaliser's sum has a rounding per token of a lane at most.
    """
    got = after.double().cpu()
    want = before.double().clone()
    bound = torch.zeros_like(want)
    for b, n in enumerate(case.lens):
        t = torch.arange(n)
        ids = case.table[b][t // case.ps].long()
        want[ids, t % case.ps] += weights[b].transpose(0, 1)
        e = score_error(case, err)[b].view(case.hkv, case.g).amax(1)
        rel = torch.expm1(2 * e) + (1024 + 32 + n) * 2.0**-24
        bound[ids, t % case.ps] = (rel.unsqueeze(1) * weights[b]).transpose(0, 1) + 2.0**-23 * want[ids, t % case.ps].abs()
    off = (got - want).abs()
    assert (off <= bound).all(), f"weights off by {float(off.max()):.3g}, over by {float((off - bound).max()):.3g}"


def eviction_case(lens, hkv, ps, seed, ties=False):
    """Random weights (a few NaN, infinite, negative, equal ones) and positions of a cache."""
    rng = random.Random(seed)
    table, pages = shuffled_table(lens, ps, spare_pages=2, extra_cols=1, seed=seed)
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(pages, ps, hkv, generator=g).exp()
    if ties:
        w = torch.randint(0, 4, w.shape, generator=g).float()
        odd = torch.tensor([math.nan, math.inf, -math.inf, -0.0, 0.0, -1.0, 1e-42])
        at = torch.rand(w.shape, generator=g) < 0.2
        w = torch.where(at, odd[torch.randint(0, len(odd), w.shape, generator=g)], w)
    pos = torch.full((pages, ps, hkv), -7, dtype=torch.int32)
    for b, n in enumerate(lens):
        for h in range(hkv):
            order = list(range(n))
            rng.shuffle(order)
            t = torch.arange(n)
            pos[table[b][t // ps].long(), t % ps, h] = torch.tensor(order, dtype=torch.int32) * 3
    return table, pages, w, pos
