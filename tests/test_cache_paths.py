"""MX4 and accumulating decodes along every path of the launcher: long units, many units, ranges, two-level and
shared folds, large batches, every page mode and layout.  Against attention in 64 bits, computed on the GPU."""

from __future__ import annotations

import math
import random

import pytest
import torch

import paged_attention_decode_amd as pad
from tests.cache_helpers import QTYPES

pytestmark = pytest.mark.gpu

E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def mx4_values(codes, scales):
    """The caches' values in 64 bits."""
    table = torch.tensor(E2M1 + [-x for x in E2M1], dtype=torch.float64, device="cuda")
    both = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    return table[both] * torch.pow(2.0, scales.double() - 127).repeat_interleave(32, -1)


def build(lens, hq, hkv, d, ps, q="bf16", kv="mx4", seed=0, layout="head", extra_cols=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = [-(-n // ps) for n in lens]
    total = sum(pages) + 1
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).int()
    table = torch.full((len(lens), max(pages) + extra_cols), int(perm[-1]), dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = perm[at:at + n]
        at += n
    q_t = torch.randn(len(lens), hq, d, generator=g, device="cuda").to(QTYPES[q])

    def ints(width, lo, hi):
        t = torch.randint(lo, hi, (total, hkv, ps, width), generator=g, device="cuda", dtype=torch.uint8).transpose(1, 2)
        return t if layout == "head" else t.contiguous()

    if kv == "mx4":
        k, v, ks, vs = ints(d // 2, 0, 256), ints(d // 2, 0, 256), ints(d // 32, 122, 127), ints(d // 32, 122, 128)
        return q_t, k, v, table, {"k_scale": ks, "v_scale": vs}
    k, v = (torch.randn(total, ps, hkv, d, generator=g, device="cuda") for _ in range(2))
    if kv == "e4m3":
        return q_t, (8 * k).to(torch.float8_e4m3fn), (8 * v).to(torch.float8_e4m3fn), table, {"k_scale": 0.125,
                                                                                              "v_scale": 0.125}
    return q_t, k.to(q_t.dtype), v.to(q_t.dtype), table, {}


def check(lens, q, k, v, table, scales, out, gained=None):
    """Bounds per element from the roundings made (see cache_helpers.check_output and check_weights)."""
    batch, hq, d = q.shape
    hkv, ps = k.shape[2], k.shape[1]
    u = torch.finfo(q.dtype).eps / 2
    for b, n in enumerate(lens):
        if n == 0:
            assert (out[b] == 0).all()
            continue
        ids = table[b, :-(-n // ps)].cuda().long()

        def rows(cache, scale):
            if isinstance(scale, torch.Tensor):
                x = mx4_values(cache[ids], scale[ids])
            elif cache.element_size() == 1:
                x = cache.view(torch.uint8)[ids].view(cache.dtype).double() * scale
            else:
                x = cache[ids].double()
            return x.flatten(0, 1)[:n].transpose(0, 1).contiguous()

        kk, vv = rows(k, scales.get("k_scale")), rows(v, scales.get("v_scale"))
        qq = q[b].double().view(hkv, hq // hkv, d)
        kt = kk.transpose(1, 2).contiguous()
        p = torch.softmax(qq @ kt / math.sqrt(d), -1)
        want = (p @ vv).view(hq, d)
        heavy = (p @ vv.abs()).view(hq, d)
        score = (qq.abs() @ kt.abs()).amax(-1) / math.sqrt(d) * (d + 4) * 2.0**-24
        e = torch.expm1(2 * score)
        # Sums: a lane's tokens one after the other, at most n of them.
        bound = u * want.abs() + (2 * u + e.view(hq, 1) + (16 + n) * 2.0**-24) * heavy
        # What lies below the normal numbers of 32 bits (2^-126) may be taken as 0: a weight (its
        # token's |v| times that is lost) and a product or the sum itself.
        bound = bound + 2.0**-126 * (1 + vv.abs().sum(1).repeat_interleave(hq // hkv, 0))
        if q.dtype == torch.float16:
            bound = bound + 2.0**-25 * (vv.abs().sum(1).repeat_interleave(hq // hkv, 0) + n * heavy) + 2.0**-24
        off = (out[b].double() - want).abs()
        assert (off <= bound).all(), f"sequence {b} of {n}: off {float(off.max()):.3g}, over by {float((off - bound).max()):.3g}"
        if gained is not None:
            t = torch.arange(n, device="cuda")
            got = gained[ids[t // ps], t % ps].double().transpose(0, 1)
            w = p.sum(1)
            assert ((got - w).abs() <= ((e.amax(-1) + (1056 + n) * 2.0**-24)[:, None] * w) + 2.0**-23 * w).all()


def run(lens, hq, hkv, d, ps, q="bf16", kv="mx4", seed=0, layout="head", weights=False, splits=None, extra_cols=0):
    q_t, k, v, table, scales = build(lens, hq, hkv, d, ps, q, kv, seed, layout, extra_cols)
    tab, sl = table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")
    if kv == "mx4":
        out = pad.paged_attention_decode_mx4(q_t, k, v, scales["k_scale"], scales["v_scale"], tab, sl, num_splits=splits)
        check(lens, q_t, k, v, table, scales, out)
    if weights or kv != "mx4":
        acc = torch.zeros(k.shape[0], hkv, ps, device="cuda").transpose(1, 2)
        out = pad.paged_attention_decode_weights(q_t, k, v, acc, tab, sl, num_splits=splits, **scales)
        check(lens, q_t, k, v, table, scales, out, acc)
        # Slots of no token stay 0: what was gained is one of each query head.
        live = sum(1 for n in lens if n) * hq
        assert abs(float(acc.double().sum()) - live) < 1e-3 * max(live, 1)


def ragged(batch, hi, seed):
    rng = random.Random(seed)
    lens = [rng.randint(0, hi) for _ in range(batch)]
    lens[rng.randrange(batch)] = hi
    lens[rng.randrange(batch)] = 0
    return lens


@pytest.mark.parametrize("kv", ["mx4", "16", "e4m3"])
@pytest.mark.parametrize("lens,hq,hkv,d,ps", [
    ([65536], 8, 1, 128, 16),              # hundreds of splits: two levels
    ([30001, 2], 4, 1, 64, 16),
    ([8192] * 4, 16, 1, 256, 16),          # large partials: the shared fold
    ([16384, 16000], 16, 1, 256, 32),
    ([4096] * 16, 12, 2, 128, 16),         # full tables
    (ragged(20, 3000, 1), 32, 8, 128, 16),
    (ragged(48, 2500, 2), 12, 2, 128, 32),
    (ragged(100, 700, 3), 24, 6, 128, 48),
    ([777] * 130, 8, 4, 64, 16),
    (ragged(40, 2048, 4), 16, 4, 256, 16),
])
def test_launch_paths(kv, lens, hq, hkv, d, ps):
    run(lens, hq, hkv, d, ps, kv=kv, weights=True, seed=len(lens))


@pytest.mark.parametrize("q", ["fp16", "bf16"])
@pytest.mark.parametrize("kv", ["mx4", "16"])
@pytest.mark.parametrize("hkv,d", [(8, 128), (4, 64), (8, 256), (2, 128)])
@pytest.mark.parametrize("ps", [16, 1, 8, 3, 64])
def test_many_units(q, kv, hkv, d, ps):
    """Rows long and many enough for the range kernel."""
    lens = ragged(70, 1500, ps)
    run(lens, 2 * hkv, hkv, d, ps, q, kv, weights=True, seed=ps, layout="token" if ps in (8, 64) else "head")


@pytest.mark.parametrize("kv", ["mx4", "16"])
@pytest.mark.parametrize("batch,hi", [(257, 200), (300, 900), (520, 600)])
def test_large_batches(kv, batch, hi):
    run(ragged(batch, hi, batch), 8, 4, 128, 16, kv=kv, weights=True, seed=batch)


@pytest.mark.parametrize("kv", ["mx4", "16"])
def test_tables_wider_than_the_lengths(kv):
    run(ragged(30, 300, 7), 32, 8, 128, 16, kv=kv, weights=True, extra_cols=400)
    run([1, 2, 3], 4, 4, 64, 16, kv=kv, weights=True, extra_cols=2000)


def test_sixteen_query_heads_and_one():
    run([2000, 31, 900], 128, 8, 128, 16, weights=True)
    run([2000, 31, 900], 8, 8, 128, 16, weights=True)


def test_scores_far_apart():
    """Scores of hundreds: running maxima move, far tokens weigh nothing."""
    q, k, v, table, s = build([3000, 500], 8, 2, 128, 16, seed=3)
    g = torch.Generator(device="cuda").manual_seed(12)
    s["k_scale"][:] = torch.randint(118, 133, s["k_scale"].shape, generator=g, device="cuda", dtype=torch.uint8)
    tab, sl = table.cuda(), torch.tensor([3000, 500], dtype=torch.int32, device="cuda")
    acc = torch.zeros(k.shape[0], 16, 2, device="cuda")
    out = pad.paged_attention_decode_weights(q, k, v, acc, tab, sl, **s)
    check([3000, 500], q, k, v, table, s, out)
    assert torch.isfinite(acc).all() and abs(float(acc.sum()) - 16) < 1e-3
