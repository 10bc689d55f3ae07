"""Cache operators on the GPU against their definitions in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

import paged_attention_decode_amd as pad
from oracle import cache as oracle
from tests.cache_helpers import (E4M3, E5M2, FP8, MX4, Case, QTYPES, check_output, check_weights, cuda_like,
                                 eviction_case, head_major)

pytestmark = pytest.mark.gpu


def bits(t):
    t = t.contiguous()
    return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32, 8: torch.int64}[t.element_size()]).cpu()


def rows(tokens, hkv, d, dtype, seed=0):
    """Rows that meet the rounding's corners: ties, saturation, zeros, tiny and huge blocks."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, hkv, d, generator=g, dtype=torch.float64)
    flat = x.view(-1, 32)
    kinds = torch.arange(flat.shape[0]) % 7
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.5, -0.25, -0.75, -1.25, -1.75, -2.5, -5.0])
    flat[kinds == 1] = ties.repeat(2).double()
    flat[kinds == 2] = 0.0
    flat[kinds == 3] *= 2.0**-13
    flat[kinds == 4] *= 1000.0
    flat[kinds == 5, ::3] = -0.0
    return x.to(dtype)


# ------------------------------------------------------------------ append, read


@pytest.mark.parametrize("q", ["fp16", "bf16"])
@pytest.mark.parametrize("kv", ["16", E4M3, E5M2, MX4])
@pytest.mark.parametrize("tokens,hkv,d,ps", [(1, 1, 64, 1), (5, 2, 128, 16), (67, 3, 128, 12), (33, 8, 256, 8),
                                             (300, 2, 64, 3)])
def test_append_then_read(q, kv, tokens, hkv, d, ps):
    dtype = QTYPES[q]
    pages = -(-2 * tokens // ps)
    k, v = rows(tokens, hkv, d, dtype, 1), rows(tokens, hkv, d, dtype, 2)
    g = torch.Generator().manual_seed(3)
    slots = torch.randperm(pages * ps, generator=g)[:tokens]
    slots[torch.rand(tokens, generator=g) < 0.2] = -1
    live = slots >= 0
    scales = {}
    if kv == MX4:
        (kc, ks), (vc, vs) = pad.mx4_cache(pages, ps, hkv, d), pad.mx4_cache(pages, ps, hkv, d)
        scales = {"k_scale": ks, "v_scale": vs}
    else:
        kc, vc = (torch.zeros(pages, ps, hkv, d, dtype=FP8.get(kv, dtype), device="cuda") for _ in range(2))
        if kv != "16":
            scales = {"k_scale": 0.37, "v_scale": 2.5}
    for t in (kc, vc):
        t.view(torch.uint8).fill_(0x25)  # slots without a token keep it
    if kv == MX4:
        ks.fill_(120)
        vs.fill_(120)
    weights, positions = pad.kv_weights(pages, ps, hkv)
    weights.fill_(-3.0)
    positions.fill_(-3)
    tw, tp = torch.rand(tokens, hkv, generator=g), torch.arange(tokens, dtype=torch.int32) + 7
    kc0, vc0 = kc.clone(), vc.clone()
    pad.paged_kv_append(k.cuda(), v.cuda(), kc, vc, slots.cuda(), **scales, weights=weights, positions=positions,
                        token_weights=tw.cuda(), token_positions=tp.cuda())
    page, at = slots[live] // ps, slots[live] % ps
    want_w, want_p = torch.full((pages, ps, hkv), -3.0), torch.full((pages, ps, hkv), -3, dtype=torch.int32)
    want_w[page, at] = tw[live]
    want_p[page, at] = tp[live, None].expand(-1, hkv)
    assert torch.equal(weights.cpu(), want_w) and torch.equal(positions.cpu(), want_p)
    back = pad.paged_kv_read(kc, vc, slots.cuda(), **scales, dtype=dtype)
    for x, cache, cache0, scale, name, got in ((k, kc, kc0, scales.get("k_scale"), "k", back[0]),
                                               (v, vc, vc0, scales.get("v_scale"), "v", back[1])):
        want = bits(cache0).clone()
        if kv == MX4:
            codes, sc = oracle.mx4_encode(x)
            want[page, at] = codes[live]
            want_s = torch.full((pages, ps, hkv, d // 32), 120, dtype=torch.uint8)
            want_s[page, at] = sc[live]
            assert torch.equal(scale.cpu(), want_s)
            values = oracle.mx4_decode(codes, sc).float()
        elif kv == "16":
            want[page, at] = bits(x)[live]
            values = x.float()
        else:
            most = torch.finfo(FP8[kv]).max
            codes = (x.float() / torch.tensor(scale)).clamp(-most, most).to(FP8[kv])
            want[page, at] = bits(codes)[live]
            values = codes.float() * torch.tensor(scale)
        assert torch.equal(bits(cache), want), name
        values = torch.where(live[:, None, None], values, 0.0).to(dtype)
        assert torch.equal(got.float().cpu(), values.float()), name


@pytest.mark.parametrize("q", ["fp16", "bf16"])
def test_append_values_that_are_no_numbers(q):
    dtype = QTYPES[q]
    x = torch.ones(6, 1, 64, dtype=dtype)
    x[0, 0, 5] = math.nan
    x[1, 0, 40] = math.inf
    x[2, 0, 40] = -math.inf
    x[3] = torch.finfo(dtype).max
    x[4] = torch.finfo(dtype).smallest_normal / 8  # subnormal
    x[5, 0, ::2] = -torch.finfo(dtype).tiny
    (kc, ks), (vc, vs) = pad.mx4_cache(2, 4, 1, 64), pad.mx4_cache(2, 4, 1, 64)
    slots = torch.arange(6).cuda()
    pad.paged_kv_append(x.cuda(), x.cuda(), kc, vc, slots, ks, vs)
    codes, scales = oracle.mx4_encode(x)
    assert torch.equal(kc.cpu().reshape(8, 1, 32)[:6], codes) and torch.equal(ks.cpu().reshape(8, 1, 2)[:6], scales)
    got = pad.paged_kv_read(kc, vc, slots, ks, vs, dtype=torch.bfloat16)[0].double().cpu()
    want = oracle.mx4_decode(codes, scales)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(), want.to(torch.bfloat16).double().nan_to_num())
    for kv, most in ((torch.float8_e4m3fn, 448.0), (torch.float8_e5m2, 57344.0)):
        c, c2 = (torch.zeros(2, 4, 1, 64, dtype=kv, device="cuda") for _ in range(2))
        pad.paged_kv_append(x.cuda(), x.cuda(), c, c2, slots, 2.0**-8, 2.0**-8)
        got = c.float().cpu().reshape(8, 64)[:6]
        want = (x.float().view(6, 64) * 256).clamp(-most, most).to(kv).float()
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(), want.nan_to_num())


def test_append_of_strided_rows_int32_slots_and_no_tokens():
    d, hkv, ps = 128, 2, 16
    both = torch.randn(10, 2, hkv, d + 8, dtype=torch.float16, device="cuda")
    k, v = both[:, 0, :, :d], both[:, 1, :, :d]
    kc, vc = (torch.zeros(4, ps, hkv, d, dtype=torch.float16, device="cuda") for _ in range(2))
    slots = torch.tensor([0, 17, 63, 64, -5, 2**31 - 1, 5, 6, 30, 40], dtype=torch.int32, device="cuda")
    pad.paged_kv_append(k, v, kc, vc, slots)
    gk, gv = pad.paged_kv_read(kc, vc, slots.long())
    live = (slots >= 0) & (slots < 64)
    assert torch.equal(gk, torch.where(live[:, None, None], k, 0)) and torch.equal(
        gv, torch.where(live[:, None, None], v, 0))
    odd = torch.randn(3, hkv, d + 1, dtype=torch.float16, device="cuda")[:, :, 1:]  # rows not 16-byte aligned
    pad.paged_kv_append(odd, odd, kc, vc, slots[:3])
    assert torch.equal(pad.paged_kv_read(kc, vc, slots[:3])[0], odd)
    before = kc.clone()
    pad.paged_kv_append(k[:0], v[:0], kc, vc, slots[:0])
    assert torch.equal(kc, before) and pad.paged_kv_read(kc, vc, slots[:0])[0].shape == (0, hkv, d)


def test_append_and_read_past_32_bit_offsets():
    # The last pages of a cache of more than 2^32 bytes.
    ps, hkv, d = 16, 8, 128
    pages = (1 << 32) // (ps * hkv * d) + 9
    kc, vc = (torch.empty(pages, ps, hkv, d, dtype=torch.float16, device="cuda") for _ in range(2))
    x = torch.randn(20, hkv, d, dtype=torch.float16, device="cuda")
    slots = pages * ps - 1 - 7 * torch.arange(20, device="cuda")
    pad.paged_kv_append(x, 2 * x, kc, vc, slots)
    k, v = pad.paged_kv_read(kc, vc, slots)
    assert torch.equal(k, x) and torch.equal(v, 2 * x) and torch.equal(kc[-1, -1], x[0])


# ------------------------------------------------------------------ MX4 decode

LENS = {"short": [1, 0, 2, 15, 16, 17, 31, 32, 33, 48], "ragged": [700, 1, 0, 333, 95], "even": [256] * 3,
        "long": [4097]}


@pytest.mark.parametrize("q", ["fp16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", [(12, 2, 128), (8, 8, 64), (16, 1, 256), (3, 3, 128), (32, 2, 128)])
@pytest.mark.parametrize("ps", [16, 1, 3, 32])
@pytest.mark.parametrize("lens", ["short", "ragged"])
def test_mx4_decode(q, hq, hkv, d, ps, lens):
    case = Case(LENS[lens], hq, hkv, d, ps, q, MX4, seed=hq + d + ps)
    dq, k, v, table, sl, scales = case.gpu()
    out = pad.paged_attention_decode_mx4(dq, k, v, scales["k_scale"], scales["v_scale"], table, sl)
    assert out.dtype == dq.dtype
    expected, _, err = case.expected()
    check_output(case, out, expected, err)
    assert (out[sl == 0] == 0).all()


@pytest.mark.parametrize("splits", [None, 1, 3, 16, 64])
@pytest.mark.parametrize("lens", ["even", "long", "ragged"])
@pytest.mark.parametrize("layout", ["head", "token"])
def test_mx4_decode_splits_and_layouts(splits, lens, layout):
    case = Case(LENS[lens], 8, 2, 128, 16, "fp16", MX4, seed=9, stretch=4.0, layout=layout)
    dq, k, v, table, sl, scales = case.gpu()
    out = pad.paged_attention_decode_mx4(dq, k, v, scales["k_scale"], scales["v_scale"], table.long(), sl.long(),
                                         num_splits=splits)
    expected, _, err = case.expected()
    check_output(case, out, expected, err)


def test_mx4_decode_equals_the_widened_caches():
    # Same values in bfloat16 caches (exact there), and torch's own element types.
    case = Case([500, 64, 129], 12, 2, 128, 16, "bf16", MX4, seed=4)
    dq, k, v, table, sl, s = case.gpu()
    out = pad.paged_attention_decode_mx4(dq, k, v, s["k_scale"], s["v_scale"], table, sl)
    wide_k, wide_v = case.k_values.bfloat16().cuda(), case.v_values.bfloat16().cuda()
    expected, _, err = case.expected()
    check_output(case, pad.paged_attention_decode_ex(dq, wide_k, wide_v, table, sl), expected, err)
    check_output(case, out, expected, err)
    again = pad.paged_attention_decode_mx4(
        dq, k.view(torch.float4_e2m1fn_x2), v.view(torch.float4_e2m1fn_x2), s["k_scale"].view(torch.float8_e8m0fnu),
        s["v_scale"].view(torch.float8_e8m0fnu), table, sl)
    assert torch.equal(bits(out), bits(again))


def test_mx4_stale_slots_and_wild_pages():
    """Codes and scales behind a sequence (NaN scales among them) and page ids outside the cache change nothing."""
    case = Case([37, 5, 0, 65], 8, 2, 128, 16, "fp16", MX4, seed=2)
    dq, k, v, table, sl, s = case.gpu()
    clean = pad.paged_attention_decode_mx4(dq, k, v, s["k_scale"], s["v_scale"], table, sl)
    live = torch.zeros(k.shape[:2], dtype=torch.bool)
    for b, n in enumerate(case.lens):
        t = torch.arange(n)
        live[case.table[b][t // 16].long(), t % 16] = True
    dead = ~live.cuda()
    for t, fill in ((k, 0x7f), (v, 0xff), (s["k_scale"], 255), (s["v_scale"], 255)):
        t[dead] = fill
    for b, n in enumerate(case.lens):
        table[b, -(-n // 16):] = 2**30 if b % 2 else -5
    out = pad.paged_attention_decode_mx4(dq, k, v, s["k_scale"], s["v_scale"], table, sl)
    assert torch.equal(bits(out), bits(clean))


# ------------------------------------------------------------------ weights


@pytest.mark.parametrize("q,kv", [("fp16", None), ("bf16", None), ("fp16", E4M3), ("bf16", E5M2), ("bf16", E4M3),
                                  ("fp16", E5M2), ("fp16", MX4), ("bf16", MX4)])
@pytest.mark.parametrize("hq,hkv,d", [(12, 2, 128), (4, 4, 64), (16, 1, 256)])
@pytest.mark.parametrize("ps", [16, 1, 8, 12])
def test_weights(q, kv, hq, hkv, d, ps):
    case = Case([1, 0, 17, 400, 64, 5], hq, hkv, d, ps, q, kv, seed=d + ps, layout="token" if ps == 8 else "head")
    dq, k, v, table, sl, scales = case.gpu()
    expected, weights, err = case.expected()
    acc = head_major(case.weights.unsqueeze(-1)).squeeze(-1)
    dev = cuda_like(acc)
    out = pad.paged_attention_decode_weights(dq, k, v, dev, table, sl, **scales)
    check_output(case, out, expected, err)
    check_weights(case, case.weights, dev, weights, err)


@pytest.mark.parametrize("d", [32, 96])
@pytest.mark.parametrize("ps", [2, 4, 16, 48])
def test_weights_other_head_dims(d, ps):
    case = Case([3, 130, 0, 77], 6, 2, d, ps, "fp16", seed=d, layout="token")
    dq, k, v, table, sl, _ = case.gpu()
    expected, weights, err = case.expected()
    dev = case.weights.cuda()
    out = pad.paged_attention_decode_weights(dq, k, v, dev, table, sl)
    check_output(case, out, expected, err)
    check_weights(case, case.weights, dev, weights, err)


@pytest.mark.parametrize("splits", [None, 1, 5, 64])
@pytest.mark.parametrize("kv", [None, MX4])
def test_weights_splits_twice_and_the_same_bits(splits, kv):
    case = Case([3000, 40, 1111], 8, 2, 128, 16, "fp16", kv, seed=11, stretch=3.0)
    dq, k, v, table, sl, scales = case.gpu()
    expected, weights, err = case.expected()
    dev = case.weights.cuda()
    out = pad.paged_attention_decode_weights(dq, k, v, dev, table, sl, num_splits=splits, **scales)
    check_output(case, out, expected, err)
    check_weights(case, case.weights, dev, weights, err)
    again = case.weights.cuda()
    out2 = pad.paged_attention_decode_weights(dq, k, v, again, table, sl, num_splits=splits, **scales)
    assert torch.equal(bits(out), bits(out2)) and torch.equal(bits(dev), bits(again))
    once = dev.clone()
    pad.paged_attention_decode_weights(dq, k, v, dev, table, sl, num_splits=splits, **scales)
    check_weights(case, once.cpu(), dev, weights, err)


# ------------------------------------------------------------------ eviction


def _evicted(case_caches, weights, positions, table, lens, keep, recent, ps):
    """The caches after the oracle's moves."""
    new_lens, moves = oracle.evict(weights, positions, table, lens, keep, recent)
    tensors = [t.clone() for t in (*case_caches, weights, positions)]
    for (b, h), pairs in moves.items():
        for s, d in pairs:
            for t in tensors:
                t[int(table[b, d // ps]), d % ps, h] = t[int(table[b, s // ps]), s % ps, h]
    return new_lens, tensors


@pytest.mark.parametrize("kv", ["fp16", "bf16", E4M3, MX4])
@pytest.mark.parametrize("hkv,d,ps", [(2, 128, 16), (1, 64, 1), (3, 256, 12)])
@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 5), (20, 3), (64, 64), (100, 1000), (5000, 10)])
@pytest.mark.parametrize("ties", [False, True])
def test_evict(kv, hkv, d, ps, keep, recent, ties):
    lens = [0, 1, 2, 20, 65, 300, 1100]
    table, pages, w, pos = eviction_case(lens, hkv, ps, seed=keep + recent + ps, ties=ties)
    width = {MX4: d // 2}.get(kv, d)
    dtype = {MX4: torch.uint8, E4M3: torch.uint8}.get(kv, torch.int16)
    g = torch.Generator().manual_seed(1)
    made = [torch.randint(0, 120, (pages, ps, hkv, width), generator=g, dtype=dtype) for _ in range(2)]
    if kv == MX4:
        made += [torch.randint(0, 255, (pages, ps, hkv, d // 32), generator=g, dtype=torch.uint8) for _ in range(2)]
    new_lens, want = _evicted(made, w, pos, table, lens, keep, recent, ps)
    dev = [head_major(t).cuda() if i % 2 else t.cuda() for i, t in enumerate(made)]
    view = {"fp16": torch.float16, "bf16": torch.bfloat16, E4M3: torch.float8_e4m3fn}.get(kv, torch.uint8)
    k, v = dev[0].view(view), dev[1].view(view)
    scales = {"k_scale": dev[2], "v_scale": dev[3]} if kv == MX4 else {}
    dw, dp = cuda_like(w.transpose(1, 2).contiguous().transpose(1, 2)), pos.cuda()
    got = pad.paged_kv_evict(k, v, dw, dp, table.cuda(), torch.tensor(lens).cuda(), keep, recent, **scales)
    assert got.dtype == torch.int32 and got.tolist() == new_lens
    for x, y in zip((*dev, dw, dp), want):
        assert torch.equal(bits(x), bits(y))


@pytest.mark.parametrize("n,keep", [(1024, 1023), (1025, 512), (16384, 9000), (16385, 16000), (40000, 3), (70001, 35000)])
@pytest.mark.parametrize("ties", [False, True])
def test_evict_long_sequences(n, keep, ties):
    ps, hkv, d = 16, 1, 64
    lens = [n, n // 3]
    table, pages, w, pos = eviction_case(lens, hkv, ps, seed=n, ties=ties)
    g = torch.Generator().manual_seed(1)
    made = [torch.randint(0, 1 << 15, (pages, ps, hkv, d), generator=g, dtype=torch.int16) for _ in range(2)]
    keeps = torch.tensor([keep, n // 3 - 1])
    new_lens, want = _evicted(made, w, pos, table, lens, keeps, 32, ps)
    dev = [t.cuda() for t in made]
    dw, dp = w.cuda(), pos.cuda()
    got = pad.paged_kv_evict(dev[0].view(torch.float16), dev[1].view(torch.float16), dw, dp, table.cuda(),
                             torch.tensor(lens, dtype=torch.int32).cuda(), keeps.cuda(), 32)
    assert got.tolist() == new_lens
    for x, y in zip((*dev, dw, dp), want):
        assert torch.equal(bits(x), bits(y))


def test_evict_keeps_of_zero_and_long_lengths():
    """A per-sequence keep of 0 (or less) empties a sequence; a length past its table counts as the table."""
    ps, hkv, d = 4, 2, 64
    table, pages, w, pos = eviction_case([12, 12, 12], hkv, ps, seed=3)
    table = table[:, :3].contiguous()
    k, v = (torch.randn(pages, ps, hkv, d, dtype=torch.float16, device="cuda") for _ in range(2))
    k0 = k.clone()
    got = pad.paged_kv_evict(k, v, w.cuda(), pos.cuda(), table.cuda(), torch.tensor([12, 12, 2**31 - 1]).cuda(),
                             torch.tensor([0, -4, 12]).cuda())
    assert got.tolist() == [0, 0, 12] and torch.equal(k, k0)


# ------------------------------------------------------------------ together


@pytest.mark.parametrize("kv", ["fp16", E4M3, MX4])
def test_generation_with_a_bounded_cache(kv):
    """append -> decode with weights -> evict, step by step, against the same steps on the CPU."""
    hq, hkv, d, ps, keep, recent, batch = 4, 2, 64, 16, 40, 8, 3
    pages_each = 4  # 64 slots a sequence
    pages = batch * pages_each
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(0)).view(batch, pages_each).int()
    dt = FP8.get(kv, torch.float16)
    if kv == MX4:
        (k, ks), (v, vs) = pad.mx4_cache(pages, ps, hkv, d), pad.mx4_cache(pages, ps, hkv, d)
        scales = {"k_scale": ks, "v_scale": vs}
    else:
        k, v = (torch.zeros(pages, ps, hkv, d, dtype=dt, device="cuda") for _ in range(2))
        scales = {"k_scale": 0.05, "v_scale": 0.05} if kv in FP8 else {}
    weights, positions = pad.kv_weights(pages, ps, hkv)
    lens = torch.zeros(batch, dtype=torch.int32, device="cuda")
    dtable = table.cuda()
    g = torch.Generator().manual_seed(1)
    held = [[dict() for _ in range(hkv)] for _ in range(batch)]  # position -> (key row, value row, weight)
    for step in range(60):
        new = [30, 50, 1][step] if step < 3 else 1
        x = torch.randn(2, batch * new, hkv, d, generator=g).half()
        if step < 3:  # a prompt's part for sequence `step` only
            slots = torch.full((batch, new), -1, dtype=torch.int64, device="cuda")
            at = lens[step].long() + torch.arange(new, device="cuda")
            slots[step] = dtable[step].long()[at // ps] * ps + at % ps
            grown = torch.zeros_like(lens)
            grown[step] = new
        else:
            at = lens.long()
            slots = (dtable.long().gather(1, (at // ps)[:, None]) * ps + (at % ps)[:, None])
            grown = torch.ones_like(lens)
        pos = (1000 * step + torch.arange(new, dtype=torch.int32)).repeat(batch).cuda()
        pad.paged_kv_append(x[0].cuda(), x[1].cuda(), k, v, slots.flatten(), **scales, weights=weights,
                            positions=positions, token_positions=pos)
        lens = lens + grown
        if kv in FP8:  # exactly: a read rounds codes times scale to 16 bits
            f, unit = slots.flatten().clamp(min=0), torch.tensor(0.05).double().cuda()
            rk, rv = (c.view(torch.uint8)[f // ps, f % ps].view(dt).double() * unit for c in (k, v))
        else:
            rk, rv = pad.paged_kv_read(k, v, slots.flatten(), **scales, dtype=torch.float16)
        for i, s in enumerate(slots.flatten().tolist()):
            if s >= 0:
                for h in range(hkv):
                    held[i // new][h][int(pos[i])] = [rk[i, h].double().cpu(), rv[i, h].double().cpu(), 0.0]
        q = torch.randn(batch, hq, d, generator=g).half()
        out = pad.paged_attention_decode_weights(q.cuda(), k, v, weights, dtable, lens, **scales)
        for b in range(batch):
            for h in range(hq):
                mine = held[b][h // 2]
                if not mine:
                    assert (out[b, h] == 0).all()
                    continue
                kk, vv = (torch.stack([r[j] for r in mine.values()]) for j in (0, 1))
                p = torch.softmax(kk @ q[b, h].double() / math.sqrt(d), 0)
                # Two roundings of weights and one of the output, 2^-11 each, of values below 6.
                assert (out[b, h].double().cpu() - p @ vv).abs().max() < 3 * 6 * 2.0**-11
                for r, w in zip(mine.values(), p.tolist()):
                    r[2] += w
        lens = pad.paged_kv_evict(k, v, weights, positions, dtable, lens, keep, recent, **{
            n: s for n, s in scales.items() if kv == MX4})
        assert int(lens.max()) <= keep
        wc, pc = weights.cpu(), positions.cpu()
        for b in range(batch):
            n = int(lens[b])
            t = torch.arange(n)
            for h in range(hkv):
                got = dict(zip(pc[table[b][t // ps].long(), t % ps, h].tolist(),
                               wc[table[b][t // ps].long(), t % ps, h].tolist()))
                mine = held[b][h]
                assert len(got) == n and set(got) <= set(mine)
                gone = set(mine) - set(got)
                if gone:
                    newest = max(mine)
                    assert all(p <= newest - recent for p in gone)
                    others = [w for p, w in got.items() if p <= newest - recent]
                    # No evicted token was heavier than a kept one, but for the roundings of the sums: a
                    # score is a sum of 64 products whose sizes add up to less than 16, 68 roundings of
                    # 2^-24 of that, 7e-5 of a weight; the weights of a step's two heads are at most 2 together.
                    assert not others or max(mine[p][2] for p in gone) <= min(others) + 1e-4
                for p in gone:
                    del mine[p]
                assert all(abs(w - mine[p][2]) < 1e-4 * (1 + w) for p, w in got.items())


def _state(kv="fp16"):
    case = Case([200, 33, 1], 8, 2, 128, 16, "fp16", kv, seed=6)
    return case, case.gpu()


def test_graph_replays_with_new_inputs():
    case, (q, k, v, table, lens, s) = _state(MX4)
    weights, positions = (t.contiguous() for t in pad.kv_weights(case.pages, 16, 2))
    positions.copy_(torch.arange(positions.numel(), device="cuda", dtype=torch.int32).view_as(positions))
    rows_k, rows_v = (torch.randn(3, 2, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    slots = torch.zeros(3, dtype=torch.int64, device="cuda")
    tp = torch.zeros(3, dtype=torch.int32, device="cuda")

    def step(lens_in):
        pad.paged_kv_append(rows_k, rows_v, k, v, slots, **s, weights=weights, positions=positions, token_positions=tp)
        a = pad.paged_attention_decode_mx4(q, k, v, s["k_scale"], s["v_scale"], table, lens_in)
        b = pad.paged_attention_decode_weights(q, k, v, weights, table, lens_in, **s)
        return a, b, pad.paged_kv_evict(k, v, weights, positions, table, lens_in, 64, 4, **s)

    stream = torch.cuda.Stream()
    static_lens = lens.clone()
    saved = [t.clone() for t in (k, v, s["k_scale"], s["v_scale"], weights, positions)]
    live = (k, v, s["k_scale"], s["v_scale"], weights, positions)

    def restore():
        for t, x in zip(live, saved):
            t.copy_(x)

    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(static_lens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = step(static_lens)
    for i in range(4):
        g = torch.Generator().manual_seed(50 + i)
        rows_k.copy_(torch.randn(3, 2, 128, generator=g).half())
        rows_v.copy_(torch.randn(3, 2, 128, generator=g).half())
        q.copy_(torch.randn(q.shape, generator=g).half())
        slots.copy_(torch.randperm(case.pages * 16, generator=g)[:3])
        tp.fill_(10**6 + i)
        static_lens.copy_(torch.tensor([200 - 60 * i, 33 - i, i]))
        restore()
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in (*got, *live)]
        restore()
        eager = step(static_lens)
        torch.cuda.synchronize()
        for x, y in zip(replayed, (*eager, *live)):
            assert torch.equal(bits(x), bits(y))


def test_another_stream_and_two_at_once():
    case, (q, k, v, table, lens, s) = _state(MX4)
    want = pad.paged_attention_decode_mx4(q, k, v, s["k_scale"], s["v_scale"], table, lens)
    streams = [torch.cuda.Stream() for _ in range(2)]
    acc = [torch.zeros(case.pages, 16, 2, device="cuda") for _ in range(2)]
    one = torch.zeros(case.pages, 16, 2, device="cuda")
    pad.paged_attention_decode_weights(q, k, v, one, table, lens, **s)
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for st, a in zip(streams, acc):
            with torch.cuda.stream(st):
                outs.append(pad.paged_attention_decode_mx4(q, k, v, s["k_scale"], s["v_scale"], table, lens))
                a.zero_()
                pad.paged_attention_decode_weights(q, k, v, a, table, lens, **s)
    torch.cuda.synchronize()
    assert all(torch.equal(bits(o), bits(want)) for o in outs)
    assert all(torch.equal(bits(a), bits(one)) for a in acc)


def test_views_of_larger_buffers():
    """Codes and scales of K and V in one buffer per page, tables and lengths as strided views: the same bits."""
    case, (q, k, v, table, lens, s) = _state(MX4)
    pages, ps, hkv, d = case.pages, 16, 2, 128
    weights, positions = pad.kv_weights(pages, ps, hkv)
    positions.copy_(torch.randperm(pages * ps, device="cuda").view(pages, ps, 1).expand(-1, -1, hkv))
    code, scale = ps * hkv * d // 2, ps * hkv * d // 32
    buf = torch.full((pages, 2 * (code + scale) + 64), 0x5a, dtype=torch.uint8, device="cuda")
    step = buf.shape[1]

    def view(at, width):
        return buf.as_strided((pages, ps, hkv, width), (step, hkv * width, width, 1), at)

    k2, v2, ks2, vs2 = view(0, d // 2), view(code, d // 2), view(2 * code, d // 32), view(2 * code + scale, d // 32)
    for x, y in ((k2, k), (v2, v), (ks2, s["k_scale"]), (vs2, s["v_scale"])):
        x.copy_(y)
    state = torch.zeros(pages, hkv, 3, ps, 2, device="cuda")
    w2 = state[:, :, 1, :, 0].transpose(1, 2)
    p2 = torch.zeros(ps, pages, hkv, dtype=torch.int32, device="cuda").transpose(0, 1)
    p2.copy_(positions)
    wide = torch.full((len(case.lens), 2 * table.shape[1]), -1, dtype=torch.int32, device="cuda")
    wide[:, ::2] = table
    t2, l2 = wide[:, ::2], torch.stack([lens, lens + 7], 1)[:, 0]
    rows = torch.randn(3, 2, hkv, d, dtype=torch.float16, device="cuda")
    slots = torch.tensor([3, -1, 40], device="cuda")
    tp = torch.tensor([900, 901, 902], dtype=torch.int32, device="cuda")
    for kk, vv, a, b, w, p in ((k, v, s["k_scale"], s["v_scale"], weights, positions), (k2, v2, ks2, vs2, w2, p2)):
        pad.paged_kv_append(rows[:, 0], rows[:, 1], kk, vv, slots, a, b, weights=w, positions=p, token_positions=tp)
    assert torch.equal(bits(pad.paged_kv_read(k, v, slots, s["k_scale"], s["v_scale"])[1]),
                       bits(pad.paged_kv_read(k2, v2, slots, ks2, vs2)[1]))
    one = pad.paged_attention_decode_weights(q, k, v, weights, table, lens, **s)
    two = pad.paged_attention_decode_weights(q, k2, v2, w2, t2, l2, k_scale=ks2, v_scale=vs2)
    assert torch.equal(bits(one), bits(two)) and torch.equal(bits(weights), bits(w2))
    assert torch.equal(bits(pad.paged_attention_decode_mx4(q, k, v, s["k_scale"], s["v_scale"], table, lens)),
                       bits(pad.paged_attention_decode_mx4(q, k2, v2, ks2, vs2, t2, l2)))
    n1 = pad.paged_kv_evict(k, v, weights, positions, table, lens, 30, 4, **s)
    n2 = pad.paged_kv_evict(k2, v2, w2, p2, t2, l2, 30, 4, k_scale=ks2, v_scale=vs2)
    assert torch.equal(n1, n2)
    for x, y in ((k, k2), (v, v2), (s["k_scale"], ks2), (s["v_scale"], vs2), (weights, w2), (positions, p2)):
        assert torch.equal(bits(x), bits(y))
    assert (buf[:, -64:] == 0x5a).all() and (state[:, :, 0] == 0).all() and (state[..., 1] == 0).all()


def test_sixteen_bit_caches_with_kv_interleaved():
    """K and V as halves of one buffer, kv heads outermost: append, weights and eviction as on plain caches."""
    ps, hkv, d, lens_l = 12, 3, 96, [50, 0, 7, 121]
    table, pages, w, p = eviction_case(lens_l, hkv, ps, seed=8)
    both = torch.randn(hkv, pages, ps, 2, d, dtype=torch.float16, device="cuda")
    k2, v2 = both[:, :, :, 0].permute(1, 2, 0, 3), both[:, :, :, 1].permute(1, 2, 0, 3)
    k1, v1 = k2.contiguous(), v2.contiguous()
    lens = torch.tensor(lens_l, dtype=torch.int32, device="cuda")
    dt = table.cuda()
    q = torch.randn(4, 6, d, dtype=torch.float16, device="cuda")
    w1, p1, w2, p2 = w.cuda(), p.cuda(), head_major(w.unsqueeze(-1)).squeeze(-1).cuda(), p.cuda()
    rows = torch.randn(5, hkv, d, dtype=torch.float16, device="cuda")
    slots = torch.tensor([0, 5, 12, 31, -2], dtype=torch.int32, device="cuda")
    results = []
    for k, v, ww, pp in ((k1, v1, w1, p1), (k2, v2, w2, p2)):
        pad.paged_kv_append(rows, 2 * rows, k, v, slots)
        out = pad.paged_attention_decode_weights(q, k, v, ww, dt, lens)
        n = pad.paged_kv_evict(k, v, ww, pp, dt, lens, 20, 5)
        results.append([out, n, k, v, ww, pp, *pad.paged_kv_read(k, v, slots)])
    for x, y in zip(*results):
        assert torch.equal(bits(x), bits(y))


def test_wild_page_ids_write_nothing():
    """An id outside the cache neither faults nor gives page 0 weights or rows."""
    case, (q, k, v, table, lens, s) = _state(MX4)
    weights, positions = (x.contiguous() for x in pad.kv_weights(case.pages, 16, 2))
    bad = table.clone()
    bad[0, 3], bad[0, 12], bad[1, 0] = 2**30, -1, case.pages
    pad.paged_attention_decode_weights(q, k, v, weights, bad, lens, **s)
    real = torch.zeros(case.pages, 16, dtype=torch.bool, device="cuda")
    for b, n in enumerate(case.lens):
        t = torch.arange(n, device="cuda")
        ids = bad[b].long()[t // 16]
        ok = (ids >= 0) & (ids < case.pages)
        real[ids[ok], (t % 16)[ok]] = True
    assert (weights[~real] == 0).all() and (weights[real] > 0).all()
    before = [x.clone() for x in (k, v, *s.values(), weights, positions)]
    n = pad.paged_kv_evict(k, v, weights, positions, bad, lens, 20, 0, **s)
    assert n.tolist() == [20, 20, 1]
    for x, y in zip((k, v, *s.values(), weights, positions), before):
        assert torch.equal(bits(x)[~real.cpu()], bits(y)[~real.cpu()])


def test_empty_batch_and_empty_tables():
    k, v = (torch.zeros(2, 16, 2, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    w, p = pad.kv_weights(2, 16, 2)
    none = torch.zeros(0, 3, dtype=torch.int32, device="cuda")
    lens = torch.zeros(0, dtype=torch.int32, device="cuda")
    q = torch.zeros(0, 4, 128, dtype=torch.float16, device="cuda")
    assert pad.paged_attention_decode_weights(q, k, v, w, none, lens).shape == (0, 4, 128)
    assert pad.paged_kv_evict(k, v, w, p, none, lens, 4).shape == (0,)
    table, lens = torch.zeros(2, 0, dtype=torch.int32, device="cuda"), torch.tensor([0, 9], device="cuda")
    q = torch.ones(2, 4, 128, dtype=torch.float16, device="cuda")
    assert (pad.paged_attention_decode_weights(q, k, v, w, table, lens) == 0).all()
    assert pad.paged_kv_evict(k, v, w, p, table, lens, 4).tolist() == [0, 0]
    (kc, ks), (vc, vs) = pad.mx4_cache(2, 16, 2, 128), pad.mx4_cache(2, 16, 2, 128)
    assert (pad.paged_attention_decode_mx4(q, kc, vc, ks, vs, table, lens) == 0).all()
    assert (w == 0).all()


# ------------------------------------------------------------------ refusals


def test_refusals():
    case, (q, k, v, table, lens, s) = _state(MX4)
    ks, vs = s["k_scale"], s["v_scale"]
    w, p = pad.kv_weights(case.pages, 16, 2)
    x = torch.zeros(3, 2, 128, dtype=torch.float16, device="cuda")
    slots = torch.zeros(3, dtype=torch.int64, device="cuda")
    half = torch.zeros(case.pages, 16, 2, 128, dtype=torch.float16, device="cuda")
    e4 = half.to(torch.float8_e4m3fn)
    A, R, M, W, E = (pad.paged_kv_append, pad.paged_kv_read, pad.paged_attention_decode_mx4,
                     pad.paged_attention_decode_weights, pad.paged_kv_evict)
    calls = [
        lambda: M(q.cpu(), k, v, ks, vs, table, lens),
        lambda: M(q, half, half, None, None, table, lens),
        lambda: M(q, k, v, 1.0, 1.0, table, lens),
        lambda: M(q, k, v, ks[:, :, :, :2], vs, table, lens),
        lambda: M(q.float(), k, v, ks, vs, table, lens),
        lambda: M(q[:, :7], k, v, ks, vs, table, lens),
        lambda: M(q[:, :, :64], k, v, ks, vs, table, lens),
        lambda: M(q, k, v, ks, vs, table[:2], lens),
        lambda: M(q, k, v, ks, vs, table, lens.float()),
        lambda: M(q, k, v, ks, vs, table, lens, num_splits=0),
        lambda: M(torch.zeros(3, 64, 128, dtype=torch.float16, device="cuda"), k, v, ks, vs, table, lens),
        lambda: W(q, half, half, w.double(), table, lens),
        lambda: W(q, half, half, w[:, :8], table, lens),
        lambda: W(q, half, half, w[:1, :1].expand(*w.shape), table, lens),
        lambda: W(q.bfloat16(), half, half, w, table, lens),
        lambda: W(q, half, half, w, table, lens, k_scale=2.0),
        lambda: W(q, e4, e4, w, table, lens, k_scale=0.0),
        lambda: W(q, e4, e4, w, table, lens, k_scale=ks),
        lambda: W(q, k, v, w, table, lens),
        lambda: A(x, x, half, half, slots[:2]),
        lambda: A(x.bfloat16(), x.bfloat16(), half, half, slots),
        lambda: A(x.float(), x.float(), half, half, slots),
        lambda: A(x, x, k, v, slots),
        lambda: A(x, x, half, half, slots.float()),
        lambda: A(x, x, half, half, slots, positions=p),
        lambda: A(x, x, half, half, slots, token_weights=torch.zeros(3, 2, device="cuda")),
        lambda: A(x, x, half, half, slots, token_positions=torch.zeros(3, dtype=torch.int32, device="cuda")),
        lambda: A(x, x, half, half, slots, weights=w, token_weights=torch.zeros(3, 1, device="cuda")),
        lambda: A(x, x, half[:, :, :1].expand(-1, -1, 2, -1), half, slots),
        lambda: A(x[:, :1], x[:, :1], half, half, slots),
        lambda: R(half, half, slots, dtype=torch.bfloat16),
        lambda: R(half, half, slots, dtype=torch.float32),
        lambda: R(half, half.bfloat16(), slots),
        lambda: R(half, half, slots.view(1, 3)),
        lambda: E(half, half, w, p, table, lens, 0),
        lambda: E(half, half, w, p, table, lens, 4, -1),
        lambda: E(half, half, w, p.long(), table, lens, 4),
        lambda: E(half, half, w, p, table, lens, torch.ones(2, dtype=torch.int32, device="cuda")),
        lambda: E(k, v, w, p, table, lens, 4),
        lambda: E(half, half, w, p, table.cpu(), lens, 4),
        lambda: pad.mx4_cache(2, 16, 2, 96),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(AssertionError):
            call()
            pytest.fail(f"call {i} was taken")
    # Rows that the kernels cannot read 16 bytes at a time.
    odd = torch.zeros(case.pages, 16, 2, 68, dtype=torch.uint8, device="cuda")[..., :64]
    with pytest.raises(RuntimeError):
        M(q, odd, odd, ks, vs, table, lens)
    with pytest.raises(RuntimeError):
        A(x, x, odd, odd, slots, ks, vs)
