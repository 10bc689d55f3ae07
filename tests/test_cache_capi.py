"""The C ABI of the cache operators (include/pa_cache.h): declarations, sizes and refusals (no GPU), and a call."""

from __future__ import annotations

import ctypes
import math
import os
import re
import shutil
import subprocess

import pytest
import torch

from oracle import cache as oracle
from paged_attention_decode_amd import _native

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "pa_cache.h")
# pad_status and formats of include/pa_decode.h, pa_cache.h
NULL, SHAPE, DIM, GQA, STRIDE, ALIGN, WORKSPACE, FORMAT = 1, 2, 3, 4, 5, 6, 7, 12
FP16, E4M3, BF16, MX4 = 0, 1, 3, 6
PTR = 1 << 20  # never read: every call here is refused, or has nothing to do


def cache(**over):
    c = _native.PadKvCache()
    c.k = c.v = c.k_scales = c.v_scales = c.weights = c.positions = PTR
    for name, t in (("k_stride", (4096, 256, 128)), ("v_stride", (4096, 256, 128)), ("ks_stride", (64, 4, 4)),
                    ("vs_stride", (64, 4, 4)), ("w_stride", (32, 2, 1)), ("p_stride", (32, 2, 1))):
        getattr(c, name)[:] = t
    c.num_pages, c.page_size, c.num_kv_heads, c.head_dim, c.kv_format = 8, 16, 2, 128, FP16
    c.k_scale = c.v_scale = 1.0
    for name, value in over.items():
        if isinstance(value, tuple):
            getattr(c, name)[:] = value
        else:
            setattr(c, name, value)
    return c


def rows(**over):
    r = _native.PadKvRows()
    r.k = r.v = r.slots = PTR
    r.k_stride[:] = r.v_stride[:] = (256, 128)
    r.tokens, r.slots64, r.bf16 = 4, 1, 0
    for name, value in over.items():
        if isinstance(value, tuple):
            getattr(r, name)[:] = value
        else:
            setattr(r, name, value)
    return r


def evict_call(**over):
    e = _native.PadKvEvictCall()
    e.block_table = e.seq_lens = e.new_lens = e.workspace = PTR
    e.workspace_bytes = 1 << 30
    e.bt_stride[:] = (4, 1)
    e.sl_stride, e.batch, e.max_pages, e.keep, e.recent = 1, 2, 4, 8, 0
    for name, value in over.items():
        setattr(e, name, value)
    return e


def test_header_and_exports():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    declared = sorted(set(re.findall(r"^\s*int\s+(pad_\w+)\s*\(", text, flags=re.M)))
    assert declared == sorted(_native.CACHE_SIGNATURES)
    for name in declared:
        assert hasattr(_native.capi(), name)


@pytest.mark.parametrize("over,status", [
    ({"k": None}, NULL), ({"v": None}, NULL), ({"kv_format": 99}, FORMAT), ({"kv_format": 4}, FORMAT),
    ({"page_size": 0}, SHAPE), ({"num_kv_heads": 0}, SHAPE), ({"num_pages": 0}, SHAPE), ({"head_dim": 48}, DIM),
    ({"kv_format": E4M3, "head_dim": 96}, DIM), ({"kv_format": MX4, "head_dim": 32}, DIM),
    ({"kv_format": MX4, "k_scales": None}, NULL), ({"kv_format": E4M3, "k_scale": 0.0}, FORMAT),
    ({"kv_format": E4M3, "v_scale": math.nan}, FORMAT), ({"k": PTR + 2}, ALIGN), ({"k_stride": (4096, 252, 128)}, ALIGN),
    ({"kv_format": MX4, "v_stride": (4096, 100, 64)}, ALIGN),
])
def test_cache_refusals(over, status):
    lib = _native.capi()
    c = cache(**over)
    assert lib.pad_kv_append(c, rows(), PTR, PTR, None) == status
    assert lib.pad_kv_read(c, rows(), None) == status
    assert lib.pad_kv_evict(c, evict_call(), None) == status


@pytest.mark.parametrize("over,status", [
    ({"k": None}, NULL), ({"slots": None}, NULL), ({"tokens": -1}, SHAPE), ({"tokens": 1 << 50}, SHAPE),
    ({"v": PTR + 8}, ALIGN), ({"k_stride": (252, 128)}, ALIGN), ({"bf16": 1}, FORMAT), ({"tokens": 0, "k": None}, 0),
])
def test_rows_refusals(over, status):
    lib = _native.capi()
    assert lib.pad_kv_append(cache(), rows(**over), PTR, PTR, None) == status
    assert lib.pad_kv_read(cache(), rows(**over), None) == status


def test_append_state_refusals():
    lib = _native.capi()
    assert lib.pad_kv_append(cache(), rows(), None, None, None) == NULL  # positions without token_positions
    assert lib.pad_kv_append(cache(weights=None, positions=None), rows(), PTR, None, None) == NULL
    assert lib.pad_kv_append(None, rows(), None, None, None) == NULL
    assert lib.pad_kv_append(cache(), None, None, None, None) == NULL


@pytest.mark.parametrize("over,status", [
    ({"batch": -1}, SHAPE), ({"batch": 70000}, SHAPE), ({"keep": -1}, SHAPE), ({"recent": -1}, SHAPE),
    ({"max_pages": -1}, SHAPE), ({"max_pages": 1 << 27}, SHAPE), ({"block_table": None}, NULL), ({"seq_lens": None}, NULL),
    ({"new_lens": None}, NULL), ({"workspace": None}, WORKSPACE), ({"workspace_bytes": 100}, WORKSPACE),
    ({"batch": 0, "workspace": None}, 0),
])
def test_evict_refusals(over, status):
    assert _native.capi().pad_kv_evict(cache(), evict_call(**over), None) == status


def test_evict_needs_weights_and_positions():
    lib = _native.capi()
    assert lib.pad_kv_evict(cache(weights=None), evict_call(), None) == NULL
    assert lib.pad_kv_evict(cache(positions=None), evict_call(), None) == NULL


def test_evict_workspace():
    lib, n = _native.capi(), ctypes.c_size_t()
    assert lib.pad_kv_evict_workspace_bytes(3, 2, 10, 16, ctypes.byref(n)) == 0
    assert n.value >= 6 * (4 + 8 * 80)  # a count and 80 moves of 8 bytes a unit
    assert lib.pad_kv_evict_workspace_bytes(3, 2, 10, 16, None) == NULL
    for bad in ((-1, 2, 10, 16), (3, 0, 10, 16), (3, 2, -1, 16), (3, 2, 10, 0), (3, 2, 1 << 31, 16)):
        assert lib.pad_kv_evict_workspace_bytes(*bad, ctypes.byref(n)) == SHAPE


def _dims(d=128, hq=8, hkv=2, **over):
    dm = _native.PadDims()
    dm.batch, dm.num_q_heads, dm.num_kv_heads, dm.head_dim = 2, hq, hkv, d
    dm.page_size, dm.max_pages, dm.num_pages = 16, 4, 8
    dm.q_stride[:] = dm.out_stride[:] = (hq * d, d, 1)
    dm.k_stride[:] = dm.v_stride[:] = (16 * hkv * d // 2, hkv * d // 2, d // 2, 1)
    dm.bt_stride[:], dm.sl_stride = (4, 1), 1
    for name, value in over.items():
        setattr(dm, name, value)
    return dm


def test_logits_bytes():
    lib, n = _native.capi(), ctypes.c_size_t()
    assert lib.pad_cache_logits_bytes(_dims(), ctypes.byref(n)) == 0
    assert n.value >= 2 * 8 * (64 + 1) * 4
    assert lib.pad_cache_logits_bytes(_dims(), None) == NULL
    assert lib.pad_cache_logits_bytes(_dims(hkv=3), ctypes.byref(n)) == GQA


@pytest.mark.parametrize("call,dims,status", [
    ({}, {"head_dim": 96}, DIM), ({}, {"head_dim": 48}, DIM), ({"indptr": PTR}, {}, SHAPE), ({"worklist": PTR}, {}, SHAPE),
    ({"engine": 1}, {}, FORMAT), ({"kv_format": FP16}, {}, FORMAT), ({"kv_format": 77}, {}, FORMAT),
    ({"kv_format": FP16, "engine": 1, "weights": PTR}, {}, FORMAT), ({"k_scales": None}, {}, NULL),
    ({}, {"page_size": 1 << 20, "max_pages": 1 << 12}, SHAPE), ({}, {"hkv": 3}, GQA),
    ({"weights": PTR}, {"page_size": 1 << 16, "max_pages": 1 << 12}, SHAPE),
])
def test_decode_refusals(call, dims, status):
    dims = dict(dims)
    dm = _dims(hkv=dims.pop("hkv", 2), **dims)
    c = _native.PadCacheCall()
    for name in ("q", "k_cache", "v_cache", "block_table", "seq_lens", "out", "workspace", "counters"):
        setattr(c.call, name, PTR)
    c.call.kv_format, c.call.scale = MX4, 1.0
    c.call.k_scale = c.call.v_scale = 1.0
    c.k_scales = c.v_scales = PTR
    for name, value in call.items():
        setattr(c if hasattr(c, name) else c.call, name, value)
    assert _native.capi().pad_cache_decode(c, dm, None) == status


def test_decode_refuses_rows_of_eight_bytes():
    dm = _dims()
    dm.k_stride[1] = 136
    c = _native.PadCacheCall()
    c.call.kv_format = MX4
    c.k_scales = c.v_scales = PTR
    assert _native.capi().pad_cache_decode(c, dm, None) == ALIGN
    assert _native.capi().pad_cache_decode(None, dm, None) == NULL


def test_structures_match_the_header(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not found")
    structs = {"pad_cache_call": _native.PadCacheCall, "pad_kv_cache": _native.PadKvCache,
               "pad_kv_rows": _native.PadKvRows, "pad_kv_evict_call": _native.PadKvEvictCall}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "pa_cache.h"', "int main(void) {"]
    for cname, py in structs.items():
        lines.append(f'  printf("{cname} sizeof %zu\\n", sizeof({cname}));')
        for fname, _ in py._fields_:
            lines.append(f'  printf("{cname} {fname} %zu\\n", offsetof({cname}, {fname}));')
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join([*lines, "  return 0;", "}"]) + "\n")
    subprocess.run([gcc, "-std=c99", f"-I{os.path.dirname(HEADER)}", str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        cname, field, value = line.split()
        py = structs[cname]
        want = ctypes.sizeof(py) if field == "sizeof" else getattr(py, field).offset
        assert int(value) == want, (cname, field, int(value), want)


@pytest.mark.gpu
def test_decode_through_the_c_abi():
    """Caller-owned scratch of the queried sizes: the package's bits, with weights, twice from the same counters."""
    import paged_attention_decode_amd as pad
    from tests.cache_helpers import Case

    case = Case([900, 3, 0, 64], 8, 2, 128, 16, "fp16", "mx4", seed=5)
    q, k, v, table, lens, s = case.gpu()
    acc = torch.zeros(case.pages, 16, 2, device="cuda")
    want = pad.paged_attention_decode_weights(q, k, v, acc, table, lens, **s)
    lib, out, got = _native.capi(), torch.empty_like(want), torch.zeros_like(acc)
    dm = _native.dims_for(q, k, v, table, lens, out)
    ws, logits, count = ctypes.c_size_t(), ctypes.c_size_t(), ctypes.c_int64()
    assert lib.pad_cache_scratch(dm, MX4, 0, 0, ctypes.byref(ws), ctypes.byref(count)) == 0
    assert lib.pad_cache_scratch(dm, 99, 0, 0, ctypes.byref(ws), ctypes.byref(count)) == FORMAT
    assert lib.pad_cache_logits_bytes(dm, ctypes.byref(logits)) == 0
    scratch = torch.empty(max(ws.value, 1), dtype=torch.uint8, device="cuda")
    counters = torch.zeros(max(count.value, 1), dtype=torch.int32, device="cuda")
    scores = torch.empty(logits.value, dtype=torch.uint8, device="cuda")
    c = _native.PadCacheCall()
    for name, t in (("q", q), ("k_cache", k), ("v_cache", v), ("block_table", table), ("seq_lens", lens), ("out", out),
                    ("workspace", scratch), ("counters", counters)):
        setattr(c.call, name, t.data_ptr())
    c.call.workspace_bytes, c.call.num_counters = scratch.numel(), counters.numel()
    c.call.kv_format, c.call.scale = MX4, case.scale
    c.k_scales, c.v_scales = s["k_scale"].data_ptr(), s["v_scale"].data_ptr()
    c.ks_stride[:], c.vs_stride[:] = s["k_scale"].stride()[:3], s["v_scale"].stride()[:3]
    c.weights, c.logits, c.logits_bytes = got.data_ptr(), scores.data_ptr(), scores.numel()
    c.w_stride[:] = got.stride()
    stream = torch.cuda.current_stream().cuda_stream
    for times in (1, 2):
        assert lib.pad_cache_decode(c, dm, stream) == 0
        torch.cuda.synchronize()
        assert torch.equal(out, want) and (counters == 0).all()
    assert torch.equal(got, acc + acc)
    c.logits_bytes -= 300
    assert lib.pad_cache_decode(c, dm, stream) == WORKSPACE


# ------------------------------------------------------------------ the oracle itself


def test_oracle_mx4_known_values():
    x = torch.zeros(1, 64)
    x[0, :8] = torch.tensor([4.0, 0.25, 0.75, 1.25, -1.75, 2.5, 3.5, -5.0])  # scale 1
    x[0, 32] = 65504.0  # 2^13, 7.996 saturates
    codes, scales = oracle.mx4_encode(x)
    assert scales.tolist() == [[127, 127 + 13]]
    got = oracle.mx4_decode(codes, scales)
    assert got[0, :8].tolist() == [4.0, 0.0, 1.0, 1.0, -2.0, 2.0, 4.0, -4.0]
    assert got[0, 32] == 6.0 * 2**13
    assert oracle.mx4_encode(torch.full((1, 32), math.nan))[1].item() == 255
    assert oracle.mx4_encode(torch.zeros(1, 32))[1].item() == 0


def test_oracle_evict_known_moves():
    table = torch.tensor([[1, 0]])
    w, p = torch.zeros(2, 3, 1), torch.zeros(2, 3, 1, dtype=torch.int32)
    for t, (wt, pt) in enumerate([(5.0, 0), (1.0, 1), (9.0, 2), (1.0, 3), (0.0, 4), (7.0, 5)]):
        w[[1, 0][t // 3], t % 3, 0], p[[1, 0][t // 3], t % 3, 0] = wt, pt
    # newest two: slots 4, 5; then 9.0 (slot 2): slot 4 -> 0, slot 5 -> 1
    assert oracle.evict(w, p, table, [6], 3, 2) == ([3], {(0, 0): [(4, 0), (5, 1)]})
    # by weight alone: 9, 7, 5, then the lower of the two of 1.0
    assert oracle.evict(w, p, table, [6], 4, 0) == ([4], {(0, 0): [(5, 3)]})
