"""The cache operators next to the decode: what they are measured on, and their plain forms.

A case is one call (or the short run of calls that belong together) as a
serving program makes it.  ``op`` names the operator:

* ``mx4_write``: new tokens' K/V rows are stored in MX4 caches
  (``paged_kv_append``) and read back as the caches stand for them
  (``paged_kv_read``), as a prompt that is prefilled in chunks does;
* ``mx4_decode``: one decode step's attention over MX4 caches
  (``paged_attention_decode_mx4``);
* ``weights``: a decode step that also adds every token's attention weight to
  its slot (``paged_attention_decode_weights``);
* ``evict``: new tokens are appended with the weights that they come with, and
  the sequences are cut back to ``keep`` tokens (``paged_kv_append``,
  ``paged_kv_evict``).

Fields: ``batch``, ``hq``, ``hkv``, ``d``, ``ps`` as elsewhere (page size);
``lo``, ``hi``: lengths are uniform in [lo, hi], drawn from ``lens``, the two
ends among them; ``room``: tokens that a table row has columns for; ``q``: the
type of q, of new rows and of the output; ``kv``: the caches' type.
``mx4_write`` has ``tokens`` rows, of which a share ``skip`` is padding;
``evict`` has ``keep``, ``recent`` and ``new`` tokens per sequence.
"""

import math
import random

import torch

own = False

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2,
          "mx4": torch.uint8}
_FP8_MAX = {"e4m3": 448.0, "e5m2": 57344.0}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
# One key row in this many is scaled by 8: outliers that move a running
# softmax maximum in the middle of a sequence.
_OUTLIERS = 4096


def _write(name, tokens, hkv, d, ps, q, skip=0.0):
    c = {"name": name} if name else {}
    c.update(op="mx4_write", tokens=tokens, hkv=hkv, d=d, ps=ps, q=q, kv="mx4", skip=skip)
    return c


def _decode(name, op, batch, hq, hkv, d, ps, lo, hi, q="fp16", kv="mx4", room=None, lens=1):
    c = {"name": name} if name else {}
    c.update(op=op, batch=batch, hq=hq, hkv=hkv, d=d, ps=ps, lo=lo, hi=hi, room=room or hi, q=q, kv=kv, lens=lens)
    return c


def _evict(name, batch, hkv, d, ps, keep, recent, new, q="fp16", kv=None):
    c = {"name": name} if name else {}
    c.update(op="evict", batch=batch, hkv=hkv, d=d, ps=ps, keep=keep, recent=recent, new=new, q=q, kv=kv or q)
    return c


def listed():
    return [
        # The new tokens of one decode step of 64 sequences.
        _write("write_step_64", 64, 8, 128, 16, "bf16"),
        # A chunk of prompts, padded: some tokens have no slot.
        _write("write_prompt_16k", 16000, 8, 128, 16, "fp16", skip=0.05),
        # One user, a short context: the smallest attention call.
        _decode("mx4_b1_1k", "mx4_decode", 1, 12, 2, 128, 16, 1024, 1024),
        # The ordinary uniform batch.
        _decode("mx4_b64_4k", "mx4_decode", 64, 12, 2, 128, 16, 4096, 4096),
        # A ragged batch, from one token to 8192, of a bfloat16 model.
        _decode("mx4_b64_ragged_8k", "mx4_decode", 64, 32, 8, 128, 32, 1, 8192, q="bf16"),
        # One long document.
        _decode("mx4_b1_128k", "mx4_decode", 1, 32, 8, 128, 16, 131072, 131072),
        # A small head dimension in an odd batch over a token-granular pool.
        _decode("mx4_b27_d64_page1", "mx4_decode", 27, 32, 8, 64, 1, 1, 4096, q="bf16"),
        # A few users: latency of the accumulating step.
        _decode("weights_b4_2k", "weights", 4, 12, 2, 128, 16, 100, 2048, kv="fp16"),
        # The ordinary uniform batch, accumulating.
        _decode("weights_b64_4k", "weights", 64, 12, 2, 128, 16, 4096, 4096, kv="fp16"),
        # A ragged batch over fp8 caches, its table wider than the lengths.
        _decode("weights_b48_fp8_ragged", "weights", 48, 32, 8, 128, 16, 1, 6000, q="bf16", kv="e4m3", room=8192),
        # Every step one token comes and one goes.
        _evict("evict_step_b64", 64, 2, 128, 16, 2048, 64, 1),
        # A long prompt comes in chunks of 1024 tokens into a cache of 4096.
        _evict("evict_chunk_b16", 16, 8, 128, 16, 4096, 1024, 1024, q="bf16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)) - 1e-9))))


# (query heads, kv heads, head_dim)
_HEADS = [(12, 2, 128), (12, 2, 128), (32, 8, 128), (32, 8, 128), (64, 8, 128), (8, 1, 128), (16, 2, 128),
          (32, 32, 128), (32, 8, 64), (16, 16, 64), (16, 4, 256), (16, 1, 256)]
_PAGES = [16, 16, 16, 32, 64, 1, 8, 2, 4, 3, 12, 24, 48]


def draw(rng):
    """One more case of the listed ranges."""
    op = rng.choice(["mx4_write", "mx4_decode", "mx4_decode", "weights", "weights", "evict"])
    hq, hkv, d = rng.choice(_HEADS)
    ps = rng.choice(_PAGES)
    q = rng.choice(["fp16", "bf16"])
    if op == "mx4_write":
        most = 16000 * 8 * 128 // (hkv * d)
        return _write(None, _log_int(rng, 1, most), hkv, d, ps, q, rng.choice([0.0, 0.0, 0.1, 0.5]))
    if op == "evict":
        kv = rng.choice([q, q, q, "e4m3", "e5m2"])
        batch = _log_int(rng, 1, 64)
        keep = _log_int(rng, 16, max(17, min(16384, (1 << 26) // (batch * hkv * d))))
        new = _log_int(rng, 1, max(2, keep // 2))
        return _evict(None, batch, hkv, d, ps, keep, rng.randint(0, keep), new, q, kv)
    kv = "mx4" if op == "mx4_decode" else rng.choice([q, q, q, "e4m3", "e5m2", "mx4"])
    batch = _log_int(rng, 1, 128)
    most = int(min(131072, max(64, (1 << 27) / (hkv * d * batch))))
    hi = _log_int(rng, 64, most)
    lo = hi if rng.random() < 0.35 else rng.randint(1, max(1, hi // 2))
    room = hi if rng.random() < 0.6 else min(131072, hi * rng.randint(2, 4))
    return _decode(None, op, batch, hq, hkv, d, ps, lo, hi, q, kv, room, rng.randrange(1 << 30))


def _lengths(case):
    """The lengths of the case's sequences, in no order that means anything."""
    rng = random.Random(case["lens"])
    lens = [rng.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
    lens[-1] = case["hi"]
    if case["batch"] > 1:
        lens[0] = case["lo"]
    return lens


def _pages(n, ps):
    return -(-n // ps)


# MX4 caches: two e2m1 codes a byte (the even element in the low nibble) and
# one power-of-two scale a 32 elements, rows of one kv head next to each
# other within a page.


def _quantise(x):
    """Rows of values -> (codes, scale codes)."""
    x = x.float()
    blocks = x.unflatten(-1, (-1, 32))
    top = blocks.abs().amax(-1)
    bad = ~torch.isfinite(top)
    e = (torch.frexp(top)[1] - 3).clamp(-127, 127)  # floor(log2) - 2
    e = torch.where((top == 0) | bad, -127, e)
    y = torch.ldexp(blocks.double(), -e.unsqueeze(-1)).float()
    a = y.abs()
    # Half-way values go to the even code.
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int()
            + (a >= 3.5).int() + (a > 5.0).int())
    code = torch.where(bad.unsqueeze(-1), 0, code + 8 * torch.signbit(y).int()).flatten(-2)
    return ((code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8),
            torch.where(bad, 255, e + 127).to(torch.uint8))


def _values(codes, scales):
    """(codes, scale codes) -> rows of values, in 32 bits."""
    table = torch.tensor(_E2M1, device=codes.device)
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    scale = torch.exp2(scales.float() - 127)
    scale = torch.where(scales == 255, float("nan"), scale)
    return (table[c].unflatten(-1, (-1, 32)) * scale.unsqueeze(-1)).flatten(-2)


def _head_major(pages, ps, hkv, width, dtype):
    return torch.zeros(pages, hkv, ps, width, dtype=dtype, device="cuda").transpose(1, 2)


def _store(cache, slots, rows):
    """Rows into the cache's slots, whatever its strides."""
    ps = cache.shape[1]
    cache[slots // ps, slots % ps] = rows


def _caches(case, gen, num_pages):
    """K and V as a serving program holds them: normal, a few outlying keys; quantised caches of such values."""
    ps, hkv, d, kv = case["ps"], case["hkv"], case["d"], case["kv"]
    made, scales = [], []
    for which in ("k", "v"):
        shape = (num_pages, ps, hkv, d)
        if kv == "mx4":
            codes = _head_major(num_pages, ps, hkv, d // 2, torch.uint8)
            scale = _head_major(num_pages, ps, hkv, d // 32, torch.uint8)
            step = max(1, (1 << 25) // (ps * hkv * d))
            for p in range(0, num_pages, step):
                n = min(step, num_pages - p)
                x = torch.randn(n, ps, hkv, d, generator=gen, device="cuda")
                if which == "k":
                    hot = torch.rand(n, ps, hkv, 1, generator=gen, device="cuda") < 1.0 / _OUTLIERS
                    x = torch.where(hot, 8 * x, x)
                codes[p:p + n], scale[p:p + n] = _quantise(x)
            made.append(codes)
            scales.append(scale)
            continue
        x = torch.randn(shape, generator=gen, device="cuda", dtype=_TYPES[case["q"]])
        if which == "k":
            rows = x.view(-1, hkv, d)
            hot = torch.randint(0, rows.shape[0], (max(1, rows.shape[0] // _OUTLIERS),), generator=gen, device="cuda")
            rows[hot] = rows[hot] * 8
        scale = None
        if kv in _FP8_MAX:
            scale = float(x.abs().max()) / (0.875 * _FP8_MAX[kv])
            x = (x.float() / scale).to(_TYPES[kv])
        made.append(x)
        scales.append(scale)
    return made, scales


def _table(case, lens, gen_seed, spare=0):
    """A block table over scattered pages, and how many pages there are."""
    ps = case["ps"]
    pages = [_pages(n, ps) for n in lens]
    total = sum(pages) + spare
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(gen_seed)).to(torch.int32)
    width = max(_pages(case.get("room", 0), ps), max(pages))
    table = torch.zeros(len(lens), width, dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, total


def prepare(case, seed):
    """The caches, the page index and this step's rows, as the program holds them before the call."""
    rng = random.Random(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, ps, hkv, d = _TYPES[case["q"]], case["ps"], case["hkv"], case["d"]
    st = {"case": dict(case)}
    if case["op"] == "mx4_write":
        t = case["tokens"]
        pages = _pages(2 * t, ps)
        st["k_cache"], st["v_cache"] = (_head_major(pages, ps, hkv, d // 2, torch.uint8) for _ in range(2))
        st["k_scale"], st["v_scale"] = (_head_major(pages, ps, hkv, d // 32, torch.uint8) for _ in range(2))
        slots = torch.randperm(pages * ps, generator=gen, device="cuda")[:t]
        if case["skip"]:
            slots[torch.rand(t, generator=gen, device="cuda") < case["skip"]] = -1
        st["slots"] = slots
        st["k"], st["v"] = (torch.randn(t, hkv, d, generator=gen, device="cuda").mul_(2.0).to(dt) for _ in range(2))
        return st
    if case["op"] == "evict":
        b, n, new = case["batch"], case["keep"], case["new"]
        table, total = _table(case, [n + new] * b, seed)
        (st["k_cache"], st["v_cache"]), (st["k_scale"], st["v_scale"]) = _caches(case, gen, total)
        st["table"] = table.cuda()
        st["lens"] = torch.full((b,), n + new, dtype=torch.int32, device="cuda")
        # Attention weights are spread over many orders of magnitude.
        shape = (total, hkv, ps)
        st["weights"] = torch.randn(shape, generator=gen, device="cuda").mul_(3.0).exp_().transpose(1, 2)
        at = torch.arange(n + new)
        slots = (table[:, at // ps].long() * ps + at % ps).cuda()
        st["positions"] = torch.zeros(shape, dtype=torch.int32, device="cuda").transpose(1, 2)
        ages = torch.argsort(torch.rand(b, hkv, n, generator=gen, device="cuda"), -1).int()  # a cache cut before
        _store(st["positions"], slots[:, :n].flatten(), ages.transpose(1, 2).flatten(0, 1))
        st["slots"] = slots[:, n:].flatten().contiguous()
        t = b * new
        st["k"], st["v"] = (torch.randn(t, hkv, d, generator=gen, device="cuda").to(dt) for _ in range(2))
        st["token_weights"] = torch.randn(t, hkv, generator=gen, device="cuda").mul_(3.0).exp_()
        st["token_positions"] = (n - new + torch.arange(new, dtype=torch.int32)).repeat(b).cuda()
        return st
    lens = _lengths(case)
    rng.shuffle(lens)
    table, total = _table(case, lens, seed)
    (st["k_cache"], st["v_cache"]), (st["k_scale"], st["v_scale"]) = _caches(case, gen, total)
    st["q"] = torch.randn(case["batch"], case["hq"], d, generator=gen, device="cuda", dtype=dt)
    st["table"], st["lens"] = table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    if case["op"] == "weights":
        st["weights"] = torch.rand(total, hkv, ps, generator=gen, device="cuda").transpose(1, 2)
    st["host"] = (lens, table)
    return st


# ------------------------------------------------------------ plain forms


def _plain_encode(rows, kv, scale):
    if kv in _FP8_MAX:
        return (rows.float() / scale).clamp(-_FP8_MAX[kv], _FP8_MAX[kv]).to(_TYPES[kv])
    return rows


def _bytes(x):
    """Codes as bytes: fp8 tensors cannot be indexed."""
    return x.view(torch.uint8) if x.element_size() == 1 else x


def _plain_rows(cache, scale, kv, slots):
    """Rows of the named slots, in 32 bits."""
    ps = cache.shape[1]
    page, at = slots // ps, slots % ps
    if kv == "mx4":
        return _values(cache[page, at], scale[page, at])
    x = _bytes(cache)[page, at].view(cache.dtype)
    return x.float() * (1.0 if scale is None else scale)


def _plain_write(st):
    c, slots = st["case"], st["slots"]
    live = slots >= 0
    at = slots[live]
    out = []
    for rows, cache, scale in ((st["k"], st["k_cache"], st["k_scale"]), (st["v"], st["v_cache"], st["v_scale"])):
        codes, s = _quantise(rows)
        _store(cache, at, codes[live])
        _store(scale, at, s[live])
        back = _plain_rows(cache, scale, "mx4", slots.clamp(min=0))
        out.append(torch.where(live[:, None, None], back, 0.0).to(_TYPES[c["q"]]))
    return out


def _plain_attention(st):
    """(output, attention weights [batch, kv heads, tokens], slots [batch, tokens], which of them are tokens)."""
    c, q, table, lens = st["case"], st["q"], st["table"], st["lens"]
    ps, hkv, hq, d = c["ps"], c["hkv"], c["hq"], c["d"]
    t = torch.arange(min(c["hi"], table.shape[1] * ps), device="cuda")
    slots = table[:, t // ps].long() * ps + t % ps
    live = t < lens[:, None]
    k = _plain_rows(st["k_cache"], st["k_scale"], c["kv"], slots)
    s = q.float().unflatten(1, (hkv, hq // hkv)) @ k.permute(0, 2, 3, 1).contiguous()
    s = (s / math.sqrt(d)).masked_fill(~live[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    w = p / p.sum(-1, keepdim=True)
    del k, s, p
    v = _plain_rows(st["v_cache"], st["v_scale"], c["kv"], slots).transpose(1, 2).contiguous()
    return (w @ v).flatten(1, 2).to(q.dtype), w.sum(2), slots, live


def _plain_weights(st):
    out, w, slots, live = _plain_attention(st)
    acc, ps = st["weights"], st["case"]["ps"]
    at = slots[live]
    acc[at // ps, at % ps] += w.transpose(1, 2)[live]
    return [out, acc]


def _plain_evict(st):
    c = st["case"]
    ps, keep = c["ps"], c["keep"]
    table, lens, acc, pos = st["table"], st["lens"], st["weights"], st["positions"]
    k_cache, v_cache = _bytes(st["k_cache"]), _bytes(st["v_cache"])
    _store(k_cache, st["slots"], _bytes(_plain_encode(st["k"], c["kv"], st["k_scale"])))
    _store(v_cache, st["slots"], _bytes(_plain_encode(st["v"], c["kv"], st["v_scale"])))
    _store(acc, st["slots"], st["token_weights"])
    _store(pos, st["slots"], st["token_positions"][:, None].expand(-1, c["hkv"]))
    new_lens = lens.clamp(max=keep)
    t = torch.arange(table.shape[1] * ps, device="cuda")
    page, at = table[:, t // ps].long()[:, None], (t % ps)[None, None]
    h = torch.arange(c["hkv"], device="cuda")[None, :, None]
    live = (t < lens[:, None])[:, None]
    p = pos[page, at, h].long()
    newest = live & (p > p.masked_fill(~live, -(1 << 40)).amax(-1, keepdim=True) - c["recent"])
    w = acc[page, at, h]
    # Newest first, then the heaviest; a stable sort keeps ties in slot order.
    w = torch.where(newest, math.inf, w).masked_fill(~live, -math.inf)
    order = torch.argsort(w, dim=-1, descending=True, stable=True)
    rank = torch.empty_like(order).scatter_(-1, order, t.expand_as(order))
    n = new_lens[:, None, None]
    kept = (rank < n) & live
    hole, mover = ~kept & (t < n), kept & (t >= n)
    # The i-th kept slot past the end goes to the i-th hole.
    src, dst = mover.nonzero(), hole.nonzero()
    sp, so = table[src[:, 0], src[:, 2] // ps].long(), src[:, 2] % ps
    dp, do = table[dst[:, 0], dst[:, 2] // ps].long(), dst[:, 2] % ps
    hh = src[:, 1]
    for x in (k_cache, v_cache, acc, pos):
        x[dp, do, hh] = x[sp, so, hh]
    return [new_lens, st["k_cache"], st["v_cache"], acc, pos]


def run(st):
    c = st["case"]
    op = c["op"]
    if op == "evict":
        st["token_positions"] += c["new"]  # the next tokens
    if not own:
        if op == "mx4_write":
            return _plain_write(st)
        if op == "mx4_decode":
            return _plain_attention(st)[0]
        return _plain_weights(st) if op == "weights" else _plain_evict(st)
    import paged_attention_decode_amd as pad

    scales = {"k_scale": st["k_scale"], "v_scale": st["v_scale"]}
    if op == "mx4_write":
        pad.paged_kv_append(st["k"], st["v"], st["k_cache"], st["v_cache"], st["slots"], **scales)
        return list(pad.paged_kv_read(st["k_cache"], st["v_cache"], st["slots"], **scales, dtype=_TYPES[c["q"]]))
    if op == "mx4_decode":
        return pad.paged_attention_decode_mx4(st["q"], st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"],
                                              st["table"], st["lens"])
    if op == "weights":
        return [pad.paged_attention_decode_weights(st["q"], st["k_cache"], st["v_cache"], st["weights"], st["table"],
                                                   st["lens"], **scales), st["weights"]]
    pad.paged_kv_append(st["k"], st["v"], st["k_cache"], st["v_cache"], st["slots"], **scales, weights=st["weights"],
                        positions=st["positions"], token_weights=st["token_weights"],
                        token_positions=st["token_positions"])
    lens = pad.paged_kv_evict(st["k_cache"], st["v_cache"], st["weights"], st["positions"], st["table"], st["lens"],
                              c["keep"], c["recent"])
    return [lens, st["k_cache"], st["v_cache"], st["weights"], st["positions"]]


def _row_bytes(case):
    return {"mx4": case["d"] // 2 + case["d"] // 32, "e4m3": case["d"], "e5m2": case["d"]}.get(case["kv"], 2 * case["d"])


def work(case):
    """Every input read once, every output written once; two products of two operations in an attention."""
    hkv, d, row = case["hkv"], case["d"], _row_bytes(case)
    if case["op"] == "mx4_write":
        t = case["tokens"]
        live = t * (1 - case["skip"])
        return {"bytes": 2 * hkv * (live * (2 * d + row) + live * row + t * 2 * d) + 16 * t, "flops": 0}
    if case["op"] == "evict":
        b, n, new = case["batch"], case["keep"], case["new"]
        moved = min(new, case["recent"])  # of the new tokens at least these move below the others
        append = b * new * (hkv * (2 * (2 * d + row) + 8 + 4) + 12)
        return {"bytes": append + b * hkv * (8 * (n + new) + 2 * moved * (2 * row + 8)) + 8 * b, "flops": 0}
    lens = _lengths(case)
    tokens, b = sum(lens), case["batch"]
    index = 4 * sum(_pages(n, case["ps"]) for n in lens) + 4 * b
    total = 2 * tokens * hkv * row + 2 * b * case["hq"] * d * 2 + index
    if case["op"] == "weights":
        total += 8 * tokens * hkv
    return {"bytes": total, "flops": 4 * tokens * case["hq"] * d}


# ------------------------------------------------- the definition, in 64 bits


def _exact_rows(cache, scale, kv, ids, n):
    """The first n rows of pages ids, [heads, n, d], in 64 bits."""
    if kv == "mx4":
        c, s = cache[ids].flatten(0, 1)[:n].long(), scale[ids].flatten(0, 1)[:n].long()
        out = torch.empty(*c.shape[:2], 2 * c.shape[2], dtype=torch.float64, device=c.device)
        for half, nibble in ((0, c % 16), (1, c // 16)):
            e, m = (nibble // 2) % 4, nibble % 2
            mag = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * torch.pow(2.0, (e - 1).double()))
            out[..., half::2] = torch.where(nibble >= 8, -mag, mag)
        out *= torch.pow(2.0, (s - 127).double()).repeat_interleave(32, -1)
    else:
        out = _bytes(cache)[ids].view(cache.dtype).flatten(0, 1)[:n]
        out = out.double() * (1.0 if scale is None else scale)
    return out.transpose(0, 1).contiguous()


def exact(case, seed):
    """Outputs of run() for these inputs from the definitions, sequence by sequence."""
    st = prepare(case, seed)
    ps, hkv, d = case["ps"], case["hkv"], case["d"]
    if case["op"] == "mx4_write":
        got = []
        grid = torch.tensor(_E2M1[:8], dtype=torch.float64, device="cuda")
        for x in (st["k"].double(), st["v"].double()):
            block = x.reshape(-1, 32)
            unit = torch.pow(2.0, torch.floor(torch.log2(block.abs().amax(1, keepdim=True).clamp(min=2.0**-120))) - 2)
            y = torch.empty_like(block)
            for part, o, u in zip(block.split(1 << 20), y.split(1 << 20), unit.split(1 << 20)):
                far = (part.abs() / u).unsqueeze(-1) - grid
                # The nearest value; of two as near, the one with the even code.
                cost = far.abs() + torch.arange(8, device="cuda") % 2 * 1e-9
                o.copy_(torch.sign(part) * grid[cost.argmin(-1)] * u)
            y = y.reshape(x.shape)
            y[st["slots"] < 0] = 0.0
            got.append(y)
        return got
    if case["op"] == "evict":
        return None  # nothing is computed: rows move
    lens, table = st["host"]
    hq, w_all = case["hq"], None
    out = torch.zeros(case["batch"], hq, d, dtype=torch.float64, device="cuda")
    if case["op"] == "weights":
        w_all = st["weights"].double()
    for b, n in enumerate(lens):
        ids = table[b, :_pages(n, ps)].cuda().long()
        k = _exact_rows(st["k_cache"], st["k_scale"], case["kv"], ids, n)
        v = _exact_rows(st["v_cache"], st["v_scale"], case["kv"], ids, n)
        q = st["q"][b].double().view(hkv, hq // hkv, d)
        p = torch.softmax((q @ k.transpose(1, 2).contiguous()) / math.sqrt(d), dim=-1)
        out[b] = (p @ v).view(hq, d)
        if w_all is not None:
            t = torch.arange(n, device="cuda")
            w_all[ids[t // ps], t % ps] += p.sum(1).transpose(0, 1)
    return out if w_all is None else [out, w_all]
