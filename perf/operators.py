"""Timing cases of the attention operators around the quantized cache, with their plain forms.

Three operators, as a decoder layer calls them around its projections:

  rope    RMS norm of every query and key head, multiplier 1 + w, and the position rotation of the
          first `rot` features of each head (angle = position x frequency);
  cache   keys and values quantized per group of 64 features to 4 or 8 bits (the rule of
          quantize_weight) as they are written to a paged cache, and read back;
  attend  causal attention of each sequence's newest tokens over its paged quantized cache.

`own = False` runs them as elementary torch operations in 32 bits, `own = True` as the calls of
marlin_q4.  Both read and write the same cache bytes; the layout is spelled out at `_unit_maps`.
"""
import math
import os
import random
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.getcwd(), "marlin-mlx_b200"))

own = False

GROUP = 64
EPS = 1e-6
UNIT = 16  # cache rows stored together


def listed():
    return [
        # the newest token of one conversation: what a decode step waits for in every layer
        dict(name="rope_one_token", op="rope", tokens=1, heads=8, kv_heads=2, dim=256, rot=64, pairs="half", axes=1, kind="bf16", far=900),
        # a batch of decode steps at far positions, adjacent pairs, all of the head rotated
        dict(name="rope_batch", op="rope", tokens=61, heads=32, kv_heads=8, dim=128, rot=128, pairs="adjacent", axes=1, kind="bf16", far=900000),
        # a prompt with image patches: three position axes, 32-bit projections (after a 32-bit norm)
        dict(name="rope_prompt", op="rope", tokens=2048, heads=8, kv_heads=2, dim=256, rot=64, pairs="half", axes=3, kind="f32", far=4096),
        # one new token for each of 32 running sequences
        dict(name="cache_step", op="cache", tokens=32, kv_heads=8, dim=128, bits=4, page=16, step=True, kind="bf16"),
        # a whole prompt's keys and values
        dict(name="cache_prompt", op="cache", tokens=4096, kv_heads=2, dim=256, bits=8, page=64, step=False, kind="f32"),
        # the first words of a conversation
        dict(name="step_short", op="attend", batch=1, new=1, longest=19, heads=4, kv_heads=2, dim=64, bits=4, page=16, ragged=False),
        # one long conversation, one token at a time
        dict(name="step_long", op="attend", batch=1, new=1, longest=131072, heads=8, kv_heads=2, dim=256, bits=4, page=64, ragged=False),
        # a server's batch of conversations of different lengths
        dict(name="step_batch", op="attend", batch=32, new=1, longest=6000, heads=32, kv_heads=8, dim=128, bits=8, page=16, ragged=True),
        # a few drafted tokens at once, checked against the cache
        dict(name="few_tokens", op="attend", batch=6, new=4, longest=2500, heads=8, kv_heads=2, dim=128, bits=4, page=32, ragged=True),
        # a prompt from its start
        dict(name="prompt", op="attend", batch=1, new=2048, longest=2048, heads=8, kv_heads=2, dim=256, bits=4, page=64, ragged=False),
        # chunks of several prompts packed together
        dict(name="chunks_packed", op="attend", batch=5, new=700, longest=5000, heads=16, kv_heads=2, dim=64, bits=8, page=16, ragged=True),
        # a chunk of a long document behind what is cached already
        dict(name="chunk_long", op="attend", batch=1, new=512, longest=16384, heads=32, kv_heads=8, dim=128, bits=4, page=128, ragged=False),
    ]


def _spread(rng, low, high):
    """A whole number between the two, its logarithm spread evenly."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    dim = rng.choice([64, 128, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 6, 8])
    bits, page = rng.choice([4, 8]), 16 * rng.choice([1, 2, 3, 4, 8])
    op = rng.choice(["rope", "cache", "attend", "attend"])
    if op == "rope":
        return dict(op=op, tokens=_spread(rng, 1, 2500), heads=kv_heads * group, kv_heads=kv_heads, dim=dim, rot=16 * rng.randint(1, dim // 16),
                    pairs=rng.choice(["half", "adjacent"]), axes=rng.choice([1, 1, 2, 3]), kind=rng.choice(["bf16", "f32"]), far=_spread(rng, 10, 1000000))
    if op == "cache":
        step = rng.random() < 0.5
        return dict(op=op, tokens=_spread(rng, 1, 200 if step else 5000), kv_heads=kv_heads, dim=dim, bits=bits, page=page, step=step, kind=rng.choice(["bf16", "f32"]))
    new = rng.choice([1, 1, rng.randint(2, 8), _spread(rng, 9, 2048)])
    batch = _spread(rng, 1, 32)
    longest = new + _spread(rng, 1, 131072)
    # no more than the largest listed case: its scores, and its cache read into 32 bits
    while batch * new * longest * kv_heads * group > 512 * 16384 * 32 or batch * longest * kv_heads * dim > 32 * 6000 * 8 * 128:
        if batch > 1:
            batch -= 1
        else:
            longest = new + (longest - new) // 2
            new = max(1, new * 3 // 4)
    return dict(op=op, batch=batch, new=new, longest=longest, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, bits=bits, page=page, ragged=rng.random() < 0.7)


# ---- the cache's bytes -----------------------------------------------------------------------------


def _row_bytes(dim, bits):
    return dim * bits // 8


def _unit_bytes(dim, bits):
    return UNIT * 2 * (_row_bytes(dim, bits) + 4 * (dim // GROUP))


def _unit_maps(dim, bits, device):
    """Where the bytes of 16 rows of one head are in their unit: codes of the keys [16, row bytes],
    scale and bias of the keys [16, 4 x groups], and the same of the values.

    A unit is [key codes | key scales and biases | value codes | value scales and biases].  Scales
    and biases are bf16 pairs, row by row.  Key codes are column panels of up to 64 bytes, each with
    its 16 rows one after the other; value codes are 16-byte pieces, piece c of row r at
    (c / 2) 32 + (r % 2 + 2 (r / 8)) 8 + (c % 2) 4 + (r / 2) % 4."""
    rb, sb = _row_bytes(dim, bits), 4 * (dim // GROUP)
    r = torch.arange(UNIT, device=device)[:, None]
    j = torch.arange(rb, device=device)[None, :]
    panel = min(64, rb)
    keys = (j // panel) * (panel * UNIT) + r * panel + j % panel
    c = j // 16
    piece = (c // 2) * 32 + (r % 2 + 2 * (r // 8)) * 8 + (c % 2) * 4 + (r // 2) % 4
    values = piece * 16 + j % 16
    scales = r * sb + torch.arange(sb, device=device)[None, :]
    at_values = UNIT * (rb + sb)
    return keys, UNIT * rb + scales, at_values + values, at_values + UNIT * rb + scales


def _round_away(x):
    x = x.double()
    return (torch.sign(x) * torch.floor(x.abs() + 0.5)).float()


def _quantized(x, bits):
    """Codes [..., dim] as bytes' values and (scale, bias) [..., dim / 64, 2] as bf16, of x [..., dim]."""
    x = x.to(torch.bfloat16).float().unflatten(-1, (-1, GROUP))
    top = float(2**bits - 1)
    high, low = x.amax(-1, keepdim=True).clamp(min=0.0), x.amin(-1, keepdim=True)
    # by a tensor: a division by a plain number is a product with its rounded reciprocal on the device
    scale = ((high - low) / torch.full_like(high, top)).clamp(min=1e-7)
    side = low.abs() > high.abs()
    scale = torch.where(side, scale, -scale)
    edge = torch.where(side, low, high)
    steps = _round_away(edge / scale)
    some = steps != 0
    scale = torch.where(some, edge / torch.where(some, steps, torch.ones_like(steps)), scale)
    bias = torch.where(some, edge, torch.zeros_like(edge))
    codes = _round_away((x - bias) / scale).clamp(0.0, top).flatten(-2).to(torch.uint8)
    return codes, torch.cat([scale, bias], -1).to(torch.bfloat16)


def _packed(codes, bits):
    return codes if bits == 8 else codes[..., 0::2] | (codes[..., 1::2] << 4)


def _values(codes, pairs, bits):
    """scale x code + bias in 32 bits: codes [..., row bytes] and pairs [..., 4 x groups] as bytes."""
    if bits == 4:
        codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    pairs = pairs.contiguous().view(torch.bfloat16).float().unflatten(-1, (-1, 2))
    x = codes.float().unflatten(-1, (-1, GROUP))
    return (x * pairs[..., 0:1] + pairs[..., 1:2]).flatten(-2)


def _write(pool, k, v, slots, dim, bits):
    maps = _unit_maps(dim, bits, pool.device)
    heads, units, size = pool.shape[1], pool.shape[2], pool.shape[3]
    unit, row = slots.long() // UNIT, slots.long() % UNIT
    base = ((unit // units)[:, None] * heads + torch.arange(heads, device=pool.device)) * units + (unit % units)[:, None]
    for x, at, at_pairs in ((k, maps[0], maps[1]), (v, maps[2], maps[3])):
        codes, pairs = _quantized(x, bits)
        pool.view(-1)[base[..., None] * size + at[row][:, None]] = _packed(codes, bits)
        pool.view(-1)[base[..., None] * size + at_pairs[row][:, None]] = pairs.flatten(-2).view(torch.uint8)


def _read(pool, slots, dim, bits):
    maps = _unit_maps(dim, bits, pool.device)
    heads, units, size = pool.shape[1], pool.shape[2], pool.shape[3]
    unit, row = slots.long() // UNIT, slots.long() % UNIT
    base = ((unit // units)[:, None] * heads + torch.arange(heads, device=pool.device)) * units + (unit % units)[:, None]
    got = []
    for at, at_pairs in ((maps[0], maps[1]), (maps[2], maps[3])):
        codes = pool.view(-1)[base[..., None] * size + at[row][:, None]]
        pairs = pool.view(-1)[base[..., None] * size + at_pairs[row][:, None]]
        got.append(_values(codes, pairs, bits).to(torch.bfloat16))
    return got


# ---- inputs ----------------------------------------------------------------------------------------


def _lengths(case):
    """(new tokens, cached tokens with the new ones) of every sequence of an attend case."""
    rng = random.Random(case["batch"] * 1000003 + case["longest"] * 101 + case["new"])
    new, total = [], []
    for i in range(case["batch"]):
        n, m = case["new"], case["longest"]
        if case["ragged"] and i:
            n = rng.randint(1, n) if n > 1 else 1
            m = n + _spread(rng, 1, m - n + 1) - 1 if m > n else n
        new.append(n)
        total.append(max(n, m))
    return new, total


def _normal(shape, g, size=1.0):
    return torch.randn(shape, generator=g, device="cuda") * size


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s = dict(case)
    dim, kvh = case["dim"], case["kv_heads"]
    if case["op"] == "rope":
        heads, t, kind = case["heads"], case["tokens"], torch.bfloat16 if case["kind"] == "bf16" else torch.float32
        # one projection holds queries, keys and values: the operator sees strided heads
        fused = _normal((t, heads + 2 * kvh, dim), g, 1.5).to(kind)
        s["q"], s["k"] = fused[:, :heads], fused[:, heads:heads + kvh]
        s["q_weight"] = (0.1 + _normal((dim,), g, 0.05)).to(torch.bfloat16)
        s["k_weight"] = (0.1 + _normal((dim,), g, 0.05)).to(torch.bfloat16)
        start = torch.randint(0, case["far"], (case["axes"], 1), generator=g, device="cuda")
        s["positions"] = (start + torch.arange(t, device="cuda") // torch.tensor([[1], [7], [5]], device="cuda")[:case["axes"]]).int()
        i = torch.arange(case["rot"] // 2, device="cuda", dtype=torch.float64)
        s["freqs"] = (1e6 ** (-2.0 * i / case["rot"])).float()
        s["axis_of"] = [f % case["axes"] for f in range(case["rot"] // 2)]
        return s
    if case["op"] == "cache":
        t, page = case["tokens"], case["page"]
        pages = (t + 3 if case["step"] else (t + page - 1) // page + 2)
        kind = torch.bfloat16 if case["kind"] == "bf16" else torch.float32
        fused = _normal((t, 2 * kvh, dim), g).to(kind)
        s["k"], s["v"] = fused[:, :kvh], fused[:, kvh:]
        order = torch.randperm(pages, generator=g, device="cuda")
        i = torch.arange(t, device="cuda")
        if case["step"]:  # one token in a page of each sequence
            slots = order[:t] * page + torch.randint(0, page, (t,), generator=g, device="cuda")
        else:
            slots = order[i // page] * page + i % page
        s["slots"] = slots.int()
        s["pool"] = torch.zeros((pages, kvh, page // UNIT, _unit_bytes(dim, case["bits"])), dtype=torch.uint8, device="cuda")
        return s
    new, total = _lengths(case)
    page, heads = case["page"], case["heads"]
    most = max((m + page - 1) // page for m in total)
    pages = sum((m + page - 1) // page for m in total) + 1
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.full((case["batch"], most), -1, dtype=torch.int32, device="cuda")
    pool = torch.empty((pages, kvh, page // UNIT, _unit_bytes(dim, case["bits"])), dtype=torch.uint8, device="cuda")
    used = 0
    for b, m in enumerate(total):
        n = (m + page - 1) // page
        table[b, :n] = order[used:used + n]
        used += n
    step = max(1, (1 << 25) // (page * kvh * dim))
    for p in range(0, pages, step):  # what stands behind the last token of a page is an older sequence's
        slots = torch.arange(p * page, min(pages, p + step) * page, device="cuda")
        _write(pool, _normal((len(slots), kvh, dim), g), _normal((len(slots), kvh, dim), g), slots, dim, case["bits"])
    s["pool"], s["table"] = pool, table
    s["q"] = _normal((sum(new), heads, dim), g, 1.5).to(torch.bfloat16)
    s["lengths"] = torch.tensor(total, dtype=torch.int32, device="cuda")
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    s["most_new"] = max(new)
    s["scale"] = dim ** -0.5
    return s


# ---- the operators ---------------------------------------------------------------------------------


def _rope_plain(s):
    axis = torch.tensor(s["axis_of"], device="cuda")
    # 64 bits for the angle: a position near 10^6 leaves 32 bits no digits behind the point
    angle = s["positions"].double()[axis].T * s["freqs"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    half = s["rot"] // 2
    out = []
    for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
        x = x.float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * (1.0 + w.float())
        turn, rest = x[..., :s["rot"]], x[..., s["rot"]:]
        if s["pairs"] == "half":
            a, b = turn[..., :half], turn[..., half:]
            turn = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        else:
            a, b = turn[..., 0::2], turn[..., 1::2]
            turn = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        out.append(torch.cat([turn, rest], -1).to(torch.bfloat16))
    return out


def _attend_plain(s):
    dim, bits, kvh, heads = s["dim"], s["bits"], s["kv_heads"], s["heads"]
    maps = _unit_maps(dim, bits, "cuda")
    got = s["pool"][s["table"].long().clamp(min=0)].transpose(1, 2)  # [batch, head, pages, units, bytes]
    keys = _values(got[..., maps[0]], got[..., maps[1]], bits).flatten(2, 4)
    values = _values(got[..., maps[2]], got[..., maps[3]], bits).flatten(2, 4)
    del got
    starts, lengths, most = s["starts"].long(), s["lengths"].long(), s["most_new"]
    new = starts[1:] - starts[:-1]
    i = torch.arange(most, device="cuda")
    take = (starts[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][take].float().unflatten(2, (kvh, heads // kvh)).permute(0, 2, 3, 1, 4)  # [batch, kv head, group, new, dim]
    at = torch.arange(keys.shape[2], device="cuda")
    seen = at <= (lengths - new)[:, None, None] + i[:, None]
    seen = (seen & (at < lengths[:, None, None]))[:, None, None]
    keys = torch.where((at < lengths[:, None])[:, None, :, None], keys, 0.0)
    values = torch.where((at < lengths[:, None])[:, None, :, None], values, 0.0)
    p = torch.matmul(q.flatten(2, 3), keys.transpose(-1, -2)).unflatten(2, q.shape[2:4]) * s["scale"]
    p = torch.where(seen, p, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = torch.exp(p - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.flatten(2, 3), values).unflatten(2, q.shape[2:4])
    out = torch.where(total > 0, out / total, 0.0).permute(0, 3, 1, 2, 4).flatten(2, 3).to(torch.bfloat16)
    return out[i < new[:, None]]


def run(state):
    s = state
    if own:
        import marlin_q4 as mq
        if s["op"] == "rope":
            rotary = mq.Rotary(s["freqs"], interleaved=s["pairs"] == "adjacent", axes=s["axis_of"] if s["axes"] > 1 else None)
            return mq.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["positions"], rotary, eps=EPS)
        cache = mq.KVCache(s["pool"], s["dim"], s["bits"])
        if s["op"] == "cache":
            mq.kv_write(cache, s["k"], s["v"], s["slots"])
            return mq.kv_read(cache, s["slots"])
        return mq.paged_attention(s["q"], cache, s["table"], s["lengths"], s["starts"], s["most_new"], scale=s["scale"])
    if s["op"] == "rope":
        return _rope_plain(s)
    if s["op"] == "cache":
        _write(s["pool"], s["k"], s["v"], s["slots"], s["dim"], s["bits"])
        return _read(s["pool"], s["slots"], s["dim"], s["bits"])
    return _attend_plain(s)


def work(case):
    dim, kvh = case["dim"], case["kv_heads"]
    if case["op"] == "rope":
        n = case["tokens"] * (case["heads"] + kvh) * dim
        size = 2 if case["kind"] == "bf16" else 4
        return {"bytes": n * (size + 2) + 4 * dim + case["tokens"] * case["axes"] * 4 + 2 * case["rot"], "flops": 10 * n}
    row = 2 * kvh * (_row_bytes(dim, case["bits"]) + 4 * (dim // GROUP))  # a token's keys and values in the cache
    if case["op"] == "cache":
        n = case["tokens"] * 2 * kvh * dim
        size = 2 if case["kind"] == "bf16" else 4
        return {"bytes": n * (size + 2) + 2 * case["tokens"] * row + 4 * case["tokens"], "flops": 12 * n}
    new, total = _lengths(case)
    seen = sum(n * m - n * (n - 1) // 2 for n, m in zip(new, total))
    return {"bytes": sum(total) * row + 2 * 2 * sum(new) * case["heads"] * dim + 4 * sum((m + case["page"] - 1) // case["page"] for m in total),
            "flops": 4 * seen * case["heads"] * dim}


# ---- the definitions in 64 bits --------------------------------------------------------------------


def _exact_rope(s):
    got = []
    pos = s["positions"].double().cpu().numpy()
    freq = s["freqs"].double().cpu().numpy()
    rot, half = s["rot"], s["rot"] // 2
    turn = np.stack([np.exp(1j * pos[s["axis_of"][f]] * freq[f]) for f in range(half)], 1)[:, None, :]
    first = np.arange(half) if s["pairs"] == "half" else 2 * np.arange(half)
    second = first + (half if s["pairs"] == "half" else 1)
    for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
        x = x.double().cpu().numpy()
        x = x / np.sqrt((x**2).sum(-1, keepdims=True) / s["dim"] + EPS) * (1 + w.double().cpu().numpy())
        z = (x[..., first] + 1j * x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
        got.append(torch.from_numpy(x))
    return got


def _exact_cache(s):
    # The rule's quotients are binary32 values (quantize_weight's definition): a code next to a border
    # goes by that rounding, so it is part of the definition; the values are 64-bit from there on.
    got, top = [], 2 ** s["bits"] - 1

    def quotient(a, b):
        return (a / b).astype(np.float32).astype(np.float64)

    for x in (s["k"], s["v"]):
        x = x.to(torch.bfloat16).double().cpu().numpy()
        y = np.empty_like(x)
        for a in range(0, s["dim"], GROUP):
            w = x[..., a:a + GROUP]
            high, low = np.maximum(w.max(-1), 0), w.min(-1)
            step = np.maximum(quotient((high - low).astype(np.float32).astype(np.float64), top), float(np.float32(1e-7)))
            below = np.abs(low) > np.abs(high)
            edge, step = np.where(below, low, high), np.where(below, step, -step)
            count = np.trunc(quotient(edge, step) + 0.5 * np.sign(edge * step))
            bias = np.where(count != 0, edge, 0.0)
            step = np.where(count != 0, quotient(edge, np.where(count != 0, count, 1)), step)
            z = quotient((w - bias[..., None]).astype(np.float32).astype(np.float64), step[..., None])
            code = np.clip(np.trunc(z + 0.5 * np.sign(z)), 0, top)
            kept = [torch.from_numpy(v).to(torch.bfloat16).double().numpy() for v in (step, bias)]
            y[..., a:a + GROUP] = code * kept[0][..., None] + kept[1][..., None]
        got.append(torch.from_numpy(y))
    return got


def _exact_head(unit, head, dim, bits):
    """Keys and values [rows, dim] in 64 bits of the units [n, heads, bytes] of one head, from the layout's words."""
    rb, groups = dim * bits // 8, dim // GROUP
    raw = unit[:, head]
    got = []
    for which in range(2):
        part = raw[:, which * 16 * (rb + 4 * groups):]
        if which == 0:
            wide = min(64, rb)
            codes = part[:, :16 * rb].reshape(-1, rb // wide, 16, wide).transpose(0, 2, 1, 3).reshape(-1, 16, rb)
        else:  # [pair of pieces, r / 8, r % 2, piece of the pair, (r / 2) % 4, byte]
            codes = part[:, :16 * rb].reshape(-1, rb // 32, 2, 2, 2, 4, 16).transpose(0, 2, 5, 3, 1, 4, 6).reshape(-1, 16, rb)
        pair = np.ascontiguousarray(part[:, 16 * rb:16 * (rb + 4 * groups)]).view(np.uint16).reshape(-1, 16, groups, 2)
        pair = (pair.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
        if bits == 4:
            codes = np.stack([codes % 16, codes // 16], -1).reshape(-1, 16, dim)
        x = codes.reshape(-1, 16, groups, GROUP) * pair[..., :1] + pair[..., 1:]
        got.append(x.reshape(-1, dim))
    return got


def _exact_attend(s):
    new, total = _lengths(s)
    if sum(n * m for n, m in zip(new, total)) * s["heads"] * s["dim"] > 1.5e11 or sum(total) * s["kv_heads"] * s["dim"] > 2.5e8:
        return None
    out, start, group = [], 0, s["heads"] // s["kv_heads"]
    for b, (n, m) in enumerate(zip(new, total)):
        pages = s["table"][b, :(m + s["page"] - 1) // s["page"]].long()
        unit = s["pool"][pages].transpose(1, 2).flatten(0, 1).cpu().numpy()
        q = s["q"][start:start + n].double()
        start += n
        of = []
        for head in range(s["kv_heads"]):
            k, v = (torch.from_numpy(x[:m]).cuda() for x in _exact_head(unit, head, s["dim"], s["bits"]))
            for h in range(head * group, (head + 1) * group):
                p = q[:, h] @ k.T * s["scale"]
                last = torch.arange(m - n, m, device="cuda")[:, None]
                p = torch.softmax(p.masked_fill(torch.arange(m, device="cuda") > last, -math.inf), -1)
                of.append(p @ v)
        out.append(torch.stack(of, 1))
    return torch.cat(out)


def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "cache": _exact_cache, "attend": _exact_attend}[case["op"]](s)
