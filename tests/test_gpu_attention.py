"""GPU tests of the attention operators around the quantized cache against 64-bit restatements.

Tolerances, from the roundings (bf16: half a step is 2^-8 of the value, binary32: 2^-24):
  norm_rope   bf16 output: 2^-8 |y| for the one rounding, and binary32 arithmetic of a few dozen
              operations (2^-18 of the row's largest value, which also bounds a turned pair);
  attention   f16 operands (half a step is 2^-11 of the value), binary32 sums, a bf16 output.  Keys and
              values are codes (exact) or rounded to f16 once, queries are exact in f16: a score moves by at
              most e = 2^-10 spread (spread = scale sum |q| |k|; twice the rounding, for the binary32 sum of
              1024-offset codes), so a weight by a factor within exp(2 e).  Weights, weights times scales
              and values are each rounded once: with mix = sum p |v|
                |error| <= (exp(2 e) (1 + 2^-10)^2 - 1) mix + 2^-12 mix (binary32) + 2^-8 |out|
                           + 2^-11 sum p |s (code - mid)|   (p s rounded, the offset part b + mid s not).
              There mid = 8 or 128 and |s| = |edge| / n with edge the group's largest value (its bias, code
              0) and n >= top / 2 rounded, so mid |s| <= 8 / 7.5 |edge| (1 + 2^-8) < 1.1 max |v| of the group.
              The roundings are independent, so the 2-norm of the error stays near the output's own (2^-9.2,
              0.17 %): asserted below 0.3 %.
"""
import math

import numpy as np
import pytest
import torch

import attn_ref as ref
import marlin_q4 as mq

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0**-8


@pytest.fixture(autouse=True)
def no_device_error():
    mq.device_error()
    yield
    torch.cuda.synchronize()
    assert mq.device_error() == 0


def rand(shape, seed, dtype=torch.bfloat16, size=1.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (torch.randn(shape, generator=g) * size).to(dtype).to(DEV)


def f64(t):
    return t.double().cpu().numpy()


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def decode_unit(unit, dim, bits):
    """Codes and (scale, bias) of the 16 rows of one unit, from the documented layout: keys, then values."""
    rb, groups = dim * bits // 8, dim // 64
    got = []
    for which in range(2):
        part = unit[which * 16 * (rb + 4 * groups):]
        codes = np.zeros((16, rb), np.uint8)
        for r in range(16):
            for j in range(rb):
                if which == 0:
                    p = min(64, rb)
                    at = (j // p) * p * 16 + r * p + j % p
                else:
                    c = j // 16
                    at = ((c // 2) * 32 + (r % 2 + 2 * (r // 8)) * 8 + (c % 2) * 4 + (r // 2) % 4) * 16 + j % 16
                codes[r, j] = part[at]
        if bits == 4:
            codes = np.stack([codes & 15, codes >> 4], -1).reshape(16, dim)
        pair = part[16 * rb:16 * (rb + 4 * groups)].copy().view(np.uint16).reshape(16, groups, 2)
        pair = (pair.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
        got.append((codes.astype(np.int64), pair[..., 0], pair[..., 1]))
    return got


# ---- head norms and rotation -----------------------------------------------------------------------


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype,out", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16),
                                       (torch.bfloat16, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,kv_heads,rot", [(1, 8, 2, 64), (3, 1, 1, 16), (37, 5, 3, 48), (400, 12, 4, 64)])
def test_norm_rope(dim, dtype, out, interleaved, tokens, heads, kv_heads, rot):
    fused = rand((tokens, heads + 2 * kv_heads, dim), tokens + dim, dtype, 1.7)
    q, k = fused[:, :heads], fused[:, heads:heads + kv_heads]
    qw, kw = rand((dim,), 5, size=0.2), rand((dim,), 6, size=0.2)
    pos = torch.arange(tokens, dtype=torch.int32, device=DEV) * 2731 + 3  # to about 10^6
    freqs = (1e4 ** (-torch.arange(rot // 2, dtype=torch.float64) * 2 / rot)).float().to(DEV)
    got = mq.qk_norm_rope(q, k, qw, kw, pos, mq.Rotary(freqs, interleaved), out_dtype=out)
    for x, w, y in ((q, qw, got[0]), (k, kw, got[1])):
        assert y.dtype == out and y.is_contiguous()
        want = ref.norm_rope(f64(x), f64(w), pos[None].cpu().numpy(), freqs.cpu().numpy(), 1e-6, interleaved)
        top = np.abs(want).max(-1, keepdims=True)
        bound = 2.0**-18 * top + (U * np.abs(want) if out == torch.bfloat16 else 0)
        assert (np.abs(f64(y) - want) <= bound).all()


def test_norm_rope_axes_far_positions_full_head():
    tokens, heads, dim, rot = 19, 6, 128, 128
    q, k = rand((tokens, heads, dim), 1, torch.float32), rand((tokens, 2, dim), 2, torch.float32)
    w = rand((dim,), 3, size=0.1)
    pos = torch.stack([torch.arange(tokens) + 2**30, torch.arange(tokens) // 4 - 7, 999983 - torch.arange(tokens)]).int().to(DEV)
    freqs = (1e6 ** (-torch.arange(rot // 2, dtype=torch.float64) * 2 / rot)).float().to(DEV)
    axes = [(7 * i) % 3 for i in range(rot // 2)]
    got = mq.qk_norm_rope(q, k, w, w, pos, mq.Rotary(freqs, axes=axes), eps=1e-5, out_dtype=torch.float32)
    for x, y in ((q, got[0]), (k, got[1])):
        want = ref.norm_rope(f64(x), f64(w), pos.cpu().numpy(), freqs.cpu().numpy(), 1e-5, False, axes)
        assert (np.abs(f64(y) - want) <= 2.0**-18 * np.abs(want).max(-1, keepdims=True)).all()


def test_norm_rope_zero_row_and_many_heads():
    q, k = torch.zeros((2, 130, 64), device=DEV), rand((2, 7, 64), 4, torch.float32)
    q[1] = rand((130, 64), 9, torch.float32)
    w, freqs = rand((64,), 3, size=0.1), torch.ones(8, device=DEV)
    qo, ko = mq.qk_norm_rope(q, k, w, w, ints([0, 5]), mq.Rotary(freqs), out_dtype=torch.float32)
    assert not qo[0].any()
    for x, y in ((q, qo), (k, ko)):
        want = ref.norm_rope(f64(x), f64(w), np.array([[0, 5]]), np.ones(8), 1e-6, False)
        assert (np.abs(f64(y) - want) <= 2.0**-18 * np.abs(want).max(-1, keepdims=True)).all()


# ---- cache write and read --------------------------------------------------------------------------


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,kv_heads,page", [(1, 1, 16), (45, 3, 48), (33, 8, 16)])
def test_write_and_read(dim, bits, dtype, tokens, kv_heads, page):
    pages = 4 + tokens // page
    cache = mq.KVCache.empty(pages, page, kv_heads, dim, bits)
    cache.data.random_(0, 256, generator=torch.Generator(device=DEV).manual_seed(3))
    before = cache.data.clone()
    fused = rand((tokens, 2 * kv_heads + 1, dim), dim + bits, dtype, 2.0)
    if dtype == torch.float32:
        fused = fused * 1.001953  # digits that the rounding to bf16 drops
    fused[0, 0, :64] = 0.0        # a group of zeros
    fused[-1, -1, 64 * (dim // 64 - 1):] = -3.25  # one of equal values
    k, v = fused[:, :kv_heads], fused[:, kv_heads + 1:]
    order = np.random.RandomState(7).permutation(pages * page)[:tokens].astype(np.int32)
    slots = order.copy()
    if tokens > 3:
        slots[2] = -1
    mq.kv_write(cache, k, v, ints(slots))
    got = mq.kv_read(cache, ints(slots))
    flat, unit = cache.data.cpu().numpy(), 0
    same = before.cpu().numpy().copy()
    want = [ref.quantize(f64(x), bits) for x in (k, v)]
    for i, s in enumerate(slots):
        if s < 0:
            assert not got[0][i].any() and not got[1][i].any()
            continue
        for h in range(kv_heads):
            unit = flat[s // page, h, s % page // 16]
            for which, (codes, scale, bias) in enumerate(decode_unit(unit, dim, bits)):
                wc, ws, wb = (x[i, h] for x in want[which])
                assert np.array_equal(codes[s % 16], wc)
                assert np.array_equal(scale[s % 16], ws) and np.array_equal(bias[s % 16], wb)
                assert np.array_equal(f64(got[which][i, h]), ref.bf16(ref.dequantize(wc, ws, wb)))
    # nothing else moved: writing the old rows' decode back is the only difference
    touched = {(int(s) // page, int(s) % page // 16) for s in slots if s >= 0}
    for p in range(pages):
        for u in range(page // 16):
            rows = [int(s) % 16 for s in slots if s >= 0 and int(s) // page == p and int(s) % page // 16 == u]
            for h in range(kv_heads):
                if (p, u) not in touched:
                    assert np.array_equal(flat[p, h, u], same[p, h, u])
                elif tokens < 40:
                    for (a, sa, ba), (b, sb, bb) in zip(decode_unit(flat[p, h, u], dim, bits), decode_unit(same[p, h, u], dim, bits)):
                        keep = [r for r in range(16) if r not in rows]
                        assert np.array_equal(a[keep], b[keep]) and np.array_equal(sa[keep], sb[keep], equal_nan=True)
                        assert np.array_equal(ba[keep], bb[keep], equal_nan=True)


def test_four_bit_rows_are_quantize_weight():
    """A cached row holds exactly what quantize_weight makes of it."""
    x = rand((29, 2, 128), 12)
    cache = mq.KVCache.empty(3, 16, 2, 128, 4)
    slots = torch.arange(29, dtype=torch.int32, device=DEV) + 7
    mq.kv_write(cache, x, x, slots)
    q = mq.quantize_weight(x.reshape(58, 128))
    w = q.weight.cpu().numpy().view(np.uint32)
    codes = (w[..., None] >> (4 * np.arange(8)) & 15).reshape(58, 128)
    want = ref.bf16(ref.dequantize(codes, f64(q.scales), f64(q.biases))).reshape(29, 2, 128)
    for y in mq.kv_read(cache, slots):
        assert np.array_equal(f64(y), want)


def test_many_groups_are_quantize_weight():
    """A million groups over all binary orders of magnitude, ties and equal values among them: the cache's own
    division gives the codes of quantize_weight (which divides by __fdiv_rn) every time."""
    g = torch.Generator(device=DEV).manual_seed(5)
    n = 1 << 18
    x = torch.randn((n, 4, 64), generator=g, device=DEV)
    x = x * torch.exp2(torch.randint(-40, 40, (n, 4, 1), generator=g, device=DEV).float())
    x[::7] = torch.randint(-20, 20, x[::7].shape, generator=g, device=DEV).float()  # quotients that tie
    x[::31] = x[::31].abs()
    x[::37] *= 2.0**-100
    x[::41] *= 2.0**80
    x = x.bfloat16().reshape(n, 1, 256)
    cache = mq.KVCache.empty(n // 1024, 1024, 1, 256, 4)
    slots = torch.arange(n, dtype=torch.int32, device=DEV)
    mq.kv_write(cache, x, x, slots)
    q = mq.quantize_weight(x.reshape(n, 256))
    codes = (q.weight[..., None] >> (4 * torch.arange(8, device=DEV)) & 15).reshape(n, 4, 64)
    want = (codes.double() * q.scales.double()[..., None] + q.biases.double()[..., None]).reshape(n, 1, 256)
    for y in mq.kv_read(cache, slots):
        assert torch.equal(y, want.bfloat16())  # double products and sums are exact, one rounding
    # 8 bits: the codes differ from the exact quotient's only where it ties
    cache = mq.KVCache.empty(n // 1024, 1024, 1, 256, 8)
    mq.kv_write(cache, x, x, slots)
    sample = torch.randint(0, n, (4096,), generator=g, device=DEV)
    k, _ = mq.kv_read(cache, sample.int())
    c, s, b = ref.quantize(f64(x[sample]), 8)
    assert np.array_equal(f64(k), ref.bf16(ref.dequantize(c, s, b)))


def test_slots_outside_the_pool_are_refused_on_the_device():
    cache = mq.KVCache.empty(2, 16, 1, 64, 8)
    x = rand((4, 1, 64), 1)
    mq.kv_write(cache, x, x, ints([32, 5, 2**31 - 1, -(2**31)]))
    torch.cuda.synchronize()
    assert mq.device_error() == 3
    k, _ = mq.kv_read(cache, ints([5, 32]))
    torch.cuda.synchronize()
    assert mq.device_error() == 3
    assert not k[1].any() and k[0].any()


def test_write_to_rows_past_32_bits():
    """The last page of a pool of more than 4 GB."""
    page, kvh, dim = 1024, 4, 256
    unit = 16 * 2 * (256 + 16)
    pages = (1 << 32) // (kvh * (page // 16) * unit) + 2
    cache = mq.KVCache(torch.empty((pages, kvh, page // 16, unit), dtype=torch.uint8, device=DEV), dim, 8)
    assert cache.data.numel() > 1 << 32
    x = rand((2, kvh, dim), 3)
    slots = ints([pages * page - 1, (pages - 1) * page])
    mq.kv_write(cache, x, -x, slots)
    k, v = mq.kv_read(cache, slots)
    c, s, b = ref.quantize(f64(x), 8)
    assert np.array_equal(f64(k), ref.bf16(ref.dequantize(c, s, b)))
    q = rand((1, 8, dim), 4)
    out = mq.paged_attention(q, cache, ints([[pages - 1]]), ints([1]))  # that page alone, its first row
    c, s, b = ref.quantize(f64(-x), 8)
    want = ref.dequantize(c, s, b)[1].repeat(2, 0)
    assert (np.abs(f64(out)[0] - want) <= (2 * U + U * U) * np.abs(want)).all()


# ---- attention -------------------------------------------------------------------------------------


def make_cache(lens, kvh, dim, bits, page, seed, spare=2, poison=True):
    """A cache with random keys and values of every sequence in shuffled pages, NaN scales everywhere else;
    the dequantized rows in 64 bits and the table."""
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    cache = mq.KVCache.empty(pages, page, kvh, dim, bits)
    if poison:
        cache.data.fill_(0xFF)  # scales and biases of -nan, codes of the top
    order = np.random.RandomState(seed).permutation(pages)
    table = np.full((len(lens), max([1] + need)), -1, np.int32)
    ks, vs, used = [], [], 0
    for b, n in enumerate(lens):
        table[b, :need[b]] = order[used:used + need[b]]
        used += need[b]
        k, v = rand((n, kvh, dim), seed + 17 * b + 1), rand((n, kvh, dim), seed + 17 * b + 2)
        if n:
            i = np.arange(n)
            mq.kv_write(cache, k, v, ints((table[b, i // page].astype(np.int64) * page + i % page).astype(np.int32)))
        for x, to in ((k, ks), (v, vs)):
            c, s, z = ref.quantize(f64(x), bits) if n else (np.zeros((0, kvh, dim), int),) + (np.zeros((0, kvh, dim // 64)),) * 2
            to.append(ref.dequantize(c, s, z))
    return cache, torch.from_numpy(table).to(DEV), ks, vs


def check(out, q, ks, vs, lens, starts, scale):
    want, mix, top, spread = (x[:starts[-1]] for x in ref.attention(f64(q), ks, vs, lens, starts, scale))
    got = f64(out)[:starts[-1]]
    rise = np.exp(2 * 2.0**-10 * spread)[..., None] * (1 + 2.0**-10) ** 2 - 1
    bound = (rise + 2.0**-12) * mix + 2.0**-11 * 1.1 * top + U * np.abs(want)
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= bound).all(), float((np.abs(got - want) - bound).max())
    if np.linalg.norm(want) > 0:
        assert np.linalg.norm(got - want) <= 0.003 * np.linalg.norm(want)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (3, 3), (7, 1), (16, 1), (24, 1)])
@pytest.mark.parametrize("page", [16, 48])
def test_one_token_each(dim, bits, heads, kv_heads, page):
    lens = [1, 15, 16, 17, 31, 33, 127, 300, 0, 64]
    cache, table, ks, vs = make_cache(lens, kv_heads, dim, bits, page, dim + bits)
    q = rand((len(lens), heads + 1, dim), 77, size=1.5)[:, :heads]
    out = mq.paged_attention(q, cache, table, ints(lens))
    check(out, q, ks, vs, lens, list(range(len(lens) + 1)), dim ** -0.5)
    assert not out[8].any()  # no position at all


@pytest.mark.parametrize("dim,bits", [(64, 4), (128, 8), (256, 4), (256, 8)])
@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (5, 1)])
def test_packed_chunks(dim, bits, heads, kv_heads):
    """Chunks of different lengths behind different histories, from one token to more than a tile of rows."""
    new = [1, 5, 40, 2, 0, 129, 17]
    lens = [1, 5, 40, 700, 9, 133, 160]
    starts = np.concatenate([[0], np.cumsum(new)]).tolist()
    cache, table, ks, vs = make_cache(lens, kv_heads, dim, bits, 32, 5)
    q = rand((starts[-1] + 3, heads, dim), 78, size=1.5)
    out = torch.full_like(q, 7.0)
    got = mq.paged_attention(q, cache, table, ints(lens), ints(starts), max(new), scale=0.07, out=out)
    assert got is out
    check(out, q, ks, vs, lens, starts, 0.07)
    assert (out[starts[-1]:] == 7.0).all()  # rows behind the last sequence stay


@pytest.mark.parametrize("dim,bits", [(64, 8), (128, 4), (256, 4)])
@pytest.mark.parametrize("new", [2, 3, 4, 8, 16])
def test_few_tokens(dim, bits, new):
    lens = [new, new + 1, 95, 260]
    starts = [new * i for i in range(5)]
    cache, table, ks, vs = make_cache(lens, 2, dim, bits, 16, new)
    q = rand((4 * new, 4, dim), 3, size=1.5)
    out = mq.paged_attention(q, cache, table, ints(lens), ints(starts), new)
    check(out, q, ks, vs, lens, starts, dim ** -0.5)


@pytest.mark.parametrize("new,max_q", [(3, 3), (70, 70)])
def test_rows_that_see_nothing_are_zero(new, max_q):
    """More new tokens than cached positions: the first ones see none."""
    cache, table, ks, vs = make_cache([2, 1], 2, 128, 4, 16, 9)
    q = rand((2 * new, 8, 128), 1)
    starts = [0, new, 2 * new]
    out = mq.paged_attention(q, cache, table, ints([2, 1]), ints(starts), max_q)
    check(out, q, ks, vs, [2, 1], starts, 128 ** -0.5)
    assert not out[:new - 2].any() and out[new - 2].any() and not out[new:2 * new - 1].any()


def on_gpu(q, ks, vs, n_pos, scale):
    """64-bit attention of one sequence's newest rows on the GPU, for lengths too long for numpy loops."""
    n, heads, dim = q.shape
    group = heads // ks.shape[1]
    k, v = torch.from_numpy(ks).to(DEV), torch.from_numpy(vs).to(DEV)
    last = torch.arange(n_pos - n, n_pos, device=DEV)[:, None]
    hide = torch.arange(n_pos, device=DEV) > last
    return torch.stack([torch.softmax((q[:, h].double() @ k[:, h // group].T * scale).masked_fill(hide, -math.inf), -1)
                        @ v[:, h // group] for h in range(heads)], 1)


@pytest.mark.parametrize("dim,bits,heads,kv_heads,new,n_pos", [
    (256, 4, 8, 2, 1, 20011), (128, 8, 4, 1, 1, 33333), (64, 4, 6, 2, 1, 9999), (128, 4, 8, 2, 4, 7001),
    (256, 4, 8, 2, 600, 1500), (256, 8, 2, 2, 257, 257), (128, 4, 8, 2, 500, 3000), (128, 8, 16, 1, 130, 2222), (64, 8, 6, 2, 333, 1999),
    (64, 4, 3, 1, 1000, 1000)])
def test_long(dim, bits, heads, kv_heads, new, n_pos):
    cache, table, ks, vs = make_cache([n_pos], kv_heads, dim, bits, 64, 21)
    q = rand((new, heads, dim), 8, size=1.5)
    out = mq.paged_attention(q, cache, table, ints([n_pos]), ints([0, new]), new)
    want = on_gpu(q, ks[0], vs[0], n_pos, dim ** -0.5)
    err = float((out.double() - want).norm() / want.norm())
    assert err <= 0.003, err
    # no output is far off on its own (a lost or doubled position would be)
    rms = want.square().mean(-1, keepdim=True).sqrt()
    assert float(((out.double() - want).abs() / (rms + want.abs())).max()) <= 0.03


def test_large_scores_and_late_maximum():
    """The running maximum grows late and far: weights of the earlier positions fall to nothing."""
    dim, n_pos = 128, 500
    cache = mq.KVCache.empty(32, 16, 1, dim, 8)
    k = torch.zeros((n_pos, 1, dim), device=DEV, dtype=torch.bfloat16)
    k[:, 0, 0] = torch.linspace(-4, 4, n_pos, device=DEV).bfloat16()
    v = rand((n_pos, 1, dim), 4)
    mq.kv_write(cache, k, v, torch.arange(n_pos, dtype=torch.int32, device=DEV))
    table = torch.arange(32, dtype=torch.int32, device=DEV)[None]
    for sign in (100.0, -100.0, 0.0):
        for new in (1, 40):
            q = torch.zeros((new, 2, dim), device=DEV, dtype=torch.bfloat16)
            q[:, :, 0] = sign
            out = mq.paged_attention(q, cache, table, ints([n_pos]), ints([0, new]), new, scale=1.0)
            kk, vv = mq.kv_read(cache, torch.arange(n_pos, dtype=torch.int32, device=DEV))
            check(out, q, [f64(kk)], [f64(vv)], [n_pos], [0, new], 1.0)


def test_bad_pages_and_lengths_are_recorded():
    cache, table, ks, vs = make_cache([40, 20], 1, 64, 4, 16, 2, poison=False)
    q = rand((2, 2, 64), 1)
    for bad_table, lens in ((ints([[0, 99, 1], [0, 1, 2]]), [40, 20]), (ints([[-1, 0, 1], [0, 1, 2]]), [40, 20]),
                            (table, [49, 20]), (table, [-3, 20])):
        out = mq.paged_attention(q, cache, bad_table, ints(lens))
        torch.cuda.synchronize()
        assert mq.device_error() == 3
        assert torch.isfinite(out).all()
    # starts that run backwards or past the rows, more new tokens than max_q
    for starts, most in (([0, 5, 2], 5), ([0, 1, 9], 9), ([-4, 1, 2], 2), ([0, 2, 2], 1)):
        mq.paged_attention(q, cache, table, ints([40, 20]), ints(starts), most)
        torch.cuda.synchronize()
        assert mq.device_error() == 3


def test_same_bits_every_time_and_any_workspace():
    lens = [900, 31, 4000]
    cache, table, _, _ = make_cache(lens, 2, 128, 4, 32, 6)
    q = rand((3, 8, 128), 5)
    first = mq.paged_attention(q, cache, table, ints(lens))
    size = mq.attention_workspace_size(3, 8, 2, 128, 3)
    for fill in (0, 255):
        ws = torch.full((size,), fill, dtype=torch.uint8, device=DEV)
        for _ in range(3):
            assert torch.equal(first, mq.paged_attention(q, cache, table, ints(lens), workspace=ws))
    with pytest.raises(mq.MarlinQ4Error):
        mq.paged_attention(q, cache, table, ints(lens), workspace=ws[:256])


@pytest.mark.parametrize("batch", [129, 1024])
def test_many_sequences(batch):
    rng = np.random.RandomState(batch)
    lens = rng.randint(0, 50, batch).tolist()
    cache, table, ks, vs = make_cache(lens, 1, 64, 4, 16, 1)
    q = rand((batch, 2, 64), 2)
    out = mq.paged_attention(q, cache, table, ints(lens))
    check(out, q, ks, vs, lens, list(range(batch + 1)), 0.125)
    with pytest.raises(mq.MarlinQ4Error):
        mq.paged_attention(q[:1].expand(1025, 2, 64), cache, table[:1].expand(1025, -1), ints([1] * 1025))


def serve_step(cache, w, pos, rot, slots, table, lens, fused, cu=None, most=1):
    q, k, v = fused[:, :4], fused[:, 4:6], fused[:, 6:]
    q, k = mq.qk_norm_rope(q, k, w, w, pos, rot)
    mq.kv_write(cache, k, v.to(k.dtype), slots)
    return mq.paged_attention(q, cache, table, lens, cu, most)


def test_prompt_then_steps_as_served():
    """A prompt in two chunks, then single tokens: each output equals attention over the rows read back."""
    dim, page, bits = 128, 16, 8
    cache = mq.KVCache.empty(9, page, 2, dim, bits)
    table = ints([[7, 2, 5, 0, 8, 1]])
    w, freqs = rand((dim,), 1, size=0.1), (1e4 ** (-torch.arange(16, dtype=torch.float64) / 16)).float().to(DEV)
    rot = mq.Rotary(freqs)
    total = 0
    for step, new in enumerate([33, 20, 1, 1, 5, 1]):
        fused = rand((new, 8, dim), 50 + step, torch.float32)
        i = torch.arange(total, total + new, device=DEV)
        slots = (table[0, i // page] * page + i % page).int()
        total += new
        out = serve_step(cache, w, i.int(), rot, slots, table, ints([total]), fused, ints([0, new]), new)
        j = torch.arange(total, device=DEV)
        k, v = mq.kv_read(cache, (table[0, j // page] * page + j % page).int())
        q, _ = mq.qk_norm_rope(fused[:, :4], fused[:, 4:6], w, w, i.int(), rot)
        check(out, q, [f64(k)], [f64(v)], [total], [0, new], dim ** -0.5)


def test_captured_step_replays_on_new_lengths():
    dim, page = 256, 16
    cache = mq.KVCache.empty(40, page, 2, dim, 4)
    table = torch.arange(40, dtype=torch.int32, device=DEV).reshape(2, 20)
    w, rot = rand((dim,), 1, size=0.1), mq.Rotary(torch.full((32,), 0.01, device=DEV))
    fused = torch.zeros((2, 8, dim), device=DEV)
    pos, slots, lens = ints([0, 0]), ints([0, 0]), ints([0, 0])
    ws = torch.empty(mq.attention_workspace_size(2, 4, 2, dim, 2), dtype=torch.uint8, device=DEV)

    def step():
        q, k = mq.qk_norm_rope(fused[:, :4], fused[:, 4:6], w, w, pos, rot)
        mq.kv_write(cache, k, fused[:, 6:].bfloat16(), slots)
        return mq.paged_attention(q, cache, table, lens, workspace=ws)

    step()
    torch.cuda.synchronize()
    cache.data.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(60):
        fused.copy_(rand((2, 8, dim), 100 + i, torch.float32))
        at = [i, i // 3]
        pos.copy_(ints(at)), lens.copy_(ints([a + 1 for a in at]))
        slots.copy_(ints([int(table[b, at[b] // page]) * page + at[b] % page for b in range(2)]))
        graph.replay()
        torch.cuda.synchronize()
        if i % 13 == 0 or i == 59:
            assert torch.equal(out, step())


def test_other_stream_and_pdl_off():
    lens = [700, 64]
    cache, table, _, _ = make_cache(lens, 2, 128, 8, 32, 6)
    q = rand((2, 8, 128), 5)
    n = ints(lens)
    want = mq.paged_attention(q, cache, table, n)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = mq.paged_attention(q, cache, table, n)
    side.synchronize()
    assert torch.equal(got, want)
    mq.set_pdl(False)
    try:
        assert torch.equal(mq.paged_attention(q, cache, table, n), want)
    finally:
        mq.set_pdl(True)


def test_nan_query_stays_in_its_row():
    cache, table, ks, vs = make_cache([100], 2, 128, 4, 16, 3)
    q = rand((4, 8, 128), 1)
    clean = mq.paged_attention(q, cache, table, ints([100]), ints([0, 4]), 4)
    q[2, 5, 7] = float("nan")
    out = mq.paged_attention(q, cache, table, ints([100]), ints([0, 4]), 4)
    bad = torch.isnan(out).any(-1)
    assert bad[2, 5] and bad.sum() == 1
    bad[2, 5] = True
    assert torch.equal(out[~bad], clean[~bad])


def test_no_tokens():
    cache = mq.KVCache.empty(1, 16, 2, 64, 4)
    q = torch.empty((0, 4, 64), dtype=torch.bfloat16, device=DEV)
    assert mq.paged_attention(q, cache, ints([[0]])[:0], ints([])).shape == (0, 4, 64)
    assert mq.paged_attention(q, cache, ints([[0]]), ints([3]), ints([0, 0]), 1).shape == (0, 4, 64)
    k = torch.empty((0, 2, 64), dtype=torch.bfloat16, device=DEV)
    mq.kv_write(cache, k, k, ints([]))
    assert mq.kv_read(cache, ints([]))[0].shape == (0, 2, 64)
    w = rand((64,), 1)
    assert mq.qk_norm_rope(q, k, w, w, ints([]), mq.Rotary(torch.ones(8, device=DEV)))[1].shape == (0, 2, 64)
