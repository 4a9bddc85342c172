"""The token-step operators (4-bit weights, 8-bit key/value cache, sampling)
against their definitions in 64 bits, on the CPU path and on the GPU kernels.

Tolerances: an output in t is off by at most half a step, finfo(t).eps / 2 of
its value, beside what the fp32 sums before it lose; each test writes that down.
Codes, scales and tokens have to be equal."""
import math

import numpy as np
import pytest
import torch

from mi355 import ops
from mi355.ops import torch_ref

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def gen(seed, device="cpu"):
    return torch.Generator(device=device).manual_seed(seed)


def randn(*shape, seed, device, dtype=FP32):
    return torch.randn(*shape, generator=gen(seed)).to(device=device, dtype=dtype)


# --------------------------------------------------------------------------- #
# 4-bit weights                                                               #
# --------------------------------------------------------------------------- #
def w4_values(codes, exps):
    """fp64 weights from the format's definition, code by code."""
    def value(c):
        e, m = c >> 1 & 3, c & 1
        v = m * 0.5 if e == 0 else (1 + m / 2) * 2.0 ** (e - 1)
        return -v if c & 8 else v

    table = np.array([value(c) for c in range(16)])
    codes, exps = codes.cpu().numpy(), exps.cpu().numpy()
    w = np.empty((codes.shape[0], codes.shape[1] * 2))
    w[:, 0::2], w[:, 1::2] = table[codes & 15], table[codes >> 4]
    return torch.from_numpy(w * np.repeat(2.0 ** (exps.astype(np.float64) - 127), 32, 1))


def random_w4(n, k, seed, device, lo=115, hi=125):
    g = gen(seed)
    return ops.W4Weight(torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8).to(device),
                        torch.randint(lo, hi, (n, k // 32), generator=g, dtype=torch.uint8).to(device))


def check_linear(x, w, y):
    ref_w = w4_values(w.codes, w.exps)
    x64 = x.double().cpu().reshape(-1, x.shape[-1])
    ref = x64 @ ref_w.t()
    # one rounding to y's type, and a sum of K products in fp32 (products of
    # 16-bit numbers are exact): at most K half steps of the sum of sizes
    size = x64.abs() @ ref_w.abs().t()
    info = torch.finfo(y.dtype)
    tol = info.eps / 2 * ref.abs() + x.shape[-1] * 2.0 ** -24 * size + info.tiny
    err = (y.double().cpu().reshape(ref.shape) - ref).abs()
    over = ref.abs() > info.max
    assert bool(((err <= tol) | over).all()), (err / tol).max()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,n,k", [(1, 1, 32), (1, 16, 64), (1, 2304, 768), (3, 17, 96), (5, 48, 2048),
                                   (16, 100, 1024), (17, 33, 160), (31, 129, 128), (64, 65, 512),
                                   (65, 200, 736), (130, 257, 320), (256, 64, 4096), (300, 512, 768),
                                   (40, 130, 4128), (100, 2050, 4640), (260, 8200, 96), (9, 8200, 160), (8, 8200, 4640), (129, 2700, 128),
                                   (2, 16390, 288)])
def test_linear_w4(device, dtype, m, n, k):
    w = random_w4(n, k, seed=m * 7 + n, device=device)
    x = randn(m, k, seed=k, device=device, dtype=dtype)
    check_linear(x, w, ops.linear_w4(x, w))


@pytest.mark.parametrize("device", DEVICES)
def test_linear_w4_layouts(device):
    """Leading dims, rows with gaps, offsets that are not 16-byte aligned, a
    transposed input, no rows, slices of output rows, ops.linear."""
    w = random_w4(70, 192, seed=1, device=device)
    base = randn(9, 400, seed=2, device=device, dtype=BF16)
    for x in (base[:, :192], base[:, 8:200], base[:, 3:195], base.t()[:192].t()[:, :192].expand(9, 192),
              randn(192, 9, seed=3, device=device, dtype=BF16).t(),
              randn(2, 3, 192, seed=4, device=device, dtype=BF16), base[:1, 5:197]):
        check_linear(x, w, ops.linear_w4(x, w))
        assert torch.equal(ops.linear(x, w), ops.linear_w4(x, w))
    assert ops.linear_w4(base[:0, :192], w).shape == (0, 70)
    part = w.rows(13, 40)
    x = base[:, :192]
    assert torch.equal(ops.linear_w4(x, part), ops.linear_w4(x, w)[:, 13:40])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_linear_w4_far_exponents(device, dtype):
    """Scales of one row that are up to 2^22 apart stay exact in both types;
    the smallest exponent byte is a scale too."""
    w = random_w4(40, 256, seed=5, device=device, lo=100, hi=123)
    x = randn(4, 256, seed=6, device=device, dtype=dtype)
    check_linear(x, w, ops.linear_w4(x, w))
    w = random_w4(8, 64, seed=7, device=device, lo=0, hi=3)
    check_linear(x[:, :64], w, ops.linear_w4(x[:, :64], w))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,n,k", [(1, 40, 32), (2, 24, 96), (1, 16400, 288), (8, 40, 416), (12, 40, 160),
                                   (12, 8210, 160), (40, 40, 416), (70, 70, 4128), (130, 8200, 160)])
def test_linear_w4_infinite_inputs(device, dtype, m, n, k):
    """An infinity makes infinite outputs (no NaN) of its own row alone, also
    among the last inputs; NaN makes NaN."""
    codes = torch.full((n, k // 2), 0x22, dtype=torch.uint8, device=device)      # ones
    w = ops.W4Weight(codes, torch.full((n, k // 32), 127, dtype=torch.uint8, device=device))
    x = torch.ones(m, k, device=device, dtype=dtype)
    x[m - 1, k - 1] = math.inf
    if m > 1:
        x[0, k - 32] = -math.inf
    if m > 2:
        x[1, k - 7] = math.nan
    y = ops.linear_w4(x, w)
    assert bool((y[m - 1] == math.inf).all())
    if m > 1:
        assert bool((y[0] == -math.inf).all())
    if m > 2:
        assert bool(y[1].isnan().all()) and bool((y[2:m - 1] == k).all() or dtype == BF16)
        assert bool(y[2:m - 1].isfinite().all())


@pytest.mark.parametrize("device", DEVICES)
def test_w4_empty_strided_and_refused(device):
    """A weight without rows, one that is a view, and what cannot be quantized."""
    w = ops.quantize_w4(torch.zeros(0, 64, device=device))
    assert w.shape == (0, 64) and w.dequantize().shape == (0, 64)
    assert ops.linear_w4(torch.ones(3, 64, device=device, dtype=BF16), w).shape == (3, 0)
    weight = randn(64, 40, seed=11, device=device)
    assert torch.equal(ops.quantize_w4(weight.t()).codes, ops.quantize_w4(weight.t().contiguous()).codes)
    for bad in (math.nan, math.inf, -math.inf):
        weight[5, 7] = bad
        with pytest.raises(ValueError):
            ops.quantize_w4(weight.t())


@pytest.mark.parametrize("device", DEVICES)
def test_linear_w4_same_twice(device):
    w = random_w4(500, 1024, seed=8, device=device)
    x = randn(20, 1024, seed=9, device=device, dtype=BF16)
    first = ops.linear_w4(x, w)
    assert all(torch.equal(first, ops.linear_w4(x, w)) for _ in range(3))


def test_quantize_w4_is_nearest():
    """Every code is a nearest one at its group's scale, no group's largest
    value is off by over a sixth, and the scale is the better of two."""
    weight = randn(24, 96, seed=10, device="cpu") * torch.logspace(-6, 4, 24)[:, None]
    weight[3] = 0
    weight[4, :32] = 6.0
    w = ops.quantize_w4(weight)
    got = w4_values(w.codes, w.exps)
    assert torch.equal(w.dequantize().double(), got)
    assert torch.equal(got[3], torch.zeros(96, dtype=torch.float64))
    assert torch.equal(got[4, :32], torch.full((32,), 6.0, dtype=torch.float64))
    grid = torch.tensor(torch_ref.E2M1, dtype=torch.float64)
    grid = torch.cat([-grid, grid])

    def off(exps):
        scale = 2.0 ** (exps.double() - 127).repeat_interleave(32, 1)
        return ((weight.double() / scale)[..., None] - grid).abs().amin(-1) * scale

    near = off(w.exps)
    assert torch.allclose((got - weight.double()).abs(), near, rtol=1e-12, atol=0)
    for other in (w.exps + 1, w.exps.clamp(min=1) - 1):
        worse = off(other).square().view(24, 3, 32).sum(-1) - near.square().view(24, 3, 32).sum(-1)
        assert bool((worse >= -1e-12 * near.square().view(24, 3, 32).sum(-1)).all())


# --------------------------------------------------------------------------- #
# 8-bit cache                                                                 #
# --------------------------------------------------------------------------- #
def round_e4m3(x):
    step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -6))) - 3)
    return np.clip(np.round(x / step) * step, -448, 448)


class Plain8:
    """The cache's definition in 64 bits, token by token."""

    def __init__(self, b, h, cap, d):
        self.nb = -(-cap // 64)
        self.codes = np.zeros((2, b, h, self.nb, 64, d))
        self.scale = np.full((2, b, h, self.nb), 2.0 ** -120)

    def append(self, k, v, start, counts=None):
        b, h, s, d = k.shape
        for which, new in enumerate((k, v)):
            new = new.double().cpu().numpy()
            for i in range(b):
                at = int(start[i]) if torch.is_tensor(start) else start
                n = s if counts is None else min(s, int(counts[i]))
                if at < 0 or n <= 0:
                    continue
                end = min(at + n, self.nb * 64)
                for blk in range(at // 64, -(-end // 64)):
                    lo, hi = max(at, blk * 64), min(end, blk * 64 + 64)
                    fresh = new[i, :, lo - at:hi - at]
                    size = np.where(np.isfinite(fresh), np.abs(fresh), 0).max((1, 2))
                    with np.errstate(divide="ignore"):
                        e = np.ceil(np.log2(size / 448))
                    scale = 2.0 ** np.clip(e, -120, 120)
                    begun = lo - blk * 64
                    if begun:
                        old = self.scale[which, i, :, blk].copy()
                        scale = np.maximum(scale, old)
                        part = self.codes[which, i, :, blk, :begun]
                        self.codes[which, i, :, blk, :begun] = round_e4m3(part * (old / scale)[:, None, None])
                    self.codes[which, i, :, blk, begun:begun + hi - lo] = round_e4m3(fresh / scale[:, None, None])
                    self.scale[which, i, :, blk] = scale

    def same(self, cache):
        b, h, nb, _, d = self.codes.shape[1:]
        k = cache.k.double().cpu().numpy().reshape(b, h, nb, 64, d)
        v = cache.v.double().cpu().numpy().swapaxes(-1, -2)
        for got, want in ((k, self.codes[0]), (v, self.codes[1]), (cache.k_scale.double().cpu().numpy(), self.scale[0]),
                          (cache.v_scale.double().cpu().numpy(), self.scale[1])):
            np.testing.assert_array_equal(got, want)


def tokens(b, h, s, d, seed, device, dtype, spread=6.0):
    """(B,H,S,D) as projections give them: a view of (B,S,H,D), sizes spread
    over some octaves so that scales grow while tokens come."""
    g = gen(seed)
    t = torch.randn(b, s, h, d, generator=g) * 2.0 ** (spread * (torch.rand(b, s, h, 1, generator=g) - 0.5))
    return t.to(device=device, dtype=dtype).transpose(1, 2)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("cap,steps", [(1, [1]), (64, [64]), (200, [70, 1, 1, 57, 2]), (130, [1] * 130),
                                       (300, [0, 63, 1, 1, 128, 100])])
def test_kv8_append(device, dtype, d, cap, steps):
    b, h = 2, 3
    cache, plain = ops.KVCache8(b, h, cap, d, device=device), Plain8(b, h, cap, d)
    at = 0
    for i, s in enumerate(steps):
        k, v = (tokens(b, h, s, d, 100 * i + j, device, dtype) for j in (1, 2))
        ops.kv8_append(cache, k, v, at)
        plain.append(k, v, at)
        at += s
    plain.same(cache)


@pytest.mark.parametrize("device", DEVICES)
def test_kv8_append_ragged(device):
    """Starts and counts of each sequence's own: in the middle of blocks, back
    over tokens that are there (codes behind stay), none, negative, past the
    capacity."""
    b, h, d, cap = 7, 2, 64, 256
    cache, plain = ops.KVCache8(b, h, cap, d, device=device), Plain8(b, h, cap, d)
    k, v = (tokens(b, h, 150, d, j, device, BF16) for j in (3, 4))
    ops.kv8_append(cache, k, v, 0)
    plain.append(k, v, 0)
    start = torch.tensor([150, 40, 64, 0, -5, 250, 2_000_000_000], dtype=torch.int32, device=device)
    counts = torch.tensor([70, 1, 3, 0, 9, 70, 70], dtype=torch.int32, device=device)
    k, v = (tokens(b, h, 70, d, j, device, BF16) for j in (5, 6))
    ops.kv8_append(cache, k, v, start, counts)
    plain.append(k, v, start, counts)
    plain.same(cache)
    counts = torch.tensor([-1, 5000, 0, 2, 0, 0, 0], dtype=torch.int32, device=device)
    ops.kv8_append(cache, k, v, torch.zeros_like(start), counts)
    plain.append(k, v, torch.zeros(b, dtype=torch.int32), counts)
    plain.same(cache)


@pytest.mark.parametrize("device", DEVICES)
def test_kv8_append_strides_and_specials(device):
    """Other strides, unaligned views, infinities (saturate, do not widen the
    scale), NaN (stays), zeros, the smallest and largest numbers."""
    b, h, s, d = 2, 2, 66, 32
    plain = Plain8(b, h, 66, d)
    cache = ops.KVCache8(b, h, 66, d, device=device)
    wide = randn(b, h, d + 9, s, seed=7, device=device, dtype=BF16)
    k, v = wide[:, :, 3:3 + d].transpose(2, 3), randn(b, h, s, d + 8, seed=8, device=device, dtype=BF16)[..., 1:1 + d]
    ops.kv8_append(cache, k, v, 0)
    plain.append(k, v, 0)
    plain.same(cache)
    k = torch.zeros(b, h, 2, d, device=device, dtype=BF16)
    v = k.clone()
    k[0, 0, 0, :4] = torch.tensor([3e38, -3e38, 1e-38, 1.0])
    v[0, 0, 1, :2] = torch.tensor([1e-38, -1e-38])
    v[1, 1, 0, 5] = 0.125
    cache, plain = ops.KVCache8(b, h, 2, d, device=device), Plain8(b, h, 2, d)
    ops.kv8_append(cache, k, v, 0)
    plain.append(k, v, 0)
    plain.same(cache)
    k[1, 0, 0, 0], k[1, 0, 0, 1], k[1, 0, 0, 2], k[1, 0, 0, 3] = math.inf, -math.inf, math.nan, 2.0
    ops.kv8_append(cache, k, v, 0)
    got = (cache.k.float()[1, 0, 0, :4]).tolist()
    assert float(cache.k_scale[1, 0, 0]) == 2.0 ** -7       # of 2.0: 448 * 2^-7 = 3.5
    assert got[:2] == [448.0, -448.0] and math.isnan(got[2]) and got[3] == 256.0


def attention_case(b, h, grp, d, length, dtype, device, seed, bias=None, kpad=None, ragged=False, cap=None):
    cap = cap or max(length, 1)
    cache = ops.KVCache8(b, h, cap, d, device=device)
    if length:
        k = tokens(b, h, length, d, seed, device, dtype, spread=2.0)
        v = tokens(b, h, length, d, seed + 1, device, dtype, spread=2.0)
        ops.kv8_append(cache, k, v, 0)
    q = tokens(b, h * grp, 1, d, seed + 2, device, dtype, spread=1.0)
    lengths = length
    if ragged:
        lengths = torch.randint(0, length + 1, (b,), generator=gen(seed + 3), dtype=torch.int32)
        lengths[0], lengths[-1] = length, 0
        lengths = lengths.to(device)
    if bias is not None:
        bias = randn(bias, h * grp, 1, length, seed=seed + 4, device=device)
    if kpad:
        pad = torch.where(torch.rand(b, length, generator=gen(seed + 5)) < 0.4, kpad, 0.0)
        kpad = pad.to(device)
    else:
        kpad = None
    return q, cache, lengths, bias, kpad


def check_attention(q, cache, lengths, bias, kpad, scale, out, max_len=None):
    b, hq, _, d = q.shape
    k, v = (t.double().cpu() for t in cache.dequantize())
    h = k.shape[1]
    assert out.shape == q.shape and out.dtype == q.dtype
    for i in range(b):
        n = int(lengths[i]) if torch.is_tensor(lengths) else lengths
        n = max(0, min(n, cache.capacity if max_len is None else max_len))
        if n == 0:
            assert bool((out[i] == 0).all())
            continue
        qi = q[i].double().cpu().view(h, hq // h, d)
        kk, vv = k[i, :, None, :n], v[i, :, None, :n]                   # (H,1,n,D)
        s = (qi[:, :, None] * kk).sum(-1) * scale
        size = (qi[:, :, None].abs() * kk.abs()).sum(-1) * abs(scale)    # what the fp32 sum runs over
        if bias is not None:
            add = bias[i if bias.shape[0] > 1 else 0, :, 0, :n].double().cpu().view(h, -1, n)
            s, size = s + add, size + add.abs()
        if kpad is not None:
            add = kpad[i, None, None, :n].double().cpu()
            s = torch.where(add == -math.inf, -math.inf, s + add)
            size = size + torch.where(add == -math.inf, 0.0, add.abs())
        o = out[i].double().cpu().view(h, -1, d)
        if bool((s == -math.inf).all()):
            assert bool((o == 0).all())
            continue
        p = torch.softmax(s, -1)
        ref = (p[..., None] * vv).sum(2)
        spread = (p[..., None] * vv.abs()).sum(2)
        # a score: D + 4 roundings of its sum of sizes; a weight: the score's
        # error, that of the difference from the maximum and of its exp (2^-21
        # together, relative), 2^-16 for hi + lo; sums of n weights; twice,
        # for numerator and denominator
        delta = ((d + 4) * 2.0 ** -24 * size * (p > 0)).amax(-1, keepdim=True) * 2
        delta = delta + 2.0 ** -21 * (1 + (s.amax(-1, keepdim=True) - s).clamp(max=60).amax(-1, keepdim=True))
        delta = delta + 2.0 ** -16 + n * 2.0 ** -24
        tol = torch.finfo(q.dtype).eps / 2 * ref.abs() + 2 * delta * spread + torch.finfo(q.dtype).tiny
        err = (o - ref).abs()
        assert bool((err <= tol).all()), (i, n, float((err / tol).max()))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("b,h,grp,d,length", [
    (1, 1, 1, 64, 1), (2, 3, 1, 64, 63), (2, 2, 1, 64, 64), (1, 12, 1, 64, 65), (3, 2, 4, 128, 200),
    (2, 1, 8, 32, 257), (1, 2, 7, 64, 513), (1, 1, 16, 64, 130), (1, 2, 9, 128, 300), (1, 1, 33, 32, 70),
    (1, 1, 1, 128, 3000), (1, 2, 20, 64, 2100)])
def test_decode_attention_kv8(device, dtype, b, h, grp, d, length):
    q, cache, lengths, _, _ = attention_case(b, h, grp, d, length, dtype, device, 11)
    scale = d ** -0.5
    check_attention(q, cache, lengths, None, None, scale,
                    ops.decode_attention_kv8(q, cache, lengths, scale=scale))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bias", [None, 1, 3])
@pytest.mark.parametrize("kpad", [None, -1e9, torch.finfo(FP32).min, -math.inf])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("grp,length", [(1, 45), (2, 130), (12, 1000)])
def test_decode_attention_kv8_masks(device, bias, kpad, ragged, grp, length):
    q, cache, lengths, bias, kpad = attention_case(3, 2, grp, 64, length, BF16, device, 21, bias, kpad, ragged)
    out = ops.decode_attention_kv8(q, cache, lengths, bias=bias, kpad=kpad, max_len=length)
    check_attention(q, cache, lengths, bias, kpad, 1.0, out, max_len=length)


@pytest.mark.parametrize("device", DEVICES)
def test_decode_attention_kv8_nothing_left(device):
    """Rows whose mask leaves nothing, lengths of zero, a cache that was never
    written, a capacity of zero."""
    q, cache, _, _, kpad = attention_case(3, 2, 2, 64, 100, BF16, device, 31, None, -math.inf)
    kpad[1] = -math.inf
    out = ops.decode_attention_kv8(q, cache, 100, kpad=kpad)
    check_attention(q, cache, 100, None, kpad, 1.0, out)
    assert bool((out[1] == 0).all())
    # finite masks of the lowest value leave an even row, as a softmax does
    low = torch.full_like(kpad, torch.finfo(FP32).min)
    check_attention(q, cache, 100, None, low, 1.0, ops.decode_attention_kv8(q, cache, 100, kpad=low))
    for lengths in (0, torch.zeros(3, dtype=torch.int32, device=device),
                    torch.full((3,), -4, dtype=torch.int32, device=device)):
        assert bool((ops.decode_attention_kv8(q, cache, lengths) == 0).all())
    empty = ops.KVCache8(3, 2, 0, 64, device=device)
    assert bool((ops.decode_attention_kv8(q, empty, 0) == 0).all())


@pytest.mark.parametrize("device", DEVICES)
def test_decode_attention_kv8_garbage_does_not_leak(device):
    """NaN codes and scales-with-NaN-keys where nothing is: behind the length,
    in blocks behind it, and under a mask of -inf.  NaN where something is
    comes out."""
    q, cache, _, _, kpad = attention_case(2, 2, 1, 64, 150, BF16, device, 41, None, -math.inf, cap=320)
    want = ops.decode_attention_kv8(q, cache, 150, kpad=kpad)
    check_attention(q, cache, 150, None, kpad, 1.0, want)
    for name in ("k", "v"):
        raw = getattr(cache, name).view(torch.uint8)
        plane = raw if name == "k" else raw.transpose(-1, -2).reshape(2, 2, -1, 64)
        plane = plane.clone()
        plane[:, :, 150:] = 0x7f
        for i in range(2):
            plane[i][:, :150][:, kpad[i, :150] == -math.inf] = 0xff
        if name == "k":
            raw.copy_(plane)
        else:
            raw.copy_(plane.view(2, 2, -1, 64, 64).transpose(-1, -2))
    assert torch.equal(ops.decode_attention_kv8(q, cache, 150, kpad=kpad), want)
    assert torch.equal(ops.decode_attention_kv8(q, cache, torch.full((2,), 150, dtype=torch.int32, device=device),
                                                kpad=torch.nn.functional.pad(kpad, (0, 170))), want)
    cache.k.view(torch.uint8)[0, 0, 0, 0] = 0x7f
    kpad[0, 0] = 0
    out = ops.decode_attention_kv8(q, cache, 150, kpad=kpad)
    assert bool(out[0, 0].isnan().all()) and torch.equal(out[1], want[1])


@pytest.mark.parametrize("device", DEVICES)
def test_decode_attention_kv8_strides(device):
    """Masks wider than the length, with strides and offsets of their own, in
    another type; queries of other strides."""
    q, cache, _, _, _ = attention_case(2, 2, 3, 64, 190, BF16, device, 51)
    bias = randn(2, 6, 5, 301, seed=52, device=device)[:, :, 2:3, 7:]
    kpad = randn(2, 400, seed=53, device=device)[:, 1::2]
    check_attention(q, cache, 190, bias, kpad, 0.5,
                    ops.decode_attention_kv8(q, cache, 190, bias=bias, kpad=kpad, scale=0.5))
    low = bias.to(FP16)
    check_attention(q, cache, 190, low, None, 0.5, ops.decode_attention_kv8(q, cache, 190, bias=low, scale=0.5))
    one = bias[:1].expand(2, -1, -1, -1)
    check_attention(q, cache, 190, one, None, 1.0, ops.decode_attention_kv8(q, cache, 190, bias=one))
    q2 = randn(2, 65, 6, 1, seed=54, device=device, dtype=BF16)[:, 1:].permute(0, 2, 3, 1)
    check_attention(q2, cache, 190, None, None, 1.0, ops.decode_attention_kv8(q2, cache, 190))


@pytest.mark.parametrize("device", DEVICES)
def test_decode_attention_kv8_max_len(device):
    """Lengths are clamped to max_len, and max_len to the capacity."""
    q, cache, _, _, _ = attention_case(3, 2, 1, 64, 256, FP16, device, 61)
    lengths = torch.tensor([256, 10, 2_000_000_000], dtype=torch.int32, device=device)
    for max_len in (100, 5000, None):
        out = ops.decode_attention_kv8(q, cache, lengths, max_len=max_len)
        check_attention(q, cache, lengths, None, None, 1.0, out, max_len=min(max_len or 256, 256))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("capacity", [0, 70])
def test_decode_attention_kv8_no_length_with_masks(device, capacity):
    """No keys at all, however that is said, with masks of any width: 0."""
    cache = ops.KVCache8(2, 3, capacity, 64, device=device)
    q = randn(2, 6, 1, 64, seed=105, device=device, dtype=BF16)
    none = torch.zeros(2, dtype=torch.int32, device=device)
    for width in (0, 5):
        bias, kpad = torch.zeros(1, 6, 1, width, device=device), torch.zeros(2, width, device=device)
        for lengths, most in ((0, None), (none, 0), (none + 9, 0), (none, min(width, capacity))):
            for masks in (dict(), dict(bias=bias), dict(kpad=kpad), dict(bias=bias, kpad=kpad)):
                out = ops.decode_attention_kv8(q, cache, lengths, max_len=most, **masks)
                assert out.shape == q.shape and not bool(out.any())


@gpu
def test_kv8_offsets_over_32_bits():
    """Heads whose codes begin 4.3 GB into the cache."""
    cache = ops.KVCache8(1, 34, 1 << 20, 128, device="cuda")
    k, v, q = (tokens(1, 34, n, 128, j, "cuda", BF16) for j, n in ((1, 200), (2, 200), (3, 1)))
    at = (1 << 20) - 200
    for start in (0, at):
        ops.kv8_append(cache, k[:, :, :199], v[:, :, :199], start)
        ops.kv8_append(cache, k[:, :, 199:], v[:, :, 199:], start + 199)
    small = ops.KVCache8(1, 34, 256, 128, device="cuda")
    ops.kv8_append(small, k, v, 0)
    assert torch.equal(ops.decode_attention_kv8(q, cache, 200), ops.decode_attention_kv8(q, small, 200))
    # of the whole cache all but the last 200 tokens are masked
    kpad = torch.full((1, 1 << 20), -math.inf, device="cuda")
    kpad[:, at:] = 0
    out = ops.decode_attention_kv8(q, cache, 1 << 20, kpad=kpad, scale=0.1)
    part = ops.KVCache8(1, 34, 256, 128, device="cuda")
    first = at // 64 * 64
    part.k[:, :, :(1 << 20) - first] = cache.k[:, :, first:]
    n = ((1 << 20) - first) // 64
    part.v[:, :, :n], part.k_scale[:, :, :n], part.v_scale[:, :, :n] = (
        cache.v[:, :, -n:], cache.k_scale[:, :, -n:], cache.v_scale[:, :, -n:])
    check_attention(q, part, (1 << 20) - first, None, kpad[:, first:], 0.1, out)


# --------------------------------------------------------------------------- #
# sampling                                                                    #
# --------------------------------------------------------------------------- #
def sample_by_definition(logits, u, temperature, top_k, top_p, min_p):
    """Row by row, sorted, in 64 bits."""
    logits, u = logits.double().cpu().numpy(), u.double().cpu().numpy()
    opts = [np.broadcast_to(o.double().cpu().numpy() if torch.is_tensor(o) else float(o), len(u))
            for o in (temperature, top_k, top_p, min_p)]
    ids = []
    for x, r, t, k, p, floor in zip(logits, u, *opts):
        x = np.where(np.isnan(x), -np.inf, x)
        order = np.argsort(-x, kind="stable")
        if x.max() == -np.inf:
            ids.append(-1)
            continue
        if not t > 0:
            ids.append(int(order[0]))
            continue
        order = order[:int(k)] if k > 0 else order
        top = x[order[0]]
        with np.errstate(invalid="ignore"):
            w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / t))
        n = len(order)
        if p < 1:
            cum = np.cumsum(w)
            n = max(1, int((cum < p * cum[-1]).sum()) + 1)
        n = max(1, min(n, int((w >= min(floor, 1.0)).sum())))
        index = np.sort(order[:n])
        weight = dict(zip(order[:n], w[:n]))
        cum = np.cumsum([weight[i] for i in index])
        ids.append(int(index[min(int((cum <= r * cum[-1]).sum()), n - 1)]))
    return ids


def uniform(n, seed, device, dtype=FP32):
    return torch.rand(n, generator=gen(seed), dtype=dtype).to(device)


OPTIONS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=5), dict(top_k=300), dict(top_p=0.9),
           dict(top_p=0.0), dict(top_p=0.3, temperature=1.7), dict(min_p=0.1), dict(min_p=1.0),
           dict(top_k=40, top_p=0.8, min_p=0.02, temperature=0.9), dict(temperature=0.0),
           dict(temperature=100.0, top_p=0.5), dict(temperature=1e-3), dict(top_k=10 ** 9, top_p=0.999)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (4, 2), (3, 7), (5, 64), (3, 1000), (2, 8191), (2, 32128), (2, 50257)])
def test_sample_tokens(device, dtype, rows, vocab):
    logits = (randn(rows, vocab, seed=vocab, device=device) * 3).to(dtype)
    for i, o in enumerate(OPTIONS):
        opt = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, **o}
        u = uniform(rows, 1000 * i + rows, device, torch.float64 if i % 2 else FP32)
        got = ops.sample_tokens(logits, u, **opt)
        assert got.dtype == torch.int64 and got.tolist() == sample_by_definition(logits, u, **opt), opt


@pytest.mark.parametrize("device", DEVICES)
def test_sample_tokens_ties_and_flat_rows(device):
    """Equal logits: cuts go by index, whole rows of one value among them."""
    for vocab in (5, 64, 3000, 20000):
        rows = [torch.zeros(vocab), torch.arange(vocab) % 3 * 1.0, (torch.arange(vocab) // 7 % 2) * 4.0,
                torch.where(torch.arange(vocab) == vocab // 2, 9.0, 0.0), torch.full((vocab,), -1e9)]
        logits = torch.stack(rows).to(device)
        for i, o in enumerate([dict(top_k=2), dict(top_k=vocab // 2), dict(top_p=0.5), dict(top_p=0.75, top_k=vocab - 1),
                               dict(), dict(min_p=0.5), dict(temperature=0.0)]):
            opt = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, **o}
            for seed in range(3):
                u = uniform(len(rows), seed + 10 * i, device)
                assert ops.sample_tokens(logits, u, **opt).tolist() == sample_by_definition(logits, u, **opt), (vocab, opt)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_sample_tokens_masked(device, dtype):
    """-inf, the type's lowest value, -1e4, NaN and +inf among the logits; a
    row with one left, a row with none."""
    vocab = 4100
    g = gen(71)
    logits = (torch.randn(8, vocab, generator=g) * 2).to(dtype)
    drop = torch.rand(8, vocab, generator=g) < 0.9
    for r, value in enumerate([-math.inf, torch.finfo(dtype).min, -1e4, math.nan]):
        logits[r, drop[r]] = value
    logits[4] = -math.inf
    logits[4, 77] = -3.0
    logits[5] = -math.inf
    logits[6, [5, 900, 901]] = math.inf
    logits[7] = math.nan
    logits = logits.to(device)
    for i, o in enumerate(OPTIONS):
        opt = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, **o}
        u = uniform(8, 72 + i, device)
        got = ops.sample_tokens(logits, u, **opt).tolist()
        assert got == sample_by_definition(logits, u, **opt), opt
        assert got[4] == 77 and got[5] == got[7] == -1 and got[6] in (5, 900, 901)
    assert ops.sample_tokens(logits, u, empty_token=3).tolist()[5] == 3


@pytest.mark.parametrize("device", DEVICES)
def test_sample_tokens_per_row_and_strides(device):
    """Options of each row's own (0 turns top_k off, out of range counts as
    the nearest), rows with gaps, unaligned, transposed, no rows; u at its ends."""
    rows, vocab = 9, 1303
    base = randn(rows, vocab + 20, seed=81, device=device, dtype=BF16) * 3
    u = uniform(rows, 82, device)
    u[0], u[1], u[2] = 0.0, 1.0 - 2.0 ** -24, 1.0
    t = torch.tensor([1.0, 0.5, 0.0, 2.0, 1.0, 0.7, -1.0, 1.0, 0.1], device=device)
    k = torch.tensor([0, 1, 10, 0, 50, 2000, 3, -2, 7], dtype=torch.int32, device=device)
    p = torch.tensor([1.0, 0.9, 0.5, 0.0, 0.8, 1.0, 0.2, 2.0, -1.0], device=device)
    m = torch.tensor([0.0, 0.0, 0.1, 0.0, 0.01, 0.2, 0.0, 5.0, 0.0], device=device)
    for logits in (base[:, :vocab], base[:, 3:3 + vocab], base[:, 8:8 + vocab].contiguous(),
                   base[:, :vocab].t().contiguous().t()):
        got = ops.sample_tokens(logits, u, temperature=t, top_k=k.long(), top_p=p, min_p=m)
        assert got.tolist() == sample_by_definition(logits, u, t, k, p.clamp(0, 1), m)
    assert ops.sample_tokens(base[:0], u[:0]).shape == (0,)


@pytest.mark.parametrize("device", DEVICES)
def test_sample_tokens_odd_options(device):
    """Temperatures so small that all weight is the maximum's and so large that
    none is less than another's, infinite and NaN options of a row, NaN as u."""
    logits = randn(6, 3001, seed=101, device=device) * 3 + 20
    u = uniform(6, 102, device)
    best = logits.argmax(1)
    for t in (1e-30, 1e-9, 1e-6):
        opt = {"temperature": t, "top_k": 0, "top_p": 1.0, "min_p": 0.0}
        assert ops.sample_tokens(logits, u, **opt).tolist() == sample_by_definition(logits, u, **opt)
        assert torch.equal(ops.sample_tokens(logits, u, temperature=t), best)
    inf, nan = math.inf, math.nan
    t = torch.tensor([inf, nan, -inf, 1e30, 1.0, 1.0], device=device)
    p = torch.tensor([1.0, 1.0, 1.0, 0.5, nan, 1.0], device=device)
    m = torch.tensor([0.0, 0.0, 0.0, 0.0, 0.0, nan], device=device)
    logits[0, :1000] = -inf
    got = ops.sample_tokens(logits, u, temperature=t, top_p=p, min_p=m).tolist()
    even = 1000 + int(math.floor(float(u[0].double()) * 2001))       # 2001 weights of 1
    assert got[0] == even and got[1] == int(logits[1].argmax()) and got[2] == int(logits[2].argmax())
    plain = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0}
    assert got[4:] == sample_by_definition(logits, u, **plain)[4:]
    half = torch.sort(logits[3].double(), descending=True, stable=True).indices[:1501]
    index = torch.sort(half).values                                   # 1501 >= 0.5 * 3001
    assert got[3] == int(index[int(math.floor(float(u[3].double()) * 1501))])
    first = ops.sample_tokens(logits, torch.full_like(u, nan), **plain)
    assert torch.equal(first, ops.sample_tokens(logits, torch.zeros_like(u), **plain))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("temperature", [1e-300, 1e-310, 5e-324])
def test_sample_tokens_tiniest_temperatures(device, dtype, temperature):
    """Down to the smallest number over 0 the maximum has weight 1 and equal
    ones share: nothing else weighs anything."""
    logits = randn(5, 900, seed=103, device=device, dtype=dtype)
    logits[2, [5, 70, 800]] = logits[2].max() + 1
    for opt in (dict(), dict(top_k=20), dict(top_k=100, top_p=0.9), dict(top_p=0.9)):
        opt = {"temperature": temperature, "top_k": 0, "top_p": 1.0, "min_p": 0.0} | opt
        for r in (0.0, 0.5, 0.9999):
            got = ops.sample_tokens(logits, torch.full((5,), r, device=device), **opt)
            want = logits.double().argmax(1)
            want[2] = 70 if r == 0.5 else 800 if r > 0.5 else 5
            assert got.tolist() == want.tolist(), (opt, r)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("vocab", [44, 4619, 32128])
def test_sample_tokens_zeros_of_both_signs(device, dtype, vocab):
    """0 and -0 are equal: the lower index comes first, at every kind of border."""
    zeros = torch.where(torch.arange(vocab) % 3 == 0, -0.0, 0.0)
    levels = (randn(4, vocab, seed=104, device="cpu") * 2).round() / 2
    levels[0] = zeros
    levels[1, 5:] = zeros[5:]
    logits = levels.to(device=device, dtype=dtype)
    u = torch.tensor([0.9, 0.71, 0.93, 0.4], device=device)
    for opt in (dict(top_k=30), dict(top_k=vocab // 2), dict(top_k=vocab * 2 // 3), dict(top_p=0.517),
                dict(top_p=0.7131, top_k=vocab * 3 // 4), dict(temperature=30.0, top_p=0.517)):
        opt = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0} | opt
        assert ops.sample_tokens(logits, u, **opt).tolist() == sample_by_definition(logits, u, **opt), opt


@pytest.mark.parametrize("device", DEVICES)
def test_sample_tokens_fewer_than_top_k(device):
    """A top-k that finds fewer than it may keep leaves nothing behind for the
    nucleus: fifty weights of 1 and one of 2^-24, of which 25 * 2^-44 have to
    be in."""
    v, small = 4000, -16.635532333438686
    logits = torch.full((8, v), -math.inf, device=device)
    at = torch.arange(50, device=device) * 61 + 3
    logits[:, at] = 0.0
    logits[:, 3900] = small
    e = math.exp(float(torch.tensor(small)))
    p = (50 + 25 * 2.0 ** -44) / (50 + e)
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.99, 1 - 2.0 ** -40, 1 - 2.0 ** -41, 1.0], dtype=torch.float64, device=device)
    opt = {"temperature": 1.0, "top_k": 600, "top_p": p, "min_p": 0.0}
    got = ops.sample_tokens(logits, u, **opt).tolist()
    assert got == sample_by_definition(logits, u, **opt)
    assert got[5:] == [3900] * 3


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("vocab", [8, 9, 65543, 131071, 1 << 19])
def test_sample_tokens_vocabularies(device, vocab):
    """The smallest and largest rows, and cuts that keep a few, some thousand
    and most of a row."""
    logits = randn(2, vocab, seed=vocab % 1000, device=device).mul_(2.5).to(BF16)
    for i, o in enumerate([dict(), dict(top_k=3), dict(top_k=300), dict(top_k=600), dict(top_k=3000, top_p=0.7),
                           dict(top_k=7000, top_p=0.99), dict(top_p=0.3), dict(top_p=0.9999), dict(min_p=1e-5),
                           dict(temperature=50.0, top_p=0.95)]):
        opt = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, **o}
        u = uniform(2, 110 + i, device)
        assert ops.sample_tokens(logits, u, **opt).tolist() == sample_by_definition(logits, u, **opt), opt


@pytest.mark.parametrize("device", DEVICES)
def test_sample_tokens_follows_the_distribution(device):
    """u on an even grid: every token comes as often as its share says, to
    within one grid step at either of its two borders."""
    n = 4000
    logits = (randn(1, 50, seed=91, device=device) * 1.5)
    got = ops.sample_tokens(logits.expand(n, 50), ((torch.arange(n, dtype=torch.float64) + 0.5) / n).to(device),
                            temperature=0.8)
    share = torch.softmax(logits[0].double() / 0.8, 0).cpu()
    count = torch.bincount(got.cpu(), minlength=50)
    assert bool(((count - n * share).abs() <= 1.0 + 1e-9).all())


# --------------------------------------------------------------------------- #
# refusals                                                                    #
# --------------------------------------------------------------------------- #
@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    w = random_w4(8, 64, seed=1, device=device)
    x = randn(2, 64, seed=2, device=device, dtype=BF16)
    u8 = torch.uint8
    for codes, exps in ((w.codes.int(), w.exps), (w.codes[:, :8], w.exps), (w.codes, w.exps[:4]),
                        (w.codes[0], w.exps), (w.codes[:, :0], w.exps[:, :0])):
        with pytest.raises(ValueError):
            ops.W4Weight(codes, exps)
    with pytest.raises(ValueError):
        ops.quantize_w4(torch.zeros(4, 33))
    with pytest.raises(ValueError):
        ops.linear_w4(x[:, :32], w)
    with pytest.raises(RuntimeError):
        ops.linear_w4(x.clone().requires_grad_(), w)
    with torch.no_grad():
        ops.linear_w4(x.clone().requires_grad_(), w)

    cache = ops.KVCache8(2, 3, 100, 64, device=device)
    k = randn(2, 3, 4, 64, seed=3, device=device, dtype=BF16)
    start = torch.zeros(2, dtype=torch.int32, device=device)
    for bad in (lambda: ops.KVCache8(1, 1, 10, 48), lambda: ops.kv8_append(cache, k, k[:, :, :3], 0),
                lambda: ops.kv8_append(cache, k[:, :2], k[:, :2], 0), lambda: ops.kv8_append(cache, k[..., :32], k[..., :32], 0),
                lambda: ops.kv8_append(cache, k, k.to(FP16), 0), lambda: ops.kv8_append(cache, k, k, -1),
                lambda: ops.kv8_append(cache, k, k, 125), lambda: ops.kv8_append(cache, k, k, start[:1]),
                lambda: ops.kv8_append(cache, k, k, 0, counts=4),
                lambda: ops.KVCache8.from_tensors(cache.k, cache.v.transpose(-1, -2), cache.k_scale, cache.v_scale),
                lambda: ops.KVCache8.from_tensors(cache.k.view(u8), cache.v.view(u8), cache.k_scale, cache.v_scale),
                lambda: ops.KVCache8.from_tensors(cache.k, cache.v, cache.k_scale[:, :2], cache.v_scale)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        ops.kv8_append(cache, k.clone().requires_grad_(), k, 0)

    q = randn(2, 6, 1, 64, seed=4, device=device, dtype=BF16)
    bias, kpad = torch.zeros(1, 6, 1, 50, device=device), torch.zeros(2, 50, device=device)
    for bad in (lambda: ops.decode_attention_kv8(q[:, :5], cache, 10), lambda: ops.decode_attention_kv8(q[..., :32], cache, 10),
                lambda: ops.decode_attention_kv8(q.expand(2, 6, 2, 64), cache, 10), lambda: ops.decode_attention_kv8(q[:1], cache, 10),
                lambda: ops.decode_attention_kv8(q, cache, 129), lambda: ops.decode_attention_kv8(q, cache, -1),
                lambda: ops.decode_attention_kv8(q, cache, 10, max_len=9), lambda: ops.decode_attention_kv8(q, cache, start[:1]),
                lambda: ops.decode_attention_kv8(q, cache, 51, bias=bias), lambda: ops.decode_attention_kv8(q, cache, 51, kpad=kpad),
                lambda: ops.decode_attention_kv8(q, cache, start, bias=bias), lambda: ops.decode_attention_kv8(q, cache, 10, bias=bias[:, :3]),
                lambda: ops.decode_attention_kv8(q, cache, 10, kpad=kpad[:1])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        ops.decode_attention_kv8(q, cache, 10, bias=bias.clone().requires_grad_())

    logits, u = torch.zeros(3, 10, device=device), torch.zeros(3, device=device)
    for bad in (lambda: ops.sample_tokens(logits[0], u), lambda: ops.sample_tokens(logits, u[:2]),
                lambda: ops.sample_tokens(logits, u.to(FP16)), lambda: ops.sample_tokens(logits[:, :0], u),
                lambda: ops.sample_tokens(logits, u, temperature=-0.1), lambda: ops.sample_tokens(logits, u, temperature=math.nan),
                lambda: ops.sample_tokens(logits, u, top_p=1.1), lambda: ops.sample_tokens(logits, u, top_k=-1),
                lambda: ops.sample_tokens(logits, u, min_p=2.0), lambda: ops.sample_tokens(logits, u, top_p=u[:1]),
                lambda: ops.sample_tokens(torch.zeros(1, 2 ** 19 + 1, device=device), u[:1])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        ops.sample_tokens(logits.clone().requires_grad_(), u)
    if device == "cuda":
        for bad in (lambda: ops.linear_w4(x.float(), w), lambda: ops.linear_w4(x.cpu(), w),
                    lambda: ops.kv8_append(cache, k.float(), k.float(), 0), lambda: ops.kv8_append(cache, k.cpu(), k.cpu(), 0),
                    lambda: ops.kv8_append(cache, k, k, start.cpu()), lambda: ops.decode_attention_kv8(q.float(), cache, 1),
                    lambda: ops.decode_attention_kv8(q, cache, 1, kpad=kpad.cpu()),
                    lambda: ops.sample_tokens(logits, u.cpu()), lambda: ops.sample_tokens(logits, u, top_p=u.cpu())):
            with pytest.raises(ValueError):
                bad()
        with pytest.raises(RuntimeError):
            ops.sample_tokens(logits.double(), u)


# --------------------------------------------------------------------------- #
# together                                                                    #
# --------------------------------------------------------------------------- #
def one_step(x, wqkv, wo, head, cache, start, u, heads, d):
    """A layer's token step as a server has it: projections, cache, attention,
    vocabulary, token."""
    b = x.shape[0]
    q, k, v = ops.linear(x, wqkv).view(b, 3, heads, d).unbind(1)
    ops.kv8_append(cache, k[:, :, None], v[:, :, None], start)
    o = ops.decode_attention_kv8(q[:, :, None], cache, start + 1, scale=d ** -0.5, max_len=cache.capacity)
    logits = ops.linear(x + ops.linear(o.reshape(b, heads * d), wo), head)
    return logits, ops.sample_tokens(logits, u, temperature=0.9, top_k=40, top_p=0.95)


def step_state(b, device, seed):
    heads, d, vocab = 3, 64, 1000
    inner = heads * d
    w = [random_w4(n, inner, seed + i, device, lo=119, hi=123) for i, n in enumerate((3 * inner, inner, vocab))]
    cache = ops.KVCache8(b, heads, 150, d, device=device)
    k, v = (tokens(b, heads, 140, d, seed + 5 + j, device, BF16) for j in (0, 1))
    start = torch.randint(0, 130, (b,), generator=gen(seed + 7), dtype=torch.int32).to(device)
    ops.kv8_append(cache, k, v, 0, counts=start)
    return (randn(b, inner, seed=seed + 8, device=device, dtype=BF16), *w, cache, start, uniform(b, seed + 9, device), heads, d)


@gpu
def test_steps_in_a_graph_match_eager():
    """A token step captured into a graph, replayed with other inputs, starts
    and numbers, with eager work and synchronizations between; two graphs
    captured after each other and replayed in turn on streams of their own."""
    def state(seed):
        return step_state(5, "cuda", seed)

    graphs = []
    for seed in (200, 300):
        args = state(seed)
        one_step(*args)                                   # warm
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = one_step(*args)
        graphs.append((g, args, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(4):
        for (g, args, _), s in zip(graphs, streams):
            fresh = state(1000 + 50 * i)
            for to, of in zip(args, fresh):
                if torch.is_tensor(to):
                    to.copy_(of)
                elif isinstance(to, ops.KVCache8):
                    for name in ("k", "v", "k_scale", "v_scale"):
                        getattr(to, name).view(torch.uint8).copy_(getattr(of, name).view(torch.uint8))
                elif isinstance(to, ops.W4Weight):
                    for name in ("codes", "exps", "row_exp"):
                        getattr(to, name).copy_(getattr(of, name))
        torch.cuda.synchronize()
        for (g, _, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        want_args = state(1000 + 50 * i)
        want = one_step(*want_args)
        for _, args, out in graphs:
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
            assert torch.equal(args[4].k.view(torch.uint8), want_args[4].k.view(torch.uint8))
            assert torch.equal(args[4].v_scale, want_args[4].v_scale)


@gpu
def test_steps_on_two_streams():
    """The same work at once on two streams gives what it gives alone."""
    a, b = step_state(4, "cuda", 400), step_state(4, "cuda", 500)
    want = [one_step(*step_state(4, "cuda", s)) for s in (400, 500)]
    torch.cuda.synchronize()
    got = []
    for args in (a, b):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            got.append([one_step(*args) for _ in range(3)][-1])
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])


def test_step_on_the_cpu():
    logits, ids = one_step(*step_state(3, "cpu", 600))
    assert logits.shape == (3, 1000) and ids.shape == (3,) and bool(((ids >= 0) & (ids < 1000)).all())
