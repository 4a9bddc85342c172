"""The token-step operators where an error hides behind larger terms unless the
inputs bring it out: weights that nearly cancel, scales that lie far apart,
numbers that need 64 bits."""
import math

import pytest
import torch

from mi355 import ops

from test_token_step import (BF16, DEVICES, FP16, FP32, Plain8, gen, gpu, sample_by_definition,  # noqa: F401
                             uniform, w4_values)


# --------------------------------------------------------------------------- #
# 4-bit weights                                                               #
# --------------------------------------------------------------------------- #
# every kernel, of few rows and of many: x in LDS (of eight waves, of four), x from
# the caches (of one, two and four tiles), tiles of 128, of 64 with and without
# shared K, of 32
W4_SHAPES = [(1, 40, 96), (2, 24, 512), (8, 40, 416), (2, 16390, 96), (8, 40, 4640), (12, 40, 160), (8, 8200, 4640),
             (12, 8210, 160), (130, 8200, 96), (70, 70, 4128), (129, 2700, 128), (40, 40, 416),
             (3, 20490, 96), (12, 4200, 160), (7, 4100, 4640), (130, 11100, 96), (20, 4100, 4128)]
SPANS = [0, 20, 22, 23, 24, 30, 35, 36, 37, 38, 50, 60, 99, 101, 134]     # octaves between a row's scales


def check_group_sums(x, w, y):
    """Against 64 bits, with what fp32 sums of the terms that are there can
    lose (terms that are 0 add no error) and y's own rounding: half a step, of
    the subnormal numbers where y is one."""
    ref_w = w4_values(w.codes, w.exps)
    x64 = x.double().cpu()
    ref, size = x64 @ ref_w.t(), x64.abs() @ ref_w.abs().t()
    terms = int((x64 != 0).sum(1).max()) + 4
    info = torch.finfo(y.dtype)
    tol = info.eps / 2 * ref.abs() + terms * 2.0 ** -24 * size + info.smallest_normal * info.eps / 2
    err = (y.double().cpu() - ref).abs()
    assert bool((err <= tol).all()), (float((err / tol).max()), (err > tol).nonzero()[:5].tolist())


def far_w4(n, k, device, big, empty=False, low=120):
    """Rows whose group `big` has a scale SPANS[row] octaves over the others';
    with `empty` all codes of that group are 0 or -0."""
    g = gen(n + k)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    exps = torch.full((n, k // 32), low, dtype=torch.uint8)
    exps[:, big] = low + torch.tensor([SPANS[i % len(SPANS)] for i in range(n)], dtype=torch.uint8)
    if empty:
        codes[:, 16 * big:16 * big + 16] &= 0x88
    return ops.W4Weight(codes.to(device), exps.to(device))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,n,k", W4_SHAPES)
def test_linear_w4_small_scales_beside_large_ones(device, dtype, m, n, k):
    """What the small scales of a row contribute is there in full where the
    group of the large scale contributes nothing: its inputs are 0, or its
    codes."""
    if device == "cpu" and m * n * k > 10 ** 7:
        n = n % 509
    groups = k // 32
    for big in {0, groups - 1}:
        x = torch.randn(m, k, generator=gen(m)).to(device, dtype)
        w = far_w4(n, k, device, big, empty=True)
        check_group_sums(x, w, ops.linear_w4(x, w))
        w = far_w4(n, k, device, big)
        x[:, 32 * big:32 * big + 32] = 0
        check_group_sums(x, w, ops.linear_w4(x, w))
        # one group alone
        only = torch.zeros_like(x)
        at = 32 * ((big + 1) % groups)
        only[:, at:at + 32] = x[:, at:at + 32]
        check_group_sums(only, w, ops.linear_w4(only, w))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_linear_w4_each_distance(device, dtype):
    """Rows with a scale for every distance from 0 to 130 octaves, x in one
    group at a time; dense x; an infinity in the group of the smallest scale."""
    k = 32 * 131
    codes = torch.randint(0, 256, (6, k // 2), generator=gen(1), dtype=torch.uint8)
    exps = torch.stack([torch.arange(131).flip(0) + 100, torch.arange(131) + 5,
                        torch.randperm(131, generator=gen(2)) + 110, torch.full((131,), 121),
                        torch.arange(131) % 37 + 100, torch.arange(131) % 38 + 100]).to(torch.uint8)
    w = ops.W4Weight(codes.to(device), exps.to(device))
    x = torch.randn(131, k, generator=gen(3)) * torch.eye(131).repeat_interleave(32, 1)
    if dtype == FP16:
        # outputs stay in range where x * scale does
        x = torch.where(x.abs() * 200 * 2.0 ** (exps.amax(0).float() - 127).repeat_interleave(32) < 60000, x, 0.0)
    x = x.to(device, dtype)
    y = ops.linear_w4(x, w)
    check_group_sums(x, w, y)
    for rows in (1, 7, 16, 40):
        check_group_sums(x[:rows], w, ops.linear_w4(x[:rows], w))
        check_group_sums(x[-rows:], w, ops.linear_w4(x[-rows:], w))
    dense = torch.randn(3, k, generator=gen(4)).to(device, BF16)
    check_group_sums(dense, w, ops.linear_w4(dense, w))
    ones = ops.W4Weight(torch.full_like(w.codes, 0x22), w.exps)
    x = torch.zeros(2, k, device=device, dtype=dtype)
    x[0, k - 5] = math.inf
    x[1, 3] = -math.inf
    y = ops.linear_w4(x, ones)
    assert bool((y[0] == math.inf).all()) and bool((y[1] == -math.inf).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("span", [25, 26, 27, 28])
def test_linear_w4_where_rows_are_summed_by_groups(device, dtype, span):
    """On both sides of the border, all groups of one row alike."""
    k = 160
    w = ops.W4Weight(*(t.to(device) for t in (
        torch.randint(0, 256, (300, k // 2), generator=gen(span), dtype=torch.uint8),
        torch.tensor([120, 120 + span, 121, 120 + span // 2, 120], dtype=torch.uint8).repeat(300, 1))))
    assert bool((w.row_exp == (255 if span > 26 else 120 + span)).all())
    x = torch.randn(140, k, generator=gen(5)).to(device, dtype)
    for keep in ((0,), (4,), (0, 4), (2, 4), (3,), (0, 2, 3, 4)):
        part = torch.zeros_like(x)
        for at in keep:
            part[:, 32 * at:32 * at + 32] = x[:, 32 * at:32 * at + 32]
        if dtype == FP16 and 3 in keep:
            part = part / 4
        for rows in (1, 9, 17, 140):
            check_group_sums(part[:rows], w, ops.linear_w4(part[:rows], w))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,n,k", W4_SHAPES)
def test_linear_w4_no_scale(device, dtype, m, n, k):
    """An exponent byte of 255, over codes of 0 as well, makes its own row's
    outputs not finite and no other's."""
    if device == "cpu" and m * n * k > 10 ** 7:
        n = n % 509
    codes = torch.full((n, k // 2), 0x22, dtype=torch.uint8)
    exps = torch.full((n, k // 32), 127, dtype=torch.uint8)
    codes[3], exps[3, k // 32 - 1] = 0, 255
    exps[n - 1, 0] = 255
    y = ops.linear_w4(torch.ones(m, k, device=device, dtype=dtype), ops.W4Weight(codes.to(device), exps.to(device)))
    bad = torch.zeros(n, dtype=torch.bool)
    bad[[3, n - 1]] = True
    assert torch.equal(~y.isfinite().cpu(), bad.expand(m, n))
    assert bool((y.cpu()[:, ~bad].double() == torch.tensor(float(k)).to(dtype).double()).all())


def test_w4_weight_loads_and_slices():
    """What is made from the exponents follows a load, and slices share it."""
    a, b = far_w4(30, 96, "cpu", 0), far_w4(30, 96, "cpu", 2, empty=True)
    before = a.row_exp.clone()
    state = b.state_dict()
    state["row_exp"] = torch.zeros_like(state["row_exp"])           # as if another rule had made it
    a.load_state_dict(state)
    assert torch.equal(a.row_exp, b.row_exp) and not torch.equal(a.row_exp, before)
    part = b.rows(7, 20)
    assert part.shape == (13, 96) and torch.equal(part.row_exp, b.row_exp[7:20])
    for name in ("codes", "exps"):
        assert getattr(part, name).data_ptr() == getattr(b, name)[7:].data_ptr()


@pytest.mark.parametrize("octaves", [-110, -80, -60, 50, 70, 100, 120])
def test_quantize_w4_at_any_size(octaves):
    """Weights that are a power of two larger or smaller get the same codes, and
    exponents that far apart: the better of two scales is found where the squares
    of its errors are over or under fp32's range too."""
    weight = torch.randn(64, 256, generator=gen(7)).clamp(-6, 6)
    w, far = ops.quantize_w4(weight), ops.quantize_w4(weight * 2.0 ** octaves)
    assert torch.equal(far.codes, w.codes) and torch.equal(far.exps.int(), w.exps.int() + octaves)


def test_quantize_w4_refuses_what_32_bits_do_not_hold():
    for bad in (1e39, -1e300):
        weight = torch.zeros(2, 32, dtype=torch.float64)
        weight[1, 5] = bad
        with pytest.raises(ValueError):
            ops.quantize_w4(weight)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n,k", [(1, 32), (5, 64), (300, 96), (67, 2048), (9, 4640), (130, 4128)])
def test_w4_row_exponents(device, n, k):
    """Each row's largest exponent of groups with codes other than 0 and -0; 255
    where two of those lie over 26 apart or a byte is 255.  Codes and exponents
    that begin at any byte."""
    g = gen(n + k)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8).view(n, k // 32, 16)
    codes[torch.rand(n, k // 32, generator=g) < 0.5] &= 0x88
    codes[0] &= 0x88
    width = torch.randint(1, 40, (n, 1), generator=g)
    exps = (torch.rand(n, k // 32, generator=g) * width).to(torch.uint8) + torch.randint(0, 210, (n, 1), generator=g, dtype=torch.uint8)
    exps[torch.rand(n, k // 32, generator=g) < 0.3 / n] = 255
    want = []
    for c, e in zip(codes, exps.tolist()):
        have = [x for x, group in zip(e, c) if bool((group & 0x77).any())]
        far = 255 in e or (have and max(have) - min(have) > 26)
        want.append(255 if far else max(have, default=0))
    codes = codes.view(n, k // 2)
    assert ops.W4Weight(codes.to(device), exps.to(device)).row_exp.tolist() == want
    if device == "cuda":
        for off in (1, 4, 7):
            c, e = (torch.zeros(t.numel() + off, dtype=torch.uint8, device=device) for t in (codes, exps))
            c[off:], e[off:] = codes.reshape(-1).to(device), exps.reshape(-1).to(device)
            assert ops.W4Weight(c[off:].view(n, k // 2), e[off:].view(n, k // 32)).row_exp.tolist() == want


def test_w4_weight_leaves_a_loaded_state_alone():
    """A load, an assigning one too, writes nothing into what it was given."""
    for assign in (False, True):
        a, b = far_w4(30, 96, "cpu", 0), far_w4(30, 96, "cpu", 2, empty=True)
        state = {k: v.clone() for k, v in b.state_dict().items()}
        state["row_exp"].zero_()
        at = a.row_exp.data_ptr()
        a.load_state_dict(state, assign=assign)
        assert torch.equal(a.row_exp, b.row_exp) and not bool(state["row_exp"].any())
        assert assign or a.row_exp.data_ptr() == at                  # a captured graph reads it there


# --------------------------------------------------------------------------- #
# attention over the 8-bit cache                                              #
# --------------------------------------------------------------------------- #
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("grp", [1, 2, 3, 8, 16])
@pytest.mark.parametrize("d,length,at", [(64, 2, (0, 1)), (32, 70, (66, 3)), (128, 200, (17, 190)),
                                         (64, 2100, (2099, 40))])
def test_decode_attention_kv8_weights_have_32_bits(device, dtype, grp, d, length, at):
    """Two tokens with values 1 and -1 and nearly equal weights: the output is
    the small difference of the two, so an error of the weights shows.

    Scores are the bias alone (keys are 0), 0 and -x with x under 2^-6.  In 32
    bits exp(-x) is off by under 2^-23 (a step of the exponential, and 2^-24 x of
    its argument), o = (1 - e^-x) / (1 + e^-x) by half of that, by some steps of
    2^-24 for its sums and by its own rounding: 2^-20 beside half a step of o.
    Weights of 16 significant bits are off by up to 2^-17, o by up to 2^-18."""
    b, h = 2, 3
    cache = ops.KVCache8(b, h, length, d)
    v = torch.zeros(b, h, cache.capacity, d)
    v[:, :, at[0]], v[:, :, at[1]] = 1.0, -1.0
    cache.v.copy_(v.view(b, h, -1, 64, d).transpose(-1, -2))
    cache.v_scale.fill_(1.0)
    cache = ops.KVCache8.from_tensors(*(t.to(device) for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)))
    x = 2.0 ** (-10 + 4 * torch.rand(b, h * grp, generator=gen(grp)))
    bias = torch.zeros(b, h * grp, 1, length)
    bias[:, :, 0, at[1]] = -x
    kpad = torch.full((b, length), -math.inf)
    kpad[:, list(at)] = 0.0
    q = torch.ones(b, h * grp, 1, d, device=device, dtype=dtype)
    out = ops.decode_attention_kv8(q, cache, length, bias=bias.to(device), kpad=kpad.to(device))
    want = torch.tanh(x.double() / 2)[:, :, None, None]              # (1 - e^-x) / (1 + e^-x)
    err = (out.double().cpu() - want).abs()
    tol = torch.finfo(dtype).eps / 2 * want + 2.0 ** -20
    assert bool((err <= tol).all()), float((err / tol).max())


# --------------------------------------------------------------------------- #
# append to the 8-bit cache                                                   #
# --------------------------------------------------------------------------- #
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_kv8_append_one_grows_at_every_offset(device, dtype, d):
    """One token at each position of a block, larger than all before it: the
    old codes follow the new scale, the new code is there, and the codes behind
    it keep their bytes, whichever of a word's bytes it takes."""
    b, h = 64, 3
    cache, plain = ops.KVCache8(b, h, 64, d, device=device), Plain8(b, h, 64, d)
    old, new = (torch.randn(2, b, h, 64, d, generator=gen(j)).to(device, dtype) for j in (1, 2))
    new = new[:, :, :, :1] * 40
    ops.kv8_append(cache, old[0], old[1], 0)
    plain.append(old[0], old[1], 0)
    before = cache.k_scale.clone(), cache.v_scale.clone()
    start = torch.arange(b, dtype=torch.int32, device=device)
    ops.kv8_append(cache, new[0], new[1], start)
    plain.append(new[0], new[1], start)
    plain.same(cache)
    assert bool((cache.k_scale > before[0]).all()) and bool((cache.v_scale > before[1]).all())


# --------------------------------------------------------------------------- #
# sampling                                                                    #
# --------------------------------------------------------------------------- #
@pytest.mark.parametrize("device", DEVICES)
def test_sample_tokens_options_of_64_bits(device):
    """A row's options in 64 bits are those numbers, as one number for all rows
    is: 0.3 of ten equal weights is three of them, and what fp32 makes of it four."""
    logits = torch.zeros(4, 10, device=device)
    u = torch.full((4,), 0.9999, device=device)
    p = torch.full((4,), 0.3, dtype=torch.float64, device=device)
    assert ops.sample_tokens(logits, u, top_p=0.3).tolist() == [2] * 4
    assert ops.sample_tokens(logits, u, top_p=p).tolist() == [2] * 4
    assert ops.sample_tokens(logits, u, top_p=p.float()).tolist() == [3] * 4
    g = gen(31)
    logits = (torch.randn(40, 3001, generator=g) * 3).to(device)
    u = uniform(40, 32, device, torch.float64)
    r = torch.rand(3, 40, generator=g, dtype=torch.float64).to(device)
    opt = dict(temperature=0.3 + r[0], top_k=0, top_p=1 - 0.3 * r[1], min_p=0.05 * r[2])
    assert ops.sample_tokens(logits, u, **opt).tolist() == sample_by_definition(logits, u, **opt)
    rows = dict(opt, temperature=opt["temperature"].float(), top_p=opt["top_p"][:1].expand(40))
    assert ops.sample_tokens(logits, u, **rows).tolist() == sample_by_definition(logits, u, **rows)


# --------------------------------------------------------------------------- #
# whole numbers of another type                                               #
# --------------------------------------------------------------------------- #
@pytest.mark.parametrize("device", DEVICES)
def test_whole_numbers_of_64_bits_keep_their_value(device):
    """Positions, counts, lengths and top-k of int64 mean what they say: none is
    taken modulo 2^32."""
    def whole(*v):
        return torch.tensor(v, dtype=torch.int64, device=device)

    b, h, d, s = 5, 2, 64, 70
    k, v = (torch.randn(2, b, h, s, d, generator=gen(41)).to(device, BF16))
    start, counts = whole(2 ** 32, -2 ** 32 - 1, 2 ** 33 + 5, 3, 60), whole(4, 4, 4, 2 ** 32 + 1, -2 ** 33)
    cache, plain = ops.KVCache8(b, h, 256, d, device=device), Plain8(b, h, 256, d)
    ops.kv8_append(cache, k, v, start, counts)
    plain.append(k, v, start, counts)
    plain.same(cache)
    one, plain1 = ops.KVCache8(b, h, 256, d, device=device), Plain8(b, h, 256, d)
    ops.kv8_append(one, k[:, :, :1], v[:, :, :1], start)
    plain1.append(k[:, :, :1], v[:, :, :1], start)
    plain1.same(one)
    q = torch.randn(b, h, 1, d, generator=gen(42)).to(device, BF16)
    ops.kv8_append(cache, k, v, 0)
    got = ops.decode_attention_kv8(q, cache, whole(2 ** 32, 2 ** 40 + 3, -2 ** 32 + 9, 3, 70), max_len=70)
    want = ops.decode_attention_kv8(q, cache, torch.tensor([70, 70, 0, 3, 70], dtype=torch.int32, device=device), max_len=70)
    assert torch.equal(got, want)
    logits, u = torch.randn(5, 1000, generator=gen(43)).to(device), torch.full((5,), 0.97, device=device)
    every = ops.sample_tokens(logits, u, temperature=3.0)
    assert torch.equal(ops.sample_tokens(logits, u, temperature=3.0, top_k=whole(2 ** 32 + 1, 2 ** 62, 0, -2 ** 32 + 1, 10 ** 6)), every)
    for top_k in (torch.tensor([1e12, 2.0 ** 31, math.inf, 0.0, -1e12], device=device), whole(0, 0, 0, 0, 0).to(torch.uint8)):
        assert torch.equal(ops.sample_tokens(logits, u, temperature=3.0, top_k=top_k), every)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [FP32, FP16, torch.float64, torch.bool])
def test_positions_that_are_no_whole_numbers_are_refused(device, dtype):
    cache = ops.KVCache8(2, 3, 100, 64, device=device)
    k = torch.randn(2, 3, 4, 64, generator=gen(44)).to(device, BF16)
    at = torch.ones(2, dtype=dtype, device=device)
    for bad in (lambda: ops.kv8_append(cache, k, k, at), lambda: ops.kv8_append(cache, k, k, 0, counts=at),
                lambda: ops.decode_attention_kv8(k[:, :, :1], cache, at)):
        with pytest.raises(ValueError):
            bad()


# --------------------------------------------------------------------------- #
# sizes over what a launch can have                                           #
# --------------------------------------------------------------------------- #
@gpu
def test_more_workgroups_than_a_launch_has_are_refused():
    """A launch has fewer than 2^32 threads: as many rows, heads and tokens as
    would take more are refused before anything runs."""
    def wide(*shape, dtype=BF16):
        return torch.zeros([1] * len(shape), dtype=dtype, device="cuda").expand(shape)

    n = 1 << 22                                          # rows of 1024 threads
    with pytest.raises(ValueError):
        ops.sample_tokens(wide(n, 8), wide(n, dtype=FP32))
    n = 1 << 29                                          # 32 rows for 256 threads
    w = ops.quantize_w4(torch.zeros(1, 32, device="cuda"))
    with pytest.raises(ValueError):
        ops.linear_w4(torch.zeros(32, dtype=BF16, device="cuda").expand(n, 32), w)
    start = torch.zeros(1, dtype=torch.int32, device="cuda")
    for heads, tokens in ((1 << 26, 1), (1 << 23, 2)):   # four heads, and half a head, for 256 threads
        cache = ops.KVCache8(1, heads, 0, 32, device="cuda")
        k = torch.zeros(32, dtype=BF16, device="cuda").expand(1, heads, tokens, 32)
        with pytest.raises(ValueError):
            ops.kv8_append(cache, k, k, start)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,n,k", [(1, 20480, 992), (8, 20479, 736), (1, 20480, 1024), (9, 4096, 288), (16, 4097, 288),
                                   (13, 8192, 288), (13, 8193, 288), (65, 16384, 96), (65, 16385, 96), (64, 32800, 64),
                                   (33, 8256, 96), (33, 8192, 96), (32, 8256, 96), (128, 4096, 4096), (129, 2752, 4096),
                                   (17, 8192, 4096)])
def test_linear_w4_where_one_kernel_follows_another(device, dtype, m, n, k):
    """Sizes at which another kernel takes over."""
    if device == "cpu" and m * n * k > 10 ** 8:
        n = n % 1021
    codes = torch.randint(0, 256, (n, k // 2), generator=gen(m + n), dtype=torch.uint8)
    exps = torch.randint(117, 124, (n, k // 32), generator=gen(k), dtype=torch.uint8)
    w = ops.W4Weight(codes.to(device), exps.to(device))
    x = torch.randn(m, k, generator=gen(51)).to(device, dtype)
    check_group_sums(x, w, ops.linear_w4(x, w))
