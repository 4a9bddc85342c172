"""The token-step operators where an error hides behind larger terms unless the
inputs bring it out: weights that nearly cancel, scales that lie far apart,
numbers that need 64 bits."""
import math

import pytest
import torch

from mi355 import ops

from test_token_step import BF16, DEVICES, FP16, FP32, Plain8, gen, gpu  # noqa: F401


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
