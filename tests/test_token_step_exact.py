"""The token-step operators where an error hides behind larger terms unless the
inputs bring it out: weights that nearly cancel, scales that lie far apart,
numbers that need 64 bits."""
import math

import pytest
import torch

from mi355 import ops

from test_token_step import BF16, DEVICES, FP16, FP32, gen, gpu  # noqa: F401


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
