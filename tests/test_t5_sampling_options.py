"""Sampling options of generate()."""
import pytest
import torch

from test_t5_token_step import DEVICES, gpu, model, prompt, seeded  # noqa: F401


@pytest.mark.parametrize("device", DEVICES)
def test_options_of_none_are_off(device):
    """A caller that hands its configuration on passes None for what is not set."""
    m, (ids, mask) = model(device), prompt(device, pad=True)

    def call(**options):
        return m.generate(input_ids=ids, attention_mask=mask, max_new_tokens=6, min_new_tokens=6,
                          generator=seeded(device, 4), **options)

    off = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    want = call(do_sample=True, **off)
    assert torch.equal(call(do_sample=True, **dict.fromkeys(off)), want)
    for name in off:
        assert torch.equal(call(do_sample=True, **{**off, name: None}), want)
    greedy = call()
    assert torch.equal(call(do_sample=None, **dict.fromkeys(off)), greedy)
    with pytest.raises(ValueError):
        call(do_sample=True, top_k=-1)
