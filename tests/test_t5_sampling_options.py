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


@gpu
@pytest.mark.parametrize("cache", [None, "fp8"])
def test_other_options_replay_the_same_graph(cache):
    """Each call has its own options, without a new capture, and the tokens of
    the eager loop, which has them as numbers of 64 bits."""
    m, (ids, mask) = model("cuda"), prompt("cuda", pad=True)
    state = None
    for i, options in enumerate([dict(temperature=0.7, top_k=50, top_p=0.95), dict(temperature=1.3, top_k=0),
                                 dict(temperature=0.0), dict(temperature=2.1, top_k=10 ** 12, top_p=0.9, min_p=0.01),
                                 dict(top_k=3), dict(top_k=None, min_p=1.0), dict(temperature=1e-300),
                                 dict(temperature=0.7, top_k=50, top_p=0.95)]):
        calls = [m.generate(input_ids=ids, attention_mask=mask, max_new_tokens=20, min_new_tokens=20, use_graph=g,
                            do_sample=True, generator=seeded("cuda", i), kv_cache_dtype=cache, **options)
                 for g in (True, False, True)]
        torch.cuda.synchronize()
        assert torch.equal(calls[0], calls[1]) and torch.equal(calls[2], calls[1]), options
        assert state is None or m._gen_graph is state
        state = m._gen_graph
    assert not getattr(m, "_gen_graph_warned", False)
    m.generate(input_ids=ids, attention_mask=mask, max_new_tokens=20, min_new_tokens=20, kv_cache_dtype=cache)
    assert m._gen_graph is not state                                 # greedy is another loop
