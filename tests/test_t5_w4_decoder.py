"""quantize_decoder_w4() of models that cannot be held in 4 bits."""
import pytest
import torch

from mi355 import ops

from test_t5_token_step import DEVICES, model, prompt


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("where", ["first", "last"])
def test_a_refused_quantization_leaves_the_model_as_it_was(device, where):
    m, ids = model(device), prompt(device)[0]
    want = m.generate(input_ids=ids, max_new_tokens=4, min_new_tokens=4)
    lin = m.lm_head if where == "first" else m.decoder.block[-1].layer[2].DenseReluDense.wo
    was = float(lin.weight.detach()[3, 5])
    with torch.no_grad():
        lin.weight[3, 5] = float("nan")
    with pytest.raises(ValueError):
        m.quantize_decoder_w4()
    assert not any(isinstance(x, ops.W4Weight) for x in m.modules())
    with torch.no_grad():
        lin.weight[3, 5] = was
    assert torch.equal(m.generate(input_ids=ids, max_new_tokens=4, min_new_tokens=4), want)
    m.quantize_decoder_w4()
    assert isinstance(lin.weight, ops.W4Weight)
