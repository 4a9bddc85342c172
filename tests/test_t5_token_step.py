"""The token-step operators on T5's own paths: generate() with sampling, with
8-bit caches, with 4-bit decoder weights."""
import pytest
import torch

from mi355 import ops
from mi355.models.t5.configuration import t5_config
from mi355.models.t5.modeling import T5ForConditionalGeneration
from mi355.ops import torch_ref

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]


def model(device, seed=0):
    torch.manual_seed(seed)
    cfg = t5_config("flan-t5-small", num_layers=2, num_decoder_layers=2, d_model=128, d_ff=256,
                    num_heads=2, d_kv=64, vocab_size=512, dropout_rate=0.0)
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    return T5ForConditionalGeneration(cfg).to(device, dtype).eval()


def prompt(device, b=3, s=12, pad=False):
    ids = torch.randint(2, 512, (b, s), generator=torch.Generator().manual_seed(1)).to(device)
    mask = torch.ones_like(ids)
    if pad:
        mask[0, 7:] = 0
        mask[2, 2:] = 0
    return ids, mask


def seeded(device, seed):
    return torch.Generator(device=device).manual_seed(seed)


@pytest.mark.parametrize("device", DEVICES)
def test_sampling_in_generate(device):
    m = model(device)
    ids, mask = prompt(device, pad=True)
    call = lambda **k: m.generate(input_ids=ids, attention_mask=mask, max_new_tokens=9, min_new_tokens=9, **k)  # noqa: E731
    greedy = call()
    # one token left is the greedy one, however it is cut
    for cut in (dict(top_k=1), dict(temperature=0.0), dict(top_p=0.0), dict(min_p=1.0)):
        assert torch.equal(call(do_sample=True, **cut), greedy), cut
    # options without do_sample change nothing, as before
    assert torch.equal(call(temperature=5.0, top_k=3), greedy)
    a, b = (call(do_sample=True, temperature=3.0, generator=seeded(device, s)) for s in (5, 5))
    c = call(do_sample=True, temperature=3.0, generator=seeded(device, 6))
    assert torch.equal(a, b) and not torch.equal(a, c)
    assert bool(((a >= 0) & (a < 512)).all()) and not bool((a == m.config.eos_token_id).any())
    with pytest.raises(ValueError):
        call(do_sample=True, top_p=1.5)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("static", [False, True])
def test_attention_over_8_bit_cache(device, static):
    """The layer's output is attention over what the cache holds."""
    m = model(device)
    att = m.decoder.block[0].layer[1 if static else 0]
    att = att.EncDecAttention if static else att.SelfAttention
    dt = m.shared.weight.dtype
    h, d = 2, 64
    cache = ops.KVCache8(2, h, 20, d, device=device)
    state = {"kv8": cache, "len": 0}
    g = torch.Generator().manual_seed(3)
    if static:
        kv = torch.randn(2, 2, h, 17, d, generator=g).to(device, dt)
        ops.kv8_append(cache, kv[0], kv[1], 0)
        state.update(len=17, static=True)
    bias = None if static else torch.randn(1, h, 1, 20, generator=g).to(device)
    kpad = torch.zeros(2, 17, device=device)
    kpad[1, 5:] = -1e9
    with torch.no_grad():
        for t in range(4):
            x = torch.randn(2, 1, 128, generator=g).to(device, dt)
            out = att(x, position_bias=bias, kpad=kpad if static else None, kv_cache=state)
            n = state["len"]
            assert n == (17 if static else t + 1)
            k, v = (c[:, :, :n] for c in cache.dequantize())
            q = att._shape(att.q(x), 2)
            want = torch_ref.attention(q.float(), k, v, bias=None if static else bias[..., :n],
                                       kpad=kpad if static else None).to(dt)
            want = att.o(want.transpose(1, 2).reshape(2, 1, h * d))
            # two ways to the same attention: its rounding to dt (half a step,
            # of either) carried through a product of h*d = 128 summands, and the
            # product's own rounding
            size = want.new_tensor(1.0).double() * (v.abs().amax().double() * att.o.weight.double().abs().sum(1).max())
            step = torch.finfo(dt).eps
            assert float((out.double() - want.double()).abs().max()) <= float(step * (size + want.double().abs().max())) + 1e-4 * float(size)


@pytest.mark.parametrize("device", DEVICES)
def test_generate_with_8_bit_cache(device):
    m = model(device)
    ids, mask = prompt(device, pad=True)
    out = m.generate(input_ids=ids, attention_mask=mask, max_new_tokens=70, min_new_tokens=70, kv_cache_dtype="fp8")
    assert out.shape == (3, 70) and bool(((out >= 0) & (out < 512)).all())
    if device == "cpu":
        # padding is not there: the same rows without it (on a GPU the
        # encoder's products of another size round otherwise)
        alone = m.generate(input_ids=ids[:1, :7], max_new_tokens=3, min_new_tokens=3, kv_cache_dtype="fp8")
        assert torch.equal(alone, out[:1, :3])
    with pytest.raises(ValueError):
        m.generate(input_ids=ids, max_new_tokens=2, kv_cache_dtype="int3")


@pytest.mark.parametrize("device", DEVICES)
def test_decoder_in_4_bits(device):
    """Every token comes from the weights that the codes stand for: a model
    that holds those values in its own type generates the same."""
    m = model(device)
    twin = model(device)
    m.quantize_decoder_w4()
    assert m.quantize_decoder_w4() is m
    held = 0
    for name, a in m.named_modules():
        if isinstance(a, ops.W4Weight):
            twin.get_parameter(name).data.copy_(a.dequantize(twin.shared.weight.dtype))
            held += 1
    assert held == 2 * 6 + 1
    ids, mask = prompt(device, pad=True)
    with torch.no_grad():
        a = m(input_ids=ids, attention_mask=mask, decoder_input_ids=ids).logits
        b = twin(input_ids=ids, attention_mask=mask, decoder_input_ids=ids).logits
    # the same products in another order of fp32 sums; where a sum falls next to
    # a rounding border of dt it is a step apart, and a few layers of 128 to
    # 256 summands carry that on: 8 steps of the largest logit
    tol = (8 * torch.finfo(a.dtype).eps if a.dtype != torch.float32 else 1e-4) * float(b.abs().max())
    assert float((a - b).abs().max()) <= tol
    out = m.generate(input_ids=ids, attention_mask=mask, max_new_tokens=6, min_new_tokens=6,
                     kv_cache_dtype="fp8", do_sample=True, generator=seeded(device, 3))
    assert out.shape == (3, 6)
    with pytest.raises(RuntimeError):
        m.save_pretrained("/tmp/never")
    m.train()
    with pytest.raises(RuntimeError):
        m(input_ids=ids, labels=ids)


@gpu
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("options", [dict(), dict(kv_cache_dtype="fp8"), dict(do_sample=True, temperature=1.5, top_p=0.9),
                                     dict(do_sample=True, top_k=20, kv_cache_dtype="fp8")])
def test_captured_loop_matches_eager(quantized, options):
    """The graph of the whole loop, replayed for other prompts, masks and
    numbers with eager work between, gives the eager tokens each time."""
    m = model("cuda")
    if quantized:
        m.quantize_decoder_w4()
    for seed in (1, 2, 3, 4):
        ids = torch.randint(2, 512, (3, 12), generator=torch.Generator().manual_seed(seed)).cuda()
        mask = torch.ones_like(ids)
        mask[seed % 3, 3 + seed:] = 0
        calls = [m.generate(input_ids=ids, attention_mask=mask, max_new_tokens=67, min_new_tokens=67, use_graph=g,
                            generator=seeded("cuda", seed), **options) for g in (True, False)]
        torch.cuda.synchronize()
        assert torch.equal(*calls), seed
        junk = [torch.randn(512, 512, device="cuda") for _ in range(8)]     # eager work that reuses freed memory
        del junk
    assert not getattr(m, "_gen_graph_warned", False) and m._gen_graph is not None


@pytest.mark.parametrize("device", DEVICES)
def test_w4_decoder_with_dropout(device):
    """In training mode without gradients the 4-bit decoder drops out like any
    other; with gradients it is refused."""
    m = model(device)
    m.quantize_decoder_w4()
    for mod in m.modules():
        if hasattr(mod, "dropout") and isinstance(mod.dropout, torch.nn.Dropout):
            mod.dropout.p = 0.1
    m.train()
    ids, mask = prompt(device)
    out = m.generate(input_ids=ids, attention_mask=mask, max_new_tokens=4, min_new_tokens=4)
    assert out.shape == (3, 4)
    with torch.no_grad():
        loss = m(input_ids=ids, attention_mask=mask, labels=ids).loss
    assert bool(loss.isfinite())
    with pytest.raises(RuntimeError):
        m(input_ids=ids, attention_mask=mask, labels=ids)
