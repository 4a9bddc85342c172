"""The captured decode loop of generate() follows what became of the model since
the capture."""
import copy
import threading

import pytest
import torch

from test_t5_token_step import gpu, model, prompt, seeded


def both(m, **options):
    """Tokens of the captured loop and of the eager one."""
    ids, mask = prompt("cuda", pad=True)
    out = [m.generate(input_ids=ids, attention_mask=mask, max_new_tokens=9, min_new_tokens=9, use_graph=g,
                      generator=seeded("cuda", 2), **options) for g in (True, False)]
    torch.cuda.synchronize()
    assert not getattr(m, "_gen_graph_warned", False)
    return out


def churn():
    """Eager work that takes freed memory and fills it."""
    for n in (64, 4096, 1 << 16, 1 << 20):
        for _ in range(20):
            torch.randn(n, device="cuda")


@gpu
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("options", [dict(), dict(kv_cache_dtype="fp8", do_sample=True, temperature=2.0)])
def test_captured_loop_after_weights_moved(quantized, options):
    m = model("cuda")
    if quantized:
        m.quantize_decoder_w4()
    other = model("cuda", seed=9)
    if quantized:
        other.quantize_decoder_w4()

    def assign():
        m.load_state_dict(copy.deepcopy(other.state_dict()), assign=True)

    for change in (lambda: None, m.half, lambda: m.to("cpu").to("cuda"), m.bfloat16, assign):
        change()
        churn()
        assert torch.equal(*both(m, **options))
        churn()
        assert torch.equal(*both(m, **options))


@gpu
def test_captured_loop_after_tokens_of_the_config_changed():
    m = model("cuda")
    for start in (m.config.decoder_start_token_id, 17, 400):
        m.config.decoder_start_token_id = start
        assert torch.equal(*both(m))
    # every token banned but by the mask of the sampler: rows without a logit
    with torch.no_grad():
        m.lm_head.weight.fill_(float("nan"))
    for pad in (m.config.pad_token_id, 5):
        m.config.pad_token_id = pad
        out = both(m, do_sample=True)
        assert torch.equal(*out) and bool((out[0] == pad).all())


@gpu
def test_captured_loop_keeps_its_graph():
    """Weights that are written in place do not cost a new capture."""
    m = model("cuda")
    both(m)
    state = m._gen_graph
    with torch.no_grad():
        for w in m.parameters():
            w.mul_(1.01)
    assert torch.equal(*both(m)) and m._gen_graph is state


@gpu
@pytest.mark.parametrize("options", [dict(), dict(kv_cache_dtype="fp8")])
def test_captured_loop_follows_the_position_bias(options):
    """The bias of the relative positions is the present one, not that of the
    capture."""
    m = model("cuda")
    assert torch.equal(*both(m, **options))
    state = m._gen_graph
    weight = m.decoder.block[0].layer[0].SelfAttention.relative_attention_bias.weight
    before = both(m, **options)[0]
    for seed in (3, 4):
        with torch.no_grad():
            weight.copy_(torch.randn(weight.shape, generator=torch.Generator().manual_seed(seed)) * 30)
        out = both(m, **options)
        assert torch.equal(*out) and not torch.equal(out[0], before)
    assert m._gen_graph is state


@gpu
@pytest.mark.parametrize("options", [dict(), dict(kv_cache_dtype="fp8", do_sample=True, temperature=2.0)])
@pytest.mark.parametrize("threads", [False, True])
def test_captured_loop_on_streams_and_threads(options, threads):
    """Calls on streams of their own, and from threads, without a
    synchronization between: each gives the tokens of its own prompt."""
    m = model("cuda")
    ids = torch.randint(2, 512, (6, 3, 12), generator=torch.Generator().manual_seed(8)).cuda()
    streams = [torch.cuda.Stream() for _ in range(3)]

    def call(i, use_graph):
        return m.generate(input_ids=ids[i], max_new_tokens=40, min_new_tokens=40, use_graph=use_graph,
                          generator=seeded("cuda", i), **options)

    want = [call(i, False) for i in range(6)]
    call(0, True)
    torch.cuda.synchronize()
    got = [[] for _ in range(6)]

    def run(i):
        with torch.cuda.stream(streams[i % 3]):
            for _ in range(4):
                got[i].append(call(i, True))

    if threads:
        workers = [threading.Thread(target=run, args=(i,)) for i in range(6)]
        for w in workers:
            w.start()
        for w in workers:
            w.join()
    else:
        for i in range(6):
            run(i)
    torch.cuda.synchronize()
    assert all(len(g) == 4 and torch.equal(x, w) for g, w in zip(got, want) for x in g)
    assert not getattr(m, "_gen_graph_warned", False)
