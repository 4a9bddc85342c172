"""Measured cases of the token-step operators: what one generated token costs a
served language model, in a plain torch form and through ``mi355.ops``.

Four operators, told apart by a case's ``"op"``:

* ``sample``  - one token per row of logits from given uniform numbers, with
  temperature, top-k, top-p and min-p (``ops.sample_tokens``);
* ``append``  - new keys and values into a cache held in 8 bits, with a scale
  for each block of 64 tokens and head (``ops.kv8_append``);
* ``step``    - one decode step of a layer on that cache: append one token,
  attend over it (``ops.kv8_append`` + ``ops.decode_attention_kv8``);
* ``w4``      - products of a few rows with 4-bit weights that carry a scale
  for each group of 32 inputs (``ops.linear_w4``).

``run`` computes the plain form unless ``own`` is set.
"""
import math

import torch

own = False

BLOCK = 64          # tokens that share a scale in the cache
GROUP = 32          # inputs that share a scale in a 4-bit weight
E_MIN, E_MAX = -120, 120   # exponents of a cache scale
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# --------------------------------------------------------------------------- #
# cases                                                                       #
# --------------------------------------------------------------------------- #
def listed():
    return [
        # a single chat request: one row over the T5 vocabulary, one set of
        # sampling options for the call
        {"name": "sample_1_row", "op": "sample", "dtype": "bf16", "rows": 1, "vocab": 32128,
         "temperature": 0.8, "top_k": 50, "top_p": 0.95, "min_p": 0.0, "per_row": False},
        # batch generation at the benchmark's batch 256: nucleus sampling
        {"name": "sample_256_nucleus", "op": "sample", "dtype": "fp16", "rows": 256, "vocab": 32128,
         "temperature": 1.0, "top_k": 0, "top_p": 0.9, "min_p": 0.0, "per_row": False},
        # a server that batches requests with options of their own, 32-bit
        # logits, an odd vocabulary
        {"name": "sample_33_per_row", "op": "sample", "dtype": "fp32", "rows": 33, "vocab": 50257,
         "temperature": 0.7, "top_k": 200, "top_p": 0.8, "min_p": 0.02, "per_row": True},
        # the encoder's keys and values of a batch-256 generation (512 tokens),
        # written once per layer before the decode loop
        {"name": "append_prompt_256x512", "op": "append", "dtype": "fp16", "batch": 256, "heads": 12,
         "dim": 64, "tokens": 512, "capacity": 512, "ragged": False},
        # a server's next chunks of prompts of unlike lengths, begun in the
        # middle of blocks
        {"name": "append_chunk_ragged", "op": "append", "dtype": "bf16", "batch": 8, "heads": 8,
         "dim": 128, "tokens": 137, "capacity": 4096, "ragged": True},
        # one request, an early decoder step of flan-t5-base with its
        # relative-position bias: latency alone counts
        {"name": "step_1_short", "op": "step", "dtype": "bf16", "batch": 1, "heads": 12, "group": 1,
         "dim": 64, "length": 45, "bias": True, "kpad": False, "ragged": False},
        # the last decoder step of batch-256 generation, 128 new tokens
        {"name": "step_256x128", "op": "step", "dtype": "fp16", "batch": 256, "heads": 12, "group": 1,
         "dim": 64, "length": 128, "bias": True, "kpad": False, "ragged": False},
        # flan-t5-xl's heads over a long document, keys of padding masked
        {"name": "step_8x5000_padded", "op": "step", "dtype": "bf16", "batch": 8, "heads": 32, "group": 1,
         "dim": 64, "length": 5000, "bias": False, "kpad": True, "ragged": False},
        # a server's step: grouped heads, sequences of unlike lengths, long
        {"name": "step_16x16k_grouped", "op": "step", "dtype": "bf16", "batch": 16, "heads": 8, "group": 4,
         "dim": 128, "length": 16384, "bias": False, "kpad": False, "ragged": True},
        # one request, flan-t5-base's fused qkv projection: latency
        {"name": "w4_1x2304x768", "op": "w4", "dtype": "bf16", "rows": 1, "out": 2304, "inp": 768},
        # one request, flan-t5-xxl's gated feed-forward input projection:
        # weight bandwidth
        {"name": "w4_1x20480x4096", "op": "w4", "dtype": "bf16", "rows": 1, "out": 20480, "inp": 4096},
        # batch 256, flan-t5-xl's feed-forward input projection: matrix rate
        {"name": "w4_256x10240x2048", "op": "w4", "dtype": "fp16", "rows": 256, "out": 10240, "inp": 2048},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["sample", "append", "step", "w4"])
    if op == "sample":
        vocab = _log(rng, 300, 130000)
        return {"op": op, "dtype": rng.choice(["bf16", "fp16", "fp32"]), "vocab": vocab,
                "rows": _log(rng, 1, max(1, min(256, 8000000 // vocab))),
                "temperature": rng.choice([0.0, 0.5, 0.8, 1.0, 1.3]),
                "top_k": rng.choice([0, 0, _log(rng, 1, vocab)]),
                "top_p": rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
                "min_p": rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.2), 4)]),
                "per_row": rng.random() < 0.5}
    if op == "append":
        dim, heads = rng.choice([32, 64, 128]), _log(rng, 1, 32)
        tokens = _log(rng, 1, 2048)
        batch = _log(rng, 1, max(1, min(256, 90000000 // (dim * heads * tokens))))
        return {"op": op, "dtype": rng.choice(["bf16", "fp16"]), "batch": batch, "heads": heads, "dim": dim,
                "tokens": tokens, "capacity": tokens + rng.randrange(0, 700), "ragged": rng.random() < 0.5}
    if op == "step":
        dim, heads = rng.choice([32, 64, 128]), _log(rng, 1, 32)
        length = _log(rng, 1, 16384)
        batch = _log(rng, 1, max(1, min(256, 250000000 // (dim * heads * length))))
        return {"op": op, "dtype": rng.choice(["bf16", "fp16"]), "batch": batch, "heads": heads,
                "group": rng.choice([1, 1, 2, 4, 7, 8]), "dim": dim, "length": length,
                "bias": rng.random() < 0.4, "kpad": rng.random() < 0.4, "ragged": rng.random() < 0.5}
    inp = GROUP * _log(rng, 2, 320)
    out = _log(rng, 16, 32768)
    rows = _log(rng, 1, max(1, min(256, 5000000000 // (inp * out))))
    return {"op": op, "dtype": rng.choice(["bf16", "fp16"]), "rows": rows, "out": out, "inp": inp}


# --------------------------------------------------------------------------- #
# inputs                                                                      #
# --------------------------------------------------------------------------- #
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return {"sample": _prepare_sample, "append": _prepare_append, "step": _prepare_step,
            "w4": _prepare_w4}[case["op"]](case, gen)


def _prepare_sample(c, gen):
    n, v = c["rows"], c["vocab"]
    logits = torch.randn(n, v, device="cuda", generator=gen) * 2.5
    # a trained model puts most of a row's mass on some tokens
    top = torch.randint(0, v // 24, (n, 24), device="cuda", generator=gen) + torch.arange(24, device="cuda") * (v // 24)
    logits.scatter_add_(1, top, torch.rand(n, 24, device="cuda", generator=gen) * 10)
    s = {"op": c["op"], "logits": logits.to(DTYPES[c["dtype"]]),
         "u": torch.rand(n, device="cuda", generator=gen)}
    if c["per_row"]:
        r = torch.rand(4, n, device="cuda", generator=gen)
        s["temperature"] = c["temperature"] * (0.5 + r[0])
        s["top_k"] = (c["top_k"] * (0.5 + r[1])).to(torch.int32)
        s["top_p"] = torch.full((n,), c["top_p"], device="cuda") ** (0.5 + r[2])
        s["min_p"] = c["min_p"] * r[3]
    else:
        s.update({k: c[k] for k in ("temperature", "top_k", "top_p", "min_p")})
    return s


def _empty_cache(b, h, capacity, d):
    nb = -(-capacity // BLOCK)
    e4m3 = torch.float8_e4m3fn
    return {"k": torch.zeros(b, h, nb * BLOCK, d, device="cuda", dtype=e4m3),
            "v": torch.zeros(b, h, nb, d, BLOCK, device="cuda", dtype=e4m3),
            "k_scale": torch.full((b, h, nb), 2.0 ** E_MIN, device="cuda"),
            "v_scale": torch.full((b, h, nb), 2.0 ** E_MIN, device="cuda")}


def _filled_cache(b, h, capacity, d, length, gen):
    """A cache whose first ``length`` tokens hold what a model wrote earlier:
    keys with some wide channels, values of unit size."""
    cache = _empty_cache(b, h, capacity, d)
    if length:
        wide = 1.0 + 3.0 * torch.rand(1, h, 1, d, device="cuda", generator=gen) ** 8
        start = torch.zeros(b, device="cuda", dtype=torch.int32)
        count = torch.full((b,), length, device="cuda", dtype=torch.int32)
        k = (torch.randn(b, h, length, d, device="cuda", generator=gen) * wide).to(torch.bfloat16)
        _append(cache["k"].view(b, h, -1, BLOCK, d), cache["k_scale"], k, start, count)
        v = torch.randn(b, h, length, d, device="cuda", generator=gen).to(torch.bfloat16)
        _append(cache["v"].transpose(-1, -2), cache["v_scale"], v, start, count)
    return cache


def _own_cache(cache):
    from mi355 import ops
    return ops.KVCache8.from_tensors(cache["k"], cache["v"], cache["k_scale"], cache["v_scale"])


def _prepare_append(c, gen):
    b, h, d, t = c["batch"], c["heads"], c["dim"], c["tokens"]
    room = c["capacity"] - t
    s = {"op": c["op"], "start": 0, "counts": None}
    if c["ragged"]:
        s["start"] = torch.randint(0, room + 1, (b,), device="cuda", generator=gen, dtype=torch.int32)
        s["counts"] = torch.randint((t + 1) // 2, t + 1, (b,), device="cuda", generator=gen, dtype=torch.int32)
    s["cache"] = _filled_cache(b, h, c["capacity"], d, room if c["ragged"] else 0, gen)
    # projections come out as (batch, tokens, heads, dim)
    dt = DTYPES[c["dtype"]]
    s["k"] = torch.randn(b, t, h, d, device="cuda", generator=gen).to(dt).transpose(1, 2)
    s["v"] = torch.randn(b, t, h, d, device="cuda", generator=gen).to(dt).transpose(1, 2)
    if own:
        s["own_cache"] = _own_cache(s["cache"])
    return s


def _prepare_step(c, gen):
    b, h, g, d, n = c["batch"], c["heads"], c["group"], c["dim"], c["length"]
    dt = DTYPES[c["dtype"]]
    s = {"op": c["op"], "start": n - 1, "lengths": n, "counts": None, "scale": 1.0 / math.sqrt(d),
         "bias": None, "kpad": None, "max_len": n}
    if c["ragged"]:
        s["start"] = torch.randint((n - 1) // 2, n, (b,), device="cuda", generator=gen, dtype=torch.int32)
        s["lengths"] = s["start"] + 1
    s["cache"] = _filled_cache(b, h, n, d, n - 1, gen)
    s["q"] = torch.randn(b, 1, h * g, d, device="cuda", generator=gen).to(dt).transpose(1, 2)
    s["k"] = torch.randn(b, 1, h, d, device="cuda", generator=gen).to(dt).transpose(1, 2)
    s["v"] = torch.randn(b, 1, h, d, device="cuda", generator=gen).to(dt).transpose(1, 2)
    if c["bias"]:
        s["bias"] = torch.randn(1, h * g, 1, n, device="cuda", generator=gen)
    if c["kpad"]:
        # up to a third of the keys is padding, at the front
        pad = torch.randint(0, n // 3 + 1, (b, 1), device="cuda", generator=gen)
        s["kpad"] = torch.where(torch.arange(n, device="cuda") < pad, -1e9, 0.0)
    if own:
        s["own_cache"] = _own_cache(s["cache"])
    return s


def _prepare_w4(c, gen):
    n, k = c["out"], c["inp"]
    codes = torch.randint(0, 256, (n, k // 2), device="cuda", generator=gen, dtype=torch.uint8)
    # groups of 32 of a trained weight: largest values within some octaves
    exps = torch.randint(117, 124, (n, k // GROUP), device="cuda", generator=gen, dtype=torch.uint8)
    s = {"op": c["op"], "codes": codes, "exps": exps,
         "x": torch.randn(c["rows"], k, device="cuda", generator=gen).to(DTYPES[c["dtype"]])}
    if own:
        from mi355 import ops
        s["w"] = ops.W4Weight(codes, exps)
    return s


# --------------------------------------------------------------------------- #
# one pass                                                                    #
# --------------------------------------------------------------------------- #
def run(state):
    if own:
        return _run_own(state)
    return {"sample": _plain_sample, "append": _plain_append, "step": _plain_step,
            "w4": _plain_w4}[state["op"]](state)


def _run_own(s):
    from mi355 import ops
    if s["op"] == "sample":
        return ops.sample_tokens(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                                 top_p=s["top_p"], min_p=s["min_p"])
    if s["op"] == "w4":
        return ops.linear_w4(s["x"], s["w"])
    ops.kv8_append(s["own_cache"], s["k"], s["v"], s["start"], counts=s["counts"])
    out = {k: s["cache"][k] for k in ("k", "v", "k_scale", "v_scale")}
    if s["op"] == "step":
        out["o"] = ops.decode_attention_kv8(s["q"], s["own_cache"], s["lengths"], bias=s["bias"],
                                            kpad=s["kpad"], scale=s["scale"], max_len=s["max_len"])
    return out


def _column(v, like, dtype):
    if torch.is_tensor(v):
        return v.to(dtype)[:, None]
    return torch.full((like.shape[0], 1), v, device=like.device, dtype=dtype)


def _plain_sample(s):
    # 64 bits: which token it is hangs on sums next to a border
    x = s["logits"].double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    t = _column(s["temperature"], x, torch.float64)
    k = _column(s["top_k"], x, torch.int64)
    top_p = _column(s["top_p"], x, torch.float64)
    min_p = _column(s["min_p"], x, torch.float64)
    k = torch.where(t == 0, 1, torch.where(k <= 0, x.shape[1], k))
    t = torch.where(t == 0, 1.0, t)
    m = x.amax(1, keepdim=True)
    w = torch.where(x == m, 1.0, torch.exp((x - m) / t))
    w = torch.where(m == -math.inf, 0.0, w)
    _, order = torch.sort(x, dim=1, descending=True, stable=True)
    rank = torch.arange(x.shape[1], device=x.device)[None]
    ws = torch.where(rank < k, w.gather(1, order), 0.0)
    cum = ws.cumsum(1)
    before = torch.cat([torch.zeros_like(cum[:, :1]), cum[:, :-1]], 1)
    keep = (rank < k) & ((rank == 0) | (top_p >= 1) | (before < top_p * cum[:, -1:])) & (ws >= min_p)
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, ws, 0.0))
    cum = kept.cumsum(1)
    r = s["u"].double()[:, None] * cum[:, -1:]
    ids = ((cum > r) & (kept > 0)).to(torch.int8).argmax(1)
    return torch.where(cum[:, -1] > 0, ids, -1)


def _scale_for(amax):
    """2^ceil(log2(amax / 448)), by exponents: exact."""
    f, e = torch.frexp(amax)                     # amax = f 2^e, f in [0.5, 1)
    e = e - 9 + (f > 0.875).to(e.dtype)          # 448 = 0.875 * 2^9
    e = torch.where(amax > 0, e.clamp(E_MIN, E_MAX), E_MIN)
    return torch.ldexp(torch.ones_like(amax), e)


def _append(codes, scales, new, start, counts):
    """codes (B,H,nb,64,D), written in place, as are scales (B,H,nb);
    new (B,H,S,D)."""
    b, h, nb, _, d = codes.shape
    n = new.shape[2]
    nw = (n + BLOCK - 2) // BLOCK + 1            # blocks that n tokens can touch
    first = (start // BLOCK).long()
    win = first[:, None] + torch.arange(nw, device=codes.device)
    valid = (win < nb) & (win * BLOCK < (start + counts)[:, None]) & (counts > 0)[:, None]
    src = torch.where(valid, win, first.clamp(max=nb - 1)[:, None])
    rows = torch.arange(b, device=codes.device)[:, None]
    old_codes = codes.view(torch.uint8)[rows, :, src].view(codes.dtype)     # (B,nw,H,64,D)
    old_scale = scales[rows, :, src]                                        # (B,nw,H)
    pos = win[:, :, None] * BLOCK + torch.arange(BLOCK, device=codes.device)
    at = pos - start[:, None, None]
    is_new = ((at >= 0) & (at < counts[:, None, None]))[:, :, None, :, None]
    is_old = (at < 0)[:, :, None, :, None]
    fresh = new.transpose(1, 2)[rows[:, :, None], at.clamp(0, n - 1)].transpose(2, 3).float()
    fresh = torch.where(is_new, fresh, 0.0)                                 # (B,nw,H,64,D)
    scale = _scale_for(fresh.abs().amax((-1, -2)))
    begun = (win * BLOCK < start[:, None])[:, :, None]
    scale = torch.where(begun, torch.maximum(scale, old_scale), scale)
    s5 = scale[..., None, None]
    value = torch.where(is_new, fresh, torch.where(is_old, old_codes.float() * old_scale[..., None, None], 0.0))
    value = (value / s5).clamp(-448, 448).to(codes.dtype).view(torch.uint8)
    # codes behind the last new token stay as they were
    touched = valid[:, :, None, None, None] & (is_new | is_old)
    value = torch.where(touched, value, old_codes.view(torch.uint8))
    scale = torch.where(valid[:, :, None], scale, old_scale)
    # a window that is not valid repeats the first one's outcome
    value = torch.where(valid[:, :, None, None, None], value, value[:, :1])
    scale = torch.where(valid[:, :, None], scale, scale[:, :1])
    codes.view(torch.uint8)[rows, :, src] = value
    scales[rows, :, src] = scale


def _plain_append(s):
    c, k, v = s["cache"], s["k"], s["v"]
    b, h, n, d = k.shape
    start, counts = s["start"], s["counts"]
    if not torch.is_tensor(start):
        start = torch.full((b,), start, device=k.device, dtype=torch.int32)
    if counts is None:
        counts = torch.full((b,), n, device=k.device, dtype=torch.int32)
    _append(c["k"].view(b, h, -1, BLOCK, d), c["k_scale"], k, start, counts)
    _append(c["v"].transpose(-1, -2), c["v_scale"], v, start, counts)
    return {x: c[x] for x in ("k", "v", "k_scale", "v_scale")}


def _plain_step(s):
    out = _plain_append(s)
    c, q = s["cache"], s["q"]
    b, h, cap, d = c["k"].shape
    k = (c["k"].view(b, h, -1, BLOCK, d).float() * c["k_scale"][..., None, None]).view(b, h, cap, d)
    v = (c["v"].float() * c["v_scale"][..., None, None]).transpose(-1, -2).reshape(b, h, cap, d)
    qf = q.float().reshape(b, h, -1, d)
    score = torch.matmul(qf, k.transpose(-1, -2).contiguous()) * s["scale"]       # (B,H,G,cap)
    n = s["max_len"]
    score = score[..., :n]
    if s["bias"] is not None:
        score = score + s["bias"].reshape(1, h, -1, n)
    if s["kpad"] is not None:
        score = score + s["kpad"][:, None, None]
    lengths = s["lengths"] if torch.is_tensor(s["lengths"]) else torch.full((b,), n, device=q.device)
    score = torch.where(torch.arange(n, device=q.device) < lengths[:, None, None, None], score, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    o = torch.matmul(p, v[:, :, :n].contiguous()) / p.sum(-1, keepdim=True)
    out["o"] = o.reshape(b, -1, 1, d).to(q.dtype)
    return out


def _plain_w4(s):
    n, half = s["codes"].shape
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=s["x"].device)
    nibbles = torch.stack([s["codes"] & 15, s["codes"] >> 4], -1).view(n, 2 * half)
    scale = torch.ldexp(torch.ones((), device=s["x"].device), s["exps"].int() - 127)
    w = table[nibbles.int()].view(n, -1, GROUP) * scale[..., None]
    return (s["x"].float() @ w.view(n, -1).t()).to(s["x"].dtype)


# --------------------------------------------------------------------------- #
# what a pass cannot do without                                               #
# --------------------------------------------------------------------------- #
def work(case):
    c = case
    size = 4 if c["dtype"] == "fp32" else 2
    if c["op"] == "sample":
        n = c["rows"] * c["vocab"]
        return {"bytes": n * size + c["rows"] * 12, "flops": 12 * n}   # an exp and a sum a logit
    if c["op"] == "w4":
        m, n, k = c["rows"], c["out"], c["inp"]
        return {"bytes": n * k // 2 + n * k // GROUP + (m * k + m * n) * size, "flops": 2 * m * n * k}
    rows = c["batch"] * c["heads"] * c["dim"]
    if c["op"] == "append":
        tokens = c["tokens"] * (0.75 if c["ragged"] else 1.0)
        return {"bytes": 2 * rows * tokens * (size + 1), "flops": 4 * rows * tokens}
    length = c["length"] * (0.75 if c["ragged"] else 1.0)
    scales = c["batch"] * c["heads"] * 8 * length / BLOCK
    masks = 4 * length * (c["bias"] * c["heads"] * c["group"] + c["kpad"] * c["batch"])
    return {"bytes": 2 * rows * length + scales + masks + 2 * rows * (1 + c["group"]) * size,
            "flops": 4 * rows * c["group"] * length}


# --------------------------------------------------------------------------- #
# the definitions in 64 bits, row by row                                      #
# --------------------------------------------------------------------------- #
def exact(case, seed):
    s = prepare(case, seed)
    return {"sample": _exact_sample, "append": _exact_append, "step": _exact_step,
            "w4": _exact_w4}[case["op"]](s)


def _exact_sample(s):
    import numpy as np
    logits = s["logits"].double().cpu().numpy()
    n, vocab = logits.shape
    opt = {k: (s[k].double().cpu().numpy() if torch.is_tensor(s[k]) else np.full(n, float(s[k])))
           for k in ("temperature", "top_k", "top_p", "min_p")}
    u = s["u"].double().cpu().numpy()
    ids = np.empty(n, dtype=np.int64)
    for i in range(n):
        x = np.where(np.isnan(logits[i]), -np.inf, logits[i])
        if x.max() == -np.inf:
            ids[i] = -1
            continue
        order = np.argsort(-x, kind="stable")            # ties: the lower index first
        if opt["temperature"][i] == 0:
            ids[i] = order[0]
            continue
        k = int(opt["top_k"][i])
        order = order[:k] if k > 0 else order
        w = np.where(x[order] == x[order[0]], 1.0, np.exp((x[order] - x[order[0]]) / opt["temperature"][i]))
        size = len(order)
        if opt["top_p"][i] < 1:
            size = max(1, int(np.searchsorted(np.cumsum(w), opt["top_p"][i] * np.cumsum(w)[-1])) + 1)
        size = min(size, max(1, int((w >= opt["min_p"][i]).sum())))
        by_index = np.argsort(order[:size])
        cum = np.cumsum(w[:size][by_index])
        at = min(int(np.searchsorted(cum, u[i] * cum[-1], side="right")), size - 1)
        ids[i] = order[:size][by_index][at]
    return torch.from_numpy(ids)


def _round_e4m3(x):
    """Nearest value with 4 significant bits and steps of at least 2^-9, ties
    to even, of at most 448 in size."""
    step = torch.exp2((torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3))
    return (torch.round(x / step) * step).clamp(-448, 448)


def _exact_cache(s):
    """The cache after the append, as 64-bit codes and scales."""
    c, n = s["cache"], s["k"].shape[2]
    b, h, cap, d = c["k"].shape
    got = {}
    for name in ("k", "v"):
        codes = c[name].double().view(b, h, -1, BLOCK, d) if name == "k" else \
            c[name].double().transpose(-1, -2).contiguous()
        scale = c[name + "_scale"].double()
        for i in range(b):
            at = int(s["start"][i]) if torch.is_tensor(s["start"]) else s["start"]
            end = at + (int(s["counts"][i]) if s["counts"] is not None else n)
            for blk in range(at // BLOCK, -(-min(end, cap) // BLOCK)):
                lo, hi = blk * BLOCK, min((blk + 1) * BLOCK, end)
                value = torch.zeros(h, hi - lo, d, dtype=torch.float64, device=codes.device)
                began, grow = max(at, lo), torch.full((h,), 2.0 ** E_MIN, dtype=torch.float64, device=codes.device)
                if at > lo:
                    grow = scale[i, :, blk].clone()
                    value[:, :at - lo] = codes[i, :, blk, :at - lo] * grow[:, None, None]
                fresh = s[name][i, :, began - at:hi - at].double()
                value[:, began - lo:] = fresh
                big = fresh.abs().amax((1, 2))
                need = torch.exp2(torch.ceil(torch.log2(big / 448)))
                grow = torch.maximum(grow, torch.where(big > 0, need, 2.0 ** E_MIN))
                codes[i, :, blk, :hi - lo] = _round_e4m3(value / grow[:, None, None])
                scale[i, :, blk] = grow
        got[name + "_scale"] = scale
        got[name] = codes.view(b, h, cap, d) if name == "k" else codes.transpose(-1, -2).contiguous()
    return got


def _exact_append(s):
    return _exact_cache(s)


def _exact_step(s):
    got = _exact_cache(s)
    b, hq, _, d = s["q"].shape
    h = got["k"].shape[1]
    o = torch.zeros(b, hq, 1, d, dtype=torch.float64, device="cuda")
    for i in range(b):
        n = int(s["lengths"][i]) if torch.is_tensor(s["lengths"]) else s["lengths"]
        k = (got["k"][i].view(h, -1, BLOCK, d) * got["k_scale"][i][..., None, None]).view(h, -1, d)[:, :n]
        v = (got["v"][i] * got["v_scale"][i][..., None, None]).transpose(-1, -2).reshape(h, -1, d)[:, :n]
        q = s["q"][i].double().reshape(h, hq // h, d)
        score = (q[:, :, None] * k[:, None]).sum(-1) * s["scale"] if n < 256 else \
            torch.bmm(q, k.transpose(1, 2).contiguous()) * s["scale"]
        if s["bias"] is not None:
            score = score + s["bias"][0, :, 0, :n].double().view(h, -1, n)
        if s["kpad"] is not None:
            score = score + s["kpad"][i, :n].double()
        o[i] = torch.bmm(torch.softmax(score, -1), v).reshape(hq, 1, d)
    got["o"] = o
    return got


def _exact_w4(s):
    values = torch.tensor([(-1.0 if c & 8 else 1.0) * ((c & 1) * 0.5 if c & 6 == 0 else (1 + (c & 1) / 2) * 2.0 ** ((c & 7) // 2 - 1))
                           for c in range(16)], dtype=torch.float64, device="cuda")
    n, half = s["codes"].shape
    w = torch.empty(n, 2 * half, dtype=torch.float64, device="cuda")
    w[:, 0::2] = values[(s["codes"] % 16).long()]
    w[:, 1::2] = values[(s["codes"] // 16).long()]
    w *= torch.exp2(s["exps"].double() - 127).repeat_interleave(GROUP, 1)
    return torch.matmul(s["x"].double(), w.t())
