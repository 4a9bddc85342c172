"""Plain-PyTorch reference implementations of every mi355 hot op.

These are the semantics contract for the hand-written HIP/CDNA4 kernels in
``mi355/csrc/kernels``: each HIP kernel is validated against the op here in
fp32 (see tests/test_ops_numerics.py). On CPU these are also the execution
path (the reference workshop runs its distributed trainer on CPU with
``no_cuda=True`` — see SURVEY.md §4.2, reference
Scaling_model_training.ipynb:cell-47).

All functions are differentiable plain-torch compositions.
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    """T5LayerNorm: RMS norm, no mean subtraction, no bias.

    Matches the reference model's T5 layer norm semantics:
    accumulate the mean-square in fp32, scale in the input dtype.
    """
    dt = x.dtype
    xf = x.float()
    var = xf.pow(2).mean(dim=-1, keepdim=True)
    xf = xf * torch.rsqrt(var + eps)
    return (xf.to(dt)) * weight


def gelu_tanh(x: torch.Tensor) -> torch.Tensor:
    """gelu_new / tanh approximation (T5 v1.1 gated act)."""
    return 0.5 * x * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (x + 0.044715 * x.pow(3.0))))


def geglu(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """Gated-GELU elementwise combine: gelu_tanh(gate) * up  (SURVEY.md K6)."""
    return gelu_tanh(gate) * up


def attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    bias: torch.Tensor | None = None,
    causal: bool = False,
    scale: float = 1.0,
    kpad: torch.Tensor | None = None,
    p_drop: float = 0.0,
) -> torch.Tensor:
    """Attention core with additive bias (T5 relative-position bias), unscaled
    by default (T5 absorbs 1/sqrt(d) into init — SURVEY.md K4).

    q: (B, H, Sq, D); k, v: (B, H, Sk, D); bias broadcastable to (B, H, Sq, Sk).
    """
    scores = torch.matmul(q, k.transpose(-1, -2))
    if scale != 1.0:
        scores = scores * scale
    if bias is not None:
        scores = scores + bias
    if kpad is not None:
        scores = scores + kpad.view(kpad.shape[0], 1, 1, kpad.shape[-1]).to(scores.dtype)
    if causal:
        sq, sk = scores.shape[-2], scores.shape[-1]
        idx_q = torch.arange(sq, device=scores.device).unsqueeze(-1) + (sk - sq)
        idx_k = torch.arange(sk, device=scores.device).unsqueeze(0)
        neg = torch.finfo(scores.dtype).min
        scores = scores.masked_fill(idx_k > idx_q, neg)
    probs = F.softmax(scores.float(), dim=-1).to(q.dtype)
    if p_drop > 0.0:
        probs = F.dropout(probs, p=p_drop, training=True)
    return torch.matmul(probs, v)


def cross_entropy(logits: torch.Tensor, labels: torch.Tensor, ignore_index: int = -100):
    """Token-mean CE over the vocab, fp32 log-softmax."""
    return F.cross_entropy(
        logits.float().view(-1, logits.shape[-1]),
        labels.view(-1),
        ignore_index=ignore_index,
    )


def adamw_step(
    params_f32: list[torch.Tensor],
    grads: list[torch.Tensor],
    exp_avgs: list[torch.Tensor],
    exp_avg_sqs: list[torch.Tensor],
    *,
    lr: float,
    beta1: float,
    beta2: float,
    eps: float,
    weight_decay: float,
    step: int,
    grad_scale: float = 1.0,
    outs_lowp: list[torch.Tensor] | None = None,
):
    """Decoupled AdamW on fp32 master params.

    ``outs_lowp`` optionally receives the updated params cast to its dtype
    (bf16 model weights while masters stay fp32).
    """
    bc1 = 1.0 - beta1**step
    bc2 = 1.0 - beta2**step
    for i, (p, g, m, v) in enumerate(zip(params_f32, grads, exp_avgs, exp_avg_sqs)):
        gf = g.float()
        if grad_scale != 1.0:
            gf = gf * grad_scale
        m.mul_(beta1).add_(gf, alpha=1.0 - beta1)
        v.mul_(beta2).addcmul_(gf, gf, value=1.0 - beta2)
        denom = (v / bc2).sqrt_().add_(eps)
        p.mul_(1.0 - lr * weight_decay)
        p.addcdiv_(m / bc1, denom, value=-lr)
        if outs_lowp is not None:
            outs_lowp[i].copy_(p)


def softmax_bias(scores: torch.Tensor, bias: torch.Tensor | None) -> torch.Tensor:
    out = scores if bias is None else scores + bias
    return F.softmax(out.float(), dim=-1).to(scores.dtype)


def seg_postprocess(logits: torch.Tensor, size) -> torch.Tensor:
    """Bilinear-upsample class logits to ``size`` and argmax over channels
    (SURVEY.md K17 — reference post_process_semantic_segmentation)."""
    up = F.interpolate(logits.float(), size=size, mode="bilinear",
                       align_corners=False)
    return up.argmax(dim=1).to(torch.int32)


# --------------------------------------------------------------------------- #
# 4-bit weights                                                               #
# --------------------------------------------------------------------------- #
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
W4_SPAN = 26        # octaves between scales that weights in 16 bits hold (csrc/kernels/w4_linear.hip)


def w4_dequantize(codes: torch.Tensor, exps: torch.Tensor, dtype=torch.float32) -> torch.Tensor:
    """(N, K/2) codes and (N, K/32) exponents -> (N, K); a byte of 255 is NaN."""
    n, half = codes.shape
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device, dtype=dtype)
    nibbles = torch.stack([codes & 15, codes >> 4], -1).view(n, half // 16, 32)
    scale = torch.ldexp(torch.ones((), device=codes.device, dtype=dtype), exps.int() - 127)
    scale = torch.where(exps == 255, math.nan, scale)
    return (table[nibbles.int()] * scale[..., None]).view(n, 2 * half)


def w4_row_exp(codes: torch.Tensor, exps: torch.Tensor) -> torch.Tensor:
    """(N,) uint8, what the kernels scale a row against: its largest exponent
    byte of a group that holds more than zeros; 255 where those of the row lie
    over W4_SPAN apart, or one is no scale: such a row is summed group by
    group."""
    there = (codes & 0x77).view(*exps.shape, 16).amax(-1) > 0
    most = torch.where(there, exps, 0).amax(1)
    least = torch.where(there, exps, 255).amin(1)
    apart = (most.int() - least.int() > W4_SPAN) | (exps == 255).any(1)
    return torch.where(apart, 255, most).to(torch.uint8)


def w4_quantize(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    n, k = weight.shape
    w = weight.float().contiguous().view(n, k // 32, 32)
    amax = w.abs().amax(-1, keepdim=True)
    # 6 * 2^e >= amax for the upper of the two powers of two
    _, e = torch.frexp(amax / 6)
    e = torch.where(amax > 0, e, -126)
    # halfway values go to the even code, as the format's rounding has it
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=w.device)
    table = torch.tensor(E2M1, device=w.device)
    best = None
    e = e.clamp(-126, 126)
    for less in (0, 1):
        ee = (e - less).clamp(min=-126)
        scaled = torch.ldexp(w, -ee)
        up = torch.bucketize(scaled.abs(), edges, right=True)    # ties up
        down = torch.bucketize(scaled.abs(), edges)              # ties down
        code = torch.where(up % 2 == 0, up, down)
        # at the upper scale: squares of the weights themselves may leave fp32's range
        err = torch.ldexp(table[code] - scaled.abs(), ee - e).square().sum(-1, keepdim=True)
        code = code + 8 * (scaled < 0)
        if best is None:
            best = (err, code, ee)
        else:
            take = err < best[0]
            best = (None, torch.where(take, code, best[1]), torch.where(take, ee, best[2]))
    code = best[1].view(n, k).to(torch.uint8)
    return code[:, 0::2] | code[:, 1::2] << 4, (best[2].view(n, k // 32) + 127).to(torch.uint8)


def linear_w4(x: torch.Tensor, codes: torch.Tensor, exps: torch.Tensor) -> torch.Tensor:
    # in 64 bits: 6 * 2^127 is a weight, and over fp32's range
    return torch.matmul(x.double(), w4_dequantize(codes, exps, torch.float64).t()).to(x.dtype)


# --------------------------------------------------------------------------- #
# key/value cache in 8 bits                                                   #
# --------------------------------------------------------------------------- #
KV8_BLOCK, KV8_E_MIN, KV8_E_MAX = 64, -120, 120


def kv8_scale(amax: torch.Tensor) -> torch.Tensor:
    """2^ceil(log2(amax / 448)), within the exponents a scale may have."""
    f, e = torch.frexp(amax)                       # amax = f 2^e, f in [0.5, 1)
    e = e - 9 + (f > 0.875).to(e.dtype)            # 448 = 0.875 * 2^9
    e = torch.where(amax > 0, e.clamp(KV8_E_MIN, KV8_E_MAX), KV8_E_MIN)
    return torch.ldexp(torch.ones_like(amax), e)


def kv8_values(k, v, k_scale, v_scale) -> tuple[torch.Tensor, torch.Tensor]:
    b, h, cap, d = k.shape
    kf = (k.float().view(b, h, -1, KV8_BLOCK, d) * k_scale[..., None, None]).view(b, h, cap, d)
    vf = (v.float() * v_scale[..., None, None]).transpose(-1, -2).reshape(b, h, cap, d)
    return kf, vf


def kv8_append(kc, vc, k_scale, v_scale, k, v, start, counts=None) -> None:
    b, h, cap, d = kc.shape
    for codes, scales, new in ((kc.view(b, h, -1, KV8_BLOCK, d), k_scale, k),
                               (vc.transpose(-1, -2), v_scale, v)):
        for i in range(b):
            at = int(start[i]) if torch.is_tensor(start) else start
            n = min(int(counts[i]), new.shape[2]) if counts is not None else new.shape[2]
            if at < 0 or n <= 0:
                continue
            end = min(at + n, cap)
            for blk in range(at // KV8_BLOCK, -(-end // KV8_BLOCK)):
                base = blk * KV8_BLOCK
                lo, hi = max(at - base, 0), min(end - base, KV8_BLOCK)
                fresh = new[i, :, base + lo - at:base + hi - at].float()      # (H, n, D)
                size = torch.where(fresh.abs() < math.inf, fresh.abs(), 0.0)
                scale = kv8_scale(size.amax((1, 2)))
                if lo > 0:
                    old = scales[i, :, blk]
                    scale = torch.maximum(scale, old)
                    ratio = (old / scale)[:, None, None]
                    kept = codes[i, :, blk, :lo].float() * ratio
                    codes[i, :, blk, :lo] = kept.to(codes.dtype)
                codes[i, :, blk, lo:hi] = (fresh / scale[:, None, None]).clamp(-448, 448).to(codes.dtype)
                scales[i, :, blk] = scale


def decode_attention_kv8(q, k, v, k_scale, v_scale, lengths, bias, kpad, scale, max_len):
    b, h, cap, d = k.shape
    if max_len == 0:
        return torch.zeros_like(q)
    kf, vf = kv8_values(k, v, k_scale, v_scale)
    kf, vf = kf[:, :, :max_len], vf[:, :, :max_len]
    there = torch.arange(max_len, device=q.device) < (
        lengths[:, None] if torch.is_tensor(lengths) else torch.full((b, 1), lengths, device=q.device))
    if kpad is not None:
        there = there & (kpad[:, :max_len] != -math.inf)
    # what is not there counts for nothing, whatever it holds
    kf = torch.where(there[:, None, :, None], kf, 0.0)
    vf = torch.where(there[:, None, :, None], vf, 0.0)
    s = torch.matmul(q.float().reshape(b, h, -1, d), kf.transpose(-1, -2).contiguous()) * scale
    if bias is not None:
        s = s + bias[..., :max_len].float().reshape(bias.shape[0], h, -1, max_len)
    if kpad is not None:
        s = s + kpad[:, None, None, :max_len].float()
    s = torch.where(there[:, None, None], s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    l = p.sum(-1, keepdim=True)
    o = torch.where(l == 0, 0.0, torch.matmul(p, vf) / l)
    return o.reshape(b, -1, 1, d).to(q.dtype)


# --------------------------------------------------------------------------- #
# choosing a token                                                            #
# --------------------------------------------------------------------------- #
def sample_tokens(logits, u, temperature, top_k, top_p, min_p, empty_token: int = -1):
    x = logits.double()
    x = torch.where(torch.isnan(x), -math.inf, x)

    def column(v, dtype):
        return v.to(dtype)[:, None] if torch.is_tensor(v) else \
            torch.full((len(x), 1), v, device=x.device, dtype=dtype)

    t, k = column(temperature, torch.float64), column(top_k, torch.int64)
    t = t.clamp(max=1e30)
    p, floor = column(top_p, torch.float64), column(min_p, torch.float64).clamp(max=1.0)
    greedy = ~(t > 0)
    k = torch.where(greedy, 1, torch.where(k <= 0, x.shape[1], k))
    t = torch.where(greedy, 1.0, t)
    m = x.amax(1, keepdim=True)
    w = torch.where(x == m, 1.0, torch.exp((x - m) / t))
    w = torch.where((m == -math.inf) | (w < 2.0 ** -45), 0.0, w)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    rank = torch.arange(x.shape[1], device=x.device)[None]
    ws = torch.where(rank < k, w.gather(1, order), 0.0)
    cum = ws.cumsum(1)
    before = torch.nn.functional.pad(cum[:, :-1], (1, 0))
    keep = (rank < k) & ((rank == 0) | ~(p < 1) | (before < p * cum[:, -1:])) & ~(ws < floor)
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, ws, 0.0))
    cum = kept.cumsum(1)
    r = u.double().nan_to_num(0.0).clamp(min=0.0)[:, None] * cum[:, -1:]
    over = (cum > r) & (kept > 0)
    # u = 1 (or a rounding of u times the sum): the last one kept
    ids = torch.where(over.any(1), over.to(torch.int8).argmax(1),
                      x.shape[1] - 1 - (kept > 0).to(torch.int8).flip(1).argmax(1))
    return torch.where(cum[:, -1] > 0, ids, empty_token)
