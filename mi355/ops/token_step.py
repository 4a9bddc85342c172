"""What one generated token costs a served model: products of a few rows with
4-bit weights, a key/value cache held in 8 bits, and the choice of the token.

All of it is inference only: weights and caches are codes and tokens are whole
numbers, so inputs that ask for a gradient are refused.  On a GPU tensor the
hand-written kernels run (``csrc/kernels/{w4_linear,kv8,sample}.hip``); CPU
tensors take the plain-PyTorch forms in ``torch_ref``.

Calls here are a few microseconds on the GPU, so the GPU path goes straight to
the extension, which checks the arguments (ValueError, as on the CPU path).
"""
from __future__ import annotations

import math

import torch

from . import _load_ext, _use_hip, torch_ref

def _no_grad(what: str, *tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{what} has no backward pass: call it under torch.no_grad()")


def _per_row(v, what: str, rows: int, device, dtype):
    """(tensor or None, number): one value for every row, or a number for all."""
    if not torch.is_tensor(v):
        return None, v
    if dtype == torch.int32 and what != "top_k" and (v.is_floating_point() or v.is_complex() or v.dtype == torch.bool):
        raise ValueError(f"{what} must be whole numbers, got {v.dtype}")
    if v.shape != (rows,) or v.device != device:
        raise ValueError(f"{what} must be a number or a ({rows},) tensor on {device}, "
                         f"got {tuple(v.shape)} on {v.device}")
    if dtype == torch.int32 and v.dtype != dtype:   # no number becomes another one
        v = v.double().nan_to_num(0.0).clamp(-2.0 ** 31, 2.0 ** 31 - 1)
    wide = dtype == torch.float32 and v.dtype == torch.float64
    return (v if v.dtype == dtype or wide else v.to(dtype)).contiguous(), 0


# --------------------------------------------------------------------------- #
# 4-bit weights                                                               #
# --------------------------------------------------------------------------- #
class W4Weight(torch.nn.Module):
    """A (N, K) weight in 4.25 bits: E2M1 codes (values 0, .5, 1, 1.5, 2, 3, 4,
    6 and their negatives), two a byte with the even input in the low nibble,
    and one exponent byte e for 32 inputs of a row: w = code * 2^(e - 127).

    ``codes`` (N, K/2) uint8, ``exps`` (N, K/32) uint8; K a multiple of 32.
    An exponent of 255 is no scale (the format's NaN): its row's outputs are
    not finite.  The buffers are read as they lie: nothing is laid out anew.
    ``row_exp`` (N,) is made from them, here and when a state is loaded: they
    are not to be written over otherwise.
    """

    GROUP = 32

    def __init__(self, codes: torch.Tensor, exps: torch.Tensor):
        super().__init__()
        if codes.dtype != torch.uint8 or exps.dtype != torch.uint8 or codes.dim() != 2 or exps.dim() != 2:
            raise ValueError("W4Weight takes uint8 codes (N, K/2) and exponents (N, K/32)")
        if codes.shape[0] != exps.shape[0] or codes.shape[1] != 16 * exps.shape[1] or not codes.shape[1]:
            raise ValueError(f"codes {tuple(codes.shape)} and exponents {tuple(exps.shape)} are not "
                             "of one (N, K) weight with K a multiple of 32")
        if codes.device != exps.device:
            raise ValueError(f"codes on {codes.device}, exponents on {exps.device}")
        self.register_buffer("codes", codes.contiguous())
        self.register_buffer("exps", exps.contiguous())
        self.register_buffer("row_exp", self._row_exp())

    def _row_exp(self) -> torch.Tensor:
        make = _load_ext().w4_row_exp if _use_hip(self.codes) else torch_ref.w4_row_exp
        return make(self.codes.contiguous(), self.exps.contiguous())

    def _load_from_state_dict(self, *args, **kwargs):
        row_exp = self.row_exp
        super()._load_from_state_dict(*args, **kwargs)
        fresh = self._row_exp()
        if self.row_exp is row_exp:
            row_exp.copy_(fresh)
        else:                                   # the caller's tensor, of an assigning load
            self.row_exp = fresh

    @property
    def shape(self) -> torch.Size:
        return torch.Size((self.codes.shape[0], 2 * self.codes.shape[1]))

    def rows(self, start: int, stop: int) -> "W4Weight":
        """Output rows [start, stop) as a weight that shares the buffers."""
        part = W4Weight.__new__(W4Weight)
        torch.nn.Module.__init__(part)
        for name in ("codes", "exps", "row_exp"):
            part.register_buffer(name, self._buffers[name][start:stop])
        return part

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        return torch_ref.w4_dequantize(self.codes, self.exps).to(dtype)

    def data_ptr(self) -> int:
        return self.codes.data_ptr()

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return linear_w4(x, self)

    def extra_repr(self) -> str:
        return f"{self.shape[0]}, {self.shape[1]}"


@torch.no_grad()
def quantize_w4(weight: torch.Tensor) -> W4Weight:
    """The nearest :class:`W4Weight` of an (N, K) weight that is finite in fp32:
    for each group of 32 inputs that power of two, of the two next to amax/6,
    whose rounded codes are off by the smaller sum of squares.  Waits for the
    device once, to refuse what is not finite."""
    if weight.dim() != 2 or weight.shape[1] % W4Weight.GROUP or not weight.shape[1]:
        raise ValueError(f"quantize_w4 takes (N, K) with K a multiple of 32, got {tuple(weight.shape)}")
    weight = weight.float()
    if not torch.isfinite(weight).all():
        raise ValueError("quantize_w4 takes a finite weight")
    return W4Weight(*torch_ref.w4_quantize(weight))


def linear_w4(x: torch.Tensor, w: W4Weight) -> torch.Tensor:
    """``x @ w.T`` for x (..., K) in bf16 or fp16: sums in 32 bits, one rounding
    at the end.  Any number of rows; made for the few that decoding has.  The
    largest scale of a row of w is multiplied in after its sum: sums of x times
    codes have to stay in fp32's range (inputs under 2^125 / K and over 2^-99
    do).  A row of w whose scales lie over 26 octaves apart, groups of zeros not
    counted, is right too, but slow: its groups are summed one by one."""
    if x.is_cuda and _use_hip(x):
        b = w._buffers
        return _load_ext().w4_linear(x, b["codes"], b["exps"], b["row_exp"])
    _no_grad("linear_w4", x)
    if x.dim() == 0 or x.shape[-1] != w.shape[1]:
        raise ValueError(f"linear_w4: x {tuple(x.shape)}, the weight has {w.shape[1]} inputs")
    if w.codes.device != x.device:
        raise ValueError(f"linear_w4: x on {x.device}, the weight on {w.codes.device}")
    return torch_ref.linear_w4(x, w.codes, w.exps)


# --------------------------------------------------------------------------- #
# 8-bit key/value cache                                                       #
# --------------------------------------------------------------------------- #
class KVCache8:
    """Keys and values of ``batch`` sequences in e4m3 codes, with a power-of-two
    scale for each block of 64 tokens and head.

    ``k`` (B, H, NB*64, D) and ``v`` (B, H, NB, D, 64; a block is turned) hold
    codes, ``k_scale`` / ``v_scale`` (B, H, NB) what they are multiplied by.
    Head dims 32, 64 and 128.  The cache does not count its tokens: callers
    pass ``start`` and ``lengths``, as with :func:`decode_attention`.
    """

    BLOCK = 64

    def __init__(self, batch: int, heads: int, capacity: int, head_dim: int, device=None):
        if head_dim not in (32, 64, 128):
            raise ValueError(f"KVCache8: head dim 32, 64 or 128, got {head_dim}")
        nb = -(-capacity // self.BLOCK)
        e4m3 = torch.float8_e4m3fn
        self.k = torch.zeros(batch, heads, nb * self.BLOCK, head_dim, device=device, dtype=e4m3)
        self.v = torch.zeros(batch, heads, nb, head_dim, self.BLOCK, device=device, dtype=e4m3)
        self.k_scale = torch.full((batch, heads, nb), 2.0 ** torch_ref.KV8_E_MIN, device=device)
        self.v_scale = self.k_scale.clone()

    @classmethod
    def from_tensors(cls, k, v, k_scale, v_scale) -> "KVCache8":
        """A cache on buffers that the caller holds (shared, not copied).  The
        scales have to be powers of two from 2^-120 to 2^120, as appends make
        them; that is not checked."""
        b, h, nb, d, block = v.shape if v.dim() == 5 else (0,) * 5
        if block != cls.BLOCK or d not in (32, 64, 128) or k.shape != (b, h, nb * block, d) \
                or k_scale.shape != (b, h, nb) or v_scale.shape != (b, h, nb):
            raise ValueError(f"KVCache8: k {tuple(k.shape)}, v {tuple(v.shape)}, scales "
                             f"{tuple(k_scale.shape)}, {tuple(v_scale.shape)} are not of one cache")
        if k.dtype != torch.float8_e4m3fn or v.dtype != k.dtype or k_scale.dtype != torch.float32 \
                or v_scale.dtype != torch.float32:
            raise ValueError("KVCache8: codes are float8_e4m3fn, scales float32")
        if any(t.device != k.device or not t.is_contiguous() for t in (k, v, k_scale, v_scale)):
            raise ValueError("KVCache8: contiguous tensors of one device")
        self = cls.__new__(cls)
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        return self

    @property
    def capacity(self) -> int:
        return self.k.shape[2]

    def dequantize(self) -> tuple[torch.Tensor, torch.Tensor]:
        """(k, v) as fp32 (B, H, capacity, D)."""
        return torch_ref.kv8_values(self.k, self.v, self.k_scale, self.v_scale)


def kv8_append(cache: KVCache8, k: torch.Tensor, v: torch.Tensor, start, counts=None) -> None:
    """Write tokens k, v (B, H, S, D) at positions ``start``.. of each sequence.

    On a GPU tokens are bf16 or fp16; a CPU takes any floating type.
    ``start``: a number, or an int32 (B,) tensor.  ``counts``: int32 (B,), how
    many of the S tokens a sequence has (the first ones; default all).  A block
    that was begun keeps the larger of its old scale and what the new tokens
    need, its earlier codes follow.  Codes behind the last new token stay as
    they were.  A number is checked against the capacity; of positions from a
    tensor, those past the capacity are not written, and a negative one skips
    the sequence.  Infinities saturate and do not widen a scale; NaN stays NaN.
    """
    if counts is not None and not torch.is_tensor(counts):
        raise ValueError("kv8_append: counts is an int32 (B,) tensor")
    if k.is_cuda and _use_hip(k):
        each = torch.is_tensor(start)
        _load_ext().kv8_append(k, v, cache.k, cache.v, cache.k_scale, cache.v_scale,
                               start if each else None, 0 if each else start, counts)
        return
    _no_grad("kv8_append", k, v)
    b, h, cap, d = cache.k.shape
    if k.dim() != 4 or k.shape != v.shape or k.shape[:2] != (b, h) or k.shape[3] != d or k.dtype != v.dtype:
        raise ValueError(f"kv8_append: k {tuple(k.shape)} {k.dtype}, v {tuple(v.shape)} {v.dtype} "
                         f"do not fit a cache of (B, H, ., D) = ({b}, {h}, ., {d})")
    if k.device != cache.k.device or v.device != k.device:
        raise ValueError(f"kv8_append: tokens on {k.device}, {v.device}, cache on {cache.k.device}")
    starts, start = _per_row(start, "start", b, k.device, torch.int32)
    if starts is None and (start < 0 or start + k.shape[2] > cap):
        raise ValueError(f"kv8_append: {k.shape[2]} tokens at {start} do not fit a cache of {cap}")
    if counts is not None:
        counts, _ = _per_row(counts, "counts", b, k.device, torch.int32)
    torch_ref.kv8_append(cache.k, cache.v, cache.k_scale, cache.v_scale, k, v,
                         start if starts is None else starts, counts)


def decode_attention_kv8(q: torch.Tensor, cache: KVCache8, lengths, bias=None, kpad=None,
                         scale: float = 1.0, max_len: int | None = None) -> torch.Tensor:
    """Attention of one query token a sequence over a :class:`KVCache8`.

    q: (B, Hq, 1, D), bf16 or fp16 on a GPU, Hq a multiple of the cache's heads
    (query head i reads cache head i // (Hq/H)).  ``lengths``: a number, or an int32 (B,) tensor
    that is taken as if clamped to 0..max_len.  ``max_len``: what no length
    exceeds; it sizes the launch (default: the number, or the capacity).
    bias: (1 or B, Hq, 1, >= max_len); kpad: (B, >= max_len) additive: a key
    with -inf is not there, whatever it holds.  A row without keys is 0.
    Scores are ``scale * q.k + bias + kpad``, in fp32 as are the sums.
    """
    if q.is_cuda and _use_hip(q):
        each = torch.is_tensor(lengths)
        return _load_ext().kv8_attn(q, cache.k, cache.v, cache.k_scale, cache.v_scale,
                                    lengths if each else None, 0 if each else lengths,
                                    -1 if max_len is None else max_len, max_len is not None, bias, kpad, scale)
    _no_grad("decode_attention_kv8", q, bias, kpad)
    b, h, cap, d = cache.k.shape
    if q.dim() != 4 or q.shape[0] != b or q.shape[2] != 1 or q.shape[3] != d or not h or q.shape[1] % h:
        raise ValueError(f"decode_attention_kv8: q {tuple(q.shape)} does not fit a cache of "
                         f"(B, H, ., D) = ({b}, {h}, ., {d})")
    if q.device != cache.k.device:
        raise ValueError(f"decode_attention_kv8: q on {q.device}, cache on {cache.k.device}")
    each, length = _per_row(lengths, "lengths", b, q.device, torch.int32)
    if each is None and not 0 <= length <= cap:
        raise ValueError(f"decode_attention_kv8: length {length} in a cache of {cap}")
    if max_len is None:
        max_len = cap if each is not None else length
    elif not 0 <= max_len or (each is None and length > max_len):
        raise ValueError(f"decode_attention_kv8: max_len {max_len} under the length")
    max_len = min(max_len, cap)
    if bias is not None and (bias.dim() != 4 or bias.shape[0] not in (1, b) or bias.shape[1] != q.shape[1]
                             or bias.shape[2] != 1 or bias.shape[3] < max_len or bias.device != q.device):
        raise ValueError(f"decode_attention_kv8: bias {tuple(bias.shape)} on {bias.device} is not "
                         f"(1 or {b}, {q.shape[1]}, 1, >= {max_len})")
    if kpad is not None and (kpad.dim() != 2 or kpad.shape[0] != b or kpad.shape[1] < max_len
                             or kpad.device != q.device):
        raise ValueError(f"decode_attention_kv8: kpad {tuple(kpad.shape)} on {kpad.device} is not "
                         f"({b}, >= {max_len})")
    return torch_ref.decode_attention_kv8(q, cache.k, cache.v, cache.k_scale, cache.v_scale,
                                          length if each is None else each, bias, kpad, scale, max_len)


# --------------------------------------------------------------------------- #
# choosing the token                                                          #
# --------------------------------------------------------------------------- #
def check_sampling(temperature, top_k, top_p, min_p) -> None:
    """Refuse sampling options that are out of range."""
    if not 0 <= temperature < math.inf or not 0 <= top_p <= 1 or not 0 <= min_p <= 1 or top_k < 0:
        raise ValueError("sampling: temperature and top_k are at least 0, top_p and min_p from 0 to 1; "
                         f"got {temperature}, {top_k}, {top_p}, {min_p}")


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0,
                  min_p=0.0, empty_token: int = -1) -> torch.Tensor:
    """One token a row of logits (B, V), bf16, fp16 or fp32 on a GPU, from given
    uniform numbers u (B,).

    With w = exp((x - max)/temperature) and the order "larger logit first, of
    equal ones the lower index": keep the first ``top_k`` (0: all), of those the
    shortest prefix with a sum of at least ``top_p`` of theirs (1: all), of
    those the ones with w >= ``min_p``; the token is the lowest index whose
    running sum of kept weights, in index order, is over u times their sum.
    Weights and sums are in 64 bits.  temperature 0 takes the first of the
    order.  Options are numbers, or a value for each row: float32 or float64
    (B,) tensors (int32 for top_k); values from tensors that are out of range count as the
    nearest in range.  NaN counts as -inf; a row with nothing above -inf gives
    ``empty_token``.  Weights under 2^-45 of the largest count as 0.
    Returns int64 (B,).
    """
    if logits.is_cuda and _use_hip(logits):
        is_t = torch.is_tensor
        t, k, p, m = is_t(temperature), is_t(top_k), is_t(top_p), is_t(min_p)
        return _load_ext().sample_tokens(
            logits, u, temperature if t else None, 1.0 if t else temperature,
            top_k if k else None, 0 if k else top_k, top_p if p else None, 1.0 if p else top_p,
            min_p if m else None, 0.0 if m else min_p, empty_token)
    if logits.dim() != 2 or not 1 <= logits.shape[1] <= 1 << 19:
        raise ValueError(f"sample_tokens: logits (B, V) with V from 1 to {1 << 19}, got {tuple(logits.shape)}")
    if u.shape != logits.shape[:1] or u.device != logits.device or u.dtype not in (torch.float32, torch.float64):
        raise ValueError(f"sample_tokens: u must be fp32 or fp64 ({logits.shape[0]},) on {logits.device}, "
                         f"got {u.dtype} {tuple(u.shape)} on {u.device}")
    _no_grad("sample_tokens", logits, u)
    rows, dev = logits.shape[0], logits.device
    temps, temperature = _per_row(temperature, "temperature", rows, dev, torch.float32)
    ks, top_k = _per_row(top_k, "top_k", rows, dev, torch.int32)
    ps, top_p = _per_row(top_p, "top_p", rows, dev, torch.float32)
    mins, min_p = _per_row(min_p, "min_p", rows, dev, torch.float32)
    check_sampling(temperature, top_k, top_p, min_p)
    pick = lambda each, one: one if each is None else each  # noqa: E731
    return torch_ref.sample_tokens(logits, u, pick(temps, temperature), pick(ks, top_k), pick(ps, top_p),
                                   pick(mins, min_p), empty_token)
