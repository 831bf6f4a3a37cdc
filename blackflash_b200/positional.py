"""Attention that knows positions: sliding windows with sinks, decoding steps against a
cache, a prefix shared by a batch, rotary positions.

Torch-facing operators over the C ABI, in the manner of ops.py: checks raise RuntimeError,
work goes to the current stream of the tensors' device, outputs are fresh contiguous
tensors, and there is no CPU fallback. The reference has no counterpart of these.

Head layouts: queries [B, Hq, N, d], keys and values [B, Hkv, N, d] with Hq a multiple of
Hkv (query head h reads KV head h // (Hq // Hkv)); d = 64 or 128; bf16 or fp16. The tensors
may be strided views (a [B, N, H, d] projection transposed, a slice of a larger cache) as
long as the last axis is contiguous and the others step by multiples of 16 bytes.
"""
from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _require, _stream_handle

_HALF = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
_ANY = {**_HALF, torch.float32: _lib.DTYPE_F32}


def _view(t: torch.Tensor) -> _lib.View:
    """The last three strides of [.., heads, tokens, d], and the batch's where there is one."""
    s = t.stride()
    return _lib.View(t.data_ptr(), (ctypes.c_longlong * 3)(s[0] if t.dim() == 4 else 0, s[-3], s[-2]))


def _check(name: str, t: torch.Tensor, dims: int, like: torch.Tensor | None = None, types=_HALF) -> None:
    _require(isinstance(t, torch.Tensor), f"{name} must be a torch.Tensor")
    _require(t.is_cuda and t.dtype in types, f"{name} must be a CUDA tensor of " +
             ", ".join(str(x).removeprefix("torch.") for x in types))
    _require(t.dim() == dims, f"{name} must have {dims} axes")
    _require(t.size(-1) <= 1 or t.stride(-1) == 1, f"{name}'s last axis must be contiguous")
    if like is not None:
        _require(t.dtype == like.dtype and t.device == like.device, f"{name} must have Q's type and device")


def _check_grouped(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, names=("K", "V")) -> None:
    _check("Q", Q, 4)
    _require(Q.size(3) in (64, 128), "BlackFlash supports d=64 and d=128")
    for name, t in zip(names, (K, V)):
        _check(name, t, 4, Q)
    _require(K.shape == V.shape and K.size(0) == Q.size(0) and K.size(3) == Q.size(3),
             f"{names[0]} and {names[1]} must have one shape, with Q's batch and d")
    _require(K.size(1) > 0 and Q.size(1) % K.size(1) == 0, "query heads must be a multiple of KV heads")


def _check_scale(scale: float | None, d: int) -> float:
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    _require(math.isfinite(scale) and scale > 0, "scale must be positive and finite")
    return scale


def _check_window(window: int, sinks: int) -> tuple[int, int]:
    _require(window >= 1 and sinks >= 0, "need window >= 1 and sinks >= 0")
    return min(int(window), 0x7FFFFFFF), min(int(sinks), 0x7FFFFFFF)


# ---------------------------------------------------------------- sliding window

def window_attention_lse(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, window: int, sinks: int = 0,
                         scale: float | None = None, want_lse: bool = True):
    """Causal attention over the last `window` keys and the first `sinks` ones.

    Query i stands at position p = i + Nkv - Nq (the last query at the last key) and sees
    the keys j <= p with j > p - window or j < sinks; window >= Nkv is causal attention.
    Returns (O [B, Hq, Nq, d], lse [B, Hq, Nq] fp32); a query that sees no key (p < 0) gets
    0 and -inf. K and V must be finite in every row, those of padding too: a masked key has
    weight 0, but 0 times an infinity or NaN is NaN.
    """
    _check_grouped(Q, K, V)
    window, sinks = _check_window(window, sinks)
    scale = _check_scale(scale, Q.size(3))
    B, Hq, Nq, d = Q.shape
    Hkv, Nkv = K.size(1), K.size(2)
    O = torch.empty((B, Hq, Nq, d), dtype=Q.dtype, device=Q.device)
    lse = torch.empty((B, Hq, Nq), dtype=torch.float32, device=Q.device) if want_lse else None
    if O.numel() == 0:
        return O, lse
    if Nkv == 0:
        return O.zero_(), lse.fill_(-math.inf) if want_lse else None
    with torch.cuda.device(Q.device):
        rc = _lib.load().blackflash_window_fwd(
            _view(Q), _view(K), _view(V), O.data_ptr(), lse.data_ptr() if want_lse else None, B, Hq, Hkv, Nq, Nkv, d,
            window, sinks, scale, _HALF[Q.dtype], _stream_handle(Q.device))
    _lib.check(rc, "blackflash_window_fwd")
    return O, lse


def window_attention(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, window: int, sinks: int = 0,
                     scale: float | None = None) -> torch.Tensor:
    """`window_attention_lse` without the logsumexp; scale defaults to 1/sqrt(d)."""
    return window_attention_lse(Q, K, V, window, sinks, scale, want_lse=False)[0]


def window_attention_backward(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, O: torch.Tensor, dO: torch.Tensor,
                              lse: torch.Tensor, window: int, sinks: int = 0, scale: float | None = None):
    """Gradients (dQ, dK, dV) of `window_attention` for upstream dO; bf16.

    O and lse as `window_attention_lse` returned them; dO [B, Hq, Nq, d] may be a strided
    view. dK and dV are summed over the query heads that share a KV head."""
    _check_grouped(Q, K, V)
    _require(Q.dtype == torch.bfloat16, "the backward supports bfloat16")
    window, sinks = _check_window(window, sinks)
    scale = _check_scale(scale, Q.size(3))
    _check("O", O, 4, Q)
    _check("dO", dO, 4, Q)
    _require(O.shape == Q.shape and dO.shape == Q.shape and O.is_contiguous(), "O must be contiguous, O and dO of Q's shape")
    _require(isinstance(lse, torch.Tensor) and lse.dtype == torch.float32 and lse.device == Q.device
             and lse.is_contiguous() and lse.shape == Q.shape[:3], "lse must be a contiguous fp32 [B, Hq, Nq] tensor")
    B, Hq, Nq, d = Q.shape
    Hkv, Nkv = K.size(1), K.size(2)
    dQ, dK, dV = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (Q, K, V))
    if Q.numel() == 0 or K.numel() == 0:
        return dQ.zero_(), dK.zero_(), dV.zero_()
    lib = _lib.load()
    with torch.cuda.device(Q.device):
        nbytes = lib.blackflash_window_bwd_workspace_bytes(B, Hq, Hkv, Nq, Nkv, d, window, sinks)
        if nbytes < 0:
            _lib.check(_lib.BF_ERR_ARG, "blackflash_window_bwd_workspace_bytes")
        ws = torch.empty(nbytes, dtype=torch.uint8, device=Q.device)
        rc = lib.blackflash_window_bwd(
            _view(Q), _view(K), _view(V), O.data_ptr(), _view(dO), lse.data_ptr(), dQ.data_ptr(), dK.data_ptr(),
            dV.data_ptr(), ws.data_ptr(), nbytes, B, Hq, Hkv, Nq, Nkv, d, window, sinks, scale, _stream_handle(Q.device))
    _lib.check(rc, "blackflash_window_bwd")
    return dQ, dK, dV


class _WindowFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, Q, K, V, window, sinks, scale):
        O, lse = window_attention_lse(Q, K, V, window, sinks, scale)
        ctx.save_for_backward(Q, K, V, O, lse)
        ctx.args = (window, sinks, scale)
        return O

    @staticmethod
    @once_differentiable
    def backward(ctx, dO):
        Q, K, V, O, lse = ctx.saved_tensors
        return (*window_attention_backward(Q, K, V, O, _rows(dO), lse, *ctx.args), None, None, None)


def window_attention_with_grad(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, window: int, sinks: int = 0,
                               scale: float | None = None) -> torch.Tensor:
    """`window_attention` as a differentiable op; bf16."""
    _require(Q.dtype == torch.bfloat16, "the backward supports bfloat16")
    return _WindowFn.apply(Q, K, V, window, sinks, scale)


# ---------------------------------------------------------------- decoding steps

def _check_step(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, lengths: torch.Tensor) -> None:
    _check_grouped(Q, K, V, ("K_cache", "V_cache"))
    _require(isinstance(lengths, torch.Tensor) and lengths.is_cuda and lengths.dtype == torch.int32
             and lengths.device == Q.device and lengths.dim() == 1 and lengths.is_contiguous()
             and lengths.size(0) == Q.size(0), "lengths must be a contiguous int32 [B] tensor on Q's device")


def _step_buffers(Q: torch.Tensor, want_lse: bool, sizes: tuple):
    """O, lse and the workspace of a decoding step."""
    nbytes = _lib.load().blackflash_decode_workspace_bytes(*sizes)
    if nbytes < 0:
        _lib.check(_lib.BF_ERR_ARG, "blackflash_decode_workspace_bytes")
    O = torch.empty(Q.shape, dtype=Q.dtype, device=Q.device)
    lse = torch.empty(Q.shape[:3], dtype=torch.float32, device=Q.device) if want_lse else None
    ws = torch.empty(nbytes, dtype=torch.uint8, device=Q.device) if nbytes else None
    return O, lse, ws, nbytes


def window_decode(Q: torch.Tensor, K_cache: torch.Tensor, V_cache: torch.Tensor, lengths: torch.Tensor, window: int,
                  sinks: int = 0, scale: float | None = None, want_lse: bool = False):
    """The step of T new tokens a sequence, Q [B, Hq, T, d], against caches [B, Hkv, C, d].

    lengths [B] int32 counts the tokens in use of each cache, the T new ones among them
    (held to 0 .. C); new token t stands at position p = lengths[b] - T + t and sees the
    keys j <= p with j > p - window or j < sinks. Returns O [B, Hq, T, d], or (O, lse) with
    want_lse; a token that sees no key (p < 0) gets 0 and -inf. Cache rows at lengths[b]
    and after are never read and may hold anything.
    """
    _check_step(Q, K_cache, V_cache, lengths)
    window, sinks = _check_window(window, sinks)
    scale = _check_scale(scale, Q.size(3))
    B, Hq, T, d = Q.shape
    Hkv, C = K_cache.size(1), K_cache.size(2)
    if Q.numel() == 0 or C == 0:
        O = torch.zeros(Q.shape, dtype=Q.dtype, device=Q.device)
        return (O, torch.full((B, Hq, T), -math.inf, device=Q.device)) if want_lse else O
    Q = Q.contiguous()
    with torch.cuda.device(Q.device):
        O, lse, ws, nbytes = _step_buffers(Q, want_lse, (B, Hq, Hkv, T, 0, C, d, window, sinks))
        rc = _lib.load().blackflash_window_decode(
            Q.data_ptr(), _view(K_cache), _view(V_cache), lengths.data_ptr(), O.data_ptr(),
            lse.data_ptr() if want_lse else None, ws.data_ptr() if nbytes else None, nbytes, B, Hq, Hkv, T, C, d, window,
            sinks, scale, _HALF[Q.dtype], _stream_handle(Q.device))
    _lib.check(rc, "blackflash_window_decode")
    return (O, lse) if want_lse else O


def prefix_decode(Q: torch.Tensor, K_prefix: torch.Tensor, V_prefix: torch.Tensor, K_cache: torch.Tensor,
                  V_cache: torch.Tensor, lengths: torch.Tensor, scale: float | None = None, want_lse: bool = False):
    """The step of T new tokens a sequence, Q [B, Hq, T, d], for a batch behind one prefix.

    K_prefix, V_prefix [Hkv, P, d] are shared by all sequences and are read once for the
    whole batch; K_cache, V_cache [B, Hkv, C, d] hold what each sequence has of its own,
    lengths [B] int32 of it, the T new tokens among them. New token t of sequence b sees the
    whole prefix and the keys j <= lengths[b] - T + t of its own cache. P or C may be 0.
    Returns O [B, Hq, T, d], or (O, lse) with want_lse; a token that sees no key gets 0 and
    -inf. Cache rows at lengths[b] and after are never read and may hold anything.
    """
    _check_step(Q, K_cache, V_cache, lengths)
    for name, t in (("K_prefix", K_prefix), ("V_prefix", V_prefix)):
        _check(name, t, 3, Q)
    B, Hq, T, d = Q.shape
    Hkv, C = K_cache.size(1), K_cache.size(2)
    _require(K_prefix.shape == V_prefix.shape and K_prefix.size(0) == Hkv and K_prefix.size(2) == d,
             "K_prefix and V_prefix must be [Hkv, P, d]")
    scale = _check_scale(scale, d)
    P = K_prefix.size(1)
    if Q.numel() == 0 or P + C == 0:
        O = torch.zeros(Q.shape, dtype=Q.dtype, device=Q.device)
        return (O, torch.full((B, Hq, T), -math.inf, device=Q.device)) if want_lse else O
    Q = Q.contiguous()
    with torch.cuda.device(Q.device):
        O, lse, ws, nbytes = _step_buffers(Q, want_lse, (B, Hq, Hkv, T, P, C, d, 0x7FFFFFFF, 0))
        rc = _lib.load().blackflash_prefix_decode(
            Q.data_ptr(), _view(K_prefix), _view(V_prefix), _view(K_cache), _view(V_cache), lengths.data_ptr(),
            O.data_ptr(), lse.data_ptr() if want_lse else None, ws.data_ptr() if nbytes else None, nbytes, B, Hq, Hkv, T, P,
            C, d, scale, _HALF[Q.dtype], _stream_handle(Q.device))
    _lib.check(rc, "blackflash_prefix_decode")
    return (O, lse) if want_lse else O


# ---------------------------------------------------------------- rotary positions

def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                       original_length: int | None = None, beta_fast: float = 32.0, beta_slow: float = 1.0,
                       device: torch.device | str | None = None) -> tuple[torch.Tensor, float]:
    """Angles per position of the rotated pairs, fp64 [rotary_dim / 2], and the amplitude.

    Pair i turns by base^(-2i / rotary_dim) radians per position. `scaling` stretches a
    model's context by `factor`:
      "linear"   every frequency divided by factor (positions interpolated);
      "ntk"      the base raised to base * factor^(rotary_dim / (rotary_dim - 2)), which
                 leaves the fastest pair and divides the slowest by factor;
      "by-parts" pairs that turn more than beta_fast times within original_length stay,
                 those that turn less than beta_slow times are divided by factor, a linear
                 ramp over the pair's index between; the amplitude is 0.1 ln(factor) + 1.
    The amplitude is 1 otherwise. Both are a plan: made once and passed to every `rotary`.
    """
    _require(rotary_dim >= 2 and rotary_dim % 2 == 0, "rotary_dim must be even and at least 2")
    _require(base > 1 and factor >= 1, "need base > 1 and factor >= 1")
    _require(scaling in (None, "linear", "ntk", "by-parts"), "scaling must be None, 'linear', 'ntk' or 'by-parts'")
    if scaling == "ntk":
        _require(rotary_dim > 2, "ntk scaling needs rotary_dim > 2")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    pair = torch.arange(rotary_dim // 2, dtype=torch.float64)
    freqs = base ** (-2.0 * pair / rotary_dim)
    amplitude = 1.0
    if scaling == "linear":
        freqs = freqs / factor
    elif scaling == "by-parts":
        _require(original_length is not None and original_length >= 1 and beta_fast > beta_slow > 0,
                 "by-parts scaling needs original_length and beta_fast > beta_slow > 0")

        def index_of(turns: float) -> float:  # of the pair that turns that often within original_length
            return rotary_dim * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))

        lo = max(math.floor(index_of(beta_fast)), 0)
        hi = min(math.ceil(index_of(beta_slow)), rotary_dim - 1)
        ramp = ((pair - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        freqs = freqs * (1 - ramp) + freqs / factor * ramp
        amplitude = 0.1 * math.log(factor) + 1.0
    return freqs.to(device if device is not None else "cuda"), amplitude


def rotary(Q: torch.Tensor, K: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, interleaved: bool = False,
           amplitude: float = 1.0, inverse: bool = False):
    """Q [B, Hq, N, d] and K [B, Hk, N, d] with their first 2 * len(freqs) columns turned by
    position: pair i of a token at position n by n * freqs[i] radians, times amplitude.

    Pair i is the columns (2i, 2i + 1) with interleaved, else (i, i + len(freqs)). positions
    is [N] or [B, N], int32 or int64; freqs is fp64 (`rotary_frequencies`). Columns past the
    rotated part are copied. inverse turns the other way (the gradient's map). bf16, fp16 or
    fp32, any even d up to 1024; returns contiguous (Q', K').
    """
    _check("Q", Q, 4, types=_ANY)
    _check("K", K, 4, Q, types=_ANY)
    B, Hq, N, d = Q.shape
    _require(K.size(0) == B and K.size(2) == N and K.size(3) == d, "K must have Q's batch, tokens and d")
    for name, t in (("positions", positions), ("freqs", freqs)):
        _require(isinstance(t, torch.Tensor) and t.device == Q.device and t.is_contiguous(),
                 f"{name} must be a contiguous tensor on Q's device")
    _require(positions.dtype in (torch.int32, torch.int64) and positions.shape in ((N,), (B, N)),
             "positions must be int32 or int64, [N] or [B, N]")
    _require(freqs.dtype == torch.float64 and freqs.dim() == 1, "freqs must be fp64 [rotary_dim / 2]")
    rot = 2 * freqs.numel()
    _require(d % 2 == 0 and d <= 1024 and 2 <= rot <= d, "need an even d <= 1024 and 1 to d / 2 frequencies")
    _require(math.isfinite(amplitude), "amplitude must be finite")
    Qo = torch.empty(Q.shape, dtype=Q.dtype, device=Q.device)
    Ko = torch.empty(K.shape, dtype=Q.dtype, device=Q.device)
    if Qo.numel() + Ko.numel() == 0:
        return Qo, Ko
    with torch.cuda.device(Q.device):
        rc = _lib.load().blackflash_rotary(
            _view(Q), _view(K), Qo.data_ptr(), Ko.data_ptr(), positions.data_ptr(), positions.dtype == torch.int64,
            positions.dim() == 2, freqs.data_ptr(), B, Hq, K.size(1), N, d, rot, bool(interleaved), float(amplitude),
            bool(inverse), _ANY[Q.dtype], _stream_handle(Q.device))
    _lib.check(rc, "blackflash_rotary")
    return Qo, Ko


class _RotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, Q, K, positions, freqs, interleaved, amplitude):
        ctx.save_for_backward(positions, freqs)
        ctx.args = (interleaved, amplitude)
        return rotary(Q, K, positions, freqs, interleaved, amplitude)

    @staticmethod
    @once_differentiable
    def backward(ctx, dQ, dK):
        # The map is linear, so its gradient is its transpose: the same turn backwards.
        positions, freqs = ctx.saved_tensors
        dQ, dK = rotary(_rows(dQ), _rows(dK), positions, freqs, *ctx.args, inverse=True)
        return dQ, dK, None, None, None, None


def _rows(t: torch.Tensor) -> torch.Tensor:
    """A gradient as the kernels read it: its rows contiguous, and not broadcast."""
    return t if t.stride(-1) == 1 and 0 not in t.stride() else t.contiguous()


def rotary_with_grad(Q: torch.Tensor, K: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor,
                     interleaved: bool = False, amplitude: float = 1.0):
    """`rotary` as a differentiable op; gradients for Q and K, not for the frequencies."""
    return _RotaryFn.apply(Q, K, positions, freqs, interleaved, amplitude)
