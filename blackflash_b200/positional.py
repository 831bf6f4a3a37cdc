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

import math

import torch

from .ops import _require

_MAX = 1 << 62
_module = None


def _ext():
    """The torch binding (csrc/torch_positional.cpp): it checks the arguments, allocates outputs
    and workspaces, and calls the C ABI on the tensors' device and current stream."""
    global _module
    if _module is None:
        try:
            from . import _positional as module
        except ImportError as e:
            raise RuntimeError("blackflash_b200._positional is not built; build it with "
                               "`python -m blackflash_b200.build` (needs nvcc and g++)") from e
        _module = module
    return _module


def _tensors(**named) -> None:
    for name, t in named.items():
        _require(isinstance(t, torch.Tensor), f"{name} must be a torch.Tensor")


# ---------------------------------------------------------------- sliding window

def window_attention_lse(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, window: int, sinks: int = 0,
                         scale: float | None = None, want_lse: bool = True):
    """Causal attention over the last `window` keys and the first `sinks` ones.

    Query i stands at position p = i + Nkv - Nq (the last query at the last key) and sees
    the keys j <= p with j > p - window or j < sinks; window >= Nkv is causal attention.
    Returns (O [B, Hq, Nq, d], lse [B, Hq, Nq] fp32); a query that sees no key (p < 0) gets
    0 and -inf. K and V must be finite in every row, those of padding too: a masked key has
    weight 0, but 0 times an infinity or NaN is NaN. A row that sees a score of NaN or +inf is
    NaN.
    """
    _tensors(Q=Q, K=K, V=V)
    return _ext().window_lse(Q, K, V, min(window, _MAX), min(sinks, _MAX), scale, want_lse)


def window_attention(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, window: int, sinks: int = 0,
                     scale: float | None = None) -> torch.Tensor:
    """`window_attention_lse` without the logsumexp; scale defaults to 1/sqrt(d)."""
    return window_attention_lse(Q, K, V, window, sinks, scale, want_lse=False)[0]


def window_attention_backward(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, O: torch.Tensor, dO: torch.Tensor,
                              lse: torch.Tensor, window: int, sinks: int = 0, scale: float | None = None):
    """Gradients (dQ, dK, dV) of `window_attention` for upstream dO; bf16.

    O and lse as `window_attention_lse` returned them; dO [B, Hq, Nq, d] may be a strided
    view. dK and dV are summed over the query heads that share a KV head."""
    _tensors(Q=Q, K=K, V=V, O=O, dO=dO, lse=lse)
    return _ext().window_backward(Q, K, V, O, dO, lse, min(window, _MAX), min(sinks, _MAX), scale)


def window_attention_with_grad(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, window: int, sinks: int = 0,
                               scale: float | None = None) -> torch.Tensor:
    """`window_attention` as a differentiable op (once: no create_graph); bf16.

    Forward and backward may be captured together into a CUDA graph, except while a graph of
    the same leaves that was made on the default stream is alive: that backward is refused."""
    _tensors(Q=Q, K=K, V=V)
    return _ext().window_with_grad(Q, K, V, min(window, _MAX), min(sinks, _MAX), scale)


# ---------------------------------------------------------------- decoding steps

def window_decode(Q: torch.Tensor, K_cache: torch.Tensor, V_cache: torch.Tensor, lengths: torch.Tensor, window: int,
                  sinks: int = 0, scale: float | None = None, want_lse: bool = False):
    """The step of T new tokens a sequence, Q [B, Hq, T, d], against caches [B, Hkv, C, d].

    lengths [B] int32 counts the tokens in use of each cache, the T new ones among them
    (held to 0 .. C); new token t stands at position p = lengths[b] - T + t and sees the
    keys j <= p with j > p - window or j < sinks. Returns O [B, Hq, T, d], or (O, lse) with
    want_lse; a token that sees no key (p < 0) gets 0 and -inf. Cache rows at lengths[b]
    and after are never read and may hold anything; V's rows of the step's own tokens and of
    its window must be finite, for the other tokens too.
    """
    _tensors(Q=Q, K_cache=K_cache, V_cache=V_cache, lengths=lengths)
    O, lse = _ext().window_decode(Q, K_cache, V_cache, lengths, min(window, _MAX), min(sinks, _MAX), scale, want_lse)
    return (O, lse) if want_lse else O


def prefix_decode(Q: torch.Tensor, K_prefix: torch.Tensor, V_prefix: torch.Tensor, K_cache: torch.Tensor,
                  V_cache: torch.Tensor, lengths: torch.Tensor, scale: float | None = None, want_lse: bool = False):
    """The step of T new tokens a sequence, Q [B, Hq, T, d], for a batch behind one prefix.

    K_prefix, V_prefix [Hkv, P, d] are shared by all sequences, and a long one is read
    once for the whole batch; K_cache, V_cache [B, Hkv, C, d] hold what each sequence has of its own,
    lengths [B] int32 of it, the T new tokens among them. New token t of sequence b sees the
    whole prefix and the keys j <= lengths[b] - T + t of its own cache. P or C may be 0.
    Returns O [B, Hq, T, d], or (O, lse) with want_lse; a token that sees no key gets 0 and
    -inf. Cache rows at lengths[b] and after are never read and may hold anything.
    """
    _tensors(Q=Q, K_prefix=K_prefix, V_prefix=V_prefix, K_cache=K_cache, V_cache=V_cache, lengths=lengths)
    O, lse = _ext().prefix_decode(Q, K_prefix, V_prefix, K_cache, V_cache, lengths, scale, want_lse)
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

        # Not held to the pairs that exist: either end may lie beyond the first or the last one.
        lo, hi = math.floor(index_of(beta_fast)), math.ceil(index_of(beta_slow))
        ramp = ((pair - lo) / max(hi - lo, 1)).clamp(0, 1)
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
    _tensors(Q=Q, K=K, positions=positions, freqs=freqs)
    return _ext().rotary(Q, K, positions, freqs, interleaved, amplitude, inverse)


def rotary_with_grad(Q: torch.Tensor, K: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor,
                     interleaved: bool = False, amplitude: float = 1.0):
    """`rotary` as a differentiable op (once: no create_graph); gradients for Q and K, not for
    the frequencies. For CUDA graphs as `window_attention_with_grad`."""
    _tensors(Q=Q, K=K, positions=positions, freqs=freqs)
    return _ext().rotary_with_grad(Q, K, positions, freqs, interleaved, amplitude)