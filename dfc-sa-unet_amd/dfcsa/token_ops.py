"""Operators of a transformer block over image, video or text tokens (kernels: csrc/token_ops.hip and
csrc/window_attn.hip).  They stand beside the ViT block's LayerNorm, learned positions and multi-head
attention of transunet_ops.py, for token counts and grids that those are not made for:

  rms_norm_residual        (y, r): r = x + residual, y = rms_norm(r) * weight         differentiable
  rms_norm_residual_q8     the same with y in 8 bits (e4m3) and scales                 serving
  dequant_q8               those 8 bits back to bf16 or fp32
  rotary                   rotary positions with one to four axes on q and k           differentiable
  window_attention         sliding window + always-visible first tokens, grouped heads differentiable
  window_attention_cached  the same for new tokens at the end of a cache               serving

The host side (checks, allocation, autograd nodes) is the extension module dfcsa._tokens, built from
csrc/token_bind.cpp; a missing one raises ImportError, there is no fallback.

Types: bf16 or fp32 (the framework's two precisions), statistics and sums in fp32.  Every function
enqueues on the current stream of its tensors' device, allocates from torch's caching allocator only
(so it can be captured into a graph) and never synchronises.  Arguments are checked on the host:
ValueError for shapes and values, TypeError for types, RuntimeError for tensors that are not on the
GPU.  Results do not depend on the order in which workgroups run.  Gradients are first order only; what torch
would need an operator of its own for (forward-mode tangents, torch.func's transforms, torch.jit.trace,
make_fx and torch.export, tensor subclasses with a dispatch of their own) is refused with a RuntimeError.
"""
import ctypes
import functools
import math

import torch

from ._lib import LIB

try:
    from . import _tokens
except ImportError as e:
    raise ImportError("dfcsa/_tokens.so is missing or does not fit this torch: build it with `python -c 'import "
                      f"__graft_entry__ as g; g.build()'` (or `make -C dfc-sa-unet_amd/csrc`): {e}") from e

_tokens.bind({n: ctypes.cast(getattr(LIB, n), ctypes.c_void_p).value for n in (
    "dfcsa_rms_fwd", "dfcsa_rms_fwd_q8", "dfcsa_rms_bwd_work_floats", "dfcsa_rms_bwd", "dfcsa_dequant_q8",
    "dfcsa_rotary", "dfcsa_wattn_work_floats", "dfcsa_wattn_fwd", "dfcsa_wattn_bwd")})

E4M3 = torch.float8_e4m3fn


def _whole(v, what):
    try:
        i = int(v)
    except OverflowError:   # infinity
        raise ValueError(f"{what} {v}: a whole number is needed") from None
    if i != v:
        raise ValueError(f"{what} {v}: a whole number is needed")
    return max(-1 << 62, min(i, 1 << 62))   # more than there are tokens is as good as any number of them


# ------------------------------------------------------------------ RMS norm of the residual stream
def rms_norm_residual(x, residual, weight, eps=1e-6):
    """(y, r) of x, residual [..., C] and weight [C]: r = x + residual in residual's type (the stream),
    y = r / sqrt(mean(r^2) + eps) * weight in x's type; the norm is of r as it is stored.

    x bf16 with a bf16 or fp32 residual, or both fp32; weight fp32; C a multiple of 8 up to 16384.
    Differentiable in all three (y's and r's gradients are used; either may be missing)."""
    return _tokens.rms_norm_residual(x, residual, weight, eps)


def rms_norm_residual_q8(x, residual, weight, eps=1e-6, group=0):
    """(y8, scales, r): as rms_norm_residual, with y in 8 bits: y8 (float8_e4m3fn) * scales is y.

    scales [..., C / group] fp32, one for each `group` columns (32, 64 or 128) or, group = 0, one for
    the row: max(max|y|, 1e-12) / 448.  A NaN or infinity makes its group's scale NaN or infinite.
    For serving: it has no gradient, and refuses inputs that ask for one."""
    return _tokens.rms_norm_residual_q8(x, residual, weight, eps, group)


def dequant_q8(y8, scales, dtype=torch.bfloat16):
    """y8 * scales in bf16 or fp32, for y8 and scales as rms_norm_residual_q8 gives them."""
    return _tokens.dequant_q8(y8, scales, dtype)


# ------------------------------------------------------------------ rotary positions
@functools.lru_cache(maxsize=64)
def _turn_table(axes, base, shared):
    """Turns per position of each pair and its axis (constants of a shape, no input's)."""
    return _tokens.TurnTable([_whole(a, "axes") for a in axes], base, shared)


def rotary(q, k, positions, axes, base=10000.0, shared=False, interleaved=False):
    """(q, k) turned by their tokens' positions; q [B, N, H, D], k [B, N, Hk, D] or None (then None).

    positions: int32 or int64, [B, N, A] or [N, A]: where the token is on each of the A axes (row and
    column of a patch, or time, row and column).  axes: how many channel pairs each axis turns, e.g.
    (16, 16) for a width of 64; channels beyond 2 * sum(axes) stay as they are.  Pair i of an axis with
    n pairs turns by base^(-i/n) a position; with shared = True all axes share one ladder, pair j of the
    sum turning by base^(-j/sum).  Pairs are channels (j, sum + j), or (2j, 2j + 1) if interleaved.
    The angle is formed in 64 bits, so far positions keep their precision.  The gradient turns back.
    q and k are read in place from any strides with contiguous channels; the results are contiguous."""
    return _tokens.rotary(q, k, positions, _turn_table(tuple(axes), float(base), bool(shared)), bool(interleaved))


# ------------------------------------------------------------------ attention
def _scale(scale, q):
    return 1.0 / math.sqrt(q.shape[-1] if q.dim() and q.shape[-1] else 1) if scale is None else float(scale)


def window_attention(q, k, v, window, sinks=0, causal=True, scale=None, lengths=None):
    """Attention of each token over the tokens near it and the first `sinks` ones: [B, N, H, D] for
    q [B, N, H, D] and k, v [B, N, Hk, D], H a multiple of Hk (query head h reads key head h // (H / Hk)).

    Token p sees token j when |p - j| < window or j < sinks, and, if causal, j <= p.  window = N (or
    more) is plain attention.  scale: of the scores, 1/sqrt(D) unless given.  lengths: int32 [B], the
    valid tokens of each sequence, the first ones (clamped to [0, N]); rows behind them are padding:
    whatever they hold, they are not seen, their results and gradients are zeros.  A NaN or infinity reaches
    what sees it, however small its weight, and nothing else; it costs time (a call about four times as long).
    bf16 or fp32, D a multiple of 8 up to 128.  Differentiable in q, k and v.  Tensors are read in place
    where their channels are contiguous and their strides multiples of 16 bytes, else from a copy.
    The cost follows N * (window + sinks); nothing N x N is stored."""
    return _tokens.window_attention(q, k, v, _whole(window, "window"), _whole(sinks, "sinks"), bool(causal),
                                    _scale(scale, q), lengths)


def window_attention_cached(q, k_cache, v_cache, lengths, window, sinks=0, scale=None):
    """window_attention (causal) of the last T tokens of each sequence, q [B, T, H, D], over caches
    [B, capacity, Hk, D] that hold lengths[b] tokens (int32 [B], these T among them; clamped to
    [0, capacity]): token t is at position lengths[b] - T + t, and one before the start of its sequence
    gives zeros.  What the caches hold behind a sequence's end is not read.  For serving: it has no
    gradient, and refuses inputs that ask for one."""
    if lengths is None:
        raise TypeError("lengths: int32 [batch] is needed")
    return _tokens.window_attention_cached(q, k_cache, v_cache, lengths, _whole(window, "window"),
                                           _whole(sinks, "sinks"), _scale(scale, q))
