"""Operators of a transformer block over image, video or text tokens (kernels: csrc/token_ops.hip and
csrc/window_attn.hip).  They stand beside the ViT block's LayerNorm, learned positions and multi-head
attention of transunet_ops.py, for token counts and grids that those are not made for:

  rms_norm_residual        (y, r): r = x + residual, y = rms_norm(r) * weight         differentiable
  rms_norm_residual_q8     the same with y in 8 bits (e4m3) and scales                 serving
  dequant_q8               those 8 bits back to bf16 or fp32
  rotary                   rotary positions with one to four axes on q and k           differentiable
  window_attention         sliding window + always-visible first tokens, grouped heads differentiable
  window_attention_cached  the same for new tokens at the end of a cache               serving

Types: bf16 or fp32 (the framework's two precisions), statistics and sums in fp32.  Every function
enqueues on the current stream of its tensors' device, allocates from torch's caching allocator only
(so it can be captured into a graph) and never synchronises.  Arguments are checked on the host:
ValueError for shapes and values, TypeError for types, RuntimeError for tensors that are not on the
GPU.  Results do not depend on the order in which workgroups run.  Gradients are first order only.
"""
import ctypes
import functools
import math

import torch

from . import _lib
from ._lib import LIB, DfcsaError, call

E4M3 = torch.float8_e4m3fn
_DT = {torch.bfloat16: _lib.DT_BF16, torch.float32: _lib.DT_F32}
_INT_MAX = 2 ** 31 - 1


def _first_order(backward):
    """A backward that refuses create_graph: its kernels are not differentiated, and the second-order
    part would be missing without a word."""
    @functools.wraps(backward)
    def run(ctx, *grads):
        if torch.is_grad_enabled():
            raise RuntimeError("dfcsa.token_ops: gradients are first order only (create_graph=True is refused)")
        return backward(ctx, *grads)
    return run


def _need_gpu(*tensors):
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("dfcsa kernels need GPU tensors (MI355X/ROCm); got a CPU tensor")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f"tensors on {dev} and {t.device}: one device is needed")
    return dev


def _dtype(t, what):
    try:
        return _DT[t.dtype]
    except KeyError:
        raise TypeError(f"{what}: bfloat16 or float32 is needed, got {t.dtype}") from None


def _launch(dev, name, *args):
    """The entry point on the current stream of `dev`, whichever device is current."""
    s = torch._C._cuda_getCurrentRawStream(dev.index)
    if dev.index == torch._C._cuda_getDevice():
        return call(name, *args, s)
    with torch.cuda.device(dev):
        return call(name, *args, s)


def _packed(t):
    """Contiguous and 16-byte aligned (a copy where it is not)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


# ------------------------------------------------------------------ RMS norm of the residual stream
def _norm_args(x, residual, weight):
    dev = _need_gpu(x, residual, weight)
    ty, rt = _dtype(x, "x"), _dtype(residual, "residual")
    if x.shape != residual.shape or x.dim() < 1:
        raise ValueError(f"x {tuple(x.shape)} and residual {tuple(residual.shape)}: one shape [..., C] is needed")
    C = x.shape[-1]
    if C < 8 or C % 8 or C > 16384:
        raise ValueError(f"{C} columns: a multiple of 8 up to 16384 is needed")
    if weight.dtype != torch.float32 or weight.shape != (C,):
        raise (TypeError if weight.dtype != torch.float32 else ValueError)(
            f"weight: float32 of shape ({C},) is needed, got {weight.dtype} {tuple(weight.shape)}")
    if ty == _lib.DT_F32 and rt != _lib.DT_F32:
        raise TypeError("a float32 x needs a float32 residual")
    rows = x.numel() // C
    if rows > _INT_MAX:
        raise ValueError(f"{rows} rows: at most {_INT_MAX}")
    return dev, ty, rt, rows, C


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        dev, ty, rt, rows, C = _norm_args(x, residual, weight)
        x, residual, weight = _packed(x), _packed(residual), _packed(weight)
        y, r = torch.empty_like(x), torch.empty_like(residual)
        grad = any(ctx.needs_input_grad)
        rstd = torch.empty(rows, dtype=torch.float32, device=dev) if grad else None
        if rows:
            _launch(dev, "dfcsa_rms_fwd", ty, rt, rows, C, x.data_ptr(), residual.data_ptr(), weight.data_ptr(), eps,
                    y.data_ptr(), r.data_ptr(), rstd.data_ptr() if grad else None)
        if grad:
            ctx.save_for_backward(r, rstd, weight)
            ctx.meta = (dev, ty, rt, rows, C, x.dtype)
            ctx.set_materialize_grads(False)
        return y, r

    @staticmethod
    @_first_order
    def backward(ctx, dy, dr):
        r, rstd, weight = ctx.saved_tensors
        dev, ty, rt, rows, C, xt = ctx.meta
        need_x, need_r, need_w = ctx.needs_input_grad[:3]
        if dy is None and dr is None:
            return None, None, None, None
        dy = torch.zeros(r.shape, dtype=xt, device=dev) if dy is None else _packed(dy)
        dr = None if dr is None else _packed(dr)
        same = ty == rt   # then dx and dres are one tensor
        dx = torch.empty(r.shape, dtype=xt, device=dev) if need_x or (same and need_r) else None
        dres = torch.empty_like(r) if need_r and not same else None
        dw = work = None
        if need_w:
            dw = torch.empty_like(weight)
            work = torch.empty(LIB.dfcsa_rms_bwd_work_floats(rows, C), dtype=torch.float32, device=dev)
        if rows:
            _launch(dev, "dfcsa_rms_bwd", ty, rt, rows, C, dy.data_ptr(), None if dr is None else dr.data_ptr(),
                    r.data_ptr(), rstd.data_ptr(), weight.data_ptr(), None if dx is None else dx.data_ptr(),
                    None if dres is None else dres.data_ptr(), None if dw is None else dw.data_ptr(),
                    None if work is None else work.data_ptr(), 0 if work is None else work.numel())
        elif dw is not None:
            dw.zero_()
        return dx if need_x else None, (dx if same else dres) if need_r else None, dw, None


def rms_norm_residual(x, residual, weight, eps=1e-6):
    """(y, r) of x, residual [..., C] and weight [C]: r = x + residual in residual's type (the stream),
    y = r / sqrt(mean(r^2) + eps) * weight in x's type; the norm is of r as it is stored.

    x bf16 with a bf16 or fp32 residual, or both fp32; weight fp32; C a multiple of 8 up to 16384.
    Differentiable in all three (y's and r's gradients are used; either may be missing)."""
    return _RmsNorm.apply(x, residual, weight, _eps(eps))


def _eps(eps):
    eps = float(eps)
    if not (0.0 <= eps < math.inf):
        raise ValueError(f"eps {eps}: a finite value of at least 0 is needed")
    return eps


def _group(group, C):
    if group not in (0, 32, 64, 128):
        raise ValueError(f"group {group}: 0 (the whole row), 32, 64 or 128")
    if group and C % group:
        raise ValueError(f"{C} columns are no multiple of the group, {group}")
    return group


def rms_norm_residual_q8(x, residual, weight, eps=1e-6, group=0):
    """(y8, scales, r): as rms_norm_residual, with y in 8 bits: y8 (float8_e4m3fn) * scales is y.

    scales [..., C / group] fp32, one for each `group` columns (32, 64 or 128) or, group = 0, one for
    the row: max(max|y|, 1e-12) / 448.  A NaN or infinity makes its group's scale NaN or infinite.
    For serving: it has no gradient, and refuses inputs that ask for one."""
    if torch.is_grad_enabled() and (x.requires_grad or residual.requires_grad or weight.requires_grad):
        raise RuntimeError("rms_norm_residual_q8 has no gradient: call it under torch.no_grad(), or rms_norm_residual")
    dev, ty, rt, rows, C = _norm_args(x, residual, weight)
    group, eps = _group(group, C), _eps(eps)
    x, residual, weight = _packed(x), _packed(residual), _packed(weight)
    y8 = torch.empty(x.shape, dtype=E4M3, device=dev)
    scales = torch.empty((*x.shape[:-1], C // group if group else 1), dtype=torch.float32, device=dev)
    r = torch.empty_like(residual)
    if rows:
        _launch(dev, "dfcsa_rms_fwd_q8", ty, rt, rows, C, group, x.data_ptr(), residual.data_ptr(), weight.data_ptr(),
                eps, y8.data_ptr(), scales.data_ptr(), r.data_ptr())
    return y8, scales, r


def dequant_q8(y8, scales, dtype=torch.bfloat16):
    """y8 * scales in bf16 or fp32, for y8 and scales as rms_norm_residual_q8 gives them."""
    dev = _need_gpu(y8, scales)
    if y8.dtype != E4M3 or scales.dtype != torch.float32:
        raise TypeError(f"float8_e4m3fn values and float32 scales are needed, got {y8.dtype} and {scales.dtype}")
    if dtype not in _DT:
        raise TypeError(f"dtype: bfloat16 or float32 is needed, got {dtype}")
    if y8.dim() < 1 or scales.dim() != y8.dim() or scales.shape[:-1] != y8.shape[:-1]:
        raise ValueError(f"values {tuple(y8.shape)} and scales {tuple(scales.shape)} do not belong together")
    C, ng = y8.shape[-1], scales.shape[-1]
    if C < 8 or C % 8 or C > 16384 or ng < 1 or C % ng:
        raise ValueError(f"{ng} scales for {C} columns")
    group = 0 if ng == 1 else _group(C // ng, C)
    y8, scales = _packed(y8), scales.contiguous()
    out = torch.empty(y8.shape, dtype=dtype, device=dev)
    rows = y8.numel() // C
    if rows:
        _launch(dev, "dfcsa_dequant_q8", _DT[dtype], rows, C, group, y8.data_ptr(), scales.data_ptr(), out.data_ptr())
    return out


# ------------------------------------------------------------------ rotary positions
@functools.lru_cache(maxsize=64)
def _turn_table(axes, base, shared):
    """Turns per position of each pair and its axis, as host arrays (shape constants, no input's)."""
    total = sum(axes)
    turns = (ctypes.c_double * total)()
    axis = (ctypes.c_ubyte * total)()
    j = 0
    for a, n in enumerate(axes):
        for i in range(n):
            turns[j] = base ** (-(j / total if shared else i / n)) / (2.0 * math.pi)
            axis[j] = a
            j += 1
    return turns, axis


def _rotary_check(q, k, positions, axes, base):
    dev = _need_gpu(q, k, positions)
    ty = _dtype(q, "q")
    if q.dim() != 4 or (k is not None and k.dim() != 4):
        raise ValueError("q and k: [batch, tokens, heads, width] is needed")
    B, N, _, D = q.shape
    if k is not None:
        if k.dtype != q.dtype:
            raise TypeError(f"q {q.dtype} and k {k.dtype}: one type is needed")
        if k.shape[:2] != q.shape[:2] or k.shape[3] != D:
            raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} differ in more than their heads")
    if not axes or len(axes) > 4 or any(int(a) != a or a < 1 for a in axes):
        raise ValueError(f"axes {axes}: the rotated pairs of one to four axes, at least one each")
    total = sum(axes)
    if 2 * total > D or total > 256 or D > 1024:
        raise ValueError(f"{total} rotated pairs in a width of {D}: at most half of it, and 256")
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"positions: int32 or int64 is needed, got {positions.dtype}")
    if positions.shape != (B, N, len(axes)) and positions.shape != (N, len(axes)):
        raise ValueError(f"positions {tuple(positions.shape)}: ({B}, {N}, {len(axes)}) or ({N}, {len(axes)}) is needed")
    if not (1.0 <= base < math.inf):
        raise ValueError(f"base {base}: a finite value of at least 1 is needed")
    if B * N > _INT_MAX or q.shape[2] > 4096 or (k is not None and k.shape[2] > 4096):
        raise ValueError("at most 2^31 - 1 tokens and 4096 heads")
    return dev, ty


def _rotate(dev, ty, q, k, positions, axes, base, shared, interleaved, inverse):
    """New tensors; either of q and k may be None."""
    one = q if q is not None else k
    B, N, _, D = one.shape
    outs, d = [], _lib.RotaryDesc()
    for i, t in enumerate((q, k)):
        if t is None:
            outs.append(None)
            continue
        if t.stride(3) != 1 and D > 1:
            t = t.contiguous()
        o = torch.empty(t.shape, dtype=t.dtype, device=dev)
        outs.append(o)
        d.heads[i], d.src[i], d.dst[i] = t.shape[2], t.data_ptr(), o.data_ptr()
        d.src_sb[i], d.src_sn[i], d.src_sh[i] = t.stride(0), t.stride(1), t.stride(2)
    if any(o is not None and o.numel() for o in outs):
        turns, axis = _turn_table(axes, base, shared)
        d.dtype, d.B, d.N, d.D, d.npairs, d.naxes = ty, B, N, D, len(turns), len(axes)
        d.interleaved, d.inverse = int(interleaved), int(inverse)
        d.positions, d.pos64 = positions.data_ptr(), int(positions.dtype == torch.int64)
        d.pos_sb = positions.stride(0) if positions.dim() == 3 else 0
        d.pos_sn, d.pos_sa = positions.stride(-2), positions.stride(-1)
        d.turns, d.axis = ctypes.addressof(turns), ctypes.addressof(axis)
        _launch(dev, "dfcsa_rotary", ctypes.addressof(d))
    return outs


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, meta):
        ctx.save_for_backward(positions)
        ctx.meta = meta
        ctx.set_materialize_grads(False)
        return tuple(_rotate(*meta[:2], q, k, positions, *meta[2:], False))

    @staticmethod
    @_first_order
    def backward(ctx, gq, gk):
        meta = ctx.meta
        gq = gq if ctx.needs_input_grad[0] else None
        gk = gk if ctx.needs_input_grad[1] else None
        if gq is None and gk is None:
            return None, None, None, None
        dq, dk = _rotate(*meta[:2], gq, gk, ctx.saved_tensors[0], *meta[2:], True)
        return dq, dk, None, None


def rotary(q, k, positions, axes, base=10000.0, shared=False, interleaved=False):
    """(q, k) turned by their tokens' positions; q [B, N, H, D], k [B, N, Hk, D] or None (then None).

    positions: int32 or int64, [B, N, A] or [N, A]: where the token is on each of the A axes (row and
    column of a patch, or time, row and column).  axes: how many channel pairs each axis turns, e.g.
    (16, 16) for a width of 64; channels beyond 2 * sum(axes) stay as they are.  Pair i of an axis with
    n pairs turns by base^(-i/n) a position; with shared = True all axes share one ladder, pair j of the
    sum turning by base^(-j/sum).  Pairs are channels (j, sum + j), or (2j, 2j + 1) if interleaved.
    The angle is formed in 64 bits, so far positions keep their precision.  The gradient turns back.
    q and k are read in place from any strides with contiguous channels; the results are contiguous."""
    axes, base = tuple(axes), float(base)
    dev, ty = _rotary_check(q, k, positions, axes, base)
    meta = (dev, ty, tuple(int(a) for a in axes), base, bool(shared), bool(interleaved))
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return _Rotary.apply(q, k, positions, meta)
    return tuple(_rotate(*meta[:2], q, k, positions, *meta[2:], False))


# ------------------------------------------------------------------ attention
def _strided(t, group):
    """t with strides the kernels read in place, or a contiguous copy."""
    es = t.element_size()
    sb, st, sh, sd = t.stride()
    if (sd != 1 or t.data_ptr() % 16 or (sb * es) % 16 or (st * es) % 16 or (sh * es) % 16
            or st * es >= 1 << 23 or sh * es * group >= 1 << 29):
        t = _packed(t)
    return t


def _attn_check(q, k, v, window, sinks, scale, lengths):
    dev = _need_gpu(q, k, v, lengths)
    ty = _dtype(q, "q")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"q {q.dtype}, k {k.dtype}, v {v.dtype}: one type is needed")
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape:
        raise ValueError("q [batch, tokens, heads, width] and k, v of one shape [batch, keys, key heads, width] are "
                         f"needed, got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    B, T, H, D = q.shape
    if k.shape[0] != B or k.shape[3] != D:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} differ in batch or width")
    Hk = k.shape[2]
    if Hk < 1 or H < 1 or H % Hk or H > 65536:
        raise ValueError(f"{H} heads over {Hk} key heads: a multiple is needed")
    if D < 8 or D % 8 or D > 128:
        raise ValueError(f"width {D}: a multiple of 8 up to 128 is needed")
    if int(window) != window or window < 1:
        raise ValueError(f"window {window}: a whole number of at least 1")
    if int(sinks) != sinks or sinks < 0:
        raise ValueError(f"sinks {sinks}: a whole number of at least 0")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not (0.0 < scale < math.inf):
        raise ValueError(f"scale {scale}: a finite value above 0 is needed")
    if lengths is not None:
        if lengths.dtype != torch.int32:
            raise TypeError(f"lengths: int32 is needed, got {lengths.dtype}")
        if lengths.shape != (B,):
            raise ValueError(f"lengths {tuple(lengths.shape)}: ({B},) is needed")
    G = H // Hk
    if T * G > 1 << 29 or k.shape[1] * G > 1 << 29 or B * Hk > 1 << 24:
        raise ValueError("at most 2^29 tokens times heads per key head, and 2^24 sequences times key heads")
    return dev, ty, scale


def _desc(ty, q, k, v, window, sinks, causal, cached, scale, lengths, o, lse):
    B, T, H, _ = q.shape
    M, Hk, D = k.shape[1:]
    i64 = ctypes.c_int64 * 3
    return _lib.WattnDesc(ty, B, T, M, H, Hk, D, min(int(window), _INT_MAX), min(int(sinks), _INT_MAX), int(causal),
                          int(cached), scale, q.data_ptr(), k.data_ptr(), v.data_ptr(), i64(*q.stride()[:3]),
                          i64(*k.stride()[:3]), i64(*v.stride()[:3]),
                          None if lengths is None else lengths.data_ptr(), o.data_ptr(),
                          None if lse is None else lse.data_ptr())


def _workspace(d, backward, dev):
    n = ctypes.c_int64()
    if LIB.dfcsa_wattn_work_floats(ctypes.addressof(d), int(backward), ctypes.byref(n)) != 0:
        raise DfcsaError("dfcsa_wattn_work_floats failed: invalid argument/shape")
    if not n.value:
        return None
    work = torch.empty(n.value, dtype=torch.float32, device=dev)
    d.work, d.work_floats = work.data_ptr(), n.value
    return work


def _attend(dev, ty, q, k, v, window, sinks, causal, cached, scale, lengths, lse, rest=None):
    """o; q, k, v as _strided gives them, lengths contiguous."""
    o = torch.empty(q.shape, dtype=q.dtype, device=dev)
    d = _desc(ty, q, k, v, window, sinks, causal, cached, scale, lengths, o, lse)
    if rest is not None:
        d.o_rest = rest.data_ptr()
    work = _workspace(d, False, dev)
    _launch(dev, "dfcsa_wattn_fwd", ctypes.addressof(d))
    del work
    return o


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, meta):
        dev, ty, window, sinks, causal, scale = meta
        B, T, H, _ = q.shape
        lse = torch.empty(B * T * H, dtype=torch.float32, device=dev)
        # bf16: the backward's dO . O needs more of O than its 8 bits, so what the rounding left is kept too
        rest = torch.empty(q.shape, dtype=q.dtype, device=dev) if ty == _lib.DT_BF16 else None
        o = _attend(dev, ty, q, k, v, window, sinks, causal, False, scale, lengths, lse, rest)
        ctx.save_for_backward(q, k, v, o, lse, lengths, rest)
        ctx.meta = meta
        return o

    @staticmethod
    @_first_order
    def backward(ctx, do):
        q, k, v, o, lse, lengths, rest = ctx.saved_tensors
        dev, ty, window, sinks, causal, scale = ctx.meta
        do = _strided(do, q.shape[2] // k.shape[2])
        dq, delta = torch.empty(q.shape, dtype=q.dtype, device=dev), torch.empty_like(lse)
        dk, dv = torch.empty(k.shape, dtype=k.dtype, device=dev), torch.empty(v.shape, dtype=v.dtype, device=dev)
        d = _desc(ty, q, k, v, window, sinks, causal, False, scale, lengths, o, lse)
        d.dout, d.dout_stride[:] = do.data_ptr(), do.stride()[:3]
        d.o_rest = None if rest is None else rest.data_ptr()
        d.delta, d.dq, d.dk, d.dv = delta.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
        work = _workspace(d, True, dev)
        _launch(dev, "dfcsa_wattn_bwd", ctypes.addressof(d))
        del work
        return dq, dk, dv, None, None


class _Nothing(torch.autograd.Function):
    """The result for no tokens: zero gradients."""

    @staticmethod
    def forward(ctx, q, k, v):
        ctx.save_for_backward(q, k, v)
        return torch.zeros_like(q)

    @staticmethod
    @_first_order
    def backward(ctx, do):
        return tuple(torch.zeros_like(t) for t in ctx.saved_tensors)


def window_attention(q, k, v, window, sinks=0, causal=True, scale=None, lengths=None):
    """Attention of each token over the tokens near it and the first `sinks` ones: [B, N, H, D] for
    q [B, N, H, D] and k, v [B, N, Hk, D], H a multiple of Hk (query head h reads key head h // (H / Hk)).

    Token p sees token j when |p - j| < window or j < sinks, and, if causal, j <= p.  window = N (or
    more) is plain attention.  scale: of the scores, 1/sqrt(D) unless given.  lengths: int32 [B], the
    valid tokens of each sequence, the first ones (clamped to [0, N]); rows behind them are padding:
    whatever they hold, they are not seen, their results and gradients are zeros.
    bf16 or fp32, D a multiple of 8 up to 128.  Differentiable in q, k and v.  Tensors are read in place
    where their channels are contiguous and their strides multiples of 16 bytes, else from a copy.
    The cost follows N * (window + sinks); nothing N x N is stored."""
    dev, ty, scale = _attn_check(q, k, v, window, sinks, scale, lengths)
    if k.shape[1] != q.shape[1]:
        raise ValueError(f"{q.shape[1]} queries and {k.shape[1]} keys: as many are needed (or window_attention_cached)")
    if q.numel() == 0:
        return _Nothing.apply(q, k, v)
    G = q.shape[2] // k.shape[2]
    q, k, v = _strided(q, G), _strided(k, 1), _strided(v, 1)
    lengths = None if lengths is None else lengths.contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _WindowAttention.apply(q, k, v, lengths, (dev, ty, window, sinks, bool(causal), scale))
    return _attend(dev, ty, q, k, v, window, sinks, causal, False, scale, lengths, None)


def window_attention_cached(q, k_cache, v_cache, lengths, window, sinks=0, scale=None):
    """window_attention (causal) of the last T tokens of each sequence, q [B, T, H, D], over caches
    [B, capacity, Hk, D] that hold lengths[b] tokens (int32 [B], these T among them; clamped to
    [0, capacity]): token t is at position lengths[b] - T + t, and one before the start of its sequence
    gives zeros.  What the caches hold behind a sequence's end is not read.  For serving: it has no
    gradient, and refuses inputs that ask for one."""
    if torch.is_grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad):
        raise RuntimeError("window_attention_cached has no gradient: call it under torch.no_grad(), or window_attention")
    if lengths is None:
        raise TypeError("lengths: int32 [batch] is needed")
    dev, ty, scale = _attn_check(q, k_cache, v_cache, window, sinks, scale, lengths)
    if q.numel() == 0 or k_cache.shape[1] == 0:
        return torch.zeros(q.shape, dtype=q.dtype, device=dev)
    G = q.shape[2] // k_cache.shape[2]
    q, k, v = _strided(q, G), _strided(k_cache, 1), _strided(v_cache, 1)
    return _attend(dev, ty, q, k, v, window, sinks, True, True, scale, lengths.contiguous(), None)
