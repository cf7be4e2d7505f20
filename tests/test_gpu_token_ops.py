"""dfcsa.token_ops on the MI355X against plain 64-bit implementations.

Tolerances are bounds on the rounding errors of the computed formulas: UT, half a step of the stored type
(bf16 2^-8, fp32 2^-24); UP, the rounding of P and dS before the second products (bf16 inputs only); UF = 2^-24
for each fp32 operation, a sum of n terms counting n of them; times 1.1 for the products of two errors."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
UF = 2.0 ** -24
UT = {BF: 2.0 ** -8, F32: UF}
SLACK = 1.1
DEV = "cuda"


def tk():
    from dfcsa import token_ops
    return token_ops


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def rand(g, *shape, type=F32):
    return torch.randn(shape, generator=g, device=DEV).to(type)


def within(got, want, bound, what):
    got, want = got.detach().double(), want.detach()
    err = (got - want).abs()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = err - bound
    i = int(over.argmax()) if over.numel() else 0
    assert not over.numel() or float(over.max()) <= 0, (
        f"{what}: off by {float(err.flatten()[i]):.3g}, allowed {float(bound.expand_as(err).flatten()[i]):.3g} "
        f"(value {float(want.flatten()[i]):.3g}, {int((over > 0).sum())} of {over.numel()} over)")


# ------------------------------------------------------------------ RMS norm
TYPES = [(BF, BF), (BF, F32), (F32, F32)]


def norm_ref(x, res, w, eps):
    r = (x.float() + res.float()).to(res.dtype).double()
    rstd = (r.square().mean(-1, keepdim=True) + eps).rsqrt()
    return r, rstd, r * rstd * w.double()


@pytest.mark.parametrize("ty,st", TYPES)
@pytest.mark.parametrize("rows,C", [(1, 8), (3, 72), (5, 768), (4, 512), (7, 1032), (130, 2048), (9, 2056), (6, 4096),
                                    (5000, 40), (3, 8200), (2, 16384), (4097, 1024)])
def test_norm(rows, C, ty, st):
    g, eps = gen(rows + C), 1e-6
    x, res, w = rand(g, rows, C, type=ty), rand(g, rows, C, type=st) * 2, 1 + 0.3 * rand(g, C)
    dy, dr = rand(g, rows, C, type=ty), rand(g, rows, C, type=st)
    for t in (x, res, w):
        t.requires_grad_(True)
    y, r = tk().rms_norm_residual(x, res, w, eps)
    assert y.dtype == ty and r.dtype == st
    R, rstd, Y = norm_ref(x.detach(), res.detach(), w.detach(), eps)
    assert torch.equal(r.detach(), (x.float() + res.float()).to(st).detach())
    n = C + 20
    within(y, Y, SLACK * (UT[ty] + n * UF) * Y.abs(), "y")
    dx, dres, dw = torch.autograd.grad((y, r), (x, res, w), (dy, dr))
    W, DY = w.detach().double(), dy.double()
    xh, u = R * rstd, DY * W
    m = (u * xh).mean(-1, keepdim=True)
    D = rstd * (u - xh * m) + dr.double()
    mag = rstd * (u.abs() + xh.abs() * (u * xh).abs().mean(-1, keepdim=True)) * 2 * n * UF + 2 * UF * D.abs()
    within(dx, D, SLACK * (mag + UT[ty] * D.abs()), "dx")
    within(dres, D, SLACK * (mag + UT[st] * D.abs()), "dres")
    within(dw, (DY * xh).sum(0), SLACK * (rows + n) * UF * (DY * xh).abs().sum(0), "dw")


def test_norm_missing_gradients_and_shapes():
    g = gen(3)
    x, res, w = rand(g, 2, 3, 64, type=BF).requires_grad_(), rand(g, 2, 3, 64).requires_grad_(), (1 + rand(g, 64) * .1).requires_grad_()
    dy, dr = rand(g, 2, 3, 64, type=BF), rand(g, 2, 3, 64)
    y, r = tk().rms_norm_residual(x, res, w)
    assert y.shape == r.shape == (2, 3, 64)
    a = torch.autograd.grad(y, (x, res, w), dy, retain_graph=True)
    b = torch.autograd.grad(r, (x, res, w), dr, retain_graph=True, allow_unused=True)
    c = torch.autograd.grad((y, r), (x, res, w), (dy, dr), retain_graph=True)
    within(a[1] + b[1], c[1].double(), 4 * UF * (a[1].abs() + b[1].abs()).double(), "sum of both")
    assert torch.equal(b[1], dr) and torch.equal(a[2], c[2]) and float(b[2].abs().max()) == 0
    # one input at a time
    only = torch.autograd.grad((y, r), (w,), (dy, dr))
    assert torch.equal(only[0], c[2])
    y2, r2 = tk().rms_norm_residual(x.detach(), res, w.detach())
    assert torch.equal(torch.autograd.grad((y2, r2), res, (dy, dr))[0], c[1])
    # no rows
    e = torch.empty(0, 64, device=DEV, requires_grad=True)
    y, r = tk().rms_norm_residual(e, e, w)
    assert y.shape == (0, 64) and float(torch.autograd.grad(y.sum() + r.sum(), w)[0].abs().max()) == 0


def test_norm_strides_and_offsets():
    g = gen(4)
    big = rand(g, 6, 3, 72, type=BF)
    x, res = big[:, 1], big.transpose(0, 1)[2]          # rows apart, and the other way round
    flat = rand(g, 6 * 72 + 1, type=BF)[1:].view(6, 72)  # two bytes off a 16-byte border
    w = 1 + 0.1 * rand(g, 73)[1:]
    for a, b in ((x, res), (flat, x), (x, flat)):
        y, r = tk().rms_norm_residual(a, b, w)
        y2, r2 = tk().rms_norm_residual(a.clone(), b.clone(), w.clone())
        assert torch.equal(y, y2) and torch.equal(r, r2)


def test_norm_gradient_by_differences():
    g = gen(5)
    x, res, w = rand(g, 3, 16).requires_grad_(), rand(g, 3, 16).requires_grad_(), (1 + rand(g, 16) * .1).requires_grad_()
    dy, dr = rand(g, 3, 16), rand(g, 3, 16)

    def f(x, res, w):
        y, r = tk().rms_norm_residual(x, res, w)
        return (y.double() * dy).sum() + (r.double() * dr).sum()

    grads = torch.autograd.grad(f(x, res, w), (x, res, w))
    h = 2.0 ** -7
    for i, t in enumerate((x, res, w)):
        d = rand(g, *t.shape)
        up = [a.detach() + (h * d if j == i else 0) for j, a in enumerate((x, res, w))]
        dn = [a.detach() - (h * d if j == i else 0) for j, a in enumerate((x, res, w))]
        slope = float(f(*up) - f(*dn)) / (2 * h)
        # central differences: h^2 times a third derivative of order one, and fp32 values of order 50 over 2 h
        assert abs(slope - float((grads[i].double() * d).sum())) < 50 * h * h + 100 * UF / h


@pytest.mark.parametrize("ty,st", TYPES)
@pytest.mark.parametrize("rows,C,group", [(1, 8, 0), (4, 768, 0), (5, 96, 32), (33, 256, 64), (9, 2560, 128), (3, 384, 128),
                                          (7, 8200, 0), (3, 16384, 32), (1000, 128, 128)])
def test_norm_q8(rows, C, group, ty, st):
    g, eps = gen(rows * 7 + C), 1e-6
    x, res, w = rand(g, rows, C, type=ty), rand(g, rows, C, type=st), 1 + 0.3 * rand(g, C)
    if rows > 2:
        x[1], res[1] = 0, 0   # a row of zeros
    y8, s, r = tk().rms_norm_residual_q8(x, res, w, eps, group)
    assert y8.dtype == torch.float8_e4m3fn and s.shape == (rows, C // group if group else 1)
    R, _, Y = norm_ref(x, res, w, eps)
    assert torch.equal(r.double(), R)
    G = group or C
    amax = Y.view(rows, -1, G).abs().amax(-1)
    within(s, amax.clamp(min=1e-12) / 448, SLACK * (C + 24) * UF * amax.clamp(min=1e-12) / 448, "scales")
    S = s.double().repeat_interleave(G, -1)
    # half a step of e4m3: 2^-4 of the value, or of the smallest normal 2^-6, plus fp32's part
    half = torch.maximum(Y.abs() * 2.0 ** -4, S * 2.0 ** -10)
    within(y8.float().double() * S, Y, SLACK * half, "y8")
    assert float((y8.float().view(rows, -1, G).abs().amax(-1)[amax > 1e-9] - 448).abs().max()) == 0
    for ot in (BF, F32):
        out = tk().dequant_q8(y8, s, ot)
        assert torch.equal(out, (y8.float() * s.repeat_interleave(G, -1)).to(ot))


def test_norm_q8_rounds_to_nearest_even_and_keeps_nan():
    # weight picks the values: r = 1 in all columns, so y = weight up to rstd; scale 1 by a column of 448
    C = 64
    w = torch.ones(C, device=DEV)
    w[0] = 448.0
    w[1:9] = torch.tensor([1.0625, 1.1875, 17.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -7, -1.0625], device=DEV)
    x, res = torch.full((2, C), 0.5, device=DEV), torch.full((2, C), 0.5, device=DEV)
    x[1, 5] = float("nan")
    y8, s, r = tk().rms_norm_residual_q8(x, res, w, 0.0)
    assert float(s[0]) == 1.0
    assert y8[0, :9].float().tolist() == [448.0, 1.0, 1.25, 16.0, 20.0, 0.0, 2 * 2.0 ** -9, 2.0 ** -7, -1.0]
    assert torch.isnan(s[1]).all() and torch.isnan(y8[1].float()).all() and torch.isnan(r[1, 5])
    x[1, 5] = 0.5
    x[1] *= float("inf")
    _, s, _ = tk().rms_norm_residual_q8(x, res, w, 0.0)
    assert float(s[0]) == 1.0 and not torch.isfinite(s[1]).any()


# ------------------------------------------------------------------ rotary
def rotary_ref(x, pos, axes, base, shared, inter, sign):
    P, out, j = sum(axes), x.double().clone(), 0
    mag = torch.zeros_like(out)
    pos = pos if pos.dim() == 3 else pos[None]
    for a, n in enumerate(axes):
        for i in range(n):
            w = pos[..., a].double() * base ** -(j / P if shared else i / n)
            c, s = w.cos()[..., None], w.sin()[..., None] * sign
            ia, ib = (2 * j, 2 * j + 1) if inter else (j, P + j)
            u, v = x[..., ia].double(), x[..., ib].double()
            out[..., ia], out[..., ib] = u * c - v * s, u * s + v * c
            mag[..., ia] = mag[..., ib] = u.abs() + v.abs()
            j += 1
    return out, mag


@pytest.mark.parametrize("ty", [BF, F32])
@pytest.mark.parametrize("B,N,H,Hk,D,axes,shared,inter,far,wide", [
    (1, 1, 1, 1, 8, (4,), False, False, 0, False), (2, 9, 3, 1, 64, (16, 16), False, False, 0, False),
    (2, 17, 4, 2, 128, (16, 24, 24), True, False, 10 ** 6, False), (1, 300, 12, 12, 64, (16, 16), False, False, 0, True),
    (3, 5, 5, 5, 24, (3, 5), False, False, 100, True), (2, 6, 2, 1, 80, (9, 8, 3), True, True, 10 ** 5, False),
    (1, 33, 2, 2, 64, (4, 4, 4, 4), False, True, 10 ** 9, True), (1, 4, 1, 1, 10, (2, 1), False, False, 7, False),
    (5, 1, 16, 4, 128, (32, 32), False, True, 10 ** 6, False), (1, 70, 1, 1, 512, (256,), False, False, 50, False)])
def test_rotary(B, N, H, Hk, D, axes, shared, inter, far, wide, ty):
    g = gen(B * N + D)
    q, k = rand(g, B, N, H, D, type=ty).requires_grad_(), rand(g, B, N, Hk, D, type=ty).requires_grad_()
    pos = torch.randint(-far // 2, far + 50, (B, N, len(axes)), generator=g, device=DEV).to(torch.int64 if wide else torch.int32)
    gq, gk = rand(g, B, N, H, D, type=ty), rand(g, B, N, Hk, D, type=ty)
    oq, ok = tk().rotary(q, k, pos, axes, 10000.0, shared, inter)
    dq, dk = torch.autograd.grad((oq, ok), (q, k), (gq, gk))
    # cos and sin: the fraction of the turn to fp32 (2 pi 2^-26), 2 ulp of sincospi; then three operations
    for got, src, sign in ((oq, q, 1), (ok, k, 1), (dq, gq, -1), (dk, gk, -1)):
        want, mag = rotary_ref(src.detach(), pos, axes, 10000.0, shared, inter, sign)
        within(got, want, SLACK * (UT[ty] * want.abs() + 12 * UF * mag), "rotary")
        assert torch.equal(got[..., 2 * sum(axes):], src[..., 2 * sum(axes):])


def test_rotary_strides_shared_positions_and_missing_parts():
    g = gen(11)
    qkv = rand(g, 2, 7, 6 * 64, type=BF)
    q, k = qkv[..., :256].view(2, 7, 4, 64), qkv[..., 256:320].view(2, 7, 1, 64)
    pos = torch.randint(0, 99, (7, 2), generator=g, device=DEV).to(torch.int32)
    want = tk().rotary(q.clone(), k.clone(), pos[None].expand(2, 7, 2).contiguous(), (16, 16))
    head_major = q.transpose(1, 2).contiguous().transpose(1, 2)
    odd = rand(g, 2 * 7 * 4 * 64 + 1, type=BF)[1:].view(2, 7, 4, 64)
    odd.copy_(q)
    channels_apart = torch.stack((q, q), -1)[..., 0]
    for qq in (q, head_major, odd, channels_apart):
        got = tk().rotary(qq, k, pos, (16, 16))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # positions stepping through memory
    wide = torch.stack((pos, pos * 0 - 1), -1)[..., 0]
    assert not wide.is_contiguous() and torch.equal(tk().rotary(q, k, wide, (16, 16))[0], want[0])
    alone = tk().rotary(q, None, pos, (16, 16))
    assert torch.equal(alone[0], want[0]) and alone[1] is None
    qr, kr = q.clone().requires_grad_(), k.clone().requires_grad_()
    a, b = tk().rotary(qr, kr, pos, (16, 16))
    da = torch.autograd.grad(a.float().sum(), (qr, kr), retain_graph=True, allow_unused=True)
    assert da[1] is None
    (db,) = torch.autograd.grad(b.float().sum(), kr)
    assert db.shape == k.shape
    back, _ = tk().rotary(a.detach(), None, -pos, (16, 16))
    # two turns, each rounded: (|a| + |b|) of the pair twice
    pair = q.abs().view(2, 7, 4, 2, 32).sum(-2, keepdim=True).expand(2, 7, 4, 2, 32).reshape(q.shape)
    within(back, q.double(), 3 * UT[BF] * pair.double(), "there and back")
    e = torch.empty(2, 0, 4, 64, device=DEV)
    assert tk().rotary(e, None, torch.empty(0, 2, dtype=torch.int32, device=DEV), (16, 16))[0].shape == e.shape


# ------------------------------------------------------------------ attention
def visible(T, M, length, off, window, sinks, causal):
    p, j = torch.arange(T, device=DEV)[:, None] + off, torch.arange(M, device=DEV)[None]
    m = (p >= 0) & (p < length) & (j < length) & (((p - j).abs() < window) | (j < sinks))
    return m & (j <= p) if causal else m


def attn_ref(q, k, v, do, mask, scale, ty):
    """(o, dq, dk, dv) in 64 bits and the bounds of their errors; q [T, H, D], k, v [M, Hk, D], mask [T, M]."""
    T, H, D = q.shape
    M, Hk, _ = k.shape
    G = H // Hk
    up, ut = (2.0 ** -8, 2.0 ** -8) if ty == BF else (0.0, UF)
    Q, K, V = q.double().transpose(0, 1), k.double().repeat_interleave(G, 1).transpose(0, 1), v.double().repeat_interleave(G, 1).transpose(0, 1)
    s = scale * Q @ K.transpose(1, 2)
    sm = s.masked_fill(~mask, -math.inf)
    top = sm.amax(-1, keepdim=True).clamp(min=-1e300)
    e = (sm - top).exp()
    p = e / e.sum(-1, keepdim=True).clamp(min=1e-300)
    o = p @ V
    n = mask.sum(-1).double()[None, :, None]
    es = UF * ((D + 8) * scale * Q.abs() @ K.abs().transpose(1, 2) + 8 * s.abs()).masked_fill(~mask, 0)
    ep = 2 * es.amax(-1, keepdim=True) + (n + 32) * UF
    eo = p @ V.abs() * (up + ep + n * UF) + ut * o.abs()
    out = [o.transpose(0, 1)], [SLACK * eo.transpose(0, 1)]
    if do is not None:
        dO = do.double().transpose(0, 1)
        dp = dO @ V.transpose(1, 2)
        dl = (dO * o).sum(-1, keepdim=True)
        ds = p * (dp - dl)
        edp = D * UF * dO.abs() @ V.abs().transpose(1, 2)
        edl = (dO.abs() * eo).sum(-1, keepdim=True) + D * UF * (dO * o).abs().sum(-1, keepdim=True)
        eds = p * ((dp - dl).abs() * (ep + 8 * UF) + edp + edl) + up * ds.abs()

        def groups(x):
            return x.view(Hk, G, M, D).sum(1).transpose(0, 1)

        dq, edq = scale * ds @ K, scale * (eds + (n + 8) * UF * ds.abs()) @ K.abs()
        rows = T * G
        dk = groups(scale * ds.transpose(1, 2) @ Q)
        edk = groups(scale * (eds + (rows + 8) * UF * ds.abs()).transpose(1, 2) @ Q.abs())
        dv = groups(p.transpose(1, 2) @ dO)
        edv = groups((p * (up + ep + (rows + 8) * UF)).transpose(1, 2) @ dO.abs())
        for want, bound in ((dq.transpose(0, 1), edq.transpose(0, 1)), (dk, edk), (dv, edv)):
            out[0].append(want)
            out[1].append(SLACK * (bound + ut * want.abs()))
    return out


def check_train(q, k, v, do, window, sinks, causal, lengths=None, scale=None):
    B, N, H, D = q.shape
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    o = tk().window_attention(*leaves, window, sinks, causal=causal, lengths=n, scale=scale)
    got = (o, *torch.autograd.grad(o, leaves, do))
    plain = tk().window_attention(*(t.detach() for t in leaves), window, sinks, causal=causal, lengths=n, scale=scale)
    assert torch.equal(plain, o)
    for b in range(B):
        L = N if lengths is None else min(max(lengths[b], 0), N)
        mask = visible(N, N, L, 0, window, sinks, causal)
        clean = [torch.where((torch.arange(N, device=DEV) < L)[:, None, None], t[b].detach(), torch.zeros_like(t[b])) for t in (*leaves, do)]
        want, bound = attn_ref(*clean, mask, scale or 1 / math.sqrt(D), q.dtype)
        for name, x, w, e in zip(("o", "dq", "dk", "dv"), got, want, bound):
            within(x[b], w, e, f"{name}[{b}]")
    return got


CASES = [  # B, N, H, Hk, D, window, sinks, causal
    (1, 1, 1, 1, 8, 1, 0, True), (1, 2, 2, 1, 16, 1, 1, True), (2, 31, 3, 3, 64, 5, 0, True),
    (1, 33, 4, 2, 64, 33, 2, False), (2, 64, 2, 2, 128, 64, 0, True), (1, 65, 8, 1, 128, 9, 4, True),
    (1, 127, 2, 1, 40, 40, 0, False), (1, 128, 3, 1, 80, 7, 70, True), (2, 129, 6, 2, 96, 129, 0, True),
    (1, 200, 4, 4, 64, 57, 4, False), (1, 300, 5, 5, 32, 1, 300, True), (1, 257, 2, 2, 24, 64, 130, False),
    (1, 700, 8, 2, 128, 100, 3, True), (1, 650, 3, 1, 112, 33, 200, False), (1, 1100, 2, 1, 64, 2000, 0, True),
    (3, 385, 1, 1, 128, 128, 1, True),
    # rows beyond the window of the sinks' keys: a pass of their own, with several blocks of sinks, two-sided
    (1, 2500, 4, 2, 64, 100, 40, True), (1, 1700, 2, 2, 128, 60, 200, False), (2, 1300, 1, 1, 96, 1300, 0, True)]


@pytest.mark.parametrize("ty", [BF, F32])
@pytest.mark.parametrize("B,N,H,Hk,D,window,sinks,causal", CASES)
def test_attention(B, N, H, Hk, D, window, sinks, causal, ty):
    g = gen(N + D)
    q, k, v, do = rand(g, B, N, H, D, type=ty), rand(g, B, N, Hk, D, type=ty), rand(g, B, N, Hk, D, type=ty), rand(g, B, N, H, D, type=ty)
    check_train(q, k, v, do, window, sinks, causal)


@pytest.mark.parametrize("seed", range(24))
def test_attention_drawn(seed):
    """Sizes, windows, sinks, lengths and types at random."""
    r = random.Random(seed)
    ty = r.choice([BF, F32])
    Hk, G, D, B = r.choice([1, 2, 3]), r.choice([1, 1, 2, 3, 5, 8]), 8 * r.randint(1, 16), r.choice([1, 2, 3])
    N = r.choice([r.randint(1, 70), r.randint(60, 500), r.randint(400, 900)])
    window, sinks = r.choice([1, r.randint(1, 40), r.randint(1, N), 2 * N]), r.choice([0, 1, 5, r.randint(0, N), 70])
    lengths = [r.randint(0, N + 3) for _ in range(B)] if r.random() < 0.5 else None
    g = gen(seed)
    q, k, v, do = (rand(g, B, N, h, D, type=ty) for h in (Hk * G, Hk, Hk, Hk * G))
    check_train(q, k, v, do, window, sinks, r.random() < 0.6, lengths, scale=r.choice([None, 0.3, 0.05]))


@pytest.mark.parametrize("ty", [BF, F32])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_padded_batch(ty, causal):
    """Lengths of zero, one, inside a tile, at its border, whole and beyond; NaN and infinity in the padding."""
    B, N, H, Hk, D = 7, 150, 4, 2, 64
    lengths = [0, 1, 63, 64, 129, 150, 400]
    g = gen(9)
    q, k, v, do = rand(g, B, N, H, D, type=ty), rand(g, B, N, Hk, D, type=ty), rand(g, B, N, Hk, D, type=ty), rand(g, B, N, H, D, type=ty)
    for b, n in enumerate(lengths):
        for t, bad in ((q, math.nan), (k, math.inf), (v, math.nan), (do, -math.inf)):
            t[b, n:] = bad
    got = check_train(q, k, v, do, 20, 3, causal, lengths)
    for b, n in enumerate(lengths):
        for x in got:
            assert float(x[b, n:].abs().sum()) == 0.0   # padding: zeros


@pytest.mark.parametrize("ty", [BF, F32])
def test_attention_strides(ty):
    g = gen(21)
    B, N, H, Hk, D = 2, 90, 4, 2, 64
    qkv = rand(g, B, N, (H + 2 * Hk) * D, type=ty)
    q, k, v = (x.view(B, N, -1, D) for x in qkv.split((H * D, Hk * D, Hk * D), -1))
    do = rand(g, B, N, H, D, type=ty)
    want = check_train(q, k, v, do, 17, 2, True)

    def again(q, k, v, do):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = tk().window_attention(*leaves, 17, 2)
        for a, b in zip((o, *torch.autograd.grad(o, leaves, do)), want):
            assert torch.equal(a, b)

    hm = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v, do)]
    again(*hm)
    again(*(t.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2) for t in (q, k, v, do)))   # channels apart
    odd = rand(g, do.numel() + 1, type=ty)[1:].view(do.shape)
    odd.copy_(do)
    again(q, k, v, odd)
    # a gradient that is one number for all
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    one = torch.autograd.grad(tk().window_attention(*leaves, 17, 2).sum(), leaves)
    leaves2 = [t.detach().requires_grad_() for t in (q, k, v)]
    two = torch.autograd.grad(tk().window_attention(*leaves2, 17, 2), leaves2, torch.ones_like(do))
    assert all(torch.equal(a, b) for a, b in zip(one, two))
    # one key head broadcast to all: its gradient is the sum over the copies
    kb = k[:, :, :1].detach().requires_grad_()
    o = tk().window_attention(q, kb.expand(B, N, Hk, D), v, 17, 2)
    (dkb,) = torch.autograd.grad(o, kb, do)
    full = k[:, :, :1].expand(B, N, Hk, D).contiguous().requires_grad_()
    (dfull,) = torch.autograd.grad(tk().window_attention(q, full, v, 17, 2), full, do)
    within(dkb, dfull.double().sum(2, keepdim=True), 2 * UT[ty] * dfull.double().abs().sum(2, keepdim=True), "broadcast")


def test_attention_gradient_by_differences():
    g = gen(31)
    q, k, v, do = rand(g, 1, 40, 2, 16), rand(g, 1, 40, 1, 16), rand(g, 1, 40, 1, 16), rand(g, 1, 40, 2, 16)
    leaves = [t.requires_grad_() for t in (q, k, v)]

    def f(*a):
        return (tk().window_attention(*a, 9, 2).double() * do).sum()

    grads = torch.autograd.grad(f(*leaves), leaves)
    h = 2.0 ** -7
    for i in range(3):
        d = rand(g, *leaves[i].shape)
        up = [t.detach() + (h * d if j == i else 0) for j, t in enumerate(leaves)]
        dn = [t.detach() - (h * d if j == i else 0) for j, t in enumerate(leaves)]
        slope = float(f(*up) - f(*dn)) / (2 * h)
        # h^2 times a third derivative of order 1000 (1280 outputs of order one), fp32 values over 2 h
        assert abs(slope - float((grads[i].double() * d).sum())) < 1000 * h * h


def test_attention_large_scores():
    """Scores of +-1000 (the running maximum moves by far more than its slack, and rows differ), one key taking all."""
    g = gen(41)
    for ty in (BF, F32):
        q, k, v, do = (rand(g, 1, 260, 2, 64, type=ty) for _ in range(4))
        k = (k * torch.linspace(0.1, 30, 260, device=DEV)[:, None, None]).to(ty)
        o = tk().window_attention(q, k, v, 260)
        want, bound = attn_ref(q[0], k[0], v[0], None, visible(260, 260, 260, 0, 260, 0, True), 0.125, ty)
        within(o[0], want[0], bound[0], "o")


CACHED = [  # B, T, cap, H, Hk, D, window, sinks, lengths
    (1, 1, 1, 1, 1, 8, 1, 0, [1]), (3, 1, 40, 4, 2, 64, 7, 2, [0, 1, 40]), (2, 1, 700, 8, 1, 128, 100, 4, [700, 333]),
    (2, 1, 4100, 2, 2, 64, 5000, 0, [4100, 77]), (1, 1, 3000, 32, 1, 128, 1000, 70, [2999]),
    (3, 3, 200, 6, 3, 40, 50, 1, [2, 3, 150]), (2, 5, 300, 40, 8, 80, 300, 0, [299, 4]),
    (1, 40, 500, 4, 2, 96, 64, 5, [450]), (2, 100, 900, 2, 1, 128, 200, 16, [900, 60]), (1, 70, 5000, 8, 8, 32, 6000, 0, [5000]),
    (4, 1, 64, 3, 3, 16, 64, 0, [64, 65, 1000, -3])]


@pytest.mark.parametrize("ty", [BF, F32])
@pytest.mark.parametrize("B,T,cap,H,Hk,D,window,sinks,lengths", CACHED)
def test_attention_cached(B, T, cap, H, Hk, D, window, sinks, lengths, ty):
    g = gen(cap + D)
    q, k, v = rand(g, B, T, H, D, type=ty), rand(g, B, cap, Hk, D, type=ty), rand(g, B, cap, Hk, D, type=ty)
    for b, n in enumerate(lengths):   # behind the end, and before the window of the first new token: not read
        n = min(max(n, 0), cap)
        k[b, n:], v[b, n:] = math.nan, math.inf
        lo = n - T - window + 1
        if lo > sinks:
            k[b, sinks:lo], v[b, sinks:lo] = math.inf, math.nan
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    o = tk().window_attention_cached(q, k, v, n, window, sinks)
    for b in range(B):
        L = min(max(lengths[b], 0), cap)
        mask = visible(T, cap, L, L - T, window, sinks, True)
        seen = mask.any(0)[:, None, None]
        want, bound = attn_ref(q[b], torch.where(seen, k[b], 0), torch.where(seen, v[b], 0), None, mask, 1 / math.sqrt(D), ty)
        within(o[b], want[0], bound[0], f"o[{b}]")


@pytest.mark.parametrize("ty", [BF, F32])
@pytest.mark.parametrize("T,cap,window,n", [(1, 300, 40, 290), (5, 300, 40, 250), (40, 500, 64, 500), (90, 200, 30, 180)])
def test_attention_cached_hidden_infinities(T, cap, window, n, ty):
    """A key that some of the new tokens see and others do not: its NaN or infinity reaches those that see it only."""
    g = gen(T + cap)
    H, Hk, D = 4, 2, 64
    q, k, v = rand(g, 1, T, H, D, type=ty), rand(g, 1, cap, Hk, D, type=ty), rand(g, 1, cap, Hk, D, type=ty)
    lengths = torch.tensor([n], dtype=torch.int32, device=DEV)
    want = tk().window_attention_cached(q, k, v, lengths, window, 2)
    j = n - T // 2 - 1
    for bad in (math.nan, math.inf):
        v2 = v.clone()
        v2[0, j] = bad
        o = tk().window_attention_cached(q, k, v2, lengths, window, 2)
        p = torch.arange(T, device=DEV) + n - T
        sees = (p >= j) & (p - j < window)
        assert not torch.isfinite(o[0, sees]).any()
        # the rows formed again differ by the rounding of P and of the sums
        within(o[0, ~sees], want[0, ~sees].double(), (4 * UT[ty] + 2000 * UF) * v.double().abs().amax().expand_as(want[0, ~sees]), "others")


@pytest.mark.parametrize("ty", [BF, F32])
@pytest.mark.parametrize("N,H,Hk,D,window,sinks,causal", [(150, 4, 2, 64, 20, 3, True), (700, 2, 1, 128, 50, 4, True),
                                                          (700, 3, 3, 40, 30, 40, False), (2500, 2, 2, 64, 100, 2, True)])
def test_attention_hidden_infinities(N, H, Hk, D, window, sinks, causal, ty):
    """NaN or infinity in a q, k, v or dO row: the results of the pairs that do not involve it stay."""
    g = gen(N + D)
    t = [rand(g, 1, N, h, D, type=ty) for h in (H, Hk, Hk, H)]
    lens = torch.tensor([N - 3], dtype=torch.int32, device=DEV)

    def run(q, k, v, do):
        leaves = [x.detach().clone().requires_grad_() for x in (q, k, v)]
        o = tk().window_attention(*leaves, window, sinks, causal=causal, lengths=lens)
        return [o.detach()[0], *(x[0] for x in torch.autograd.grad(o, leaves, do))]

    clean = run(*t)
    mask = visible(N, N, N - 3, 0, window, sinks, causal)
    at = N // 2
    for which, bad in ((0, math.nan), (1, math.inf), (2, math.nan), (3, math.inf), (2, -math.inf)):
        x = [y.clone() for y in t]
        x[which][0, at] = bad
        got = run(*x)
        # what depends on the row: as a query (q, dO) or as a key (k, v), directly and through the rows that see it
        if which in (0, 3):
            rows = torch.zeros(N, dtype=torch.bool, device=DEV)
            rows[at] = True
        else:
            rows = mask[:, at]
        keys = mask[rows].any(0)
        touched = (rows if which != 3 else torch.zeros_like(rows), rows, keys | False, keys | False)
        for name, a, b, hit in zip(("o", "dq", "dk", "dv"), got, clean, touched):
            free = ~hit
            assert torch.isfinite(a[free]).all(), (which, name)
            # formed again in another order, P and dS unrounded: rounding of both sides
            scale = b.double().abs().amax()
            within(a[free], b[free].double(), (6 * UT[ty] + 4 * N * UF) * scale.expand_as(b[free]), f"{which} {name}")
        assert not torch.isfinite(got[0][rows]).all() or which == 3
        assert not torch.isfinite(got[1][rows]).all()


def test_attention_cached_is_the_last_rows_of_the_whole():
    g = gen(51)
    q, k, v = rand(g, 2, 300, 8, 64, type=BF), rand(g, 2, 300, 2, 64, type=BF), rand(g, 2, 300, 2, 64, type=BF)
    whole = tk().window_attention(q, k, v, 90, 4)
    n = torch.tensor([300, 300], dtype=torch.int32, device=DEV)
    for T in (1, 7, 130):
        part = tk().window_attention_cached(q[:, 300 - T:], k, v, n, 90, 4)
        # two roundings of P and two of the result
        within(part, whole[:, 300 - T:].double(), 4 * UT[BF] * v.double().abs().amax() * torch.ones((), device=DEV, dtype=torch.float64), "part")


def test_attention_long_cache_offsets():
    """Keys further than 2^31 bytes and elements from the cache's start."""
    cap, Hk, D = 2_200_000, 8, 128   # 4.5 GB each, 2.25e9 elements
    g = gen(61)
    k, v = torch.zeros(1, cap, Hk, D, dtype=BF, device=DEV), torch.zeros(1, cap, Hk, D, dtype=BF, device=DEV)
    for t in (k, v):
        t[0, -500:] = rand(g, 500, Hk, D, type=BF)
        t[0, :8] = rand(g, 8, Hk, D, type=BF)
    q = rand(g, 1, 1, 16, D, type=BF)
    n = torch.tensor([cap], dtype=torch.int32, device=DEV)
    o = tk().window_attention_cached(q, k, v, n, 400, 8)
    keep = torch.cat((torch.arange(8, device=DEV), torch.arange(cap - 400, cap, device=DEV)))
    want, bound = attn_ref(q[0], k[0, keep], v[0, keep], None, torch.ones(1, 408, dtype=torch.bool, device=DEV), 1 / math.sqrt(D), BF)
    within(o[0], want[0], bound[0], "o")


# ------------------------------------------------------------------ a block, streams, graphs
def block(x, stream, w1, wq, wo, w2, pos, H, Hk, D, window, sinks, lengths):
    """norm -> projection -> rotary -> windowed attention -> projection -> norm with the residual."""
    t = tk()
    B, N, C = x.shape
    y, r = t.rms_norm_residual(x, stream, w1)
    q, k, v = (y @ wq).split((H * D, Hk * D, Hk * D), -1)
    q, k = t.rotary(q.view(B, N, H, D), k.view(B, N, Hk, D), pos, (D // 4, D // 4))
    o = t.window_attention(q, k, v.view(B, N, Hk, D), window, sinks, causal=False, lengths=lengths)
    return t.rms_norm_residual(o.reshape(B, N, H * D) @ wo, r, w2)


def block_ref(x, stream, w1, wq, wo, w2, pos, H, Hk, D, window, sinks, lengths):
    B, N, C = x.shape

    def norm(a, b, w):
        r = a + b
        return r * (r.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w, r

    y, r = norm(x, stream, w1)
    q, k, v = (y @ wq).split((H * D, Hk * D, Hk * D), -1)

    def turn(t):
        P = D // 2
        w = torch.cat([pos[..., a, None].double() * 10000.0 ** -(torch.arange(D // 4, device=DEV).double() / (D // 4)) for a in range(2)], -1)
        c, s = w.cos()[:, None], w.sin()[:, None]
        a, b = t[..., :P], t[..., P:]
        return torch.cat((a * c - b * s, a * s + b * c), -1)

    q, k, v = turn(q.view(B, N, H, D)), turn(k.view(B, N, Hk, D)), v.view(B, N, Hk, D)
    k, v = k.repeat_interleave(H // Hk, 2), v.repeat_interleave(H // Hk, 2)
    out = []
    for b in range(B):
        mask = visible(N, N, int(lengths[b]), 0, window, sinks, False)
        s = (torch.einsum("nhd,mhd->hnm", q[b], k[b]) / math.sqrt(D)).masked_fill(~mask, -math.inf)
        p = torch.where(mask.any(-1)[:, None], torch.softmax(s.masked_fill(~mask.any(-1)[:, None], 0), -1), torch.zeros_like(s))
        out.append(torch.einsum("hnm,mhd->nhd", p, v[b]))
    return norm(torch.stack(out).reshape(B, N, H * D) @ wo, r, w2)


def block_inputs(ty):
    g = gen(71)
    B, N, C, H, Hk, D = 2, 90, 128, 4, 2, 32
    x, stream = rand(g, B, N, C, type=ty), rand(g, B, N, C)
    w1, w2 = 1 + 0.1 * rand(g, C), 1 + 0.1 * rand(g, C)
    wq, wo = rand(g, C, (H + 2 * Hk) * D, type=ty) / math.sqrt(C), rand(g, H * D, C, type=ty) / math.sqrt(C)
    n = torch.arange(N, device=DEV)
    pos = torch.stack((n // 10, n % 10), -1).to(torch.int32)
    lengths = torch.tensor([90, 71], dtype=torch.int32, device=DEV)
    leaves = [t.detach().requires_grad_() for t in (x, stream, w1, wq, wo, w2)]
    return leaves, (pos, H, Hk, D, 25, 3, lengths), (rand(g, B, N, C, type=ty), rand(g, B, N, C))


@pytest.mark.parametrize("ty,tol", [(F32, 2e-5), (BF, 0.04)])
def test_block(ty, tol):
    """The operators together, values and all gradients.  Relative 2-norms: fp32, about 100 roundings in a row of a
    few hundred terms each grow like their root; bf16, ten stored tensors at 2^-8 each, and as many in the gradients."""
    leaves, rest, douts = block_inputs(ty)
    got = block(*leaves, *rest)
    grads = torch.autograd.grad(got, leaves, douts)
    ref = [t.detach().double().requires_grad_() for t in leaves]
    want = block_ref(*ref, *rest)
    wgrads = torch.autograd.grad(want, ref, [d.double() for d in douts])
    for a, b in zip((*got, *grads), (*want, *wgrads)):
        assert float((a.double() - b).norm() / b.norm()) < tol


def test_everything_twice_is_bitwise_the_same():
    for ty in (BF, F32):
        leaves, rest, douts = block_inputs(ty)
        runs = []
        for _ in range(2):
            got = block(*leaves, *rest)
            runs.append((*got, *torch.autograd.grad(got, leaves, douts)))
        assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_side_stream():
    leaves, rest, douts = block_inputs(BF)
    got = block(*leaves, *rest)
    want = (*got, *torch.autograd.grad(got, leaves, douts))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = block(*leaves, *rest)
        got = (*got, *torch.autograd.grad(got, leaves, douts))
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_streams_at_once():
    """The same calls on two streams side by side: no memory is shared between calls."""
    run, _ = token_calls()
    want = run()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for _ in range(3):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(run())
    torch.cuda.synchronize()
    for out in got:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def token_calls():
    """Every entry point's call of this package alone (no library product), on inputs that can be overwritten."""
    t, g = tk(), gen(81)
    x, st, w = rand(g, 50, 256, type=BF).requires_grad_(), rand(g, 50, 256).requires_grad_(), (1 + rand(g, 256) * .1).requires_grad_()
    q, k, v = (rand(g, 1, 900, h, 64, type=BF).requires_grad_() for h in (4, 2, 2))
    pos = torch.arange(1800, device=DEV).view(900, 2).to(torch.int32)
    cq, ck, cv = rand(g, 2, 1, 8, 64, type=BF), rand(g, 2, 2000, 2, 64, type=BF), rand(g, 2, 2000, 2, 64, type=BF)
    n = torch.tensor([2000, 700], dtype=torch.int32, device=DEV)
    dy, dr, do = rand(g, 50, 256, type=BF), rand(g, 50, 256), rand(g, 1, 900, 4, 64, type=BF)

    def run():
        y, r = t.rms_norm_residual(x, st, w)
        out = [y, r, *torch.autograd.grad((y, r), (x, st, w), (dy, dr))]
        a, b = t.rotary(q, k, pos, (16, 16))
        o = t.window_attention(a, b, v, 60, 3)
        out += [o, *torch.autograd.grad(o, (q, k, v), do)]
        with torch.no_grad():
            y8, s, r = t.rms_norm_residual_q8(x, st, w, group=64)
            out += [t.dequant_q8(y8, s), s, t.window_attention_cached(cq, ck, cv, n, 1500, 4)]
        return [z.detach() for z in out]

    return run, (x, st, q, k, v, cq, ck, cv, dy, do)


def test_graph_capture_and_replay():
    """Captured once (forward and backward), replayed with new inputs between eager calls: each replay is the eager result;
    two graphs of the same calls do not share their workspaces."""
    run, inputs = token_calls()
    run()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            run()
        torch.cuda.current_stream().wait_stream(s)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = run()
        graphs.append((gr, out))
    g = gen(91)
    for turn in range(4):
        with torch.no_grad():
            for t in inputs:
                t.copy_(rand(g, *t.shape))
        want = run()
        for gr, _ in graphs:
            gr.replay()
        again = run()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want)), turn
        assert all(torch.equal(a, b) for a, b in zip(again, want))


def test_saved_tensors_are_guarded_and_second_order_refused():
    g = gen(95)
    q, k, v = (rand(g, 1, 20, 2, 16).requires_grad_() for _ in range(3))
    o = tk().window_attention(q, k, v, 5)
    with torch.no_grad():
        k.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()
    q2 = q.detach().requires_grad_()
    w = torch.ones(16, device=DEV, requires_grad=True)
    for out in (tk().window_attention(q2, k, v, 5), tk().rms_norm_residual(q2, q, w)[0], tk().rotary(q2, None, torch.zeros(
            20, 1, dtype=torch.int32, device=DEV), (4,))[0]):
        with pytest.raises(RuntimeError, match="first order"):
            torch.autograd.grad(out.sum(), q2, create_graph=True)


# ------------------------------------------------------------------ refusals
def test_refusals():
    t, g = tk(), gen(99)
    x, w = rand(g, 4, 64), torch.ones(64, device=DEV)
    b = x.to(BF)
    for bad, e in ((lambda: t.rms_norm_residual(x, x[:2], w), ValueError), (lambda: t.rms_norm_residual(x[:, :12], x[:, :12], w[:12]), ValueError),
                   (lambda: t.rms_norm_residual(x, b, w), TypeError), (lambda: t.rms_norm_residual(x.half(), x, w), TypeError),
                   (lambda: t.rms_norm_residual(x, x, w.to(BF)), TypeError), (lambda: t.rms_norm_residual(x, x, w[:8]), ValueError),
                   (lambda: t.rms_norm_residual(x, x, w, eps=-1), ValueError), (lambda: t.rms_norm_residual(x, x, w, eps=math.nan), ValueError),
                   (lambda: t.rms_norm_residual(x, x.cpu(), w), RuntimeError),
                   (lambda: t.rms_norm_residual_q8(x, x, w, group=16), ValueError), (lambda: t.rms_norm_residual_q8(x, x, w, group=128), ValueError),
                   (lambda: t.dequant_q8(x, torch.ones(4, 1, device=DEV)), TypeError),
                   (lambda: t.dequant_q8(x.to(t.E4M3), torch.ones(4, 3, device=DEV)), ValueError),
                   (lambda: t.dequant_q8(x.to(t.E4M3), torch.ones(3, 1, device=DEV)), ValueError),
                   (lambda: t.dequant_q8(x.to(t.E4M3), torch.ones(4, 1, device=DEV), torch.float16), TypeError)):
        with pytest.raises(e):
            bad()
    q, pos = rand(g, 2, 5, 4, 16), torch.zeros(5, 2, dtype=torch.int32, device=DEV)
    for bad, e in ((lambda: t.rotary(q[0], None, pos, (4, 4)), ValueError), (lambda: t.rotary(q, q[:, :4], pos, (4, 4)), ValueError),
                   (lambda: t.rotary(q, q.to(BF), pos, (4, 4)), TypeError), (lambda: t.rotary(q.half(), None, pos, (4, 4)), TypeError),
                   (lambda: t.rotary(q, q, pos, (4, 5)), ValueError), (lambda: t.rotary(q, q, pos, (4, 0)), ValueError),
                   (lambda: t.rotary(q, q, pos, ()), ValueError), (lambda: t.rotary(q, q, pos, (1,) * 5), ValueError),
                   (lambda: t.rotary(q, q, pos, (8,)), ValueError), (lambda: t.rotary(q, q, pos.float(), (4, 4)), TypeError),
                   (lambda: t.rotary(q, q, pos[:4], (4, 4)), ValueError), (lambda: t.rotary(q, q, pos, (4, 4), base=0.5), ValueError),
                   (lambda: t.rotary(q, q, pos.cpu(), (4, 4)), RuntimeError)):
        with pytest.raises(e):
            bad()
    n = torch.tensor([5, 5], dtype=torch.int32, device=DEV)
    for bad, e in ((lambda: t.window_attention(q, q, q, 0), ValueError), (lambda: t.window_attention(q, q, q, 2.5), ValueError),
                   (lambda: t.window_attention(q, q, q, 2, -1), ValueError), (lambda: t.window_attention(q, q[:, :, :3], q[:, :, :3], 2), ValueError),
                   (lambda: t.window_attention(q, q, q[:, :4], 2), ValueError), (lambda: t.window_attention(q, q[:, :4], q[:, :4], 2), ValueError),
                   (lambda: t.window_attention(q[..., :12], q[..., :12], q[..., :12], 2), ValueError),
                   (lambda: t.window_attention(rand(g, 1, 2, 1, 136), rand(g, 1, 2, 1, 136), rand(g, 1, 2, 1, 136), 2), ValueError),
                   (lambda: t.window_attention(q, q.to(BF), q, 2), TypeError), (lambda: t.window_attention(q.half(), q.half(), q.half(), 2), TypeError),
                   (lambda: t.window_attention(q, q, q, 2, scale=0.0), ValueError), (lambda: t.window_attention(q, q, q, 2, scale=math.inf), ValueError),
                   (lambda: t.window_attention(q, q, q, 2, lengths=n.long()), TypeError), (lambda: t.window_attention(q, q, q, 2, lengths=n[:1]), ValueError),
                   (lambda: t.window_attention(q, q, q, 2, lengths=n.cpu()), RuntimeError), (lambda: t.window_attention(q[0], q[0], q[0], 2), ValueError),
                   (lambda: t.window_attention_cached(q, q, q, None, 2), TypeError), (lambda: t.window_attention_cached(q, q, q, n.float(), 2), TypeError)):
        with pytest.raises(e):
            bad()
    e = torch.empty(1, 0, 2, 16, device=DEV, requires_grad=True)
    assert torch.autograd.grad(t.window_attention(e, e, e, 3).sum(), e)[0].shape == e.shape
    assert t.window_attention_cached(q, q[:, :0], q[:, :0], n, 3).abs().sum() == 0


@pytest.mark.parametrize("ty", [BF, F32])
def test_attention_dimensions_of_one_have_any_stride(ty):
    """One token of one head cut from rows of 9 elements: its strides are 9 although it is contiguous."""
    g = gen(81)
    k, v = rand(g, 1, 40, 1, 8, type=ty), rand(g, 1, 40, 1, 8, type=ty)
    n = torch.tensor([33], dtype=torch.int32, device=DEV)
    wide = rand(g, 1, 1, 1, 9, type=ty)
    for q in (wide[..., :8], wide[..., 1:]):   # the second is misaligned as well
        assert torch.equal(tk().window_attention_cached(q, k, v, n, 20, 2),
                           tk().window_attention_cached(q.reshape(8).clone().view(1, 1, 1, 8), k, v, n, 20, 2))
        leaves = [t.detach().requires_grad_() for t in (q, q + 1, q - 1)]
        do = rand(g, 1, 1, 1, 9, type=ty)[..., 1:]
        check_train(*leaves, do, 1, 0, True)


def test_attention_head_major_cache():
    cap, Hk, D = 1 << 18, 2, 128   # 8 query heads of a key head times 2^26 bytes reach 2^29
    g = gen(82)
    k, v = (torch.zeros(1, Hk, cap, D, dtype=BF, device=DEV).transpose(1, 2) for _ in range(2))
    for t in (k, v):
        t[0, -500:] = rand(g, 500, Hk, D, type=BF)
        t[0, :4] = rand(g, 4, Hk, D, type=BF)
    q = rand(g, 1, 1, 16, D, type=BF)
    n = torch.tensor([cap], dtype=torch.int32, device=DEV)
    assert torch.equal(tk().window_attention_cached(q, k, v, n, 300, 4),
                       tk().window_attention_cached(q, k.contiguous(), v.contiguous(), n, 300, 4))


def test_many_workgroups():
    """More than 2^22 workgroups of rotary and dequant_q8: a grid of two dimensions, against two halves."""
    t, g = tk(), gen(83)
    N, D = (1 << 22) + 5, 272   # one token a workgroup
    q = rand(g, 1, N, 1, D, type=BF)
    pos = torch.arange(N, dtype=torch.int32, device=DEV)[:, None]
    whole, _ = t.rotary(q, None, pos, (136,))
    for part in (slice(0, N // 2), slice(N // 2, N)):
        assert torch.equal(whole[:, part], t.rotary(q[:, part], None, pos[part], (136,))[0])
    del q, whole
    rows, C = (1 << 19) + 1, 16384   # 2^33 elements and one row
    y8 = torch.empty(rows, C, dtype=torch.uint8, device=DEV).random_(0, 127, generator=g).view(t.E4M3)   # no NaN
    s = rand(g, rows, 1)
    whole = t.dequant_q8(y8, s)
    for part in (slice(0, rows // 2), slice(rows // 2, rows)):
        assert torch.equal(whole[part], t.dequant_q8(y8[part], s[part]))
    assert torch.equal(whole[-1].float(), (y8[-1].float() * s[-1]).to(BF).float())
    del y8, whole
    torch.cuda.empty_cache()


def test_attention_limits_are_refused():
    t = tk()
    q = torch.zeros(1, 1, 1, 8, dtype=BF, device=DEV).expand(1 << 23, 1, 1, 8)
    with pytest.raises(ValueError, match="2\\^23"):
        t.window_attention(q, q, q, 1)
    wide = torch.zeros(1, 1, 1, 128, dtype=F32, device=DEV).expand(1, 1, 1 << 14, 128)
    with pytest.raises(ValueError, match="token of q"):
        t.window_attention(wide, wide, wide, 1)
    q = torch.zeros(1, 3, 1, 8, device=DEV)
    with pytest.raises(ValueError, match="scale"):
        t.window_attention(q, q, q, 1, scale=3e38)
    # a window of more than all tokens, however large
    q = rand(gen(84), 1, 40, 2, 8)
    assert torch.equal(t.window_attention(q, q, q, 1 << 70), t.window_attention(q, q, q, 40))


@pytest.mark.parametrize("ty", [BF, F32])
def test_attention_infinite_far_row_and_padded_sinks(ty):
    """More sinks than the sequence has tokens, and an infinite gradient in a row far from them: the keys
    behind the sequence's end still get zeros."""
    g = gen(85)
    N, n, D = 2048, 390, 64
    q, k, v, do = (rand(g, 1, N, 1, D, type=ty) for _ in range(4))
    do[0, 10] = math.inf
    leaves = [t.requires_grad_() for t in (q, k, v)]
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    o = tk().window_attention(*leaves, 8, 400, causal=False, lengths=lens)
    for d in torch.autograd.grad(o, leaves, do):
        assert torch.equal(d[0, n:], torch.zeros_like(d[0, n:]))


@pytest.mark.parametrize("ty", [BF, F32])
@pytest.mark.parametrize("which", [0, 1, 2, 3])
def test_attention_of_nothing_but_nan(which, ty):
    """Every result that depends on a NaN is NaN, padding keeps its zeros."""
    g = gen(86)
    N, n = 700, 690
    t = [rand(g, 1, N, h, 64, type=ty) for h in (4, 2, 2, 4)]
    t[which].fill_(math.nan)
    leaves = [x.requires_grad_() for x in t[:3]]
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    o = tk().window_attention(*leaves, 50, 4, lengths=lens)
    got = (o, *torch.autograd.grad(o, leaves, t[3]))
    # v reaches dS through dO . (V - O); dV is P^T dO, which knows of q, k and dO; O of all but dO
    hit = {0: (1, 1, 1, 1), 1: (1, 1, 1, 1), 2: (1, 1, 1, 0), 3: (0, 1, 1, 1)}[which]
    for x, nan in zip(got, hit):
        assert torch.isnan(x[0, :n]).all() if nan else torch.isfinite(x[0, :n]).all()
        assert torch.equal(x[0, n:], torch.zeros_like(x[0, n:]))


@pytest.mark.parametrize("ty", [BF, F32])
@pytest.mark.parametrize("B,N,H,Hk,D,window,sinks,causal,lengths", [
    (3, 700, 6, 2, 80, 90, 7, True, [700, 320, 0]), (3, 700, 2, 2, 128, 200, 0, False, [1, 700, 128]),
    (5, 400, 4, 1, 64, 50, 4, True, [129, 127, 128, 400, 3]), (2, 1500, 2, 1, 128, 400, 40, True, [200, 1400]),
    (4, 130, 3, 1, 32, 130, 0, False, [0, 0, 130, 0]), (2, 300, 2, 2, 40, 60, 0, True, [0, 0])])
def test_attention_padded_tiles(B, N, H, Hk, D, window, sinks, causal, lengths, ty):
    """Padding of all sizes: live tiles are dealt out first, and the backward cuts them by how many there are."""
    g = gen(B * N + D)
    q, k, v, do = (rand(g, B, N, h, D, type=ty) for h in (H, Hk, Hk, H))
    first = check_train(q, k, v, do, window, sinks, causal, lengths)
    for a, b in zip(first, check_train(q, k, v, do, window, sinks, causal, lengths)):
        assert torch.equal(a, b)
    for b, n in enumerate(lengths):
        for x in first:
            assert torch.equal(x[b, n:], torch.zeros_like(x[b, n:]))


@pytest.mark.parametrize("B", [63, 64, 65])
def test_attention_many_padded_sequences(B):
    """Up to 64 sequences' lengths are looked through by a workgroup; more take the plain order."""
    g = gen(B)
    N = 150
    q, k, v, do = (rand(g, B, N, 2, 32, type=BF) for _ in range(4))
    check_train(q, k, v, do, 40, 2, True, [(37 * b) % (N + 1) for b in range(B)])


def test_attention_padded_graph_with_other_lengths():
    """A captured call finds its tiles by the lengths of the replay, not of the capture."""
    t, g = tk(), gen(87)
    q, k, v, do = (rand(g, 3, 600, h, 64, type=F32) for h in (6, 2, 2, 6))
    leaves = [x.requires_grad_() for x in (q, k, v)]
    n = torch.tensor([600, 600, 600], dtype=torch.int32, device=DEV)

    def run():
        o = t.window_attention(*leaves, 90, 3, lengths=n)
        return [o.detach(), *torch.autograd.grad(o, leaves, do)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for lens in ([600, 10, 300], [0, 0, 0], [5, 600, 129], [600, 600, 600]):
        n.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out]
        for a, b in zip(got, run()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("B,T,cap,H,Hk,D,window,sinks,lengths", [c for c in CACHED if c[1] * c[3] // c[4] <= 64 and max(c[8]) > 1] + [
    (1, 1, 4096, 16, 4, 128, 1024, 4, [4096])])
def test_attention_few_rows_keep_p(B, T, cap, H, Hk, D, window, sinks, lengths):
    """Up to 64 rows a key head: the results' error is that of rounding the exact ones to bf16.  P in two bf16 is off by
    2^-16, fp32 sums and scores by less: independent errors add in squares, 2^-14 of the norm beside the rounding's
    2^-10.5 or more is 1.004 times it.  (P in one bf16: 1.08 to 1.35 times.)"""
    g = gen(cap + D)
    q, k, v = rand(g, B, T, H, D, type=BF), rand(g, B, cap, Hk, D, type=BF), rand(g, B, cap, Hk, D, type=BF)
    o = tk().window_attention_cached(q, k, v, torch.tensor(lengths, dtype=torch.int32, device=DEV), window, sinks)
    err = rounding = 0.0
    for b in range(B):
        L = min(max(lengths[b], 0), cap)
        want = attn_ref(q[b], k[b], v[b], None, visible(T, cap, L, L - T, window, sinks, True), 1 / math.sqrt(D), BF)[0][0]
        err += float((o[b].double() - want).square().sum())
        rounding += float((want.to(BF).double() - want).square().sum())
    assert math.sqrt(err) <= 1.03 * math.sqrt(rounding), math.sqrt(err / rounding)


@pytest.mark.parametrize("ty", [BF, F32])
@pytest.mark.parametrize("T,cap,H,Hk", [(1, 4096, 2, 2), (70, 5000, 8, 8), (4, 90, 2, 1)])
def test_attention_visible_nan_of_no_weight(T, cap, H, Hk, ty):
    """A NaN or infinity in a visible value reaches the row however small its weight is, also where the keys are split
    (the first two) and the weight of its whole split rounds to 0: 0 times it is NaN."""
    g, D = gen(cap), 64
    q, k, v = torch.ones(1, T, H, D, dtype=ty, device=DEV), rand(g, 1, cap, Hk, D, type=ty), rand(g, 1, cap, Hk, D, type=ty)
    k[0, cap - T] = 40.0   # seen by all rows: a score of 320, e^250 times all others
    n = torch.tensor([cap], dtype=torch.int32, device=DEV)
    o = tk().window_attention_cached(q, k, v, n, cap)
    within(o, v[:, cap - T, None].repeat_interleave(H // Hk, 2).expand_as(o).double(), 4 * UT[ty] * v.double().abs().amax().expand_as(o), "o")
    for bad in (math.nan, math.inf):
        for at in (5, cap // 2):
            w = v.clone()
            w[0, at] = bad
            assert not torch.isfinite(tk().window_attention_cached(q, k, w, n, cap)).any(), (bad, at)


def test_tangents_of_gradients_are_refused():
    """Forward mode over the backward pass: the gradients' tangents would be lost."""
    t, g = tk(), gen(101)
    q, x = rand(g, 1, 9, 2, 16).requires_grad_(), rand(g, 3, 16).requires_grad_()
    w, pos = torch.ones(16, device=DEV), torch.zeros(9, 1, dtype=torch.int32, device=DEV)
    for leaf, out in ((x, t.rms_norm_residual(x, x, w)[0]), (q, t.rotary(q, None, pos, (4,))[0]), (q, t.window_attention(q, q, q, 3))):
        with torch.autograd.forward_ad.dual_level():
            d = torch.autograd.forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(out, leaf, d)


@pytest.mark.parametrize("ty", [BF, F32])
@pytest.mark.parametrize("N,D,window,sinks", [(2048, 64, 30, 40), (300, 96, 30, 100), (5000, 128, 100, 4)])
def test_attention_infinite_far_gradient(N, D, window, sinks, ty):
    """An infinite gradient in one column of a row far from the sinks: their dV is infinite there (P is above 0), not NaN."""
    g = gen(N)
    q, k, v, do = (rand(g, 1, N, 1, D, type=ty) for _ in range(4))
    do[0, N - 2, 0, 5] = math.inf
    v.requires_grad_()
    (dv,) = torch.autograd.grad(tk().window_attention(q, k, v, window, sinks, causal=False), v, do)
    assert torch.isposinf(dv[0, :sinks, 0, 5]).all()
    assert torch.isfinite(dv[0, :sinks, 0, :5]).all() and torch.isfinite(dv[0, :sinks, 0, 6:]).all()


def kinds(x):
    return torch.isnan(x).int() + 2 * torch.isposinf(x).int() + 4 * torch.isneginf(x).int()


@pytest.mark.parametrize("ty", [BF, F32])
@pytest.mark.parametrize("N,H,Hk,D,window,sinks,causal", [(130, 2, 1, 32, 40, 3, True), (40, 2, 2, 64, 9, 0, False),
                                                          (300, 1, 1, 96, 30, 100, False), (900, 2, 1, 40, 60, 2, True)])
def test_attention_infinite_values(N, H, Hk, D, window, sinks, causal, ty):
    """Infinities of both signs and NaN in single places of v and dO: o and dV are infinite, NaN and finite where the
    sums over the visible pairs are."""
    g = gen(N + D)
    q, k, v, do = (rand(g, 1, N, h, D, type=ty) for h in (H, Hk, Hk, H))
    mask, scale = visible(N, N, N, 0, window, sinks, causal), 1 / math.sqrt(D)
    want, bound = attn_ref(q[0], k[0], v[0], do[0], mask, scale, ty)
    bad = torch.tensor([math.inf, -math.inf, math.nan], device=DEV)

    def spoil(x):
        x = x.clone()
        for i in range(12):
            x[0, (i * 37 + 1) % N, i % x.shape[2], (i * 5) % D] = bad[i % 3]
        return x

    vs, dos = spoil(v), spoil(do)
    leaves = [t.requires_grad_() for t in (q, k, vs)]
    o = tk().window_attention(*leaves, window, sinks, causal=causal)
    dv = torch.autograd.grad(tk().window_attention(q, k, v.requires_grad_(), window, sinks, causal=causal), v, dos)[0]
    # sign of each visible pair's term (every P is above 0), 3 for NaN: what a sum of them is
    for got, src, see, fine, eps, heads in ((o, vs, mask.int(), want[0], bound[0], True), (dv, dos, mask.int().T, want[3], bound[3], False)):
        x = src[0].detach()
        if heads:
            x = x.repeat_interleave(H // Hk, 1)
        n = [torch.einsum("ab,bhd->ahd", see.double(), c.double()) for c in (torch.isnan(x), torch.isposinf(x), torch.isneginf(x))]
        if not heads:
            n = [c.view(N, Hk, H // Hk, D).sum(2) for c in n]
        nan = (n[0] > 0) | ((n[1] > 0) & (n[2] > 0))
        kind = nan.int() + 2 * ((n[1] > 0) & ~nan).int() + 4 * ((n[2] > 0) & ~nan).int()
        assert torch.equal(kinds(got[0].detach()), kind)
        free = kind == 0
        assert free.any() and not free.all()
        within(got[0][free], fine[free], eps[free], "finite ones")


@pytest.mark.parametrize("ty", [BF, F32])
@pytest.mark.parametrize("T,cap", [(1, 4096), (4, 300), (100, 2000)])
def test_attention_cached_infinite_values(T, cap, ty):
    """The same over a cache, the keys split or not: which columns are infinite is the sum over visible pairs."""
    g, H, Hk, D, window = gen(T + cap), 4, 2, 64, cap - 100
    q, k, v = rand(g, 1, T, H, D, type=ty), rand(g, 1, cap, Hk, D, type=ty), rand(g, 1, cap, Hk, D, type=ty)
    n = torch.tensor([cap - 5], dtype=torch.int32, device=DEV)
    mask = visible(T, cap, cap - 5, cap - 5 - T, window, 3, True)
    want, bound = attn_ref(q[0], k[0], v[0], None, mask, 1 / math.sqrt(D), ty)
    w = v.clone()
    w[0, 1, 0, 3], w[0, cap // 2, 0, 3], w[0, cap - 7, 0, 5], w[0, cap - 6 - T // 2, 1, 7], w[0, cap - 3] = math.inf, -math.inf, -math.inf, math.nan, math.nan
    o = tk().window_attention_cached(q, k, w, n, window, 3)
    see = mask.double()
    x = w[0].repeat_interleave(H // Hk, 1)
    c = [torch.einsum("ab,bhd->ahd", see, torch.where(mask.any(0)[:, None, None], y, False).double()) > 0
         for y in (torch.isnan(x), torch.isposinf(x), torch.isneginf(x))]
    nan = c[0] | (c[1] & c[2])
    kind = nan.int() + 2 * (c[1] & ~nan).int() + 4 * (c[2] & ~nan).int()
    assert torch.equal(kinds(o[0]), kind)
    within(o[0][kind == 0], want[0][kind == 0], bound[0][kind == 0], "finite ones")


@pytest.mark.parametrize("ty", [BF, F32])
def test_attention_of_values_that_are_not_finite_takes_no_longer_way(ty):
    """Sums that are not finite are formed again with matrix products: a second pass of four products for one and their
    operands' classes, 10 times the first's at most, and 25 here for short times.  (One pair after the other: 34 to 63.)"""
    g, N, H, Hk, D = gen(103), 4096, 8, 2, 128
    t = [rand(g, 1, N, h, D, type=ty) for h in (H, Hk, Hk, H)]

    def times(which=None, where=slice(None), value=0.0):
        x = [y.clone() for y in t]
        if which is not None:
            x[which][where] = value
        leaves, best = [y.requires_grad_() for y in x[:3]], [math.inf, math.inf]
        for _ in range(4):
            e = [torch.cuda.Event(enable_timing=True) for _ in range(3)]
            e[0].record()
            o = tk().window_attention(*leaves, 512, 4)
            e[1].record()
            torch.autograd.grad(o, leaves, x[3])
            e[2].record()
            torch.cuda.synchronize()
            best = [min(best[0], e[0].elapsed_time(e[1])), min(best[1], e[1].elapsed_time(e[2]))]
        return best

    clean = times()
    for case in ((0, slice(None), math.nan), (1, slice(None), math.inf), (2, slice(None), math.nan), (2, slice(None), math.inf),
                 (3, slice(None), math.nan), (3, slice(None), -math.inf), (2, (0, 0), math.nan), (2, (0, 0, 0, 5), math.inf),
                 (3, (0, 2000), math.inf), (1, (0, 1), math.inf), (0, (0, 2000), math.nan)):
        spoilt = times(*case)
        assert spoilt[0] < 25 * clean[0] and spoilt[1] < 25 * clean[1], (case, spoilt, clean)


@pytest.mark.parametrize("ty", [BF, F32])
def test_attention_scores_of_minus_infinity(ty):
    """A softmax over nothing but -inf is NaN; over -inf and others it is the others'.  Padding keeps its zeros."""
    g, D = gen(107), 32
    # training: row 6 sees keys 5 and 6 alone, whose scores are -inf, row 5 sees 4 as well, row 7 itself
    for N in (40, 300):
        q, k, v, do = (rand(g, 2, N, 1, D, type=ty) for _ in range(4))
        q[..., 0] = 1.0
        k[:, 5:7, :, 0] = -math.inf
        leaves = [t.requires_grad_() for t in (q, k, v)]
        n = torch.tensor([N, 6], dtype=torch.int32, device=DEV)
        o = tk().window_attention(*leaves, 2, lengths=n)
        dq, dk, dv = torch.autograd.grad(o, leaves, do)
        hit = torch.zeros(2, N, dtype=torch.bool, device=DEV)
        hit[0, 6] = True
        assert torch.isnan(o[hit]).all() and torch.isfinite(o[~hit]).all()
        assert torch.isnan(dq[hit]).all()
        within(o[0, 5], v[0, 4].double(), 4 * UT[ty] * v[0, 4].double().abs(), "row 5")
        within(o[0, 7], v[0, 7].double(), 4 * UT[ty] * v[0, 7].double().abs(), "row 7")
        assert torch.equal(o[1, 6:], torch.zeros_like(o[1, 6:]))
    # a cache, whole and split, one of two sequences with nothing but -inf; the first token lies before its start
    for T, cap in ((1, 30), (1, 4096), (100, 4096)):
        q, k, v = rand(g, 2, T, 2, D, type=ty), rand(g, 2, cap, 2, D, type=ty), rand(g, 2, cap, 2, D, type=ty)
        q[..., 0] = 1.0
        k[0, ..., 0] = -math.inf
        n = torch.tensor([cap, cap - 3], dtype=torch.int32, device=DEV)
        o = tk().window_attention_cached(q, k, v, n, cap)
        assert torch.isnan(o[0]).all() and torch.isfinite(o[1]).all()
        n = torch.tensor([0, T - 1], dtype=torch.int32, device=DEV)
        o = tk().window_attention_cached(q, k, v, n, cap)
        assert torch.equal(o[0], torch.zeros_like(o[0])) and torch.equal(o[1, 0], torch.zeros_like(o[1, 0]))


# Where bf16 is rounded: P and dS before the second products, and the results.  Independent roundings add in squares, so
# beside the results' own rounding (1) the first add up to 1 (less over few keys, where the largest P is 1 and the sum is
# of the rounded ones): sqrt(2) of it for dV and O, and for dQ and dK with delta's part of P's rounding 1.46 to 1.53 with
# windows of 2 to 64 keys when the formulas are put in 64 bits with those roundings alone; 1.73 and more if O's rounding
# reaches delta, 2.0 and more with its rest subtracted (windows of 2 and 3: 1.93 to 2.27 and 2.8 to 3.7).
def rel(got, want):
    """The 2-norm of the error, in that of rounding the exact result to bf16."""
    return float((got.double() - want).norm() / (want.to(BF).double() - want).norm())


@pytest.mark.parametrize("N,H,Hk,D,window,causal", [
    (60, 2, 2, 64, 2, True), (15, 16, 4, 128, 2, True), (62, 3, 3, 40, 3, False),   # up to 64 rows a key head
    (300, 8, 8, 64, 2, True), (300, 8, 2, 128, 3, True), (1100, 4, 4, 96, 2, True), (500, 6, 6, 32, 2, False), (2500, 4, 2, 128, 3, True)])
def test_attention_error_norms(N, H, Hk, D, window, causal):
    """Over few keys dS is a small difference: its error shows whether delta is formed from more than O's 8 bits."""
    g = gen(N + D)
    q, k, v, do = (rand(g, 1, N, h, D, type=BF) for h in (H, Hk, Hk, H))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = tk().window_attention(*leaves, window, causal=causal)
    got = (o.detach(), *torch.autograd.grad(o, leaves, do))
    want, _ = attn_ref(q[0].detach(), k[0].detach(), v[0].detach(), do[0], visible(N, N, N, 0, window, 0, causal), 1 / math.sqrt(D), BF)
    for name, a, b, limit in zip(("o", "dq", "dk", "dv"), got, want, (1.45, 1.65, 1.65, 1.5)):
        assert rel(a[0], b) <= limit, (name, rel(a[0], b))


@pytest.mark.parametrize("spoilt", [False, True])
@pytest.mark.parametrize("N,H,Hk,D,window,limit", [(60, 2, 2, 64, 2, 0.85), (15, 16, 4, 128, 3, 0.85), (300, 8, 8, 64, 2, 0.85),
                                                   (1100, 4, 2, 96, 3, 0.85), (2000, 1, 1, 64, 2000, 1.2)])
def test_attention_rest_of_o(N, H, Hk, D, window, limit, spoilt):
    """o and what its rounding left: together as far off as P's rounding makes them (0.33 to 0.7 of o's own over few keys,
    up to 1 over many), not more (alone 1.05 and more, 1.4 over many).  The kernels for few rows, for tiles of rows, the
    keys split and joined (the last); spoilt: rows formed again beside a NaN that they do not see.  lse as well."""
    import ctypes
    from dfcsa._lib import LIB, WattnDesc
    g = gen(N + D)
    q, k, v = rand(g, 1, N, H, D, type=BF), rand(g, 1, N, Hk, D, type=BF), rand(g, 1, N, Hk, D, type=BF)
    live, first = (N - 1, N - 12) if spoilt else (N, 0)   # the last rows are formed again beside the last key's NaN
    want, _ = attn_ref(q[0], k[0], v[0], None, visible(N, N, N, 0, window, 0, True), 1 / math.sqrt(D), BF)
    if spoilt:
        v[0, -1] = math.nan
    o, rest, lse = torch.empty_like(q), torch.empty_like(q), torch.empty(Hk * N * (H // Hk), device=DEV)
    d = WattnDesc(dtype=1, B=1, T=N, M=N, H=H, Hk=Hk, D=D, window=window, sinks=0, causal=1, cached=0, scale=1 / math.sqrt(D),
                  q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), o=o.data_ptr(), o_rest=rest.data_ptr(), lse=lse.data_ptr())
    d.q_stride[:], d.k_stride[:], d.v_stride[:] = q.stride()[:3], k.stride()[:3], v.stride()[:3]
    n = ctypes.c_int64()
    assert LIB.dfcsa_wattn_work_floats(ctypes.addressof(d), 0, ctypes.byref(n)) == 0
    assert (n.value > 0) == (N == 2000)
    work = torch.empty(max(n.value, 1), device=DEV)
    d.work, d.work_floats = work.data_ptr(), n.value
    assert LIB.dfcsa_wattn_fwd(ctypes.addressof(d), torch.cuda.current_stream().cuda_stream) == 0
    both, exact = (o.double() + rest.double())[0, first:live], want[0][first:live]
    assert rel(both, exact) <= limit, rel(both, exact)
    assert rel(o[0, first:live], exact) <= 1.45
    s = (torch.einsum("nhd,mhd->hnm", q[0].double(), k[0].double().repeat_interleave(H // Hk, 1)) / math.sqrt(D)).masked_fill(
        ~visible(N, N, N, 0, window, 0, True), -math.inf)
    got = lse.view(Hk, N, H // Hk).permute(0, 2, 1).reshape(H, N).double() * math.log(2)
    # of the rounded P: 2^-8 at most; scores and sums in fp32, and the lse's own rounding, stay below 2^-14 here
    assert float((got - torch.logsumexp(s, -1)).abs().max()) <= 2.0 ** -8 + 2.0 ** -14


@pytest.mark.parametrize("ty", [BF, F32])
@pytest.mark.parametrize("N,H,Hk,D,window,sinks,causal", [(260, 2, 2, 64, 260, 0, True), (60, 2, 1, 64, 60, 3, True), (2500, 2, 1, 64, 100, 40, True),
                                                          (700, 1, 1, 128, 700, 0, False), (1500, 2, 2, 96, 60, 4, False)])
def test_attention_large_scores_backward(N, H, Hk, D, window, sinks, causal, ty):
    """Scores of +-1000: P is formed again from the log-sum of rows whose maximum moved far, in all passes of the backward."""
    g = gen(N + 41)
    q, k, v, do = (rand(g, 1, N, h, D, type=ty) for h in (H, Hk, Hk, H))
    k = (k * torch.linspace(0.1, 30, N, device=DEV)[:, None, None]).to(ty)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = tk().window_attention(*leaves, window, sinks, causal=causal, scale=0.125)
    got = (o.detach(), *torch.autograd.grad(o, leaves, do))
    want, bound = attn_ref(*(t[0].detach() for t in leaves), do[0], visible(N, N, N, 0, window, sinks, causal), 0.125, ty)
    # a P below fp32's smallest normal number, 2^-126, is 0: each of a sum's at most N * H terms is off by that times at
    # most |dP - delta| < 2^8 and |q| or |k| < 2^8 (0.125 of it)
    floor = N * H * 2.0 ** -113
    for name, a, b, e in zip(("o", "dq", "dk", "dv"), got, want, bound):
        within(a[0], b, e + floor, name)


@pytest.mark.parametrize("ty", [BF, F32])
def test_attention_one_input_at_a_time(ty):
    """Gradients of some inputs alone are those of all; without k's and v's nothing is allocated or computed for them."""
    g, N, H, D = gen(109), 3000, 4, 64
    t = [rand(g, 1, N, H, D, type=ty) for _ in range(4)]
    leaves = [x.detach().clone().requires_grad_() for x in t[:3]]
    whole = torch.autograd.grad(tk().window_attention(*leaves, 100, 3), leaves, t[3])
    for want in ((0,), (1,), (2,), (0, 1), (0, 2), (1, 2)):
        x = [y.detach().clone().requires_grad_(i in want) for i, y in enumerate(t[:3])]
        o = tk().window_attention(*x, 100, 3)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        got = torch.autograd.grad(o, [x[i] for i in want], t[3])
        peak = torch.cuda.max_memory_allocated() - before
        for i, d in zip(want, got):
            assert torch.equal(d, whole[i]), (want, i)
        # dQ and delta (a float for each row).  The allocator counts a cached block whole where it is less than 1 MiB too
        # long, for each of the two; dK and dV alone would be 3 MB or more.
        if want == (0,):
            assert peak <= t[0].numel() * t[0].element_size() + N * H * 4 + (2 << 20)


def test_norm_eps_is_finite_in_fp32():
    """An eps that fp32 holds as infinity would make every result 0."""
    x, w = torch.ones(2, 16, device=DEV), torch.ones(16, device=DEV)
    for call in (tk().rms_norm_residual, tk().rms_norm_residual_q8):
        with pytest.raises(ValueError, match="eps"):
            call(x, x, w, eps=1e39)


@pytest.mark.parametrize("ty", [BF, F32])
def test_one_tensor_in_several_places(ty):
    """The same tensor as x and residual, as q and k, as k and v, as all three: its gradient is the sum of theirs."""
    g, t = gen(113), tk()
    x, w, dy, dr = rand(g, 5, 64, type=ty), torch.ones(64, device=DEV), rand(g, 5, 64, type=ty), rand(g, 5, 64, type=ty)
    q, do, dk = rand(g, 1, 70, 2, 32, type=ty), rand(g, 1, 70, 2, 32, type=ty), rand(g, 1, 70, 2, 32, type=ty)
    pos = torch.arange(70, dtype=torch.int32, device=DEV)[:, None]
    calls = ((x, 2, lambda a, b: t.rms_norm_residual(a, b, w), (dy, dr)), (q, 2, lambda a, b: t.rotary(a, b, pos, (16,)), (do, dk)),
             (q, 2, lambda a, b: t.window_attention(q, a, b, 9, 2), do), (q, 3, lambda a, b, c: t.window_attention(a, b, c, 9, 2), do))
    for src, n, call, grads in calls:
        one, apart = src.clone().requires_grad_(), [src.clone().requires_grad_() for _ in range(n)]
        a, b = call(*[one] * n), call(*apart)
        same = zip(a, b) if isinstance(a, tuple) else ((a, b),)
        assert all(torch.equal(u, v) for u, v in same)
        (got,) = torch.autograd.grad(a, one, grads)
        parts = [p.double() for p in torch.autograd.grad(b, apart, grads)]
        # torch adds the parts in their type: half a step of each sum
        within(got, sum(parts), n * UT[ty] * sum(p.abs() for p in parts), "sum")
