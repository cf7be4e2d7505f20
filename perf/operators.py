"""Cases of the token operators (dfcsa.token_ops): what they compute, and what is timed.

Three families, the parts of one transformer block over image, video or text tokens:

  norm     residual stream r = x + residual, y = rms_norm(r) * weight; training (with its gradients) or
           serving (y as e4m3 values with a scale for each row or group of columns)
  rotary   rotary positions with one to three axes on q and k; training or serving
  attn     attention with a sliding window and always-visible first tokens, grouped key heads; training
           over (padded) sequences, or new tokens over a cache

Where `own` is false every operator is its plain form in elementary torch operations, 32 bits inside.
"""
import math
import os
import sys

import torch

own = False

BF16, F32 = torch.bfloat16, torch.float32
TYPES = {"bf16": BF16, "fp32": F32}
DEV = "cuda"


def _ops():
    pkg = os.path.join(os.getcwd(), "dfc-sa-unet_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from dfcsa import token_ops
    return token_ops


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one training step's norm of a ViT-B/16 block at 224 x 224, batch 16: bf16 branch onto the fp32 stream
        dict(name="norm train vit", op="norm", mode="train", rows=3136, C=768, type="bf16", stream="fp32"),
        # the same step of a wide model over long sequences, everything in bf16
        dict(name="norm train wide", op="norm", mode="train", rows=16384, C=4096, type="bf16", stream="bf16"),
        # serving four sequences, one new token each: latency only
        dict(name="norm q8 token", op="norm", mode="q8", rows=4, C=768, type="bf16", stream="bf16", group=0),
        # serving a prompt, an odd number of rows, a scale for each 128 columns
        dict(name="norm q8 prompt", op="norm", mode="q8", rows=8191, C=2560, type="bf16", stream="fp32", group=128),
        # ViT tokens of 14 x 14 patches, q and k read in place from the fused projection, with gradients
        dict(name="rotary train image", op="rotary", mode="train", B=16, N=196, H=12, Hk=12, D=64, axes="16,16",
             type="bf16", shared=False, interleaved=False, far=0),
        # a video prompt: time x height x width, shared frequencies, grouped key heads
        dict(name="rotary video", op="rotary", mode="serve", B=1, N=16384, H=16, Hk=4, D=128, axes="16,24,24",
             type="bf16", shared=True, interleaved=False, far=0),
        # one new token for each of eight sequences, at far positions
        dict(name="rotary token", op="rotary", mode="serve", B=8, N=1, H=16, Hk=4, D=128, axes="16,24,24",
             type="bf16", shared=True, interleaved=False, far=1000000),
        # ViT tokens plus four register tokens that everybody sees, two-sided window, with gradients
        dict(name="attn train image", op="attn", mode="train", B=16, N=200, H=12, Hk=12, D=64, window=57, sinks=4,
             causal=False, ragged=False, type="bf16"),
        # a long causal sequence with grouped key heads: the largest training call
        dict(name="attn train long", op="attn", mode="train", B=1, N=8192, H=16, Hk=4, D=128, window=1024, sinks=4,
             causal=True, ragged=False, type="bf16"),
        # a padded batch of odd lengths in full precision, head width 80
        dict(name="attn train ragged fp32", op="attn", mode="train", B=3, N=1531, H=6, Hk=2, D=80, window=300,
             sinks=7, causal=True, ragged=True, type="fp32"),
        # one stream, one new token: latency, few rows over a longer axis
        dict(name="attn decode one", op="attn", mode="decode", B=1, T=1, cap=4096, H=16, Hk=4, D=128, window=1024,
             sinks=4, type="bf16"),
        # a serving batch, one new token each, long caches and a wide window
        dict(name="attn decode batch", op="attn", mode="decode", B=32, T=1, cap=16384, H=32, Hk=8, D=128, window=4096,
             sinks=16, type="bf16"),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm train", "norm q8", "rotary train", "rotary serve", "attn train", "attn train",
                       "attn decode", "attn decode"])
    op, mode = kind.split()
    ty = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    if op == "norm":
        C = 8 * _log(rng, 4, 1024)
        rows = _log(rng, 1, max(1, min(65536, 32_000_000 // C)))
        stream = "fp32" if ty == "fp32" else rng.choice(["fp32", "bf16"])
        case = dict(op=op, mode=mode, rows=rows, C=C, type=ty, stream=stream)
        if mode == "q8":
            case["C"] = C = 128 * _log(rng, 1, 64)
            case["rows"] = max(1, min(rows, 32_000_000 // C))
            case["group"] = rng.choice([0, 0, 32, 64, 128])
        return case
    Hk = _log(rng, 1, 12)
    H = Hk * rng.choice([1, 1, 2, 3, 4, 8])
    if op == "rotary":
        D = 8 * rng.randint(2, 32)
        naxes = rng.randint(1, 3)
        left, axes = D // 2, []
        for a in range(naxes):
            n = rng.randint(1, max(1, left // (naxes - a)))
            axes.append(n)
            left -= n
        B = _log(rng, 1, 16)
        N = _log(rng, 1, max(1, min(16384, 32_000_000 // (B * (H + Hk) * D))))
        return dict(op=op, mode=mode, B=B, N=N, H=H, Hk=Hk, D=D, axes=",".join(map(str, axes)), type=ty,
                    shared=rng.random() < 0.5, interleaved=rng.random() < 0.5, far=rng.choice([0, 0, 100000, 1000000]))
    D = 8 * rng.randint(2, 16)
    sinks = rng.choice([0, 1, 4, 16, 70])
    if mode == "train":
        B = _log(rng, 1, 16)
        N = _log(rng, 1, max(1, min(6000, int(math.sqrt(600_000_000 / (B * H))))))
        window = _log(rng, 1, max(1, 2 * N))
        return dict(op=op, mode=mode, B=B, N=N, H=H, Hk=Hk, D=D, window=window, sinks=sinks,
                    causal=rng.random() < 0.7, ragged=rng.random() < 0.5, type=ty)
    B = _log(rng, 1, 64)
    T = rng.choice([1, 1, 1, 2, 5, 64])
    cap = _log(rng, T, max(T, min(32768, 300_000_000 // (B * Hk * D), 500_000_000 // (B * H * T))))
    return dict(op=op, mode=mode, B=B, T=T, cap=cap, H=H, Hk=Hk, D=D, window=_log(rng, 1, max(1, 2 * cap)),
                sinks=sinks, type=ty)


def _axes(case):
    return tuple(int(a) for a in case["axes"].split(","))


def _lengths(case):
    """The valid tokens of each sequence: part of the case, not of the seed, so that work() knows them."""
    B = case["B"]
    if case["mode"] == "train":
        N = case["N"]
        return [max(0, N - (N * b * 3) // (4 * B)) if b < B - 1 or B == 1 else min(N, 1) for b in range(B)] \
            if case["ragged"] else [N] * B
    cap, T = case["cap"], case["T"]
    return [max(min(T, cap), cap - (cap * b) // (2 * B) - b % 3) for b in range(B)]


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))

    def rand(*shape, type=F32):
        return torch.randn(shape, generator=g, device=DEV).to(type)

    ty = TYPES[case["type"]]
    s = {"case": dict(case), "ty": ty}
    train = case["mode"] == "train"
    if case["op"] == "norm":
        rows, C, st = case["rows"], case["C"], TYPES[case["stream"]]
        s["x"] = rand(rows, C, type=ty).requires_grad_(train)
        s["residual"] = rand(rows, C, type=st).mul_(2).requires_grad_(train)
        s["weight"] = (1 + 0.2 * rand(C)).requires_grad_(train)
        if train:
            s["dy"], s["dr"] = rand(rows, C, type=ty), rand(rows, C, type=st)
        return s
    B, H, Hk, D = case["B"], case["H"], case["Hk"], case["D"]
    if case["op"] == "rotary":
        N, A = case["N"], len(_axes(case))
        # the fused projection [q heads | k heads | v heads] that q and k are read from in place
        qkv = rand(B, N, (H + 2 * Hk) * D, type=ty)
        s["q"] = qkv[..., :H * D].view(B, N, H, D).requires_grad_(train)
        s["k"] = qkv[..., H * D:(H + Hk) * D].view(B, N, Hk, D).requires_grad_(train)
        side = max(1, int(round(N ** (1.0 / A))))
        n = torch.arange(N, device=DEV)
        at = [(n // side ** (A - 1 - a)) % side if a else n // side ** (A - 1) for a in range(A)]
        start = torch.randint(0, case["far"] + 1, (B, 1, A), generator=g, device=DEV)
        s["positions"] = (torch.stack(at, -1)[None] + start).to(torch.int32)
        if train:
            s["gq"], s["gk"] = rand(B, N, H, D, type=ty), rand(B, N, Hk, D, type=ty)
        return s
    if train:
        N = case["N"]
        qkv = rand(B, N, (H + 2 * Hk) * D, type=ty)
        s["q"] = qkv[..., :H * D].view(B, N, H, D).requires_grad_(True)
        s["k"] = qkv[..., H * D:(H + Hk) * D].view(B, N, Hk, D).requires_grad_(True)
        s["v"] = qkv[..., (H + Hk) * D:].view(B, N, Hk, D).requires_grad_(True)
        s["do"] = rand(B, N, H, D, type=ty)
        s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device=DEV) if case["ragged"] else None
    else:
        s["q"] = rand(B, case["T"], H, D, type=ty)
        s["k"], s["v"] = rand(B, case["cap"], Hk, D, type=ty), rand(B, case["cap"], Hk, D, type=ty)
        s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device=DEV)
    return s


# ------------------------------------------------------------------ one pass
EPS = 1e-6


def run(s):
    case = s["case"]
    if own:
        return _run_own(s, case)
    with torch.no_grad():
        if case["op"] == "norm":
            return _plain_norm(s, case)
        if case["op"] == "rotary":
            return _plain_rotary(s, case)
        return _plain_attn(s, case)


def _run_own(s, case):
    ops = _ops()
    if case["op"] == "norm":
        if case["mode"] == "q8":
            y8, scales, r = ops.rms_norm_residual_q8(s["x"], s["residual"], s["weight"], eps=EPS, group=case["group"])
            return {"y": ops.dequant_q8(y8, scales), "scales": scales, "r": r}
        y, r = ops.rms_norm_residual(s["x"], s["residual"], s["weight"], eps=EPS)
        dx, dres, dw = torch.autograd.grad((y, r), (s["x"], s["residual"], s["weight"]), (s["dy"], s["dr"]))
        return {"y": y, "r": r, "dx": dx, "dres": dres, "dw": dw}
    if case["op"] == "rotary":
        q, k = ops.rotary(s["q"], s["k"], s["positions"], _axes(case), base=10000.0, shared=case["shared"],
                          interleaved=case["interleaved"])
        if case["mode"] == "serve":
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["gq"], s["gk"]))
        return {"q": q, "k": k, "dq": dq, "dk": dk}
    if case["mode"] == "decode":
        return {"o": ops.window_attention_cached(s["q"], s["k"], s["v"], s["lengths"], case["window"], case["sinks"])}
    o = ops.window_attention(s["q"], s["k"], s["v"], case["window"], case["sinks"], causal=case["causal"],
                             lengths=s["lengths"])
    dq, dk, dv = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])
    return {"o": o, "dq": dq, "dk": dk, "dv": dv}


# The stream is what the next block adds to, so it is held in its own type and the norm is of what it
# holds: r = stream_type(x + residual), y = r / sqrt(mean(r^2) + eps) * weight.
def _plain_norm(s, case):
    ty, st = s["x"].dtype, s["residual"].dtype
    w = s["weight"].float()
    r = (s["x"].float() + s["residual"].float()).to(st)
    rf = r.float()
    rstd = torch.rsqrt((rf * rf).mean(-1, keepdim=True) + EPS)
    y = rf * rstd * w
    if case["mode"] == "q8":
        rows, C = y.shape
        g = case["group"] or C
        yg = y.view(rows, C // g, g)
        scales = yg.abs().amax(-1, keepdim=True).clamp(min=1e-12) / 448.0
        y8 = (yg * (1.0 / scales)).to(torch.float8_e4m3fn)
        return {"y": (y8.float() * scales).view(rows, C).to(BF16), "scales": scales[..., 0], "r": r}
    dy, dr = s["dy"].float(), s["dr"].float()
    wdy, xhat = dy * w, rf * rstd
    d = rstd * (wdy - xhat * (wdy * xhat).mean(-1, keepdim=True)) + dr
    return {"y": y.to(ty), "r": r, "dx": d.to(ty), "dres": d.to(st), "dw": (dy * xhat).sum(0)}


def _turns(case):
    """The frequency of each rotated pair (radians a position) and the axis it follows."""
    axes, freq, axis = _axes(case), [], []
    for a, n in enumerate(axes):
        for i in range(n):
            freq.append(10000.0 ** (-len(freq) / sum(axes)) if case["shared"] else 10000.0 ** (-i / n))
            axis.append(a)
    return freq, axis


def _plain_rotary(s, case):
    freq, axis = _turns(case)
    P, R = len(freq), 2 * len(freq)
    f = torch.tensor(freq, dtype=torch.float64, device=DEV)
    angle = s["positions"].double()[..., torch.tensor(axis, device=DEV)] * f  # far positions: 64 bits
    cos, sin = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]

    def turn(x, sin):
        xf = x.float()
        if case["interleaved"]:
            a, b = xf[..., 0:R:2], xf[..., 1:R:2]
            both = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
        else:
            a, b = xf[..., :P], xf[..., P:R]
            both = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
        return torch.cat((both, xf[..., R:]), -1).to(x.dtype)

    out = {"q": turn(s["q"], sin), "k": turn(s["k"], sin)}
    if case["mode"] == "train":
        out |= {"dq": turn(s["gq"], -sin), "dk": turn(s["gk"], -sin)}
    return out


# Query at position p sees key j where j is before the sequence's end, not after p (causal), and within
# the window, |p - j| < window, or among the first `sinks`.  A row that sees nothing gives zeros.
def _visible(case, s, M):
    T = case["N"] if case["mode"] == "train" else case["T"]
    j = torch.arange(M, device=DEV)
    if case["mode"] == "train":
        length = s["lengths"][:, None, None] if s["lengths"] is not None else torch.full((1, 1, 1), M, device=DEV)
        p = torch.arange(T, device=DEV)[None, :, None]
        alive, causal = p < length, case["causal"]
    else:
        length = s["lengths"][:, None, None]
        p = length - T + torch.arange(T, device=DEV)[None, :, None]
        alive, causal = p >= 0, True
    near = ((p - j).abs() < case["window"]) | (j < case["sinks"])
    seen = alive & (j < length) & near
    return seen & (j <= p) if causal else seen


def _plain_attn(s, case):
    H, Hk, D = case["H"], case["Hk"], case["D"]
    G, ty = H // Hk, s["q"].dtype
    B, T = s["q"].shape[:2]
    M = s["k"].shape[1]
    scale = 1.0 / math.sqrt(D)
    # [B, Hk, G * T, D]: the query heads of a key head stacked over the tokens
    q = s["q"].float().view(B, T, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * T, D)
    k, v = s["k"].float().permute(0, 2, 1, 3), s["v"].float().permute(0, 2, 1, 3)
    seen = _visible(case, s, M)[:, None, None]
    sc = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).view(B, Hk, G, T, M)
    sc = sc.masked_fill_(~seen, -math.inf)
    e = (sc - sc.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    del sc
    p = e.div_(e.sum(-1, keepdim=True).clamp(min=1e-30)).view(B, Hk, G * T, M)
    o = torch.matmul(p, v)

    def back(x):
        return x.view(B, Hk, G, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, H, D).to(ty)

    if case["mode"] == "decode":
        return {"o": back(o)}
    do = s["do"].float().view(B, T, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * T, D)
    dv = torch.matmul(p.transpose(-1, -2), do)
    ds = torch.matmul(do, v.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    del p
    dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(-1, -2), q)
    return {"o": back(o), "dq": back(dq), "dk": dk.permute(0, 2, 1, 3).to(ty), "dv": dv.permute(0, 2, 1, 3).to(ty)}


# ------------------------------------------------------------------ what a pass cannot do without
def _pairs(case):
    """Visible (query, key) pairs and keys read, over the batch."""
    pairs = keys = 0
    W, S = case["window"], case["sinks"]
    for n in _lengths(case):
        if case["mode"] == "train":
            first, causal = 0, case["causal"]
        else:
            first, causal = max(0, n - case["T"]), True
        for p in range(first, n):
            lo, hi = max(0, p - W + 1), (p + 1 if causal else min(n, p + W))
            pairs += hi - lo + min(S, lo) + (max(0, min(S, n) - hi) if not causal else 0)
        if n > first:
            lo = max(0, first - W + 1)
            keys += n - lo + min(S, lo)
    return pairs, keys


def work(case):
    es = {"bf16": 2, "fp32": 4}
    e = es[case["type"]]
    if case["op"] == "norm":
        n, C, st = case["rows"] * case["C"], case["C"], es[case["stream"]]
        if case["mode"] == "q8":  # x, residual in; stream, 8 bits and scales out (and the values as bf16)
            scales = 4 * case["rows"] * (C // case["group"] if case["group"] else 1)
            return {"bytes": n * (e + 2 * st + 1) + scales + 4 * C + n * 2, "flops": 6 * n}
        # x, residual in, y, r out; r, dy, dr in, dx, dres (one where the types are one) out
        return {"bytes": n * (2 * e + 2 * st) + n * (2 * st + e + (e if e == st else e + st)) + 12 * C,
                "flops": 14 * n}
    B, H, Hk, D = case["B"], case["H"], case["Hk"], case["D"]
    if case["op"] == "rotary":
        n = B * case["N"] * (H + Hk) * D
        passes = 2 if case["mode"] == "train" else 1
        return {"bytes": passes * (2 * n * e + 4 * B * case["N"] * len(_axes(case))), "flops": passes * 3 * n}
    pairs, keys = _pairs(case)
    if case["mode"] == "decode":
        return {"bytes": 2 * keys * Hk * D * e + 2 * B * case["T"] * H * D * e, "flops": 4 * pairs * H * D}
    n, m = B * case["N"] * H * D * e, B * case["N"] * Hk * D * e
    return {"bytes": (n + 2 * m + n) + (3 * n + 2 * m) + (n + 2 * m), "flops": 14 * pairs * H * D}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "rotary": _exact_rotary, "attn": _exact_attn}[case["op"]](s, case)


def _e4m3(v):
    """v rounded to the nearest e4m3 value, ties to even: 3 fraction bits, exponents from -6, at most 448."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp(min=-6) - 3)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def _exact_norm(s, case):
    x, w = s["x"].double(), s["weight"].double()
    r = (x + s["residual"].double()).to(s["residual"].dtype)
    rd = r.double()
    norm = torch.sqrt(rd.square().sum(-1, keepdim=True) / case["C"] + EPS)
    unit = rd / norm
    y = unit * w
    if case["mode"] == "q8":
        g = case["group"] or case["C"]
        parts = y.reshape(case["rows"], -1, g)
        scale = torch.maximum(parts.abs().amax(-1), torch.tensor(1e-12, device=DEV, dtype=torch.float64)) / 448
        return {"y": (_e4m3(parts / scale[..., None]) * scale[..., None]).reshape(y.shape), "scales": scale, "r": rd}
    dy, dr = s["dy"].double(), s["dr"].double()
    u = dy * w
    d = (u - unit * ((u * unit).sum(-1, keepdim=True) / case["C"])) / norm + dr
    return {"y": y, "r": rd, "dx": d, "dres": d, "dw": (dy * unit).sum(0)}


def _exact_rotary(s, case):
    axes = _axes(case)
    total, out, pairs = sum(axes), {}, []
    for a, n in enumerate(axes):
        for i in range(n):
            j = len(pairs)
            power = j / total if case["shared"] else i / n
            w = s["positions"][..., a].double() / 10000.0 ** power
            at = (2 * j, 2 * j + 1) if case["interleaved"] else (j, j + total)
            pairs.append((at, torch.complex(torch.cos(w), torch.sin(w))[..., None]))

    def turned(x, conj):
        y = x.double().clone()
        for (a, b), u in pairs:
            z = torch.complex(x[..., a].double(), x[..., b].double()) * (u.conj() if conj else u)
            y[..., a], y[..., b] = z.real, z.imag
        return y

    out["q"], out["k"] = turned(s["q"], False), turned(s["k"], False)
    if case["mode"] == "train":
        out["dq"], out["dk"] = turned(s["gq"], True), turned(s["gk"], True)
    return out


def _exact_attn(s, case):
    """One sequence and query head at a time; the gradients by the chain rule through the softmax."""
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    B, T, H, D = q.shape
    M, G = k.shape[1], H // case["Hk"]
    train = case["mode"] == "train"
    if B * H > 600 and B * H * T * M > 200_000_000:
        return None
    o = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    lengths = _lengths(case)
    key = torch.arange(M, device=DEV)
    for b in range(B):
        n = lengths[b]
        at = torch.arange(T, device=DEV) + (0 if train else n - T)
        t = torch.nonzero((at >= 0) & (at < n))[:, 0]
        if not len(t):
            continue
        gap = at[t][:, None] - key[None, :n]
        hidden = (gap.abs() >= case["window"]) & (key[None, :n] >= case["sinks"])
        if not train or case["causal"]:
            hidden = hidden | (gap < 0)
        for h in range(H):
            K, V, Q = k[b, :n, h // G], v[b, :n, h // G], q[b, t, h] / math.sqrt(D)
            prob = torch.softmax((Q @ K.T).masked_fill(hidden, -math.inf), -1)
            o[b, t, h] = prob @ V
            if train:
                do = s["do"][b, t, h].double()
                dprob = do @ V.T
                dscore = prob * (dprob - (dprob * prob).sum(-1, keepdim=True))
                dq[b, t, h] = dscore @ K / math.sqrt(D)
                dk[b, :n, h // G] += dscore.T @ Q
                dv[b, :n, h // G] += prob.T @ do
    return {"o": o, "dq": dq, "dk": dk, "dv": dv} if train else {"o": o}
