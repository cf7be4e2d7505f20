"""dfcsa.token_ops without a GPU: descriptor layouts, refusals at the C boundary and of host tensors, plans."""
import ctypes
import os
import subprocess

import pytest
import torch

from dfcsa import _lib, token_ops as tk
from dfcsa._lib import EINVAL, LIB

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_descriptor_layouts_match_c(tmp_path):
    fields = [("dfcsa_rotary_desc", _lib.RotaryDesc, [n for n, _ in _lib.RotaryDesc._fields_]),
              ("dfcsa_wattn_desc", _lib.WattnDesc, [n for n, _ in _lib.WattnDesc._fields_])]
    exprs, want = [], []
    for cname, py, names in fields:
        exprs.append(f"sizeof({cname})")
        want.append(ctypes.sizeof(py))
        for n in names:
            exprs.append(f"offsetof({cname}, {n})")
            want.append(getattr(py, n).offset)
    src = tmp_path / "lay.c"
    src.write_text('#include "dfcsa.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(){'
                   + "".join(f'printf("%zu\\n", (size_t){e});' for e in exprs) + "}\n")
    exe = tmp_path / "lay"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    assert [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()] == want


def test_host_tensors_are_refused():
    x, w = torch.randn(2, 8), torch.ones(8)
    q = torch.randn(1, 4, 2, 8)
    n = torch.ones(1, dtype=torch.int32)
    for call in (lambda: tk.rms_norm_residual(x, x, w), lambda: tk.rms_norm_residual_q8(x, x, w),
                 lambda: tk.dequant_q8(x.to(tk.E4M3), torch.ones(2, 1)),
                 lambda: tk.rotary(q, q, torch.zeros(4, 1, dtype=torch.int32), (2,)),
                 lambda: tk.window_attention(q, q, q, 2), lambda: tk.window_attention_cached(q, q, q, n, 2)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_serving_forms_refuse_gradients():
    x, w = torch.randn(2, 8, requires_grad=True), torch.ones(8)
    q = torch.randn(1, 4, 2, 8, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        tk.rms_norm_residual_q8(x, x, w)
    with pytest.raises(RuntimeError, match="no gradient"):
        tk.window_attention_cached(q, q, q, torch.ones(1, dtype=torch.int32), 2)


@pytest.mark.parametrize("axes,base", [((), 1e4), ((1,) * 5, 1e4), ((4, 0), 1e4), ((300,), 1e4), ((200, 200), 1e4),
                                       ((4.5,), 1e4), ((4,), 0.5), ((4,), float("inf")), ((4,), float("nan"))])
def test_rotary_table_refusals(axes, base):
    with pytest.raises(ValueError):
        tk._turn_table(axes, base, False)


P16 = 1 << 20   # an aligned address that nothing reads: every call below is refused before a launch


@pytest.mark.parametrize("ty,rt,rows,C", [(0, 1, 4, 64), (2, 0, 4, 64), (1, 2, 4, 64), (1, 0, 0, 64), (1, 0, -1, 64),
                                          (1, 0, 4, 0), (1, 0, 4, 12), (1, 0, 4, 16392)])
def test_norm_refusals(ty, rt, rows, C):
    assert LIB.dfcsa_rms_fwd(ty, rt, rows, C, P16, P16, P16, 1e-6, P16, P16, P16, None) == EINVAL
    assert LIB.dfcsa_rms_fwd_q8(ty, rt, rows, C, 0, P16, P16, P16, 1e-6, P16, P16, P16, None) == EINVAL
    assert LIB.dfcsa_rms_bwd(ty, rt, rows, C, P16, P16, P16, P16, P16, P16, P16, P16, P16, 1 << 40, None) == EINVAL


@pytest.mark.parametrize("C,group", [(64, 16), (64, 128), (96, 64), (64, -32), (64, 256)])
def test_q8_group_refusals(C, group):
    assert LIB.dfcsa_rms_fwd_q8(1, 0, 4, C, group, P16, P16, P16, 1e-6, P16, P16, P16, None) == EINVAL
    assert LIB.dfcsa_dequant_q8(1, 4, C, group, P16, P16, P16, None) == EINVAL


def test_norm_backward_needs_its_workspace():
    n = LIB.dfcsa_rms_bwd_work_floats(100, 64)
    assert n >= 64
    assert LIB.dfcsa_rms_bwd(1, 0, 100, 64, P16, P16, P16, P16, P16, P16, P16, P16, P16, n - 1, None) == EINVAL
    assert LIB.dfcsa_rms_bwd(1, 0, 100, 64, P16, P16, P16, P16, P16, P16, P16, P16, None, n, None) == EINVAL


def rotary_desc(**over):
    turns, axis = (ctypes.c_double * 8)(*[0.1] * 8), (ctypes.c_ubyte * 8)(*[0] * 4 + [1] * 4)
    d = _lib.RotaryDesc(dtype=1, B=1, N=4, D=16, npairs=8, naxes=2, positions=P16, pos_sb=8, pos_sn=2, pos_sa=1,
                        turns=ctypes.addressof(turns), axis=ctypes.addressof(axis))
    d.keep = (turns, axis)
    for i in range(2):
        d.heads[i], d.src[i], d.dst[i], d.src_sb[i], d.src_sn[i], d.src_sh[i] = 2, P16, P16, 128, 32, 16
    for k, v in over.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("over", [dict(dtype=2), dict(B=0), dict(N=0), dict(D=14), dict(D=2000), dict(npairs=0),
                                  dict(npairs=300, D=1000), dict(naxes=0), dict(naxes=5), dict(naxes=1),
                                  dict(positions=None), dict(turns=None), dict(axis=None), dict(B=1 << 20, N=1 << 20)])
def test_rotary_refusals(over):
    assert LIB.dfcsa_rotary(ctypes.addressof(rotary_desc(**over)), None) == EINVAL


def test_rotary_head_refusals():
    d = rotary_desc()
    d.heads[0] = d.heads[1] = 0
    assert LIB.dfcsa_rotary(ctypes.addressof(d), None) == EINVAL
    d = rotary_desc()
    d.src[1] = None
    assert LIB.dfcsa_rotary(ctypes.addressof(d), None) == EINVAL


def attn_desc(**over):
    i64 = ctypes.c_int64 * 3
    over = dict(over)
    strides = {k: over.pop(k) for k in list(over) if k.endswith("_stride")}
    d = _lib.WattnDesc(dtype=1, B=2, T=100, M=100, H=4, Hk=2, D=64, window=10, sinks=2, causal=1, cached=0, scale=0.125,
                       q=P16, k=P16, v=P16, q_stride=i64(25600, 256, 64), k_stride=i64(12800, 128, 64),
                       v_stride=i64(12800, 128, 64), o=P16, lse=P16, work=P16, work_floats=1 << 40, dout=P16,
                       dout_stride=i64(25600, 256, 64), delta=P16, dq=P16, dk=P16, dv=P16)
    for k, v in over.items():
        setattr(d, k, v)
    for k, v in strides.items():
        getattr(d, k)[:] = v
    return d


BAD = [dict(dtype=2), dict(B=0), dict(T=0), dict(M=0), dict(H=0), dict(Hk=0), dict(H=5), dict(D=0), dict(D=12),
       dict(D=136), dict(window=0), dict(sinks=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
       dict(q=None), dict(k=None), dict(v=None), dict(o=None), dict(q=P16 + 8), dict(v=P16 + 2), dict(T=99),
       dict(cached=1), dict(q_stride=(25600, 252, 64)), dict(k_stride=(12800, 1 << 22, 64)),
       dict(v_stride=(-12800, 128, 64)), dict(q_stride=(25600, 256, 1 << 28)), dict(T=1 << 30, M=1 << 30),
       dict(H=1 << 17, Hk=1 << 17)]


@pytest.mark.parametrize("over", BAD)
def test_attention_refusals(over):
    n = ctypes.c_int64()
    d = attn_desc(**over)
    assert LIB.dfcsa_wattn_fwd(ctypes.addressof(d), None) == EINVAL
    assert LIB.dfcsa_wattn_bwd(ctypes.addressof(d), None) == EINVAL
    assert LIB.dfcsa_wattn_work_floats(ctypes.addressof(d), 0, ctypes.byref(n)) == EINVAL


@pytest.mark.parametrize("over", [dict(lse=None), dict(delta=None), dict(dq=None), dict(dk=None), dict(dv=None),
                                  dict(dout=None), dict(dout=P16 + 4), dict(dout_stride=(25600, 255, 64)),
                                  dict(cached=1, lengths=P16)])
def test_attention_backward_refusals(over):
    assert LIB.dfcsa_wattn_bwd(ctypes.addressof(attn_desc(**over)), None) == EINVAL


def test_attention_workspace_is_checked():
    n = ctypes.c_int64()
    # one token over a long cache: the keys are split
    d = attn_desc(B=1, T=1, M=4096, window=4096, cached=1, lengths=P16)
    assert LIB.dfcsa_wattn_work_floats(ctypes.addressof(d), 0, ctypes.byref(n)) == 0 and n.value > 0
    for over in (dict(work=None), dict(work_floats=n.value - 1)):
        d = attn_desc(B=1, T=1, M=4096, window=4096, cached=1, lengths=P16, **over)
        assert LIB.dfcsa_wattn_fwd(ctypes.addressof(d), None) == EINVAL
    # sinks that all later rows see: their rows are split
    d = attn_desc(B=1, T=4096, M=4096)
    assert LIB.dfcsa_wattn_work_floats(ctypes.addressof(d), 1, ctypes.byref(n)) == 0 and n.value > 0
    d.work_floats = n.value - 1
    assert LIB.dfcsa_wattn_bwd(ctypes.addressof(d), None) == EINVAL


def test_attention_takes_head_major_caches():
    # a head of k or v is a base of its own: its stride has no limit, whatever the group
    n = ctypes.c_int64()
    for H in (2, 16):
        far = (1 << 40, 64, 1 << 34)
        d = attn_desc(B=1, T=1, M=4096, H=H, Hk=2, cached=1, lengths=P16, k_stride=far, v_stride=far)
        assert LIB.dfcsa_wattn_work_floats(ctypes.addressof(d), 0, ctypes.byref(n)) == 0


@pytest.mark.parametrize("over", [dict(B=1 << 23, T=1, M=1, sinks=0), dict(B=1 << 14, T=1 << 17, M=1 << 17, H=2, Hk=1, D=8)])
def test_attention_launches_past_32_bits_are_refused(over):
    # 2^24 workgroups of 256 threads and more
    d = attn_desc(**over)
    assert LIB.dfcsa_wattn_fwd(ctypes.addressof(d), None) == EINVAL
    assert LIB.dfcsa_wattn_bwd(ctypes.addressof(d), None) == EINVAL


def test_argument_corners():
    q, n = torch.randn(1, 4, 2, 8), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        tk.window_attention(q, q, q, float("inf"))
    with pytest.raises(ValueError):
        tk.window_attention_cached(q, q, q, n, 2, float("inf"))
    for call in (lambda: tk.window_attention(q, q, q, 1 << 70), lambda: tk.window_attention(q[0, 0, 0, 0], q, q, 2)):
        with pytest.raises(RuntimeError, match="GPU"):   # so the arguments before it are taken
            call()
    with pytest.raises(RuntimeError, match="no gradient"):
        tk.dequant_q8(torch.zeros(2, 8).to(tk.E4M3), torch.ones(2, 1, requires_grad=True))
    assert LIB.dfcsa_wattn_fwd(ctypes.addressof(attn_desc(scale=3e38)), None) == EINVAL


def calls(x, q):
    """Each entry point with one of x [2, 8] and q [1, 4, 2, 8] among its arguments."""
    n, pos = torch.ones(1, dtype=torch.int32), torch.zeros(4, 1, dtype=torch.int32)
    y, w, r = torch.ones(2, 8), torch.ones(8), torch.ones(1, 4, 2, 8)
    return (lambda: tk.rms_norm_residual(x, y, w)[0], lambda: tk.rms_norm_residual(y, x, w)[0],
            lambda: tk.rms_norm_residual_q8(y, x, w)[1], lambda: tk.dequant_q8(y.to(tk.E4M3), x[:, :1]),
            lambda: tk.rotary(q, r, pos, (2,))[0], lambda: tk.rotary(r, q, pos, (2,))[0],
            lambda: tk.window_attention(r, q, r, 2), lambda: tk.window_attention(q, r, r, 2),
            lambda: tk.window_attention_cached(r, r, q, n, 2))


@pytest.mark.parametrize("i", range(9))
def test_forward_mode_is_refused(i):
    with torch.autograd.forward_ad.dual_level():
        x, q = (torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)) for t in (torch.randn(2, 8), torch.randn(1, 4, 2, 8)))
        for grad in (torch.enable_grad, torch.no_grad):
            with grad(), pytest.raises(RuntimeError, match="forward-mode"):
                calls(x, q)[i]()


@pytest.mark.parametrize("i", range(9))
def test_tracing_is_refused(i):
    x, q = torch.randn(2, 8), torch.randn(1, 4, 2, 8)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(lambda x, q: calls(x, q)[i](), (x, q))
    for mode in ("real", "fake", "symbolic"):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.fx.experimental.proxy_tensor.make_fx(lambda x, q: calls(x, q)[i](), tracing_mode=mode)(x, q)
    with torch._subclasses.FakeTensorMode(), pytest.raises(RuntimeError, match="cannot be traced"):
        calls(torch.empty(2, 8, device="cuda"), torch.empty(1, 4, 2, 8, device="cuda"))[i]()


class Wrapped(torch.Tensor):
    """A tensor without memory of its own."""

    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_wrapper_subclass(cls, t.shape, dtype=t.dtype, device=t.device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise NotImplementedError


@pytest.mark.parametrize("i", [0, 1, 2, 4, 5, 6, 7, 8])
def test_wrapped_tensors_are_refused(i):
    x, q = torch.randn(2, 8), torch.randn(1, 4, 2, 8)
    with pytest.raises(RuntimeError, match="dense tensors"):
        torch.func.vmap(lambda x, q: calls(x, q)[i]())(x[None], q[None])
    with pytest.raises(RuntimeError, match="dense tensors|forward-mode"):
        torch.func.jvp(lambda x, q: calls(x, q)[i](), (x, q), (x, q))
    with pytest.raises(RuntimeError, match="dense tensors"):
        torch.func.grad(lambda x, q: calls(x, q)[i]().sum(), (0, 1))(x, q)
    with pytest.raises(RuntimeError, match="dense tensors"):
        calls(Wrapped(x), Wrapped(q))[i]()


def test_attention_backward_without_key_gradients():
    # neither dk nor dv: no workspace, which the same call with both has
    n = ctypes.c_int64()
    for over, some in ((dict(), True), (dict(dk=None, dv=None), False)):
        d = attn_desc(B=1, T=4096, M=4096, **over)
        assert LIB.dfcsa_wattn_work_floats(ctypes.addressof(d), 1, ctypes.byref(n)) == 0 and (n.value > 0) == some


@pytest.mark.parametrize("eps", [-1e-6, float("nan"), float("inf")])
def test_norm_eps_refusals(eps):
    assert LIB.dfcsa_rms_fwd(1, 0, 4, 64, P16, P16, P16, eps, P16, P16, P16, None) == EINVAL
    assert LIB.dfcsa_rms_fwd_q8(1, 0, 4, 64, 0, P16, P16, P16, eps, P16, P16, P16, None) == EINVAL
