"""Refusals of the operators over serialised points (K7 - K9) that need no device: the C ABI's argument checks and workspace plans, the
Python entry points' own checks, and the frequencies of the rotary positions."""
import ctypes
import math

import pytest
import torch

import serial_oracle as O


def _lib():
    import __graft_entry__  # noqa: F401  (torch first: maps the HIP runtime the library binds to)
    from gfs3d import _lib as m
    return m, m.lib()


def _window(m, **kw):
    a = m.WindowAttnArgs()
    a.B, a.N, a.S, a.H, a.G, a.D, a.type = 1, 64, 64, 2, 1, 64, m.COMPUTE_BF16
    a.left, a.right, a.sinks, a.scale = 8, 8, 0, 0.125
    a.q = a.k = a.v = a.out = 4096
    for name in ("q_stride", "k_stride", "v_stride", "dout_stride"):
        setattr(a, name, (ctypes.c_longlong * 3)(8192, 128, 64))
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,text", [
    (dict(type=5), b"type"), (dict(N=0, S=0), b"bad shape"), (dict(H=3, G=2), b"key heads"), (dict(D=60), b"head size"), (dict(D=136), b"head size"),
    (dict(left=-1), b"left"), (dict(sinks=-2), b"sinks"), (dict(scale=0.0), b"scale"), (dict(scale=float("nan")), b"scale"),
    (dict(scale=float("inf")), b"scale"), (dict(q=None), b"NULL"), (dict(k=4100), b"16 bytes"), (dict(out=4104), b"16 bytes"), (dict(S=63), b"differs"),
    (dict(v_stride=(ctypes.c_longlong * 3)(8192, 100, 64)), b"stride"), (dict(q_stride=(ctypes.c_longlong * 3)(8192, -128, 64)), b"stride"),
])
def test_window_attention_refuses(kw, text):
    m, L = _lib()
    a = _window(m, **kw)
    assert L.gfs3d_window_attn_forward(ctypes.byref(a), None) == 1 and text in L.gfs3d_last_error(), L.gfs3d_last_error()


def test_window_attention_refuses_missing_buffers_and_small_workspaces():
    m, L = _lib()
    assert L.gfs3d_window_attn_forward(None, None) == 1 and b"NULL args" in L.gfs3d_last_error()
    a = _window(m)
    assert L.gfs3d_window_attn_backward(ctypes.byref(a), None) == 1 and b"NULL buffer" in L.gfs3d_last_error()
    for name in ("lse", "dout", "dq", "dk", "dv", "workspace"):
        setattr(a, name, 4096)
    a.workspace_bytes = 64
    assert L.gfs3d_window_attn_backward(ctypes.byref(a), None) == 2 and b"workspace" in L.gfs3d_last_error()
    a = _window(m, N=1, S=100000, left=100000)
    assert L.gfs3d_window_attn_step(ctypes.byref(a), None) == 1 and b"lengths" in L.gfs3d_last_error()
    a.lengths = 4096
    need = L.gfs3d_window_attn_workspace_bytes(1, 1, 100000, 2, 1, 64, 100000, 0, 1)
    assert need > 0
    a.workspace, a.workspace_bytes = 4096, need - 1
    assert L.gfs3d_window_attn_step(ctypes.byref(a), None) == 2 and b"workspace" in L.gfs3d_last_error()
    assert L.gfs3d_window_attn_workspace_bytes(1, 0, 64, 2, 1, 64, 8, 0, 0) == 0
    assert L.gfs3d_window_attn_workspace_bytes(1, 64, 64, 2, 1, 64, 8, 8, 0) > L.gfs3d_window_attn_workspace_bytes(1, 64, 64, 2, 1, 64, 8, 0, 0)


def test_rotary_refuses():
    m, L = _lib()

    def args(**kw):
        a = m.RotaryArgs()
        a.B, a.N, a.D, a.type, a.q_heads, a.axes, a.pairs, a.magnitude = 1, 4, 64, 0, 2, 1, 32, 1.0
        a.q = a.q_out = a.positions = a.freqs = 4096
        for k, v in kw.items():
            setattr(a, k, v)
        return a
    assert L.gfs3d_rotary(None, None) == 1 and b"NULL args" in L.gfs3d_last_error()
    for kw, text in ((dict(type=7), b"type"), (dict(N=0), b"bad shape"), (dict(pairs=33), b"do not fit"), (dict(axes=4, pairs=8), b"do not fit"),
                     (dict(pairs=0), b"do not fit"), (dict(D=4096, pairs=1025), b"at most"), (dict(k=4096, k_heads=1), b"NULL"), (dict(k_heads=1), b"NULL"),
                     (dict(freqs=None), b"positions"), (dict(position_type=3), b"positions"),
                     (dict(q_stride=(ctypes.c_longlong * 3)(-1, 128, 64)), b"negative")):
        a = args(**kw)
        assert L.gfs3d_rotary(ctypes.byref(a), None) == 1 and text in L.gfs3d_last_error(), (kw, L.gfs3d_last_error())


def test_rms_norm_refuses():
    m, L = _lib()

    def args(**kw):
        a = m.RmsNormArgs()
        a.rows, a.C, a.type, a.eps = 4, 128, 1, 1e-6
        a.x = a.weight = a.y = 4096
        a.x_stride = 128
        for k, v in kw.items():
            setattr(a, k, v)
        return a
    assert L.gfs3d_rms_norm_forward(None, None) == 1 and b"NULL args" in L.gfs3d_last_error()
    for kw, text in ((dict(type=9), b"type"), (dict(rows=0), b"bad shape"), (dict(C=16385), b"bad shape"), (dict(eps=-1.0), b"eps"),
                     (dict(eps=float("nan")), b"eps"), (dict(weight=None), b"NULL"), (dict(residual=4096), b"NULL"), (dict(fp8=1), b"NULL"),
                     (dict(fp8=1, scale=4096, group=48), b"groups"), (dict(fp8=1, scale=4096, group=128, C=64), b"groups"), (dict(x_stride=-1), b"negative")):
        a = args(**kw)
        assert L.gfs3d_rms_norm_forward(ctypes.byref(a), None) == 1 and text in L.gfs3d_last_error(), (kw, L.gfs3d_last_error())
    a = args()
    assert L.gfs3d_rms_norm_backward(ctypes.byref(a), None) == 1 and b"NULL" in L.gfs3d_last_error()
    a = args(rstd=4096, dy=4096, dweight=4096, workspace=4096, workspace_bytes=10)
    assert L.gfs3d_rms_norm_backward(ctypes.byref(a), None) == 2 and b"workspace" in L.gfs3d_last_error()
    a = args(rstd=4096, dy=4096, dresidual=4096)
    assert L.gfs3d_rms_norm_backward(ctypes.byref(a), None) == 1 and b"dresidual" in L.gfs3d_last_error()


def test_entry_points_refuse_host_tensors():
    from gfs3d import ops
    q = torch.zeros(1, 4, 2, 64)
    f, _ = ops.rotary_frequencies(32)
    for call in (lambda: ops.window_attention(q, q, q), lambda: ops.window_attention_step(q, q, q, torch.ones(1, dtype=torch.int32)),
                 lambda: ops.rotary(q, q, torch.arange(4), f), lambda: ops.rms_norm(q, torch.ones(64)), lambda: ops.rms_norm_fp8(q, torch.ones(64))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_rotary_frequencies_refuse():
    from gfs3d import ops
    for bad in (dict(pairs=0), dict(pairs=4, base=1.0), dict(pairs=4, factor=0.5), dict(pairs=4, scaling="twice"), dict(pairs=4, scaling="parts"),
                dict(pairs=4, scaling="parts", original_length=64, fast=1.0, slow=2.0)):
        with pytest.raises(ValueError):
            ops.rotary_frequencies(**bad)
    f, m = ops.rotary_frequencies(1, scaling="base", factor=8.0)
    assert f.tolist() == [1.0] and m == 1.0


def test_the_oracle_s_gradients_are_those_of_its_forward():
    """The oracle's formulas against float64 automatic differentiation of a dense softmax, windows, sinks, lengths and shared heads included."""
    torch.manual_seed(0)
    B, N, H, G, D = 2, 23, 4, 2, 8
    q, k, v = (torch.randn(B, N, h, D, dtype=torch.float64, requires_grad=True) for h in (H, G, G))
    g = torch.randn(B, N, H, D, dtype=torch.float64)
    lens = [23, 17]
    ok = torch.stack([O.visible(N, N, 0, n, 5, 2, 3) for n in lens])[:, None]
    s = torch.einsum("bihd,bjhd->bhij", q, k.repeat_interleave(2, 2)) / math.sqrt(D)
    p = torch.softmax(s.masked_fill(~ok, -1e300), -1) * ok.any(-1, keepdim=True)
    out = torch.einsum("bhij,bjhd->bihd", p, v.repeat_interleave(2, 2))
    grads = torch.autograd.grad(out, (q, k, v), g)
    want = O.attention(q, k, v, 5, 2, 3, lens, dout=g)
    for name, x in zip(("out", "dq", "dk", "dv"), (out,) + grads):
        assert torch.allclose(want[name][0], x, rtol=1e-10, atol=1e-12), name
    x, w, r = (torch.randn(*s_, dtype=torch.float64, requires_grad=True) for s_ in ((5, 9), (9,), (5, 9)))
    y = (x + r) * ((x + r).square().mean(-1, keepdim=True) + 1e-5).rsqrt() * w
    dy, ds = torch.randn(5, 9, dtype=torch.float64), torch.randn(5, 9, dtype=torch.float64)
    dx, dw = torch.autograd.grad((y, x + r), (x, w), (dy, ds))
    want = O.rms(x, w, 1e-5, r, dy, ds)
    assert torch.allclose(want["dx"][0], dx) and torch.allclose(want["dw"][0], dw) and torch.allclose(want["y"][0], y)
