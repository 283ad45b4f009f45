"""Calls of the operators over serialised points (K7 - K9) at the edges of their plans, on the GPU, against the plain float64 forms
and derived bounds of serial_oracle.py."""
import pytest
import torch

import serial_oracle as O

pytestmark = pytest.mark.gpu


def ops():
    from gfs3d import ops as o
    return o


def rnd(seed, shape, dtype, mul=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * mul).to(dtype).cuda()


def test_backward_of_many_sequences_with_sinks():
    """65536 (sequence, key head) pairs whose sinks receive gradients from many rows: as the forward, the backward takes the call, and
    every copy of a sequence gets the same gradients."""
    B, copies, N, H, G, D = 8, 1024, 64, 64, 8, 8
    base = [rnd(n, (B, N, h, D), torch.bfloat16) for n, h in ((1, H), (2, G), (3, G), (4, H))]
    want = O.attention(*base[:3], 8, 0, 4, None, dout=base[3], dtype=torch.bfloat16)
    q, k, v, g = (t.repeat(copies, 1, 1, 1) for t in base)
    ins = [t.requires_grad_() for t in (q, k, v)]
    out = ops().window_attention(*ins, left=8, right=0, sinks=4)
    grads = torch.autograd.grad(out, ins, g)
    for name, x in zip(("out", "dq", "dk", "dv"), (out.detach(),) + grads):
        x = x.view(copies, B, *x.shape[1:])
        assert torch.equal(x, x[:1].expand_as(x)), name
        O.check(name, x[copies - 1], want[name])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_backward_without_the_rounding_remainder(dtype):
    """The C ABI's form with out_low = NULL: the statistics alone are kept, delta is formed from the rounded output (which the bounds count)."""
    from gfs3d import _lib
    B, N, H, G, D, left, right, sinks = 2, 130, 4, 2, 64, 2, 1, 3
    q, k, v, g = (rnd(20 + n, (B, N, h, D), dtype) for n, h in enumerate((H, G, G, H)))
    a, _, device = ops()._window_args("test", q, k, v, left, right, sinks, None, None)
    ops()._window_inputs(a, q, k, v)
    out, lse = torch.empty_like(q), torch.empty((B, H, N), device="cuda")
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    a.out, a.lse = out.data_ptr(), lse.data_ptr()
    ops()._launch("gfs3d_window_attn_forward", device, a)
    assert torch.equal(out, ops().window_attention(q, k, v, left=left, right=right, sinks=sinks))
    a.dout, a.dq, a.dk, a.dv, a.dout_stride = g.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), g.stride()[:3]
    a.workspace_bytes = _lib.lib().gfs3d_window_attn_workspace_bytes(B, N, N, H, G, D, left, sinks, 0)
    ws = torch.empty(a.workspace_bytes, dtype=torch.uint8, device="cuda")
    a.workspace = ws.data_ptr()
    ops()._launch("gfs3d_window_attn_backward", device, a)
    want = O.attention(q, k, v, left, right, sinks, None, dout=g, dtype=dtype)
    for name, x in zip(("out", "dq", "dk", "dv"), (out, dq, dk, dv)):
        O.check(name, x, want[name])


@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,pairs", [(64, 32), (40, 7), (7, 3)])
def test_rotary_in_place(D, pairs, dtype, layout):
    """The C ABI's outputs may be its inputs: the same values as into tensors of their own, and the inverse turns back."""
    from gfs3d import _lib
    B, N, H, G = 2, 37, 3, 2
    q, k = rnd(30, (B, N, H, D), dtype), rnd(31, (B, N, G, D), dtype)
    pos = torch.arange(N, device="cuda").expand(B, N).contiguous()
    freqs, _ = ops().rotary_frequencies(pairs, device="cuda")
    want = ops().rotary(q, k, pos, freqs, layout="interleaved" if layout else "half")
    p, r = q.clone(), k.clone()
    args = lambda inverse: _lib.RotaryArgs(  # noqa: E731
        B, N, D, ops()._TYPE_IDS[dtype], H, G, p.data_ptr(), r.data_ptr(), p.data_ptr(), r.data_ptr(), p.stride()[:3], r.stride()[:3],
        p.stride()[:3], r.stride()[:3], pos.data_ptr(), 1, 1, pairs, layout, inverse, freqs.data_ptr(), 1.0)
    ops()._launch("gfs3d_rotary", p.get_device(), args(0))
    assert torch.equal(p, want[0]) and torch.equal(r, want[1])
    ops()._launch("gfs3d_rotary", p.get_device(), args(1))
    # two turns of a pair, each a few u32 and one rounding of values no longer than the pair: 2 (u + 12 u32) sqrt 2 of its length
    for a, b in ((p, q), (r, k)):
        a, b = a.cpu().double(), b.cpu().double()
        assert float((a - b).abs().max()) <= 2 * (O.u(dtype) + 12 * O.U32) * 2 ** 0.5 * 2 ** 0.5 * float(b.abs().max())


# B, T, S, H, G, D, left, sinks: either side of what one workgroup takes, for each type (320 KB of keys and values, 256 workgroups)
SHORT = [
    (2, 1, 1300, 8, 2, 64, 1100, 4), (2, 1, 1300, 8, 2, 64, 1200, 4), (2, 1, 1300, 8, 2, 64, 1290, 0), (1, 2, 640, 8, 2, 64, 560, 4),
    (1, 1, 640, 4, 1, 128, 500, 4), (1, 1, 640, 4, 1, 128, 600, 4), (3, 3, 1100, 4, 1, 128, 1023, 33), (1, 1, 90, 4, 1, 128, None, 0),
    (127, 1, 80, 2, 2, 32, 50, 1), (128, 1, 80, 2, 2, 32, 50, 1), (130, 1, 600, 2, 2, 32, 500, 1), (100, 1, 700, 2, 2, 64, None, 3),
    (40, 1, 1500, 2, 2, 16, 1400, 3),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", range(len(SHORT)))
def test_step_at_the_borders_of_its_plan(case, dtype):
    B, T, S, H, G, D, left, sinks = SHORT[case]
    q, k, v = rnd(40, (B, T, H, D), dtype), rnd(41, (B, S, G, D), dtype), rnd(42, (B, S, G, D), dtype)
    lens = [max(0, S - 37 * (b % 40)) for b in range(B)]
    out = ops().window_attention_step(q, k, v, torch.tensor(lens, dtype=torch.int32, device="cuda"), left=left, sinks=sinks)
    O.check(f"{dtype} {SHORT[case]}", out, O.attention(q, k, v, left, 0, sinks, lens, step=True, dtype=dtype)["out"])
