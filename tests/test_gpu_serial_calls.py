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
