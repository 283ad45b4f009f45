"""WindowSelfAttention (K7 - K9 in a layer) and the models that hold it, on the GPU: every gradient element by element against float64
automatic differentiation of the same plain form, in all three arithmetics, and CAPL's two feature paths against each other."""
import copy
import math
import random
import types

import pytest
import torch

import serial_oracle as O

pytestmark = pytest.mark.gpu
SHAPE = dict(window=20, sinks=3, layers=2, heads=4, key_heads=2, head_dim=32)


def ops():
    from gfs3d import ops as o
    return o


def rnd(seed, shape, mul=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * mul).cuda()


def _turn(x, angle):
    a, b = x.chunk(2, -1)
    c, s = torch.cos(angle), torch.sin(angle)
    return torch.cat((a * c - b * s, b * c + a * s), -1)


def _plain(m, params, x, order, rank):
    """The learner's formula in float64 on the host; params in the order of m.parameters()."""
    L, H, G, D = len(m.qkv_maps), m.heads, m.key_heads, m.head_dim
    norms, qkvs, outs, head = params[:L + 1], params[L + 1:2 * L + 1], params[2 * L + 1:3 * L + 1], params[-1]
    B, C, N = x.shape
    pick = lambda t, at: t.gather(1, at[:, :, None].expand(-1, -1, t.shape[2]))  # noqa: E731
    norm = lambda s, w: s * (s.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w  # noqa: E731
    hidden = ~O.visible(N, N, 0, N, m.window, m.window, m.sinks)
    angle = (torch.arange(N, dtype=torch.float64)[:, None] * m.freqs.cpu())[None, :, None]
    stream, branch = pick(x.transpose(1, 2), order), None
    for n in range(L):
        stream = stream if branch is None else stream + branch
        qkv = (norm(stream, norms[n]) @ qkvs[n].t()).view(B, N, H + 2 * G, D)
        q, k = _turn(qkv[:, :, :H], angle), _turn(qkv[:, :, H:H + G], angle).repeat_interleave(H // G, 2)
        s = torch.einsum("bihd,bjhd->bhij", q, k) / math.sqrt(D)
        p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
        branch = torch.einsum("bhij,bjhd->bihd", p, qkv[:, :, H + G:].repeat_interleave(H // G, 2)).reshape(B, N, H * D) @ outs[n].t()
    return pick(norm(stream + branch, norms[L]) @ head.t(), rank).transpose(1, 2)


def _blocks(name, t, m):
    """A gradient in parts that are compared on their own scale: the q, k and v rows of a projection; otherwise the whole."""
    if "qkv_maps" not in name:
        return [(name, t)]
    H, G, D = m.heads, m.key_heads, m.head_dim
    return [(f"{name}.{p}", x) for p, x in zip("qkv", t.split((H * D, G * D, G * D)))]


@pytest.mark.parametrize("mode", ["f32", "bf16", "f16"])
def test_learner_output_and_every_gradient_against_float64(mode):
    """Bounds, per part of a gradient.  fp32, the worst case: about 27 products lie on the way to a gradient, each off by at most 256 u32
    of the sum of its terms' magnitudes, which is about 16 times the product's own size: 27 * 256 * 16 u32 = 6.6e-3 < 2^-7 of the part's
    largest element.  16 bits: each stage stores values rounded to half a step u, in the mean u / sqrt 3 of their size, independent of
    each other; 19 stages in the forward, 57 with the backward's: six deviations are 6 u sqrt(19 / 3) < 16 u, 6 u sqrt(57 / 3) < 32 u, of an
    element and the part's root mean square.  A term left out is off by the size of the elements it belongs to."""
    from gfs3d.morton import morton_order
    from model.attention import WindowSelfAttention
    torch.manual_seed(11)
    B, N, C = 2, 150, 64
    m = WindowSelfAttention(C, 32, **SHAPE).cuda()
    with torch.no_grad():
        for n in m.norms:
            n.add_(0.1 * rnd(200, n.shape))
    x, cloud, w = rnd(201, (B, C, N)).requires_grad_(), rnd(202, (B, 9, N)), rnd(203, (B, 32, N))
    with ops().compute(mode):
        out = m(x, cloud)
        got = torch.autograd.grad(out, [x] + list(m.parameters()), w)
    order, rank = (t.cpu() for t in morton_order(cloud[:, :3]))
    leaves = [t.detach().cpu().double().requires_grad_() for t in [x] + list(m.parameters())]
    ref = _plain(m, leaves[1:], leaves[0], order, rank)
    want = torch.autograd.grad(ref, leaves, w.cpu().double())
    u = {"f32": O.U32, "bf16": O.u(torch.bfloat16), "f16": O.u(torch.float16)}[mode]

    def check(name, a, b, steps):
        a, b = a.detach().cpu().double(), b.detach()
        bound = torch.full_like(b, 2.0 ** -7 * float(b.abs().max())) if mode == "f32" else steps * u * (b.square().mean().sqrt() + b.abs())
        over = (a - b).abs() / bound
        assert bool(a.isfinite().all()) and float(over.max()) <= 1, f"{name}: {float(over.max())} of the bound"

    check("out", out, ref, 16)
    for name, a, b in zip(["x"] + [n for n, _ in m.named_parameters()], got, want):
        for (part, pa), (_, pb) in zip(_blocks(name, a, m), _blocks(name, b, m)):
            check(part, pa, pb, 32)


def _capl():
    from model.attention import WindowSelfAttention
    from model.capl import mpti_net_Point_GeoAsWeight_v2
    a = types.SimpleNamespace(edgeconv_widths=[[64, 64]] * 3, dgcnn_mlp_widths=[512, 256], pc_in_dim=9, dgcnn_k=20, base_widths=[128, 64],
                              output_dim=64, eval_weight=1.2, att_window=40, att_sinks=5, att_layers=2)
    torch.manual_seed(12)
    gp = torch.randn(200, 192, generator=torch.Generator().manual_seed(13)).cuda()
    m = mpti_net_Point_GeoAsWeight_v2(classes=13, criterion=torch.nn.CrossEntropyLoss(ignore_index=255), args=a, base_num=7, gp=gp, energy=0.9).cuda()
    assert type(m.att_learner) is WindowSelfAttention
    return m


def _rel(a, b):
    return float((a - b).abs().max()) / (float(b.abs().max()) + 1e-12)


@pytest.mark.parametrize("want_onehot", [False, True])            # words and fusion as one operator; pack and fusion as one
@pytest.mark.parametrize("training", [True, False])
def test_capl_features_with_the_learner_fused_and_unfused(training, want_onehot, monkeypatch):
    """CAPL's features with args.att_window: point-major on the library's kernels against the form with torch's heads (same backbone), and
    the gradients of the learner, to the bars of the fused heads with the reference's learner (1e-4 and 5e-4 relative)."""
    m = _capl().train(training)
    x, cot = rnd(210, (2, 9, 256)).abs(), rnd(211, (2, 128, 256))
    sd = copy.deepcopy(m.state_dict())
    runs = []
    for fused in (True, False):
        m.load_state_dict(sd)
        monkeypatch.setattr(m, "_heads_fusable", lambda f=fused, orig=type(m)._heads_fusable: f and orig(m))
        with torch.set_grad_enabled(training):
            assert m._heads_fusable() == fused
            feat, semantic, _ = m._features(x, want_semantic=True, want_onehot=want_onehot)
        grads = torch.autograd.grad(feat, list(m.att_learner.parameters()), cot) if training else []
        runs.append([feat.detach(), semantic.detach()] + list(grads))
    assert runs[0][0].shape == (2, 128, 256) and runs[0][1].shape == (2, 192, 256)
    for n, (a, b) in enumerate(zip(*runs)):
        assert bool(a.any()) and _rel(a, b) < (1e-4 if n < 2 else 5e-4), (n, _rel(a, b))


@pytest.mark.parametrize("mode", ["f32", "bf16", "f16"])
def test_capl_steps_with_the_learner(mode):
    """A training step and the reference's testing pass, in all three arithmetics."""
    m = _capl().train()
    x, y = rnd(212, (4, 9, 256)).abs(), torch.randint(0, 8, (4, 256), generator=torch.Generator().manual_seed(214)).cuda()
    with ops().compute(mode):
        random.seed(0)
        pred, loss = m(x, y=y)
        loss.backward()
        assert pred.shape == (4, 256) and bool(loss.isfinite())
        assert all(bool(p.grad.isfinite().all()) and bool(p.grad.any()) for p in m.att_learner.parameters())
        m.eval()
        coding = (torch.rand(13, 200, generator=torch.Generator().manual_seed(215)) > 0.5).float().cuda()
        with torch.no_grad():
            logits, acc, _ = m(x, y=y, gened_proto=m.main_proto.detach().unsqueeze(0), eval_model=True, base_class_coding=coding[:7],
                               novel_class_coding=coding[7:])
    assert logits.shape == (4, 13, 256) and bool(logits.isfinite().all()) and 0 <= float(acc) <= 1
