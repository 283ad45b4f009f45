"""GPU parity of the operators over serialised points (K7 - K9) against plain float64 forms, with derived elementwise bounds."""
import math

import pytest
import torch

import serial_oracle as O

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def ops():
    from gfs3d import ops as o
    return o


def rnd(seed, shape, dtype, mul=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * mul).to(dtype).cuda()


# B, N, H, G, D, left, right, sinks, lengths
ATTEND = [
    (1, 1, 1, 1, 64, None, None, 0, None),
    (2, 33, 2, 1, 32, None, 0, 0, None),
    (1, 64, 1, 1, 64, 0, 0, 0, None),                       # a row sees itself alone
    (2, 130, 4, 2, 64, 7, 3, 0, None),
    (1, 257, 3, 1, 40, 50, 0, 5, None),
    (2, 200, 6, 2, 128, 31, 32, 33, [200, 77]),
    (3, 161, 2, 2, 16, 20, 0, 64, [0, 1, 161]),             # an empty sequence, one of one row
    (1, 300, 5, 5, 8, 64, 64, 1, [299]),
    (2, 96, 8, 1, 96, None, None, 0, [96, 50]),
    (1, 520, 1, 1, 64, 100, 60, 70, None),
    (1, 1100, 2, 1, 48, 33, 0, 3, [1090]),                  # several chunks of sink rows
    (1, 128, 1, 1, 80, 1000, 1000, 200, None),              # everything behind the sequence's ends
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_window_attention_forward_and_gradients(case, dtype):
    B, N, H, G, D, left, right, sinks, lens = ATTEND[case]
    q, k, v = rnd(1, (B, N, H, D), dtype), rnd(2, (B, N, G, D), dtype), rnd(3, (B, N, G, D), dtype)
    g = rnd(4, (B, N, H, D), dtype)
    lengths = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    for t in (q, k, v):
        t.requires_grad_()
    out = ops().window_attention(q, k, v, left=left, right=right, sinks=sinks, lengths=lengths)
    grads = torch.autograd.grad(out, (q, k, v), g)
    want = O.attention(q, k, v, left, right, sinks, lens, dout=g, dtype=dtype)
    for name, x in zip(("out", "dq", "dk", "dv"), (out,) + grads):
        O.check(f"{name} {dtype} {ATTEND[case]}", x, want[name])
    with torch.no_grad():                                   # the form that keeps nothing for a backward
        assert torch.equal(ops().window_attention(q, k, v, left=left, right=right, sinks=sinks, lengths=lengths), out)


@pytest.mark.parametrize("dtype", TYPES)
def test_window_attention_reads_nothing_behind_a_sequence(dtype):
    """NaN and infinities behind the lengths, in every input, change nothing; rows there are zero."""
    B, N, H, G, D = 2, 150, 4, 2, 64
    lens = torch.tensor([90, 150], device="cuda")            # int64 lengths
    base = [rnd(5, (B, N, H, D), dtype), rnd(6, (B, N, G, D), dtype), rnd(7, (B, N, G, D), dtype), rnd(8, (B, N, H, D), dtype)]
    dirty = [t.clone() for t in base]
    for n, t in enumerate(dirty):
        t[0, 90:] = (math.nan, math.inf, -math.inf, math.nan)[n]
    got = []
    for q, k, v, g in (base, dirty):
        q, k, v = (t.clone().requires_grad_() for t in (q, k, v))
        out = ops().window_attention(q, k, v, left=40, right=10, sinks=3, lengths=lens)
        got.append((out.detach(),) + torch.autograd.grad(out, (q, k, v), g))
    for a, b in zip(*got):
        assert torch.equal(a, b)
        assert not a[0, 90:].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_window_attention_large_and_equal_scores(dtype):
    """Scores of +-300 (the maximum moves far between tiles) and rows whose scores are all equal."""
    N, D = 200, 64
    q, k, v = rnd(9, (1, N, 1, D), dtype, 6.0), rnd(10, (1, N, 1, D), dtype, 6.0), rnd(11, (1, N, 1, D), dtype)
    q[0, 100:] = 0
    out = ops().window_attention(q, k, v, left=150, right=0)
    want = O.attention(q, k, v, 150, 0, 0, None, dtype=dtype)
    O.check("out", out, want["out"])
    O.check("mean", out[:, 150:151], (v[:, :151].double().cpu().mean(1, keepdim=True), O.attention(q, k, v, 150, 0, 0, None, dtype=dtype)["out"][1][:, 150:151]))


def test_window_attention_strides_and_copies():
    """Channel slices of one projection, transposed heads, an expanded gradient, an unaligned view (copied), against dense inputs."""
    B, N, H, D = 2, 70, 2, 64
    for dtype in TYPES:
        packed = rnd(12, (B, N, 3, H, D), dtype)
        q, k, v = packed.unbind(2)
        dense = [t.contiguous() for t in (q, k, v)]
        want = ops().window_attention(*dense, left=9, right=9, sinks=2)
        assert torch.equal(ops().window_attention(q, k, v, left=9, right=9, sinks=2), want)
        swapped = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in dense]
        assert torch.equal(ops().window_attention(*swapped, left=9, right=9, sinks=2), want)
        odd = torch.empty(B * N * H * D + 1, dtype=dtype, device="cuda")[1:].view(B, N, H, D)
        odd.copy_(q)
        assert torch.equal(ops().window_attention(odd, k, v, left=9, right=9, sinks=2), want)
        grads = []
        for ins in (dense, swapped):
            ins = [t.detach().requires_grad_() for t in ins]
            out = ops().window_attention(*ins, left=9, right=9, sinks=2)
            grads.append(torch.autograd.grad(out, ins, torch.ones((), dtype=dtype, device="cuda").expand_as(out)))
        assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_window_attention_gradient_against_differences():
    """The directional derivative of sum(w o) in fp32: central differences of step h are off by h^2 f'''/6 and 2 u32 |f| / h."""
    B, N, H, G, D = 1, 90, 2, 1, 32
    q, k, v, w = (rnd(n, (B, N, h, D), torch.float32) for n, h in ((13, H), (14, G), (15, G), (16, H)))
    ins = [t.requires_grad_() for t in (q, k, v)]
    f = lambda *a: float((ops().window_attention(*a, left=20, right=5, sinks=4).double() * w.double()).sum())  # noqa: E731
    grads = torch.autograd.grad(ops().window_attention(*ins, left=20, right=5, sinks=4), ins, w)
    for n in range(3):
        d = rnd(17 + n, ins[n].shape, torch.float32)
        d /= d.norm()
        h = 2.0 ** -6
        with torch.no_grad():
            moved = [[t + s * h * d if m == n else t for m, t in enumerate(ins)] for s in (1, -1)]
            slope = (f(*moved[0]) - f(*moved[1])) / (2 * h)
        at = float((grads[n].double() * d.double()).sum())
        # f is a sum of B N H D weighted means: its rounding noise is about u32 sqrt(B N H D) |w o|, far below the bound; f''' of a
        # softmax along a unit direction is below 8 |w| |v|, here about 8 * 8 * 8
        assert abs(slope - at) <= h * h * 512 / 6 + 1e-3, (n, slope, at)


def test_window_attention_offsets_past_32_bits():
    """A view whose rows and sequences lie more than 2^32 elements into its storage."""
    free = torch.cuda.mem_get_info()[0]
    need = 2 * (2 ** 32 + 2 ** 22)
    if free < 2 * need:
        pytest.skip("needs 17 GB of free memory")
    store = torch.empty(2 ** 32 + 2 ** 22, dtype=torch.bfloat16, device="cuda")
    B, N, H, D = 2, 40, 1, 64
    view = lambda off: torch.as_strided(store, (B, N, H, D), (2 ** 32, 256, 64, 1), off)  # noqa: E731
    q, k, v = (view(off) for off in (0, 64, 128))
    src = [rnd(20 + n, (B, N, H, D), torch.bfloat16) for n in range(3)]
    for t, s in zip((q, k, v), src):
        t.copy_(s)
    out = ops().window_attention(q, k, v, left=8, right=2, sinks=1)
    assert torch.equal(out, ops().window_attention(*src, left=8, right=2, sinks=1))
    lens = torch.tensor([40, 33], dtype=torch.int32, device="cuda")
    assert torch.equal(ops().window_attention_step(q[:, -2:], k, v, lens, left=8, sinks=1),
                       ops().window_attention_step(src[0][:, -2:].contiguous(), src[1], src[2], lens, left=8, sinks=1))


# B, T, S, H, G, D, left, sinks, lengths
STEP = [
    (1, 1, 1, 1, 1, 64, None, 0, [1]),
    (2, 1, 70, 4, 2, 64, 20, 3, [70, 5]),
    (3, 1, 100, 8, 1, 128, None, 0, [0, 64, 100]),           # an empty sequence
    (2, 3, 80, 6, 2, 40, 33, 40, [80, 2]),                    # rows in front of the first position
    (1, 5, 600, 8, 1, 32, 500, 7, [599]),                     # 40 columns: two tiles of them
    (1, 1, 5000, 4, 1, 64, None, 0, [4999]),                  # split over workgroups
    (2, 2, 9000, 16, 2, 128, 8191, 40, [9000, 8500]),
    (1, 1, 3000, 2, 2, 8, 100, 16, [2999]),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(STEP)))
def test_window_attention_step(case, dtype):
    B, T, S, H, G, D, left, sinks, lens = STEP[case]
    q, k, v = rnd(31, (B, T, H, D), dtype), rnd(32, (B, S, G, D), dtype), rnd(33, (B, S, G, D), dtype)
    for b, n in enumerate(lens):                              # what lies behind a sequence, or between sinks and window, is not read
        gone = max(sinks, n - T - left) if left is not None else 0
        for a_, b_ in ((n, S), (sinks, gone)):
            k[b, a_:b_] = math.nan
            v[b, a_:b_] = math.inf
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = ops().window_attention_step(q, k, v, lengths, left=left, sinks=sinks)
    k, v = k.nan_to_num(0, 0, 0), v.nan_to_num(0, 0, 0)
    O.check(f"{dtype} {STEP[case]}", out, O.attention(q, k, v, left, 0, sinks, lens, step=True, dtype=dtype)["out"])


@pytest.mark.parametrize("dtype", TYPES)
def test_step_continues_a_causal_pass(dtype):
    """The cache of a causal pass, then its last rows one at a time and together: the same numbers as the whole pass's, to rounding."""
    B, N, H, G, D = 2, 140, 4, 2, 64
    q, k, v = rnd(34, (B, N, H, D), dtype), rnd(35, (B, N, G, D), dtype), rnd(36, (B, N, G, D), dtype)
    want = O.attention(q, k, v, 30, 0, 2, None, dtype=dtype)["out"]
    whole = ops().window_attention(q, k, v, left=30, right=0, sinks=2)
    O.check("whole", whole, want)
    for n in (1, 2, 31, 140):
        one = ops().window_attention_step(q[:, n - 1:n], k, v, torch.full((B,), n, device="cuda"), left=30, sinks=2)
        O.check(f"row {n}", one, tuple(t[:, n - 1:n] for t in want))
    four = ops().window_attention_step(q[:, -4:], k, v, torch.full((B,), N, device="cuda"), left=30, sinks=2)
    O.check("four", four, tuple(t[:, -4:] for t in want))


ROTARY = [
    # B, N, H, G, D, axes, pairs, layout, positions, far
    (2, 5, 2, 1, 64, 1, 32, "half", torch.int32, 100),
    (1, 1, 8, 2, 64, 1, 32, "interleaved", torch.int64, 10 ** 9),
    (3, 40, 4, 4, 64, 3, 10, "interleaved", torch.float32, 30),
    (2, 17, 1, 2, 128, 2, 16, "half", torch.float32, 5),
    (1, 300, 3, 1, 40, 1, 7, "half", torch.int64, 10 ** 6),       # pairs that do not fill a vector, channels that stay
    (1, 33, 1, 1, 30, 3, 5, "interleaved", torch.int32, 50),
    (1, 9, 2, 2, 7, 1, 3, "interleaved", torch.int32, 50),        # an odd head
    (2, 2000, 2, 2, 16, 1, 8, "half", torch.int64, 10 ** 5),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(ROTARY)))
def test_rotary_forward_and_gradients(case, dtype):
    B, N, H, G, D, axes, P, layout, pt, far = ROTARY[case]
    q, k = rnd(41, (B, N, H, D), dtype).requires_grad_(), rnd(42, (B, N, G, D), dtype).requires_grad_()
    g = torch.Generator().manual_seed(43)
    pos = (torch.rand((B, N) if axes == 1 else (B, N, axes), generator=g, dtype=torch.float64) * 2 * far - far).to(pt).cuda()
    freqs, mag = ops().rotary_frequencies(P, scaling="parts", factor=4.0, original_length=64, device="cuda")
    qr, kr = ops().rotary(q, k, pos, freqs, magnitude=mag, layout=layout)
    gq, gk = rnd(44, q.shape, dtype), rnd(45, k.shape, dtype)
    dq, dk = torch.autograd.grad((qr, kr), (q, k), (gq, gk))
    for name, got, x, sign in (("q", qr, q, 1.0), ("k", kr, k, 1.0), ("dq", dq, gq, -1.0), ("dk", dk, gk, -1.0)):
        O.check(f"{name} {dtype} {ROTARY[case]}", got, O.rotary(x, pos, freqs, mag, layout, sign, dtype))
    alone = ops().rotary(q.detach(), None, pos, freqs, magnitude=mag, layout=layout)
    assert torch.equal(alone, qr)
    dq1, = torch.autograd.grad(ops().rotary(q, k, pos, freqs, magnitude=mag, layout=layout)[0], (q,), gq)
    assert torch.equal(dq1, dq)


def test_rotary_strides_and_broadcast_positions():
    for dtype in TYPES:
        packed = rnd(46, (2, 50, 3, 64), dtype)
        q, k = packed[:, :, :2], packed[:, :, 2:]
        freqs, mag = ops().rotary_frequencies(32, device="cuda")
        pos = torch.arange(50, device="cuda")
        want = ops().rotary(q.contiguous(), k.contiguous(), pos.expand(2, 50).contiguous(), freqs)
        got = ops().rotary(q, k, pos, freqs)
        assert mag == 1.0
        for a, b in zip(got, want):
            assert torch.equal(a, b), (dtype, float((a.double() - b.double()).abs().max()))
        cut = rnd(46, (2, 50, 3, 66), dtype)[..., 1:65]            # not aligned
        # the element-wise form may round half values once (a mixed-precision fma) where the vector form rounds twice: both are held to
        # the value's bound, not to each other
        for y in ops().rotary(cut, cut, pos, freqs):
            O.check("unaligned", y, O.rotary(cut, pos, freqs, 1.0, "half", 1.0, dtype))


@pytest.mark.parametrize("scaling,factor", [(None, 1.0), ("linear", 4.0), ("base", 8.0), ("parts", 4.0)])
def test_rotary_frequencies_turn_as_documented(scaling, factor):
    P, base, length = 32, 10000.0, 4096.0
    f, mag = ops().rotary_frequencies(P, base, scaling, factor, length)
    plain = torch.tensor([base ** (-p / P) for p in range(P)], dtype=torch.float64)
    ratio = plain / f
    if scaling is None:
        assert torch.allclose(ratio, torch.ones_like(ratio), rtol=1e-12)
    elif scaling == "linear":
        assert torch.allclose(ratio, torch.full_like(ratio, factor), rtol=1e-12)
    elif scaling == "base":
        assert abs(float(ratio[0]) - 1) < 1e-12 and abs(float(ratio[-1]) - factor) < 1e-9 and bool((ratio[1:] > ratio[:-1]).all())
    else:
        turns = length * plain / (2 * math.pi)
        assert bool((ratio[turns >= 40] < 1 + 1e-12).all()) and bool((ratio[turns <= 0.75] > factor - 1e-9).all())
        assert abs(mag - (0.1 * math.log(factor) + 1)) < 1e-15


NORM = [(1, 1), (3, 7), (5, 64), (130, 72), (2, 129), (64, 192), (33, 256), (700, 200), (9, 512), (4, 1000), (3, 2048), (2, 4095), (2, 5000), (1, 16384)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["none", "same", "f32"])
@pytest.mark.parametrize("rows,C", NORM)
def test_rms_norm_forward_and_gradients(rows, C, kind, dtype):
    x = rnd(51, (rows, C), dtype).requires_grad_()
    wt = torch.float32 if (rows + C) % 2 else dtype
    w = (1 + 0.2 * rnd(52, (C,), torch.float32)).to(wt).requires_grad_()
    r = None if kind == "none" else rnd(53, (rows, C), dtype if kind == "same" else torch.float32).requires_grad_()
    dy = rnd(54, (rows, C), dtype)
    ds = None if r is None else rnd(55, (rows, C), r.dtype)
    got = ops().rms_norm(x, w, 1e-5, residual=r)
    want = O.rms(x, w, 1e-5, r, dy, ds)
    if r is None:
        O.check("y", got, want["y"])
        dx, dw = torch.autograd.grad(got, (x, w), dy)
    else:
        O.check("y", got[0], want["y"])
        assert torch.equal(got[1].detach().cpu().double(), want["stream"][0])
        dx, dw, dr = torch.autograd.grad(got, (x, w, r), (dy, ds))
        O.check("dr", dr, want["dr"])
    O.check("dx", dx, want["dx"])
    O.check("dw", dw, (want["dw"][0], want["dw"][1] + O.u(wt) * want["dw"][0].abs()))
    with torch.no_grad():
        again = ops().rms_norm(x, w, 1e-5, residual=r)
    for a, b in zip((again,) if r is None else again, (got,) if r is None else got):
        assert torch.equal(a, b)


def test_rms_norm_partial_gradients_and_strides():
    x, w, r = rnd(56, (4, 9, 128), torch.bfloat16).requires_grad_(), torch.ones(128, device="cuda", requires_grad=True), rnd(57, (4, 9, 128), torch.float32).requires_grad_()
    y, s = ops().rms_norm(x, w, residual=r)
    full = torch.autograd.grad((y, s), (x, w, r), (torch.ones_like(y), torch.zeros_like(s)), retain_graph=True)
    only_y = torch.autograd.grad(y, (x, w, r), torch.ones_like(y), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(full, only_y))
    gs = rnd(58, s.shape, torch.float32)
    dx, dw, dr = torch.autograd.grad(s, (x, w, r), gs, allow_unused=True)
    assert torch.equal(dr, gs) and torch.equal(dx, gs.bfloat16()) and (dw is None or not dw.any())
    wide = rnd(59, (12, 300), torch.float16)
    for cut in (wide[:, 3:203], wide[:, 8:208], wide[::2, :200], wide.t()[:12]):
        w16 = torch.ones(cut.shape[1], dtype=torch.float16, device="cuda")
        assert torch.equal(ops().rms_norm(cut, w16), ops().rms_norm(cut.contiguous(), w16))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,C,group", [(1, 8, None), (7, 64, 32), (5, 100, None), (40, 128, 128), (9, 256, 64), (3, 384, 128),
                                          (6, 1024, 128), (2, 4096, 128), (3, 4096, None), (1, 16384, 64), (2, 2056, None)])
def test_rms_norm_fp8(rows, C, group, dtype):
    x, r = rnd(61, (rows, C), dtype, 3.0), rnd(62, (rows, C), dtype)
    w = 1 + 0.2 * rnd(63, (C,), torch.float32)
    if rows > 1:
        x[1], r[1] = 0, 0                                     # a row of zeros
    q, scale, s = ops().rms_norm_fp8(x, w, 1e-6, residual=r, group=group)
    want = O.rms(x, w, 1e-6, r)
    assert q.dtype == torch.float8_e4m3fn and torch.equal(s.cpu().double(), want["stream"][0])
    y = want["y"][0].view(rows, -1, group or C)
    sc = y.abs().amax(-1).clamp_min(1e-12) / 448
    O.check("scale", scale.view(rows, -1), (sc, 56 * O.U32 * sc))
    got = q.float().cpu().double().view_as(y) * scale.cpu().double().view(rows, -1, 1)
    # half a step of e4m3: 2^-4 of the value, 2^-10 scales where it is subnormal
    assert bool(((got - y).abs() <= (2.0 ** -4 + 1e-5) * y.abs() + 2.0 ** -10 * 1.0001 * sc[..., None]).all())
    if rows > 1:
        assert not q[1].float().any() and bool((scale[1] > 0).all())


def test_rms_norm_fp8_keeps_nan():
    x = torch.ones((2, 64), device="cuda")
    x[0, 5] = math.nan
    q, scale = ops().rms_norm_fp8(x, torch.ones(64, device="cuda"), group=32)
    assert bool(scale[0].isnan().all()) and bool(q[0].float().isnan().all()) and bool(q[1].float().isfinite().all())


def _layer(o, h, branch, w, wqkv, pos, freqs, H, G, D, lengths):
    """A pre-norm attention layer as it would be used: residual norm, one projection, rotary positions, window attention."""
    y, h = o.rms_norm(branch, w, residual=h)
    B, N, _ = y.shape
    qkv = (y @ wqkv).view(B, N, H + 2 * G, D)
    q, k = o.rotary(qkv[:, :, :H], qkv[:, :, H:H + G], pos, freqs)
    return h, o.window_attention(q, k, qkv[:, :, H + G:], left=24, right=24, sinks=2, lengths=lengths).reshape(B, N, H * D)


def test_a_layer_of_them_together_and_replayed():
    """The operators in a row: against the float64 forms in fp32, and a training step captured into a graph and replayed with new
    inputs between eager work, equal to the eager step."""
    o = ops()
    B, N, H, G, D = 2, 75, 4, 2, 32
    C = H * D
    freqs, _ = o.rotary_frequencies(D // 2, device="cuda")
    pos = torch.arange(N, device="cuda")
    lengths = torch.tensor([75, 60], dtype=torch.int32, device="cuda")
    new = lambda n: (rnd(70 + n, (B, N, C), torch.float32), rnd(80 + n, (B, N, C), torch.float32))  # noqa: E731
    w, wqkv = (1 + 0.1 * rnd(71, (C,), torch.float32)).requires_grad_(), (rnd(72, (C, (H + 2 * G) * D), torch.float32) / C ** 0.5).requires_grad_()
    h, x = (t.clone() for t in new(0))

    def step():
        s, y = _layer(o, h, x, w, wqkv, pos, freqs, H, G, D, lengths)
        return (s.detach(), y.detach()) + torch.autograd.grad((s + y).square().sum(), (w, wqkv))

    # (no eager graph over w and wqkv may live while a backward through them is captured: torch would make its streams part of the
    # capture, which ends the process)
    with torch.no_grad():
        s, y = _layer(o, h, x, w, wqkv, pos, freqs, H, G, D, lengths)
    rs = O.rms(x, w, 1e-6, h)
    qkv = (rs["y"][0] @ wqkv.detach().cpu().double()).view(B, N, H + 2 * G, D)
    q, k = (O.rotary(t, pos, freqs, 1.0, "half")[0] for t in (qkv[:, :, :H], qkv[:, :, H:H + G]))
    want = O.attention(q, k, qkv[:, :, H + G:], 24, 24, 2, [75, 60])["out"][0].reshape(B, N, C)
    # the projection's fp32 product of C = 128 terms is off by C u32 relative, about 1e-5 of values of a few units
    assert float((y.detach().cpu().double() - want).abs().max()) < 2e-4
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for n in range(4):
        a, b = new(n)
        h.copy_(a), x.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for got, eager in zip(held, step()):
            assert torch.equal(got, eager)


def test_other_streams():
    q, k, v = (rnd(90 + n, (1, 500, 2, 64), torch.bfloat16) for n in range(3))
    lens = torch.tensor([500], dtype=torch.int32, device="cuda")
    want = ops().window_attention(q, k, v, left=60, right=60), ops().window_attention_step(q[:, -1:], k, v, lens)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for st in streams:
        with torch.cuda.stream(st):
            got.append((ops().window_attention(q, k, v, left=60, right=60), ops().window_attention_step(q[:, -1:], k, v, lens)))
    torch.cuda.synchronize()
    for pair in got:
        assert all(torch.equal(a, b) for a, b in zip(pair, want))


def test_window_attention_learner_against_float64():
    """WindowSelfAttention, two layers, against the float64 forms in the curve's order; its gradients against differences."""
    from gfs3d.morton import morton_order
    from model.attention import WindowSelfAttention
    torch.manual_seed(3)
    B, N, C = 2, 150, 64
    m = WindowSelfAttention(C, 32, window=20, sinks=3, layers=2, heads=4, key_heads=2, head_dim=32).cuda()
    with torch.no_grad():
        for n in m.norms:
            n.add_(0.1 * rnd(100, n.shape, torch.float32))
    x, cloud = rnd(101, (B, C, N), torch.float32).requires_grad_(), rnd(102, (B, 9, N), torch.float32)
    out = m(x, cloud)
    order, rank = (t.cpu() for t in morton_order(cloud[:, :3]))
    d = lambda t: t.detach().cpu().double()  # noqa: E731
    stream, branch = d(x).transpose(1, 2).gather(1, order[:, :, None].expand(-1, -1, C)), None
    for norm, qm, om in zip(m.norms, m.qkv_maps, m.out_maps):
        stream = stream if branch is None else stream + branch
        y = O.rms(stream, norm, 1e-6, None)["y"][0]
        qkv = (y @ d(qm.weight).t()).view(B, N, 8, 32)
        q, k = (O.rotary(t, torch.arange(N), m.freqs, 1.0, "half")[0] for t in (qkv[:, :, :4], qkv[:, :, 4:6]))
        branch = O.attention(q, k, qkv[:, :, 6:], 20, 20, 3, None)["out"][0].reshape(B, N, -1) @ d(om.weight).t()
    want = O.rms(stream + branch, m.norms[2], 1e-6, None)["y"][0] @ d(m.head_map.weight).t()
    want = want.gather(1, rank[:, :, None].expand(-1, -1, 32)).transpose(1, 2)
    # five fp32 products of 64 to 128 terms and four norms of values of a few units: 128 u32 = 8e-6 each, relative to their terms' sum
    assert float((d(out) - want).abs().max()) < 2e-4
    w = rnd(103, out.shape, torch.float32)
    leaves = [x] + list(m.parameters())
    grads = torch.autograd.grad(out, leaves, w)
    assert all(bool(g.isfinite().all()) and bool(g.any()) for g in grads)
    for n in (0, 1, 4, 6, len(leaves) - 1):
        t, h = leaves[n], 2.0 ** -7
        dirn = grads[n] / grads[n].norm()                     # the steepest direction: the slope is the gradient's norm
        f = []
        for s in (h, -h):
            with torch.no_grad():
                t.add_(s * dirn)
                f.append(float((m(x, cloud).double() * w.double()).sum()))
                t.sub_(s * dirn)
        slope, at = (f[0] - f[1]) / (2 * h), float(grads[n].double().norm())
        assert abs(slope - at) <= 0.02 * at, (n, slope, at)   # h^2 f''' / 6 of a unit step: below 1e-4 of the slope times the model's curvature


def test_models_take_the_window_attention_learner():
    """args.att_window puts it into both models: training gradients reach its weights, points may be given in any order, and models
    without the option hold the reference's learner."""
    import types
    from model.attention import SelfAttention, WindowSelfAttention
    from model.dgcnn import DGCNNSeg_att
    args = types.SimpleNamespace(edgeconv_widths=[[64, 64]] * 3, dgcnn_mlp_widths=[512, 256], pc_in_dim=9, dgcnn_k=20, base_widths=[128, 64],
                                 output_dim=64, eval_weight=1.2)
    assert type(DGCNNSeg_att(args, 5).att_learner) is SelfAttention
    args.att_window, args.att_layers = 64, 2
    torch.manual_seed(4)
    net = DGCNNSeg_att(args, 5).cuda().train()
    assert type(net.att_learner) is WindowSelfAttention and len(net.att_learner.qkv_maps) == 2
    pc = rnd(104, (2, 9, 512), torch.float32)
    for mode in ("f32", "bf16"):
        with ops().compute(mode):
            net.zero_grad()
            logits = net(pc)
            logits.square().mean().backward()
        assert logits.shape == (2, 5, 512) and bool(logits.isfinite().all())
        assert all(bool(p.grad.isfinite().all()) and bool(p.grad.any()) for p in net.att_learner.parameters())
    net.eval()
    with torch.no_grad():
        perm = torch.randperm(512, generator=torch.Generator().manual_seed(5)).cuda()
        a, b = net.att_learner(pc[:, :1].expand(-1, 256, -1), pc), net.att_learner(pc[:, :1, perm].expand(-1, 256, -1), pc[:, :, perm])
    assert torch.equal(a[:, :, perm], b)                      # random coordinates: no two points on one cell of the curve, or the test's seed is bad


def test_entry_points_refuse():
    o = ops()
    q = rnd(110, (2, 8, 4, 64), torch.bfloat16)
    k = q[:, :, :2]
    f, _ = o.rotary_frequencies(32, device="cuda")
    pos, lens = torch.arange(8, device="cuda"), torch.tensor([8, 8], device="cuda")
    x, w = rnd(111, (4, 96), torch.float16), torch.ones(96, device="cuda")
    for call in (
            lambda: o.window_attention(q, k.float(), k), lambda: o.window_attention(q, k.cpu(), k), lambda: o.window_attention(q, q[:, :, :3], q[:, :, :3]),
            lambda: o.window_attention(q, k[:, :5], k[:, :5]), lambda: o.window_attention(q, k, k[:, :, :1]), lambda: o.window_attention(q.int(), k, k),
            lambda: o.window_attention(q, k, k, left=-1), lambda: o.window_attention(q, k, k, sinks=-1), lambda: o.window_attention(q, k, k, scale=0.0),
            lambda: o.window_attention(q, k, k, scale=float("inf")), lambda: o.window_attention(q, k, k, lengths=lens.float()),
            lambda: o.window_attention(q, k, k, lengths=lens.cpu()), lambda: o.window_attention(q, k, k, lengths=lens[:1]),
            lambda: o.window_attention_step(q, k, k, None), lambda: o.window_attention_step(q.requires_grad_(), k, k, lens),
            lambda: o.rotary(q, k, pos.double(), f), lambda: o.rotary(q, k, pos[:7], f), lambda: o.rotary(q, k, pos.cpu(), f),
            lambda: o.rotary(q, k, pos, f.float()), lambda: o.rotary(q, k, pos.view(1, 8, 1).expand(2, 8, 2).contiguous(), f),
            lambda: o.rotary(q, k.float(), pos, f), lambda: o.rotary(q[0], None, pos, f),
            lambda: o.rms_norm(x, w[:95]), lambda: o.rms_norm(x, w.double()), lambda: o.rms_norm(x, w.bfloat16()), lambda: o.rms_norm(x, w, -1.0),
            lambda: o.rms_norm(x, w, residual=x[:3]), lambda: o.rms_norm(x, w, residual=x.bfloat16()), lambda: o.rms_norm_fp8(x, w, group=64),
            lambda: o.rms_norm_fp8(x, w, group=48), lambda: o.rms_norm_fp8(x, w.clone().requires_grad_())):
        with pytest.raises(RuntimeError):
            call()
    q = q.detach()
    for call in (lambda: o.window_attention(q[..., :60].contiguous(), k[..., :60].contiguous(), k[..., :60].contiguous()),
                 lambda: o.rms_norm(torch.zeros((1, 16392), device="cuda"), torch.ones(16392, device="cuda"))):
        with pytest.raises(NotImplementedError):
            call()
    with pytest.raises(ValueError):
        o.rotary(q, k, pos, f, layout="quarter")
    a = q.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(o.window_attention(a, k, k).sum(), a, create_graph=True)


def test_empty_batches_and_sequences():
    o = ops()
    f, _ = o.rotary_frequencies(32, device="cuda")
    for shape in ((0, 5, 2, 64), (2, 0, 2, 64)):
        q = torch.zeros(shape, device="cuda", requires_grad=True)
        out = o.window_attention(q, q, q)
        assert out.shape == q.shape and torch.autograd.grad(out.sum(), q)[0].shape == q.shape
        assert o.rotary(q.detach(), None, torch.zeros(shape[:2], dtype=torch.int32, device="cuda"), f).shape == q.shape
        x = torch.zeros((*shape[:2], 16), device="cuda", requires_grad=True)
        w = torch.ones(16, device="cuda", requires_grad=True)
        dx, dw = torch.autograd.grad(o.rms_norm(x, w).sum(), (x, w))
        assert dx.shape == x.shape and not dw.any()
    q = torch.ones((2, 1, 2, 64), device="cuda")
    assert not o.window_attention_step(q, q[:, :0], q[:, :0], torch.zeros(2, dtype=torch.int32, device="cuda")).any()


def test_two_captured_steps_share_nothing():
    """Two captured calls with workspaces of their own, replayed in turn and with eager calls between."""
    o = ops()
    lens = [torch.tensor([n], dtype=torch.int32, device="cuda") for n in (9000, 7000)]
    ins = [[rnd(120 + 3 * i, (1, 1, 4, 64), torch.bfloat16), rnd(121 + 3 * i, (1, 9000, 1, 64), torch.bfloat16), rnd(122 + 3 * i, (1, 9000, 1, 64), torch.bfloat16)] for i in range(2)]
    want = [o.window_attention_step(*ins[i], lens[i]) for i in range(2)]
    graphs, outs = [], []
    for i in range(2):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            o.window_attention_step(*ins[i], lens[i])
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(o.window_attention_step(*ins[i], lens[i]))
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
        again = [o.window_attention_step(*ins[i], lens[i]) for i in range(2)]
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], want[i]) and torch.equal(again[i], want[i])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_large_batches_equal_their_parts(D, dtype):
    """A batch large enough for eight-wave workgroups and unsplit key gradients, against two of its sequences alone (four waves, rows of
    dK and dV split): the forward takes the same key tiles in the same order, so it is equal; the sums of the gradients differ in order."""
    o = ops()
    B, N, H, G = 130, 515, 8, 4
    lens = torch.tensor([515 - 7 * (b % 30) for b in range(B)], dtype=torch.int32, device="cuda")
    q, k, v, g = (rnd(140 + n, (B, N, h, D), dtype) for n, h in enumerate((H, G, G, H)))
    for left, right, sinks in ((70, 33, 5), (None, 0, 0)):
        whole = [t.clone().requires_grad_() for t in (q, k, v)]
        out = o.window_attention(*whole, left=left, right=right, sinks=sinks, lengths=lens)
        grads = torch.autograd.grad(out, whole, g)
        for b in (0, 31, 128):
            part = [t[b:b + 2].clone().requires_grad_() for t in (q, k, v)]
            one = o.window_attention(*part, left=left, right=right, sinks=sinks, lengths=lens[b:b + 2])
            assert torch.equal(one, out[b:b + 2])
            want = O.attention(q[b:b + 2], k[b:b + 2], v[b:b + 2], left, right, sinks, lens[b:b + 2].tolist(), dout=g[b:b + 2], dtype=dtype)
            for name, x, y in zip(("dq", "dk", "dv"), torch.autograd.grad(one, part, g[b:b + 2]), grads):
                O.check(f"{name} alone", x, want[name])
                O.check(f"{name} of the batch", y[b:b + 2], want[name])
