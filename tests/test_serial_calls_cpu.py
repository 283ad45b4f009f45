"""How the Python entry points of the operators over serialised points (K7 - K9) treat their callers' autograd state and plan their
kernels, on the CPU: the launches are recorded instead of made."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad


@pytest.fixture
def ops(monkeypatch):
    """gfs3d.ops whose launches land in ops.calls as (entry point, arguments); host tensors pass for device tensors."""
    from gfs3d import ops as o
    calls = []
    monkeypatch.setattr(o, "_need_typed", lambda who, first, *rest: first.get_device())
    monkeypatch.setattr(o, "_launch", lambda fn, device, args: calls.append((fn, args)))
    monkeypatch.setattr(o, "calls", calls, raising=False)
    return o


def _inputs(o):
    q, k = torch.randn(2, 5, 4, 64), torch.randn(2, 5, 2, 64)
    freqs, _ = o.rotary_frequencies(32)
    return {"q": q, "k": k, "v": torch.randn_like(k), "lengths": torch.tensor([5, 3], dtype=torch.int32), "freqs": freqs,
            "positions": torch.rand(2, 5), "x": torch.randn(6, 64), "weight": torch.ones(64), "residual": torch.randn(6, 64)}


CALLS = {
    "rotary": (("q", "k", "positions", "freqs"), lambda o, t: o.rotary(t["q"], t["k"], t["positions"], t["freqs"])),
    "rms_norm": (("x", "weight", "residual"), lambda o, t: o.rms_norm(t["x"], t["weight"], residual=t["residual"])),
    "rms_norm_fp8": (("x", "weight", "residual"), lambda o, t: o.rms_norm_fp8(t["x"], t["weight"], residual=t["residual"])),
    "window_attention": (("q", "k", "v"), lambda o, t: o.window_attention(t["q"], t["k"], t["v"], lengths=t["lengths"])),
    "window_attention_step": (("q", "k", "v"), lambda o, t: o.window_attention_step(t["q"], t["k"], t["v"], t["lengths"])),
}


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("who,name", [(w, n) for w, (names, _) in CALLS.items() for n in names])
def test_forward_mode_tangents_are_refused(ops, who, name, grad):
    """A tangent in any floating-point input is refused, whether or not gradients are recorded: no output may come back without it."""
    t = _inputs(ops)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        CALLS[who][1](ops, t)                               # a level alone changes nothing
        t[name] = forward_ad.make_dual(t[name], torch.ones_like(t[name]))
        del ops.calls[:]
        with pytest.raises((RuntimeError, NotImplementedError)):
            CALLS[who][1](ops, t)


@pytest.mark.parametrize("who", ["rotary", "rms_norm", "window_attention"])
def test_forward_mode_tangents_of_gradients_are_refused(ops, who):
    """Forward over reverse: a gradient that carries a tangent enters no backward that would drop it."""
    names, call = CALLS[who]
    t = _inputs(ops)
    t = {n: x.requires_grad_() if n in ("q", "k", "v", "x", "weight", "residual") else x for n, x in t.items()}
    ins = [t[n] for n in names if t[n].requires_grad]
    with forward_ad.dual_level():
        outs = call(ops, t)
        outs = outs if isinstance(outs, tuple) else (outs,)
        plain = [torch.ones_like(o) for o in outs]
        torch.autograd.grad(outs, ins, plain, retain_graph=True)
        for n in range(len(outs)):
            duals = [forward_ad.make_dual(g, torch.ones_like(g)) if m == n else g for m, g in enumerate(plain)]
            with pytest.raises(RuntimeError):
                torch.autograd.grad(outs, ins, duals, retain_graph=True)


def _lib():
    import __graft_entry__  # noqa: F401  (torch first: maps the HIP runtime the library binds to)
    from gfs3d import _lib as m
    return m.lib()


@pytest.mark.parametrize("B,N,H,G,D,left,sinks", [
    (64, 8192, 32, 8, 128, 1024, 512), (2, 65536, 8, 8, 64, 512, 16384), (8192, 512, 8, 8, 8, 8, 4), (2, 65536, 8, 8, 64, 512, 16),
    (32, 2048, 1, 1, 64, 128, 4), (1, 8192, 64, 1, 128, 0, 32), (3, 100000, 6, 2, 40, 100, 1000), (1, 33, 1, 1, 32, 0, 33)])
def test_the_backward_s_workspace_is_bounded_by_its_tensors(B, N, H, G, D, left, sinks):
    """delta; the fp32 sums of the sink keys' dK and dV in whole tiles of 32, in several chunks of rows only while there are fewer than
    2048 of them; and up to eight fp32 dK and dV where fewer than 512 workgroups of 128 keys exist."""
    dp = 32 if D <= 32 else 64 if D <= 64 else 128
    tiles = B * G * ((sinks + 31) // 32)
    floats = B * H * N + 64 + max(tiles, 2048) * 2 * dp * 32
    if B * G * ((N + 127) // 128) < 512:
        floats += 8 * 2 * B * N * G * D
    need = _lib().gfs3d_window_attn_workspace_bytes(B, N, N, H, G, D, left, sinks, 0)
    assert 4 * B * H * N < need <= 4 * floats, (need, 4 * floats)


def _attention_args(L, **kw):
    import ctypes
    from gfs3d import _lib as m
    a = m.WindowAttnArgs()
    a.B, a.N, a.S, a.H, a.G, a.D, a.type, a.scale = 1, 64, 64, 1, 1, 8, m.COMPUTE_BF16, 0.125
    for name in ("q", "k", "v", "out", "lse", "dout", "dq", "dk", "dv", "workspace", "lengths"):
        setattr(a, name, 4096)
    for name in ("q_stride", "k_stride", "v_stride", "dout_stride"):
        setattr(a, name, (ctypes.c_longlong * 3)(8, 8, 8))
    a.workspace_bytes = 2 ** 62
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


@pytest.mark.parametrize("entry,kw", [
    ("forward", dict(N=2 ** 29, S=2 ** 29, H=4)),                                # 2^24 workgroups of 256 threads
    ("backward", dict(N=2 ** 29, S=2 ** 29, H=4)),
    ("backward", dict(B=2 ** 19, N=1024, S=1024, sinks=1024)),                   # dQ and dK / dV fit, the sinks' tiles do not
    ("backward", dict(B=2 ** 24, N=64, S=64, H=1)),
    ("step", dict(B=2 ** 24, N=1, S=64)),
])
def test_calls_of_more_threads_than_a_launch_holds_are_refused_at_once(entry, kw):
    """2^32 threads are refused by their number, before anything is launched (a launch here fails for want of a device)."""
    L = _lib()
    rc = getattr(L, f"gfs3d_window_attn_{entry}")(_attention_args(L, **kw), None)
    assert rc == 1 and b"workgroups" in L.gfs3d_last_error(), (rc, L.gfs3d_last_error())


def test_rotary_refuses_more_threads_than_a_launch_holds():
    import ctypes
    from gfs3d import _lib as m
    L = _lib()
    a = m.RotaryArgs()
    a.B, a.N, a.D, a.type, a.q_heads, a.axes, a.pairs, a.magnitude = 2 ** 14, 2 ** 14, 2, 0, 1, 1, 1, 1.0
    a.q = a.q_out = a.positions = a.freqs = 4096
    assert L.gfs3d_rotary(ctypes.byref(a), None) == 1 and b"too many" in L.gfs3d_last_error(), L.gfs3d_last_error()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_window_attention_keeps_for_a_backward_only_where_one_can_follow(ops, dtype):
    """Statistics and rounding remainders are written where a gradient is recorded, not for leaves under no_grad (an evaluation pass)."""
    q, k, v = (torch.randn(1, 6, 2, 64, dtype=dtype) for _ in range(3))
    kept = lambda: (ops.calls[-1][1].lse is not None, ops.calls[-1][1].out_low is not None)  # noqa: E731
    ops.window_attention(q, k, v)
    assert kept() == (False, False)
    q.requires_grad_()
    assert ops.window_attention(q, k, v).requires_grad and kept() == (True, dtype == torch.bfloat16)
    for off in (torch.no_grad, torch.inference_mode):
        with off():
            out = ops.window_attention(q, k, v)
        assert not out.requires_grad and kept() == (False, False)


def test_the_learner_s_frequencies_stay_in_64_bits():
    """Casts of the module (and of a model that holds it) round its weights, not the angles of its rotary positions."""
    import copy
    from gfs3d import ops as o
    from model.attention import WindowSelfAttention
    want = o.rotary_frequencies(32)[0]
    m = WindowSelfAttention(64, 32, window=8)
    for cast in (lambda x: x.float(), lambda x: x.half(), lambda x: x.to(torch.bfloat16), lambda x: x.double(), lambda x: x.to("cpu"),
                 lambda x: torch.nn.Sequential(x).float()[0], copy.deepcopy):
        m = cast(m)
        assert m.freqs.dtype == torch.float64 and torch.equal(m.freqs, want)
        assert "freqs" not in m.state_dict()


def test_the_learner_refuses_to_have_no_layer():
    """args.att_layers = 0 is refused where the model is built, not in its first forward."""
    import types
    from model.attention import SelfAttention, WindowSelfAttention, attention_learner
    for layers in (0, -1):
        with pytest.raises(ValueError, match="layers"):
            WindowSelfAttention(64, 32, layers=layers)
        with pytest.raises(ValueError, match="layers"):
            attention_learner(types.SimpleNamespace(att_window=16, att_layers=layers), 64, 32)
    assert type(attention_learner(types.SimpleNamespace(att_layers=0), 64, 32)) is SelfAttention
    assert len(attention_learner(types.SimpleNamespace(att_window=16, att_layers=2), 64, 32).qkv_maps) == 2


@pytest.mark.parametrize("length,fast,slow", [(4.0, 32.0, 1.0), (6.0, 32.0, 1.0), (6.5, 32.0, 1.0), (50.0, 40.0, 10.0), (64.0, 32.0, 1.0), (4096.0, 32.0, 1.0),
                                              (1e6, 32.0, 1.0), (1e9, 2.0, 1.0)])
@pytest.mark.parametrize("pairs", [1, 2, 10, 32])
def test_parts_slow_every_pair_that_turns_too_seldom(length, fast, slow, pairs):
    """Pairs that turn at most `slow` times over the original length are slowed by the whole factor, those that turn at least `fast` times
    not at all, also where all of them or none do (short lengths: a room in metres)."""
    import math
    from gfs3d import ops as o
    factor = 4.0
    got, magnitude = o.rotary_frequencies(pairs, scaling="parts", factor=factor, original_length=length, fast=fast, slow=slow)
    plain = o.rotary_frequencies(pairs)[0]
    ratio, turns = plain / got, length * plain / (2 * math.pi)
    assert abs(magnitude - (0.1 * math.log(factor) + 1)) < 1e-15
    assert torch.allclose(ratio[turns <= slow], torch.full((), factor, dtype=torch.float64), rtol=1e-12), (ratio, turns)
    assert torch.allclose(ratio[turns >= fast], torch.ones((), dtype=torch.float64), rtol=1e-12), (ratio, turns)
    assert bool((ratio >= 1 - 1e-12).all()) and bool((ratio <= factor * (1 + 1e-12)).all()) and bool((ratio[1:] >= ratio[:-1] - 1e-12).all())


def test_every_build_of_the_kernels_leaves_packed_fp32_out():
    """The library's flags, and each line of scripts/ that compiles device code or says how, keep packed fp32 instructions out."""
    import pathlib
    from gfs3d import _lib as m
    flag = "-Xclang -target-feature -Xclang -packed-fp32-ops"
    assert flag in " ".join(m.HIPCC_FLAGS)
    root = pathlib.Path(__file__).resolve().parent.parent / "scripts"
    lines = [(f.name, line) for f in sorted(root.rglob("*")) if f.is_file() and f.suffix in (".sh", ".py", ".md", ".hip")
             for line in f.read_text().splitlines() if "--offload-arch" in line]
    assert len(lines) >= 5
    assert not [x for x in lines if flag not in x[1]]


def test_build_compiles_also_where_a_library_is_there(monkeypatch):
    import __graft_entry__
    import gfs3d
    asked = []
    monkeypatch.setattr(gfs3d, "build_library", lambda force=False, verbose=False: asked.append(force) or gfs3d.library_path())
    __graft_entry__.build()
    assert asked == [True]


def test_short_caches_are_split_where_one_workgroup_is_too_few():
    """The step's plan, seen through its workspace: one workgroup per key head only for few small caches; fp32 heads of 128 channels, wide
    16-bit caches and long ones are split; as many short ones as CUs are not."""
    need = _lib().gfs3d_window_attn_workspace_bytes
    f32, bf16 = 1, 2                                          # step: 1 + GFS3D_COMPUTE_*
    assert need(4, 1, 2048, 8, 2, 64, 1023, 4, bf16) == 0 and need(4, 1, 2048, 8, 2, 64, 255, 4, f32) == 0
    assert need(4, 1, 2048, 8, 2, 64, 1023, 4, f32) > 0       # 526 KB a key head
    assert need(1, 1, 2048, 8, 2, 128, 1023, 4, bf16) > 0 and need(4, 1, 2048, 8, 2, 128, 1023, 4, f32) > 0
    assert need(256, 1, 2048, 8, 2, 64, 1023, 4, bf16) == 0
    assert need(64, 1, 8192, 32, 4, 128, 4095, 16, bf16) == need(64, 1, 8192, 32, 4, 128, 4095, 16, f32) > 0     # lengths differ: four to a CU
    for case in ((4, 1, 2048, 8, 2, 64, 1023, 4), (3, 2, 9000, 16, 2, 128, 8191, 40), (1, 5, 600, 8, 1, 32, 500, 7)):
        assert need(*case, f32) >= need(*case, bf16) == need(*case, 3)


@pytest.mark.parametrize("name", ["positions", "freqs"])
def test_rotary_refuses_to_leave_out_the_gradient_of_positions(ops, name):
    """Coordinates that are learnt, or frequencies, would silently miss their share of the gradient: the call says so; detached they pass."""
    t = _inputs(ops)
    t["q"].requires_grad_(), t[name].requires_grad_()
    with pytest.raises(RuntimeError, match="detach"):
        CALLS["rotary"][1](ops, t)
    with torch.no_grad():
        CALLS["rotary"][1](ops, t)
    t[name] = t[name].detach()
    assert CALLS["rotary"][1](ops, t)[0].requires_grad
