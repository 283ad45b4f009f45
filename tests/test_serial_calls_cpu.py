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
