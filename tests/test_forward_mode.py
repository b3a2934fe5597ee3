"""Derivatives that are refused (CPU; before anything that needs a GPU).
Forward-mode ones do not exist for the rotary and the differentiable attention
entry points: a tensor that carries a tangent is refused, in eager calls, under
torch.compile and in a backward pass.  Positions have no gradient."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

NAMES = ("q", "k", "v", "wq", "wk", "pos")


def tensors():
    x = torch.zeros(1, 2, 3, 16, dtype=torch.bfloat16)
    return dict(q=x, k=x.clone(), v=x.clone(), wq=torch.ones(16), wk=torch.ones(16), pos=torch.zeros(3, 2))


def calls():
    import b200_pisa

    axes = (8, 8)
    return {
        "axial_rope": (("q", "pos"), lambda q, pos: b200_pisa.axial_rope(q, pos, axes)),
        "qk_norm_rope": (("q", "k", "wq", "wk", "pos"), lambda *x: b200_pisa.qk_norm_rope(*x, axes)),
        "attention": (("q", "k", "v"), lambda *x: b200_pisa.attention(*x)),
        "attention_forward": (("q", "k", "v"), lambda *x: b200_pisa.attention_forward(*x)),
        "norm_rope_attention": (NAMES, lambda *x: b200_pisa.norm_rope_attention(*x, axes)),
        "qk_norm_rope_backward": (("q", "k", "q", "k", "wq", "wk", "pos"),
                                  lambda *x: b200_pisa.qk_norm_rope_backward(*x, axes)),
        "attention_backward": (("v", "q", "k", "v", "q"),
                               lambda *x: b200_pisa.attention_backward(*x, torch.zeros(1, 2, 3))),
    }


CALLS = list(calls())


@pytest.mark.parametrize("grad", [False, True], ids=["plain", "requires_grad"])
@pytest.mark.parametrize("name", CALLS)
def test_tangents_are_refused(name, grad):
    names, call = calls()[name]
    for dual in dict.fromkeys(names):
        args = tensors()
        if grad:
            args = {n: x.requires_grad_(n != "pos") for n, x in args.items()}
        with forward_ad.dual_level():
            args[dual] = forward_ad.make_dual(args[dual], torch.ones_like(args[dual]))
            with pytest.raises(ValueError, match="forward-mode"):
                call(*(args[n] for n in names))
    with forward_ad.dual_level(), pytest.raises(ValueError, match="one CUDA device"):  # an open level alone is none
        call(*(tensors()[n] for n in names))


@pytest.mark.parametrize("name", CALLS)
def test_functional_jvp_is_refused(name):
    names, call = calls()[name]
    args = tensors()
    primals = tuple(args[n] for n in names)
    with pytest.raises(ValueError, match="forward-mode"):
        torch.func.jvp(call, primals, tuple(torch.ones_like(x) for x in primals))


@pytest.mark.parametrize("name", ["axial_rope", "qk_norm_rope", "attention", "norm_rope_attention"])
@pytest.mark.parametrize("fullgraph", [False, True])
def test_refused_under_compile(name, fullgraph):
    torch._dynamo.reset()
    names, call = calls()[name]
    args = tensors()
    compiled = torch.compile(call, backend="eager", fullgraph=fullgraph)
    with forward_ad.dual_level():
        args["q"] = forward_ad.make_dual(args["q"], torch.ones_like(args["q"]))
        # the graph is left for the eager refusal, or cannot be traced whole
        with pytest.raises(torch._dynamo.exc.Unsupported if fullgraph else ValueError, match="forward-mode"):
            compiled(*(args[n] for n in names))
    torch._dynamo.reset()


@pytest.mark.parametrize("name", ["axial_rope", "attention"])
def test_a_graph_traced_without_tangents_is_not_reused(name):
    torch._dynamo.reset()
    names, call = calls()[name]
    args = tensors()
    compiled = torch.compile(call, backend="eager")
    with pytest.raises(NotImplementedError):  # traced, but nothing here runs on the CPU
        compiled(*(args[n] for n in names))
    with forward_ad.dual_level():
        args["q"] = forward_ad.make_dual(args["q"], torch.ones_like(args["q"]))
        with pytest.raises(ValueError, match="forward-mode"):
            compiled(*(args[n] for n in names))
    torch._dynamo.reset()


@pytest.mark.parametrize("name", ["axial_rope", "qk_norm_rope", "attention", "norm_rope_attention"])
def test_a_gradient_with_a_tangent_is_refused(monkeypatch, name):
    import contextlib

    import b200_pisa
    from b200_pisa import exact, fused, rotary

    class Library:  # runs nothing
        def __getattr__(self, entry):
            return getattr(b200_pisa.LIB, entry) if entry.endswith("_bytes") else lambda *args: 0

    for module in (exact, fused, rotary):
        monkeypatch.setattr(module, "LIB", Library())
        monkeypatch.setattr(module, "on_device", lambda x: contextlib.nullcontext())
        monkeypatch.setattr(module, "raw_stream", lambda x: 0)
        monkeypatch.setattr(module, "require_one_device", lambda *args: None)
    names, call = calls()[name]
    args = tensors()
    out = call(*(args[n].requires_grad_(n != "pos") for n in names))
    out = out[0] if isinstance(out, tuple) else out
    with forward_ad.dual_level(), pytest.raises(ValueError, match="forward-mode"):
        out.backward(forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out)))


@pytest.mark.parametrize("name", ["axial_rope", "qk_norm_rope", "norm_rope_attention"])
@pytest.mark.parametrize("fullgraph", [False, True])
def test_derivatives_of_positions_are_refused_under_compile(name, fullgraph):
    torch._dynamo.reset()
    names, call = calls()[name]
    args = tensors()
    args["pos"].requires_grad_()
    compiled = torch.compile(call, backend="eager", fullgraph=fullgraph)
    with pytest.raises(torch._dynamo.exc.Unsupported if fullgraph else ValueError, match="no gradient"):
        compiled(*(args[n] for n in names))
    torch._dynamo.reset()
