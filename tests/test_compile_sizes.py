"""torch.compile of the rotary and the differentiable attention entry points with
sizes that change from call to call: traced with symbolic sizes (CPU, fakes
alone), and one compiled step over several sizes against the eager one (GPU)."""
import random

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from gpu_util import DEV

gpu = pytest.mark.gpu


def inputs(dev, batch, tokens, heads=4, kv_heads=2, dim=64, seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    q, k, v = (torch.randn(batch, tokens, h, dim, generator=gen, device=dev).to(torch.bfloat16).permute(0, 2, 1, 3)
               .requires_grad_() for h in (heads, kv_heads, kv_heads))
    w = torch.ones(dim, device=dev, dtype=torch.bfloat16, requires_grad=True)
    pos = torch.stack([torch.arange(tokens, device=dev) // n for n in (7, 1)], 1)
    lens = torch.full((batch,), tokens, dtype=torch.int32, device=dev)
    lens[-1] = tokens // 2
    return q, k, v, w, pos, lens


def steps():
    import b200_pisa

    axes = (32, 32)
    return {
        "axial_rope": lambda q, k, v, w, pos, lens: b200_pisa.axial_rope(q, pos, axes),
        "qk_norm_rope": lambda q, k, v, w, pos, lens: b200_pisa.qk_norm_rope(q, k, w, w, pos, axes),
        "attention": lambda q, k, v, w, pos, lens: b200_pisa.attention(q, k, v, causal=True, key_lengths=lens),
        "attention, all keys": lambda q, k, v, w, pos, lens: b200_pisa.attention(q, k, v),
        "flat attention": lambda q, k, v, w, pos, lens: b200_pisa.attention(q[:, 0], k[:, 0], v[:, 1]),
        "norm_rope_attention": lambda q, k, v, w, pos, lens: b200_pisa.norm_rope_attention(
            q, k, v, w, w, pos, axes, key_lengths=lens),
        "norm_rope_attention, no weights": lambda q, k, v, w, pos, lens: b200_pisa.norm_rope_attention(
            q, k, v, None, None, pos, axes),
    }


STEPS = list(steps())


@pytest.mark.parametrize("name", STEPS)
def test_symbolic_sizes_trace(monkeypatch, name):
    step = steps()[name]
    monkeypatch.setattr(torch.compiler, "_is_compiling_flag", True)  # what is_compiling() returns

    def with_gradients(*args):
        outs = step(*args)
        outs = outs if isinstance(outs, tuple) else (outs,)
        leaves = [x for x in args[:4] if x.requires_grad]
        return outs, torch.autograd.grad(outs, leaves, [torch.ones_like(x) for x in outs], allow_unused=True)

    args = inputs("cpu", 3, 70)
    graph = make_fx(with_gradients, tracing_mode="symbolic")(*args)
    values = [n.meta["val"] for n in graph.graph.nodes if n.op == "call_function" and "b200_pisa" in str(n.target)]
    assert len(values) == 2  # the operator and its backward pass
    out = values[0][0] if isinstance(values[0], (tuple, list)) else values[0]
    assert any(isinstance(n, torch.SymInt) for n in out.shape)


def test_saved_bytes_by_arithmetic():
    from b200_pisa import fused

    rng = random.Random(3)
    for _ in range(300):
        sizes = rng.randint(1, 9), rng.randint(1, 60), rng.randint(1, 60), rng.randint(1, 40000), 8 * rng.randint(1, 16)
        assert fused.saved_size(*sizes) == fused.saved_bytes(*sizes)[0]


@gpu
@pytest.mark.parametrize("dynamic", [True, None], ids=["dynamic", "automatic"])
@pytest.mark.parametrize("name", STEPS)
def test_one_compiled_step_for_several_sizes(name, dynamic):
    torch._dynamo.reset()
    step = steps()[name]
    compiled = torch.compile(step, fullgraph=True, dynamic=dynamic)
    for seed, (batch, tokens) in enumerate([(2, 70), (2, 90), (3, 333), (2, 40)]):
        args = inputs(DEV, batch, tokens, seed=seed)
        results = []
        for run in (step, compiled):
            outs = run(*args)
            outs = outs if isinstance(outs, tuple) else (outs,)
            gen = torch.Generator(device=DEV).manual_seed(9)
            douts = [torch.randn(x.shape, generator=gen, device=DEV).to(x.dtype) for x in outs]
            grads = torch.autograd.grad(outs, args[:4], douts, allow_unused=True)
            results.append([*outs, *(g for g in grads if g is not None)])
        eager, traced = results
        assert len(eager) == len(traced)
        # the same kernels on the same inputs, and at most two gradients of a leaf (the shared weight) to add
        assert all(torch.equal(a, b) for a, b in zip(eager, traced))
    torch._dynamo.reset()
