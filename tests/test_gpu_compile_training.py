"""torch.compile(fullgraph=True) of the rotary and the differentiable attention
entry points: results and gradients are those of the eager calls, bit for bit
(the same kernels on the same inputs)."""
import pytest
import torch

from gpu_util import DEV

gpu = pytest.mark.gpu


def leaf(h, t, d, seed, dtype=torch.bfloat16):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(2, t, h, d, generator=gen, device=DEV).to(dtype).permute(0, 2, 1, 3).requires_grad_()


@gpu
@pytest.mark.parametrize("weights", [True, False])
def test_training_entry_points_in_one_graph(weights):
    import b200_pisa

    torch._dynamo.reset()
    q, k, v = leaf(4, 70, 64, 1), leaf(2, 70, 64, 2), leaf(2, 70, 64, 3)
    w = torch.ones(64, device=DEV, dtype=torch.bfloat16, requires_grad=True) if weights else None
    pos = torch.stack([torch.arange(70, device=DEV) // n for n in (7, 1)], 1)
    lens = torch.tensor([70, 9], dtype=torch.int32, device=DEV)

    def step(q, k, v, w):
        a = b200_pisa.axial_rope(q, pos, (32, 16), theta=(1e4, 1e2), inverse=True)
        q1, k1 = b200_pisa.qk_norm_rope(a, k, w, w, pos, (32, 32), interleaved=False)
        b = b200_pisa.attention(q1, k1, v, causal=True)
        c = b200_pisa.norm_rope_attention(q, k, v, w, w, pos, (32, 32), key_lengths=lens)
        d = b200_pisa.attention(q1[0], k1[0].repeat_interleave(2, 0), v[0].repeat_interleave(2, 0), 0.3)
        return b, c, d

    leaves = [x for x in (q, k, v, w) if x is not None]
    eager = step(q, k, v, w)
    douts = [torch.randn_like(x) for x in eager]
    want = torch.autograd.grad(eager, leaves, douts)
    got = torch.compile(step, fullgraph=True)(q, k, v, w)
    grads = torch.autograd.grad(got, leaves, douts)
    assert all(torch.equal(x, y) and x.stride() == y.stride() for x, y in zip(eager, got))
    # sums of several gradients of one leaf may be fused, in FP32, by the compiler: one rounding of each less
    u = torch.finfo(torch.bfloat16).eps / 2
    for x, y in zip(want, grads):
        assert ((x.double() - y.double()).abs() <= 4 * u * x.double().abs().amax()).all()


@gpu
def test_ops_pass_the_library_checks():
    """Schema, fakes and autograd registration."""
    import b200_pisa  # noqa: F401

    q, k, v = leaf(4, 33, 40, 1), leaf(2, 33, 40, 2), leaf(2, 33, 40, 3)
    w = torch.ones(40, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    pos = torch.arange(33, device=DEV)[:, None]
    tests = ("test_schema", "test_faketensor", "test_autograd_registration")
    ops = torch.ops.b200_pisa
    for op, args in ((ops.axial_rope, (q, pos, (40,), [1e4], True, False)),
                     (ops.qk_norm_rope, (q, k, w, None, pos, (40,), 1e-6, [1e4], True)),
                     (ops.attention, (q, k, v, 0.2, False, None)),
                     (ops.attention, (q[0], q[1], q[1], 0.2, True, None)),
                     (ops.norm_rope_attention, (q, k, v, w, w, pos, (40,), 0.2, 1e-6, [1e4], True, True, None))):
        torch.library.opcheck(op.default, args, test_utils=tests)
