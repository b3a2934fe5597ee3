"""norm_rope_attention: refusals (CPU) and parity with a plain FP64 layer (GPU).

Tolerances, each term at its worst.  The normed and rotated q', k' are held in
FP16 (relative h = 2^-11), so a logit is off by e = scale 2 h |q'||k'|^T and a
probability by P (e + rowsum(P e)); P is rounded to v's type (u) and dS to FP16
(h); the gradients of q', k' stay in FP32 and pass through the norm's linear
backward map; results are rounded once.  The FP32 part is that of the two
operators apart (2^-18 of P, 64 * 2^-24 of the norm's terms)."""
import math

import pytest
import torch

from gpu_util import DEV
from test_attention_gradients import FP32_PART, keep_mask, make
from test_rotary import norm_ref, rotate_ref

gpu = pytest.mark.gpu
H16 = 2.0 ** -11


def rotate_abs(x, positions, axes, theta, interleaved):
    """Upper bound of a rotation of values of magnitudes x: |cos| and |sin|."""
    pos = positions.double()
    pos = pos[None] if pos.ndim == 2 else pos
    angle = torch.cat([pos[..., a, None] * torch.tensor([theta ** (-2.0 * j / d) for j in range(d // 2)],
                                                        dtype=torch.float64, device=x.device)
                       for a, d in enumerate(axes)], dim=-1)[:, None]
    c, s = angle.cos().abs(), angle.sin().abs()
    half = c.shape[-1]
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    ya, yb = a * c + b * s, a * s + b * c
    y = torch.stack((ya, yb), -1).flatten(-2) if interleaved else torch.cat((ya, yb), -1)
    return torch.cat((y, x[..., 2 * half:]), -1)


def check(name, got, want, allowed):
    allowed = allowed * (1 + 2 ** -7) + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps * 64
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), f"{name} is not finite"
    assert (off <= allowed).all(), f"{name} off by {off.max().item():.3g}, {(off / allowed).max().item():.3g} of the allowed"


CASES = [
    # b, h, hk, t, d, axes, dtype, weights, interleaved, causal, lens
    (1, 2, 2, 1, 64, (64,), torch.bfloat16, "same", True, False, None),
    (1, 4, 2, 130, 128, (44, 42, 42), torch.bfloat16, "same", False, False, None),
    (2, 3, 3, 77, 64, (24, 12, 12), torch.bfloat16, "f32", True, True, None),
    (2, 4, 1, 200, 40, (8, 8, 4), torch.float16, "same", False, False, (200, 3)),
    (3, 2, 2, 140, 128, (128,), torch.bfloat16, "f32", True, False, (0, 140, 129)),
    (1, 7, 7, 300, 120, (40, 40, 40), torch.float16, "f32", False, True, None),
    (1, 2, 1, 515, 96, (32, 32, 32), torch.bfloat16, None, False, False, None),
    (1, 3, 3, 65, 8, (2,), torch.bfloat16, "tiny", True, False, None),
    (1, 2, 2, 90, 64, (64,), torch.bfloat16, "large", True, False, None),
]


@gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)).replace("torch.", ""))
def test_layer_and_gradients_match_fp64(case):
    import b200_pisa
    from b200_pisa import _lib

    b, h, hk, t, d, axes, dtype, weights, inter, causal, lens = case
    g = h // hk
    q, k, v = make(b, h, t, d, dtype, "bthd", 1, 2.0), make(b, hk, t, d, dtype, "fused", 2), make(b, hk, t, d, dtype, "bthd", 3)
    dout = make(b, h, t, d, dtype, "bthd", 4)
    pos = torch.stack([torch.arange(t, device=DEV) // (3 * i + 1) for i in range(len(axes))], 1)
    gen = torch.Generator(device=DEV).manual_seed(5)
    wq = wk = None
    if weights:
        wt = torch.float32 if weights == "f32" else dtype
        size = {"tiny": 2.0 ** -40, "large": 2.0 ** 15}.get(weights, 1.0)
        wq, wk = ((1 + 0.3 * torch.randn(d, generator=gen, device=DEV)).to(wt) for _ in range(2))
        wq, wk = (wq * size).to(wt), (wk / size).to(wt)  # logits stay what they are
    lens_t = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=DEV)
    if lens is not None:  # what lies past the keys does not matter, not to the weights' gradients either
        k, v = k.clone(), v.clone()
        for i, n in enumerate(lens):
            k[i, :, n:], v[i, :, n:] = math.nan, math.inf
    scale = d ** -0.5
    leaves = [x.detach().requires_grad_() for x in (q, k, v, wq, wk) if x is not None]
    args = (*leaves, *([None, None] if wq is None else []), pos, axes, scale)
    run = lambda: b200_pisa.norm_rope_attention(*args, eps=1e-5, interleaved=inter, causal=causal, key_lengths=lens_t)  # noqa: E731
    out = run()
    grads = torch.autograd.grad(out, leaves, dout)
    again = torch.autograd.grad(run(), leaves, dout)
    assert all(torch.equal(x, y) for x, y in zip(grads, again))
    _lib.check_status()

    u = torch.finfo(dtype).eps / 2
    wqd, wkd = (None if w is None else w.double() for w in (wq, wk))
    alive = torch.ones(b, 1, t, 1, dtype=torch.bool, device=DEV) if lens is None else (torch.arange(t, device=DEV)[None] < lens_t[:, None])[:, None, :, None]
    kx, vx = (torch.where(alive, x.double(), 0.0) for x in (k, v))
    q1 = rotate_ref(norm_ref(q.double(), wqd, 1e-5), pos, axes, 1e4, inter)
    k1 = rotate_ref(norm_ref(kx, wkd, 1e-5), pos, axes, 1e4, inter)
    wide = lambda x: x.repeat_interleave(g, 1)  # noqa: E731
    fold = lambda x: x.unflatten(1, (hk, g)).sum(2)  # noqa: E731
    keep = keep_mask(t, t, causal, lens_t, b)
    s = (q1 @ wide(k1).transpose(-1, -2) * scale).masked_fill(~keep, -math.inf)
    lse = torch.logsumexp(s, -1, keepdim=True)
    p = torch.where(keep, (s - torch.where(lse == -math.inf, 0.0, lse)).exp(), 0.0)
    e = scale * 2 * H16 * q1.abs() @ wide(k1).abs().transpose(-1, -2)
    slack = p * (e + (p * e).sum(-1, keepdim=True)) + FP32_PART * p
    vw, do = wide(vx), dout.double()
    ref_out = p @ vw
    a_out = (slack + u * p) @ vw.abs() + u * ref_out.abs()
    check("out", out.detach(), ref_out, a_out)
    check("dv", grads[2], fold(p.transpose(-1, -2) @ do), fold((slack + u * p).transpose(-1, -2) @ do.abs()) + u * fold(p.transpose(-1, -2) @ do).abs())
    dp = do @ vw.transpose(-1, -2)
    delta = (do * ref_out).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    a_ds = slack * (do.abs() @ vw.abs().transpose(-1, -2) + delta.abs()) + p * (do.abs() * a_out).sum(-1, keepdim=True) + H16 * ds.abs()
    dq1, dk1 = scale * ds @ wide(k1), fold(scale * ds.transpose(-1, -2) @ q1)
    a_dq1 = scale * (a_ds + H16 * ds.abs()) @ wide(k1).abs()
    a_dk1 = fold(scale * (a_ds + H16 * ds.abs()).transpose(-1, -2) @ q1.abs())
    for i, (x, w, dy, a_dy, gx, name) in enumerate(((q.double(), wqd, dq1, a_dq1, grads[0], "q"),
                                                     (kx, wkd, dk1, a_dk1, grads[1], "k"))):
        dz = rotate_ref(dy, pos, axes, 1e4, inter, inverse=True)
        a_dz = rotate_abs(a_dy, pos, axes, 1e4, inter) + 64 * 2.0 ** -24 * dy.abs().amax(-1, keepdim=True)
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5)
        xh = x * r
        gg, a_g = (dz, a_dz) if w is None else (dz * w, a_dz * w.abs())
        want = r * (gg - xh * (gg * xh).mean(-1, keepdim=True))
        allowed = r * (a_g + xh.abs() * (a_g * xh.abs()).mean(-1, keepdim=True)) + u * want.abs()
        allowed = allowed + 64 * 2.0 ** -24 * r * (gg.abs().amax(-1, keepdim=True) + xh.abs() * (gg * xh).abs().mean(-1, keepdim=True))
        if name == "k":
            want, allowed = torch.where(alive, want, 0.0), torch.where(alive, allowed, 0.0)
        check("d" + name, gx, want, allowed)
        if w is not None:
            dw = (dz * xh).sum((0, 1, 2))
            uw = torch.finfo(grads[3 + i].dtype).eps / 2
            check("dw" + name, grads[3 + i], dw, (a_dz * xh.abs()).sum((0, 1, 2)) + uw * dw.abs() + 288 * 2.0 ** -24 * (dz * xh).abs().sum((0, 1, 2)))


@gpu
def test_it_is_the_two_operators_in_a_row():
    """The same layer by the two calls apart: closer to one another than the
    roundings in between allow, and the composed one closer to FP64."""
    import b200_pisa

    t, d, axes = 400, 128, (44, 42, 42)
    q, k, v = (make(1, h, t, d, torch.bfloat16, "bthd", i) for i, h in ((1, 8), (2, 2), (3, 2)))
    pos = torch.stack([torch.arange(t, device=DEV) // n for n in (100, 10, 1)], 1)
    w = (1 + 0.2 * torch.randn(d, device=DEV)).to(torch.bfloat16)
    dout = make(1, 8, t, d, torch.bfloat16, "bthd", 4)
    leaves = [x.clone().requires_grad_() for x in (q, k, v, w, w)]
    out = b200_pisa.norm_rope_attention(*leaves, pos, axes)
    one = (out.detach(), *torch.autograd.grad(out, leaves, dout))
    q1, k1 = b200_pisa.qk_norm_rope(leaves[0], leaves[1], leaves[3], leaves[4], pos, axes)
    out = b200_pisa.attention(q1, k1, leaves[2])
    two = (out.detach(), *torch.autograd.grad(out, leaves, dout))
    for a, b in zip(one, two):
        # about ten independent roundings of up to 2^-9 apart, root mean square 2^-9 / sqrt(3) each
        assert ((a.double() - b.double()).norm() / b.double().norm()).item() < 2.0 ** -7


@gpu
def test_no_gradients_wanted_saves_nothing_and_replays():
    import b200_pisa

    q, k, v = (make(1, 4, 150, 64, torch.bfloat16, "bthd", i) for i in (1, 2, 3))
    pos = torch.arange(150, device=DEV)[:, None]
    w = torch.ones(64, device=DEV, dtype=torch.bfloat16)
    call = lambda: b200_pisa.norm_rope_attention(q, k, v, w, w, pos, (64,))  # noqa: E731
    eager = call()
    assert not eager.requires_grad
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = call()
    k.mul_(2.0)
    fresh = call()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(fresh, captured)


# ---------------------------------------------------------------- refusals (CPU)
def _x(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("change,match", [
    (dict(q=_x(2, 3, 16)), r"\[B,H,T,D\]"),
    (dict(k=_x(1, 2, 4, 16), v=_x(1, 2, 4, 16)), "share"),
    (dict(k=_x(1, 3, 3, 16), v=_x(1, 3, 3, 16)), "multiple of k/v heads"),
    (dict(q=_x(1, 4, 3, 16, dtype=torch.float32), k=_x(1, 2, 3, 16, dtype=torch.float32), v=_x(1, 2, 3, 16, dtype=torch.float32)), "float16 or bfloat16"),
    (dict(w=torch.ones(8)), r"\[D\]"),
    (dict(pos=torch.zeros(4, 1)), "positions"),
    (dict(axes=(18,)), "axes_dims"),
    (dict(eps=-1.0), "eps"),
    (dict(scale=0.0), "scale"),
    (dict(key_lengths=torch.zeros(2, dtype=torch.int32)), "key_lengths"),
    (dict(), "one CUDA device"),
])
def test_refusals(change, match):
    import b200_pisa

    kw = dict(q=_x(1, 4, 3, 16), k=_x(1, 2, 3, 16), v=_x(1, 2, 3, 16), w=None, pos=torch.zeros(3, 1), axes=(16,), eps=1e-6,
              scale=None, key_lengths=None)
    kw.update(change)
    with pytest.raises(ValueError, match=match):
        b200_pisa.norm_rope_attention(kw["q"], kw["k"], kw["v"], kw["w"], kw["w"], kw["pos"], kw["axes"], kw["scale"],
                                      eps=kw["eps"], key_lengths=kw["key_lengths"])


def test_c_sizes():
    from b200_pisa import _lib

    lib = _lib.LIB
    assert lib.b2_norm_rope_attention_saved_bytes(1, 4, 2, 100, 64) >= 2 * 100 * 64 * (4 + 2)
    assert lib.b2_norm_rope_attention_saved_bytes(1, 4, 2, 100, 136) == -1
    assert lib.b2_norm_rope_attention_workspace_bytes(1, 4, 2, 100, 64) >= 4 * 100 * 64 * (4 + 2)
    assert lib.b2_norm_rope_attention_workspace_bytes(0, 4, 2, 100, 64) == -1


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("power", [60, 57, 30, -50, -75, -85])
def test_gradients_scale_with_dout(d, power):
    """Gradients of dout * 2^n are those of dout times 2^n, whatever power of two FP16 holds dS times in between: exactly
    where it can follow dout's rows.  Below, their squares leave FP32 and dS is held up to 2^10 lower than it could be,
    its small entries as subnormals: results may round to the next BF16 value, 2^-7 of theirs."""
    import b200_pisa

    t, axes = 200, (d,)
    q, k, v = (make(1, h, t, d, torch.bfloat16, "bthd", i) for i, h in ((1, 4), (2, 2), (3, 2)))
    dout = make(1, 4, t, d, torch.bfloat16, "bthd", 4)
    pos = torch.arange(t, device=DEV)[:, None]
    w = torch.ones(d, device=DEV)
    leaves = [x.clone().requires_grad_() for x in (q, k, v, w, w)]
    out = b200_pisa.norm_rope_attention(*leaves, pos, axes)
    want = torch.autograd.grad(out, leaves, dout, retain_graph=True)
    got = torch.autograd.grad(out, leaves, dout * 2.0 ** power)
    for name, a, b in zip(("dq", "dk", "dv", "dwq", "dwk"), want, got):
        a, b = a.double(), b.double() * 2.0 ** -power
        if power > -70:
            assert torch.equal(a, b), name
        else:
            assert ((a - b).norm() <= 2.0 ** -7 * a.norm()).item(), name



@gpu
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("d,dtype,layer", [(64, torch.float16, False), (128, torch.float16, False), (128, torch.bfloat16, True)])
def test_a_dout_row_that_is_not_finite_leaves_the_others(d, dtype, layer, value):
    """Their dq is that beside a row of zeros, bit for bit."""
    import b200_pisa

    q, k, v, dout = (make(1, 3, 150, d, dtype, "bthd", i) for i in range(4))
    dout *= 2.0 ** -12
    pos = torch.arange(150, device=DEV)[:, None]
    grads = []
    for x in (0.0, value):
        dout[0, 1, 77] = 0.0
        dout[0, 1, 77, 5] = x
        leaf = q.clone().requires_grad_()
        out = b200_pisa.norm_rope_attention(leaf, k, v, None, None, pos, (d,)) if layer else b200_pisa.attention(leaf, k, v)
        grads.append(torch.autograd.grad(out, leaf, dout)[0])
    assert not grads[1][0, 1, 77].isfinite().any()
    for g in grads:
        g[0, 1, 77] = 0.0
    assert torch.equal(*grads)
