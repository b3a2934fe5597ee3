"""Rotary positions with several axes and the query/key norms with that
rotation: refusals (CPU) and parity with a plain FP64 implementation (GPU).

Tolerances: the kernels compute a row in FP32 and round once.  One rounding is
at most finfo.eps / 2 of the value (half the smallest subnormal below the
normal range); the FP32 part is the angle (a fraction of a turn rounded to
FP32, then sincospif: under 4 * 2^-24), the norm (a D-term sum of squares,
rsqrt, three products) and the rotation: under 32 * 2^-24 of the pair's
magnitude in all, for D <= 256."""
import math

import pytest
import torch

from gpu_util import DEV

gpu = pytest.mark.gpu
U32 = 2.0 ** -24


def rotate_ref(x, positions, axes, theta, interleaved, inverse=False):
    """FP64 rotation by complex multiplication; x [B,H,T,D], positions [T,A] or [B,T,A]."""
    pos = positions.double()
    pos = pos[None] if pos.ndim == 2 else pos
    thetas = theta if isinstance(theta, (tuple, list)) else [theta] * len(axes)
    angle = torch.cat([pos[..., a, None] * torch.tensor([thetas[a] ** (-2.0 * j / d) for j in range(d // 2)],
                                                        dtype=torch.float64, device=x.device)
                       for a, d in enumerate(axes)], dim=-1)[:, None]
    unit = torch.polar(torch.ones_like(angle), -angle if inverse else angle)
    half = unit.shape[-1]
    rot = x[..., : 2 * half]
    if interleaved:
        y = torch.view_as_real(torch.complex(rot[..., 0::2].contiguous(), rot[..., 1::2].contiguous()) * unit).flatten(-2)
    else:
        z = torch.complex(rot[..., :half].contiguous(), rot[..., half:].contiguous()) * unit
        y = torch.cat((z.real, z.imag), dim=-1)
    return torch.cat((y, x[..., 2 * half:]), dim=-1)


def norm_ref(x, w, eps):
    z = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    return z if w is None else z * w


def close(got, want, scale, units=32):
    """Within one rounding of got's type plus ``units`` FP32 units of ``scale``."""
    info = torch.finfo(got.dtype)
    allowed = want.abs() * (info.eps / 2) * (1 + 2 ** -10) + units * U32 * scale + info.smallest_normal * info.eps / 2
    off = (got.double() - want).abs()
    assert (off <= allowed).all(), f"off by {off.max().item():.3g}, {(off / allowed).max().item():.3g} of the allowed"


def pair_scale(z, dims, interleaved):
    """Upper bound of each row's pair magnitudes."""
    return z.abs().amax(-1, keepdim=True) * math.sqrt(2.0)


def make(b, h, t, d, dtype, layout, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    if layout == "bthd":
        return torch.randn(b, t, h, d, generator=gen, device=DEV).to(dtype).permute(0, 2, 1, 3)
    if layout == "bhtd":
        return torch.randn(b, h, t, d, generator=gen, device=DEV).to(dtype)
    if layout == "fused":
        return torch.randn(b, t, 3, h, d, generator=gen, device=DEV).to(dtype)[:, :, 1].permute(0, 2, 1, 3)
    assert layout == "sliced"  # every other token of a wider storage
    return torch.randn(b, 2 * t, h + 1, d + 8, generator=gen, device=DEV).to(dtype)[:, ::2, 1:, 8:].permute(0, 2, 1, 3)


def grid_positions(t, axes, kind, batch=None):
    i = torch.arange(t, device=DEV)
    cols = [i // 35, i // 7 % 5, i % 7, i % 3][:len(axes)] if len(axes) > 1 else [i]
    pos = torch.stack(cols, dim=1)
    if kind == "float":
        pos = pos.float() * 0.37 - 2.5
    elif kind == "double":
        pos = pos.double() * 1.0001 + 1e6
    elif kind == "far":
        pos = (pos + 2_000_003).int()
    if batch:
        pos = torch.stack([pos + n for n in range(batch)])
    return pos


# ---------------------------------------------------------------- refusals (CPU)
def _good():
    return torch.zeros(1, 2, 3, 16, dtype=torch.bfloat16), torch.zeros(3, 2, dtype=torch.int64)


@pytest.mark.parametrize("change,match", [
    (dict(x=torch.zeros(2, 3, 16, dtype=torch.bfloat16)), "non-empty"),
    (dict(x=torch.zeros(1, 2, 0, 16, dtype=torch.bfloat16)), "non-empty"),
    (dict(x=torch.zeros(1, 2, 3, 16, dtype=torch.float64)), "bfloat16, float16 or float32"),
    (dict(x=torch.zeros(1, 2, 3, 12, dtype=torch.float32)), "multiple of 8"),
    (dict(x=torch.zeros(1, 2, 3, 264, dtype=torch.float32)), "256"),
    (dict(x=torch.zeros(1, 2, 3, 20, dtype=torch.bfloat16)[..., 2:18]), "16-byte"),
    (dict(x=torch.zeros(1, 2, 16, 3, dtype=torch.bfloat16).transpose(2, 3)), "contiguous head"),
    (dict(axes=(8, 9)), "axes_dims"),
    (dict(axes=(8, 10)), "axes_dims"),
    (dict(axes=()), "axes_dims"),
    (dict(axes=(2, 2, 2, 2, 2)), "axes_dims"),
    (dict(theta=0.0), "theta"),
    (dict(theta=(1e4,)), "theta"),
    (dict(theta=math.inf), "theta"),
    (dict(positions=torch.zeros(4, 2)), "positions must be"),
    (dict(positions=torch.zeros(2, 3, 2)), "positions must be"),
    (dict(positions=torch.zeros(3, 2, dtype=torch.int16)), "positions must be"),
    (dict(positions=torch.zeros(3, 2, requires_grad=True)), "no gradient"),
    (dict(), "one CUDA device"),
])
def test_axial_rope_refuses(change, match):
    import b200_pisa

    x, pos = _good()
    kw = dict(x=x, positions=pos, axes=(8, 8), theta=1e4, **{})
    kw.update(change)
    with pytest.raises(ValueError, match=match):
        b200_pisa.axial_rope(kw["x"], kw["positions"], kw["axes"], theta=kw["theta"])


@pytest.mark.parametrize("change,match", [
    (dict(k=torch.zeros(1, 2, 4, 16, dtype=torch.bfloat16)), "share"),
    (dict(k=torch.zeros(1, 2, 3, 16, dtype=torch.float16)), "share"),
    (dict(q_weight=torch.ones(8)), r"\[D\]"),
    (dict(q_weight=torch.ones(16, dtype=torch.float64)), r"\[D\]"),
    (dict(q_weight=torch.ones(32)[::2]), "contiguous"),
    (dict(q_weight=torch.ones(16), k_weight=torch.ones(16, dtype=torch.bfloat16)), "one dtype"),
    (dict(eps=-1.0), "eps"),
    (dict(eps=math.nan), "eps"),
    (dict(), "one CUDA device"),
])
def test_qk_norm_rope_refuses(change, match):
    import b200_pisa

    x, pos = _good()
    kw = dict(q=x, k=x.clone(), q_weight=None, k_weight=None, eps=1e-6)
    kw.update(change)
    with pytest.raises(ValueError, match=match):
        b200_pisa.qk_norm_rope(kw["q"], kw["k"], kw["q_weight"], kw["k_weight"], pos, (8, 8), eps=kw["eps"])


def test_non_tensors_are_type_errors():
    import b200_pisa

    x, pos = _good()
    with pytest.raises(TypeError):
        b200_pisa.axial_rope([1.0], pos, (8, 8))
    with pytest.raises(TypeError):
        b200_pisa.axial_rope(x, [[0, 0]] * 3, (8, 8))
    with pytest.raises(TypeError):
        b200_pisa.qk_norm_rope(x, x, 1.0, None, pos, (8, 8))


def test_c_entries_check_their_arguments():
    import ctypes

    from b200_pisa import _lib
    from b200_pisa._args import row_view

    lib = _lib.LIB
    x, pos = _good()
    v = row_view(x)
    rot = _lib.Rotary(pos.data_ptr(), 0, 2, 1, _lib.POS_I64, 2)
    rot.axes_dims[:2], rot.theta[:2] = [8, 8], [1e4, 1e4]
    call = lambda r, a=v, b=v: lib.b2_axial_rope(ctypes.byref(a), ctypes.byref(b), ctypes.byref(r), None)  # noqa: E731
    for field, value in (("positions", None), ("pos_dtype", 4), ("n_axes", 0), ("n_axes", 5)):
        bad = _lib.Rotary.from_buffer_copy(rot)
        setattr(bad, field, value)
        assert call(bad) == _lib.B2_ERR_INVALID, field
    bad = _lib.Rotary.from_buffer_copy(rot)
    bad.axes_dims[1] = 2147483646  # the sum must not wrap
    assert call(bad) == _lib.B2_ERR_INVALID
    bad = _lib.Rotary.from_buffer_copy(rot)
    bad.theta[0] = math.nan
    assert call(bad) == _lib.B2_ERR_INVALID
    other = row_view(torch.zeros(1, 2, 3, 24, dtype=torch.bfloat16))
    assert call(rot, v, other) == _lib.B2_ERR_INVALID
    tiled = row_view(x)
    tiled.order, tiled.grid_h, tiled.grid_w, tiled.tokens = _lib.ORDER_TILED8, 8, 8, 64
    assert call(rot, tiled, tiled) == _lib.B2_ERR_UNSUPPORTED
    assert lib.b2_qk_norm_rope_workspace_bytes(12) == -1 and lib.b2_qk_norm_rope_workspace_bytes(264) == -1
    args = [ctypes.byref(v)] * 6
    assert lib.b2_qk_norm_rope_backward(*args, None, None, _lib.B2_F32, 1e-6, ctypes.byref(rot), x.data_ptr(), None,
                                        None, None) == _lib.B2_ERR_INVALID  # weight gradients need a workspace
    assert b"workspace" in lib.b2_last_error()


# ---------------------------------------------------------------- parity (GPU)
ROPE_CASES = [
    # b, h, t, d, axes, dtype, layout, positions, interleaved
    (1, 1, 1, 8, (8,), torch.bfloat16, "bhtd", "int", True),
    (2, 3, 77, 128, (44, 42, 42), torch.bfloat16, "bthd", "int", True),
    (2, 3, 77, 128, (44, 42, 42), torch.bfloat16, "fused", "batch", False),
    (1, 16, 40, 64, (24, 12, 12), torch.float16, "sliced", "far", False),
    (1, 5, 33, 40, (8, 4, 4), torch.float32, "bthd", "float", False),
    (1, 5, 33, 40, (8, 8, 4), torch.float32, "bthd", "double", False),  # R/2 = 10: pair by pair
    (3, 2, 19, 120, (58, 30, 30), torch.float16, "bhtd", "far", False),  # R = 118
    (3, 2, 19, 120, (40, 40, 38), torch.bfloat16, "bhtd", "far", True),
    (1, 2, 21, 256, (64, 64, 64, 64), torch.bfloat16, "bthd", "double", True),
    (1, 2, 21, 256, (128, 128), torch.float32, "sliced", "float", False),
    (1, 2, 7, 256, (126, 128), torch.float32, "bhtd", "int", False),  # R = 254
    (1, 2, 9, 24, (2,), torch.bfloat16, "bhtd", "int", False),
    (1, 70, 300, 128, (128,), torch.bfloat16, "bthd", "int", False),
]


@gpu
@pytest.mark.parametrize("b,h,t,d,axes,dtype,layout,kind,inter", ROPE_CASES)
@pytest.mark.parametrize("inverse", [False, True])
def test_axial_rope_matches_fp64(b, h, t, d, axes, dtype, layout, kind, inter, inverse):
    import b200_pisa

    x = make(b, h, t, d, dtype, layout, 1)
    pos = grid_positions(t, axes, kind, b if kind == "batch" else None)
    theta = [1e4 / (n + 1) for n in range(len(axes))]
    y = b200_pisa.axial_rope(x, pos, axes, theta=theta, interleaved=inter, inverse=inverse)
    want = rotate_ref(x.double(), pos, axes, theta, inter, inverse)
    close(y, want, pair_scale(x.double(), axes, inter))
    r = sum(axes)
    assert torch.equal(y[..., r:], x[..., r:])  # columns that do not rotate keep their bits
    assert y.permute(0, 2, 1, 3).is_contiguous()


@gpu
@pytest.mark.parametrize("weights", [None, "same", "f32"])
@pytest.mark.parametrize("b,h,t,d,axes,dtype,layout,kind,inter", ROPE_CASES)
def test_qk_norm_rope_and_gradients_match_fp64(b, h, t, d, axes, dtype, layout, kind, inter, weights):
    import b200_pisa

    hk = max(1, h // 2)
    q, k = make(b, h, t, d, dtype, layout, 1), make(b, hk, t, d, dtype, "bthd", 2)
    q = (q * 3).to(dtype)
    pos = grid_positions(t, axes, kind, b if kind == "batch" else None)
    gen = torch.Generator(device=DEV).manual_seed(3)
    wq = wk = None
    if weights:
        wt = torch.float32 if weights == "f32" else dtype
        wq, wk = ((1 + 0.3 * torch.randn(d, generator=gen, device=DEV)).to(wt) for _ in range(2))
    leaves = [x.detach().requires_grad_() for x in (q, k, wq, wk) if x is not None]
    lq, lk, lwq, lwk = leaves if weights else (*leaves, None, None)
    yq, yk = b200_pisa.qk_norm_rope(lq, lk, lwq, lwk, pos, axes, eps=1e-5, interleaved=inter)
    dyq, dyk = make(b, h, t, d, dtype, "bhtd", 4), make(b, hk, t, d, dtype, layout, 5)
    grads = torch.autograd.grad((yq, yk), leaves, (dyq, dyk))
    again = torch.autograd.grad(b200_pisa.qk_norm_rope(lq, lk, lwq, lwk, pos, axes, eps=1e-5, interleaved=inter), leaves,
                                (dyq, dyk))
    assert all(torch.equal(x, y) for x, y in zip(grads, again))  # no order of blocks shows
    for i, (x, w, y, dy) in enumerate(((q, wq, yq, dyq), (k, wk, yk, dyk))):
        xd = x.double()
        wd = None if w is None else w.double()
        z = norm_ref(xd, wd, 1e-5)
        close(y, rotate_ref(z, pos, axes, 1e4, inter), pair_scale(z, axes, inter))
        # the formulas of the gradient, in FP64
        dz = rotate_ref(dy.double(), pos, axes, 1e4, inter, inverse=True)
        r = torch.rsqrt(xd.square().mean(-1, keepdim=True) + 1e-5)
        xh, g = xd * r, dz if wd is None else dz * wd
        dot = (g * xh).mean(-1, keepdim=True)
        # terms g and xh * dot carry the row's largest |g| and |xh|^2 |g|: 64 units of their sum
        close(grads[i], r * (g - xh * dot),
              r * (g.abs().amax(-1, keepdim=True) + xh.abs().amax(-1, keepdim=True) * (g * xh).abs().mean(-1, keepdim=True)) * 2,
              units=64)
        if w is not None:
            terms = dz * xh
            # FP32 sums of at most t*h terms a column over lanes, groups and blocks: chains
            # are shorter than 256 additions at these sizes, on top of a term's own error
            close(grads[2 + i], terms.sum((0, 1, 2)), (terms.abs() + dz.abs().amax(-1, keepdim=True) * xh.abs()).sum((0, 1, 2)),
                  units=256 + 32)


@gpu
def test_gradients_match_differences():
    """FP32 gradients against central differences of the FP64 forward."""
    import b200_pisa

    axes, d, t = (8, 6, 6), 24, 5
    q, k = make(1, 2, t, d, torch.float32, "bhtd", 1), make(1, 1, t, d, torch.float32, "bhtd", 2)
    w = torch.linspace(0.5, 1.5, d, device=DEV)
    pos = grid_positions(t, axes, "int")
    dy = make(1, 2, t, d, torch.float32, "bhtd", 3)
    lq, lw = q.clone().requires_grad_(), w.clone().requires_grad_()
    yq, _ = b200_pisa.qk_norm_rope(lq, k, lw, None, pos, axes, interleaved=False)
    dq, dw = torch.autograd.grad(yq, (lq, lw), dy)
    loss = lambda x, ww: (rotate_ref(norm_ref(x, ww, 1e-6), pos, axes, 1e4, False) * dy.double()).sum().item()  # noqa: E731
    step = 1e-5
    for idx in ((0, 0, 0, 0), (0, 1, 4, 23), (0, 1, 2, 11)):
        e = torch.zeros_like(q, dtype=torch.float64)
        e[idx] = step
        slope = (loss(q.double() + e, w.double()) - loss(q.double() - e, w.double())) / (2 * step)
        assert abs(dq[idx].item() - slope) < 1e-5 * max(1.0, abs(slope))  # FP32 terms and the step^2 error
    e = torch.zeros(d, device=DEV, dtype=torch.float64)
    e[7] = step
    slope = (loss(q.double(), w.double() + e) - loss(q.double(), w.double() - e)) / (2 * step)
    assert abs(dw[7].item() - slope) < 1e-5 * max(1.0, abs(slope))


@gpu
def test_rope_gradient_rotates_back_and_accepts_broadcast_gradients():
    import b200_pisa

    x = make(2, 3, 50, 64, torch.bfloat16, "fused", 1).detach().requires_grad_()
    pos = grid_positions(50, (32, 32), "float")
    y = b200_pisa.axial_rope(x, pos, (32, 32))
    (dx,) = torch.autograd.grad(y.sum(), x)  # the gradient of sum() is one broadcast value
    ones = torch.ones(2, 3, 50, 64, device=DEV, dtype=torch.float64)
    close(dx, rotate_ref(ones, pos, (32, 32), 1e4, True, inverse=True), ones * 2)
    y = b200_pisa.axial_rope(x, pos, (32, 32))
    odd = torch.randn(2, 64, 3, 50, device=DEV).to(torch.bfloat16).permute(0, 2, 3, 1)  # head dimension not contiguous
    (dx,) = torch.autograd.grad(y, x, odd)
    close(dx, rotate_ref(odd.double(), pos, (32, 32), 1e4, True, inverse=True), pair_scale(odd.double(), (32, 32), True))


@gpu
def test_only_some_gradients_wanted_and_broadcast_inputs():
    import b200_pisa

    d, axes = 32, (16, 16)
    w = torch.ones(d, device=DEV).requires_grad_()
    q = make(1, 1, 9, d, torch.float32, "bhtd", 1).expand(2, 4, 9, d)  # one row for all heads, read in place
    k = make(2, 1, 9, d, torch.float32, "bhtd", 2)
    pos = grid_positions(9, axes, "int")
    yq, yk = b200_pisa.qk_norm_rope(q, k, w, None, pos, axes)
    close(yq, rotate_ref(norm_ref(q.double(), None, 1e-6), pos, axes, 1e4, True), pair_scale(norm_ref(q.double(), None, 1e-6), axes, True))
    (dw,) = torch.autograd.grad(yq.sum(), w)  # k's output unused
    dz = rotate_ref(torch.ones_like(q, dtype=torch.float64), pos, axes, 1e4, True, inverse=True)
    terms = dz * norm_ref(q.double(), None, 1e-6)
    close(dw, terms.sum((0, 1, 2)), 2 * terms.abs().sum((0, 1, 2)) + 1, units=288)
    with torch.no_grad():
        assert not b200_pisa.qk_norm_rope(q, k, w, None, pos, axes)[0].requires_grad


@gpu
def test_nonfinite_rows_stay_in_their_rows():
    import b200_pisa

    x = make(1, 2, 8, 64, torch.bfloat16, "bthd", 1).clone()
    x[0, 1, 3, 40] = math.inf  # a column that is not rotated
    x[0, 0, 5, 2] = math.nan
    pos = grid_positions(8, (32,), "int")
    y = b200_pisa.axial_rope(x, pos, (32,))
    assert torch.equal(y[0, 1, 3, 32:], x[0, 1, 3, 32:]) and torch.isfinite(y[0, 1, 3, :32]).all()
    bad = torch.zeros_like(x, dtype=torch.bool)
    bad[0, 0, 5, 2:4] = True  # the NaN's pair
    bad[0, 1, 3, 40] = True
    assert torch.equal(~torch.isfinite(y), bad)


@gpu
def test_streams_graphs_and_repeated_replays():
    import b200_pisa

    axes, t = (44, 42, 42), 200
    q, k = make(1, 4, t, 128, torch.bfloat16, "bthd", 1), make(1, 2, t, 128, torch.bfloat16, "bthd", 2)
    w = (1 + 0.1 * torch.randn(128, device=DEV)).to(torch.bfloat16)
    pos = grid_positions(t, axes, "int")
    call = lambda: (*b200_pisa.qk_norm_rope(q, k, w, w, pos, axes),  # noqa: E731
                    *b200_pisa.qk_norm_rope_backward(q, k, q, k, w, w, pos, axes))
    eager = call()
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        on_side = call()
        with torch.cuda.graph(graph, stream=side):
            captured = call()
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(eager, on_side))
    q.mul_(2)
    pos.add_(5)
    fresh = call()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(fresh, captured))


@gpu
def test_long_rows_pass_32_bit_offsets():
    """A view whose last rows lie past 2^31 elements of its storage."""
    import b200_pisa

    storage = torch.empty(2 ** 31 + 2 ** 20, device=DEV, dtype=torch.bfloat16)
    x = storage.as_strided((1, 2, 4, 64), (0, 2 ** 31 - 64 * 2, 2 ** 17, 1))
    x.copy_(torch.randn(1, 2, 4, 64, device=DEV))
    pos = grid_positions(4, (64,), "int")
    close(b200_pisa.axial_rope(x, pos, (64,)), rotate_ref(x.double(), pos, (64,), 1e4, True), pair_scale(x.double(), (64,), True))


@gpu
def test_eps_zero_with_lanes_and_groups_left_over():
    """Heads that do not fill the groups of a block, and no eps to keep the
    empty lanes' reciprocal root finite."""
    import b200_pisa

    q, k = make(1, 3, 7, 40, torch.float32, "bthd", 1), make(1, 5, 7, 40, torch.float32, "bthd", 2)
    w = torch.ones(40, device=DEV).requires_grad_()
    lq = q.clone().requires_grad_()
    pos = grid_positions(7, (40,), "int")
    yq, yk = b200_pisa.qk_norm_rope(lq, k, w, w, pos, (40,), eps=0.0)
    dq, dw = torch.autograd.grad((yq, yk), (lq, w), (torch.ones_like(yq), torch.ones_like(yk)))
    assert all(torch.isfinite(x).all() for x in (yq, yk, dq, dw))
    z = norm_ref(q.double(), None, 0.0)
    close(yq.detach(), rotate_ref(z, pos, (40,), 1e4, True), pair_scale(z, (40,), True))


@gpu
def test_one_tensor_as_queries_and_keys():
    import b200_pisa

    x = make(1, 4, 33, 64, torch.bfloat16, "bthd", 1).requires_grad_()
    w = torch.ones(64, device=DEV, dtype=torch.bfloat16)
    pos = grid_positions(33, (64,), "int")
    yq, yk = b200_pisa.qk_norm_rope(x, x, w, w, pos, (64,))
    assert torch.equal(yq, yk)
    (dx,) = torch.autograd.grad((yq, yk), x, (torch.ones_like(yq), torch.ones_like(yk)))
    lone = x.detach().clone().requires_grad_()
    zq, _ = b200_pisa.qk_norm_rope(lone, lone.detach(), w, w, pos, (64,))
    (half,) = torch.autograd.grad(zq, lone, torch.ones_like(zq))
    assert torch.equal(dx, half * 2)


@gpu
@pytest.mark.parametrize("size", [1e-17, 1e15])
def test_tiny_and_huge_rows_without_eps(size):
    """r^3 of such rows is out of FP32's range, their gradient is not; the
    sums of squares (1e-34, 1e30) still are in it."""
    import b200_pisa

    x = (make(1, 4, 9, 64, torch.float32, "bthd", 1) * size).requires_grad_()
    dy = make(1, 4, 9, 64, torch.float32, "bthd", 2)
    w = torch.ones(64, device=DEV)
    pos = grid_positions(9, (64,), "int")
    y, _ = b200_pisa.qk_norm_rope(x, x.detach(), w, w, pos, (64,), eps=0.0)
    (dx,) = torch.autograd.grad(y, x, dy)
    leaf = x.detach().double().requires_grad_()
    ref = rotate_ref(norm_ref(leaf, None, 0.0), pos, (64,), 1e4, True)
    (want,) = torch.autograd.grad(ref, leaf, dy.double())
    close(y.detach(), ref.detach(), pair_scale(ref.detach(), (64,), True))
    # dx = r (g - xh mean(g xh)): a hundred roundings of terms as large as r |g|, r |xh| sum|g xh| / 64
    r = leaf.detach().square().mean(-1, keepdim=True).rsqrt()
    g = dy.double().abs().amax(-1, keepdim=True) * 2 ** 0.5
    xh = (leaf.detach() * r).abs()
    assert ((dx.double() - want).abs() <= 128 * 2.0 ** -24 * r * g * (1 + xh * xh.mean(-1, keepdim=True))).all()


@gpu
@pytest.mark.parametrize("h,t,d,axis", [(2, 887, 64, 64), (1, 17, 128, 128), (3, 5, 40, 40), (2, 33, 24, 12)])
def test_weight_gradients_of_ragged_token_tiles(h, t, d, axis):
    """Tokens past the last of a block's tile have no angles: what an earlier
    call left in their place (here NaN, from NaN positions) does not reach the
    sums."""
    import b200_pisa

    x = make(1, h, 20000, d, torch.float32, "bthd", 1)  # the same tiles, on every SM
    w = torch.ones(d, device=DEV)
    dirty = torch.full((20000, 1), math.nan, device=DEV)
    q, k, dq, dk = (make(1, n, t, d, torch.float32, "bthd", i) for i, n in ((1, h), (2, 1), (3, h), (4, 1)))
    pos = grid_positions(t, (axis,), "int")
    for _ in range(3):
        b200_pisa.qk_norm_rope_backward(x, x, x, x, w, w, dirty, (axis,))
        b200_pisa.qk_norm_rope(x, x, w, w, dirty, (axis,))
        got = b200_pisa.qk_norm_rope_backward(dq, dk, q, k, w, w, pos, (axis,))
        assert all(torch.isfinite(g).all() for g in got)
