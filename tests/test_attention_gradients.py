"""Exact attention with gradients: refusals (CPU) and parity of both passes
with a plain FP64 implementation (GPU).

Tolerances.  One rounding of type t is at most u = finfo(t).eps / 2 of a value.
With P the probabilities, the kernels round
  * P once before P V and P^T dO (relative u a term; the row sum is not rounded);
  * dS = P (dP - delta) once before the last two products; delta uses the
    rounded output, off by u |out| |dout| summed over D;
  * every result once.
So, each term at its worst,
  out: u (|P| |V|) + u |out|
  dV:  u (|P|^T |dO|) + u |dV|
  dQ:  scale ((u |dS| + P ddelta) |K|) + u |dQ|, ddelta = u sum |out||dout|
  dK:  scale ((u |dS| + P ddelta)^T |Q|) + u |dK|
plus the FP32 part: S is a D-term FP32 sum, exp2 and the statistics add under
2^-18 relative to P in all for the logits here (|scaled logit| <= 64, whose
product with scale and lse is rounded at 2^-24 of it), which is taken on every
P and dS with |dP| + |delta| in place of |dP - delta|.  FP16: P is held times
2^8, so what falls below FP16's normal range is at most 2^-14 of 2^-8 with a
step of 2^-24 of 2^-8: 2^-33 a key absolute."""
import math

import pytest
import torch

from gpu_util import DEV

gpu = pytest.mark.gpu
FP32_PART = 2.0 ** -18


def make(b, h, t, d, dtype, layout, seed, scale=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    if layout == "bthd":
        return (torch.randn(b, t, h, d, generator=gen, device=DEV) * scale).to(dtype).permute(0, 2, 1, 3)
    if layout == "bhtd":
        return (torch.randn(b, h, t, d, generator=gen, device=DEV) * scale).to(dtype)
    if layout == "fused":
        return (torch.randn(b, t, 3, h, d, generator=gen, device=DEV) * scale).to(dtype)[:, :, 1].permute(0, 2, 1, 3)
    assert layout == "sliced"
    return (torch.randn(b, 2 * t, h + 1, d + 8, generator=gen, device=DEV) * scale).to(dtype)[:, ::2, 1:, 8:].permute(0, 2, 1, 3)


def keep_mask(tq, tk, causal, lens, b):
    keep = torch.ones(b, 1, tq, tk, dtype=torch.bool, device=DEV)
    if causal:
        i = torch.arange(tq, device=DEV)[:, None]
        keep &= torch.arange(tk, device=DEV)[None] <= i + (tk - tq)
    if lens is not None:
        keep &= (torch.arange(tk, device=DEV)[None] < lens[:, None])[:, None, None]
    return keep


def reference(q, k, v, dout, scale, causal, lens):
    """FP64 (out, lse, dq, dk, dv) and the allowed error of each but lse, as
    functions of the rounding unit u (see the module docstring)."""
    b, h, tq, d = q.shape
    hk, tk = k.shape[1], k.shape[2]
    g = h // hk
    keep = keep_mask(tq, tk, causal, lens, b)
    valid = keep.any(2)[:, :, :, None] if lens is None else (torch.arange(tk, device=DEV)[None] < lens[:, None])[:, None, :, None]
    qd = q.double()
    kd, vd = (torch.where(valid, x.double(), 0.0).repeat_interleave(g, 1) for x in (k, v))
    s = (qd @ kd.transpose(-1, -2) * scale).masked_fill(~keep, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(keep, (s - torch.where(lse == -math.inf, 0.0, lse)[..., None]).exp(), 0.0)
    out = p @ vd
    res = {"out": out, "lse": lse}
    fp32 = FP32_PART * p
    allow = {"out": lambda u: (u * p + fp32) @ vd.abs() + u * out.abs()}
    if dout is not None:
        do = dout.double()
        dp = do @ vd.transpose(-1, -2)
        delta = (do * out).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        fold = lambda x: x.unflatten(1, (hk, g)).sum(2)  # noqa: E731
        res.update(dq=scale * ds @ kd, dk=fold(scale * ds.transpose(-1, -2) @ qd), dv=fold(p.transpose(-1, -2) @ do))
        rough = fp32 * (do.abs() @ vd.abs().transpose(-1, -2) + (do * out).abs().sum(-1, keepdim=True))
        # the rounded output delta is made from is itself within allow["out"]
        slip = lambda u: u * ds.abs() + p * (do.abs() * allow["out"](u)).sum(-1, keepdim=True) + rough  # noqa: E731
        allow["dq"] = lambda u: scale * slip(u) @ kd.abs() + u * res["dq"].abs()
        allow["dk"] = lambda u: fold(scale * slip(u).transpose(-1, -2) @ qd.abs()) + u * res["dk"].abs()
        allow["dv"] = lambda u: fold((u * p + fp32).transpose(-1, -2) @ do.abs()) + u * res["dv"].abs()
    return res, allow


def close(name, got, want, allowed):
    u16 = 2.0 ** -33 if got.dtype == torch.float16 else 0.0
    floor = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps / 2 + u16 * 64
    allowed = allowed * (1 + 2 ** -8) + floor  # products of the first-order terms
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), f"{name} is not finite"
    assert (off <= allowed).all(), f"{name} off by {off.max().item():.3g}, {(off / allowed).max().item():.3g} of the allowed"


# ---------------------------------------------------------------- refusals (CPU)
def _x(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("q,k,v,kw,match", [
    (_x(2, 4, 8), _x(1, 2, 4, 8), _x(1, 2, 4, 8), {}, "same rank"),
    (_x(1, 2, 0, 8), _x(1, 2, 4, 8), _x(1, 2, 4, 8), {}, "non-empty"),
    (_x(1, 2, 4, 8), _x(1, 2, 4, 8), _x(1, 2, 5, 8), {}, "matching"),
    (_x(1, 2, 4, 8), _x(2, 2, 4, 8), _x(2, 2, 4, 8), {}, "matching"),
    (_x(1, 2, 4, 8), _x(1, 2, 4, 16), _x(1, 2, 4, 16), {}, "matching"),
    (_x(1, 3, 4, 8), _x(1, 2, 4, 8), _x(1, 2, 4, 8), {}, "multiple of k/v heads"),
    (_x(1, 2, 4, 8, dtype=torch.float32),) * 3 + ({}, "float16 or bfloat16"),
    (_x(1, 2, 4, 8), _x(1, 2, 4, 8, dtype=torch.float16), _x(1, 2, 4, 8), {}, "float16 or bfloat16"),
    (_x(1, 2, 4, 136),) * 3 + ({}, "D <= 128"),
    (_x(1, 2, 4, 12),) * 3 + ({}, "multiple of 8"),
    (_x(1, 2, 4, 8),) * 3 + (dict(scale=0.0), "scale"),
    (_x(1, 2, 4, 8),) * 3 + (dict(scale=math.nan), "scale"),
    (_x(1, 2, 4, 8),) * 3 + (dict(scale=1e300), "scale"),
    (_x(1, 2, 4, 8),) * 3 + (dict(key_lengths=torch.zeros(2, dtype=torch.int32)), "key_lengths"),
    (_x(1, 2, 4, 8),) * 3 + (dict(key_lengths=torch.zeros(1, dtype=torch.int64)), "key_lengths"),
    (_x(1, 2, 4, 20)[..., 2:10],) * 3 + ({}, "16-byte"),
    (_x(1, 2, 8, 8).transpose(2, 3),) * 3 + ({}, "contiguous head"),
    (_x(1, 2, 4, 8),) * 3 + ({}, "one CUDA device"),
])
def test_attention_refuses(q, k, v, kw, match):
    import b200_pisa

    with pytest.raises(ValueError, match=match):
        b200_pisa.attention(q, k, v, **kw)
    with pytest.raises(ValueError, match=match):
        b200_pisa.attention_forward(q, k, v, **kw)


@pytest.mark.parametrize("change,match", [
    (dict(dout=_x(1, 2, 5, 8)), "dout"),
    (dict(out=_x(1, 2, 4, 8, dtype=torch.float16)), "out"),
    (dict(lse=torch.zeros(1, 2, 5)), "lse"),
    (dict(lse=torch.zeros(1, 2, 4, dtype=torch.float64)), "lse"),
    (dict(lse=None), "lse"),
    (dict(), "one CUDA device"),
])
def test_attention_backward_refuses(change, match):
    import b200_pisa

    x = _x(1, 2, 4, 8)
    kw = dict(dout=x, out=x, lse=torch.zeros(1, 2, 4))
    kw.update(change)
    with pytest.raises(ValueError, match=match):
        b200_pisa.attention_backward(kw["dout"], x, x, x, kw["out"], kw["lse"])


def test_c_entries_check_their_arguments():
    import ctypes

    from b200_pisa import _lib
    from b200_pisa._args import row_view

    lib = _lib.LIB
    x, kv = _x(1, 4, 8, 64), _x(1, 2, 8, 64)
    q, k = row_view(x), row_view(kv)
    fake = ctypes.c_void_p(256)

    def forward(q=q, k=k, v=k, out=q, scale=0.1, lens=None):
        return lib.b2_attention_forward(*(ctypes.byref(a) for a in (q, k, v, out)), scale, 0, lens, None, None, None)

    def backward(dq=q, dk=k, lse=fake, ws=fake):
        args = [ctypes.byref(a) for a in (q, k, k, q)]
        return lib.b2_attention_backward(*args, None, ctypes.byref(q), lse, ctypes.byref(dq), ctypes.byref(dk), ctypes.byref(k), 0.1, 0, None,
                                         ws, None)

    def changed(view, **fields):
        new = _lib.View.from_buffer_copy(view)
        for name, value in fields.items():
            setattr(new, name, value)
        return new

    invalid, unsupported = _lib.B2_ERR_INVALID, _lib.B2_ERR_UNSUPPORTED
    assert forward(scale=0.0) == invalid and forward(scale=math.inf) == invalid
    assert forward(lens=ctypes.c_void_p(2)) == invalid
    assert forward(k=changed(k, heads=3), v=changed(k, heads=3)) == invalid
    assert forward(q=changed(q, stride_h=0)) == invalid  # broadcast rows
    assert forward(out=changed(q, stride_t=-64)) == invalid
    assert forward(q=changed(q, order=_lib.ORDER_TILED8, grid_h=8, grid_w=8, tokens=64)) == unsupported
    assert forward(*(changed(a, dtype=_lib.B2_F32) for a in (q, k, k, q))) == unsupported
    wide = dict(head_dim=136, stride_t=136)
    assert forward(*(changed(a, **wide) for a in (q, k, k, q))) == unsupported
    many = dict(batch=1 << 10, heads=1 << 10, tokens=1 << 20, stride_b=64)  # more tiles than a launch has blocks
    assert forward(*(changed(a, **many) for a in (q, k, k, q))) == unsupported
    assert backward(lse=None) == invalid and backward(ws=None) == invalid and backward(ws=ctypes.c_void_p(8)) == invalid
    assert backward(dk=q) == invalid and backward(dq=changed(q, stride_t=0)) == invalid
    assert lib.b2_attention_backward_workspace_bytes(0, 1, 1, 1, 1) == -1
    assert lib.b2_attention_backward_workspace_bytes(2, 4, 2, 129, 5) >= 2 * 4 * 2 * 1024


# ---------------------------------------------------------------- parity (GPU)
CASES = [
    # b, h, hk, tq, tk, d, dtype, causal, lens, layout
    (1, 1, 1, 128, 128, 64, torch.bfloat16, False, None, "bhtd"),
    (1, 1, 1, 128, 128, 128, torch.bfloat16, False, None, "bhtd"),
    (1, 2, 2, 1, 1, 64, torch.bfloat16, False, None, "bthd"),
    (1, 2, 1, 1, 300, 128, torch.float16, False, None, "bthd"),
    (2, 2, 2, 300, 1, 40, torch.bfloat16, False, None, "fused"),
    (1, 4, 2, 257, 129, 128, torch.float16, False, None, "sliced"),
    (2, 3, 3, 65, 127, 8, torch.bfloat16, False, None, "bthd"),
    (1, 7, 1, 200, 333, 72, torch.float16, False, None, "bthd"),
    (3, 4, 4, 130, 260, 128, torch.bfloat16, False, (260, 0, 131), "bthd"),
    (3, 4, 2, 130, 260, 64, torch.float16, False, (1, 128, 129), "fused"),
    (2, 2, 2, 100, 64, 96, torch.bfloat16, False, (-5, 1000), "bhtd"),
    (1, 2, 2, 385, 385, 128, torch.bfloat16, True, None, "bthd"),
    (1, 4, 1, 513, 513, 64, torch.float16, True, None, "fused"),
    (1, 2, 2, 100, 400, 128, torch.bfloat16, True, None, "bthd"),
    (1, 2, 2, 1, 400, 128, torch.bfloat16, True, None, "bthd"),
    (2, 2, 1, 400, 100, 128, torch.bfloat16, True, None, "bthd"),  # the first 300 queries see nothing
    (2, 2, 1, 260, 260, 120, torch.float16, True, (200, 30), "sliced"),
    (1, 2, 2, 1030, 2050, 128, torch.bfloat16, False, None, "bthd"),
    (1, 2, 2, 2050, 1030, 48, torch.float16, False, None, "bthd"),
]


def run_case(b, h, hk, tq, tk, d, dtype, causal, lens, layout, seed=0, spread=1.0):
    import b200_pisa
    from b200_pisa import _lib

    q = make(b, h, tq, d, dtype, layout, seed + 1, spread)
    k, v = (make(b, hk, tk, d, dtype, layout, seed + i, spread if i == 2 else 1.0) for i in (2, 3))
    dout = make(b, h, tq, d, dtype, "bthd", seed + 4)
    lens_t = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=DEV)
    if lens is not None:  # what lies past the keys does not matter
        k, v = k.clone(), v.clone()
        for i, n in enumerate(lens):
            k[i, :, max(n, 0):], v[i, :, max(n, 0):] = math.nan, math.inf
    out, lse = b200_pisa.attention_forward(q, k, v, causal=causal, key_lengths=lens_t)
    grads = b200_pisa.attention_backward(dout, q, k, v, out, lse, causal=causal, key_lengths=lens_t)
    again = b200_pisa.attention_backward(dout, q, k, v, out, lse, causal=causal, key_lengths=lens_t)
    _lib.check_status()  # no pipeline wait ran out
    assert all(torch.equal(x, y) for x, y in zip(grads, again))
    clamped = None if lens is None else lens_t.clamp(0, tk)
    res, allow = reference(q, k, v, dout, d ** -0.5, causal, clamped)
    u = torch.finfo(dtype).eps / 2
    empty = res["lse"] == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    # sums of up to Tk FP32 terms, exp2, log2: 2^-18 of the sum
    assert ((lse.double() - res["lse"])[~empty].abs() <= FP32_PART * (1 + res["lse"][~empty].abs())).all()
    for name, got in (("out", out), ("dq", grads[0]), ("dk", grads[1]), ("dv", grads[2])):
        close(name, got, res[name], allow[name](u))
    assert (out[empty] == 0).all() and (grads[0][empty] == 0).all()
    if lens is not None:
        for i, n in enumerate(lens):
            assert (grads[1][i, :, max(n, 0):] == 0).all() and (grads[2][i, :, max(n, 0):] == 0).all()


@gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)).replace("torch.", ""))
def test_forward_and_backward_match_fp64(case):
    run_case(*case)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_peaked_rows(dtype):
    """Logits spread by 3 * 3: most of a row's weight on few keys."""
    run_case(1, 2, 2, 300, 500, 128, dtype, False, None, "bthd", seed=10, spread=3.0 ** 0.5)


# ---------------------------------------------------------------- calls no plain case makes (GPU)
def plain_grads(q, k, v, dout, scale, causal=False):
    res, allow = reference(q, k, v, dout, scale, causal, None)
    return res, allow


def check_all(got, res, allow, dtype, names=("out", "dq", "dk", "dv")):
    u = torch.finfo(dtype).eps / 2
    for name, x in zip(names, got):
        close(name, x, res[name], allow[name](u))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_autograd_broadcast_inputs_and_gradients(dtype):
    """Expanded keys and values (one head for all), and the gradient of sum(),
    which is one broadcast value."""
    import b200_pisa

    q = make(2, 4, 70, 64, dtype, "bthd", 1).requires_grad_()
    k1, v1 = (make(2, 1, 90, 64, dtype, "bhtd", i).requires_grad_() for i in (2, 3))
    out = b200_pisa.attention(q, k1.expand(2, 4, 90, 64), v1.expand(2, 4, 90, 64))
    grads = torch.autograd.grad(out.sum(), (q, k1, v1))
    res, allow = plain_grads(q.detach(), k1.detach(), v1.detach(), torch.ones_like(q), 64 ** -0.5)
    u = torch.finfo(dtype).eps / 2
    close("out", out.detach(), res["out"], allow["out"](u))
    close("dq", grads[0], res["dq"], allow["dq"](u))
    # four heads' gradients rounded to the type one by one, then summed by autograd in it
    full, fallow = plain_grads(q.detach(), k1.detach().expand(2, 4, 90, 64), v1.detach().expand(2, 4, 90, 64),
                               torch.ones_like(q), 64 ** -0.5)
    for i, name in ((1, "dk"), (2, "dv")):
        total = full[name].sum(1, keepdim=True)
        allowed = fallow[name](u).sum(1, keepdim=True) + 4 * u * full[name].abs().sum(1, keepdim=True)
        close(name, grads[i], total, allowed)


@gpu
def test_three_dimensional_calls_and_unaligned_gradients():
    import b200_pisa

    q, k, v = (make(1, 6, t, 40, torch.bfloat16, "bhtd", i)[0] for i, t in ((1, 33), (2, 65), (3, 65)))
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    out = b200_pisa.attention(*leaves, scale=0.3)
    assert out.shape == q.shape
    wide = torch.randn(6, 33, 43, device=DEV).to(torch.bfloat16)
    dout = wide[..., 1:41]  # rows off the 16-byte boundaries
    grads = torch.autograd.grad(out, leaves, dout)
    four = [x[None] for x in (q, k, v)]
    res, allow = plain_grads(*four, dout[None], 0.3)
    check_all([x[None] for x in (out.detach(), *grads)], res, allow, torch.bfloat16)


@gpu
def test_gradients_match_differences():
    """Against central differences of the FP64 formula along a few directions."""
    import b200_pisa

    q, k, v = (make(1, 2, t, 64, torch.float16, "bthd", i) for i, t in ((1, 17), (2, 23), (3, 23)))
    dout = make(1, 2, 17, 64, torch.float16, "bthd", 4)
    out, lse = b200_pisa.attention_forward(q, k, v, causal=True)
    grads = b200_pisa.attention_backward(dout, q, k, v, out, lse, causal=True)

    def loss(*x):
        res, _ = reference(*x, None, 64 ** -0.5, True, None)
        return (res["out"] * dout.double()).sum().item()

    base = [x.double() for x in (q, k, v)]
    for i, g in enumerate(grads):
        way = torch.randn_like(base[i], dtype=torch.float64)
        step = 1e-5
        moved = [[x + s * step * way if j == i else x for j, x in enumerate(base)] for s in (1, -1)]
        slope = (loss(*moved[0]) - loss(*moved[1])) / (2 * step)
        # the gradient's FP16 terms add up to half a unit of FP16 of their sum at worst, a few times over
        assert abs((g.double() * way).sum().item() - slope) <= 4 * 2.0 ** -11 * (g.double() * way).abs().sum().item() + 1e-6


@gpu
@pytest.mark.parametrize("scale_dout,scale_v", [(1e-6, 1.0), (1e-7, 1e3), (3e2, 30.0)])
def test_fp16_gradients_of_any_size(scale_dout, scale_v):
    """dS neither underflows nor overflows FP16: what is lost is the last
    rounding (step 2^-24) of results that are themselves FP16."""
    import b200_pisa

    q, k = (make(1, 2, t, 128, torch.float16, "bthd", i) for i, t in ((1, 300), (2, 500)))
    v = make(1, 2, 500, 128, torch.float16, "bthd", 3, scale_v)
    dout = make(1, 2, 300, 128, torch.float16, "bthd", 4, scale_dout)
    out, lse = b200_pisa.attention_forward(q, k, v)
    grads = b200_pisa.attention_backward(dout, q, k, v, out, lse)
    res, allow = reference(q, k, v, dout, 128 ** -0.5, False, None)
    check_all((out, *grads), res, allow, torch.float16)


@gpu
def test_few_keys_keep_their_accuracy_through_autograd():
    """With two keys delta cancels against two dP terms: the rounding of out
    (2^-9) would be several times the error of everything else."""
    import b200_pisa

    for tk, lens in ((2, None), (300, (2, 300))):
        q = make(2, 4, 128, 64, torch.bfloat16, "bthd", 1).requires_grad_()
        k, v = (make(2, 4, tk, 64, torch.bfloat16, "bthd", i).requires_grad_() for i in (2, 3))
        lens_t = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=DEV)
        dout = make(2, 4, 128, 64, torch.bfloat16, "bthd", 4)
        out = b200_pisa.attention(q, k, v, key_lengths=lens_t)
        dq, dk, _ = torch.autograd.grad(out, (q, k, v), dout)
        res, _ = reference(q.detach(), k.detach(), v.detach(), dout, 64 ** -0.5, False, lens_t)
        for got, want in ((dq[0], res["dq"][0]), (dk[0], res["dk"][0])):  # the batch of two keys
            # roundings of P's and dS's 2^-9 and the result's, uniform and independent: their
            # root mean square is 2^-9 / sqrt(3) each, 2^-9 in all; delta's would add more than that again
            assert ((got.double() - want).norm() / want.norm()).item() < 2.0 ** -8.25


@gpu
def test_streams_two_calls_at_once_and_graph_replays():
    import b200_pisa
    from b200_pisa import _lib

    q, k, v = (make(1, h, t, 128, torch.bfloat16, "bthd", i) for i, h, t in ((1, 8, 700), (2, 4, 900), (3, 4, 900)))
    dout = make(1, 8, 700, 128, torch.bfloat16, "bthd", 4)

    def call():
        out, lse = b200_pisa.attention_forward(q, k, v, causal=True)
        return (out, lse, *b200_pisa.attention_backward(dout, q, k, v, out, lse, causal=True))

    eager = call()
    streams = [torch.cuda.Stream(DEV) for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream(DEV))
    at_once = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                at_once.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for got in at_once for x, y in zip(eager, got))
    graphs, captured = [], []
    for s in streams:  # two graphs with workspaces of their own, replayed at once
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            captured.append(call())
        graphs.append(g)
    q.mul_(0.5)
    fresh = call()
    torch.cuda.synchronize()
    for _ in range(2):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for got in captured for x, y in zip(fresh, got))
    _lib.check_status()


@gpu
def test_long_sequences_and_many_heads():
    import b200_pisa
    from b200_pisa import _lib

    # 33000 keys: the whole gradient of one head against FP64
    q, k, v, dout = (make(1, 1, t, 64, torch.bfloat16, "bthd", i) for i, t in ((1, 200), (2, 33000), (3, 33000), (4, 200)))
    out, lse = b200_pisa.attention_forward(q, k, v)
    res, allow = reference(q, k, v, dout, 0.125, False, None)
    check_all((out, *b200_pisa.attention_backward(dout, q, k, v, out, lse)), res, allow, torch.bfloat16)
    # 6000 heads of 5 tokens
    q, k, v, dout = (make(2, 3000, 5, 16, torch.float16, "bhtd", i) for i in range(4))
    out, lse = b200_pisa.attention_forward(q, k, v)
    res, allow = reference(q, k, v, dout, 0.25, False, None)
    check_all((out, *b200_pisa.attention_backward(dout, q, k, v, out, lse)), res, allow, torch.float16)
    _lib.check_status()


@gpu
def test_rows_past_32_bit_offsets():
    import b200_pisa

    storage = torch.empty(2 ** 31 + 2 ** 22, device=DEV, dtype=torch.bfloat16)
    far = lambda t: storage.as_strided((1, 2, t, 64), (0, 2 ** 31, 64, 1))  # noqa: E731
    near = [make(1, 2, t, 64, torch.bfloat16, "bthd", i) for i, t in ((1, 100), (2, 200), (3, 200), (4, 100))]
    want_out, want_lse = b200_pisa.attention_forward(*near[:3])
    want = b200_pisa.attention_backward(near[3], *near[:3], want_out, want_lse)
    for i, x in enumerate(near):
        y = far(x.shape[2])
        y.copy_(x)
        args = [*near[:i], y, *near[i + 1:]]
        out, lse = b200_pisa.attention_forward(*args[:3])
        got = b200_pisa.attention_backward(args[3], *args[:3], out, lse)
        assert torch.equal(out, want_out) and all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_equal_to_full_attention_and_to_the_node_default():
    """The forward-only entry point and this one agree within the rounding of
    their results (their products and order of sums are the same)."""
    import b200_pisa

    q, k, v = (make(1, 4, t, 128, torch.bfloat16, "bthd", i) for i, t in ((1, 130), (2, 260), (3, 260)))
    a = b200_pisa.full_attention(q, k, v, 128 ** -0.5)
    b = b200_pisa.attention(q, k, v)
    assert ((a.float() - b.float()).abs() <= 2.0 ** -8 * a.float().abs() + 1e-6).all()


@gpu
def test_contiguous_gradients_off_the_16_byte_boundaries():
    """contiguous() leaves such a tensor where it is."""
    import b200_pisa

    q, k, v, dout = (make(1, 2, 40, 64, torch.bfloat16, "bhtd", i) for i in range(4))
    out, lse = b200_pisa.attention_forward(q, k, v)
    want = b200_pisa.attention_backward(dout, q, k, v, out, lse)
    off = torch.empty(dout.numel() + 1, device=DEV, dtype=torch.bfloat16)[1:].view_as(dout)
    off.copy_(dout)
    assert off.is_contiguous() and off.data_ptr() % 16
    got = b200_pisa.attention_backward(off, q, k, v, out, lse)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    pos = torch.arange(40, device=DEV)[:, None]
    x = q.clone().requires_grad_()
    y = b200_pisa.axial_rope(x, pos, (64,))
    assert torch.equal(torch.autograd.grad(y, x, off, retain_graph=True)[0], torch.autograd.grad(y, x, dout)[0])


@gpu
def test_training_step_captured_whole():
    """Forward and backward through autograd in one graph, as a captured
    training step has them (no eager graph of the leaves is alive)."""
    import b200_pisa

    q, k, v = (make(1, 4, 200, 64, torch.bfloat16, "bthd", i).requires_grad_() for i in (1, 2, 3))
    w = torch.ones(64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    pos = torch.arange(200, device=DEV)[:, None]
    dout = make(1, 4, 200, 64, torch.bfloat16, "bthd", 4)

    def step():
        a = b200_pisa.norm_rope_attention(q, k, v, w, w, pos, (64,), causal=True)
        b = b200_pisa.attention(q, k, v)
        return torch.autograd.grad((a, b), (q, k, v, w), (dout, dout))

    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream(DEV).wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    with torch.no_grad():
        q.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    got = [x.clone() for x in captured]
    assert all(torch.equal(a, b) for a, b in zip(got, step()))


@gpu
@pytest.mark.parametrize("tq,tk,lens", [(113, 113, None), (300, 300, None), (70, 200, None), (200, 70, (70, 9)), (129, 400, (400, 60))])
def test_causal_rows_of_few_keys_keep_their_accuracy(tq, tk, lens):
    """The first rows of a causal call see few keys, and with_low's rounding
    error of out takes part in their gradients."""
    import b200_pisa

    q, k, v, dout = (make(2, 2, t, 64, torch.bfloat16, "bthd", i) for i, t in ((1, tq), (2, tk), (3, tk), (4, tq)))
    lens_t = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=DEV)
    torch.cuda.empty_cache()
    out, lse, low = b200_pisa.attention_forward(q, k, v, causal=True, key_lengths=lens_t, with_low=True)
    dq, dk, dv = b200_pisa.attention_backward(dout, q, k, v, out, lse, causal=True, key_lengths=lens_t, out_low=low)
    res, allow = reference(q, k, v, dout, 0.125, True, lens_t)
    check_all((out, dq, dk, dv), res, allow, torch.bfloat16)
    seen = torch.arange(tq, device=DEV)[None] + 1 + tk - tq
    limit = torch.full((2, 1), tk, device=DEV) if lens is None else lens_t[:, None]
    few = (torch.minimum(seen.expand(2, tq), limit.long()) <= 64)[:, None, :, None].expand_as(out)
    whole = out.double() + torch.where(few, low, torch.zeros_like(low)).double()
    p = res["out"]
    # P's rounding only: the row's output is exact but for 2^-9 of its P V terms
    err = ((whole - p) * few).norm() / (p * few).norm().clamp_min(1e-30)
    plain = ((out.double() - p) * few).norm() / (p * few).norm().clamp_min(1e-30)
    assert not few.any() or err < 0.85 * plain
    rows = few[..., 0]
    if rows.any():  # as for few keys without a mask: two roundings and P's in delta
        e = (dq.double() - res["dq"])[rows].norm() / res["dq"][rows].norm().clamp_min(1e-30)
        assert e < 2.0 ** -8.25


@gpu
def test_more_heads_than_a_grid_dimension_holds():
    import b200_pisa
    from b200_pisa import _lib

    q, k, v, dout = (make(2, 35000, 3, 8, torch.float16, "bhtd", i) for i in range(4))
    out, lse = b200_pisa.attention_forward(q, k, v, causal=True)
    res, allow = reference(q, k, v, dout, 8 ** -0.5, True, None)
    check_all((out, *b200_pisa.attention_backward(dout, q, k, v, out, lse, causal=True)), res, allow, torch.float16)
    pos = torch.arange(3, device=DEV)[:, None]
    fused = b200_pisa.norm_rope_attention(q, k, v, None, None, pos, (8,), causal=True)
    some = b200_pisa.norm_rope_attention(q[1:, 34000:], k[1:, 34000:], v[1:, 34000:], None, None, pos, (8,), causal=True)
    assert torch.equal(fused[1:, 34000:], some)
    _lib.check_status()


def test_wrong_types_are_refused_with_gradients_wanted_too():
    import b200_pisa

    x = _x(1, 2, 4, 16).requires_grad_()
    for args in ((None, x, x), (x, 3.0, x), (x, x, "v")):
        with pytest.raises(TypeError):
            b200_pisa.attention(*args)
