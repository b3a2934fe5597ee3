"""Exact attention where single values decide: a dominant key over a long tail,
queries that are not numbers.

FP16 holds P = exp(s - running max) times 2^8, so a P below FP16's normal range
is off by at most half a step of 2^-24, 2^-33 of the largest; the row sum is of
the FP32 values.  Normalised, n keys are off by n 2^-33 max|v| together, beside
the terms u (P |V|) + u |out| of the two roundings and 2^-18 P |V| of the FP32
part."""
import math

import pytest
import torch

from gpu_util import DEV

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("at", [0, 1000, -1])
@pytest.mark.parametrize("d,keys", [(64, 32768), (128, 65535), (8, 9216)])
def test_a_dominant_key_over_a_long_tail(d, keys, at, dtype):
    """Tens of thousands of keys at 2^-25.5 of one: together up to 1.4e-3 of the row, which FP16 alone cannot hold."""
    import b200_pisa
    from b200_pisa import _lib

    gen = torch.Generator(device=DEV).manual_seed(keys + d)
    q = torch.zeros(1, 2, 5, d, device=DEV, dtype=dtype)
    q[..., 0] = 1.0
    q[..., 1] = 0.25
    k = torch.zeros(1, 2, keys, d, device=DEV, dtype=dtype)
    k[..., 1] = torch.randn(1, 2, keys, generator=gen, device=DEV).clamp(-1, 1).to(dtype)
    k[:, :, at, 0], k[:, :, at, 1] = 25.5 * math.log(2.0), 0.0
    v = (0.5 + torch.rand(1, 2, keys, d, generator=gen, device=DEV)).to(dtype)
    v[:, :, at] = 0.0  # the output is the tail's alone
    out, lse = b200_pisa.attention_forward(q, k, v, 1.0)
    _lib.check_status()
    s = q.double() @ k.double().transpose(-1, -2)
    want_lse = torch.logsumexp(s, -1)
    p = (s - want_lse[..., None]).exp()
    want = p @ v.double()
    u = torch.finfo(dtype).eps / 2
    allowed = (u + 2.0 ** -18) * want + u * want
    if dtype == torch.float16:
        allowed = allowed + keys * 2.0 ** -33 * v.double().abs().amax() + 2.0 ** -25  # the result's own subnormal step
    off = (out.double() - want).abs()
    assert (off <= allowed * (1 + 2 ** -8)).all(), f"off by {off.max().item():.3g} of {want.max().item():.3g}, allowed {allowed.max().item():.3g}"
    assert ((lse.double() - want_lse).abs() <= 2.0 ** -18 + 2.0 ** -22 * want_lse.abs()).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("tq,tk,causal,lens", [(200, 200, False, None), (200, 333, True, None), (300, 129, True, None),
                                               (130, 200, False, (200, 65)), (129, 65, True, (65, 3))])
def test_a_query_that_is_not_a_number_stays_one(tq, tk, causal, lens, d, dtype):
    """Its out, lse and dq are NaN, unless it sees no key; other rows do not notice, bit for bit."""
    import b200_pisa
    from b200_pisa import _lib

    gen = torch.Generator(device=DEV).manual_seed(tq)
    q, k, v, dout = (torch.randn(2, 2, t, d, generator=gen, device=DEV).to(dtype) for t in (tq, tk, tk, tq))
    k[1, 1, :, 0] = k[1, 1, :, 0].abs() + 0.5
    lens_t = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=DEV)
    kw = dict(causal=causal, key_lengths=lens_t)

    def run(q):
        q = q.clone().requires_grad_()
        out = b200_pisa.attention(q, k, v, **kw)
        return out.detach(), b200_pisa.attention_forward(q, k, v, **kw)[1], torch.autograd.grad(out, q, dout)[0]

    rows = [(0, 0, 0), (0, 1, 77), (1, 0, tq - 1), (1, 1, 5), (1, 1, 127)]
    bad = q.clone()
    for i, r in enumerate(rows):
        bad[r] = math.nan if i % 2 == 0 else bad[r]
        bad[r][0] = math.nan if i != 3 else -math.inf  # k's first column there is positive: every logit -inf
    hit = torch.zeros(2, 2, tq, dtype=torch.bool, device=DEV)
    for r in rows:
        hit[r] = True
    seen = torch.full((2, tq), tk, device=DEV) if lens is None else lens_t[:, None].expand(2, tq)
    if causal:
        seen = torch.minimum(seen, torch.arange(tq, device=DEV) + tk - tq + 1)
    sees = (seen > 0)[:, None].expand(2, 2, tq)
    clean, got = run(q), run(bad)
    _lib.check_status()
    nan = hit & sees
    assert torch.equal(got[0].isnan().all(-1), nan) and torch.equal(got[0].isnan().any(-1), nan)
    assert torch.equal(got[2].isnan().all(-1), nan) and torch.equal(got[2].isnan().any(-1), nan)
    minus = torch.zeros_like(nan)
    minus[1, 1, 5] = True  # the logarithm of a sum of zeros
    assert torch.equal(got[1].isnan(), nan & ~minus)
    assert (got[1][nan & minus] == -math.inf).all() and (got[1][~sees] == -math.inf).all()
    assert not got[0][~sees].any() and not got[2][~sees].any()
    for a, b in zip(clean, got):
        assert torch.equal(a[~nan], b[~nan])


@gpu
def test_a_layer_query_that_is_not_a_number_stays_one():
    import b200_pisa

    gen = torch.Generator(device=DEV).manual_seed(2)
    q, k, v = (torch.randn(1, 2, 150, 64, generator=gen, device=DEV).to(torch.bfloat16) for _ in range(3))
    pos = torch.arange(150, device=DEV)[:, None]
    run = lambda q: b200_pisa.norm_rope_attention(q, k, v, None, None, pos, (64,))  # noqa: E731
    clean = run(q)
    q[0, 1, 33, 7] = math.nan
    got = run(q)
    assert got[0, 1, 33].isnan().all()
    clean[0, 1, 33] = got[0, 1, 33] = 0.0
    assert torch.equal(clean, got)


@gpu
def test_the_benchmark_node_s_default_sizes_equal_full_attention():
    """1 x 4 heads, 128 tokens x 64, FP16: two kernels that round P and their result once each, at worst apart by
    both roundings of both, u (P |V|) + u |out| each, and the FP32 part 2^-18 P |V|."""
    import b200_pisa

    gen = torch.Generator(device=DEV).manual_seed(11)
    q, k, v = (torch.randn(1, 4, 128, 64, generator=gen, device=DEV).to(torch.float16) for _ in range(3))
    a = b200_pisa.full_attention(q, k, v, 64 ** -0.5).double()
    b = b200_pisa.attention(q, k, v).double()
    p = (q.double() @ k.double().transpose(-1, -2) * 64 ** -0.5).softmax(-1)
    u = 2.0 ** -11
    allowed = 2 * (((u + 2.0 ** -18) * p) @ v.double().abs() + u * (p @ v.double()).abs()) * (1 + 2 ** -8) + 128 * 2.0 ** -25 * v.abs().max()
    assert ((a - b).abs() <= allowed).all()
