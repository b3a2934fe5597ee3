"""Exact attention where single values decide: a dominant key over a long tail.

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
