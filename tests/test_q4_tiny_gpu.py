"""Quantising groups of weights so small that their scale has no reciprocal in 32 bits."""
import pytest
import torch

from conftest import load

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("exponent", [-120, -124, -126, -128, -130])
def test_tiny_weights(cuda, group, zeros, exponent):
    """Every weight to its nearest value: the step is the scale, a multiple of bf16's smallest number 2^-133, whose own rounding (half of that,
    or 2^-9 of itself) shifts the ends of 15 steps; the weights keep their signs.  A projection of unit vectors times 2^100 shows them."""
    ops = load("ops")
    N, K = 128, 256
    W = (torch.randn(N, K, generator=torch.Generator().manual_seed(group)) * 2.0 ** exponent).bfloat16()
    W[0] = 0.0
    q = ops.QuantWeight(W.to(cuda), group, zeros)
    eye = (torch.eye(K, device=cuda) * 2.0 ** 100).bfloat16()
    got = torch.cat([ops.linear(eye[i:i + 16].contiguous(), q, flags=ops.OUT_F32) for i in range(0, K, 16)]).T.cpu().double() * 2.0 ** -100
    w = W.double().view(N, K // group, group)
    if zeros:
        step = (w.amax(-1).clamp(min=0) - w.amin(-1).clamp(max=0)) / 15
    else:
        step = w.abs().amax(-1) / 7
    off = torch.maximum(2.0 ** -8 * step, torch.full_like(step, 2.0 ** -134))  # (of the scale)
    # a zero point adds half a step at the ends of the range
    limit = ((0.5 + 0.5 * zeros) * (step + off) + 15 * off)[..., None].expand_as(w).reshape(N, K)
    assert bool(((got - W.double()).abs() <= limit).all()), float(((got - W.double()).abs() / limit.clamp(min=2.0 ** -140)).max())
    far = W.double().abs() > limit
    assert bool((got[far].sign() == W.double()[far].sign()).all()) and not bool(got[0].any())
