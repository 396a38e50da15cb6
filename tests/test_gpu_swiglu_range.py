"""SwiGLU where the gate's sigmoid leaves the range of fp32 but its product with the gate does not."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24  # half a step of fp32, relative


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [64, 37])
def test_swiglu_far_gates(cuda_ok, dtype, n):
    """g sigma(g) is a normal number down to g of about -91.8, where sigma itself is none any more; it keeps its relative
    accuracy down to there, and its gradient too."""
    from gsa_b200 import ops

    g = torch.linspace(-91.5, -85.0, n, device=DEV).to(dtype)
    g[:8] = torch.tensor([-87.0, -87.5, -88.0, -88.5, -89.0, -90.0, -91.0, -91.5], device=DEV).to(dtype)
    u = torch.where(torch.arange(n, device=DEV) % 2 == 0, 1.0, 3.0).to(dtype)
    z, packed = ops.silu_mul_packed(torch.cat([g, u]).view(1, -1))
    gd, ud = g.double(), u.double()
    want = gd / (1 + torch.exp(-gd)) * ud
    half = torch.finfo(dtype).eps / 2
    # 2^t of t = -g log2 e up to 132.1, 2 steps of the function beside its argument's compensation, its reciprocal and
    # three products: under 16 U; the output's own half step, or half the smallest subnormal
    assert bool(((z[0].double() - want).abs() <= (16 * U + half) * want.abs() + 2.0 ** -126 * half).all())
    # the backward pass at the kept values: dz of 2^40 brings the gradients back into the range
    dz = torch.full((1, n), 2.0 ** 40, device=DEV, dtype=dtype)
    dgu, z2 = ops.silu_mul_packed_backward(dz, packed, want_z=True)
    kept = packed.unpack(torch.float32).double()[0]
    gk, uk = kept[0], kept[1]
    up = torch.exp(-gk)
    slope = (1 + up + gk * up) / (1 + up) ** 2
    tiny = 2.0 ** -126
    for got, ref in ((dgu[0, :n], 2.0 ** 40 * uk * slope), (dgu[0, n:], 2.0 ** 40 * gk / (1 + up)), (z2[0], gk / (1 + up) * uk)):
        ok = (got.double() - ref).abs() <= (32 * U + half) * ref.abs() + tiny
        assert bool(ok.all()), (got, ref)
    assert bool((dgu[0] != 0).all())
