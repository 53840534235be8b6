"""Global norm and clipping where the factor leaves fp32's normal range."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [5, 40000])                           # the kernel's short and long loops
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("value,max_norm", [(1e38, 1.0), (3e38, 1e-6), (2e38, 1e-37), (1e-30, 1e-38), (1.0, 1e-40)])
def test_clip_by_factors_below_the_least_normal_number(cuda, n, dtype, value, max_norm):
    """max_norm / norm may be subnormal or zero in fp32 where the clipped values are not.  Into fp32: two products and the
    factor rounded, 4 x 2^-24 relative, or 2^-149 where the result itself is subnormal."""
    from nmt_gan_amd import ops
    g = [torch.full((n,), value, device=cuda).to(dtype), torch.tensor([-value, 0.0, value / 3], device=cuda).to(dtype)]
    out = [torch.full(t.shape, 7.0, device=cuda) for t in g]
    ops.clip_global_norm(ops.TensorList(g, out=out), max_norm)
    most = torch.tensor(max_norm, dtype=torch.float32).double().item()
    norm = math.sqrt(sum(float((t.double() / value).square().sum()) for t in g)) * value
    for t, o in zip(g, out):
        want = t.double() * (most / norm)
        assert bool(((o.double() - want).abs() <= want.abs() * 2.0 ** -22 + 2.0 ** -149).all()), (o[0].item(), want[0].item())


def test_clip_by_a_tiny_scale(cuda):
    from nmt_gan_amd import ops
    g = torch.tensor([1e30, -3e37, 0.0, 1.0], device=cuda)
    scale = torch.tensor(1e-40, dtype=torch.float32).double().item()
    want = g.double() * scale
    norm = ops.clip_global_norm([g], 1.0, grad_scale=1e-40)
    assert bool(((g.double() - want).abs() <= want.abs() * 2.0 ** -22 + 2.0 ** -149).all())
    assert abs(float(norm) - 3e37 * scale) <= 3e37 * scale * 2.0 ** -20
