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


@pytest.mark.parametrize("given", [False, True])
def test_a_list_follows_its_tensors(cuda, given):
    """Tensors that get other memory, another size or another type behind the list are read and written where they are now."""
    from nmt_gan_amd import ops
    first = [torch.full((1000,), 3.0, device=cuda), torch.full((17,), 4.0, device=cuda)]
    grads = [t.clone() for t in first]
    out = [torch.zeros(1000, device=cuda), torch.zeros(17, device=cuda)] if given else None
    tensors = ops.TensorList(grads, out=out)
    before = [t.data for t in grads]                                # keeps the memory that the list was built on
    ops.global_norm(tensors)
    grads[0].data = torch.full((1000,), 30.0, device=cuda)
    grads[1].set_(torch.full((17,), 40.0, device=cuda))
    norm = ops.clip_global_norm(tensors, 1.0)
    want = math.sqrt(1000 * 900.0 + 17 * 1600.0)
    assert abs(float(norm) - want) <= want * 2.0 ** -23
    for o, value in zip(out if given else grads, (30.0, 40.0)):
        assert bool(((o.double() - value / want).abs() <= 2.0 ** -22 * value / want).all())
    assert all(torch.equal(a, b) for a, b in zip(before, first))    # nothing was written there
    grads[1].data = torch.ones(5, device=cuda)
    if given:                                                       # its output no longer fits
        with pytest.raises(ValueError):
            ops.clip_global_norm(tensors, 1.0)
    else:
        grads[0].data = torch.full((9,), 2.0, dtype=torch.float16, device=cuda)
        assert abs(float(ops.global_norm(tensors)) - math.sqrt(41.0)) <= 1e-6
    grads[0].data = torch.ones(1000)
    with pytest.raises(ValueError):
        ops.global_norm(tensors)
