"""Cross entropy of few rows over large tables."""
import pytest
import torch

from ops_reference import HALF, check, xent_reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,v,d,smoothing", [(1, 50257, 1024, 0.1), (8, 50257, 1024, 0.0), (32, 20011, 512, 0.1), (32, 50257, 520, 0.0), (31, 70001, 768, 0.1)])
def test_gradients_of_up_to_32_rows_round_results_only(cuda, m, v, d, smoothing):
    """bf16: d(logits) stay in fp32, so the bounds are those of the same operands in fp32 and one rounding of the result."""
    from nmt_gan_amd import ops
    g = torch.Generator().manual_seed(m)
    h = torch.randn(m, d, generator=g).to(torch.bfloat16).to(cuda)
    w = (torch.randn(v, d, generator=g) * 2.0 * d ** -0.5).to(torch.bfloat16).to(cuda)
    labels = torch.randint(0, v, (m,), generator=g, dtype=torch.int32).to(cuda)
    labels[m // 2:m // 2 + m // 8] = -1
    weight = (torch.rand(m, generator=g) / m).to(cuda)
    loss, lse = ops.linear_xent(h, w, labels, smoothing=smoothing)
    dh, dw = ops.linear_xent_grads(h, w, labels, lse, weight, smoothing=smoothing)
    want = xent_reference(h.float(), w.float(), labels, smoothing, weight)
    half = HALF[torch.bfloat16]
    for name, x in (("loss", loss), ("lse", lse)):
        check(name, x, want[name])
    for name, x in (("dh", dh), ("dw", dw)):
        value, bound = want[name]
        check(name, x, (value, bound + half * (value.abs() + bound)))
