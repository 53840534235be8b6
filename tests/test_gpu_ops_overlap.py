"""Calls of span attention and cross entropy whose outputs lie between their inputs, and over them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_outputs_over_inputs_are_refused(cuda):
    from nmt_gan_amd import NmtGanError, ops
    q, k, v, out, do = (torch.randn(40, 128, device=cuda) for _ in range(5))
    lo, hi = torch.zeros(40, dtype=torch.int32, device=cuda), torch.arange(1, 41, dtype=torch.int32, device=cuda)
    o, lse = ops.attn_span(q, k, v, lo, hi, heads=2)
    w, labels = torch.randn(33, 128, device=cuda), torch.zeros(40, dtype=torch.int32, device=cuda)
    _, z = ops.linear_xent(q, w, labels)
    buf = torch.randn(41, 128, device=cuda)
    bad = [
        lambda: ops.attn_span(q, k, v, lo, hi, heads=2, out=q), lambda: ops.attn_span(q, k, v, lo, hi, heads=2, out=k),
        lambda: ops.attn_span_step(q, k, v, lo, hi, heads=2, max_keys=40, out=v), lambda: ops.attn_span(buf[1:], k, v, lo, hi, heads=2, out=buf[:40]),
        lambda: ops.attn_span_grads(do, q, k, v, o, lse, lo, hi, heads=2, dq=q), lambda: ops.attn_span_grads(do, q, k, v, o, lse, lo, hi, heads=2, dq=do),
        lambda: ops.attn_span_grads(do, q, k, v, o, lse, lo, hi, heads=2, dk=out, dv=out), lambda: ops.linear_xent_grads(q, w, labels, z, dh=q),
        lambda: ops.linear_xent_grads(q, w, labels, z, dw=w), lambda: ops.linear_xent_grads(q, w, labels, z, dh=buf[:40], dw=buf[8:]),
    ]
    before = [t.clone() for t in (q, k, v, do, w)]
    for n, call in enumerate(bad):
        with pytest.raises(NmtGanError, match="overlaps"):
            call()
            raise AssertionError("call %d was taken" % n)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, (q, k, v, do, w)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_columns_of_one_buffer_are_taken(cuda, dtype):
    """q, k, v, the result, its gradient and theirs as columns of one buffer: side by side, not over each other."""
    from nmt_gan_amd import ops
    g = torch.Generator().manual_seed(1)
    src = [torch.randn(300, 128, generator=g).to(dtype).to(cuda) for _ in range(4)]
    lo, hi = torch.zeros(300, dtype=torch.int32, device=cuda), torch.arange(1, 301, dtype=torch.int32, device=cuda)
    o, lse = ops.attn_span(*src[:3], lo, hi, heads=2)
    step = ops.attn_span_step(*src[:3], lo, hi, heads=2, max_keys=3000)
    want = ops.attn_span_grads(src[3], *src[:3], o, lse, lo, hi, heads=2)
    buf = torch.full((300, 9 * 128), 7.0, dtype=dtype, device=cuda)
    col = [buf[:, 128 * i:128 * i + 128] for i in range(9)]
    for c, t in zip(col[:4], src):
        c.copy_(t)
    _, lse2 = ops.attn_span(*col[:3], lo, hi, heads=2, out=col[4])
    got = ops.attn_span_grads(col[3], *col[:3], col[4], lse2, lo, hi, heads=2, dq=col[5], dk=col[6], dv=col[7])
    ops.attn_span_step(*col[:3], lo, hi, heads=2, max_keys=3000, out=col[8])
    for a, b in zip((lse2, col[4], col[8]) + got, (lse, o, step) + want):
        assert torch.equal(a, b)
    labels = torch.arange(300, dtype=torch.int32, device=cuda) % 50
    w = torch.randn(50, 128, generator=g).to(dtype).to(cuda)
    _, z = ops.linear_xent(src[0], w, labels)
    dh, dw = ops.linear_xent_grads(src[0], w, labels, z)
    table = torch.zeros(50, 256, dtype=dtype, device=cuda)
    table[:, :128] = w
    dh2, dw2 = ops.linear_xent_grads(col[0], table[:, :128], labels, z, dh=col[1], dw=table[:, 128:])
    assert torch.equal(dh, dh2) and torch.equal(dw, dw2)
