"""Torch's version counters of tensors that an operator writes."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _rises(tensors, call):
    before = [t._version for t in tensors]
    call()
    return [t._version > b for t, b in zip(tensors, before)]


def test_written_tensors_get_a_new_version(cuda):
    from nmt_gan_amd import ops
    q, k, v, do, o, dq, dk, dv = (torch.randn(20, 64, device=cuda) for _ in range(8))
    lo, hi = torch.zeros(20, dtype=torch.int32, device=cuda), torch.arange(1, 21, dtype=torch.int32, device=cuda)
    w, dw, labels = torch.randn(30, 64, device=cuda), torch.empty(30, 64, device=cuda), torch.zeros(20, dtype=torch.int32, device=cuda)
    read = [q, k, v, do, lo, hi, w, labels]
    versions = [t._version for t in read]
    assert all(_rises([o], lambda: ops.attn_span(q, k, v, lo, hi, heads=1, out=o)))
    lse = ops.attn_span(q, k, v, lo, hi, heads=1)[1]
    assert all(_rises([o], lambda: ops.attn_span_step(q, k, v, lo, hi, heads=1, max_keys=20, out=o)))
    assert all(_rises([dq, dk, dv], lambda: ops.attn_span_grads(do, q, k, v, o, lse, lo, hi, heads=1, dq=dq, dk=dk, dv=dv)))
    z = ops.linear_xent(q, w, labels)[1]
    assert all(_rises([dq, dw], lambda: ops.linear_xent_grads(q, w, labels, z, dh=dq, dw=dw)))
    assert all(_rises([dq, dw], lambda: ops.clip_global_norm([dq, dw], 1.0)))
    flat = torch.empty(dq.numel() + dw.numel(), device=cuda)
    tensors = ops.TensorList([dq, dw], out=ops.split_flat(flat, [dq, dw]))
    assert _rises([dq, dw, flat], lambda: ops.clip_global_norm(tensors, 1.0)) == [False, False, True]
    assert not any(_rises([dq, dw, flat], lambda: ops.global_norm(tensors)))
    assert [t._version for t in read] == versions


def test_autograd_sees_a_saved_tensor_that_was_written(cuda):
    from nmt_gan_amd import ops
    x = torch.randn(20, 64, device=cuda, requires_grad=True)
    y = x * 2
    loss = (y * y).sum()                                            # keeps y for its gradient
    ops.clip_global_norm([y.detach()], 1e-3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_tensors_of_inference_mode(cuda):
    from nmt_gan_amd import ops
    with torch.inference_mode():
        q, k, v, o = (torch.randn(20, 64, device=cuda) for _ in range(4))
        lo, hi = torch.zeros(20, dtype=torch.int32, device=cuda), torch.arange(1, 21, dtype=torch.int32, device=cuda)
        ops.attn_span(q, k, v, lo, hi, heads=1, out=o)
    assert torch.equal(ops.attn_span(q, k, v, lo, hi, heads=1)[0], o)
    ops.clip_global_norm([o], 1.0)                                  # outside of it too
