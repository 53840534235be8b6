"""Refusals of the span attention, cross-entropy and global-norm entry points: everything the host can see is refused
with a message before any launch, so these run without a GPU (the pointers below are never followed)."""
import ctypes as C

import pytest

from nmt_gan_amd import _lib as L

P = 1 << 20                                                         # a 16-byte aligned address nobody reads


def _span(**kw):
    a = L.SpanArgs(dtype=L.NMTGAN_F32, M=4, N=4, heads=2, kv_heads=2, dh=64, q=P, ldq=128, k=P, ldk=128, v=P, ldv=128, lo=P, hi=P,
                   scale=1.0, cap=0.0, out=P, ldo=128, lse=P)
    for n, x in kw.items():
        setattr(a, n, x)
    return a


def _refused(rc, part):
    assert rc != 0
    assert part in L.lib.nmtgan_last_error().decode(), L.lib.nmtgan_last_error()


@pytest.mark.parametrize("kw,part", [
    (dict(dtype=7), "dtype"), (dict(M=-1), "shape"), (dict(N=-1), "shape"), (dict(M=2**31 - 65000), "shape"), (dict(N=2**31 - 1), "shape"), (dict(heads=0), "heads"), (dict(kv_heads=0), "heads"),
    (dict(heads=3), "heads"), (dict(dh=0), "head width"), (dict(dh=60), "head width"), (dict(dh=136), "head width"),
    (dict(scale=float("inf")), "finite"), (dict(cap=-1.0), "cap"), (dict(cap=float("nan")), "cap"), (dict(q=None), "null"),
    (dict(lo=None), "null"), (dict(hi=None), "null"), (dict(out=None), "null"), (dict(k=None), "null"), (dict(v=None), "null"),
    (dict(q=P + 4), "16-byte"), (dict(ldq=127), "16-byte"), (dict(ldq=64), "16-byte"), (dict(ldk=64), "16-byte"), (dict(ldv=130), "16-byte"),
    (dict(ldo=100), "16-byte"), (dict(v=P + 8), "16-byte")])
def test_span_refusals(kw, part):
    _refused(L.lib.nmtgan_attn_span(C.byref(_span(**kw)), None), part)
    _refused(L.lib.nmtgan_attn_span_step(C.byref(_span(**kw)), 4, P, 1 << 30, None), part)


def test_span_null_arguments_and_workspaces():
    _refused(L.lib.nmtgan_attn_span(None, None), "null")
    _refused(L.lib.nmtgan_attn_span_step(C.byref(_span()), 4000, P, 16, None), "workspace")
    _refused(L.lib.nmtgan_attn_span_step(C.byref(_span()), 4000, None, 1 << 30, None), "workspace")
    _refused(L.lib.nmtgan_attn_span_step(C.byref(_span()), -1, P, 1 << 30, None), "max_keys")
    assert L.lib.nmtgan_attn_span(C.byref(_span(M=0, q=None, lo=None, hi=None, out=None)), None) == 0      # nothing to do
    assert L.lib.nmtgan_attn_span_step_workspace_bytes(0, 2, 2, 64, 100) == 0


@pytest.mark.parametrize("kw,gkw,part", [
    (dict(dtype=L.NMTGAN_F16), {}, "bf16 or fp32"), (dict(lse=None), {}, "null"), ({}, dict(dout=None), "null"), ({}, dict(dq=None), "null"),
    ({}, dict(dk=None), "null"), ({}, dict(dv=None), "null"), ({}, dict(ld_dq=64), "16-byte"), ({}, dict(ld_dk=129), "16-byte"),
    ({}, dict(dv=P + 4), "16-byte"), ({}, dict(ld_dout=127), "16-byte")])
def test_span_grads_refusals(kw, gkw, part):
    g = L.SpanGrads(dout=P, ld_dout=128, dq=P, ld_dq=128, dk=P, ld_dk=128, dv=P, ld_dv=128)
    for n, x in gkw.items():
        setattr(g, n, x)
    _refused(L.lib.nmtgan_attn_span_grads(C.byref(_span(**kw)), C.byref(g), P, 1 << 30, None), part)
    if not kw and not gkw:
        _refused(L.lib.nmtgan_attn_span_grads(C.byref(_span()), C.byref(g), P, 16, None), "workspace")


def test_span_grads_workspace_and_null():
    g = L.SpanGrads(dout=P, ld_dout=128, dq=P, ld_dq=128, dk=P, ld_dk=128, dv=P, ld_dv=128)
    _refused(L.lib.nmtgan_attn_span_grads(C.byref(_span()), C.byref(g), P, 16, None), "workspace")
    _refused(L.lib.nmtgan_attn_span_grads(C.byref(_span()), None, P, 1 << 30, None), "null")


def _xent(**kw):
    a = L.XentArgs(dtype=L.NMTGAN_F32, M=4, V=10, d=64, h=P, ldh=64, w=P, ldw=64, labels=P, smoothing=0.0)
    for n, x in kw.items():
        setattr(a, n, x)
    return a


@pytest.mark.parametrize("kw,part", [
    (dict(dtype=3), "dtype"), (dict(M=-1), "shape"), (dict(V=0), "shape"), (dict(d=0), "shape"), (dict(d=62), "16 bytes"),
    (dict(smoothing=1.0), "smoothing"), (dict(smoothing=-0.1), "smoothing"), (dict(smoothing=0.1, V=1), "smoothing"), (dict(h=None), "null"),
    (dict(labels=None), "null"), (dict(w=None), "null"), (dict(w=P + 4), "16-byte"), (dict(ldw=60), "16-byte"), (dict(ldh=65), "16-byte"),
    (dict(M=2**31 - 1), "shape"), (dict(V=2**31 - 1), "shape"), (dict(M=2**30, V=2**30), "tiles"), (dict(ldw=2**21), "apart"), (dict(ldh=2**21), "apart")])
def test_xent_refusals(kw, part):
    _refused(L.lib.nmtgan_linear_xent(C.byref(_xent(**kw)), P, P, P, 1 << 30, None), part)
    _refused(L.lib.nmtgan_linear_xent_grads(C.byref(_xent(**kw)), P, None, P, 64, P, 64, P, 1 << 30, None), part)


def test_xent_other_refusals():
    _refused(L.lib.nmtgan_linear_xent(None, P, P, P, 1 << 30, None), "null")
    _refused(L.lib.nmtgan_linear_xent(C.byref(_xent()), None, P, P, 1 << 30, None), "null")
    _refused(L.lib.nmtgan_linear_xent(C.byref(_xent()), P, P, P, 8, None), "workspace")
    _refused(L.lib.nmtgan_linear_xent_grads(C.byref(_xent(dtype=L.NMTGAN_F16)), P, None, P, 64, P, 64, P, 1 << 30, None), "bf16 or fp32")
    _refused(L.lib.nmtgan_linear_xent_grads(C.byref(_xent()), None, None, P, 64, P, 64, P, 1 << 30, None), "null")
    _refused(L.lib.nmtgan_linear_xent_grads(C.byref(_xent()), P, None, P, 60, P, 64, P, 1 << 30, None), "dh")
    _refused(L.lib.nmtgan_linear_xent_grads(C.byref(_xent()), P, None, P, 64, None, 64, P, 1 << 30, None), "dw")
    _refused(L.lib.nmtgan_linear_xent_grads(C.byref(_xent()), P, None, P, 64, P, 64, P, 8, None), "workspace")
    _refused(L.lib.nmtgan_linear_xent_grads(C.byref(_xent(M=2**22 + 1)), P, None, P, 64, P, 64, P, 1 << 40, None), "2^22 rows")


def _list(*refs):
    return (L.GradRef * len(refs))(*[L.GradRef(*r) for r in refs]), len(refs)


@pytest.mark.parametrize("refs,part", [
    ([(P, P, -1, 1, 1)], "size"), ([(P, P, 5, 9, 9)], "dtype"), ([(None, P, 5, 1, 1)], "null"), ([(P + 2, P + 2, 5, 1, 1)], "misaligned"),
    ([(P, None, 5, 1, 1)], "null"), ([(P, P + 4096, 5, 1, 0)], "type"), ([(P, P, 5, 0, 1)], "in place"),
    ([(P, P, 5, 1, 1), (P, P, 5, 1, 1)], "overlap"), ([(P, P, 5, 1, 1), (P + 16, P + 16, 5, 1, 1)], "overlap"),
    ([(P, P + 16, 5, 1, 1)], "overlaps an output"), ([(P + 4096, P, 5, 1, 1), (P + 8192, P + 4096, 5, 1, 1)], "overlaps an output")])
def test_clip_refusals(refs, part):
    a, n = _list(*refs)
    _refused(L.lib.nmtgan_clip_global_norm(a, n, 1.0, 1.0, P, P, 1 << 20, None), part)


def test_norm_other_refusals():
    a, n = _list((P, P, 5, 1, 1))
    _refused(L.lib.nmtgan_clip_global_norm(a, n, 0.0, 1.0, P, P, 1 << 20, None), "max_norm")
    _refused(L.lib.nmtgan_clip_global_norm(a, n, 1.0, float("nan"), P, P, 1 << 20, None), "scale")
    _refused(L.lib.nmtgan_clip_global_norm(a, n, 1.0, 1.0, None, P, 1 << 20, None), "null")
    _refused(L.lib.nmtgan_clip_global_norm(a, n, 1.0, 1.0, P, P, 8, None), "workspace")
    _refused(L.lib.nmtgan_global_norm(a, n, 1.0, P, P, 8, None), "workspace")
    _refused(L.lib.nmtgan_global_norm(None, 3, 1.0, P, P, 1 << 20, None), "null")
    _refused(L.lib.nmtgan_global_norm(a, -1, 1.0, P, P, 1 << 20, None), "null")
    assert L.lib.nmtgan_global_norm_workspace_bytes(200) >= 3 * 1024 * 8


def test_tensor_calls_refuse_what_is_not_on_a_gpu():
    import torch

    from nmt_gan_amd import ops
    q, i = torch.zeros(4, 64), torch.zeros(4, dtype=torch.int32)
    for call in (lambda x: ops.attn_span(x, q, q, i, i, heads=1), lambda x: ops.attn_span_step(x, q, q, i, i, heads=1, max_keys=4),
                 lambda x: ops.attn_span_grads(q, x, q, q, q, q[:, 0], i, i, heads=1), lambda x: ops.linear_xent(x, q, i),
                 lambda x: ops.linear_xent_grads(x, q, i, q[:, 0]), lambda x: ops.global_norm([x]), lambda x: ops.clip_global_norm([x], 1.0)):
        for x in (q, None, q.numpy(), q.double()):
            with pytest.raises(ValueError):
                call(x)
    with pytest.raises(ValueError):
        ops.clip_global_norm([q], None)
