"""Operators of teacher-forced training, prompts and single tokens as functions of torch tensors over the C ABI
(include/nmtgan.h: nmtgan_attn_span*, nmtgan_linear_xent*, nmtgan_*global_norm).

Every function checks its arguments on the host (ValueError; NmtGanError with the library's message for what the library
refuses, outputs that lie over an input among it), allocates outputs and scratch through torch's caching allocator and enqueues on
the current stream of the tensors' device without synchronising; inside a graph capture the scratch belongs to the graph's pool.  Tensors made on another stream are the caller's to order, as with any kernel.
There is no autograd: gradients are explicit calls, as everywhere in this package, inputs that require gradients are taken as
they are, and torch's version of every tensor that a call writes goes up.  (The checks and calls themselves are
compiled: csrc/calls.cpp.)
"""
from __future__ import annotations

import ctypes as C

from ._lib import lib

_ENTRIES = ("nmtgan_attn_span", "nmtgan_attn_span_step", "nmtgan_attn_span_step_workspace_bytes", "nmtgan_attn_span_grads",
            "nmtgan_attn_span_grads_workspace_bytes", "nmtgan_linear_xent", "nmtgan_linear_xent_grads",
            "nmtgan_linear_xent_workspace_bytes", "nmtgan_global_norm_workspace_bytes", "nmtgan_global_norm", "nmtgan_clip_global_norm")


class _FirstUse:
    """Stands for the compiled calls until one is made: they are built against one torch, and nothing else in the package needs
    them.  There is no other path: without them a call raises."""

    def __getattr__(self, name):
        global _calls
        if name.startswith("__"):
            raise AttributeError(name)
        import torch                                       # noqa: F401  (the library that _calls.so is linked against)
        try:
            from . import _calls as found
        except ImportError as e:
            raise ImportError("nmt_gan_amd/_calls.so is missing or does not fit this torch: make -C nmt_gan_amd/csrc") from e
        found.bind({n: C.cast(getattr(lib, n), C.c_void_p).value for n in _ENTRIES})
        _calls = found
        return getattr(found, name)


_calls = _FirstUse()


# ---------------------------------------------------------------------------------------------- span attention
def attn_span(q, k, v, lo, hi, *, heads, kv_heads=None, scale=1.0, cap=0.0, slopes=None, pos=None, out=None):
    """(out [M, heads dh], lse [M, heads] fp32) of q [M, heads dh] over k, v [N, kv_heads dh]; row i sees keys lo[i] <= j < hi[i].

    score = scale q.k, with cap > 0 cap tanh(score / cap), minus slopes[h] |pos[i] - j| (pos: hi - 1 unless given; pos[i] - j has to
    fit 32 bits).  A row that sees nothing gets 0 and -inf.  For many rows (training, prompts); attn_span_step is the form for single tokens.
    """
    return _calls.attn_span(q, k, v, lo, hi, heads, kv_heads, scale, cap, slopes, pos, out)


def attn_span_step(q, k, v, lo, hi, *, heads, max_keys, kv_heads=None, scale=1.0, cap=0.0, slopes=None, pos=None, out=None):
    """attn_span for a few rows over long spans (one token for each of many requests): spans are cut along their keys.
    max_keys: the longest span expected (a hint: longer ones are right too)."""
    return _calls.attn_span_step(q, k, v, lo, hi, heads, kv_heads, scale, cap, slopes, pos, max_keys, out)


def attn_span_grads(dout, q, k, v, out, lse, lo, hi, *, heads, kv_heads=None, scale=1.0, cap=0.0, slopes=None, pos=None,
                    dq=None, dk=None, dv=None):
    """(dq, dk, dv) of attn_span for its results `out`, `lse` and the output gradient `dout`; bfloat16 or float32."""
    return _calls.attn_span_grads(q, k, v, lo, hi, heads, kv_heads, scale, cap, slopes, pos, dout, out, lse, dq, dk, dv)


# ---------------------------------------------------------------------------------------------- cross entropy
def linear_xent(h, w, labels, *, smoothing=0.0):
    """(loss [M], lse [M]), fp32: label-smoothed cross entropy of softmax(h w^T) row by row, h [M, d], w [V, d], without the
    [M, V] logits.  A label outside [0, V) gives loss 0."""
    return _calls.linear_xent(h, w, labels, smoothing)


def linear_xent_grads(h, w, labels, lse, grad_row=None, *, smoothing=0.0, dh=None, dw=None):
    """(dh, dw) of sum_i grad_row[i] loss[i] (grad_row None: 1 each) with linear_xent's lse; bfloat16 or float32."""
    return _calls.linear_xent_grads(h, w, labels, smoothing, lse, grad_row, dh, dw)


# ---------------------------------------------------------------------------------------------- global norm
def split_flat(flat, tensors):
    """Views of the one-dimensional `flat`, one for each tensor and of its shape, back to back (an optimizer's flat buffer)."""
    sizes = [t.numel() for t in tensors]
    if flat.dim() != 1 or flat.numel() != sum(sizes):
        raise ValueError("split_flat: the tensors hold %d elements, the buffer %s" % (sum(sizes), tuple(flat.shape)))
    return [f.view(t.shape) for f, t in zip(flat.split(sizes), tensors)]


class TensorList:
    """A list of contiguous gradient tensors (bfloat16, float16, float32, mixed) on one GPU, and where their clipped values
    go: `out` holds a tensor of the same size for each, of its type or float32; without it they are clipped in place.
    Built once for buffers that live as long as the list, which keeps them alive; every call looks at the tensors again, so one
    that has been given other memory (t.data = ..., t.set_(...)) since is read and written there."""

    def __init__(self, grads, out=None):
        self.grads = list(grads)
        self.out = self.grads if out is None else list(out)
        _calls.check_list(self.grads, self.out)
        self.device = self.grads[0].device


def _lists(tensors):
    if isinstance(tensors, TensorList):
        return tensors.grads, tensors.out
    grads = list(tensors)
    return grads, grads


def global_norm(tensors, *, grad_scale=1.0):
    """sqrt(sum (grad_scale g)^2) over a TensorList (or a list of tensors), as a float32 scalar on the device."""
    return _calls.global_norm(*_lists(tensors), grad_scale, None)


def clip_global_norm(tensors, max_norm, *, grad_scale=1.0):
    """Writes grad_scale g min(1, max_norm / norm) to the list's outputs and returns the norm (before clipping), a float32
    scalar on the device.  A gradient that is not finite makes every output NaN."""
    if max_norm is None:
        raise ValueError("clip_global_norm: max_norm=None")
    return _calls.global_norm(*_lists(tensors), grad_scale, max_norm)
