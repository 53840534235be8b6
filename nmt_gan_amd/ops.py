"""Operators of teacher-forced training, prompts and single tokens as functions of torch tensors over the C ABI
(include/nmtgan.h: nmtgan_attn_span*, nmtgan_linear_xent*, nmtgan_*global_norm).

Every function checks its arguments on the host (ValueError), allocates outputs and scratch through torch's caching
allocator and enqueues on the current stream of the tensors' device without synchronising; inside a graph capture the
scratch belongs to the graph's pool.  Tensors made on another stream are the caller's to order, as with any kernel.
There is no autograd: gradients are explicit calls, as everywhere in this package.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib as L
from ._lib import lib

_CODE = {torch.bfloat16: L.NMTGAN_BF16, torch.float16: L.NMTGAN_F16, torch.float32: L.NMTGAN_F32}
_SIZE = {torch.bfloat16: 2, torch.float16: 2, torch.float32: 4}
_raw_stream = torch._C._cuda_getCurrentRawStream      # the hipStream_t of torch.cuda.current_stream(index)


def _fail(what, text):
    raise ValueError("%s: %s" % (what, text))


def _rows(what, name, t, width, device, dtype):
    """(address, row stride) of a [rows, width] matrix whose rows are contiguous and 16-byte aligned."""
    shape, at = t.shape, t.data_ptr()
    if len(shape) != 2 or shape[1] != width:
        _fail(what, "%s must be [rows, %d], is %s" % (name, width, tuple(shape)))
    if t.dtype != dtype or t.device != device:
        _fail(what, "%s is %s on %s, expected %s on %s" % (name, t.dtype, t.device, dtype, device))
    step, one = t.stride()
    if shape[0] < 2:
        step = width
    if (one != 1 and width > 1) or step < width or step * _SIZE[dtype] % 16 or at % 16:
        _fail(what, "%s needs contiguous rows that start at 16-byte boundaries" % name)
    return at, step


def _vector(what, name, t, n, device, dtype):
    if t.shape != (n,) or t.dtype != dtype or t.device != device or (n > 1 and t.stride(0) != 1):
        _fail(what, "%s must be a contiguous %s vector of %d on %s" % (name, dtype, n, device))
    return t.data_ptr()


def _target(what, name, t, rows, width, device, dtype):
    """An output given by the caller, or a new one."""
    if t is None:
        return torch.empty(rows, width, device=device, dtype=dtype)
    if t.shape[0] != rows:
        _fail(what, "%s must have %d rows" % (name, rows))
    return t


def _gpu(what, t):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _fail(what, "tensors on a GPU are needed")
    if t.dtype not in _CODE:
        _fail(what, "bfloat16, float16 or float32 expected, got %s" % t.dtype)
    return t.device


def _run(what, device, fn, *args):
    """Calls an entry point on the current stream of `device`."""
    index = device.index
    if index == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _raw_stream(index))
    if rc:
        L.check(rc, what)


def _scratch(n, device):
    return torch.empty(max(int(n), 1), device=device, dtype=torch.uint8)


# ---------------------------------------------------------------------------------------------- span attention
def _span(what, q, k, v, lo, hi, heads, kv_heads, scale, cap, slopes, pos):
    dev, dt = _gpu(what, q), q.dtype
    kv_heads = heads if kv_heads is None else kv_heads
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        _fail(what, "heads=%r must be a multiple of kv_heads=%r" % (heads, kv_heads))
    if q.dim() != 2 or k.dim() != 2 or q.shape[1] % heads:
        _fail(what, "q must be [rows, heads * dh] and k [keys, kv_heads * dh]")
    dh = q.shape[1] // heads
    if dh < 1 or dh % 8 or dh > 128:
        _fail(what, "the head width %d must be a multiple of 8, at most 128" % dh)
    if not math.isfinite(scale) or not math.isfinite(cap) or cap < 0:
        _fail(what, "scale and cap must be finite, cap >= 0")
    m, n = q.shape[0], k.shape[0]
    if m >= 1 << 31 or n >= 1 << 31 or v.shape[0] != n:
        _fail(what, "k has %d rows, v %d" % (n, v.shape[0]))
    a = L.SpanArgs(_CODE[dt], m, n, heads, kv_heads, dh, *_rows(what, "q", q, heads * dh, dev, dt),
                   *_rows(what, "k", k, kv_heads * dh, dev, dt), *_rows(what, "v", v, kv_heads * dh, dev, dt),
                   _vector(what, "lo", lo, m, dev, torch.int32), _vector(what, "hi", hi, m, dev, torch.int32),
                   None if pos is None else _vector(what, "pos", pos, m, dev, torch.int32),
                   None if slopes is None else _vector(what, "slopes", slopes, heads, dev, torch.float32), scale, cap)
    return a, dev, dt


def attn_span(q, k, v, lo, hi, *, heads, kv_heads=None, scale=1.0, cap=0.0, slopes=None, pos=None, out=None):
    """(out [M, heads dh], lse [M, heads] fp32) of q [M, heads dh] over k, v [N, kv_heads dh]; row i sees keys lo[i] <= j < hi[i].

    score = scale q.k, with cap > 0 cap tanh(score / cap), minus slopes[h] |pos[i] - j| (pos: hi - 1 unless given).  A row
    that sees nothing gets 0 and -inf.  For many rows (training, prompts); attn_span_step is the form for single tokens.
    """
    a, dev, dt = _span("attn_span", q, k, v, lo, hi, heads, kv_heads, scale, cap, slopes, pos)
    out = _target("attn_span", "out", out, a.M, q.shape[1], dev, dt)
    lse = torch.empty(a.M, heads, device=dev, dtype=torch.float32)
    a.out, a.ldo = _rows("attn_span", "out", out, q.shape[1], dev, dt)
    a.lse = lse.data_ptr()
    _run("attn_span", dev, lib.nmtgan_attn_span, C.byref(a))
    return out, lse


def attn_span_step(q, k, v, lo, hi, *, heads, max_keys, kv_heads=None, scale=1.0, cap=0.0, slopes=None, pos=None, out=None):
    """attn_span for a few rows over long spans (one token for each of many requests): spans are cut along their keys.
    max_keys: the longest span expected (a hint: longer ones are right too)."""
    a, dev, dt = _span("attn_span_step", q, k, v, lo, hi, heads, kv_heads, scale, cap, slopes, pos)
    if not 0 <= max_keys < 1 << 31:
        _fail("attn_span_step", "max_keys=%r" % max_keys)
    out = _target("attn_span_step", "out", out, a.M, q.shape[1], dev, dt)
    a.out, a.ldo = _rows("attn_span_step", "out", out, q.shape[1], dev, dt)
    n = lib.nmtgan_attn_span_step_workspace_bytes(a.M, heads, a.kv_heads, a.dh, max_keys)
    ws = _scratch(n, dev) if n else None
    _run("attn_span_step", dev, lib.nmtgan_attn_span_step, C.byref(a), max_keys, L.ptr(ws), n)
    return out


def attn_span_grads(dout, q, k, v, out, lse, lo, hi, *, heads, kv_heads=None, scale=1.0, cap=0.0, slopes=None, pos=None,
                    dq=None, dk=None, dv=None):
    """(dq, dk, dv) of attn_span for its results `out`, `lse` and the output gradient `dout`; bfloat16 or float32."""
    what = "attn_span_grads"
    a, dev, dt = _span(what, q, k, v, lo, hi, heads, kv_heads, scale, cap, slopes, pos)
    if dt == torch.float16:
        _fail(what, "bfloat16 or float32 (float16 gradients would underflow without loss scaling)")
    wq, wk = q.shape[1], k.shape[1]
    for name, t in (("dout", dout), ("out", out)):
        if t.shape[0] != a.M:
            _fail(what, "%s must have %d rows" % (name, a.M))
    if lse.shape != (a.M, heads) or lse.dtype != torch.float32 or lse.device != dev or not lse.is_contiguous():
        _fail(what, "lse must be attn_span's [%d, %d] float32 result" % (a.M, heads))
    dq = _target(what, "dq", dq, a.M, wq, dev, dt)
    dk = _target(what, "dk", dk, a.N, wk, dev, dt)
    dv = _target(what, "dv", dv, a.N, wk, dev, dt)
    a.out, a.ldo = _rows(what, "out", out, wq, dev, dt)
    a.lse = lse.data_ptr()
    g = L.SpanGrads(*_rows(what, "dout", dout, wq, dev, dt), *_rows(what, "dq", dq, wq, dev, dt),
                    *_rows(what, "dk", dk, wk, dev, dt), *_rows(what, "dv", dv, wk, dev, dt))
    n = lib.nmtgan_attn_span_grads_workspace_bytes(a.M, heads)
    ws = _scratch(n, dev)
    _run(what, dev, lib.nmtgan_attn_span_grads, C.byref(a), C.byref(g), ws.data_ptr(), n)
    return dq, dk, dv


# ---------------------------------------------------------------------------------------------- cross entropy
def _xent(what, h, w, labels, smoothing):
    dev, dt = _gpu(what, h), h.dtype
    if h.dim() != 2 or w.dim() != 2 or w.shape[0] < 1 or h.shape[1] < 1:
        _fail(what, "h must be [rows, d] and w [vocabulary, d]")
    if not 0.0 <= smoothing < 1.0 or (smoothing and w.shape[0] < 2):
        _fail(what, "smoothing must be in [0, 1), and 0 for a vocabulary of one")
    if h.shape[1] * h.element_size() % 16 or max(h.shape[0], w.shape[0], w.shape[1]) >= 1 << 31:
        _fail(what, "a row of h must be a multiple of 16 bytes")
    m, v, d = h.shape[0], w.shape[0], h.shape[1]
    a = L.XentArgs(_CODE[dt], m, v, d, *_rows(what, "h", h, d, dev, dt), *_rows(what, "w", w, d, dev, dt),
                   _vector(what, "labels", labels, m, dev, torch.int32), smoothing)
    return a, dev, dt


def linear_xent(h, w, labels, *, smoothing=0.0):
    """(loss [M], lse [M]), fp32: label-smoothed cross entropy of softmax(h w^T) row by row, h [M, d], w [V, d], without the
    [M, V] logits.  A label outside [0, V) gives loss 0."""
    a, dev, _ = _xent("linear_xent", h, w, labels, smoothing)
    loss, lse = torch.empty(2, a.M, device=dev, dtype=torch.float32).unbind(0)
    n = lib.nmtgan_linear_xent_workspace_bytes(C.byref(a), 0)
    ws = _scratch(n, dev)
    _run("linear_xent", dev, lib.nmtgan_linear_xent, C.byref(a), loss.data_ptr(), lse.data_ptr(), ws.data_ptr(), n)
    return loss, lse


def linear_xent_grads(h, w, labels, lse, grad_row=None, *, smoothing=0.0, dh=None, dw=None):
    """(dh, dw) of sum_i grad_row[i] loss[i] (grad_row None: 1 each) with linear_xent's lse; bfloat16 or float32."""
    what = "linear_xent_grads"
    a, dev, dt = _xent(what, h, w, labels, smoothing)
    if dt == torch.float16:
        _fail(what, "bfloat16 or float32 (float16 gradients would underflow without loss scaling)")
    dh = _target(what, "dh", dh, a.M, a.d, dev, dt)
    dw = _target(what, "dw", dw, a.V, a.d, dev, dt)
    dh_at, dw_at = _rows(what, "dh", dh, a.d, dev, dt), _rows(what, "dw", dw, a.d, dev, dt)
    ls = _vector(what, "lse", lse, a.M, dev, torch.float32)
    g = None if grad_row is None else _vector(what, "grad_row", grad_row, a.M, dev, torch.float32)
    n = lib.nmtgan_linear_xent_workspace_bytes(C.byref(a), 1)
    ws = _scratch(n, dev)
    _run(what, dev, lib.nmtgan_linear_xent_grads, C.byref(a), ls, g, *dh_at, *dw_at, ws.data_ptr(), n)
    return dh, dw


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
    Built once for buffers that live as long as the list, which keeps them alive."""

    def __init__(self, grads, out=None):
        grads = list(grads)
        out = grads if out is None else list(out)
        if not grads:
            raise ValueError("TensorList: no tensors")
        if len(out) != len(grads):
            raise ValueError("TensorList: %d gradients, %d outputs" % (len(grads), len(out)))
        self.device = _gpu("TensorList", grads[0])
        self.grads, self.out = grads, out
        self._refs = (L.GradRef * len(grads))()
        for i, (g, o) in enumerate(zip(grads, out)):
            for t in (g, o):
                if t.device != self.device or t.dtype not in _CODE or not t.is_contiguous():
                    raise ValueError("TensorList: tensor %d must be contiguous, floating and on %s" % (i, self.device))
            if o.numel() != g.numel() or (o.dtype != g.dtype and o.dtype != torch.float32):
                raise ValueError("TensorList: output %d must have its gradient's size, and its type or float32" % i)
            r = self._refs[i]
            r.g, r.out, r.n, r.dtype, r.out_dtype = g.data_ptr(), o.data_ptr(), g.numel(), _CODE[g.dtype], _CODE[o.dtype]
        self._bytes = lib.nmtgan_global_norm_workspace_bytes(len(grads))


def _norm_args(what, tensors, grad_scale):
    if not isinstance(tensors, TensorList):
        tensors = TensorList(tensors)
    if not math.isfinite(grad_scale):
        _fail(what, "grad_scale=%r" % grad_scale)
    return tensors, torch.empty((), device=tensors.device, dtype=torch.float32), _scratch(tensors._bytes, tensors.device)


def global_norm(tensors, *, grad_scale=1.0):
    """sqrt(sum (grad_scale g)^2) over a TensorList (or a list of tensors), as a float32 scalar on the device."""
    t, norm, ws = _norm_args("global_norm", tensors, grad_scale)
    _run("global_norm", t.device, lib.nmtgan_global_norm, t._refs, len(t._refs), grad_scale, norm.data_ptr(), ws.data_ptr(), t._bytes)
    return norm


def clip_global_norm(tensors, max_norm, *, grad_scale=1.0):
    """Writes grad_scale g min(1, max_norm / norm) to the list's outputs and returns the norm (before clipping), a float32
    scalar on the device.  A norm that is not finite makes every output NaN."""
    if not (math.isfinite(max_norm) and max_norm > 0):
        _fail("clip_global_norm", "max_norm=%r" % max_norm)
    t, norm, ws = _norm_args("clip_global_norm", tensors, grad_scale)
    _run("clip_global_norm", t.device, lib.nmtgan_clip_global_norm, t._refs, len(t._refs), max_norm, grad_scale, norm.data_ptr(),
         ws.data_ptr(), t._bytes)
    return norm
