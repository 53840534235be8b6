"""64-bit references of nmt_gan_amd.ops, and how far a right kernel may be from them.

Every bound is derived from the arithmetic a kernel of this library may do, before it ran: operands are exact in their
type, products and sums are fp32 (an n-term sum is off by at most n 2^-24 of the sum of its terms' magnitudes, whatever its
order), probabilities and score gradients are rounded once to the operand type on their way into a matrix product (`u`,
half a step of the type; nothing in fp32), and results are rounded once more.
"""
import math

import torch

E = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def heads_of(t, heads):
    """[rows, heads dh] -> [heads, rows, dh] in 64 bits."""
    return t.double().reshape(t.shape[0], heads, t.shape[1] // heads).transpose(0, 1)


def rows_of(t):
    return t.transpose(0, 1).reshape(t.shape[1], t.shape[0] * t.shape[2])


def span_reference(q, k, v, lo, hi, heads, kv_heads, scale, cap=0.0, slopes=None, pos=None, dout=None):
    """{name: (value, bound)} of out, lse and - with dout - dq, dk, dv.  Rows outside every span are zeroed first (the
    operator does not read them)."""
    dt, n, g = q.dtype, k.shape[0], heads // kv_heads
    u = 0.0 if dt == torch.float32 else HALF[dt]
    tiny = 2.0 ** -25 if dt == torch.float16 else 0.0               # a probability below 2^-14 in fp16
    dh = q.shape[1] // heads
    if n == 0:
        zero = [torch.zeros(x.shape, dtype=torch.float64, device=q.device) for x in (q, k)]
        minus = torch.full((q.shape[0], heads), -math.inf, dtype=torch.float64, device=q.device)
        return {"out": (zero[0], zero[0]), "lse": (minus, minus), "dq": (zero[0], zero[0]), "dk": (zero[1], zero[1]), "dv": (zero[1], zero[1])}
    at = torch.arange(n, device=q.device)
    a, b = lo.long().clamp(min=0), hi.long().clamp(max=n)
    vis = (at[None] >= a[:, None]) & (at[None] < b[:, None])
    K = heads_of(torch.where(vis.any(0)[:, None], k, torch.zeros_like(k)), kv_heads).repeat_interleave(g, 0)
    V = heads_of(torch.where(vis.any(0)[:, None], v, torch.zeros_like(v)), kv_heads).repeat_interleave(g, 0)
    some = vis.any(1)
    Q = heads_of(torch.where(some[:, None], q, torch.zeros_like(q)), heads)
    s = scale * (Q @ K.transpose(1, 2))
    size = abs(scale) * (Q.abs() @ K.abs().transpose(1, 2))
    err = (dh + 4) * E * size
    turn = torch.full_like(s, scale)
    if cap:
        t = torch.tanh(s / cap)
        s, turn = cap * t, scale * (1 - t * t)
        err = err + 8 * E * cap
    if slopes is not None:
        p = (hi - 1 if pos is None else pos).double()
        bias = slopes.double()[:, None, None] * (p[:, None] - at[None].double()).abs()
        s = s - bias
        err = err + 4 * E * bias
    s = s.masked_fill(~vis, -math.inf)
    lse = torch.logsumexp(s, -1)
    P = torch.where(vis & some[:, None], torch.exp(s - lse.masked_fill(~some, 0.0)[..., None]), torch.zeros_like(s))
    out = P @ V
    # relative error of a probability: its score, the exponent's argument, the exponential
    top = torch.where(vis, s.abs() + lse.abs().masked_fill(~some, 0.0)[..., None] + 2, torch.zeros_like(s))
    rho = (torch.where(vis, err, torch.zeros_like(err)) + 8 * E * top).amax(-1, keepdim=True)
    cnt = vis.sum(1).double()[None, :, None]
    PV = P @ V.abs()
    e_out = (2 * rho + (cnt + 8) * E + u) * PV + tiny * (vis.double() @ V.abs())
    res = {"out": (rows_of(out), rows_of(e_out + HALF[dt] * (out.abs() + e_out) + 1e-30)),
           "lse": (lse.transpose(0, 1), ((2 * rho + (cnt + 8) * E).squeeze(-1)
                                         + 4 * E * lse.abs().masked_fill(~some, 0.0)).transpose(0, 1))}
    if dout is None:
        return res
    D = heads_of(torch.where(some[:, None], dout, torch.zeros_like(dout)), heads)
    dp, DV = D @ V.transpose(1, 2), D.abs() @ V.abs().transpose(1, 2)
    delta = (D * out).sum(-1, keepdim=True)
    e_delta = (D.abs() * (e_out + HALF[dt] * (out.abs() + e_out))).sum(-1, keepdim=True) + (dh + 2) * E * (D.abs() * out.abs()).sum(-1, keepdim=True)
    core = dp - delta
    dr = P * core * turn
    e_turn = 32 * E * abs(scale)
    e_dr = P * ((4 * rho + 8 * E) * core.abs() * turn.abs() + turn.abs() * ((dh + 2) * E * DV + e_delta) + e_turn * core.abs())
    e_dr = e_dr + u * (dr.abs() + e_dr)
    e_p = P * (2 * rho + u)
    n_q = vis.sum(0).double()[None, :, None] * 1.0

    def group(t):
        return t.reshape(kv_heads, g, n, dh).sum(1)

    dq = dr @ K
    e_dq = e_dr @ K.abs() + (cnt + 4) * E * (dr.abs() @ K.abs())
    dk, dv = group(dr.transpose(1, 2) @ Q), group(P.transpose(1, 2) @ D)
    e_dk = group(e_dr.transpose(1, 2) @ Q.abs() + (g * n_q + 4) * E * (dr.abs().transpose(1, 2) @ Q.abs()))
    e_dv = group(e_p.transpose(1, 2) @ D.abs() + (g * n_q + 4) * E * (P.transpose(1, 2) @ D.abs()))
    for name, x, e in (("dq", dq, e_dq), ("dk", dk, e_dk), ("dv", dv, e_dv)):
        res[name] = (rows_of(x), rows_of(e + HALF[dt] * (x.abs() + e) + 1e-30))
    return res


def xent_reference(h, w, labels, smoothing=0.0, grad_row=None):
    """{name: (value, bound)} of loss, lse, dh, dw."""
    dt, v, d = h.dtype, w.shape[0], h.shape[1]
    u = 0.0 if dt == torch.float32 else HALF[dt]
    used = (labels >= 0) & (labels < v)
    H, W = h.double(), w.double()
    z, size = H @ W.t(), H.abs() @ W.abs().t()
    e_z = (d + 4) * E * size
    wanted = torch.full_like(z, smoothing / (v - 1) if v > 1 else 0.0)
    wanted[torch.arange(h.shape[0], device=h.device), labels.clamp(0, v - 1).long()] = 1.0 - smoothing
    lse = torch.logsumexp(z, 1)
    far = (z.amax(1) - z.amin(1))
    e_lse = e_z.amax(1) + (128 + v / 64 + 8 * far.clamp(max=88.0)) * E + 4 * E * lse.abs()
    loss = lse - (wanted * z).sum(1)
    e_loss = e_lse + (wanted * e_z).sum(1) + (wanted * z.abs()).sum(1) * (136 + v / 64) * E + 4 * E * (loss.abs() + lse.abs())
    res = {"loss": (torch.where(used, loss, torch.zeros_like(loss)), torch.where(used, e_loss, torch.zeros_like(loss))),
           "lse": (lse, e_lse)}
    g = (torch.ones_like(lse) if grad_row is None else grad_row.double()) * used
    H = torch.where((g != 0)[:, None], H, torch.zeros_like(H))
    P = torch.exp(z - lse[:, None])
    dz = torch.where((g != 0)[:, None], (P - wanted) * g[:, None], torch.zeros_like(z))
    e_dz = torch.where((g != 0)[:, None], (P * (e_z + e_lse[:, None] + 8 * E * (2 + far[:, None])) + 4 * E * wanted) * g[:, None].abs(),
                       torch.zeros_like(z))
    # on its way into the products the entry-dependent part, p / high - [label], is rounded once: g high u |p / high - [label]|
    # <= g u (p + [label]) as |high| <= 1; the constant part of label smoothing is summed apart in fp32
    label_part = torch.zeros_like(z)
    label_part[torch.arange(h.shape[0], device=h.device), labels.clamp(0, v - 1).long()] = 1.0
    e_img = u * ((P + label_part) * g[:, None].abs() * (g != 0)[:, None] + e_dz).nan_to_num(0.0)
    e_dz = e_dz + e_img
    rows = float(h.shape[0])
    dh, dw = dz @ W, dz.t() @ H
    e_dh = e_dz @ W.abs() + (v + 8) * E * (dz.abs() @ W.abs())
    # dw's other factor is g h, rounded once too: u |g h| per term of the same size, (1 + u) for the two roundings together
    e_dw = (e_dz + (1 + u) * e_img).t() @ H.abs() + (rows + 64) * E * (dz.abs().t() @ H.abs())
    res["dh"] = (dh, e_dh + HALF[dt] * (dh.abs() + e_dh) + 1e-30)
    res["dw"] = (dw, e_dw + HALF[dt] * (dw.abs() + e_dw) + 1e-30)
    return res


def check(name, got, want):
    """Every element of `got` within its bound; infinities and NaN in the same places."""
    value, bound = want
    got = got.double()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(value)), name
    assert torch.equal(torch.isinf(got), torch.isinf(value)), name
    fine = torch.isfinite(value)
    assert torch.equal(got[~fine & ~torch.isnan(value)], value[~fine & ~torch.isnan(value)]), name
    off = ((got - value).abs() - bound)[fine]
    if off.numel():
        i = int(off.argmax())
        assert off[i] <= 0, "%s: off by %.3g where %.3g is allowed (value %.3g)" % (
            name, (got - value).abs()[fine][i], bound[fine][i], value[fine][i])
