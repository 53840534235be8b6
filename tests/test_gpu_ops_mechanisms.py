"""What the wider bounds of ops_reference.py would not show: the corrected delta of 16-bit gradients, scales below and at zero,
lse of the single-token form."""
import math
import random

import pytest
import torch

from ops_reference import E, HALF, TYPES, check, heads_of, rows_of, span_reference
from ops_step import step_with_lse

pytestmark = pytest.mark.gpu


def _ops():
    from nmt_gan_amd import ops
    return ops


def _normal(g, *shape, dt, times=1.0):
    return (torch.randn(*shape, generator=g) * times).to(dt)


def _whole(values, cuda):
    return torch.tensor(values, dtype=torch.int32, device=cuda)


def _corrected(q, k, v, lo, hi, heads, kv_heads, scale, cap, dout):
    """{name: (value, bound, value without the correction)} of bf16 dq and dk in which delta does not carry the rounding of `out`.

    delta is the walk's own sum of p dp: off by the probabilities' error rho and fp32 sums.  The walk multiplies
    c (dp - delta16), c = p (1 - t^2), delta16 = dout . out off by e_off, rounds that to bf16 (u), and adds
    (delta16 - delta) sum c k with c rounded (u): u |dr| as ever and twice u c e_off, of second order."""
    dt, dh, g = q.dtype, q.shape[1] // heads, heads // kv_heads
    u, half = HALF[dt], HALF[dt]
    at = torch.arange(k.shape[0], device=q.device)
    vis = (at[None] >= lo[:, None]) & (at[None] < hi[:, None])
    cnt = vis.sum(1).double()[None, :, None]
    Q, D = heads_of(q, heads), heads_of(dout, heads)
    K, V = (heads_of(t, kv_heads).repeat_interleave(g, 0) for t in (k, v))
    s = scale * (Q @ K.transpose(1, 2))
    size = abs(scale) * (Q.abs() @ K.abs().transpose(1, 2))
    err = (dh + 4) * E * size + 8 * E * cap
    turn = torch.full_like(s, scale)
    if cap:
        t = torch.tanh(s / cap)
        s, turn = cap * t, scale * (1 - t * t)
    s = s.masked_fill(~vis, -math.inf)
    lse = torch.logsumexp(s, -1, keepdim=True)
    P = torch.exp(s - lse)
    top = torch.where(vis, s.abs() + lse.abs() + 2, torch.zeros_like(s))
    rho = (torch.where(vis, err, torch.zeros_like(err)) + 8 * E * top).amax(-1, keepdim=True)
    out, PV = P @ V, P @ V.abs()
    dp, DV = D @ V.transpose(1, 2), D.abs() @ V.abs().transpose(1, 2)
    delta = (D * out).sum(-1, keepdim=True)
    e_out = (2 * rho + (cnt + 8) * E + u) * PV
    e_off = (D.abs() * (e_out + half * (out.abs() + e_out))).sum(-1, keepdim=True) + (dh + 2) * E * (D.abs() * out.abs()).sum(-1, keepdim=True)
    e_delta = (2 * rho + (cnt + 8) * E) * (P * dp.abs()).sum(-1, keepdim=True) + (dh + 2) * E * (P * DV).sum(-1, keepdim=True)
    core, turn_size = dp - delta, turn.abs() + 32 * E * abs(scale)
    dr = P * core * turn
    e_dr = P * ((4 * rho + 8 * E) * core.abs() * turn_size + turn_size * ((dh + 2) * E * DV + e_delta) + 32 * E * abs(scale) * core.abs()
                + 4 * E * turn_size * (dp.abs() + delta.abs() + e_off))
    e_dr = e_dr + u * (dr.abs() + e_dr) + 2 * u * (1 + u) * P * turn_size * e_off
    seen = vis.sum(0).double()[None, :, None]

    def group(t):
        return t.reshape(kv_heads, g, t.shape[1], dh).sum(1)

    delta16 = (D * heads_of(rows_of(out).to(dt), heads)).sum(-1, keepdim=True)
    dr16 = P * (dp - delta16) * turn
    res = {}
    for name, x, e, wrong in (("dq", dr @ K, e_dr @ K.abs() + (2 * cnt + 8) * E * (dr.abs() @ K.abs()), dr16 @ K),
                              ("dk", group(dr.transpose(1, 2) @ Q), group(e_dr.transpose(1, 2) @ Q.abs() + (g * seen + 4) * E * (dr.abs().transpose(1, 2) @ Q.abs())),
                               group(dr16.transpose(1, 2) @ Q))):
        res[name] = (rows_of(x), rows_of(e + half * (x.abs() + e) + 1e-30), rows_of(wrong))
    return res


@pytest.mark.parametrize("heads,kv_heads,dh,cap", [(2, 2, 64, 0.0), (2, 1, 128, 0.0), (4, 2, 32, 5.0), (64, 64, 64, 0.0), (64, 32, 32, 20.0)])
def test_delta_does_not_carry_the_rounding_of_out(cuda, heads, kv_heads, dh, cap):
    """Documents of one to four rows; heads * blocks on both sides of the choice between shared and single walks."""
    ops, dt = _ops(), torch.bfloat16
    g, rng = torch.Generator().manual_seed(dh), random.Random(dh)
    m, lo, hi = 1100, [], []
    while len(lo) < m:
        a, n = len(lo), min(rng.randint(1, 4), m - len(lo))
        lo, hi = lo + [a] * n, hi + [a + i + 1 for i in range(n)]
    q, dout = (_normal(g, m, heads * dh, dt=dt).to(cuda) for _ in range(2))
    k, v = (_normal(g, m, kv_heads * dh, dt=dt).to(cuda) for _ in range(2))
    lo, hi = _whole(lo, cuda), _whole(hi, cuda)
    how = dict(heads=heads, kv_heads=kv_heads, scale=dh ** -0.5, cap=cap)
    out, lse = ops.attn_span(q, k, v, lo, hi, **how)
    got = dict(zip(("dq", "dk"), ops.attn_span_grads(dout, q, k, v, out, lse, lo, hi, **how)))
    want = _corrected(q, k, v, lo, hi, heads, kv_heads, dh ** -0.5, cap, dout)
    for name, x in got.items():
        value, bound, wrong = want[name]
        assert bool(((wrong - value).abs() > bound).any()), name     # without the correction the check below would fail
        check(name, x, (value, bound))


@pytest.mark.parametrize("op", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("scale", [-0.125, -1.0, 0.0])
@pytest.mark.parametrize("heads,kv_heads,dh,cap,bias", [(2, 2, 64, 0.0, False), (4, 2, 32, 3.0, False), (2, 1, 128, 0.0, True), (2, 2, 64, 200.0, True),
                                                         (64, 64, 32, 0.0, False)])
def test_scales_below_and_at_zero(cuda, op, scale, heads, kv_heads, dh, cap, bias):
    """The largest score is the smallest product, or all scores are one number."""
    ops, dt = _ops(), TYPES[op]
    g = torch.Generator().manual_seed(heads + dh)
    m = 1100 if heads == 64 else 333
    q = _normal(g, m, heads * dh, dt=dt).to(cuda)
    k, v = (_normal(g, m, kv_heads * dh, dt=dt).to(cuda) for _ in range(2))
    dout = _normal(g, m, heads * dh, dt=dt, times=0.1).to(cuda)
    lo, hi = _whole([i // 90 * 90 for i in range(m - 3)] + [0] * 3, cuda), _whole([i + 1 for i in range(m - 3)] + [0] * 3, cuda)
    slopes = torch.tensor([2.0 ** (-8 * (h + 1) / heads) for h in range(heads)], device=cuda) if bias else None
    how = dict(heads=heads, kv_heads=kv_heads, scale=scale, cap=cap, slopes=slopes)
    grads = None if dt == torch.float16 else dout
    want = span_reference(q, k, v, lo, hi, heads, kv_heads, scale, cap, slopes, dout=grads)
    out, lse = ops.attn_span(q, k, v, lo, hi, **how)
    got = {"out": out, "lse": lse}
    if grads is not None:
        got["dq"], got["dk"], got["dv"] = ops.attn_span_grads(dout, q, k, v, out, lse, lo, hi, **how)
    for name, x in got.items():
        check(name, x, want[name])
    for keys in (1, 5000):
        check("step", ops.attn_span_step(q, k, v, lo, hi, max_keys=keys, **how), want["out"])


@pytest.mark.parametrize("op", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("heads,kv_heads,dh,cap,bias", [(8, 8, 64, 0.0, False), (8, 2, 64, 30.0, True), (6, 3, 24, 0.0, True), (16, 1, 128, 5.0, False)])
def test_lse_of_single_tokens(cuda, op, heads, kv_heads, dh, cap, bias):
    """In one part and in several, and a row without keys."""
    dt, rows, cache = TYPES[op], 5, 2500
    g = torch.Generator().manual_seed(dh)
    q = _normal(g, rows, heads * dh, dt=dt).to(cuda)
    k, v = (_normal(g, rows * cache, kv_heads * dh, dt=dt).to(cuda) for _ in range(2))
    lo = torch.arange(rows, dtype=torch.int32, device=cuda) * cache
    hi = lo + _whole([cache, 0, 1, 300, 2047], cuda)
    slopes = torch.rand(heads, generator=g).to(cuda) * 0.1 if bias else None
    want = span_reference(q, k, v, lo, hi, heads, kv_heads, dh ** -0.5, cap, slopes)
    for keys in (1, 1024, cache, 40 * cache):
        out, lse = step_with_lse(q, k, v, lo, hi, heads, kv_heads, dh ** -0.5, cap, slopes, max_keys=keys)
        check("out of %d" % keys, out, want["out"])
        check("lse of %d" % keys, lse, want["lse"])
