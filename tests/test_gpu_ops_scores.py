"""Scores of span attention where a form could lose them: wide caps, small capped scores of short spans, packed beside long ones."""
import pytest
import torch

from ops_reference import E, TYPES, check, heads_of, span_reference
from ops_step import step_with_lse

pytestmark = pytest.mark.gpu


def _ops():
    from nmt_gan_amd import ops
    return ops


def _normal(g, *shape, dt, times=1.0):
    return (torch.randn(*shape, generator=g) * times).to(dt)


def _whole(values, cuda):
    return torch.tensor(values, dtype=torch.int32, device=cuda)


@pytest.mark.parametrize("op", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("heads,kv_heads,dh", [(2, 2, 64), (4, 1, 32), (2, 1, 128)])
@pytest.mark.parametrize("cap", [100.0, 3e4, 1e6, 1e30])
def test_wide_caps(cuda, op, heads, kv_heads, dh, cap):
    """A cap far above the scores changes next to nothing, and loses nothing.  A capped score is its product through a
    hyperbolic tangent and a few products, relative errors of 8 E in all on top of (dh + 4) E of the sum's magnitude: the bounds
    of the same scores without a cap, 1 + 8 / (dh + 4) <= 1.25 times.  (The cap itself moves a probability by s^3 / (3 cap^2) < 2 %.)"""
    ops, dt = _ops(), TYPES[op]
    g = torch.Generator().manual_seed(dh)
    m = 300
    q = _normal(g, m, heads * dh, dt=dt).to(cuda)
    k, v = (_normal(g, m, kv_heads * dh, dt=dt).to(cuda) for _ in range(2))
    dout = _normal(g, m, heads * dh, dt=dt, times=0.1).to(cuda)
    lo, hi = _whole([0] * 40 + [i // 30 * 30 for i in range(40, m - 2)] + [0, 0], cuda), _whole(list(range(1, m - 1)) + [0, 0], cuda)
    how = dict(heads=heads, kv_heads=kv_heads, scale=dh ** -0.5, cap=cap)
    grads = None if dt == torch.float16 else dout
    value = span_reference(q, k, v, lo, hi, heads, kv_heads, dh ** -0.5, cap, dout=grads)
    bound = span_reference(q, k, v, lo, hi, heads, kv_heads, dh ** -0.5, dout=grads)
    out, lse = ops.attn_span(q, k, v, lo, hi, **how)
    got = {"out": out, "lse": lse}
    if grads is not None:
        got["dq"], got["dk"], got["dv"] = ops.attn_span_grads(dout, q, k, v, out, lse, lo, hi, **how)
    for name, x in got.items():
        check(name, x, (value[name][0], 1.25 * bound[name][1]))
    for keys in (1, 5000):                                          # in one part, in several
        out, lse = step_with_lse(q, k, v, lo, hi, heads, kv_heads, dh ** -0.5, cap, max_keys=keys)
        check("step", out, (value["out"][0], 1.25 * bound["out"][1]))
        check("step lse", lse, (value["lse"][0], 1.25 * bound["lse"][1]))


@pytest.mark.parametrize("op", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (64, 64), (4, 1)])
def test_small_capped_scores_beside_a_long_document(cuda, op, heads, kv_heads):
    """Rows that see one key: lse is the score itself.  Its error: dh E of the sum's magnitude for the product, 12 E of the score
    for the tangent (4 E), the scale, the cap and the passage through log 2.  It is the same bits wherever the row is packed."""
    ops, dt, dh, cap = _ops(), TYPES[op], 64, 50.0
    g = torch.Generator().manual_seed(heads)
    m = 1100
    q = _normal(g, m, heads * dh, dt=dt, times=0.2).to(cuda)
    k, v = (_normal(g, m, kv_heads * dh, dt=dt, times=0.2).to(cuda) for _ in range(2))
    # rows 0 .. 999 one causal document, of its rows every fifth one sees itself only; the rest see themselves only
    alone = [i % 5 == 3 or i >= 1000 for i in range(m)]
    lo, hi = _whole([i if a else 0 for i, a in enumerate(alone)], cuda), _whole([i + 1 for i in range(m)], cuda)
    mine = torch.tensor(alone, device=cuda)
    scores = dh ** -0.5 * heads_of(q, heads) * heads_of(k, kv_heads).repeat_interleave(heads // kv_heads, 0)
    value = (cap * torch.tanh(scores.sum(-1) / cap)).transpose(0, 1)
    bound = (dh + 16) * E * scores.abs().sum(-1).transpose(0, 1)
    how = dict(heads=heads, kv_heads=kv_heads, scale=dh ** -0.5, cap=cap)
    lse = ops.attn_span(q, k, v, lo, hi, **how)[1]
    check("lse", lse[mine], (value[mine], bound[mine]))
    by_itself = ops.attn_span(q, k, v, hi - 1, hi, **how)[1]
    assert torch.equal(lse[mine], by_itself[mine])
    for keys in (1, 5000):
        check("step lse", step_with_lse(q, k, v, lo, hi, heads, kv_heads, dh ** -0.5, cap, max_keys=keys)[1][mine], (value[mine], bound[mine]))


def test_a_cap_that_float32_does_not_have_is_refused(cuda):
    """Rounded to zero it would mean no cap; the least one that there is makes all scores equal."""
    ops = _ops()
    g = torch.Generator().manual_seed(3)
    q, k, v = (_normal(g, 50, 64, dt=torch.float32, times=4.0).to(cuda) for _ in range(3))
    lo, hi = _whole([0] * 50, cuda), _whole(range(1, 51), cuda)
    o, lse = ops.attn_span(q, k, v, lo, hi, heads=1)
    for call in (lambda c: ops.attn_span(q, k, v, lo, hi, heads=1, cap=c), lambda c: ops.attn_span_step(q, k, v, lo, hi, heads=1, max_keys=50, cap=c),
                 lambda c: ops.attn_span_grads(o, q, k, v, o, lse, lo, hi, heads=1, cap=c)):
        with pytest.raises(ValueError, match="cap"):
            call(1e-60)
    out, lse = ops.attn_span(q, k, v, lo, hi, heads=1, cap=1e-36)
    mean = v.double().cumsum(0) / hi.double()[:, None]
    assert bool(((out.double() - mean).abs() <= 60 * E * v.double().abs().cumsum(0) / hi.double()[:, None]).all())
    assert bool(((lse[:, 0].double() - hi.double().log()).abs() <= 8 * E * (1 + hi.double().log())).all())
