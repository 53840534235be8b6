"""nmt_gan_amd.ops on the GPU against 64-bit references (ops_reference.py, where the tolerances are derived)."""
import math
import random

import pytest
import torch

from ops_reference import HALF, TYPES, check, span_reference, xent_reference

pytestmark = pytest.mark.gpu


def _ops():
    from nmt_gan_amd import ops
    return ops


def _normal(g, *shape, dt, times=1.0):
    return (torch.randn(*shape, generator=g) * times).to(dt)


def _documents(rows, longest, kind, seed, tail=3):
    """Spans of documents packed one behind the other, `tail` rows at the end that see nothing."""
    rng = random.Random(seed)
    lo, hi = [], []
    while len(lo) < rows - tail:
        a, n = len(lo), min(rows - tail - len(lo), rng.randint(1, longest))
        seen = {"causal": 0, "document": n, "prefix": rng.randint(0, n), "window": 0}[kind]
        lo += [max(a, a + i - 4) if kind == "window" else a for i in range(n)]
        hi += [a + max(i + 1, seen) for i in range(n)]
    return lo + [0] * min(tail, rows), hi + [0] * min(tail, rows)


def _span_case(cuda, ops, dt, lo, hi, n, heads, kv_heads, dh, cap=0.0, bias=False, grads=True, seed=0, own_place=True, fused=False,
               times=1.0):
    g = torch.Generator().manual_seed(seed)
    m = len(lo)
    q = _normal(g, m, heads * dh, dt=dt, times=times).to(cuda)
    if fused:                                                       # one [rows, q | k | v] buffer, as a fused projection writes it
        buf = _normal(g, max(m, n), (heads + 2 * kv_heads) * dh, dt=dt).to(cuda)
        q, k, v = buf[:m, :heads * dh], buf[:n, heads * dh:(heads + kv_heads) * dh], buf[:n, (heads + kv_heads) * dh:]
    else:
        k, v = _normal(g, n, kv_heads * dh, dt=dt, times=times).to(cuda), _normal(g, n, kv_heads * dh, dt=dt).to(cuda)
    dout = _normal(g, m, heads * dh, dt=dt, times=0.1).to(cuda)
    lo, hi = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in (lo, hi))
    pos = torch.arange(m, dtype=torch.int32, device=cuda) if bias and own_place else None
    slopes = torch.tensor([2.0 ** (-8 * (h + 1) / heads) for h in range(heads)], device=cuda) if bias else None
    how = dict(heads=heads, kv_heads=kv_heads, scale=dh ** -0.5, cap=cap, slopes=slopes, pos=pos)
    out, lse = ops.attn_span(q, k, v, lo, hi, **how)
    got = {"out": out, "lse": lse}
    grads = grads and dt != torch.float16
    if grads:
        got["dq"], got["dk"], got["dv"] = ops.attn_span_grads(dout, q, k, v, out, lse, lo, hi, **how)
    torch.cuda.synchronize()
    want = span_reference(q, k, v, lo, hi, heads, kv_heads, dh ** -0.5, cap, slopes, pos, dout if grads else None)
    for name, x in got.items():
        check(name, x, want[name])
    return got


@pytest.mark.parametrize("op", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,longest,kind,heads,kv_heads,dh,cap,bias", [
    (70, 20, "causal", 2, 2, 64, 0.0, False),
    (300, 50, "causal", 8, 8, 64, 0.0, False),
    (333, 333, "causal", 4, 2, 64, 20.0, True),
    (200, 90, "prefix", 4, 1, 32, 0.0, False),
    (257, 128, "document", 2, 2, 128, 5.0, False),
    (130, 70, "window", 3, 3, 48, 0.0, True),
    (129, 129, "causal", 4, 4, 16, 0.0, False),
    (65, 40, "prefix", 6, 2, 24, 2.0, True),
    (100, 64, "document", 2, 1, 8, 0.0, False),
    (190, 150, "causal", 2, 2, 96, 0.0, True),
    (64, 64, "document", 1, 1, 80, 0.0, False),
    (5, 2, "causal", 2, 2, 64, 0.0, False),
])
def test_span_documents(cuda, op, rows, longest, kind, heads, kv_heads, dh, cap, bias):
    lo, hi = _documents(rows, longest, kind, rows)
    _span_case(cuda, _ops(), TYPES[op], lo, hi, rows, heads, kv_heads, dh, cap, bias, seed=rows)


@pytest.mark.parametrize("op", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("heads,kv_heads,dh,longest,kind,cap,bias", [
    (64, 64, 64, 50, "causal", 0.0, False), (64, 64, 8, 50, "prefix", 3.0, True), (72, 72, 128, 30, "document", 0.0, True),
    (128, 64, 32, 40, "causal", 0.0, False), (64, 64, 16, 600, "causal", 0.0, False)])
def test_span_many_blocks(cuda, op, heads, kv_heads, dh, longest, kind, cap, bias):
    """Launches with so many blocks of rows that waves walk short spans alone; a long document among them does not."""
    lo, hi = _documents(1100, longest, kind, heads + dh)
    if longest < 100:
        lo, hi = lo[:700] + [700] * 400, hi[:700] + [700 + i + 1 for i in range(400)]
        hi = [min(h, 700) if i < 700 else h for i, h in enumerate(hi)]
    _span_case(cuda, _ops(), TYPES[op], lo, hi, 1100, heads, kv_heads, dh, cap, bias, seed=dh)


@pytest.mark.parametrize("op", ["bf16", "fp32"])
@pytest.mark.parametrize("heads,kv_heads,crossing", [(1, 1, 50), (2, 2, 50), (4, 2, 700)])
def test_span_more_row_blocks_than_one_list(cuda, op, heads, kv_heads, crossing):
    """40000 rows of short documents and one of `crossing` rows over row 32768; checked where the lists begin and end."""
    ops, dt, dh, n = _ops(), TYPES[op], 64, 40000
    rng, starts = random.Random(heads), [0]
    while starts[-1] < n:
        at = starts[-1]
        if at < 32768 - crossing // 2 <= at + 50:
            starts += [32768 - crossing // 2, 32768 - crossing // 2 + crossing]
        else:
            starts.append(min(n, at + rng.randint(1, 50)))
    lo = [a for a, b in zip(starts, starts[1:]) for _ in range(a, b)]
    lo, hi = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in (lo, range(1, n + 1)))
    g = torch.Generator().manual_seed(heads)
    q, dout = (_normal(g, n, heads * dh, dt=dt).to(cuda) for _ in range(2))
    k, v = (_normal(g, n, kv_heads * dh, dt=dt).to(cuda) for _ in range(2))
    how = dict(heads=heads, kv_heads=kv_heads, scale=dh ** -0.5)
    out, lse = ops.attn_span(q, k, v, lo, hi, **how)
    got = dict(zip(("dq", "dk", "dv"), ops.attn_span_grads(dout, q, k, v, out, lse, lo, hi, **how)), out=out, lse=lse)
    for near in (0, 32768 - 900, n - 900):
        a = max(x for x in starts if x <= near)
        b = min(x for x in starts if x >= min(a + 1500, n))
        want = span_reference(q[a:b], k[a:b], v[a:b], lo[a:b] - a, hi[a:b] - a, heads, kv_heads, dh ** -0.5, dout=dout[a:b])
        for name, x in got.items():
            check("%s from row %d" % (name, a), x[a:b], want[name])


@pytest.mark.parametrize("op", ["bf16", "fp32"])
@pytest.mark.parametrize("m,n", [(1, 1), (1, 200), (200, 1), (3, 0), (0, 5), (77, 500), (500, 77), (1025, 1300)])
def test_span_shapes_and_cross_attention(cuda, op, m, n):
    """Query rows over another buffer: random spans, some empty, some reaching outside (cut), in no order."""
    rng = random.Random(m * 1000 + n)
    lo = [rng.randint(-3, max(n, 1)) for _ in range(m)]
    hi = [a + rng.randint(-2, max(n, 1)) for a in lo]
    _span_case(cuda, _ops(), TYPES[op], lo, hi, n, 4, 2, 64, seed=m + n, bias=m == 77)


@pytest.mark.parametrize("op", ["bf16", "fp32"])
def test_span_long_rows(cuda, op):
    lo, hi = _documents(2100, 2100, "causal", 1)
    lo, hi = lo[:2000] + [0] * 100, hi[:2000] + [2100] * 100
    _span_case(cuda, _ops(), TYPES[op], lo, hi, 2100, 2, 1, 64, seed=9)


@pytest.mark.parametrize("op", ["bf16", "fp16", "fp32"])
def test_span_strided_rows(cuda, op):
    lo, hi = _documents(150, 60, "causal", 4)
    _span_case(cuda, _ops(), TYPES[op], lo, hi, 150, 4, 2, 64, seed=11, fused=True)


@pytest.mark.parametrize("op", ["bf16", "fp32"])
def test_span_large_scores(cuda, op):
    """Scores of several hundred: the running maximum has to carry them."""
    lo, hi = _documents(140, 140, "causal", 4)
    _span_case(cuda, _ops(), TYPES[op], lo, hi, 140, 2, 2, 64, seed=12, times=12.0)


@pytest.mark.parametrize("op", ["bf16", "fp32"])
def test_span_outputs_given_and_rows_behind(cuda, op):
    """Results go into the caller's strided buffers; what lies beside and behind the rows stays as it was."""
    ops, dt = _ops(), TYPES[op]
    lo, hi = _documents(60, 30, "causal", 2)
    g = torch.Generator().manual_seed(5)
    q, k, v, do = (_normal(g, 60, 128, dt=dt).to(cuda) for _ in range(4))
    lo, hi = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in (lo, hi))
    want, lse = ops.attn_span(q, k, v, lo, hi, heads=2)
    grads = ops.attn_span_grads(do, q, k, v, want, lse, lo, hi, heads=2)
    bufs = [torch.full((64, 160), 7.0, dtype=dt, device=cuda) for _ in range(4)]
    views = [b[:60, 16:144] for b in bufs]
    out, lse2 = ops.attn_span(q, k, v, lo, hi, heads=2, out=views[0])
    assert out is views[0] and torch.equal(lse2, lse)
    ops.attn_span_grads(do, q, k, v, views[0], lse, lo, hi, heads=2, dq=views[1], dk=views[2], dv=views[3])
    torch.cuda.synchronize()
    for b, x in zip(bufs, (want,) + grads):
        assert torch.equal(b[:60, 16:144], x)
        b[:60, 16:144] = 7.0
        assert bool((b == 7.0).all())


@pytest.mark.parametrize("op", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
@pytest.mark.parametrize("heads,m", [(2, 200), (64, 1100)])
def test_span_unseen_rows_may_hold_anything(cuda, op, poison, heads, m):
    """Padding rows between documents (seen by nobody) and query rows that see nothing hold NaN or infinities."""
    ops, dt = _ops(), TYPES[op]
    g = torch.Generator().manual_seed(6)
    docs = [(0, 37), (50, 64), (64, 65), (70, 150), (150, 190)]
    lo, hi = [0] * m, [0] * m
    for a, b in docs:
        for i in range(a, b):
            lo[i], hi[i] = a, i + 1
    q, k, v, do = (_normal(g, m, heads * 64, dt=dt).to(cuda) for _ in range(4))
    off = torch.tensor([h == 0 for h in hi], device=cuda)
    lo, hi = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in (lo, hi))
    want = span_reference(q, k, v, lo, hi, heads, heads, 0.125, dout=do)
    for t in (q, k, v, do):
        t[off] = poison
    out, lse = ops.attn_span(q, k, v, lo, hi, heads=heads, scale=0.125)
    check("out", out, want["out"])
    check("lse", lse, want["lse"])
    check("step", ops.attn_span_step(q, k, v, lo, hi, heads=heads, scale=0.125, max_keys=80), want["out"])
    if dt != torch.float16:
        for name, x in zip(("dq", "dk", "dv"), ops.attn_span_grads(do, q, k, v, out, lse, lo, hi, heads=heads, scale=0.125)):
            check(name, x, want[name])


@pytest.mark.parametrize("op", ["bf16", "fp32"])
@pytest.mark.parametrize("where", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("heads,m", [(2, 160), (64, 1100)])
def test_span_nan_reaches_its_own_document_only(cuda, op, where, heads, m):
    ops, dt = _ops(), TYPES[op]
    g = torch.Generator().manual_seed(7)
    lo, hi = _documents(m, 30, "document", 3, tail=0)
    bad = next(i for i in range(60, m) if hi[i] - lo[i] > 3)
    mine = torch.tensor([a == lo[bad] for a in lo], device=cuda)
    t = {n: _normal(g, m, heads * 64, dt=dt).to(cuda) for n in ("q", "k", "v", "dout")}
    lo, hi = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in (lo, hi))
    want = span_reference(t["q"], t["k"], t["v"], lo, hi, heads, heads, 0.125, dout=t["dout"])
    t[where][bad] = float("nan")
    out, lse = ops.attn_span(t["q"], t["k"], t["v"], lo, hi, heads=heads, scale=0.125)
    got = dict(zip(("dq", "dk", "dv"), ops.attn_span_grads(t["dout"], t["q"], t["k"], t["v"], out, lse, lo, hi, heads=heads, scale=0.125)))
    got.update(out=out, lse=lse)
    for name, x in got.items():
        check(name, x[~mine], (want[name][0][~mine], want[name][1][~mine]))
    seen = {"q": "out", "k": "out", "v": "out", "dout": "dq"}[where]
    assert bool(torch.isnan(got[seen][bad]).all())
    if where != "q":                                                # a NaN query row spoils itself, in the forward pass
        assert bool(torch.isnan(got["dv" if where == "dout" else "out"][mine]).all())


@pytest.mark.parametrize("op", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,cache,heads,kv_heads,dh,cap,bias", [
    (1, 300, 8, 8, 64, 0.0, False), (3, 1, 2, 1, 64, 0.0, False), (5, 5000, 8, 2, 64, 30.0, True), (17, 700, 4, 1, 128, 0.0, True),
    (40, 90, 4, 4, 32, 0.0, False), (2, 2049, 8, 1, 64, 5.0, False), (2, 515, 3, 3, 48, 0.0, True), (1, 3000, 4, 2, 8, 0.0, False),
    (3, 260, 16, 1, 24, 0.0, False)])
def test_span_step(cuda, op, rows, cache, heads, kv_heads, dh, cap, bias):
    """One token for each of `rows` requests; request 1 has an empty cache, and the hint may be far off."""
    ops, dt = _ops(), TYPES[op]
    g = torch.Generator().manual_seed(rows + cache)
    rng = random.Random(cache)
    n = rows * cache
    q = _normal(g, rows, heads * dh, dt=dt).to(cuda)
    k, v = (_normal(g, n, kv_heads * dh, dt=dt).to(cuda) for _ in range(2))
    lens = [rng.randint(1, cache) for _ in range(rows)]
    if rows > 1:
        lens[1] = 0
    lens[0] = cache
    lo = torch.tensor([i * cache for i in range(rows)], dtype=torch.int32, device=cuda)
    hi = lo + torch.tensor(lens, dtype=torch.int32, device=cuda)
    slopes = torch.rand(heads, generator=g).to(cuda) * 0.1 if bias else None
    how = dict(heads=heads, kv_heads=kv_heads, scale=dh ** -0.5, cap=cap, slopes=slopes)
    want = span_reference(q, k, v, lo, hi, heads, kv_heads, dh ** -0.5, cap, slopes)["out"]
    for hint in (cache, 0, 20 * cache + 7):
        check("hint %d" % hint, ops.attn_span_step(q, k, v, lo, hi, max_keys=hint, **how), want)
    check("rows form", ops.attn_span(q, k, v, lo, hi, **how)[0], want)


@pytest.mark.parametrize("op,heads,kv_heads", [("bf16", 8, 2), ("fp16", 2, 2), ("fp32", 4, 1)])
def test_span_step_captured_and_replayed(cuda, op, heads, kv_heads):
    """Tokens over growing caches by replays of one graph, with eager calls between."""
    ops, dt = _ops(), TYPES[op]
    g = torch.Generator().manual_seed(heads)
    rows, cache, dh = 3, 3000, 64
    q = _normal(g, rows, heads * dh, dt=dt).to(cuda)
    k, v = (_normal(g, rows * cache, kv_heads * dh, dt=dt).to(cuda) for _ in range(2))
    lo = torch.arange(rows, dtype=torch.int32, device=cuda) * cache
    hi = lo.clone()
    how = dict(heads=heads, kv_heads=kv_heads, scale=0.125, cap=20.0, max_keys=cache)
    ops.attn_span_step(q, k, v, lo, hi, **how)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.attn_span_step(q, k, v, lo, hi, **how)
    for n in (0, 1, 33, 600, 3000):
        hi.copy_(lo + n)
        q.copy_(_normal(g, rows, heads * dh, dt=dt))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.attn_span_step(q, k, v, lo, hi, **how)), n
        check("replay", out, span_reference(q, k, v, lo, hi, heads, kv_heads, 0.125, 20.0)["out"])


def test_span_offsets_beyond_32_bits(cuda):
    """A key buffer of more than 2^32 bytes and 2^31 elements, spans at its end."""
    ops = _ops()
    n, w = (1 << 25) + 300, 64
    k, v = (torch.zeros(n, w, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    g = torch.Generator().manual_seed(3)
    k[-200:], v[-200:] = _normal(g, 200, w, dt=torch.bfloat16).to(cuda), _normal(g, 200, w, dt=torch.bfloat16).to(cuda)
    q = _normal(g, 70, w, dt=torch.bfloat16).to(cuda)
    lo = torch.tensor([n - 200 + i for i in range(70)], dtype=torch.int32, device=cuda)
    hi = torch.tensor([n - i for i in range(70)], dtype=torch.int32, device=cuda)
    want = span_reference(q, k[-200:].contiguous(), v[-200:].contiguous(), lo - (n - 200), hi - (n - 200), 1, 1, 0.125)
    check("out", ops.attn_span(q, k, v, lo, hi, heads=1, scale=0.125)[0], want["out"])
    check("step", ops.attn_span_step(q, k, v, lo, hi, heads=1, scale=0.125, max_keys=200)[0:70], want["out"])


def test_span_gradients_against_differences(cuda):
    """fp32 gradients against central differences of the 64-bit forward formula along random directions."""
    ops = _ops()
    lo, hi = _documents(90, 40, "prefix", 5)
    g = torch.Generator().manual_seed(8)
    t = {n: _normal(g, 90, w, dt=torch.float32).to(cuda) for n, w in (("q", 128), ("k", 64), ("v", 64), ("dout", 128))}
    lo, hi = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in (lo, hi))
    slopes = torch.tensor([0.1, 0.05], device=cuda)
    pos = torch.arange(90, dtype=torch.int32, device=cuda)
    how = dict(heads=2, kv_heads=1, scale=0.3, cap=2.0, slopes=slopes, pos=pos)
    out, lse = ops.attn_span(t["q"], t["k"], t["v"], lo, hi, **how)
    grads = ops.attn_span_grads(t["dout"], t["q"], t["k"], t["v"], out, lse, lo, hi, **how)

    def value(**moved):
        x = {n: moved.get(n, t[n].double()) for n in "qkv"}
        o = span_reference(x["q"], x["k"], x["v"], lo, hi, 2, 1, 0.3, 2.0, slopes, pos)["out"][0]
        return float((o * t["dout"].double()).sum())

    HALF[torch.float64] = 2.0 ** -53
    for name, dx in zip("qkv", grads):
        way = torch.randn(t[name].shape, generator=g).to(cuda).double()
        step = 1e-5
        diff = (value(**{name: t[name].double() + step * way}) - value(**{name: t[name].double() - step * way})) / (2 * step)
        have = float((dx.double() * way).sum())
        # third derivatives times step^2 stay below 1e-8; fp32 gradients are off by 1e-5 of the sum of magnitudes at most
        assert abs(have - diff) <= 1e-5 * float((dx.double() * way).abs().sum()) + 1e-7, (name, have, diff)


# -------------------------------------------------------------------------------------------------- cross entropy
def _xent_case(cuda, ops, dt, m, v, d, smoothing, weights, seed=0, strided=False, times=1.0):
    g = torch.Generator().manual_seed(seed)
    pad = 16 if strided else 0
    h = _normal(g, m, d + pad, dt=dt, times=times).to(cuda)[:, :d]
    w = _normal(g, v, d + pad, dt=dt, times=2.0 * d ** -0.5).to(cuda)[:, :d]
    labels = torch.randint(0, v, (m,), generator=g).to(torch.int32)
    for i, bad in zip(range(1, m, 5), (-1, v, -100, v + 5) * m):
        labels[i] = bad
    labels = labels.to(cuda)
    gr = (torch.rand(m, generator=g) / m).to(cuda) if weights else None
    loss, lse = ops.linear_xent(h, w, labels, smoothing=smoothing)
    got = {"loss": loss, "lse": lse}
    if dt != torch.float16:
        got["dh"], got["dw"] = ops.linear_xent_grads(h, w, labels, lse, gr, smoothing=smoothing)
    torch.cuda.synchronize()
    want = xent_reference(h, w, labels, smoothing, gr)
    for name, x in got.items():
        check(name, x, want[name])
    return h, w, labels, gr, got


@pytest.mark.parametrize("op", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("m,v,d,smoothing,weights", [
    (1, 1, 64, 0.0, False), (1, 300, 64, 0.1, True), (97, 509, 64, 0.1, True), (130, 1000, 256, 0.0, False), (64, 64, 8, 0.2, True),
    (300, 4099, 512, 0.1, True), (777, 1, 128, 0.0, True), (20, 2, 40, 0.3, False), (500, 2050, 448, 0.0, True),
    (1111, 3001, 1024, 0.1, True), (33, 20011, 512, 0.05, True)])
def test_xent(cuda, op, m, v, d, smoothing, weights):
    _xent_case(cuda, _ops(), TYPES[op], m, v, d, smoothing, weights, seed=m + v)


@pytest.mark.parametrize("op", ["bf16", "fp32"])
def test_xent_many_pieces(cuda, op):
    """Enough rows and entries that the vocabulary is taken in several pieces."""
    _xent_case(cuda, _ops(), TYPES[op], 3001, 30011 if op == "bf16" else 18013, 128, 0.1, True, seed=2)


@pytest.mark.parametrize("op", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("m,v,d", [(700, 3600, 136), (700, 2600, 256), (601, 7003, 256), (2500, 6001, 256), (3001, 30011, 64),
                                   (9001, 70, 40), (70001, 2100, 64)])
def test_xent_more_work(cuda, op, m, v, d):
    """Sizes on both sides of the choices between the products' forms, their tiles and one or several pieces."""
    h, w, labels, gr, got = _xent_case(cuda, _ops(), TYPES[op], m, v, d, 0.1, True, seed=m, strided=True)
    if op == "fp16":
        return
    ops, off = _ops(), (labels < 0) | (labels >= v)
    h[off] = float("nan")
    loss, lse = ops.linear_xent(h, w, labels, smoothing=0.1)
    dh, dw = ops.linear_xent_grads(h, w, labels, lse, gr, smoothing=0.1)
    for x, y in ((loss, got["loss"]), (lse[~off], got["lse"][~off]), (dh, got["dh"]), (dw, got["dw"])):
        assert torch.equal(x, y)                     # rows without a label count nowhere, and sums have one order


def test_xent_partial_sums_of_pieces(cuda):
    """More partial sums of dh than are kept apart: the second piece adds to the first one's."""
    _xent_case(cuda, _ops(), torch.bfloat16, 262145, 700, 512, 0.1, True, seed=9)


@pytest.mark.parametrize("op", ["bf16", "fp32"])
@pytest.mark.parametrize("m,v,d,smoothing", [(300, 2, 64, 0.5), (300, 2, 64, 0.9), (300, 3, 64, 2 / 3), (300000, 3, 512, 0.9)])
def test_xent_smoothing_beyond_the_uniform_distribution(cuda, op, m, v, d, smoothing):
    """The label's own weight 1 - smoothing at or below the others'."""
    _xent_case(cuda, _ops(), TYPES[op], m, v, d, smoothing, True, seed=10)


@pytest.mark.parametrize("op", ["bf16", "fp32"])
def test_xent_two_million_rows(cuda, op):
    """More row tiles than a grid's second dimension would hold."""
    _xent_case(cuda, _ops(), TYPES[op], 2100003, 9, 8, 0.1, True, seed=8)


@pytest.mark.parametrize("op", ["bf16", "fp32"])
def test_xent_strided_and_large_logits(cuda, op):
    _xent_case(cuda, _ops(), TYPES[op], 150, 700, 256, 0.1, True, seed=3, strided=True)
    _xent_case(cuda, _ops(), TYPES[op], 150, 700, 256, 0.0, True, seed=4, times=30.0)


@pytest.mark.parametrize("op", ["bf16", "fp32"])
def test_xent_rows_without_a_label_may_hold_anything(cuda, op):
    ops, dt = _ops(), TYPES[op]
    h, w, labels, gr, _ = _xent_case(cuda, ops, dt, 200, 999, 128, 0.1, True, seed=5)
    want = xent_reference(h, w, labels, 0.1, gr)
    off = (labels < 0) | (labels >= 999)
    h[off] = float("nan")
    loss, lse = ops.linear_xent(h, w, labels, smoothing=0.1)
    dh, dw = ops.linear_xent_grads(h, w, labels, lse, gr, smoothing=0.1)
    check("loss", loss, want["loss"])
    check("dh", dh, want["dh"])
    check("dw", dw, want["dw"])


def test_xent_without_rows(cuda):
    ops = _ops()
    h, w = torch.empty(0, 64, device=cuda), torch.randn(77, 64, device=cuda)
    labels = torch.empty(0, dtype=torch.int32, device=cuda)
    loss, lse = ops.linear_xent(h, w, labels)
    dw = torch.full_like(w, 3.0)
    dh, dw = ops.linear_xent_grads(h, w, labels, lse, dw=dw)
    assert loss.shape == (0,) and dh.shape == (0, 64) and bool((dw == 0).all())


def test_xent_gradients_against_differences(cuda):
    ops = _ops()
    h, w, labels, gr, got = _xent_case(cuda, ops, torch.float32, 60, 333, 64, 0.1, True, seed=7)
    g = torch.Generator().manual_seed(1)
    HALF[torch.float64] = 2.0 ** -53
    for name, x in (("dh", h), ("dw", w)):
        way = torch.randn(x.shape, generator=g).to(cuda).double()

        def value(step):
            y = x.double() + step * way
            return float((xent_reference(y if name == "dh" else h.double(), y if name == "dw" else w.double(), labels, 0.1)["loss"][0] * gr.double()).sum())

        diff, have = (value(1e-5) - value(-1e-5)) / 2e-5, float((got[name].double() * way).sum())
        assert abs(have - diff) <= 1e-5 * float((got[name].double() * way).abs().sum()) + 1e-7, (name, have, diff)


# -------------------------------------------------------------------------------------------------- global norm
def _norm_ok(norm, tensors, scale=1.0):
    want = abs(scale) * math.sqrt(sum(float(t.double().square().sum()) for t in tensors))
    assert abs(float(norm) - want) <= want * 2 ** -23, (float(norm), want)
    return want


@pytest.mark.parametrize("op", ["bf16", "fp16", "fp32", "mixed"])
@pytest.mark.parametrize("sizes,max_norm,scale", [
    ([1], 0.5, 1.0), ([5, 0, 3], 1e9, 1.0), ([16384, 16385, 1, 40001], 1.0, 0.25), ([7] * 300, 2.0, -1.0), ([3000001], 10.0, 1.0),
    ([17] * 96 + [50000], 1.0, 1.0)])
def test_clip_global_norm(cuda, op, sizes, max_norm, scale):
    ops = _ops()
    g = torch.Generator().manual_seed(len(sizes))
    kinds = list(TYPES.values())
    ts = [_normal(g, n, dt=kinds[i % 3] if op == "mixed" else TYPES[op]).to(cuda) for i, n in enumerate(sizes)]
    _norm_ok(ops.global_norm(ts, grad_scale=scale), ts, scale)
    flat = torch.full((sum(sizes) + 1,), 9.0, device=cuda)          # odd offsets inside the flat buffer
    views = ops.split_flat(flat[:-1], ts)
    want = _norm_ok(ops.clip_global_norm(ops.TensorList(ts, out=views), max_norm, grad_scale=scale), ts, scale)
    f = scale * min(1.0, max_norm / want)
    for t, o in zip(ts, views):
        assert bool(((o.double() - t.double() * f).abs() <= t.double().abs() * abs(f) * 2 ** -22).all())
    assert float(flat[-1]) == 9.0
    before = [t.clone() for t in ts]
    _norm_ok(ops.clip_global_norm(ts, max_norm, grad_scale=scale), before, scale)          # in place
    for t, b in zip(ts, before):
        # fp16 results below 2^-14 are rounded to steps of 2^-24
        room = b.double().abs() * abs(f) * (HALF[t.dtype] + 2 ** -22) + (2.0 ** -25 if t.dtype == torch.float16 else 0.0)
        assert bool(((t.double() - b.double() * f).abs() <= room).all())


def test_clip_extreme_values(cuda):
    ops = _ops()
    big = [torch.full((5000,), 1e38, device=cuda), torch.full((3,), -2e38, device=cuda)]
    norm = ops.clip_global_norm(big, 1.0)
    assert math.isinf(float(norm)) or float(norm) > 1e39                 # 7e39 does not fit fp32: the norm reads inf
    assert all(bool(torch.isfinite(t).all()) and float(t.abs().max()) < 1.0 for t in big)
    small = [torch.full((100,), 1e-30, device=cuda)]
    _norm_ok(ops.global_norm(small), small)
    zero = [torch.zeros(10, device=cuda)]
    assert float(ops.clip_global_norm(zero, 1.0)) == 0.0 and bool((zero[0] == 0).all())
    for bad in (float("nan"), float("inf")):
        ts = [torch.ones(100, device=cuda), torch.ones(5, device=cuda)]
        ts[1][2] = bad
        norm = ops.clip_global_norm(ts, 1.0)
        assert not math.isfinite(float(norm)) and all(bool(torch.isnan(t).all()) for t in ts)
    assert float(ops.global_norm([torch.empty(0, device=cuda)])) == 0.0
    assert float(ops.clip_global_norm([torch.empty(0, device=cuda)], 1.0)) == 0.0


# -------------------------------------------------------------------------------------------------- together
def _train_step(ops, L, s, out_bufs=None):
    """One teacher-forced step of an attention layer under the vocabulary loss: forward, loss, gradients, clipping by the
    global norm, RMSProp on the flat master weights."""
    how = dict(heads=4, kv_heads=2, scale=s["scale"], cap=0.0)
    q, k, v = s["qkv"][:, :256], s["qkv"][:, 256:384], s["qkv"][:, 384:]
    out, lse = ops.attn_span(q, k, v, s["lo"], s["hi"], **how)
    loss, z = ops.linear_xent(out, s["w"], s["labels"], smoothing=0.1)
    dh, dw = ops.linear_xent_grads(out, s["w"], s["labels"], z, s["weight"], smoothing=0.1)
    dqkv = torch.empty_like(s["qkv"])
    ops.attn_span_grads(dh, q, k, v, out, lse, s["lo"], s["hi"], dq=dqkv[:, :256], dk=dqkv[:, 256:384], dv=dqkv[:, 384:], **how)
    flat = torch.empty(dw.numel() + dqkv.numel(), device=dw.device)
    norm = ops.clip_global_norm(ops.TensorList([dw, dqkv], out=ops.split_flat(flat, [dw, dqkv])), s["max_norm"])
    L.check(L.lib.nmtgan_rmsprop_update(s["master"].data_ptr(), s["ms"].data_ptr(), None, flat.data_ptr(), flat.numel(), 1e-3, 0.9,
                                        0.0, 1e-10, 1.0, 0.0, None, L.NMTGAN_F32, L.stream_ptr()), "rmsprop")
    return loss, dw, dqkv, flat, norm


def _train_state(cuda, dt, seed):
    g = torch.Generator().manual_seed(seed)
    lo, hi = _documents(250, 50, "causal", seed)
    s = {"qkv": _normal(g, 250, 512, dt=dt).to(cuda), "w": _normal(g, 1009, 256, dt=dt, times=0.1).to(cuda), "scale": 0.125,
         "lo": torch.tensor(lo, dtype=torch.int32, device=cuda), "hi": torch.tensor(hi, dtype=torch.int32, device=cuda),
         "labels": torch.randint(-1, 1009, (250,), generator=g).to(torch.int32).to(cuda), "weight": torch.full((250,), 1 / 250, device=cuda),
         "max_norm": 0.05}
    n = s["w"].numel() + s["qkv"].numel()
    s["master"], s["ms"] = torch.zeros(n, device=cuda), torch.ones(n, device=cuda)
    return s


@pytest.mark.parametrize("op", ["bf16", "fp32"])
def test_training_step_of_all_operators(cuda, op):
    """The run against autograd of the same formulas in 64 bits."""
    from nmt_gan_amd import _lib as L
    ops, s = _ops(), _train_state(cuda, TYPES[op], 3)
    loss, dw, dqkv, flat, norm = _train_step(ops, L, s)
    x, w = s["qkv"].double().requires_grad_(), s["w"].double().requires_grad_()
    q = x[:, :256].reshape(250, 4, 64).transpose(0, 1)
    k, v = (x[:, a:a + 128].reshape(250, 2, 64).transpose(0, 1).repeat_interleave(2, 0) for a in (256, 384))
    at = torch.arange(250, device=cuda)
    vis = (at >= s["lo"][:, None]) & (at < s["hi"][:, None])
    sc = (q @ k.transpose(1, 2) * 0.125).masked_fill(~vis, -1e300)
    p = torch.softmax(sc, -1) * vis.any(1)[:, None]
    o = (p @ v).transpose(0, 1).reshape(250, 256)
    if op == "bf16":                                                # the operator hands its rounded output on
        o = o + (o.detach().to(torch.bfloat16).double() - o.detach())
    logp = torch.log_softmax(o @ w.t(), -1)
    wanted = torch.full_like(logp, 0.1 / 1008).scatter(1, s["labels"].clamp(min=0).long()[:, None], 0.9)
    want = -(wanted * logp).sum(1) * (s["labels"] >= 0)
    (want * s["weight"]).sum().backward()
    # bf16: dz, dh, p, dr and the results are rounded by at most 2^-8 each, five roundings between the loss and dqkv whose
    # errors have no common sign; fp32: sums of at most 1009 terms
    tol = 5 * 2.0 ** -8 if op == "bf16" else 1009 * 2.0 ** -24
    for name, a, b in (("loss", loss, want), ("dw", dw, w.grad), ("dqkv", dqkv, x.grad)):
        off = float((a.double() - b.detach()).norm() / b.detach().norm())
        assert off <= tol, (name, off, tol)
    total = math.sqrt(float(dw.double().square().sum() + dqkv.double().square().sum()))
    assert abs(float(norm) - total) <= total * 2 ** -23
    f = min(1.0, 0.05 / total)
    both = torch.cat([dw.flatten(), dqkv.flatten()]).double()
    assert float((flat.double() - both * f).norm()) <= 2 ** -22 * f * total
    ms = 1 + (flat.double() ** 2 - 1) * 0.1
    step = 1e-3 * flat.double() / (ms + 1e-10).sqrt()
    assert float((s["master"].double() + step).norm()) <= 1e-5 * float(step.norm())


@pytest.mark.parametrize("op", ["bf16", "fp32"])
def test_training_step_captured_and_replayed(cuda, op):
    """Two captured steps that share torch's graph pool, replayed in turn with other inputs and eager work between, give
    the bits of the eager step every time."""
    from nmt_gan_amd import _lib as L
    ops, dt = _ops(), TYPES[op]
    states = [_train_state(cuda, dt, 3), _train_state(cuda, dt, 4)]
    _train_step(ops, L, states[0])                                  # warm
    torch.cuda.synchronize()
    pool, graphs, results = torch.cuda.graph_pool_handle(), [], []
    for s in states:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool, capture_error_mode="relaxed"):
            r = _train_step(ops, L, s)
        graphs.append(graph)
        results.append(r)
    for turn in range(3):
        for s, graph, r in zip(states, graphs, results):
            fresh = _train_state(cuda, dt, 10 + turn)
            for n in ("qkv", "w", "lo", "hi", "labels", "master", "ms"):
                s[n].copy_(fresh[n])
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in r] + [s["master"].clone()]
            want = list(_train_step(ops, L, fresh)) + [fresh["master"]]
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a, b), turn


def test_calls_on_two_streams(cuda):
    """The same calls on two side streams at once: results of both are those of one call after the other."""
    ops = _ops()
    from nmt_gan_amd import _lib as L
    s = [_train_state(cuda, torch.bfloat16, 20 + i) for i in range(2)]
    want = [_train_step(ops, L, dict(x, master=x["master"].clone(), ms=x["ms"].clone())) for x in s]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in s]
    got = []
    for x, st in zip(s, streams):
        with torch.cuda.stream(st):
            got.append(_train_step(ops, L, x))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


# -------------------------------------------------------------------------------------------------- refusals
def test_python_refusals(cuda):
    ops = _ops()
    q = torch.zeros(10, 128, device=cuda)
    i = torch.zeros(10, dtype=torch.int32, device=cuda)
    ok = dict(heads=2)
    ops.attn_span(q, q, q, i, i, **ok)
    bad = [
        lambda: ops.attn_span(q.cpu(), q, q, i, i, **ok), lambda: ops.attn_span(q.double(), q, q, i, i, **ok),
        lambda: ops.attn_span(q, q.half(), q, i, i, **ok), lambda: ops.attn_span(q, q, q[:9], i, i, **ok),
        lambda: ops.attn_span(q, q, q, i[:9], i, **ok), lambda: ops.attn_span(q, q, q, i.long(), i, **ok),
        lambda: ops.attn_span(q, q, q, i, i, heads=3), lambda: ops.attn_span(q, q, q, i, i, heads=2, kv_heads=4),
        lambda: ops.attn_span(q, q, q, i, i, heads=0), lambda: ops.attn_span(q, q, q, i, i, heads=32),
        lambda: ops.attn_span(q, q, q, i, i, heads=2, cap=-1.0), lambda: ops.attn_span(q, q, q, i, i, heads=2, scale=float("nan")),
        lambda: ops.attn_span(q.t(), q.t(), q.t(), i, i, **ok), lambda: ops.attn_span(q, q, q, i, i, slopes=i[:2], **ok),
        lambda: ops.attn_span(q, q, q, i, i, slopes=torch.zeros(3, device=cuda), **ok),
        lambda: ops.attn_span(q, q, q, i, i, out=torch.zeros(9, 128, device=cuda), **ok),
        lambda: ops.attn_span(torch.zeros(10 * 129 + 1, device=cuda)[1:1281].view(10, 128), q, q, i, i, **ok),
        lambda: ops.attn_span_step(q, q, q, i, i, max_keys=-1, **ok),
        lambda: ops.attn_span_grads(q.half(), q.half(), q.half(), q.half(), q.half(), q[:, :2], i, i, **ok),
        lambda: ops.attn_span_grads(q, q, q, q, q, q[:, :3], i, i, **ok), lambda: ops.attn_span_grads(q[:9], q, q, q, q, q[:, :2].contiguous(), i, i, **ok),
        lambda: ops.linear_xent(q, q[:, :64], i), lambda: ops.linear_xent(q, q, i.long()), lambda: ops.linear_xent(q, q, i, smoothing=1.0),
        lambda: ops.linear_xent(q, q[:1], i, smoothing=0.1), lambda: ops.linear_xent(q[:, :3], q[:, :3], i),
        lambda: ops.linear_xent_grads(q.half(), q.half(), i, q[:, 0].contiguous()), lambda: ops.linear_xent_grads(q, q, i, q[0]),
        lambda: ops.TensorList([]), lambda: ops.TensorList([q.t()]), lambda: ops.TensorList([q], out=[q.half()]),
        lambda: ops.TensorList([q], out=[q[:5]]), lambda: ops.TensorList([q, q.cpu()]), lambda: ops.clip_global_norm([q], 0.0),
        lambda: ops.clip_global_norm([q], float("inf")), lambda: ops.global_norm([q], grad_scale=float("nan")),
        lambda: ops.split_flat(q.flatten()[:7], [q]),
    ]
    for n, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            raise AssertionError("call %d was taken" % n)


def test_overlapping_lists_are_refused(cuda):
    ops = _ops()
    from nmt_gan_amd import NmtGanError
    x = torch.ones(100, device=cuda)
    for call in (lambda: ops.clip_global_norm([x, x], 1.0), lambda: ops.clip_global_norm([x[:60], x[50:]], 1.0),
                 lambda: ops.clip_global_norm(ops.TensorList([x[:50], x[50:]], out=[x[25:75], torch.empty(50, device=cuda)]), 1.0)):
        with pytest.raises(NmtGanError):
            call()
    ops.global_norm([x, x])                                         # reading twice is fine
    assert float(ops.global_norm([x, x])) == pytest.approx(math.sqrt(200.0))
