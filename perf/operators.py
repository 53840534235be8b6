"""What the training and serving operators of nmt_gan_amd.ops cost, case by case.

Three operators, each in its plain form (elementary torch operations in 32 bits) and as the framework's own calls:

  attention   span attention: every query row sees the keys [lo, hi) of a packed key buffer - forward, gradients, and
              the form for single tokens over a long cache
  xent        softmax cross entropy of hidden rows against a vocabulary table, with label smoothing, and its gradient
  clip        global gradient norm over a list of tensors, and the clipped gradients in one flat fp32 buffer
"""
import math
import random

import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # a training batch at the width of the benchmark: sentences of at most 50 tokens, packed
        {"name": "attn train sentences", "op": "attn", "rows": 2048, "longest": 50, "layout": 1, "d": 512, "heads": 8,
         "kv_heads": 8, "mask": "causal", "cap": 0.0, "bias": False, "type": "bf16", "grads": True},
        # packed documents of very different lengths, capped scores and a distance bias
        {"name": "attn train documents", "op": "attn", "rows": 8192, "longest": 4096, "layout": 2, "d": 512, "heads": 8,
         "kv_heads": 8, "mask": "causal", "cap": 30.0, "bias": True, "type": "bf16", "grads": True},
        # the parity tier's training step at the small generator's width, source part visible to all (prefix mask)
        {"name": "attn train fp32 prefix", "op": "attn", "rows": 999, "longest": 160, "layout": 3, "d": 256, "heads": 4,
         "kv_heads": 4, "mask": "prefix", "cap": 0.0, "bias": False, "type": "fp32", "grads": True},
        # prompts read before decoding: shared key heads of width 128
        {"name": "attn prompts shared heads", "op": "attn", "rows": 5000, "longest": 3000, "layout": 4, "d": 1024, "heads": 8,
         "kv_heads": 2, "mask": "causal", "cap": 0.0, "bias": False, "type": "fp16", "grads": False},
        # one token for each of 48 requests whose caches hold up to 16384 tokens
        {"name": "attn step long caches", "op": "step", "rows": 48, "cache": 16384, "layout": 5, "d": 512, "heads": 8,
         "kv_heads": 2, "cap": 30.0, "bias": False, "type": "fp16"},
        # one token of one request with a short cache: latency
        {"name": "attn step one short", "op": "step", "rows": 1, "cache": 300, "layout": 6, "d": 512, "heads": 8,
         "kv_heads": 8, "cap": 0.0, "bias": True, "type": "bf16"},
        # the loss of a training batch of the generator over its 32000 tokens, with label smoothing
        {"name": "xent train batch", "op": "xent", "rows": 3200, "vocab": 32000, "d": 512, "smoothing": 0.1, "ignored": 0.05,
         "type": "bf16", "grads": True},
        # the same loss for a large packed batch, a wider model and an odd vocabulary
        {"name": "xent train large", "op": "xent", "rows": 8000, "vocab": 50257, "d": 1024, "smoothing": 0.0, "ignored": 0.0,
         "type": "bf16", "grads": True},
        # scoring a held-out set (no gradient)
        {"name": "xent score", "op": "xent", "rows": 1601, "vocab": 32000, "d": 512, "smoothing": 0.0, "ignored": 0.1,
         "type": "fp16", "grads": False},
        # the parity tier at the smallest configuration of the tests
        {"name": "xent train fp32 small", "op": "xent", "rows": 97, "vocab": 509, "d": 64, "smoothing": 0.1, "ignored": 0.1,
         "type": "fp32", "grads": True},
        # gradients of the whole six-block generator (16 bits each) into the flat fp32 buffer of the optimizer
        {"name": "clip generator", "op": "clip", "d": 512, "blocks": 6, "vocab": 32000, "odd": False, "max_norm": 1.0,
         "type": "bf16"},
        # a handful of small tensors of odd sizes: latency
        {"name": "clip small", "op": "clip", "d": 60, "blocks": 1, "vocab": 77, "odd": True, "max_norm": 5.0, "type": "fp32"},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "step", "step", "xent", "xent", "clip"])
    if op == "clip":
        return {"op": "clip", "d": rng.choice([60, 64, 128, 250, 256, 500, 512]), "blocks": rng.randint(1, 6),
                "vocab": _spread(rng, 70, 32000), "odd": rng.random() < 0.5, "max_norm": round(rng.uniform(0.5, 20.0), 3),
                "type": rng.choice(["bf16", "fp16", "fp32"])}
    if op == "xent":
        grads = rng.random() < 0.7
        kind = rng.choice(["bf16", "bf16", "fp32"]) if grads else rng.choice(["fp16", "bf16", "fp32"])
        small = kind == "fp32"
        return {"op": "xent", "rows": _spread(rng, 1, 900 if small else 6000), "vocab": _spread(rng, 300, 9000 if small else 40000),
                "d": rng.choice([64, 128, 256, 512] if small else [64, 128, 256, 448, 512, 768, 1024]),
                "smoothing": rng.choice([0.0, 0.1, 0.2]), "ignored": rng.choice([0.0, 0.1, 0.4]), "type": kind, "grads": grads}
    width = rng.choice([32, 64, 128])
    heads = rng.choice([h for h in (2, 4, 8) if h * width <= 1024])
    kv_heads = rng.choice([h for h in (1, 2, 4, 8) if h <= heads])
    if op == "step":
        rows = _spread(rng, 1, 48)
        return {"op": "step", "rows": rows, "cache": _spread(rng, 20, min(16384, 400000 // rows)), "layout": rng.randint(10, 10 ** 6),
                "d": heads * width, "heads": heads, "kv_heads": kv_heads, "cap": rng.choice([0.0, 0.0, 20.0]),
                "bias": rng.random() < 0.3, "type": rng.choice(["bf16", "fp16", "fp32"])}
    grads = rng.random() < 0.6
    kind = rng.choice(["bf16", "bf16", "fp32"]) if grads else rng.choice(["bf16", "fp16", "fp32"])
    # one-row documents have no gradient of their scores at all: a training batch holds longer ones too
    least = 16 if grads else 1
    rows = _spread(rng, least, 1200 if kind == "fp32" else 6000)
    return {"op": "attn", "rows": rows, "longest": _spread(rng, min(least, 8), max(2, rows)), "layout": rng.randint(10, 10 ** 6),
            "d": heads * width, "heads": heads, "kv_heads": kv_heads, "mask": rng.choice(["causal", "causal", "prefix", "document"]),
            "cap": rng.choice([0.0, 0.0, 20.0, 50.0]), "bias": rng.random() < 0.3, "type": kind, "grads": grads}


# ------------------------------------------------------------------------------------------------------- inputs
def _spans(case):
    """(lo, hi) of every query row of a packed buffer: documents of 1 to `longest` rows one behind the other, the last
    rows (one in forty) belong to none."""
    rng = random.Random(case["layout"])
    rows, lo, hi = case["rows"], [], []
    used = rows - rows // 40
    while len(lo) < used:
        first = len(lo)
        n = min(used - first, max(1, min(case["longest"], _spread(rng, max(1, case["longest"] / 16), case["longest"]))))
        seen = rng.randint(0, n) if case["mask"] == "prefix" else n if case["mask"] == "document" else 0
        lo += [first] * n
        hi += [first + max(i + 1, seen) for i in range(n)]
    return lo + [0] * (rows - used), hi + [0] * (rows - used)


def _lengths(case):
    rng = random.Random(case["layout"])
    return [max(1, int(case["cache"] * rng.uniform(0.3, 1.0))) for _ in range(case["rows"])]


def _slopes(heads, device):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], device=device, dtype=torch.float32)


def _sizes(case):
    d, v, more = case["d"], case["vocab"], 1 if case["odd"] else 0
    block = [(3 * d, d), (3 * d + more,), (d, d), (d,), (4 * d, d), (4 * d + more,), (d, 4 * d), (d,), (d,), (d,), (d,), (d,)]
    cross = [(d, d), (d + more,), (2 * d, d), (2 * d,), (d, d), (d,), (d,), (d,)]
    return [(v, d), (v, d), (v, d + more)] + case["blocks"] * block + case["blocks"] * (block + cross)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    kind = TYPES[case["type"]]

    def normal(*shape, times=1.0, kind=kind):
        return (torch.randn(*shape, generator=g, device=DEVICE) * times).to(kind)

    def whole(values):
        return torch.tensor(values, device=DEVICE, dtype=torch.int32)

    s = dict(case)
    if case["op"] == "clip":
        s["grads"] = [normal(*shape, times=0.02) for shape in _sizes(case)]
        s["flat"] = torch.zeros(sum(t.numel() for t in s["grads"]), device=DEVICE)
        if own:
            from nmt_gan_amd import ops
            s["list"] = ops.TensorList(s["grads"], out=ops.split_flat(s["flat"], s["grads"]))
        return s
    if case["op"] == "xent":
        n, v, d = case["rows"], case["vocab"], case["d"]
        s["h"], s["w"] = normal(n, d), normal(v, d, times=2.0 * d ** -0.5)
        labels = torch.randint(0, v, (n,), generator=g, device=DEVICE)
        out = torch.rand(n, generator=g, device=DEVICE) < case["ignored"]
        s["labels"] = torch.where(out, torch.full_like(labels, -1), labels).to(torch.int32)
        s["weight"] = torch.full((n,), 1.0 / n, device=DEVICE)
        return s
    width = case["d"] // case["heads"]
    s["scale"] = width ** -0.5
    s["slopes"] = _slopes(case["heads"], DEVICE) if case["bias"] else None
    if case["op"] == "step":
        lengths = _lengths(case)
        keys = case["rows"] * case["cache"]
        s["lo"] = whole([i * case["cache"] for i in range(case["rows"])])
        s["hi"] = whole([i * case["cache"] + n for i, n in enumerate(lengths)])
        s["q"] = normal(case["rows"], case["d"])
    else:
        lo, hi = _spans(case)
        keys = case["rows"]
        s["lo"], s["hi"] = whole(lo), whole(hi)
        s["pos"] = torch.arange(keys, device=DEVICE, dtype=torch.int32)
        s["q"] = normal(case["rows"], case["d"])
        s["dout"] = normal(case["rows"], case["d"], times=0.01)
    s["k"], s["v"] = normal(keys, case["kv_heads"] * width), normal(keys, case["kv_heads"] * width)
    return s


# ------------------------------------------------------------------------------------------------- plain forms
def _by_head(t, heads):
    return t.float().view(t.shape[0], heads, -1).transpose(0, 1).contiguous()


def _probabilities(s, r, pos, at, visible, slopes):
    """p, lse and the factor d(score)/d(r) of raw scores r."""
    slope = 1.0
    if s["cap"]:
        t = torch.tanh(r / s["cap"])
        r, slope = s["cap"] * t, 1.0 - t * t
    if slopes is not None:
        r = r - slopes * (pos - at).abs()
    r = torch.where(visible, r, -math.inf)
    top = r.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = torch.where(visible, torch.exp(r - top), 0.0)
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, torch.ones_like(total)), (top + torch.log(total)).squeeze(-1), slope


def _plain_attn(s):
    heads, shared = s["heads"], s["heads"] // s["kv_heads"]
    q, k, v = _by_head(s["q"], heads), _by_head(s["k"], s["kv_heads"]), _by_head(s["v"], s["kv_heads"])
    k, v = k.repeat_interleave(shared, 0), v.repeat_interleave(shared, 0)
    at = torch.arange(k.shape[1], device=k.device)
    visible = (at >= s["lo"][:, None]) & (at < s["hi"][:, None])
    slopes = None if s["slopes"] is None else s["slopes"][:, None, None]
    r = torch.matmul(q, k.transpose(1, 2).contiguous()) * s["scale"]
    p, lse, slope = _probabilities(s, r, s["pos"][:, None], at, visible, slopes)
    del r

    def rows(t, n=heads):
        t = t.view(n, heads // n, t.shape[1], -1).sum(1)
        return t.transpose(0, 1).reshape(t.shape[1], -1).to(s["q"].dtype)

    answer = {"out": rows(torch.matmul(p, v)), "lse": lse.transpose(0, 1).contiguous()}
    if s["grads"]:
        do = _by_head(s["dout"], heads)
        dv = torch.matmul(p.transpose(1, 2).contiguous(), do)
        dp = torch.matmul(do, v.transpose(1, 2).contiguous())
        dr = p * (dp - (p * dp).sum(-1, keepdim=True)) * slope * s["scale"]
        answer["dq"] = rows(torch.matmul(dr, k))
        answer["dk"] = rows(torch.matmul(dr.transpose(1, 2).contiguous(), q), s["kv_heads"])
        answer["dv"] = rows(dv, s["kv_heads"])
    return answer


def _plain_step(s):
    n, heads, kv = s["rows"], s["heads"], s["kv_heads"]
    q = s["q"].float().view(n, kv, heads // kv, -1)
    k = s["k"].float().view(n, s["cache"], kv, -1).permute(0, 2, 3, 1).contiguous()
    v = s["v"].float().view(n, s["cache"], kv, -1).transpose(1, 2).contiguous()
    at = torch.arange(s["cache"], device=q.device)
    length = (s["hi"] - s["lo"])[:, None, None, None]
    slopes = None if s["slopes"] is None else s["slopes"].view(1, kv, heads // kv, 1)
    p, _, _ = _probabilities(s, torch.matmul(q, k) * s["scale"], length - 1, at, at < length, slopes)
    return {"out": torch.matmul(p, v).reshape(n, -1).to(s["q"].dtype)}


def _plain_xent(s):
    h, w, v = s["h"].float(), s["w"].float(), s["vocab"]
    low = s["smoothing"] / (v - 1)
    high = 1.0 - s["smoothing"] - low
    used = s["labels"] >= 0
    label = s["labels"].clamp(min=0).long()[:, None]
    z = torch.matmul(h, w.t())
    top = z.amax(1, keepdim=True)
    lse = (top + torch.log(torch.exp(z - top).sum(1, keepdim=True))).squeeze(1)
    loss = lse - high * z.gather(1, label).squeeze(1)
    if low:
        loss = loss - low * z.sum(1)
    answer = {"loss": torch.where(used, loss, torch.zeros_like(loss)), "lse": lse}
    if s["grads"]:
        dz = torch.exp(z - lse[:, None]) - low
        dz.scatter_add_(1, label, torch.full_like(label, -high, dtype=torch.float32))
        dz = dz * torch.where(used, s["weight"], torch.zeros_like(s["weight"]))[:, None]
        answer["dh"] = torch.matmul(dz, w).to(s["h"].dtype)
        answer["dw"] = torch.matmul(dz.t(), h).to(s["h"].dtype)
    return answer


def _plain_clip(s):
    g = torch.cat([t.reshape(-1).float() for t in s["grads"]])
    norm = g.double().square().sum().sqrt().float()
    return {"norm": norm, "flat": g * torch.clamp(s["max_norm"] / norm, max=1.0)}


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    s = state
    if not own:
        return {"attn": _plain_attn, "step": _plain_step, "xent": _plain_xent, "clip": _plain_clip}[s["op"]](s)
    from nmt_gan_amd import ops
    if s["op"] == "clip":
        norm = ops.clip_global_norm(s["list"], s["max_norm"])
        return {"norm": norm, "flat": s["flat"]}
    if s["op"] == "xent":
        loss, lse = ops.linear_xent(s["h"], s["w"], s["labels"], smoothing=s["smoothing"])
        answer = {"loss": loss, "lse": lse}
        if s["grads"]:
            answer["dh"], answer["dw"] = ops.linear_xent_grads(s["h"], s["w"], s["labels"], lse, s["weight"],
                                                               smoothing=s["smoothing"])
        return answer
    how = {"heads": s["heads"], "kv_heads": s["kv_heads"], "scale": s["scale"], "cap": s["cap"], "slopes": s["slopes"]}
    if s["op"] == "step":
        return {"out": ops.attn_span_step(s["q"], s["k"], s["v"], s["lo"], s["hi"], max_keys=s["cache"], **how)}
    how["pos"] = s["pos"]
    out, lse = ops.attn_span(s["q"], s["k"], s["v"], s["lo"], s["hi"], **how)
    answer = {"out": out, "lse": lse}
    if s["grads"]:
        answer["dq"], answer["dk"], answer["dv"] = ops.attn_span_grads(s["dout"], s["q"], s["k"], s["v"], out, lse, s["lo"],
                                                                       s["hi"], **how)
    return answer


# ------------------------------------------------------------------------------------------------ what it costs
def work(case):
    size = 4 if case["type"] == "fp32" else 2
    if case["op"] == "clip":
        n = sum(math.prod(shape) for shape in _sizes(case))
        return {"bytes": n * (size + 4), "flops": 3 * n}
    if case["op"] == "xent":
        n, v, d = case["rows"], case["vocab"], case["d"]
        both = 2 if case["grads"] else 1
        return {"bytes": both * size * (n + v) * d + 16 * n, "flops": (6 if case["grads"] else 2) * n * v * d}
    kv = case["d"] // case["heads"] * case["kv_heads"]
    if case["op"] == "step":
        seen = sum(_lengths(case))
        return {"bytes": size * (2 * case["rows"] * case["d"] + 2 * seen * kv), "flops": 4 * seen * case["d"]}
    lo, hi = _spans(case)
    seen = sum(b - a for a, b in zip(lo, hi))
    rows = case["rows"]
    if case["grads"]:
        return {"bytes": size * rows * (4 * case["d"] + 4 * kv) + 4 * rows * case["heads"], "flops": 14 * seen * case["d"]}
    return {"bytes": size * rows * (2 * case["d"] + 2 * kv) + 4 * rows * case["heads"], "flops": 4 * seen * case["d"]}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        parts = [t.double().flatten() for t in s["grads"]]
        norm = math.sqrt(sum(float(torch.dot(t, t)) for t in parts))
        return {"norm": torch.tensor(norm, dtype=torch.float64), "flat": torch.cat(parts) * min(1.0, case["max_norm"] / norm)}
    if case["op"] == "xent":
        return _exact_xent(case, s)
    width, shared = case["d"] // case["heads"], case["heads"] // case["kv_heads"]
    q, k, v = (s[x].double() for x in "qkv")
    step = case["op"] == "step"
    out = torch.zeros(case["rows"], case["d"], dtype=torch.float64, device=q.device)
    lse = torch.full((case["rows"], case["heads"]), -math.inf, dtype=torch.float64, device=q.device)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    lo, hi = s["lo"].tolist(), s["hi"].tolist()
    # runs of rows that start at the same key are one document (or one request); the rows behind them see nothing
    first = 0
    while first < case["rows"] and hi[first] > lo[first]:
        last = first
        while last < case["rows"] and lo[last] == lo[first] and hi[last] > lo[last]:
            last += 1
        mine, keys = slice(first, last), slice(lo[first], max(hi[first:last]))
        at = torch.arange(keys.start, keys.stop, device=q.device)
        where = s["hi"][mine].long() - 1 if step else s["pos"][mine].long()
        hidden = at[None, :] >= s["hi"][mine, None]
        for h in range(case["heads"]):
            a, b = slice(h * width, (h + 1) * width), slice(h // shared * width, (h // shared + 1) * width)
            x = q[mine, a] @ k[keys, b].t() * s["scale"]
            turn = torch.ones_like(x)
            if case["cap"]:
                turn = 1.0 / torch.cosh(x / case["cap"]) ** 2
                x = case["cap"] * torch.tanh(x / case["cap"])
            if case["bias"]:
                x = x - float(s["slopes"][h]) * (where[:, None] - at[None, :]).abs()
            x = x.masked_fill(hidden, -math.inf)
            lse[mine, h] = torch.logsumexp(x, 1)
            p = torch.exp(x - lse[mine, h, None])
            out[mine, a] = p @ v[keys, b]
            if not step and case["grads"]:
                do = s["dout"][mine, a].double()
                dv[keys, b] += p.t() @ do
                dx = p * (do @ v[keys, b].t() - (do * out[mine, a]).sum(1, keepdim=True)) * turn * s["scale"]
                dq[mine, a] = dx @ k[keys, b]
                dk[keys, b] += dx.t() @ q[mine, a]
        first = last
    if step:
        return {"out": out}
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv} if case["grads"] else {"out": out, "lse": lse}


def _exact_xent(case, s):
    """Blocks of rows, so that the logits of one block at a time are held in 64 bits."""
    n, v = case["rows"], case["vocab"]
    w = s["w"].double()
    loss, lse = torch.zeros(n, dtype=torch.float64, device=w.device), torch.zeros(n, dtype=torch.float64, device=w.device)
    dh, dw = torch.zeros(n, case["d"], dtype=torch.float64, device=w.device), torch.zeros_like(w)
    for first in range(0, n, 1024):
        part = slice(first, min(n, first + 1024))
        h, label = s["h"][part].double(), s["labels"][part].long()
        used = label >= 0
        wanted = torch.full((h.shape[0], v), case["smoothing"] / (v - 1), dtype=torch.float64, device=w.device)
        wanted[torch.arange(h.shape[0], device=w.device), label.clamp(min=0)] = 1.0 - case["smoothing"]
        z = h @ w.t()
        lse[part] = torch.logsumexp(z, 1)
        loss[part] = (lse[part] - (wanted * z).sum(1)) * used
        if case["grads"]:
            dz = (torch.exp(z - lse[part, None]) - wanted) * (used * s["weight"][part].double())[:, None]
            dh[part] = dz @ w
            dw += dz.t() @ h
    return {"loss": loss, "lse": lse, "dh": dh, "dw": dw} if case["grads"] else {"loss": loss, "lse": lse}
