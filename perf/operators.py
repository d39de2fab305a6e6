"""The operators around the sparse layers of a training step, as cases to measure.

A case is one call of one of them, at one size:

  loss   the language-model head and its loss, linear_cross_entropy: `train` is the loss with
         the gradients of the hidden states and of the head, `score` the loss of every token
         (no gradient), as when candidate tokens are scored
  norm   residual_norm, what stands between two blocks: r = x + scale * gate * post(branch),
         y = pre(r), with LayerNorm or RMSNorm before and, if asked for, after the block:
         `train` is forward plus backward, `infer` forward under no_grad
  adamw  one AdamW step over a list of tensors, moments in 32 or in 8 bits
  carry  moments that follow their weights after a SET / RigL rewrite of a padded-CSR matrix

Where `own` is false the same is computed in plain torch, in 32 bits. `exact` states it in 64.
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F

own = False

DEV = "cuda"
PADDING = 0.2  # spare capacity of a padded-CSR row
BLOCK = 256    # elements that share one scale of an 8-bit moment
IGNORE = -100
LR, BETA1, BETA2, EPS, DECAY, STEP = 1e-3, 0.9, 0.95, 1e-8, 0.1, 1000
NORM_EPS = 1e-5
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def listed():
    return [
        # the 10M char-GPT's head over its training batch of 8192 tokens: 65 characters
        {"name": "loss_char_train", "kind": "loss", "mode": "train", "n": 8192, "d": 384, "v": 65,
         "ignored": 0.0, "dtype": "float32"},
        # a word-piece vocabulary on the 60M mini-GPT's width; packed prompts whose instruction
        # part (three tokens in ten) carries no loss, an odd number of tokens
        {"name": "loss_32k_train", "kind": "loss", "mode": "train", "n": 4001, "d": 768,
         "v": 32000, "ignored": 0.3, "dtype": "float32"},
        # a wide model's head under mixed precision: the largest
        {"name": "loss_100k_train_bf16", "kind": "loss", "mode": "train", "n": 8192, "d": 4096,
         "v": 100000, "ignored": 0.0, "dtype": "bfloat16"},
        # eight candidate tokens scored while generating
        {"name": "loss_32k_score_8", "kind": "loss", "mode": "score", "n": 8, "d": 768,
         "v": 32000, "ignored": 0.0, "dtype": "float32"},
        # one token each of eight sequences being generated: where latency counts
        {"name": "norm_decode_8", "kind": "norm", "mode": "infer", "b": 8, "t": 1, "d": 768,
         "norm": "layer", "post": False, "gate": "none", "cols": False, "dtype": "float32"},
        # between two blocks of the 10M char-GPT, whose sparse layers keep activations
        # feature-major
        {"name": "norm_10m_train", "kind": "norm", "mode": "train", "b": 32, "t": 256, "d": 384,
         "norm": "layer", "post": False, "gate": "none", "cols": True, "dtype": "float32"},
        # a wide block with norms before and after it and a gate of each sequence
        {"name": "norm_4096_gate_train_bf16", "kind": "norm", "mode": "train", "b": 8, "t": 2048,
         "d": 4096, "norm": "rms", "post": True, "gate": "sequence", "cols": False,
         "dtype": "bfloat16"},
        # the optimizer of the 784 -> 512 -> 10 MLP
        {"name": "adamw_mlp", "kind": "adamw", "model": "mlp", "k": 784, "h": 512, "m": 10,
         "bits": 32, "dtype": "float32"},
        # the optimizer of the whole 10M char-GPT: 53 tensors from 384 to 159252 elements
        {"name": "adamw_10m", "kind": "adamw", "model": "gpt", "d": 384, "f": 1536, "layers": 6,
         "vocab": 65, "ctx": 256, "bits": 32, "dtype": "float32"},
        # four large sparse layers (16384 x 16384 at 95%) with 8-bit moments
        {"name": "adamw_4x16m_8bit", "kind": "adamw", "model": "flat", "tensors": 4,
         "size": 16113000, "bits": 8, "dtype": "float32"},
        # after a SET rewrite of the 60M mini-GPT's FFN-up
        {"name": "carry_ffn_up", "kind": "carry", "m": 3072, "k": 768, "sparsity": 0.9,
         "rows": "uniform", "bits": 32},
        # after a RigL rewrite of the benchmark's largest layer, long-tailed rows, 8-bit moments
        {"name": "carry_16k_95_8bit", "kind": "carry", "m": 16384, "k": 16384, "sparsity": 0.95,
         "rows": "zipf", "bits": 8},
    ]


# ───────────────────────────── drawn cases ─────────────────────────────

def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size of [lo, hi]: half the time a multiple of 64 where one fits, else any."""
    v = _log_int(rng, lo, hi)
    if rng.random() < 0.5 and v >= 64:
        v = min(hi, 64 * max(1, round(v / 64)))
    return v


def draw(rng):
    kind = rng.choice(["loss"] * 4 + ["norm"] * 4 + ["adamw"] * 3 + ["carry"])
    if kind == "loss":
        mode = rng.choice(["train", "train", "score"])
        return {"kind": kind, "mode": mode, "n": _size(rng, 1 if mode == "score" else 16, 8192),
                "d": _size(rng, 64, 4096), "v": _size(rng, 65, 100000),
                "ignored": rng.choice([0.0, 0.0, 0.3, 0.7]),
                "dtype": rng.choice(["float32", "bfloat16"])}
    if kind == "norm":
        mode = rng.choice(["train", "train", "infer"])
        c = {"kind": kind, "mode": mode, "b": _log_int(rng, 1, 32), "t": _log_int(rng, 1, 2048),
             "d": _size(rng, 64, 8192), "norm": rng.choice(["layer", "rms"]),
             "post": rng.random() < 0.5,
             "gate": rng.choice(["none", "feature", "sequence", "element"]),
             "cols": rng.random() < 0.4, "dtype": rng.choice(["float32", "bfloat16"])}
        while c["b"] * c["t"] * c["d"] > 8 * 2048 * 4096:
            c["t"] = (c["t"] + 1) // 2
        return c
    if kind == "adamw":
        model = rng.choice(["mlp", "gpt", "flat"])
        bits, dtype = rng.choice([8, 32]), rng.choice(["float32", "float32", "bfloat16"])
        c = {"kind": kind, "model": model, "bits": bits, "dtype": dtype}
        if model == "mlp":
            c |= {"k": _size(rng, 64, 1024), "h": _size(rng, 64, 1024), "m": _size(rng, 10, 100)}
        elif model == "gpt":
            d = _size(rng, 64, 1024)
            c |= {"d": d, "f": 4 * d, "layers": rng.randint(1, 6), "vocab": _size(rng, 65, 32000),
                  "ctx": _size(rng, 64, 1024)}
        else:
            c |= {"tensors": rng.randint(1, 16), "size": _size(rng, 300, 4000000)}
        return c
    return {"kind": kind, "m": _size(rng, 64, 8192), "k": _size(rng, 64, 8192),
            "sparsity": rng.choice([0.7, 0.9, 0.95, 0.99]),
            "rows": rng.choice(["uniform", "zipf"]), "bits": rng.choice([8, 32])}


# ───────────────────────────── inputs ─────────────────────────────

def _gen(seed, part):
    return torch.Generator(device=DEV).manual_seed(seed * 64 + part)


def _normal(shape, seed, part, scale=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=_gen(seed, part), device=DEV) * scale).to(dtype)


def _loss_inputs(case, seed):
    """Normalised hidden states that lean towards their target's row of the head, as a trained
    model's do; ignored tokens at random places."""
    n, d, v, dt = case["n"], case["d"], case["v"], DTYPES[case["dtype"]]
    w = _normal((v, d), seed, 1, 2.0 / math.sqrt(d))
    target = torch.randint(0, v, (n,), generator=_gen(seed, 2), device=DEV)
    h = _normal((n, d), seed, 3) + 1.5 * w[target]
    skip = torch.rand(n, generator=_gen(seed, 4), device=DEV) < case["ignored"]
    return h.to(dt), w.to(dt), target.masked_fill(skip, IGNORE)


def _columns(t):
    """The same N x D values, stored feature by feature."""
    return t.t().contiguous().t()


def _norm_inputs(case, seed):
    b, t, d, dt = case["b"], case["t"], case["d"], DTYPES[case["dtype"]]
    n, layer = b * t, case["norm"] == "layer"
    part = iter(range(1, 20))

    def rows(scale=1.0):
        return _normal((n, d), seed, next(part), scale, dt)

    def vector(mean, scale):
        return (mean + _normal((d,), seed, next(part), scale)).to(dt)

    s = {"x": rows(2.0), "u": rows(), "w": vector(1.0, 0.1),
         "b": vector(0.0, 0.1) if layer else None,
         "pw": vector(1.0, 0.1) if case["post"] else None,
         "pb": vector(0.0, 0.1) if case["post"] and layer else None,
         "gate": {"none": None, "feature": (d,), "sequence": (b, 1, d),
                  "element": (b, t, d)}[case["gate"]]}
    if s["gate"] is not None:
        s["gate"] = _normal(s["gate"], seed, next(part), 0.5, dt)
    s["dy"], s["dr"] = rows(), rows()
    if case["cols"]:
        s["u"], s["dy"] = _columns(s["u"]), _columns(s["dy"])
    else:
        s = {k: x.reshape(b, t, d) if k in ("x", "u", "dy", "dr") else x for k, x in s.items()}
    if s["gate"] is not None and case["cols"] and case["gate"] == "element":
        s["gate"] = s["gate"].reshape(n, d)
    elif s["gate"] is not None and case["cols"] and case["gate"] == "sequence":
        # N x D activations of several sequences: the gate of sequence i serves its t rows
        s["gate"] = s["gate"].reshape(b, d)
    return s


NORM_SCALE = 0.5


def _capacity(m, k, sparsity):
    nnz = round((1 - sparsity) * k)
    return m * max(1, math.ceil(nnz * (1 + PADDING)))


def _adamw_sizes(case):
    if case["model"] == "mlp":
        k, h, m = case["k"], case["h"], case["m"]
        return [_capacity(h, k, 0.9), h, _capacity(m, h, 0.9), m]
    if case["model"] == "gpt":
        d, f = case["d"], case["f"]
        block = [d, d, _capacity(3 * d, d, 0.7), _capacity(d, d, 0.7), d, d,
                 _capacity(f, d, 0.9), _capacity(d, f, 0.9)]
        return [case["vocab"] * d, case["ctx"] * d] + block * case["layers"] + [
            d, d, case["vocab"] * d]
    return [case["size"] + 37 * i for i in range(case["tensors"])]


def _blocks(sizes):
    return [-(-n // BLOCK) for n in sizes]


def _encode(x, signed):
    """(codes, scales) of whole blocks of a flat float32 x: the code of |x| / scale is its
    square root (first moment) or fourth root (second), so that small values keep digits."""
    x = x.view(-1, BLOCK)
    scale = x.abs().amax(1, keepdim=True)
    a = torch.where(scale > 0, x.abs() / scale, 0.0)
    if signed:
        return (torch.copysign(torch.round(torch.sqrt(a) * 127.0), x).to(torch.int8).view(-1),
                scale.view(-1))
    q = torch.round(torch.sqrt(torch.sqrt(a)) * 255.0)
    return torch.where(x > 0, q.clamp(min=1.0), q).to(torch.uint8).view(-1), scale.view(-1)


def _decode(codes, scales):
    if codes.dtype == torch.int8:
        t = codes.float() / 127.0
        return ((t * t.abs()).view(-1, BLOCK) * scales[:, None]).view(-1)
    t = codes.float() / 255.0
    t = t * t
    return ((t * t).view(-1, BLOCK) * scales[:, None]).view(-1)


def _moments(total, live, seed):
    """Flat first and second moments (0 between tensors) as after some thousand steps: each
    element with a gradient scale of its own, over three decades."""
    size = 1e-4 * torch.exp(1.5 * torch.randn(total, generator=_gen(seed, 2), device=DEV))
    m = 0.3 * size * torch.randn(total, generator=_gen(seed, 3), device=DEV)
    v = size.square() * torch.rand(total, generator=_gen(seed, 4), device=DEV).add_(0.5)
    return m * live, v * live, size


def _adamw_inputs(case, seed):
    sizes, dt = _adamw_sizes(case), DTYPES[case["dtype"]]
    spans = [BLOCK * b for b in _blocks(sizes)]
    total = sum(spans)
    live = torch.cat([x for n, s in zip(sizes, spans)
                      for x in (torch.ones(n, device=DEV), torch.zeros(s - n, device=DEV))])
    m, v, size = _moments(total, live, seed)
    p = torch.randn(total, generator=_gen(seed, 1), device=DEV) * 0.02
    g = size * torch.randn(total, generator=_gen(seed, 5), device=DEV)

    def split(flat):
        return [x[:n] for x, n in zip(flat.split(spans), sizes)]

    s = {"kind": "adamw", "sizes": sizes, "spans": spans, "p": [x.to(dt) for x in split(p)],
         "g": [x.to(dt) for x in split(g)]}
    if case["bits"] == 8:
        (m, ms), (v, vs) = _encode(m, True), _encode(v, False)
        s |= {"ms_flat": ms, "vs_flat": vs, "ms": list(ms.split(_blocks(sizes))),
              "vs": list(vs.split(_blocks(sizes)))}
    else:
        s |= {"ms": None, "vs": None}
    return s | {"m_flat": m, "v_flat": v, "m": split(m), "v": split(v)}


def _row_counts(case):
    m, k = case["m"], case["k"]
    total = round((1.0 - case["sparsity"]) * m * k)
    if case["rows"] == "uniform":
        return torch.full((m,), max(1, total // m))
    rank = torch.arange(1, m + 1, dtype=torch.float64) ** -1.1
    lo, hi = 0.0, float(k) * m
    for _ in range(100):
        mid = 0.5 * (lo + hi)
        if (mid * rank).floor().clamp(1, k).sum() < total:
            lo = mid
        else:
            hi = mid
    return (hi * rank).floor().clamp(1, k).long()


def _first(score, counts):
    """A mask of counts[i] columns of row i, those of the lowest score."""
    inside = torch.arange(score.shape[1], device=DEV) < counts[:, None]
    return torch.zeros_like(inside).scatter_(1, score.argsort(dim=1), inside)


def _carry_inputs(case, seed):
    """A padded-CSR topology before and after a rewrite that moved three in ten of its
    connections, and the moments of its slots."""
    m, k = case["m"], case["k"]
    shuffle = torch.randperm(m, generator=torch.Generator().manual_seed(seed))
    cnt = _row_counts(case)[shuffle].to(DEV)
    cap = (cnt.double() * (1.0 + PADDING)).ceil().clamp(min=1).long()
    start = cap.cumsum(0) - cap
    total = int(cap.sum())
    old, new = (torch.full((total,), -1, dtype=torch.int32, device=DEV) for _ in range(2))
    g, step = _gen(seed, 1), max(1, (1 << 26) // k)
    for r0 in range(0, m, step):
        c = cnt[r0:r0 + step]
        was = _first(torch.rand(c.numel(), k, generator=g, device=DEV), c)
        score = torch.rand(c.numel(), k, generator=g, device=DEV)
        kept = was & (score > 0.3)
        now = _first(torch.where(was, torch.where(kept, -1.0, 2.0), score), c)
        for mask, to in ((was, old), (now, new)):
            rows, cols = mask.nonzero(as_tuple=True)
            at = torch.arange(rows.numel(), device=DEV) - (c.cumsum(0) - c)[rows]
            to[start[r0 + rows] + at] = cols.int()
    spans = BLOCK * -(-total // BLOCK)
    live = torch.zeros(spans, device=DEV)
    live[:total] = (old >= 0).float()
    first, second, _ = _moments(spans, live, seed)
    s = {"kind": "carry", "start": start.int(), "old": old, "new": new, "nnz": cnt.int(),
         "k": k, "total": total}
    if case["bits"] == 8:
        (a, sa), (b, sb) = _encode(first, True), _encode(second, False)
        return s | {"m": a[:total], "v": b[:total], "ms": sa, "vs": sb}
    return s | {"m": first[:total].clone(), "v": second[:total].clone(), "ms": None, "vs": None}


def prepare(case, seed):
    if case["kind"] == "loss":
        h, w, target = _loss_inputs(case, seed)
        train = case["mode"] == "train"
        return {"kind": "loss", "train": train, "h": h.requires_grad_(train),
                "w": w.requires_grad_(train), "target": target}
    if case["kind"] == "norm":
        s, train = _norm_inputs(case, seed), case["mode"] == "train"
        for k in ("x", "u", "w", "b", "pw", "pb", "gate"):
            if s[k] is not None:
                s[k].requires_grad_(train)
        return s | {"kind": "norm", "train": train, "norm": case["norm"], "cols": case["cols"]}
    if case["kind"] == "adamw":
        return _adamw_inputs(case, seed)
    return _carry_inputs(case, seed)


# ───────────────────────────── one pass, plain ─────────────────────────────

def _plain_loss(s):
    h, w, target = s["h"].detach().float(), s["w"].detach().float(), s["target"]
    live = target != IGNORE
    t = torch.where(live, target, 0)[:, None]
    z = h @ w.t()
    top = z.amax(1, keepdim=True)
    zt = z.gather(1, t)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    each = torch.where(live, (top + torch.log(total) - zt).squeeze(1), 0.0)
    if not s["train"]:
        return each
    count = live.sum()
    p = e / total
    p.scatter_add_(1, t, torch.full_like(zt, -1.0))
    p = p * torch.where(live, 1.0 / count, 0.0)[:, None]
    return (each.sum() / count, (p @ w).to(s["h"].dtype), (p.t() @ h).to(s["w"].dtype))


def _plain_stats(x, layer):
    xc = x - x.mean(-1, keepdim=True) if layer else x
    rstd = 1.0 / torch.sqrt(xc.square().mean(-1, keepdim=True) + NORM_EPS)
    return xc * rstd, rstd


def _plain_norm_back(g, xhat, rstd, layer):
    g = g - xhat * (g * xhat).mean(-1, keepdim=True) - (g.mean(-1, keepdim=True) if layer else 0)
    return g * rstd


def _rows_of(t):
    return t.detach().float().reshape(-1, t.shape[-1])


def _plain_norm(s):
    layer, dt, shape = s["norm"] == "layer", s["x"].dtype, s["x"].shape
    x, u, w = _rows_of(s["x"]), _rows_of(s["u"]), s["w"].detach().float()
    pw = s["pw"].detach().float() if s["pw"] is not None else None
    o, gate = u, None
    if pw is not None:
        uhat, urstd = _plain_stats(u, layer)
        o = uhat * pw + (s["pb"].detach().float() if layer else 0.0)
    branch = o
    if s["gate"] is not None:
        gate = _rows_of(s["gate"]) if s["gate"].dim() > 1 else s["gate"].detach().float()[None]
        groups = gate.shape[0]
        gate = gate[:, None].expand(groups, x.shape[0] // groups, -1).reshape(x.shape)
        branch = o * gate
    r = x + NORM_SCALE * branch
    xhat, rstd = _plain_stats(r, layer)
    y = xhat * w + (s["b"].detach().float() if layer else 0.0)
    out = [r.to(dt).reshape(shape), y.to(dt).reshape(shape)]
    if not s["train"]:
        return out
    dy = _rows_of(s["dy"])
    dr = _rows_of(s["dr"]) + _plain_norm_back(dy * w, xhat, rstd, layer)
    do = NORM_SCALE * dr
    grads = [dr, None, (dy * xhat).sum(0)] + ([dy.sum(0)] if layer else [])
    dgate = None
    if gate is not None:
        dgate = (do * o).reshape(groups, -1, x.shape[1]).sum(1).reshape(s["gate"].shape)
        do = do * gate
    grads[1] = do
    if pw is not None:
        grads += [(do * uhat).sum(0)] + ([do.sum(0)] if layer else [])
        grads[1] = _plain_norm_back(do * pw, uhat, urstd, layer)
    grads += [dgate] if gate is not None else []
    grads[0], grads[1] = grads[0].reshape(shape), grads[1].reshape(shape)
    return out + [g.to(dt) for g in grads]


def _plain_adamw(s):
    """On all tensors at once, each in whole blocks of one flat array."""
    g = torch.cat([x for g, n, span in zip(s["g"], s["sizes"], s["spans"])
                   for x in (g.float(), g.new_zeros(span - n, dtype=torch.float32))])
    p = torch.cat([x for p, n, span in zip(s["p"], s["sizes"], s["spans"])
                   for x in (p.float(), p.new_zeros(span - n, dtype=torch.float32))])
    m, v = s["m_flat"], s["v_flat"]
    if s["ms"] is not None:
        m, v = _decode(m, s["ms_flat"]), _decode(v, s["vs_flat"])
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * (g * g)
    root = torch.sqrt(v) / math.sqrt(1 - BETA2 ** STEP) + EPS
    p = p * (1 - LR * DECAY) - (LR / (1 - BETA1 ** STEP)) * (m / root)
    s["p"] = [x[:n].to(q.dtype) for x, n, q in zip(p.split(s["spans"]), s["sizes"], s["p"])]
    if s["ms"] is None:
        s["m_flat"], s["v_flat"] = m, v
        return [*s["p"], m, v]
    (s["m_flat"], s["ms_flat"]), (s["v_flat"], s["vs_flat"]) = _encode(m, True), _encode(v, False)
    return [*s["p"], _decode(s["m_flat"], s["ms_flat"]), _decode(s["v_flat"], s["vs_flat"])]


def _whole(x):
    return F.pad(x, (0, -x.numel() % BLOCK))


def _plain_carry(s):
    total, k = s["total"], s["k"] + 1
    rows = torch.searchsorted(s["start"], torch.arange(total, device=DEV, dtype=torch.int32),
                              right=True) - 1
    # ascending keys: a row's padding slots come after its live ones
    was = rows * k + torch.where(s["old"] >= 0, s["old"].long(), k - 1)
    now = rows * k + torch.where(s["new"] >= 0, s["new"].long(), k - 1)
    at = torch.searchsorted(was, now).clamp(max=total - 1)
    found = (was[at] == now) & (s["new"] >= 0)
    if s["ms"] is None:
        return [torch.where(found, x[at], 0.0) for x in (s["m"], s["v"])]
    m, v = (_decode(_whole(x), y)[:total] for x, y in ((s["m"], s["ms"]), (s["v"], s["vs"])))
    m, v = (torch.where(found, x[at], 0.0) for x in (m, v))
    return [_decode(*_encode(_whole(m), True))[:total],
            _decode(*_encode(_whole(v), False))[:total]]


# ───────────────────────────── one pass ─────────────────────────────

def run(s):
    kind = s["kind"]
    if not own:
        return {"loss": _plain_loss, "norm": _plain_norm, "adamw": _plain_adamw,
                "carry": _plain_carry}[kind](s)
    import sparsecore_amd as slk

    if kind == "loss":
        if not s["train"]:
            with torch.no_grad():
                return slk.linear_cross_entropy(s["h"], s["w"], s["target"], reduction="none")
        loss = slk.linear_cross_entropy(s["h"], s["w"], s["target"])
        return (loss.detach(), *torch.autograd.grad(loss, [s["h"], s["w"]]))
    if kind == "norm":
        with torch.set_grad_enabled(s["train"]):
            r, y = slk.residual_norm(s["x"], s["w"], s["b"], branch=s["u"], gate=s["gate"],
                                     post_weight=s["pw"], post_bias=s["pb"], scale=NORM_SCALE,
                                     kind=s["norm"], eps=NORM_EPS, feature_major=s["cols"])
        if not s["train"]:
            return [r, y]
        of = [s[k] for k in ("x", "u", "w", "b", "pw", "pb", "gate") if s[k] is not None]
        return [r.detach(), y.detach(), *torch.autograd.grad([r, y], of, [s["dr"], s["dy"]])]
    if kind == "adamw":
        slk.optim.adamw_step(s["p"], s["g"], s["m"], s["v"], exp_avg_scales=s["ms"],
                             exp_avg_sq_scales=s["vs"], step=STEP, lr=LR, betas=(BETA1, BETA2),
                             eps=EPS, weight_decay=DECAY)
        if s["ms"] is None:
            return [*s["p"], s["m_flat"], s["v_flat"]]
        return [*s["p"], slk.optim.dequantize(s["m_flat"], s["ms_flat"]),
                slk.optim.dequantize(s["v_flat"], s["vs_flat"])]
    states = [s["m"], s["v"]] if s["ms"] is None else [(s["m"], s["ms"]), (s["v"], s["vs"])]
    states = slk.optim.carry_slots(s["start"], (s["old"], s["nnz"]), (s["new"], s["nnz"]), states)
    return states if s["ms"] is None else [slk.optim.dequantize(*x) for x in states]


# ───────────────────────────── its work ─────────────────────────────

def work(case):
    if case["kind"] == "loss":
        n, d, v = case["n"], case["d"], case["v"]
        e = 4 if case["dtype"] == "float32" else 2
        live = 1 - case["ignored"]
        if case["mode"] == "score":
            return {"bytes": e * (live * n * d + v * d) + 12 * n, "flops": 2 * live * n * d * v}
        return {"bytes": e * ((1 + live) * n * d + 2 * v * d) + 8 * n,
                "flops": 6 * live * n * d * v}
    if case["kind"] == "norm":
        d, n = case["d"], case["b"] * case["t"]
        e = 4 if case["dtype"] == "float32" else 2
        gate = {"none": 0, "feature": d, "sequence": case["b"] * d,
                "element": n * d}[case["gate"]]
        if case["mode"] == "infer":
            return {"bytes": e * (4 * n * d + gate), "flops": 12 * n * d}
        # forward as above; backward reads dy, dr, r and the branch, writes dx and its gradient
        return {"bytes": e * (10 * n * d + 3 * gate), "flops": 40 * n * d}
    if case["kind"] == "adamw":
        e = 4 if case["dtype"] == "float32" else 2
        state = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
        n = sum(_adamw_sizes(case))
        return {"bytes": n * (3 * e + state), "flops": 15 * n}
    nnz = (1 - case["sparsity"]) * case["m"] * case["k"]
    cap = nnz * (1 + PADDING) + 0.5 * case["m"]
    state = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    return {"bytes": 8 * nnz + state * cap + 8 * case["m"], "flops": 2 * cap}


# ───────────────────────────── the same in 64 bits ─────────────────────────────

def _exact_loss(case, seed):
    h, w, target = _loss_inputs(case, seed)
    if case["mode"] == "score":
        return F.cross_entropy(h.double() @ w.double().t(), target, reduction="none",
                               ignore_index=IGNORE)
    count = (target != IGNORE).sum()
    w = w.double()
    loss, dh, dw = torch.zeros((), dtype=torch.float64, device=DEV), [], torch.zeros_like(w)
    for part, t in zip(h.split(2048), target.split(2048)):
        part = part.double()
        z = (part @ w.t()).requires_grad_()
        each = F.cross_entropy(z, t, reduction="sum", ignore_index=IGNORE) / count
        dz, = torch.autograd.grad(each, z)
        loss += each.detach()
        dh.append(dz @ w)
        dw += dz.t() @ part
    return loss, torch.cat(dh), dw


def _exact_norm(case, seed):
    s = _norm_inputs(case, seed)
    d, layer, train = case["d"], case["norm"] == "layer", case["mode"] == "train"
    p = {k: s[k].double().requires_grad_(train)
         for k in ("x", "u", "w", "b", "pw", "pb", "gate") if s[k] is not None}

    def norm(v, w, b):
        if layer:
            return F.layer_norm(v, (d,), p[w], p[b], NORM_EPS)
        return F.rms_norm(v, (d,), p[w], NORM_EPS)

    o = norm(p["u"], "pw", "pb") if case["post"] else p["u"]
    if "gate" in p:
        gate = p["gate"]
        if case["cols"] and case["gate"] == "sequence":
            gate = gate.repeat_interleave(case["t"], 0)
        o = o * gate
    r = p["x"] + NORM_SCALE * o
    y = norm(r, "w", "b")
    if not train:
        return [r, y]
    grads = torch.autograd.grad([r, y], list(p.values()), [s["dr"].double(), s["dy"].double()])
    return [r.detach(), y.detach(), *grads]


def _exact_adamw(case, seed):
    s = _adamw_inputs(case, seed)
    m, v = s["m_flat"], s["v_flat"]
    if case["bits"] == 8:
        a, b = m.double() / 127, v.double() / 255
        m = (a * a.abs()).view(-1, BLOCK) * s["ms_flat"].double()[:, None]
        v = (b ** 4).view(-1, BLOCK) * s["vs_flat"].double()[:, None]
    g = torch.zeros(m.numel(), dtype=torch.float64, device=DEV)
    at = 0
    for x, n, span in zip(s["g"], s["sizes"], s["spans"]):
        g[at:at + n] = x
        at += span
    m, v = m.double().view(-1), v.double().view(-1)
    m, v = torch.lerp(g, m, BETA1), torch.lerp(g ** 2, v, BETA2)
    update = (m / (1 - BETA1 ** STEP)) / ((v / (1 - BETA2 ** STEP)).sqrt() + EPS)
    p = [(1 - LR * DECAY) * x.double() - LR * u[:x.numel()]
         for x, u in zip(s["p"], update.split(s["spans"]))]
    # 8-bit moments are codes, not computed numbers
    return [*p, None, None] if case["bits"] == 8 else [*p, m, v]


def exact(case, seed):
    if case["kind"] == "loss":
        return _exact_loss(case, seed)
    if case["kind"] == "norm":
        return _exact_norm(case, seed)
    return _exact_adamw(case, seed) if case["kind"] == "adamw" else None
