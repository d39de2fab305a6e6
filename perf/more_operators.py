"""More operators around the sparse layers of a training step, as cases to measure.

A case is one call of one of them, at one size:

  attn   attention between the QKV projection and the output projection: causal or not, grouped
         heads (several query heads share a key head), a batch, a padded batch or packed
         sequences of different lengths, with or without a learned bias of the relative position
         (one value a head and bucket of distances). `train` is forward plus backward, `infer`
         forward under no_grad, and `decode` one or a few new tokens against long key and value
         arrays of which each sequence fills a part
  act    an activation between two layers that keeps its input in 8 bits for its backward pass:
         forward plus backward

Where `own` is false the same is computed in plain torch, in 32 bits. `exact` states it in 64.
"""

from __future__ import annotations

import decimal
import math

import torch
import torch.nn.functional as F

own = False

DEV = "cuda"
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
BLOCK = 256     # consecutive elements of an activation that share one scale
TINY = 2.0 ** -100  # a block whose largest magnitude is below this is kept as zeros
CHUNK = 1 << 28  # scores that a plain or exact pass holds at once


def listed():
    return [
        # the 10M char-GPT's attention over its training batch: the QKV projection is a sparse
        # layer, whose output is feature-major
        {"name": "attn_10m_train", "kind": "attn", "mode": "train", "layout": "batch", "b": 32,
         "t": 256, "h": 6, "g": 6, "d": 64, "causal": True, "buckets": 0, "cols": True,
         "dtype": "float32"},
        # the 60M mini-GPT's, with a learned relative position bias in place of position vectors
        {"name": "attn_60m_bias_train", "kind": "attn", "mode": "train", "layout": "batch",
         "b": 16, "t": 512, "h": 12, "g": 12, "d": 64, "causal": True, "buckets": 32,
         "cols": True, "dtype": "float32"},
        # an encoder over padded sentences: both directions, bias, odd sizes
        {"name": "attn_padded_bias_train_bf16", "kind": "attn", "mode": "train",
         "layout": "padded", "b": 24, "t": 333, "h": 8, "g": 8, "d": 64, "causal": False,
         "buckets": 32, "cols": False, "dtype": "bfloat16"},
        # documents of very different lengths packed into one row of 8191 tokens, grouped heads
        {"name": "attn_packed_train_bf16", "kind": "attn", "mode": "train", "layout": "packed",
         "b": 23, "t": 8191, "h": 16, "g": 4, "d": 128, "causal": True, "buckets": 0,
         "cols": False, "dtype": "bfloat16"},
        # one long document: the largest
        {"name": "attn_16k_train_bf16", "kind": "attn", "mode": "train", "layout": "batch",
         "b": 1, "t": 16384, "h": 32, "g": 8, "d": 128, "causal": True, "buckets": 0,
         "cols": False, "dtype": "bfloat16"},
        # a prompt of the 60M mini-GPT being read
        {"name": "attn_prompt_1001", "kind": "attn", "mode": "infer", "layout": "batch", "b": 1,
         "t": 1001, "h": 12, "g": 12, "d": 64, "causal": True, "buckets": 0, "cols": True,
         "dtype": "float32"},
        # one token each of eight sequences of the char-GPT being generated: where latency counts
        {"name": "attn_decode_8", "kind": "attn", "mode": "decode", "b": 8, "t": 1, "s": 256,
         "h": 6, "g": 6, "d": 64, "causal": True, "buckets": 0, "dtype": "float32"},
        # sixteen long conversations, grouped heads
        {"name": "attn_decode_16x8k_bf16", "kind": "attn", "mode": "decode", "b": 16, "t": 1,
         "s": 8192, "h": 32, "g": 8, "d": 128, "causal": True, "buckets": 0,
         "dtype": "bfloat16"},
        # one very long context with a relative position bias
        {"name": "attn_decode_131k_bias", "kind": "attn", "mode": "decode", "b": 1, "t": 1,
         "s": 131071, "h": 12, "g": 12, "d": 64, "causal": True, "buckets": 32,
         "dtype": "float32"},
        # the hidden layer of the 784 -> 512 -> 10 MLP
        {"name": "act_mlp_relu", "kind": "act", "n": 256, "d": 512, "act": "relu", "cols": True,
         "dtype": "float32"},
        # the 10M char-GPT's feed-forward part, feature-major between two sparse layers
        {"name": "act_10m_gelu", "kind": "act", "n": 8192, "d": 1536, "act": "gelu",
         "cols": True, "dtype": "float32"},
        # a wide feed-forward part under mixed precision, an odd number of tokens
        {"name": "act_16k_silu_bf16", "kind": "act", "n": 8191, "d": 16384, "act": "silu",
         "cols": False, "dtype": "bfloat16"},
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
    kind = rng.choice(["attn"] * 3 + ["act"])
    dtype = rng.choice(["float32", "bfloat16"])
    if kind == "act":
        return {"kind": kind, "n": _size(rng, 1, 8192), "d": _size(rng, 16, 16384),
                "act": rng.choice(["gelu", "gelu_tanh", "silu", "relu"]),
                "cols": rng.random() < 0.5, "dtype": dtype}
    mode = rng.choice(["train", "train", "infer", "decode"])
    g = rng.choice([1, 2, 3, 4, 6, 8, 12, 16])
    c = {"kind": kind, "mode": mode, "h": g * rng.choice([1, 1, 2, 4]), "g": g,
         "d": rng.choice([32, 64, 64, 128, 128, 40, 80]), "causal": rng.random() < 0.7,
         "buckets": rng.choice([0, 0, 16, 32]), "dtype": dtype}
    if mode == "decode":
        c |= {"b": _log_int(rng, 1, 32), "t": rng.choice([1, 1, 1, 2, 5]), "causal": True,
              "s": _size(rng, 16, 65536)}
        while c["b"] * c["s"] * g * c["d"] > 1 << 28:
            c["s"] = (c["s"] + 1) // 2
        return c
    c |= {"layout": rng.choice(["batch", "padded", "packed"]), "cols": rng.random() < 0.5}
    c |= {"t": _size(rng, 1, 8192), "b": _log_int(rng, 1, 48)}
    if c["layout"] == "packed":
        c["t"] = max(c["t"], c["b"])
        return c
    while c["b"] * c["t"] > 16384:
        c["b"] = (c["b"] + 1) // 2
    return c


# ───────────────────────────── inputs ─────────────────────────────

def _gen(seed, part):
    return torch.Generator(device=DEV).manual_seed(seed * 64 + part)


def _normal(shape, seed, part, scale=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=_gen(seed, part), device=DEV) * scale).to(dtype)


def _lengths(case, seed):
    """Host lengths of the sequences. Padded sentences fill half of their row or more; packed
    documents spread over a factor of a hundred and fill the row but for a few tokens."""
    gen = torch.Generator().manual_seed(seed)
    b, t = case["b"], case["t"]
    if case["layout"] == "batch":
        return [t] * b
    if case["layout"] == "padded":
        return (t - torch.randint(0, t // 2 + 1, (b,), generator=gen)).tolist()
    share = torch.exp(4.6 * torch.rand(b, generator=gen))
    n = (share / share.sum() * (t - b) * 0.999).floor().long() + 1
    return n.tolist()


def _columns(x):
    """The same rows, stored feature by feature."""
    return x.t().contiguous().t()


def _attn_inputs(case, seed):
    """Queries and keys as projections give them: scores of a standard deviation of about 1.5,
    all keys with a part in common (so that some queries look everywhere and some at few)."""
    h, g, d, dt = case["h"], case["g"], case["d"], DTYPES[case["dtype"]]
    s = {"scale": d ** -0.5, "causal": case["causal"], "mode": case["mode"]}
    if case["buckets"]:
        s["bias"] = _normal((case["buckets"], h), seed, 9, 0.7, dt)
    if case["mode"] == "decode":
        b, t, n = case["b"], case["t"], case["s"]
        gen = torch.Generator().manual_seed(seed)
        low = max(t, (3 * n) // 4)
        lens = torch.randint(low, max(n, low) + 1, (b,), generator=gen)
        n = max(n, int(lens.max()))
        s |= {"host": [(t, int(x)) for x in lens], "k_lengths": lens.int().to(DEV),
              "q": _normal((b, t, h, d), seed, 1, 1.2, dt),
              "k": (_normal((b, n, g, d), seed, 2) + _normal((g, d), seed, 3, 0.5)).to(dt),
              "v": _normal((b, n, g, d), seed, 4, 1.0, dt)}
        return s
    lens = _lengths(case, seed)
    packed = case["layout"] == "packed"
    rows = case["t"] if packed else case["b"] * case["t"]
    x = _normal((rows, (h + 2 * g) * d), seed, 1, 1.2)
    x[:, h * d:(h + g) * d] += _normal((g * d,), seed, 3, 0.5)
    x = x.to(dt)
    lead = (rows,) if packed else (case["b"], case["t"])
    dout = _normal((rows, h * d), seed, 5, 1e-3, dt)
    if case["cols"]:
        x, dout = _columns(x), _columns(dout)
    q, k, v = x.split([h * d, g * d, g * d], dim=1)
    s |= {"q": q.unflatten(1, (h, d)), "k": k.unflatten(1, (g, d)), "v": v.unflatten(1, (g, d)),
          "dout": dout.unflatten(1, (h, d)), "host": [(n, n) for n in lens], "lead": lead,
          "cols": case["cols"]}
    for key in ("q", "k", "v", "dout"):
        s[key] = s[key].unflatten(0, lead)
    if packed:
        off = torch.tensor([0] + lens).cumsum(0).int()
        s["offsets"] = off.to(DEV)
    elif case["layout"] == "padded":
        s["lengths"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    return s


def _act_inputs(case, seed):
    """Pre-activations, a few features much larger than the others, and the gradient of the
    output, one memory layout for all."""
    n, d, dt = case["n"], case["d"], DTYPES[case["dtype"]]
    size = torch.exp(0.5 * torch.randn(d, generator=_gen(seed, 1), device=DEV))
    x = (_normal((n, d), seed, 2) * size).to(dt)
    dy = _normal((n, d), seed, 3, 1e-3, dt)
    if case["cols"]:
        x, dy = _columns(x), _columns(dy)
    return {"x": x, "dy": dy, "act": case["act"], "cols": case["cols"]}


def prepare(case, seed):
    if case["kind"] == "act":
        s = _act_inputs(case, seed)
        s["x"].requires_grad_()
        return s | {"kind": "act"}
    s = _attn_inputs(case, seed)
    if case["mode"] == "train":
        for key in ("q", "k", "v", "bias"):
            if key in s:
                s[key] = s[key].detach().requires_grad_()
    return s | {"kind": "attn"}


# ───────────────────────────── one pass, plain ─────────────────────────────

MAX_DISTANCE = 128


def _plain_buckets(buckets, causal):
    """The bucket of each distance 0..MAX_DISTANCE of one direction: the first half one
    distance each, then logarithmic. With r of those and e exact ones bucket e + t begins at
    the first n with (n / e)^r >= (MAX_DISTANCE / e)^t, in whole numbers."""
    one = buckets if causal else buckets // 2
    e = one // 2
    r = one - e
    out = []
    for n in range(MAX_DISTANCE + 1):
        t = sum(n ** r * e ** k >= e ** r * MAX_DISTANCE ** k for k in range(1, r))
        out.append(n if n < e else e + t)
    return out


def _plain_bucket_of(tq, tk, buckets, causal):
    """tq x tk buckets; the last query stands at the last key."""
    near = torch.tensor(_plain_buckets(buckets, causal), device=DEV)
    at = torch.arange(tq, device=DEV)[:, None] + (tk - tq)
    away = at - torch.arange(tk, device=DEV)
    which = near[away.abs().clamp(max=MAX_DISTANCE)]
    return which if causal else which + (away < 0) * (buckets // 2)


def _sequences(s):
    """(query rows, key rows) of each sequence as index pairs of the row-flattened arrays."""
    out, packed = [], "offsets" in s
    q0 = k0 = 0
    tq = 0 if packed else s["q"].shape[1]
    tk = 0 if packed else s["k"].shape[1]
    for nq, nk in s["host"]:
        out.append((q0, nq, k0, nk))
        q0, k0 = (q0 + nq, k0 + nk) if packed else (q0 + tq, k0 + tk)
    return out


def _flat(x):
    return x.detach().reshape(-1, *x.shape[-2:])


def _groups(seqs, heads):
    """Runs of neighbouring sequences of one size, and the heads of a piece."""
    i = 0
    while i < len(seqs):
        _, nq, _, nk = seqs[i]
        j = i + 1
        step_q, step_k = (seqs[j][0] - seqs[i][0], seqs[j][2] - seqs[i][2]) if j < len(seqs) \
            else (nq, nk)
        each = max(1, nq * nk * heads)
        while j < len(seqs) and seqs[j][1] == nq and seqs[j][3] == nk and \
                (j + 1 - i) * each <= CHUNK and \
                seqs[j][0] - seqs[j - 1][0] == step_q and seqs[j][2] - seqs[j - 1][2] == step_k:
            j += 1
        yield i, j, step_q, step_k
        i = j


def _plain_attn(s):
    q, k, v = _flat(s["q"]), _flat(s["k"]), _flat(s["v"])
    h, g, train = q.shape[1], k.shape[1], s["mode"] == "train"
    rep = h // g
    bias = s["bias"].detach().float() if "bias" in s else None
    out = torch.zeros(q.shape, device=DEV)
    if train:
        dout = _flat(s["dout"])
        dq, dk, dv = (torch.zeros(x.shape, device=DEV) for x in (q, k, v))
        dbias = torch.zeros_like(bias) if bias is not None else None
    seqs = _sequences(s)
    for i, j, step_q, step_k in _groups(seqs, h):
        q0, nq, k0, nk = seqs[i]
        b = j - i
        qi = torch.arange(nq, device=DEV) + q0 + step_q * torch.arange(b, device=DEV)[:, None]
        ki = torch.arange(nk, device=DEV) + k0 + step_k * torch.arange(b, device=DEV)[:, None]
        hidden = None
        if s["causal"]:
            hidden = torch.arange(nk, device=DEV) > \
                torch.arange(nq, device=DEV)[:, None] + (nk - nq)
        which = _plain_bucket_of(nq, nk, bias.shape[0], s["causal"]) if bias is not None else None
        heads = max(1, min(g, CHUNK // max(1, b * nq * nk * rep)))
        for g0 in range(0, g, heads):
            gs, hs = slice(g0, g0 + heads), slice(g0 * rep, (g0 + heads) * rep)
            qf = q[:, hs][qi].float().transpose(1, 2).contiguous()  # b, heads, nq, d
            kf, vf = (x[:, gs][ki].float().transpose(1, 2).repeat_interleave(rep, 1).contiguous()
                      for x in (k, v))
            z = (qf @ kf.transpose(2, 3).contiguous()) * s["scale"]
            if bias is not None:
                z += bias[:, hs].t()[:, which]
            if hidden is not None:
                z.masked_fill_(hidden, -math.inf)
            top = z.amax(3, keepdim=True)
            p = torch.exp(z - top)
            del z
            p /= p.sum(3, keepdim=True)
            o = p @ vf
            out[:, hs][qi] = o.transpose(1, 2)
            if not train:
                continue
            go = dout[:, hs][qi].float().transpose(1, 2).contiguous()
            shape = (b, -1, rep, nk, q.shape[2])
            dv[:, gs][ki] = (p.transpose(2, 3).contiguous() @ go).view(shape).sum(2).transpose(1, 2)
            ds = go @ vf.transpose(2, 3).contiguous()
            ds -= (go * o).sum(3, keepdim=True)
            ds *= p
            del p
            if bias is not None:
                per = ds.sum(0).view(-1, nq * nk).t()
                dbias[:, hs] += torch.zeros_like(dbias[:, hs]).index_add_(0, which.view(-1), per)
            dq[:, hs][qi] = (ds @ kf).transpose(1, 2) * s["scale"]
            dk[:, gs][ki] = (ds.transpose(2, 3).contiguous() @ qf).view(shape).sum(2) \
                .transpose(1, 2) * s["scale"]
    dt = s["q"].dtype
    out = out.to(dt).view(s["q"].shape)
    if not train:
        return out
    grads = [x.to(dt).view(s[n].shape) for x, n in ((dq, "q"), (dk, "k"), (dv, "v"))]
    return [out, *grads] + ([dbias.to(dt)] if bias is not None else [])


def _blocks(x, cols):
    """x as float32 rows of BLOCK consecutive elements of its memory, zeros behind the last."""
    flat = (x.t() if cols else x).reshape(-1).float()
    return F.pad(flat, (0, -flat.numel() % BLOCK)).view(-1, BLOCK)


def _kept(x, cols):
    """What 8 bits keep of x: whole multiples of a 127th of a block's largest magnitude."""
    rows = _blocks(x, cols)
    top = rows.abs().amax(1, keepdim=True)
    inv = torch.where(top >= TINY, torch.full_like(top, 127.0) / top, 0.0)
    kept = torch.round(rows * inv) * (top * torch.tensor(1.0 / 127.0, device=DEV))
    n, d = x.shape
    kept = kept.view(-1)[:n * d]
    return kept.view(d, n).t() if cols else kept.view(n, d)


ROOT_2_PI, TANH_CUBE = math.sqrt(2.0 / math.pi), 0.044715


def _plain_act(s):
    x, dy, act, dt = s["x"].detach(), s["dy"].float(), s["act"], s["x"].dtype
    xf, xk = x.float(), _kept(x, s["cols"])

    def normal(z):
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))

    if act == "relu":
        y, slope = torch.where(xf > 0, xf, 0.0), (xk > 0).float()
    elif act == "silu":
        y = xf / (1.0 + torch.exp(-xf))
        sig = 1.0 / (1.0 + torch.exp(-xk))
        slope = sig * (1.0 + xk * (1.0 - sig))
    elif act == "gelu":
        y = xf * normal(xf)
        slope = normal(xk) + xk * torch.exp(-0.5 * xk * xk) / math.sqrt(2.0 * math.pi)
    else:
        y = 0.5 * xf * (1.0 + torch.tanh(ROOT_2_PI * (xf + TANH_CUBE * xf ** 3)))
        t = torch.tanh(ROOT_2_PI * (xk + TANH_CUBE * xk ** 3))
        slope = 0.5 * (1.0 + t) + 0.5 * xk * (1.0 - t * t) * ROOT_2_PI * \
            (1.0 + 3.0 * TANH_CUBE * xk * xk)
    return [y.to(dt), (dy * slope).to(dt)]


# ───────────────────────────── one pass ─────────────────────────────

def run(s):
    if not own:
        return _plain_attn(s) if s["kind"] == "attn" else _plain_act(s)
    import sparsecore_amd as slk

    if s["kind"] == "act":
        y = slk.activation(s["x"], s["act"], save_bits=8)
        return [y.detach(), *torch.autograd.grad(y, [s["x"]], [s["dy"]])]
    more = {k: s[k] for k in ("offsets", "lengths", "k_lengths", "bias") if k in s}
    if "bias" in s:
        more["max_distance"] = MAX_DISTANCE
    train = s["mode"] == "train"
    with torch.set_grad_enabled(train):
        out = slk.attention(s["q"], s["k"], s["v"], causal=s["causal"], scale=s["scale"],
                            feature_major=s.get("cols", False), **more)
    if not train:
        return out
    of = [s[k] for k in ("q", "k", "v", "bias") if k in s]
    return [out.detach(), *torch.autograd.grad(out, of, [s["dout"]])]


# ───────────────────────────── its work ─────────────────────────────

def _pairs(nq, nk, causal):
    """(query, key) pairs that see each other."""
    if not causal:
        return nq * nk
    full = max(0, min(nq, nk))
    return full * (full + 1) // 2 + (nk - full) * full


def work(case):
    e = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "act":
        n = case["n"] * case["d"]
        # forward x -> y and a code, backward dy and the code -> dx
        return {"bytes": n * (4 * e + 2 + 8 / BLOCK), "flops": 30 * n}
    h, g, d = case["h"], case["g"], case["d"]
    if case["mode"] == "decode":
        b, t, live = case["b"], case["t"], 0.875 * case["s"]
        return {"bytes": e * b * d * (2 * t * h + 2 * live * g),
                "flops": 4 * d * h * b * t * live}
    if case["layout"] == "padded":
        rows = 0.75 * case["b"] * case["t"]
        pairs = case["b"] * _pairs(round(0.75 * case["t"]), round(0.75 * case["t"]),
                                   case["causal"])
    else:
        lens = _lengths(case, 0)
        rows = sum(lens)
        pairs = sum(_pairs(n, n, case["causal"]) for n in lens)
    if case["mode"] == "infer":
        return {"bytes": e * rows * d * (2 * h + 2 * g), "flops": 4 * d * h * pairs}
    # forward q, k, v -> out; backward q, k, v, out, dout -> dq, dk, dv: seven products
    return {"bytes": e * rows * d * (6 * h + 6 * g), "flops": 14 * d * h * pairs}


# ───────────────────────────── the same in 64 bits ─────────────────────────────

def _exact_bucket(away, buckets, causal):
    """Bucket of a query `away` positions behind its key, with logarithms of fifty digits."""
    first, one = (0, buckets) if causal else ((buckets // 2) * (away < 0), buckets // 2)
    n, e = abs(away), one // 2
    if n < e:
        return first + n
    with decimal.localcontext() as ctx:
        ctx.prec = 50
        at = (decimal.Decimal(n) / e).ln() / (decimal.Decimal(MAX_DISTANCE) / e).ln() * (one - e)
        return first + min(one - 1, e + int(at + decimal.Decimal("1e-40")))


def _exact_bias(table, nq, nk, causal):
    """heads x nq x nk biases of a (buckets, heads) table."""
    far = torch.arange(-MAX_DISTANCE, MAX_DISTANCE + 1).tolist()
    which = [0 if causal and n < 0 else _exact_bucket(n, table.shape[0], causal) for n in far]
    per = table[torch.tensor(which, device=DEV)]  # distances x heads
    away = (torch.arange(nq, device=DEV)[:, None] + (nk - nq)) - torch.arange(nk, device=DEV)
    return per.t()[:, away.clamp(-MAX_DISTANCE, MAX_DISTANCE) + MAX_DISTANCE]


def _exact_attn(case, seed):
    s = _attn_inputs(case, seed)
    train = case["mode"] == "train"
    h, g = case["h"], case["g"]
    rep = h // g
    rows = {key: s[key].reshape(-1, *s[key].shape[-2:]) for key in ("q", "k", "v", "dout")
            if key in s}
    out = torch.zeros(rows["q"].shape, dtype=torch.float64, device=DEV)
    grads = [torch.zeros(rows[key].shape, dtype=torch.float64, device=DEV)
             for key in ("q", "k", "v")] if train else []
    table = s["bias"].double().requires_grad_(train) if "bias" in s else None
    dtable = torch.zeros_like(table) if train and table is not None else None
    for q0, nq, k0, nk in _sequences(s):
        if not nq or not nk:
            continue
        step = max(1, CHUNK // (2 * nq * nk * rep))
        for g0 in range(0, g, step):
            g1 = min(g, g0 + step)
            hs = slice(g0 * rep, g1 * rep)
            q = rows["q"][q0:q0 + nq, hs].double().transpose(0, 1).requires_grad_(train)
            k, v = (rows[key][k0:k0 + nk, g0:g1].double().transpose(0, 1).requires_grad_(train)
                    for key in ("k", "v"))
            z = torch.bmm(q, k.repeat_interleave(rep, 0).mT.contiguous()) * s["scale"]
            if table is not None:
                z = z + _exact_bias(table[:, hs], nq, nk, case["causal"])
            if case["causal"]:
                seen = torch.ones(nq, nk, dtype=torch.bool, device=DEV).tril(nk - nq)
                z = z.masked_fill(~seen, -math.inf)
            o = torch.bmm(torch.softmax(z, 2), v.repeat_interleave(rep, 0))
            out[q0:q0 + nq, hs] = o.detach().transpose(0, 1)
            if not train:
                continue
            up = rows["dout"][q0:q0 + nq, hs].double().transpose(0, 1)
            of = [q, k, v] + ([table] if table is not None else [])
            d = torch.autograd.grad(o, of, up)
            grads[0][q0:q0 + nq, hs] = d[0].transpose(0, 1)
            grads[1][k0:k0 + nk, g0:g1] = d[1].transpose(0, 1)
            grads[2][k0:k0 + nk, g0:g1] = d[2].transpose(0, 1)
            if table is not None:
                dtable += d[3]
    out = out.view(s["q"].shape)
    if not train:
        return out
    grads = [x.view(s[key].shape) for x, key in zip(grads, ("q", "k", "v"))]
    return [out, *grads] + ([dtable] if dtable is not None else [])


def _exact_act(case, seed):
    s = _act_inputs(case, seed)
    f = {"relu": F.relu, "silu": F.silu, "gelu": F.gelu,
         "gelu_tanh": lambda z: F.gelu(z, approximate="tanh")}[case["act"]]
    # a code is what float32 operations make of it: 127 / top, rounded, times x, rounded
    x = s["x"].t() if case["cols"] else s["x"]
    n = x.numel()
    flat = torch.zeros(-(-n // BLOCK) * BLOCK, device=DEV)
    flat[:n] = x.reshape(-1)
    flat = flat.view(-1, BLOCK)
    top = flat.abs().max(1).values
    code = flat.mul((torch.full_like(top, 127.0) / top.clamp(min=TINY))[:, None]).round()
    code.masked_fill_((top < TINY)[:, None], 0.0)
    kept = code.double() * (top.double() / 127)[:, None]
    kept = kept.view(-1)[:n].view(x.shape)
    kept = (kept.t() if case["cols"] else kept).requires_grad_()
    y = f(s["x"].double())
    dx, = torch.autograd.grad(f(kept), kept, s["dy"].double())
    return [y, dx]


def exact(case, seed):
    return _exact_attn(case, seed) if case["kind"] == "attn" else _exact_act(case, seed)
