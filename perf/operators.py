"""Cases and plain forms of the operators that regularise training: counter-based dropout, the norms that add a
residual, attention with dropout on its probabilities, and the embedding with a sorted gradient.

``run`` computes one forward and backward pass of a case, in elementary torch operations where ``own`` is false and
through the framework's entry points where it is true. ``exact`` states the same results in 64 bits.
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_LOW = 0xFFFFFFFF
HEAD = 64  # columns of an attention head
BUCKETS, MAX_POSITION, SPAN = 256, 512, 256  # position buckets of the DeBERTa-v3 presets


def listed():
    return [
        # the embedding output of a base model's micro-batch (32 x 512 tokens)
        {"name": "dropout base", "op": "dropout", "rows": 16384, "cols": 768, "dtype": "bf16", "p": 0.1, "residual": False},
        # the residual branch of one short sentence of the xsmall model, in the type of a CPU-parity run
        {"name": "dropout_add sentence", "op": "dropout", "rows": 37, "cols": 384, "dtype": "fp32", "p": 0.1, "residual": True},
        # post-norm block output of the base model: LayerNorm(dropout(branch) + residual)
        {"name": "add_layer_norm base", "op": "norm", "rows": 16384, "cols": 768, "dtype": "bf16", "rms": False, "p": 0.1},
        # rotary backbone without dropout at the large width, four sequences of 4096 tokens
        {"name": "add_rms_norm large", "op": "norm", "rows": 16384, "cols": 1024, "dtype": "bf16", "rms": True, "p": 0.0},
        # a ragged batch tail at a width that is no multiple of eight
        {"name": "add_rms_norm odd", "op": "norm", "rows": 61, "cols": 770, "dtype": "fp16", "rms": True, "p": 0.15},
        # the base model's attention layer on a padded micro-batch
        {"name": "disentangled base", "op": "attention", "kind": "disentangled", "batch": 32, "length": 512, "heads": 12,
         "mask": "pad", "p": 0.1},
        # two short padded sentences of the xsmall model: latency
        {"name": "disentangled sentences", "op": "attention", "kind": "disentangled", "batch": 2, "length": 93, "heads": 6,
         "mask": "pad", "p": 0.1},
        # packed documents in long rows of the rotary backbone
        {"name": "rotary packed 4096", "op": "attention", "kind": "rotary", "batch": 2, "length": 4096, "heads": 12,
         "mask": "docs", "p": 0.1},
        # unmasked long rows at the large width
        {"name": "rotary 2048", "op": "attention", "kind": "rotary", "batch": 4, "length": 2048, "heads": 16,
         "mask": "none", "p": 0.05},
        # word embeddings of a base micro-batch: Zipf-distributed tokens, a seventh of them the mask token
        {"name": "embedding base", "op": "embedding", "tokens": 16384, "vocab": 128100, "hidden": 768, "dtype": "bf16",
         "scale": 1.0},
        # a large-width micro-batch with the square-root scaling of the table
        {"name": "embedding large", "op": "embedding", "tokens": 32768, "vocab": 128100, "hidden": 1024, "dtype": "bf16",
         "scale": 32.0},
        # one short sentence on a small synthetic vocabulary
        {"name": "embedding sentence", "op": "embedding", "tokens": 57, "vocab": 4096, "hidden": 384, "dtype": "fp32",
         "scale": 1.0},
    ]


def _between(rng, low, high):
    """A whole number of [low, high], uniform over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["dropout", "norm", "attention", "embedding"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op in ("dropout", "norm"):
        cols = rng.choice([384, 768, 1024, _between(rng, 8, 2048), 8 * _between(rng, 1, 256)])
        rows = _between(rng, 1, min(32768, (16384 * 1024) // cols))
        p = rng.choice([0.05, 0.1, 0.15, round(rng.uniform(0.01, 0.6), 3)])
        case = {"op": op, "rows": rows, "cols": cols, "dtype": dtype}
        if op == "dropout":
            return {**case, "p": p, "residual": rng.random() < 0.5}
        return {**case, "rms": rng.random() < 0.5, "p": rng.choice([0.0, p])}
    if op == "embedding":
        vocab = rng.choice([128100, 50265, _between(rng, 100, 128100)])
        hidden = rng.choice([384, 768, 1024, 8 * _between(rng, 1, 128), _between(rng, 8, 1024)])
        scale = rng.choice([1.0, round(math.sqrt(hidden), 3)])
        return {"op": op, "tokens": _between(rng, 1, 32768), "vocab": vocab, "hidden": hidden, "dtype": dtype, "scale": scale}
    kind = rng.choice(["disentangled", "rotary"])
    heads = rng.choice([1, 3, 6, 12, 16])
    length = _between(rng, 16, 1024 if kind == "disentangled" else 4096)
    most = max(1, min(16384 // length, 2 * 12 * 4096 * 4096 // (4 * heads * length * length)))
    return {"op": op, "kind": kind, "batch": _between(rng, 1, most), "length": length, "heads": heads,
            "mask": rng.choice(["none", "pad", "docs"]), "p": rng.choice([0.05, 0.1, round(rng.uniform(0.01, 0.5), 3)])}


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))

    def normal(*shape, dtype, scale=1.0, shift=0.0):
        return (torch.randn(*shape, device=dev, generator=g) * scale + shift).to(dtype)

    state = {"case": case, "seed": torch.randint(0, 1 << 62, (1,), device=dev, generator=g)}
    op = case["op"]
    if op == "embedding":
        dtype = _DTYPES[case["dtype"]]
        n, vocab = case["tokens"], case["vocab"]
        rank = torch.rand(n, device=dev, generator=g, dtype=torch.float64)
        ids = (vocab ** rank).long().clamp_(0, vocab - 1)  # frequency of an id falls as its inverse
        ids[torch.rand(n, device=dev, generator=g) < 0.15] = min(4, vocab - 1)  # the mask token
        ids[torch.rand(n, device=dev, generator=g) < 0.05] = 0  # padding, which has no gradient
        state.update(ids=ids, table=normal(vocab, case["hidden"], dtype=dtype, scale=0.02).requires_grad_(True),
                     grad=normal(n, case["hidden"], dtype=dtype))
    elif op == "attention":
        b, s, h = case["batch"], case["length"], case["heads"]
        for name in ("q", "k", "v"):
            state[name] = normal(b, s, h * HEAD, dtype=torch.bfloat16).requires_grad_(True)
        state["grad"] = normal(b, s, h * HEAD, dtype=torch.bfloat16)
        state["keep"] = state["docs"] = None
        if case["mask"] == "pad":
            kept = torch.randint(max(1, s // 2), s + 1, (b, 1), device=dev, generator=g)
            kept[-1] = 0 if b > 1 else s - s // 4  # the last row of a batch is empty
            state["keep"] = torch.arange(s, device=dev)[None] < kept
        elif case["mask"] == "docs":
            starts = torch.rand(b, s, device=dev, generator=g) < 1.0 / 300
            docs = 1 + starts.long().cumsum(1)
            docs[:, s - s // 16:] = 0
            state["docs"] = docs
        if case["kind"] == "disentangled":
            state["pos_k"] = normal(2 * SPAN, h * HEAD, dtype=torch.bfloat16).requires_grad_(True)
            state["pos_q"] = normal(2 * SPAN, h * HEAD, dtype=torch.bfloat16).requires_grad_(True)
        else:
            rate = 10000.0 ** (-torch.arange(0, HEAD, 2, device=dev, dtype=torch.float64) / HEAD)
            angle = torch.arange(s, device=dev, dtype=torch.float64)[:, None] * rate.repeat_interleave(2)[None]
            state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    else:
        dtype, rows, cols = _DTYPES[case["dtype"]], case["rows"], case["cols"]
        state["x"] = normal(rows, cols, dtype=dtype).requires_grad_(True)
        state["residual"] = normal(rows, cols, dtype=dtype).requires_grad_(True)
        state["grad"] = normal(rows, cols, dtype=dtype)
        if op == "norm":
            state["grad_total"] = normal(rows, cols, dtype=dtype)
            state["weight"] = normal(cols, dtype=dtype, scale=0.1, shift=1.0).requires_grad_(True)
            state["bias"] = None if case["rms"] else normal(cols, dtype=dtype, scale=0.1).requires_grad_(True)
            state["eps"] = 1e-6
    return state


def run(state):
    op = state["case"]["op"]
    if own:
        return {"dropout": _own_dropout, "norm": _own_norm, "attention": _own_attention, "embedding": _own_embedding}[op](state)
    with torch.no_grad():
        return {"dropout": _dropout, "norm": _norm, "attention": _attention, "embedding": _embedding}[op](state)


# ---- the framework's entry points -------------------------------------------------------------------------------------
def _own_dropout(s):
    from deberta_b200.ops.dropout import dropout, dropout_add

    p = s["case"]["p"]
    out = dropout_add(s["x"], s["residual"], p, s["seed"]) if s["case"]["residual"] else dropout(s["x"], p, s["seed"])
    (dx,) = torch.autograd.grad(out, (s["x"],), s["grad"])
    return {"out": out, "dx": dx}


def _own_norm(s):
    from deberta_b200.ops.norm import add_layer_norm, add_rms_norm

    kw = {"dropout_p": s["case"]["p"], "seed": s["seed"]}
    leaves = {"dx": s["x"], "dresidual": s["residual"], "dweight": s["weight"]}
    if s["case"]["rms"]:
        y, total = add_rms_norm(s["x"], s["residual"], s["weight"], s["eps"], **kw)
    else:
        y, total = add_layer_norm(s["x"], s["residual"], s["weight"], s["bias"], s["eps"], **kw)
        leaves["dbias"] = s["bias"]
    grads = torch.autograd.grad((y, total), tuple(leaves.values()), (s["grad"], s["grad_total"]))
    return {"y": y, "total": total, **dict(zip(leaves, grads))}


def _own_attention(s):
    from deberta_b200.ops.attention import disentangled_attention, rope_attention

    c = s["case"]
    kw = {"heads": c["heads"], "key_keep": s["keep"], "doc_ids": s["docs"], "dropout_p": c["p"], "training": True,
          "dropout_seed": s["seed"]}
    leaves = {"dq": s["q"], "dk": s["k"], "dv": s["v"]}
    if c["kind"] == "disentangled":
        out = disentangled_attention(s["q"], s["k"], s["v"], s["pos_k"], s["pos_q"], scale_factor=3, bucket_size=BUCKETS,
                                     max_position=MAX_POSITION, att_span=SPAN, **kw)
        leaves.update(dpos_k=s["pos_k"], dpos_q=s["pos_q"])
    else:
        out = rope_attention(s["q"], s["k"], s["v"], s["cos"], s["sin"], rotary_dim=HEAD, **kw)
    return {"out": out, **dict(zip(leaves, torch.autograd.grad(out, tuple(leaves.values()), s["grad"])))}


def _own_embedding(s):
    from deberta_b200.ops.embedding import scaled_embedding

    out = scaled_embedding(s["ids"], s["table"], s["case"]["scale"], padding_idx=0)
    (dtable,) = torch.autograd.grad(out, (s["table"],), s["grad"])
    return {"out": out, "dtable": dtable}


# ---- plain forms -------------------------------------------------------------------------------------------------------
def _threshold(p):
    return int(p * 65536 + 0.5)


def _factor(rows, cols, p, seed):
    """fp32 ``[rows, cols]``: 0 for dropped places, the inverse of the kept share elsewhere.

    Column c of row r takes 16 of the 128 bits of Philox4x32 with seven rounds (Salmon, Moraes, Dror and Shaw, "Parallel
    random numbers: as easy as 1, 2, 3", SC 2011) at counter (c >> 3, r mod 2^32, r >> 32, 0) under the seed's 64 bits,
    and is kept where they are at least ``p`` in units of 2^-16."""
    dev, t = seed.device, _threshold(p)
    row = torch.arange(rows, device=dev)[:, None]
    c0, c1, c2 = torch.arange((cols + 7) // 8, device=dev)[None, :], row & _LOW, row >> 32
    c3 = torch.zeros_like(row)
    k0, k1 = seed & _LOW, (seed >> 32) & _LOW
    for _ in range(7):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # modulo 2^64, as the type has it
        c0, c1, c2, c3 = ((b >> 32) & _LOW) ^ c1 ^ k0, b & _LOW, ((a >> 32) & _LOW) ^ c3 ^ k1, a & _LOW
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    words = torch.stack(torch.broadcast_tensors(c0, c1, c2, c3), dim=-1)
    halves = torch.stack((words & 0xFFFF, words >> 16), dim=-1).reshape(rows, -1)[:, :cols]
    return (halves >= t).float() * (65536.0 / max(1, 65536 - t))


def _dropout(s):
    x, f = s["x"], _factor(s["case"]["rows"], s["case"]["cols"], s["case"]["p"], s["seed"])
    out = x.float() * f
    if s["case"]["residual"]:
        out = out + s["residual"].float()
    return {"out": out.to(x.dtype), "dx": (s["grad"].float() * f).to(x.dtype)}


def _norm(s):
    c, dtype = s["case"], s["x"].dtype
    f = _factor(c["rows"], c["cols"], c["p"], s["seed"]) if c["p"] else 1.0
    total = s["residual"].float() + s["x"].float() * f
    w, dy = s["weight"].float(), s["grad"].float()
    centred = total if c["rms"] else total - total.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + s["eps"])
    unit = centred * rstd
    y = unit * w if c["rms"] else unit * w + s["bias"].float()
    g = dy * w
    d = g - unit * (g * unit).mean(-1, keepdim=True)
    if not c["rms"]:
        d = d - g.mean(-1, keepdim=True)
    dtotal = d * rstd + s["grad_total"].float()
    out = {"y": y, "total": total, "dx": dtotal * f, "dresidual": dtotal, "dweight": (dy * unit).sum(0)}
    if not c["rms"]:
        out["dbias"] = dy.sum(0)
    return {name: t.to(dtype) for name, t in out.items()}


def _bucket_rows(length, dev):
    """Rows of the two position tables that each (query, key) pair reads: ``[S, S]`` twice."""
    at = torch.arange(length, device=dev)
    rel = (at[:, None] - at[None, :]).clamp(1 - MAX_POSITION, MAX_POSITION - 1)
    mid = BUCKETS // 2
    far = torch.log(rel.abs().clamp_min(1).double() / mid) / math.log((MAX_POSITION - 1) / mid) * (mid - 1)
    far = (torch.ceil(far - 1e-9).long() + mid) * torch.sign(rel)  # (the last bucket's edge is a whole number)
    rel = torch.where(rel.abs() < mid, rel, far).clamp(-SPAN, SPAN)
    return (rel + SPAN).clamp(0, 2 * SPAN - 1), (SPAN - rel).clamp(0, 2 * SPAN - 1)


def _turn(x, cos, sin):
    """Rotates the pairs of neighbouring columns of ``[B, heads, S, 64]``."""
    even, odd = x[..., 0::2], x[..., 1::2]
    c, sn = cos[:, 0::2], sin[:, 0::2]
    return torch.stack((even * c - odd * sn, odd * c + even * sn), dim=-1).flatten(-2)


def _attention(s):
    c, dev = s["case"], s["q"].device
    b, n, h = c["batch"], c["length"], c["heads"]
    split = lambda x: x.float().view(-1, n, h, HEAD).transpose(1, 2)  # noqa: E731
    merge = lambda x: x.transpose(1, 2).reshape(b, n, h * HEAD).to(torch.bfloat16)  # noqa: E731
    q, k, v, do = split(s["q"]), split(s["k"]), split(s["v"]), split(s["grad"])
    position = c["kind"] == "disentangled"
    if position:
        pk = s["pos_k"].float().view(2 * SPAN, h, HEAD).transpose(0, 1)
        pq = s["pos_q"].float().view(2 * SPAN, h, HEAD).transpose(0, 1)
        to_key, to_query = (i.expand(b, h, n, n) for i in _bucket_rows(n, dev))
        scores = q @ k.transpose(-1, -2) + (q @ pk.transpose(-1, -2)).gather(-1, to_key)
        scores += (k @ pq.transpose(-1, -2)).gather(-1, to_query.transpose(-1, -2)).transpose(-1, -2)
        scale = 1.0 / math.sqrt(3.0 * HEAD)
    else:
        q, k = _turn(q, s["cos"], s["sin"]), _turn(k, s["cos"], s["sin"])
        scores, scale = q @ k.transpose(-1, -2), 1.0 / math.sqrt(HEAD)
    scores *= scale
    seen = torch.ones(b, n, n, dtype=torch.bool, device=dev)
    if s["keep"] is not None:
        seen = s["keep"][:, :, None] & s["keep"][:, None, :]
    elif s["docs"] is not None:
        seen = (s["docs"][:, :, None] == s["docs"][:, None, :]) & (s["docs"] != 0)[:, :, None]
    scores = scores.masked_fill(~seen[:, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    prob = e / e.sum(-1, keepdim=True).clamp_min(1e-30)  # rows that see nothing stay zero
    f = _factor(b * h * n, n, c["p"], s["seed"]).view(b, h, n, n)
    dropped = prob * f
    out = dropped @ v
    dv = dropped.transpose(-1, -2) @ do
    dp = (do @ v.transpose(-1, -2)) * f
    ds = prob * (dp - (prob * dp).sum(-1, keepdim=True)) * scale
    dq, dk = ds @ k, ds.transpose(-1, -2) @ q
    if not position:
        return {"out": merge(out), "dq": merge(_turn(dq, s["cos"], -s["sin"])), "dk": merge(_turn(dk, s["cos"], -s["sin"])),
                "dv": merge(dv)}
    by_key = torch.zeros(b, h, n, 2 * SPAN, device=dev).scatter_add_(-1, to_key, ds)
    by_query = torch.zeros(b, h, n, 2 * SPAN, device=dev).scatter_add_(-1, to_query.transpose(-1, -2), ds.transpose(-1, -2))
    dq, dk = dq + by_key @ pk, dk + by_query @ pq
    table = lambda g, x: (g.transpose(-1, -2) @ x).sum(0).transpose(0, 1).reshape(2 * SPAN, h * HEAD).to(torch.bfloat16)  # noqa: E731
    return {"out": merge(out), "dq": merge(dq), "dk": merge(dk), "dv": merge(dv), "dpos_k": table(by_key, q),
            "dpos_q": table(by_query, k)}


def _embedding(s):
    ids, table, scale = s["ids"], s["table"], s["case"]["scale"]
    out = (table[ids].float() * scale).to(table.dtype)
    rows = s["grad"].float() * (ids != 0)[:, None]
    dtable = torch.zeros(table.shape, device=table.device).index_add_(0, ids, rows) * scale
    return {"out": out, "dtable": dtable.to(table.dtype)}


# ---- what it costs at least -------------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    size = 4 if case.get("dtype") == "fp32" else 2
    if op == "embedding":
        n, v, h = case["tokens"], case["vocab"], case["hidden"]
        rows = min(n, v)  # table rows that are read, at most
        return {"bytes": size * h * (rows + 2 * n + v) + 16 * n, "flops": 2 * n * h}
    if op == "attention":
        b, n, h = case["batch"], case["length"], case["heads"]
        tables = 4 * 2 * SPAN * h * HEAD if case["kind"] == "disentangled" else 0
        # what a document mask leaves of the map: about 300 of the row's keys at a time, twice that seen from a key
        pairs = b * h * n * (min(n, 600) if case["mask"] == "docs" else n)
        if case["mask"] == "pad":
            pairs = pairs * 0.55
        return {"bytes": 2 * (8 * b * n * h * HEAD + tables), "flops": 14 * HEAD * pairs}
    cells = case["rows"] * case["cols"] * size
    if op == "dropout":
        return {"bytes": cells * (5 if case["residual"] else 4), "flops": 12 * case["rows"] * case["cols"]}
    return {"bytes": cells * (4 + 4 + (case["p"] > 0)) + 6 * size * case["cols"], "flops": 30 * case["rows"] * case["cols"]}


# ---- definitions in 64 bits -------------------------------------------------------------------------------------------
def _exact_kept(rows, cols, p, seed):
    """bool ``[rows, cols]`` of the kept places. The products are built from 16-bit pieces, so no step wraps."""
    dev = seed.device
    group = torch.arange(-(-cols // 8), device=dev).repeat(rows)
    row = torch.arange(rows, device=dev).repeat_interleave(-(-cols // 8))
    x = [group, row % 2**32, row // 2**32, torch.zeros_like(row)]
    key = [int(seed) % 2**32, int(seed) // 2**32 % 2**32]

    def times(a, m):
        low = (a & 0xFFFF) * m  # < 2^48
        high = (a >> 16) * m + (low >> 16)  # < 2^49: the product's bits from 16 up
        return high >> 16, ((high & 0xFFFF) << 16) | (low & 0xFFFF)

    for _ in range(7):
        h0, l0 = times(x[0], 0xD2511F53)
        h1, l1 = times(x[2], 0xCD9E8D57)
        x = [h1 ^ x[1] ^ key[0], l1, h0 ^ x[3] ^ key[1], l0]
        key = [(key[0] + 0x9E3779B9) % 2**32, (key[1] + 0xBB67AE85) % 2**32]
    bits = torch.empty(rows * -(-cols // 8), 8, dtype=torch.int32, device=dev)
    for i in range(4):
        bits[:, 2 * i], bits[:, 2 * i + 1] = x[i] % 65536, x[i] // 65536
    return (bits >= math.floor(p * 65536 + 0.5)).view(rows, -1)[:, :cols]


def _exact_dropout(x, p, seed):
    """Dropout of the last axis of a 64-bit tensor, differentiable."""
    if p == 0:
        return x
    kept = _exact_kept(x.numel() // x.shape[-1], x.shape[-1], p, seed).view(x.shape)
    return torch.where(kept, x / (1 - math.floor(p * 65536 + 0.5) / 65536), torch.zeros((), dtype=x.dtype, device=x.device))


def exact(case, seed):
    s = prepare(case, seed)
    wide = {n: t.detach().double().requires_grad_(t.requires_grad) for n, t in s.items()
            if torch.is_tensor(t) and t.is_floating_point()}
    op = case["op"]
    if op == "dropout":
        out = _exact_dropout(wide["x"], case["p"], s["seed"])
        if case["residual"]:
            out = out + wide["residual"]
        (dx,) = torch.autograd.grad(out, (wide["x"],), wide["grad"])
        return {"out": out.detach(), "dx": dx}
    if op == "norm":
        total = wide["residual"] + _exact_dropout(wide["x"], case["p"], s["seed"])
        leaves = {"dx": wide["x"], "dresidual": wide["residual"], "dweight": wide["weight"]}
        if case["rms"]:
            y = total / (total.pow(2).mean(-1, keepdim=True) + s["eps"]).sqrt() * wide["weight"]
        else:
            leaves["dbias"] = wide["bias"]
            y = (total - total.mean(-1, keepdim=True)) / (total.var(-1, unbiased=False, keepdim=True) + s["eps"]).sqrt()
            y = y * wide["weight"] + wide["bias"]
        grads = torch.autograd.grad((y, total), tuple(leaves.values()), (wide["grad"], wide["grad_total"]))
        return {"y": y.detach(), "total": total.detach(), **dict(zip(leaves, grads))}
    if op == "embedding":
        # one row per distinct token: the rows of its places are summed through the inverse map
        values, place = torch.unique(s["ids"], return_inverse=True)
        sums = torch.zeros(len(values), case["hidden"], dtype=torch.float64, device=values.device)
        sums.index_put_((place,), wide["grad"], accumulate=True)
        dtable = torch.zeros(case["vocab"], case["hidden"], dtype=torch.float64, device=values.device)
        dtable[values] = sums * case["scale"]
        dtable[0] = 0
        return {"out": wide["table"].detach().index_select(0, s["ids"]) * case["scale"], "dtable": dtable}
    return _exact_attention(case, s, wide)


def _exact_attention(case, s, wide):
    b, n, h = case["batch"], case["length"], case["heads"]
    q, k, v = (wide[x].view(b, n, h, HEAD).permute(0, 2, 1, 3) for x in ("q", "k", "v"))
    leaves = {"dq": wide["q"], "dk": wide["k"], "dv": wide["v"]}
    if case["kind"] == "disentangled":
        leaves.update(dpos_k=wide["pos_k"], dpos_q=wide["pos_q"])
        edge, width = BUCKETS // 2, math.log((MAX_POSITION - 1) / (BUCKETS // 2))

        def bucket(d):
            m = min(abs(d), MAX_POSITION - 1)
            if m >= edge:
                m = edge + math.ceil(math.log(m / edge) / width * (edge - 1) - 1e-9)
            return int(math.copysign(m, d))

        offset = torch.arange(n, device=q.device)[:, None] - torch.arange(n, device=q.device)[None, :] + n - 1
        line = torch.tensor([bucket(d) for d in range(1 - n, n)], device=q.device)
        key_row = (line + SPAN).clamp(0, 2 * SPAN - 1)[offset]
        query_row = (SPAN - line).clamp(0, 2 * SPAN - 1)[offset]
        pk, pq = (wide[x].view(2 * SPAN, h, HEAD).permute(1, 2, 0) for x in ("pos_k", "pos_q"))
        rows, cols = torch.arange(n, device=q.device)[:, None], torch.arange(n, device=q.device)[None, :]
        scores = q @ k.transpose(-1, -2) + (q @ pk)[:, :, rows, key_row] + (k @ pq)[:, :, cols, query_row]
        scores = scores / math.sqrt(3 * HEAD)
    else:
        c, sn = wide["cos"][:, ::2], wide["sin"][:, ::2]
        turn = torch.complex(c, sn)
        q, k = (torch.view_as_real(torch.view_as_complex(x.reshape(b, h, n, HEAD // 2, 2)) * turn).flatten(-2) for x in (q, k))
        scores = q @ k.transpose(-1, -2) / math.sqrt(HEAD)
    if s["keep"] is not None:
        live = s["keep"]
        pair = live[:, None, None, :] & live[:, None, :, None]
    elif s["docs"] is not None:
        live = s["docs"] > 0
        pair = ((s["docs"][:, None, :] == s["docs"][:, :, None]) & live[:, :, None])[:, None]
    else:
        live = torch.ones(b, n, dtype=torch.bool, device=q.device)
        pair = live[:, None, None, :]
    prob = torch.softmax(scores.masked_fill(~pair, -1e300), dim=-1) * live[:, None, :, None]
    out = _exact_dropout(prob, case["p"], s["seed"]) @ v
    out = out.permute(0, 2, 1, 3).reshape(b, n, h * HEAD)
    grads = torch.autograd.grad(out, tuple(leaves.values()), wide["grad"])
    return {"out": out.detach(), **dict(zip(leaves, grads))}
