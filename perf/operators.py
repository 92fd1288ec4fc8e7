"""Cases and plain forms of the transformer-layer operators (dorado_amd.ops): RMS norm with the residual's addition and an optional
8-bit output, rotary positions, masked attention.

`own` False: every operator in its plain form, elementary torch operations in 32 bits (64 for the angles of far positions).
`own` True: the calls a user makes of dorado_amd.ops on the same state."""
import math
import random

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
E4M3_MAX = 448.0


# ------------------------------------------------------------------------------------------------------------------ cases
def _norm(name, rows, cols, type, residual=True, total=False, quant="none", group=0, weight="f32"):
    c = {"name": name, "op": "norm", "rows": rows, "cols": cols, "type": type, "residual": residual, "sum": total,
         "quant": quant, "group": group, "weight": weight}
    return c


def _rope(name, batch, tokens, heads, kv_heads, head_dim, rot_dim, type, interleaved=False, scaling="none", positions="start",
          far=0):
    return {"name": name, "op": "rope", "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "rot_dim": rot_dim, "type": type, "interleaved": interleaved, "scaling": scaling,
            "positions": positions, "far": far}


def _att(name, batch, q_tokens, k_tokens, heads, kv_heads, head_dim, type, back=-1, ahead=-1, cap=0.0, slopes=False,
         lengths=False, prefix=0, documents=0, lse=False, packed=False):
    return {"name": name, "op": "attention", "batch": batch, "q_tokens": q_tokens, "k_tokens": k_tokens, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "type": type, "back": back, "ahead": ahead, "cap": cap,
            "slopes": slopes, "lengths": lengths, "prefix": prefix, "documents": documents, "lse": lse, "packed": packed}


def listed():
    return [
        # one new token of 8 sequences, wide model: what a layer does per token when it answers; latency counts
        _norm("norm tokens", 8, 4096, "bf16", total=True, weight="bf16"),
        # the encoder's own width: 256 signal chunks of 1024 tokens, residual scaled and added, normalised in f16
        _norm("norm chunks", 262144, 512, "f16"),
        # a long prompt before an 8-bit product: sum kept for the next layer, e4m3 with one scale per 128 columns
        _norm("norm e4m3 groups", 16383, 4096, "bf16", total=True, quant="e4m3", group=128, weight="bf16"),
        # one new token of 16 sequences at far positions, interleaved pairs, context stretched by parts
        _rope("rope tokens", 16, 1, 32, 8, 128, 128, "bf16", interleaved=True, scaling="by_parts", positions="given", far=1000000),
        # the encoder's own q | k projection (8 heads of 64, f16, half layout), 64 chunks, views of one buffer
        _rope("rope chunks", 64, 1024, 8, 8, 64, 64, "f16"),
        # a very long text, half of each head rotated
        _rope("rope long part", 1, 100001, 32, 8, 128, 64, "bf16", scaling="linear"),
        # one new token of 48 sequences over a cache of up to 8192, ragged lengths, shared heads, scores capped
        _att("attention tokens", 48, 1, 8192, 32, 8, 128, "bf16", ahead=0, cap=30.0, lengths=True),
        # one token against one very long cache: the long axis has to be split
        _att("attention long token", 1, 1, 131072, 16, 2, 128, "bf16", ahead=0),
        # the encoder's own attention: chunks of 1024 tokens, 8 heads of 64, window 127 | 128, q | k | v in one buffer
        _att("attention window", 64, 1024, 1024, 8, 8, 64, "f16", back=127, ahead=128, packed=True),
        # a long prompt, causal, shared heads, capped scores
        _att("attention causal cap", 1, 16384, 16384, 16, 4, 128, "bf16", ahead=0, cap=50.0),
        # documents packed into one batch row, bias by distance, statistics kept
        _att("attention documents", 1, 16000, 16000, 8, 8, 64, "f16", slopes=True, documents=37, lse=True),
        # four prompts whose first part is seen both ways, odd length
        _att("attention prefix", 4, 2111, 2111, 12, 4, 128, "f16", ahead=0, prefix=301, lse=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "rope", "attention", "attention"])
    kind = rng.choice(["f16", "bf16", "bf16", "f16", "f32"]) if op != "attention" else rng.choice(["f16", "bf16"])
    if op == "norm":
        cols = rng.choice([_log(rng, 64, 16384), 8 * _log(rng, 8, 2048), 128 * _log(rng, 1, 128)])
        rows = _log(rng, 1, max(1, min(262144, (1 << 26) // cols)))
        quant = rng.choice(["none", "none", "e4m3", "int8"])
        c = _norm("", rows, cols, kind, residual=rng.random() < 0.7, total=rng.random() < 0.5, quant=quant,
                  group=128 if quant != "none" and cols % 128 == 0 and rng.random() < 0.5 else 0,
                  weight=rng.choice(["f32", kind]))
    elif op == "rope":
        hd = rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
        kvh = rng.choice([1, 2, 4, 8])
        batch = _log(rng, 1, 64)
        heads = kvh * rng.choice([1, 2, 3, 4])
        tokens = _log(rng, 1, max(1, min(100000, (1 << 27) // (batch * heads * hd))))
        c = _rope("", batch, tokens, heads, kvh, hd, rng.choice([hd, hd, hd // 2]), kind, interleaved=rng.random() < 0.5,
                  scaling=rng.choice(["none", "linear", "base", "by_parts"]), positions=rng.choice(["start", "given"]),
                  far=rng.choice([0, 4097, 1000000]))
    else:
        hd = rng.choice([64, 128])
        kvh = rng.choice([1, 2, 4, 8])
        heads = kvh * rng.choice([1, 1, 2, 4, 7])
        cap = rng.choice([0.0, 0.0, 30.0, 50.0])
        slopes = rng.random() < 0.3
        shape = rng.choice(["token", "self", "self", "cross", "documents"])
        if shape == "token":
            batch = _log(rng, 1, 64)
            k_tokens = _log(rng, 1, max(1, min(131072, (1 << 28) // (batch * kvh * hd))))
            q_tokens = min(k_tokens, rng.choice([1, 1, 1, 2, 5]))
            c = _att("", batch, q_tokens, k_tokens, heads, kvh, hd, kind, ahead=0, cap=cap, slopes=slopes,
                     back=rng.choice([-1, -1, 1023]), lengths=rng.random() < 0.6)
        else:
            most = (1 << 31) // heads    # score elements of one head over the batch
            batch = 1 if shape == "documents" else _log(rng, 1, 16)
            tokens = _log(rng, 16, max(16, min(12288, int(math.sqrt(most / batch)))))
            if shape == "documents":
                c = _att("", 1, tokens, tokens, heads, kvh, hd, kind, back=rng.choice([-1, 255]), ahead=rng.choice([-1, 0]),
                         cap=cap, slopes=slopes, documents=1 + _log(rng, 1, max(1, tokens // 8)), lse=rng.random() < 0.5)
            elif shape == "cross":
                q_tokens = _log(rng, 6, tokens)
                c = _att("", batch, q_tokens, tokens, heads, kvh, hd, kind, ahead=rng.choice([-1, 0]), cap=cap, slopes=slopes,
                         lengths=rng.random() < 0.5, lse=rng.random() < 0.5)
            else:
                back, ahead = rng.choice([(-1, -1), (-1, 0), (127, 128), (500, 0)])
                c = _att("", batch, tokens, tokens, heads, kvh, hd, kind, back=back, ahead=ahead, cap=cap, slopes=slopes,
                         prefix=_log(rng, 1, tokens) if ahead == 0 and rng.random() < 0.5 else 0, lse=rng.random() < 0.5,
                         packed=rng.random() < 0.5)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------- what belongs to a case
def _lengths(case):
    """Keys in use per batch row: the last row's cache is full, the others hold between a quarter and all of it."""
    r, n = random.Random(case["k_tokens"] * 31 + case["batch"]), case["k_tokens"]
    return [n if b == case["batch"] - 1 else r.randint(max(1, n // 4), n) for b in range(case["batch"])]


def _offsets(case):
    """Document borders: cuts at random places, a few tokens behind the last document belong to none."""
    r, n = random.Random(case["documents"] * 17 + case["q_tokens"]), case["q_tokens"]
    end = n - n // 100
    cuts = sorted(r.randint(1, max(1, end)) for _ in range(case["documents"] - 1))
    return [0] + cuts + [end]


def _seen(n, m, start, back, ahead, prefix):
    """Visible (query, key) pairs of n queries at positions start.. over m keys."""
    total = 0
    for i in range(start, start + n):
        lo = max(0, i - back) if back >= 0 else 0
        hi = min(m, i + ahead + 1) if ahead >= 0 else m
        p = min(prefix, m)
        w = max(0, hi - lo)
        total += w + p - max(0, min(hi, p) - lo if w else 0)
    return total


def _frequencies(case, dtype):
    """Radians per position of each rotated pair, and the factor on the result."""
    d = case["rot_dim"]
    i = torch.arange(d // 2, dtype=dtype)
    theta, factor, length = 10000.0, 8.0, 4096.0
    if case["scaling"] == "base":       # a larger base: the lowest frequency slows by the factor, the highest stays
        theta = theta * factor ** (d / (d - 2)) if d > 2 else theta
    f = theta ** (-2.0 * i / d)
    if case["scaling"] == "linear":     # positions squeezed
        f = f / factor
    if case["scaling"] == "by_parts":   # pairs with few turns over the trained length are squeezed, fast ones stay
        turns = length * f / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        f = f * (keep + (1 - keep) / factor)
        return f, 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _randn(g, shape, dtype, mul=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * mul).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = TYPES[case["type"]]
    s = {"case": case}
    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        s["x"] = _randn(g, (rows, cols), dt, 2.0)
        s["residual"] = _randn(g, (rows, cols), dt) if case["residual"] else None
        s["weight"] = (1.0 + 0.2 * _randn(g, (cols,), torch.float32)).to(TYPES[case["weight"]])
        s["alpha"] = 2.5 if case["type"] == "f16" else 1.0   # the f16 encoder scales its residual
    elif case["op"] == "rope":
        b, t, h, kh, d = (case[k] for k in ("batch", "tokens", "heads", "kv_heads", "head_dim"))
        both = _randn(g, (b, t, h + kh, d), dt)
        s["q"], s["k"] = both[:, :, :h], both[:, :, h:]      # views of one projection's result
        f, s["amplitude"] = _frequencies(case, torch.float64)
        s["freqs"] = f.cuda()
        s["positions"] = None
        if case["positions"] == "given":
            s["positions"] = torch.randint(0, case["far"] + t, (b, t), generator=g, device="cuda")
    else:
        b, n, m, h, kh, d = (case[k] for k in ("batch", "q_tokens", "k_tokens", "heads", "kv_heads", "head_dim"))
        if case["packed"]:
            qkv = _randn(g, (b, n, h + 2 * kh, d), dt)
            s["q"], s["k"], s["v"] = qkv[:, :, :h], qkv[:, :, h:h + kh], qkv[:, :, h + kh:]
        else:
            s["q"], s["k"], s["v"] = (_randn(g, (b, c, x, d), dt) for c, x in ((n, h), (m, kh), (m, kh)))
        s["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], device="cuda") if case["slopes"] else None
        s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda") if case["lengths"] else None
        s["offsets"] = torch.tensor(_offsets(case), dtype=torch.int32, device="cuda") if case["documents"] else None
        s["prefix"] = torch.full((b,), case["prefix"], dtype=torch.int32, device="cuda") if case["prefix"] else None
    return s


# ------------------------------------------------------------------------------------------------------------ plain forms
def _plain_norm(s):
    c = s["case"]
    x = s["x"].float()
    if c["residual"]:
        x = x + s["alpha"] * s["residual"].float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5) * s["weight"].float()
    dt = s["x"].dtype
    total = (x.to(dt),) if c["sum"] else ()
    if c["quant"] == "none":
        return (y.to(dt),) + total
    g = y.view(c["rows"], -1, c["group"] or c["cols"])
    top = g.abs().amax(-1, keepdim=True)
    scale = torch.where(top == 0, torch.ones_like(top), top / (E4M3_MAX if c["quant"] == "e4m3" else 127.0))
    if c["quant"] == "e4m3":
        q = (g / scale).to(torch.float8_e4m3fn).view(c["rows"], c["cols"])
    else:
        q = (g / scale).round().to(torch.int8).view(c["rows"], c["cols"])
    return _quantised(c, dt, q, scale.view(c["rows"], -1)) + total


def _quantised(c, dt, q, scale):
    """8-bit floats and their scales as they are; whole numbers as the values they stand for."""
    if c["quant"] == "e4m3":
        return (q, scale)
    g = q.view(c["rows"], -1, c["group"] or c["cols"])
    return ((g * scale[:, :, None]).to(torch.float16 if dt == torch.float32 else dt).view(c["rows"], c["cols"]), scale)


def _plain_rotate(x, cos, sin, c):
    r, half = c["rot_dim"], c["rot_dim"] // 2
    f = x.float()
    a, b = (f[..., 0:r:2], f[..., 1:r:2]) if c["interleaved"] else (f[..., :half], f[..., half:r])
    u, v = a * cos - b * sin, a * sin + b * cos
    y = torch.stack((u, v), -1).flatten(-2) if c["interleaved"] else torch.cat((u, v), -1)
    return torch.cat((y, f[..., r:]), -1).to(x.dtype)


def _plain_rope(s):
    c = s["case"]
    p = s["positions"]
    if p is None:
        p = torch.arange(c["far"], c["far"] + c["tokens"], device=s["q"].device)[None]
    angle = p[..., None].double() * s["freqs"]
    cos = (angle.cos() * s["amplitude"]).float()[:, :, None]
    sin = (angle.sin() * s["amplitude"]).float()[:, :, None]
    return _plain_rotate(s["q"], cos, sin, c), _plain_rotate(s["k"], cos, sin, c)


def _plain_visible(s):
    """[batch or 1][query][key]: which keys a query sees, and both their positions."""
    c = s["case"]
    j = torch.arange(c["k_tokens"], device=s["q"].device)[None, None]
    t = torch.arange(c["q_tokens"], device=s["q"].device)[None, :, None]
    length = s["lengths"].long()[:, None, None] if c["lengths"] else torch.full_like(j[:, :, :1], c["k_tokens"])
    i = t + length - c["q_tokens"]
    see = torch.ones_like(i == j)
    if c["back"] >= 0:
        see = see & (j >= i - c["back"])
    if c["ahead"] >= 0:
        see = see & (j <= i + c["ahead"])
    if c["prefix"]:
        see = see | (j < s["prefix"].long()[:, None, None])
    see = see & (j < length)
    if c["documents"]:
        o = s["offsets"].long()
        mine = (t >= o).sum(-1, keepdim=True)
        its = (j[..., None] >= o).sum(-1)
        see = see & (mine == its) & (mine > 0) & (mine < o.numel())
    return see, (i - j).abs()


def _plain_attention(s):
    c = s["case"]
    b, n, m, h, kh, d = (c[k] for k in ("batch", "q_tokens", "k_tokens", "heads", "kv_heads", "head_dim"))
    q = s["q"].float().transpose(1, 2).reshape(b, kh, h // kh * n, d)
    k = s["k"].float().permute(0, 2, 3, 1)
    score = torch.matmul(q, k).view(b, h, n, m).mul_(d ** -0.5)
    if c["cap"]:
        score = torch.tanh(score / c["cap"]) * c["cap"]
    see, far = _plain_visible(s)
    if c["slopes"]:
        score = score - s["slopes"][None, :, None, None] * far[:, None]
    score = score.masked_fill(~see[:, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    base = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = torch.exp(score - base)
    total = p.sum(-1, keepdim=True)
    v = s["v"].float().transpose(1, 2)
    out = torch.matmul(p.view(b, kh, h // kh * n, m), v).view(b, h, n, d)
    out = torch.where(total > 0, out / total, torch.zeros_like(out)).transpose(1, 2).contiguous().to(s["q"].dtype)
    return (out, (base + torch.log(total))[..., 0]) if c["lse"] else (out,)


# -------------------------------------------------------------------------------------------------------------------- run
def _own(s):
    from dorado_amd import ops

    c = s["case"]
    if c["op"] == "norm":
        r = ops.rms_norm(s["x"], s["weight"], residual=s["residual"], alpha=s["alpha"], eps=1e-5,
                         quant=None if c["quant"] == "none" else c["quant"], group=c["group"], return_sum=c["sum"])
        r = r if isinstance(r, tuple) else (r,)
        return r if c["quant"] == "none" else _quantised(c, s["x"].dtype, r[0], r[1]) + r[2:]
    if c["op"] == "rope":
        return ops.rope(s["q"], s["k"], freqs=s["freqs"], positions=s["positions"], start=c["far"],
                        interleaved=c["interleaved"], amplitude=s["amplitude"])
    r = ops.attention(s["q"], s["k"], s["v"], window=(c["back"], c["ahead"]), softcap=c["cap"], slopes=s["slopes"],
                      k_len=s["lengths"], prefix=s["prefix"], doc_offsets=s["offsets"], return_lse=c["lse"])
    return r if isinstance(r, tuple) else (r,)


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "rope": _plain_rope, "attention": _plain_attention}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------------------------- work
def _hull(n, m, start, back, ahead, prefix):
    """Keys that at least one of n queries at positions start.. sees."""
    lo = max(0, start - back) if back >= 0 else 0
    hi = max(0, min(m, start + n + ahead)) if ahead >= 0 else m
    lo = min(lo, hi)
    p = min(prefix, m)
    return hi - lo + p - max(0, min(hi, p) - lo)


def work(case):
    e = {"f16": 2, "bf16": 2, "f32": 4}[case["type"]]
    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        n = rows * cols
        out = n * e if case["quant"] == "none" else n + 4 * rows * (cols // (case["group"] or cols))
        return {"bytes": n * e * (1 + case["residual"] + case["sum"]) + out + cols * (4 if case["weight"] == "f32" else e),
                "flops": 6 * n}
    if case["op"] == "rope":
        tokens = case["batch"] * case["tokens"]
        n = tokens * (case["heads"] + case["kv_heads"])
        return {"bytes": 2 * n * case["head_dim"] * e + (8 * tokens if case["positions"] == "given" else 0),
                "flops": 3 * n * case["rot_dim"]}
    b, n, m, h, kh, d = (case[k] for k in ("batch", "q_tokens", "k_tokens", "heads", "kv_heads", "head_dim"))
    rule = (case["back"], case["ahead"], case["prefix"])
    if case["documents"]:
        o = _offsets(case)
        parts = [(y - x, y - x, 0) for x, y in zip(o, o[1:])]
    else:
        parts = [(n, x, x - n) for x in (_lengths(case) if case["lengths"] else [m] * b)]
    pairs = sum(_seen(*p, *rule) for p in parts)
    keys = sum(_hull(*p, *rule) for p in parts)
    return {"bytes": e * (2 * b * n * h * d + 2 * keys * kh * d) + (4 * b * n * h if case["lse"] else 0),
            "flops": 4 * d * h * pairs}


# ------------------------------------------------------------------------------------------------------------------ exact
def _exact_norm(s):
    c, dt = s["case"], torch.float64
    rows, cols = c["rows"], c["cols"]
    out, sums, scales = [], [], []
    for x, r in zip(s["x"].split(8192), s["residual"].split(8192) if c["residual"] else s["x"].split(8192)):
        a = x.to(dt)
        if c["residual"]:
            a += s["alpha"] * r.to(dt)
        y = a / (a.pow(2).sum(1, keepdim=True) / cols + 1e-5).sqrt() * s["weight"].to(dt)
        if c["quant"] != "none":
            g = y.reshape(y.shape[0], -1, c["group"] or cols)
            top = g.abs().amax(2)
            scale = top / (E4M3_MAX if c["quant"] == "e4m3" else 127.0)
            scale[top == 0] = 1.0
            scales.append(scale)
            g = g / scale[:, :, None]
            y = (g if c["quant"] == "e4m3" else g.round() * scale[:, :, None]).reshape(y.shape)
        out.append(y)
        sums.append(a)
    r = [torch.cat(out)]
    if c["quant"] != "none":
        r.append(torch.cat(scales))
    if c["sum"]:
        r.append(torch.cat(sums))
    return tuple(r)


def _exact_rope(s):
    c, dt = s["case"], torch.float64
    r = c["rot_dim"]
    p = s["positions"] if s["positions"] is not None else torch.arange(c["tokens"], device=s["q"].device)[None] + c["far"]
    turn = torch.polar(torch.full_like(p[..., None] * s["freqs"], s["amplitude"]), p[..., None] * s["freqs"])[:, :, None]
    got = []
    for x in (s["q"], s["k"]):
        y = x.to(dt)
        pair = y[..., :r].unflatten(-1, (r // 2, 2)) if c["interleaved"] else y[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
        z = z.flatten(-2) if c["interleaved"] else z.transpose(-1, -2).flatten(-2)
        got.append(torch.cat((z, y[..., r:]), -1))
    return tuple(got)


def _exact_rows(q, k, v, lo, hi, start, scale, cap, slope, head):
    """One head: queries q at positions start.., each over its keys [0, head) and [lo, hi)."""
    j = torch.arange(k.shape[0], device=q.device)
    score = q @ k.T * scale
    if cap:
        score = cap * torch.tanh(score / cap)
    if slope is not None:
        i = torch.arange(start, start + q.shape[0], device=q.device)
        score = score - slope.double() * (i[:, None] - j).abs()
    hidden = ((j < lo[:, None]) | (j >= hi[:, None])) & (j >= head)
    lse = torch.logsumexp(score.masked_fill(hidden, -math.inf), 1)
    p = torch.exp(score - lse[:, None].nan_to_num(neginf=0.0)).masked_fill(hidden, 0.0)
    return p @ v, lse


def _exact_attention(s):
    c = s["case"]
    b, n, m, h, kh, d = (c[k] for k in ("batch", "q_tokens", "k_tokens", "heads", "kv_heads", "head_dim"))
    out = torch.zeros(b, n, h, d, dtype=torch.float64, device=s["q"].device)
    lse = torch.full((b, h, n), -math.inf, dtype=torch.float64, device=s["q"].device)
    if c["documents"]:
        o = _offsets(c)
        parts = [(0, x, y - x, x, y - x, 0) for x, y in zip(o, o[1:]) if y > x]   # row, first query, queries, first key, keys, position
    else:
        size = _lengths(c) if c["lengths"] else [m] * b
        parts = [(r, 0, n, 0, size[r], size[r] - n) for r in range(b)]
    for row, q0, nq, k0, nk, at in parts:
        for x in range(h):
            k, v = (s[y][row, k0:k0 + nk, x * kh // h].double() for y in ("k", "v"))
            for first in range(0, nq, 4096):
                count = min(4096, nq - first)
                q = s["q"][row, q0 + first:q0 + first + count, x].double()
                i = torch.arange(at + first, at + first + count, device=q.device)
                lo = (i - c["back"]).clamp(min=0) if c["back"] >= 0 else torch.zeros_like(i)
                hi = (i + c["ahead"] + 1).clamp(max=nk) if c["ahead"] >= 0 else torch.full_like(i, nk)
                y, z = _exact_rows(q, k, v, lo, hi, at + first, d ** -0.5, c["cap"], s["slopes"][x] if c["slopes"] else None,
                                   min(c["prefix"], nk))
                out[row, q0 + first:q0 + first + count, x] = y
                lse[row, x, q0 + first:q0 + first + count] = z
    return (out, lse) if c["lse"] else (out,)


def exact(case, seed):
    if case["op"] == "attention":
        # about 2 ms for each head of a part, and the products of 64-bit numbers
        parts = case["documents"] or case["batch"]
        if parts * case["heads"] > 4000 or work(case)["flops"] > 4e12:
            return None
    s = prepare(case, seed)
    return {"norm": _exact_norm, "rope": _exact_rope, "attention": _exact_attention}[case["op"]](s)
