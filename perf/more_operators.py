"""Measured cases of the attention operators: the norm of queries and keys for each head with
the rotation by positions (one or several axes) and its backward pass, and attention with a
sliding window and first tokens that stay visible: prompts, padded training batches, single
tokens over a cache, and its backward pass.

``run`` computes a case in plain torch operations (binary32, angles in binary64, rounded once
at the end), or, with ``own`` set, through the library's entry points.  ``exact`` is the same
in binary64.  Sizes are generic ones of transformer attention layers; 16384 tokens are the rows
of the repository's layer norm workload."""
import math

import torch

own = False

EPS = 1e-6
DT = {"f16": torch.float16, "f32": torch.float32}
ES = {"f16": 2, "f32": 4}


def _rot(name, op, dtype, tokens, hq, hk, d, rot, sections=(0, 0, 0), pairs=False, packed=True, far=0):
    """tokens with hq query and hk key heads of d columns, the first rot of them rotated.
    sections: pairs that go by the time, height and width axis (0, 0, 0: one axis); pairs:
    neighbouring columns are a pair, else column i and i + rot / 2; packed: queries and keys
    are views of one [tokens, hq + 2 hk, d] projection; far: the first token's position."""
    return {"name": name, "op": op, "dtype": dtype, "tokens": tokens, "hq": hq, "hk": hk, "d": d, "rot": rot,
            "s0": sections[0], "s1": sections[1], "s2": sections[2], "pairs": pairs, "packed": packed, "far": far}


def _att(name, op, dtype, b, sq, sk, hq, hk, d, window=0, sinks=0, ragged=False, keep=False):
    """b sequences of sq queries over sk keys; window 0: all earlier tokens; sinks: first tokens
    that stay visible; ragged: each sequence has a length of its own; keep: the forward pass also
    returns each row's logarithm of the sum of exponentials."""
    return {"name": name, "op": op, "dtype": dtype, "b": b, "sq": sq, "sk": sk, "hq": hq, "hk": hk, "d": d,
            "window": window, "sinks": sinks, "ragged": ragged, "keep": keep}


def listed():
    return [
        # one new token of each of 8 sequences, far into their contexts: latency
        _rot("rotary_8_f16", "rot", "f16", 8, 32, 8, 128, 128, far=100000),
        # a training batch or a long prompt
        _rot("rotary_16384_f16", "rot", "f16", 16384, 32, 8, 128, 128),
        # images and video: three axes, neighbouring columns as pairs
        _rot("rotary_3001_f32", "rot", "f32", 3001, 16, 16, 80, 80, sections=(8, 16, 16), pairs=True),
        # the training batch's gradients
        _rot("rotary_bwd_16384_f16", "rot_bwd", "f16", 16384, 32, 8, 128, 128),
        # half of each head rotated, an odd number of pairs: no vector access fits
        _rot("rotary_bwd_515_f32", "rot_bwd", "f32", 515, 12, 4, 100, 50, packed=False),
        # a long prompt through a windowed layer
        _att("attention_8192_f16", "att", "f16", 1, 8192, 8192, 32, 8, 128, window=4096, sinks=4),
        # a padded training batch, every earlier token visible
        _att("attention_pad_6x1000_f16", "att", "f16", 6, 1000, 1000, 12, 12, 64, ragged=True, keep=True),
        # binary32, ragged sizes
        _att("attention_777_f32", "att", "f32", 2, 777, 777, 8, 2, 80, window=256, sinks=4, keep=True),
        # a batch's next tokens over its cache
        _att("decode_16x8192_f16", "att", "f16", 16, 1, 8192, 32, 8, 128, ragged=True),
        # one sequence's next token in a windowed layer: latency
        _att("decode_1x2000_f16", "att", "f16", 1, 1, 2000, 16, 2, 64, window=512, sinks=4, ragged=True),
        # a training batch's gradients
        _att("attention_bwd_4096_f16", "att_bwd", "f16", 2, 4096, 4096, 16, 2, 128, window=2048, sinks=4),
        # binary32 gradients of a small padded batch
        _att("attention_bwd_200_f32", "att_bwd", "f32", 3, 200, 200, 6, 3, 72, ragged=True),
    ]


def _size(rng, lo, hi):
    """Log-uniform in [lo, hi]."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    dtype = rng.choice(["f16", "f16", "f32"])
    op = rng.choice(["rot", "rot_bwd", "att", "decode", "att_bwd"])
    hk = rng.choice([1, 2, 3, 4, 8])
    hq = hk * rng.choice([1, 2, 3, 4, 8])
    if op in ("rot", "rot_bwd"):
        d = rng.choice([32, 64, 80, 96, 100, 128, 128, 256])
        rot = rng.choice([d, d, d // 2])
        sections = (0, 0, 0)
        if rng.random() < 0.4:
            a = rot // 8
            sections = (rot // 2 - 2 * a, a, a)
        most = 16384 * 40 * 128 * 2 // ((hq + hk) * d * ES[dtype])
        return _rot("", op, dtype, _size(rng, 1, min(16384, most)), hq, hk, d, rot, sections, rng.random() < 0.4,
                    rng.random() < 0.7, rng.choice([0, 0, 5000, 1000000]))
    d = rng.choice([32, 64, 64, 72, 80, 96, 128, 128])
    window, sinks = rng.choice([(0, 0), (0, 0), (_size(rng, 16, 4096), rng.choice([0, 1, 4, 130]))])
    ragged = rng.random() < 0.6
    if op == "decode":
        b = _size(rng, 1, 32)
        sk = _size(rng, 1, min(32768, 16 * 8192 * 8 * 128 * 2 // (b * hk * d * ES[dtype])))
        sq = min(sk, rng.choice([1, 1, 1, 2, 5]))
        return _att("", "att", dtype, b, sq, sk, hq, hk, d, window, sinks, ragged)
    cost = (6 if dtype == "f32" else 1) * (3 if op == "att_bwd" else 1)  # of one pair of tokens
    s = _size(rng, 1, min(4096, int(math.sqrt(8192 * 8192 * 32 / (cost * 4 * hq)))))
    b = _size(rng, 1, max(1, min(8, 8192 * 8192 * 32 // (cost * 4 * hq * s * s))))
    sk = s if op == "att_bwd" or rng.random() < 0.7 else s + _size(rng, 1, 512)
    return _att("", op, dtype, b, s, sk, hq, hk, d, window, sinks, ragged, keep=op == "att" and rng.random() < 0.5)


def _lengths(case):
    """Queries and keys of each sequence; they go by the case alone, so that work() knows them."""
    b, sq, sk = case["b"], case["sq"], case["sk"]
    if not case["ragged"]:
        return [sq] * b, [sk] * b
    lk = [max(min(sq, sk), sk - (i * 2654435761 + 40503) % 1009 * sk // 1010) for i in range(b)]
    if sq == sk:  # a padded batch: as many queries as keys
        lk = [max(1, sk - (i * 40503) % 101 * sk // 202) for i in range(b)]
        return list(lk), lk
    return [sq] * b, lk


def _visible(nq, nk, window, sinks):
    """Pairs of a query and a key that it sees."""
    total = 0
    for p in range(max(0, nk - nq), nk):
        first = max(0, p - window + 1) if window else 0
        total += p + 1 - first + min(sinks, first)
    return total


def work(case):
    es, d = ES[case["dtype"]], case["d"]
    if case["op"] in ("rot", "rot_bwd"):
        n = case["tokens"] * (case["hq"] + case["hk"]) * d
        moved = 3 if case["op"] == "rot_bwd" else 2
        axes = 3 if case["s1"] else 1
        w = 2 * d * 4 * (2 if case["op"] == "rot_bwd" else 1)
        return {"bytes": moved * n * es + case["tokens"] * axes * 4 + case["rot"] // 2 * 4 + w,
                "flops": (25 if case["op"] == "rot_bwd" else 10) * n}
    nq, nk = _lengths(case)
    seen = sum(_visible(a, b, case["window"], case["sinks"]) for a, b in zip(nq, nk)) * case["hq"]
    rows = case["b"] * case["sq"] * case["hq"]
    used = 0  # keys that some query sees
    for a, b in zip(nq, nk):
        first = max(0, b - a - case["window"] + 1) if case["window"] else 0
        used += b - first + min(case["sinks"], first)
    queries, keys = sum(nq) * case["hq"] * d, used * case["hk"] * d
    if case["op"] == "att":
        return {"bytes": (queries + rows * d + 2 * keys) * es + (rows * 4 if case["keep"] else 0), "flops": 4 * seen * d}
    kv = case["b"] * case["sk"] * case["hk"] * d
    return {"bytes": (3 * queries + rows * d + 2 * keys + 2 * kv) * es + sum(nq) * case["hq"] * 4,
            "flops": 10 * seen * d}


# ---- inputs -------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DT[case["dtype"]]

    def normal(*shape, mean=0.0, std=1.0):
        return torch.randn(shape, generator=gen, device="cuda") * std + mean

    s = {"case": dict(case)}
    if case["op"] in ("rot", "rot_bwd"):
        t, hq, hk, d, rot = case["tokens"], case["hq"], case["hk"], case["d"], case["rot"]
        if case["packed"]:
            qkv = normal(t, hq + 2 * hk, d).to(dt)
            s["q"], s["k"] = qkv[:, :hq], qkv[:, hq:hq + hk]
        else:
            s["q"], s["k"] = normal(t, hq, d).to(dt), normal(t, hk, d).to(dt)
        s["wq"], s["wk"] = normal(d, mean=1.0, std=0.2), normal(d, mean=1.0, std=0.2)
        i = torch.arange(t, device="cuda", dtype=torch.int32)
        if case["s1"]:  # a clip of frames of 24 x 36 patches, moved by a random offset
            off = torch.randint(0, 64, (3,), generator=gen, device="cuda", dtype=torch.int32)
            s["pos"] = (torch.stack([i // 864, i // 36 % 24, i % 36], 1) + off + case["far"]).to(torch.int32).contiguous()
        else:
            off = torch.randint(0, 4096, (), generator=gen, device="cuda", dtype=torch.int32)
            s["pos"] = (i + off + case["far"]).to(torch.int32)
        s["freq"] = (10000.0 ** (-torch.arange(rot // 2, device="cuda", dtype=torch.float64) * 2 / rot)).float()
        if case["op"] == "rot_bwd":
            s["gq"], s["gk"] = normal(t, hq, d).to(dt), normal(t, hk, d).to(dt)
        return s
    b, sq, sk, hq, hk, d = (case[x] for x in ("b", "sq", "sk", "hq", "hk", "d"))
    s["q"] = normal(b, sq, hq, d, std=1.5).to(dt)
    s["k"], s["v"] = normal(b, sk, hk, d).to(dt), normal(b, sk, hk, d).to(dt)
    s["nq"] = s["nk"] = None
    if case["ragged"]:
        nq, nk = _lengths(case)
        s["nk"] = torch.tensor(nk, device="cuda", dtype=torch.int32)
        s["nq"] = torch.tensor(nq, device="cuda", dtype=torch.int32) if sq == sk else None
    if case["op"] == "att_bwd":
        s["do"] = normal(b, sq, hq, d).to(dt)
        o, s["lse"] = _attention(s)
        s["o"] = o.to(dt)
    return s


# ---- plain form ---------------------------------------------------------------------------
def _angles(s):
    c = s["case"]
    pos = s["pos"].double()
    if c["s1"]:
        axis = torch.repeat_interleave(torch.arange(3, device="cuda"),
                                       torch.tensor([c["s0"], c["s1"], c["s2"]], device="cuda"))
        pos = pos[:, axis]
    else:
        pos = pos[:, None]
    a = pos * s["freq"].double()
    return torch.cos(a).float()[:, None], torch.sin(a).float()[:, None]


def _split(x, rot, pairs):
    return (x[..., 0:rot:2], x[..., 1:rot:2]) if pairs else (x[..., :rot // 2], x[..., rot // 2:rot])


def _join(a, b, x, rot, pairs):
    r = torch.stack([a, b], -1).flatten(-2) if pairs else torch.cat([a, b], -1)
    return torch.cat([r, x[..., rot:]], -1)


def _rotate(x, cos, sin, rot, pairs):
    a, b = _split(x, rot, pairs)
    return _join(a * cos - b * sin, b * cos + a * sin, x, rot, pairs)


def _plain_rotary(s):
    c = s["case"]
    dt, rot, pairs = DT[c["dtype"]], c["rot"], c["pairs"]
    cos, sin = _angles(s)
    out, sums = [], []
    for x, w, g in ((s["q"], s["wq"], s.get("gq")), (s["k"], s["wk"], s.get("gk"))):
        x = x.float()
        rstd = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
        xh = x * rstd
        if g is None:
            out.append(_rotate(xh * w, cos, sin, rot, pairs).to(dt))
            continue
        g = _rotate(g.float(), cos, -sin, rot, pairs)
        h = g * w
        out.append((rstd * (h - xh * (h * xh).mean(-1, keepdim=True))).to(dt))
        sums.append((g * xh).sum((0, 1)))
    return out + sums


def _scores(s):
    """Masked scores [b, hk, group, sq, sk] and the mask."""
    c = s["case"]
    b, sq, sk, hq, hk, d = (c[x] for x in ("b", "sq", "sk", "hq", "hk", "d"))
    q = s["q"].float().view(b, sq, hk, hq // hk, d).permute(0, 2, 3, 1, 4)
    k = s["k"].float().permute(0, 2, 3, 1)[:, :, None]
    nq = s["nq"] if s["nq"] is not None else torch.full((b,), sq, device="cuda", dtype=torch.int32)
    nk = s["nk"] if s["nk"] is not None else torch.full((b,), sk, device="cuda", dtype=torch.int32)
    i, j = torch.arange(sq, device="cuda")[None, :, None], torch.arange(sk, device="cuda")[None, None, :]
    p = i + (nk - nq)[:, None, None]
    seen = (j <= p) & (i < nq[:, None, None])
    if c["window"]:
        seen &= (j > p - c["window"]) | (j < c["sinks"])
    seen = seen[:, None, None]
    return torch.where(seen, (q @ k) * d ** -0.5, -math.inf), seen


def _attention(s):
    c = s["case"]
    b, sq, hq, d = c["b"], c["sq"], c["hq"], c["d"]
    z, _ = _scores(s)
    m = z.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(z - m)
    total = p.sum(-1, keepdim=True)
    o = (p @ s["v"].float().permute(0, 2, 1, 3)[:, :, None]) / torch.where(total == 0, 1.0, total)
    return o.permute(0, 3, 1, 2, 4).reshape(b, sq, hq, d), (m + torch.log(total)).view(b, hq, sq)


def _plain_attention_backward(s):
    c = s["case"]
    dt = DT[c["dtype"]]
    b, sq, sk, hq, hk, d = (c[x] for x in ("b", "sq", "sk", "hq", "hk", "d"))
    z, seen = _scores(s)
    p = torch.where(seen, torch.exp(z - s["lse"].view(b, hk, hq // hk, sq, 1)), 0.0)
    g = s["do"].float().view(b, sq, hk, hq // hk, d).permute(0, 2, 3, 1, 4)
    q = s["q"].float().view(b, sq, hk, hq // hk, d).permute(0, 2, 3, 1, 4)
    dp = g @ s["v"].float().permute(0, 2, 3, 1)[:, :, None]
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * d ** -0.5
    dq = ds @ s["k"].float().permute(0, 2, 1, 3)[:, :, None]
    dk, dv = (ds.transpose(-1, -2) @ q).sum(2), (p.transpose(-1, -2) @ g).sum(2)
    return [dq.permute(0, 3, 1, 2, 4).reshape(b, sq, hq, d).to(dt), dk.permute(0, 2, 1, 3).contiguous().to(dt),
            dv.permute(0, 2, 1, 3).contiguous().to(dt)]


def _plain(s):
    c = s["case"]
    if c["op"] in ("rot", "rot_bwd"):
        return _plain_rotary(s)
    if c["op"] == "att_bwd":
        return _plain_attention_backward(s)
    o, lse = _attention(s)
    return [o.to(DT[c["dtype"]])] + ([lse] if c["keep"] else [])


# ---- the library's calls --------------------------------------------------------------------
_ctx = None


def _own_setup(s):
    """The context, descriptors and output buffers that a program keeps between calls."""
    global _ctx
    from quasarml_b200 import abi
    if _ctx is None:
        _ctx = abi.Context(0)
    c = s["case"]
    dt, f32 = DT[c["dtype"]], torch.float32

    def desc(t):
        return None if t is None else abi.desc_of(t)

    def new(*shape, dtype=dt):
        return torch.empty(shape, dtype=dtype, device="cuda")

    if c["op"] in ("rot", "rot_bwd"):
        t, hq, hk, d = c["tokens"], c["hq"], c["hk"], c["d"]
        how = {"eps": EPS, "sections": [c["s0"], c["s1"], c["s2"]] if c["s1"] else None,
               "pairing": abi.ROTARY_PAIRS if c["pairs"] else abi.ROTARY_HALVES}
        a = [desc(s[x]) for x in ("q", "k", "wq", "wk", "pos", "freq")]
        out = [new(t, hq, d), new(t, hk, d)]
        if c["op"] == "rot":
            a += [desc(x) for x in out]
            return out, lambda: _ctx.norm_rotary(*a, **how)
        out += [new(d, dtype=f32), new(d, dtype=f32)]
        a += [desc(s["gq"]), desc(s["gk"])] + [desc(x) for x in out]
        return out, lambda: _ctx.norm_rotary_backward(*a, **how)
    b, sq, sk, hq, hk, d = (c[x] for x in ("b", "sq", "sk", "hq", "hk", "d"))
    how = {"scale": d ** -0.5, "window": c["window"], "sinks": c["sinks"], "q_lengths": desc(s["nq"]),
           "k_lengths": desc(s["nk"])}
    q, k, v = desc(s["q"]), desc(s["k"]), desc(s["v"])
    if c["op"] == "att":
        out = [new(b, sq, hq, d)] + ([new(b, hq, sq, dtype=f32)] if c["keep"] else [])
        o, lse = desc(out[0]), desc(out[1]) if c["keep"] else None
        return out, lambda: _ctx.attention(q, k, v, o, lse=lse, **how)
    out = [new(b, sq, hq, d), new(b, sk, hk, d), new(b, sk, hk, d)]
    a = [q, k, v] + [desc(s[x]) for x in ("o", "lse", "do")] + [desc(x) for x in out]
    return out, lambda: _ctx.attention_backward(*a, **how)


def run(state):
    if not own:
        return _plain(state)
    if "own" not in state:
        state["own"] = _own_setup(state)
    out, call = state["own"]
    call()
    return out


# ---- binary64 -------------------------------------------------------------------------------
def _exact_rotary(case, s):
    c, half = case, case["rot"] // 2
    pos = s["pos"].double().view(c["tokens"], -1)
    counts = [c["s0"], c["s1"], c["s2"]] if c["s1"] else [half]
    turn = torch.cat([pos[:, a:a + 1].expand(-1, n) for a, n in enumerate(counts)], 1) * s["freq"].double()
    unit = torch.polar(torch.ones_like(turn), turn)[:, None]  # e^(i angle)
    first = torch.arange(half, device="cuda") * (2 if c["pairs"] else 1)
    second = first + (1 if c["pairs"] else half)

    def turned(x, u):
        y = x.clone()
        z = torch.complex(x[..., first], x[..., second]) * u
        y[..., first], y[..., second] = z.real, z.imag
        return y

    out, sums = [], []
    for n in ("q", "k"):
        x, w = s[n].double(), s["w" + n].double()
        r = ((x ** 2).sum(-1, keepdim=True) / c["d"] + EPS) ** -0.5
        if c["op"] == "rot":
            out.append(turned(x * r * w, unit))
            continue
        g = turned(s["g" + n].double(), unit.conj())
        along = (g * w * x).sum(-1, keepdim=True) / c["d"]
        out.append(r * g * w - r ** 3 * x * along)
        sums.append(torch.einsum("thd,thd->d", g, x * r))
    return out + sums


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("rot", "rot_bwd"):
        return _exact_rotary(case, s)
    b, sq, sk, hq, hk, d = (case[x] for x in ("b", "sq", "sk", "hq", "hk", "d"))
    nq, nk = _lengths(case)
    f64 = {"dtype": torch.float64, "device": "cuda"}
    o, lse = torch.zeros(b, sq, hq, d, **f64), torch.full((b, hq, sq), -math.inf, **f64)
    dq, dk, dv = torch.zeros(b, sq, hq, d, **f64), torch.zeros(b, sk, hk, d, **f64), torch.zeros(b, sk, hk, d, **f64)
    for n in range(b):
        rows, cols = nq[n], nk[n]
        at = torch.arange(cols - rows, cols, device="cuda")[:, None]
        key = torch.arange(cols, device="cuda")[None]
        hidden = key > at
        if case["window"]:
            hidden |= (at - key >= case["window"]) & (key >= case["sinks"])
        for h in range(hq):
            g = h // (hq // hk)
            q, k, v = s["q"][n, :rows, h].double(), s["k"][n, :cols, g].double(), s["v"][n, :cols, g].double()
            z = torch.mm(q, k.t()).div_(math.sqrt(d)).masked_fill_(hidden, -math.inf)
            norm = torch.logsumexp(z, 1)
            p = z.sub_(norm.clamp(min=-1e300)[:, None]).exp_()
            if case["op"] == "att":
                o[n, :rows, h], lse[n, h, :rows] = torch.mm(p, v), norm
                continue
            do = s["do"][n, :rows, h].double()
            dv[n, :cols, g] += torch.mm(p.t(), do)
            dp = torch.mm(do, v.t())
            p *= dp - (p * dp).sum(1, keepdim=True)
            dq[n, :rows, h] = torch.mm(p, k) / math.sqrt(d)
            dk[n, :cols, g] += torch.mm(p.t(), q) / math.sqrt(d)
    if case["op"] == "att":
        return [o] + ([lse] if case["keep"] else [])
    return [dq, dk, dv]
