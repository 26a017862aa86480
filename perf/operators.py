"""Measured cases of the feed-forward operators: layer norm's backward pass, the linear
layer with its epilogue (bias, activation, residual) and its backward pass, and the gated
linear layer and its backward pass.

``run`` computes a case in plain torch operations (binary32, rounded once at the end), or,
with ``own`` set, through the library's entry points.  ``exact`` is the same in binary64.
Sizes are those of the repository's layer norm and matmul workloads (16384 x 4096,
2048 x 1024 x 2048) and generic ones of transformer feed-forward layers."""
import torch

own = False

EPS = 1e-5
DT = {"f16": torch.float16, "f32": torch.float32}
ES = {"f16": 2, "f32": 4}


def _case(name, op, dtype, m, k, n, act="none", bias=False, residual=False, keep=False, wt=False, pitch=0):
    """m rows, k input and n output features (layer norm: m rows of n).  bias: with a bias (and
    its gradient); residual: added after the activation; keep: the forward pass also writes what
    the backward pass reads; wt: the weight is stored [n, k] and used as its transpose; pitch:
    extra elements between the rows of x."""
    return {"name": name, "op": op, "dtype": dtype, "m": m, "k": k, "n": n, "act": act, "bias": bias,
            "residual": residual, "keep": keep, "wt": wt, "pitch": pitch}


def listed():
    return [
        # a training step's normalisation of 16384 tokens (the layer norm workload's tensor)
        _case("ln_bwd_16384x4096_f16", "ln_bwd", "f16", 16384, 0, 4096),
        # binary32 rows whose width is odd: no vector access fits
        _case("ln_bwd_6007x1537_f32", "ln_bwd", "f32", 6007, 0, 1537),
        # fine tuning with a batch of a few short sequences: latency
        _case("ln_bwd_200x1024_f16", "ln_bwd", "f16", 200, 0, 1024),
        # one new token through a down projection with its residual
        _case("linear_1x11008x4096_f16", "linear", "f16", 1, 11008, 4096, bias=False, residual=True),
        # a prompt or training batch through a plain feed-forward layer's first product
        _case("linear_8192x4096x4096_f16", "linear", "f16", 8192, 4096, 4096, act="gelu", bias=True, keep=True),
        # ragged binary32 layer: no size fits a vector
        _case("linear_1000x1027x2050_f32", "linear", "f32", 1000, 1027, 2050, act="relu", bias=True, residual=True),
        # training step of a layer of the batched matmul workload's sizes, 8 sequences of 2048
        _case("linear_bwd_16384x1024x2048_f16", "linear_bwd", "f16", 16384, 1024, 2048, act="gelu", bias=True),
        # binary32 training step of a small layer whose weight is stored transposed
        _case("linear_bwd_777x1024x1000_f32", "linear_bwd", "f32", 777, 1024, 1000, act="silu", bias=True, wt=True),
        # a few tokens decoded together through the gated projection
        _case("gated_5x4096x11008_f16", "gated", "f16", 5, 4096, 11008, act="silu"),
        # a training batch through the gated projection
        _case("gated_8192x2048x5632_f16", "gated", "f16", 8192, 2048, 5632, act="silu", keep=True),
        # its backward pass
        _case("gated_bwd_8192x2048x5632_f16", "gated_bwd", "f16", 8192, 2048, 5632, act="silu"),
        # ragged binary32 backward pass of a small gated layer with biases
        _case("gated_bwd_515x520x1366_f32", "gated_bwd", "f32", 515, 520, 1366, act="gelu", bias=True),
    ]


def _size(rng, lo, hi):
    """Log-uniform in [lo, hi], half of the time rounded to a multiple of 64 (a model's width)."""
    v = int(round(lo * (hi / lo) ** rng.random()))
    if v >= 64 and rng.random() < 0.5:
        v = v // 64 * 64
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["ln_bwd", "linear", "linear_bwd", "gated", "gated_bwd"])
    dtype = rng.choice(["f16", "f16", "f32"])
    if op == "ln_bwd":
        n = _size(rng, 8, 20000)
        return _case("", op, dtype, _size(rng, 1, min(16384, (1 << 26) // n)), 0, n)
    k, n = _size(rng, 16, 8192), _size(rng, 16, 11264)
    most = (1 << 36) // (4 if dtype == "f32" else 1) // (2 if op in ("gated", "gated_bwd") else 1)
    m = _size(rng, 1, max(1, min(16384, most // (k * n) // (2 if op.endswith("_bwd") else 1))))
    gated = op.startswith("gated")
    return _case("", op, dtype, m, k, n,
                 act=rng.choice(["relu", "gelu", "silu", "sigmoid"] + ([] if gated else ["none"])),
                 bias=rng.random() < 0.5, residual=op == "linear" and rng.random() < 0.5,
                 keep=op in ("linear", "gated") and rng.random() < 0.5, wt=rng.random() < 0.25,
                 pitch=rng.choice([0, 0, 0, 8, 3]))


def work(case):
    m, k, n, es = case["m"], case["k"], case["n"], ES[case["dtype"]]
    op = case["op"]
    if op == "ln_bwd":
        return {"bytes": 3 * m * n * es + 3 * n * 4, "flops": 16 * m * n}
    b = n * 4 if case["bias"] else 0
    kept = 1 if case["keep"] else 0
    if op == "linear":
        moved = m * k + k * n + m * n * (1 + kept + (1 if case["residual"] else 0))
        return {"bytes": moved * es + b, "flops": 2 * m * k * n}
    if op == "linear_bwd":
        read = m * k + k * n + m * n * (2 if case["act"] != "none" else 1)
        return {"bytes": (read + m * k + k * n) * es + b, "flops": 4 * m * k * n}
    if op == "gated":
        return {"bytes": (m * k + 2 * k * n + m * n * (1 + 2 * kept)) * es + 2 * b, "flops": 4 * m * k * n}
    return {"bytes": (2 * m * k + 4 * k * n + 3 * m * n) * es + 2 * b, "flops": 8 * m * k * n}


# ---- inputs -------------------------------------------------------------------------------
def _weight(gen, case):
    k, n = case["k"], case["n"]
    w = torch.randn((n, k) if case["wt"] else (k, n), generator=gen, device="cuda") * k ** -0.5
    w = w.to(DT[case["dtype"]])
    return w.t() if case["wt"] else w


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DT[case["dtype"]]
    m, k, n, op = case["m"], case["k"], case["n"], case["op"]

    def normal(*shape, mean=0.0, std=1.0):
        return torch.randn(shape, generator=gen, device="cuda") * std + mean

    s = {"case": dict(case)}
    if op == "ln_bwd":
        s["x"] = normal(m, n, mean=0.5, std=2.0).to(dt)
        s["gamma"] = normal(n, mean=1.0, std=0.1)
        s["dy"] = normal(m, n).to(dt)
        return s
    s["x"] = normal(m, k + case["pitch"]).to(dt)[:, :k]
    gated = op.startswith("gated")
    s["w"] = _weight(gen, case)
    s["b"] = normal(n, std=0.1) if case["bias"] else None
    if gated:
        s["w2"] = _weight(gen, case)
        s["b2"] = normal(n, std=0.1) if case["bias"] else None
    if op == "linear":
        s["residual"] = normal(m, n).to(dt) if case["residual"] else None
    if op.endswith("_bwd"):
        s["dy"] = normal(m, n).to(dt)
        # what the forward pass kept
        z = s["x"].float() @ s["w"].float()
        s["pre"] = (z if s["b"] is None else z + s["b"]).to(dt)
        if gated:
            z = s["x"].float() @ s["w2"].float()
            s["up"] = (z if s["b2"] is None else z + s["b2"]).to(dt)
    return s


# ---- plain form ---------------------------------------------------------------------------
GELU_S, GELU_C = 0.7978845608, 0.044715


def _sigmoid(z):
    return 1.0 / (1.0 + torch.exp(-z))


def _act(z, act):
    if act == "relu":
        return torch.clamp(z, min=0.0)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.tanh(GELU_S * (z + GELU_C * z * z * z)))
    if act == "silu":
        return z * _sigmoid(z)
    if act == "sigmoid":
        return _sigmoid(z)
    return z


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        t = torch.tanh(GELU_S * (z + GELU_C * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * GELU_S * (1.0 + 3.0 * GELU_C * z * z)
    if act == "silu":
        s = _sigmoid(z)
        return s * (1.0 + z * (1.0 - s))
    if act == "sigmoid":
        s = _sigmoid(z)
        return s * (1.0 - s)
    return torch.ones_like(z)


def _plain(s):
    c = s["case"]
    dt, op, act = DT[c["dtype"]], c["op"], c["act"]
    x = s["x"].float()
    if op == "ln_bwd":
        dy = s["dy"].float()
        d = x - x.mean(1, keepdim=True)
        rstd = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
        xh = d * rstd
        h = dy * s["gamma"]
        dx = rstd * (h - h.mean(1, keepdim=True) - xh * (h * xh).mean(1, keepdim=True))
        return [dx.to(dt), (dy * xh).sum(0), dy.sum(0)]
    w = s["w"].float()
    if op == "linear":
        z = x @ w
        if s["b"] is not None:
            z = z + s["b"]
        y = _act(z, act)
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return [y.to(dt)] + ([z.to(dt)] if c["keep"] else [])
    if op == "linear_bwd":
        dz = s["dy"].float() * _act_grad(s["pre"].float(), act)
        out = [(dz @ w.t()).to(dt), (x.t() @ dz).to(dt)]
        return out + ([dz.sum(0)] if c["bias"] else [])
    w2 = s["w2"].float()
    if op == "gated":
        g, u = x @ w, x @ w2
        if c["bias"]:
            g, u = g + s["b"], u + s["b2"]
        y = _act(g, act) * u
        return [y.to(dt)] + ([g.to(dt), u.to(dt)] if c["keep"] else [])
    dy, g, u = s["dy"].float(), s["pre"].float(), s["up"].float()
    dg, du = dy * u * _act_grad(g, act), dy * _act(g, act)
    out = [(dg @ w.t() + du @ w2.t()).to(dt), (x.t() @ dg).to(dt), (x.t() @ du).to(dt)]
    return out + ([dg.sum(0), du.sum(0)] if c["bias"] else [])


# ---- the library's calls --------------------------------------------------------------------
_ctx = None


def _own_setup(s):
    """The context, descriptors and output buffers that a program keeps between calls."""
    global _ctx
    from quasarml_b200 import abi
    if _ctx is None:
        _ctx = abi.Context(0)
    c = s["case"]
    op, act = c["op"], getattr(abi, "ACT_" + c["act"].upper())
    dt = DT[c["dtype"]]

    def desc(t):
        return None if t is None else abi.desc_of(t)

    def new(*shape, dtype=dt):
        return torch.empty(shape, dtype=dtype, device="cuda")

    m, k, n = c["m"], c["k"], c["n"]
    x, f32 = desc(s["x"]), torch.float32
    if op == "ln_bwd":
        out = [new(m, n), new(n, dtype=f32), new(n, dtype=f32)]
        a = [x, desc(s["gamma"]), desc(s["dy"]), EPS] + [desc(t) for t in out]
        return out, lambda: _ctx.layer_norm_backward(*a)
    w, b = desc(s["w"]), desc(s["b"])
    if op == "linear":
        out = [new(m, n)] + ([new(m, n)] if c["keep"] else [])
        a = [x, w, b, act, desc(s["residual"]), desc(out[1]) if c["keep"] else None, desc(out[0])]
        return out, lambda: _ctx.linear(*a)
    if op == "linear_bwd":
        out = [new(m, k), new(k, n)] + ([new(n, dtype=f32)] if c["bias"] else [])
        a = [x, w, act, desc(s["pre"]), desc(s["dy"]), desc(out[0]), desc(out[1]),
             desc(out[2]) if c["bias"] else None]
        return out, lambda: _ctx.linear_backward(*a)
    w2, b2 = desc(s["w2"]), desc(s["b2"])
    if op == "gated":
        out = [new(m, n)] + ([new(m, n), new(m, n)] if c["keep"] else [])
        kept = [desc(out[1]), desc(out[2])] if c["keep"] else [None, None]
        a = [x, w, w2, b, b2, act] + kept + [desc(out[0])]
        return out, lambda: _ctx.gated_linear(*a)
    out = [new(m, k), new(k, n), new(k, n)] + ([new(n, dtype=f32), new(n, dtype=f32)] if c["bias"] else [])
    db = [desc(out[3]), desc(out[4])] if c["bias"] else [None, None]
    a = [x, w, w2, act, desc(s["pre"]), desc(s["up"]), desc(s["dy"]), desc(out[0]), desc(out[1]), desc(out[2])] + db
    return out, lambda: _ctx.gated_linear_backward(*a)


def run(state):
    if not own:
        return _plain(state)
    if "own" not in state:
        state["own"] = _own_setup(state)
    out, call = state["own"]
    call()
    return out


# ---- binary64 -------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op, act = case["op"], case["act"]
    f64 = {key: v.double() for key, v in s.items() if isinstance(v, torch.Tensor)}

    def f(z):  # the activation and its derivative
        if act == "none":
            return z, torch.ones_like(z)
        if act == "relu":
            return torch.where(z > 0, z, torch.zeros_like(z)), torch.where(z > 0, 1.0, 0.0).double()
        if act == "gelu":
            # 0.5 (1 + tanh v) = sigmoid(2 v)
            v2, dv2 = 2 * GELU_S * (z + GELU_C * z ** 3), 2 * GELU_S * (1 + 3 * GELU_C * z ** 2)
            p = torch.special.expit(v2)
            return z * p, p + z * p * (1 - p) * dv2
        p = torch.special.expit(z)
        return (z * p, p + z * p * (1 - p)) if act == "silu" else (p, p * (1 - p))

    x = f64["x"]
    if op == "ln_bwd":
        n = x.shape[1]
        mean = x.sum(1, keepdim=True) / n
        var = ((x - mean) ** 2).sum(1, keepdim=True) / n
        xh = (x - mean) / (var + EPS) ** 0.5
        h = f64["dy"] * f64["gamma"]
        along = h.sum(1, keepdim=True) / n + xh * ((h * xh).sum(1, keepdim=True) / n)
        return [(h - along) / (var + EPS) ** 0.5, torch.einsum("rc,rc->c", f64["dy"], xh), f64["dy"].sum(0)]
    w, zero = f64["w"], x.new_zeros(())
    if op == "linear":
        z = torch.addmm(f64.get("b", zero).expand(case["n"]), x, w)
        y = f(z)[0] + f64.get("residual", zero)
        return [y] + ([z] if case["keep"] else [])
    if op == "linear_bwd":
        dz = f64["dy"] * f(f64["pre"])[1]
        return [torch.mm(dz, w.t()), torch.mm(x.t(), dz)] + ([dz.sum(0)] if case["bias"] else [])
    w2 = f64["w2"]
    if op == "gated":
        g = torch.addmm(f64.get("b", zero).expand(case["n"]), x, w)
        u = torch.addmm(f64.get("b2", zero).expand(case["n"]), x, w2)
        return [f(g)[0] * u] + ([g, u] if case["keep"] else [])
    a, da = f(f64["pre"])
    dg, du = f64["dy"] * f64["up"] * da, f64["dy"] * a
    out = [torch.addmm(torch.mm(dg, w.t()), du, w2.t()), torch.mm(x.t(), dg), torch.mm(x.t(), du)]
    return out + ([dg.sum(0), du.sum(0)] if case["bias"] else [])
