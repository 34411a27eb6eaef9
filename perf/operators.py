"""What is timed of the encoder operators: layer norm, linear with its epilogue, the gated linear
recurrence and the AdamW step, each as a user of ``torchwarp_b200`` calls it.

Every case has a plain form in elementary torch operations, in 32 bits and rounded once at the
end, and ``exact`` restates the operators' definitions in 64 bits.
"""

import math

import torch

#: False: the plain forms.  True: the calls of torchwarp_b200.
own = False

_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}
_EPS = 1e-5
_BLOCK = 256  # values that share one scale in the 8-bit optimizer states
_ADAM = {"lr": 1e-3, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": 1e-2}


# ------------------------------------------------------------------- cases

def listed():
    return [
        # One new frame of four streams, normalised while a live sequence is encoded.
        {"name": "layer_norm token", "op": "layer_norm", "dtype": "float32", "rows": 4, "dim": 256,
         "train": False},
        # 50 series of 140 frames, a training step with an odd feature count.
        {"name": "layer_norm f32 odd", "op": "layer_norm", "dtype": "float32", "rows": 7000,
         "dim": 257, "train": True},
        # A training batch of 32 sequences of 1024 frames.
        {"name": "layer_norm bf16 train", "op": "layer_norm", "dtype": "bfloat16", "rows": 32768,
         "dim": 1024, "train": True},
        # Eight streams, one frame each, through the wide layer of an encoder block.
        {"name": "linear token", "op": "linear", "dtype": "bfloat16", "rows": 8, "inner": 1024,
         "outer": 4096, "act": "silu", "residual": False, "train": False},
        # A small float32 forecaster's hidden layer, odd sizes, forward and backward.
        {"name": "linear f32 odd train", "op": "linear", "dtype": "float32", "rows": 7000,
         "inner": 257, "outer": 385, "act": "silu", "residual": False, "train": True},
        # The narrow layer of a block with its residual, for 4096 frames of a support set.
        {"name": "linear bf16 residual", "op": "linear", "dtype": "bfloat16", "rows": 4096,
         "inner": 4096, "outer": 1024, "act": "none", "residual": True, "train": False},
        # The wide layer in a training step of 32 sequences of 1024 frames.
        {"name": "linear bf16 train", "op": "linear", "dtype": "bfloat16", "rows": 32768,
         "inner": 1024, "outer": 4096, "act": "gelu", "residual": False, "train": True},
        # One frame of 64 streams against their running states.
        {"name": "scan token", "op": "scan_step", "dtype": "bfloat16", "batch": 64, "dim": 1024},
        # A training batch of 32 sequences of 1024 frames.
        {"name": "scan bf16 train", "op": "scan", "dtype": "bfloat16", "batch": 32, "time": 1024,
         "dim": 1024, "ragged": False, "train": True},
        # Four long recordings of different lengths, few features.
        {"name": "scan f32 long ragged", "op": "scan", "dtype": "float32", "batch": 4,
         "time": 32768, "dim": 256, "ragged": True, "train": True},
        # A small encoder's weights (bfloat16, odd sizes among them), 8-bit states.
        {"name": "adamw 8 bit small", "op": "adamw", "dtype": "bfloat16", "bits": 8, "width": 257,
         "layers": 4},
        # An encoder of 8 blocks, 32-bit states: 106 tensors, 67 million weights.
        {"name": "adamw 32 bit", "op": "adamw", "dtype": "float32", "bits": 32, "width": 1024,
         "layers": 8},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    op = rng.choice(["layer_norm", "linear", "scan", "scan_step", "adamw"])
    if op == "layer_norm":
        dim = _log_int(rng, 8, 8192)
        return {"op": op, "dtype": dtype, "rows": _log_int(rng, 1, min(65536, (1 << 25) // dim)),
                "dim": dim, "train": rng.random() < 0.6}
    if op == "linear":
        inner, outer = _log_int(rng, 1, 4096), _log_int(rng, 1, 4096)
        train = rng.random() < 0.6
        act = rng.choice(["none", "relu", "gelu", "silu", "sigmoid"])
        if act == "relu" and train and dtype == "float32":
            act = "silu"  # relu's slope at a z within rounding of zero is either 0 or 1
        return {"op": op, "dtype": dtype, "inner": inner, "outer": outer,
                "rows": _log_int(rng, 1, 16384), "act": act,
                "residual": rng.random() < 0.4, "train": train}
    if op == "scan":
        dim = _log_int(rng, 1, 2048)
        batch = _log_int(rng, 1, 64)
        return {"op": op, "dtype": dtype, "batch": batch, "dim": dim,
                "time": _log_int(rng, 1, min(32768, (1 << 25) // (dim * batch))),
                "ragged": rng.random() < 0.4, "train": rng.random() < 0.6}
    if op == "scan_step":
        return {"op": op, "dtype": dtype, "batch": _log_int(rng, 1, 512),
                "dim": _log_int(rng, 1, 4096)}
    return {"op": op, "dtype": dtype, "bits": rng.choice([8, 32]), "width": _log_int(rng, 8, 900),
            "layers": rng.randint(1, 8)}


def _adam_shapes(case):
    """The weights of an encoder of `layers` blocks: 13 tensors a block, and 2 for all."""
    d = case["width"]
    block = [(2 * d, d), (2 * d,), (d, d), (d,), (4 * d, d), (4 * d,), (d, d), (d,), (d,), (d,),
             (d,), (d,), (d,)]
    return block * case["layers"] + [(d,), (d,)]


def _padded(shape):
    return -(-math.prod(shape) // _BLOCK) * _BLOCK


def work(case):
    s = _BYTES[case["dtype"]]
    if case["op"] == "layer_norm":
        n, d = case["rows"] * case["dim"], case["dim"]
        if case["train"]:  # x, dy -> y, dx; weight, bias and their gradients
            return {"bytes": s * (4 * n + 4 * d), "flops": 20 * n}
        return {"bytes": s * (2 * n + 2 * d), "flops": 8 * n}
    if case["op"] == "linear":
        m, k, n = case["rows"], case["inner"], case["outer"]
        res = m * n if case["residual"] else 0
        if case["train"]:  # x, w, b, r, dy -> y, dx, dw, db
            return {"bytes": s * (2 * m * k + 2 * n * k + 2 * n + res + 2 * m * n),
                    "flops": 6 * m * n * k}
        return {"bytes": s * (m * k + n * k + n + res + m * n), "flops": 2 * m * n * k}
    if case["op"] == "scan":
        n, st = case["batch"] * case["time"] * case["dim"], case["batch"] * case["dim"]
        if case["train"]:  # x, gate, dy -> y, dx, dgate; states in 32 bits
            return {"bytes": s * 6 * n + 16 * st, "flops": 25 * n}
        return {"bytes": s * 3 * n + 8 * st, "flops": 8 * n}
    if case["op"] == "scan_step":
        n = case["batch"] * case["dim"]
        return {"bytes": 3 * s * n + 8 * n, "flops": 8 * n}
    n = sum(math.prod(x) for x in _adam_shapes(case))
    state = 16 if case["bits"] == 32 else 4 + 16 / _BLOCK
    return {"bytes": n * (3 * s + state), "flops": 15 * n}


# ------------------------------------------------------------------ inputs

def _make(case, seed):
    """The case's inputs, on the GPU, from the seed alone."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, dtype=dt):
        return torch.randn(*shape, device=dev, generator=g).mul_(std).add_(mean).to(dtype)

    op = case["op"]
    if op == "layer_norm":
        r, d = case["rows"], case["dim"]
        # activations with an offset and a scale per frame, as a residual stream has them
        x = (torch.randn(r, d, device=dev, generator=g)
             * (0.5 + torch.rand(r, 1, device=dev, generator=g))
             + torch.randn(r, 1, device=dev, generator=g)).to(dt)
        return {"x": x, "weight": normal(d, std=0.1, mean=1.0), "bias": normal(d, std=0.1),
                "dy": normal(r, d)}
    if op == "linear":
        m, k, n = case["rows"], case["inner"], case["outer"]
        return {"x": normal(m, k), "weight": normal(n, k, std=k ** -0.5),
                "bias": normal(n, std=0.1),
                "residual": normal(m, n) if case["residual"] else None, "dy": normal(m, n)}
    if op == "scan":
        b, t, d = case["batch"], case["time"], case["dim"]
        lengths = None
        if case["ragged"]:
            lengths = torch.randint(0, t + 1, (b,), device=dev, generator=g)
            lengths[0] = t
        # gates that keep most of the state, as a trained recurrence has them
        return {"x": normal(b, t, d), "gate": normal(b, t, d, std=1.5, mean=2.0),
                "state": normal(b, d, dtype=torch.float32), "lengths": lengths,
                "dy": normal(b, t, d), "dstate": normal(b, d, dtype=torch.float32)}
    if op == "scan_step":
        b, d = case["batch"], case["dim"]
        return {"x": normal(b, d), "gate": normal(b, d, std=1.5, mean=2.0),
                "state": normal(b, d, dtype=torch.float32)}
    shapes = _adam_shapes(case)
    total = sum(_padded(s) for s in shapes)
    live = torch.cat([torch.arange(_padded(s), device=dev) < math.prod(s) for s in shapes])
    # gradients whose size differs from one run of weights to the next
    size = torch.exp(torch.randn(total // _BLOCK, 1, device=dev, generator=g))
    grad = torch.randn(total, device=dev, generator=g).view(-1, _BLOCK).mul_(size).mul_(1e-3)
    grad = grad.view(-1).mul_(live).to(dt)
    param = torch.randn(total, device=dev, generator=g).mul_(0.02).mul_(live).to(dt)
    return {"param": param, "grad": grad, "shapes": shapes, "seed": seed & 0xFFFF}


def prepare(case, seed):
    s = {"case": dict(case), **_make(case, seed)}
    if case.get("train"):
        for k in ("x", "weight", "bias", "gate", "state"):
            if s.get(k) is not None:
                s[k].requires_grad_(True)
    if case["op"] != "adamw":
        return s
    # All weights lie in one buffer, each on a boundary of 256 values, and the optimizer keeps
    # its states in buffers of the same layout.
    if own:
        import torchwarp_b200 as tw
        params, at = [], 0
        for shape in s["shapes"]:
            n = math.prod(shape)
            p = torch.nn.Parameter(s["param"][at:at + n].view(shape))
            p.grad = s["grad"][at:at + n].view(shape)
            params.append(p)
            at += _padded(shape)
        s["optimizer"] = tw.AdamW(params, state_bits=case["bits"], seed=s["seed"], **_ADAM)
        return s
    n, dev = s["param"].numel(), s["param"].device
    if case["bits"] == 32:
        s["exp_avg"] = torch.zeros(n, device=dev)
        s["exp_avg_sq"] = torch.zeros(n, device=dev)
    else:
        for k in ("exp_avg", "exp_avg_sqrt"):
            s[k] = torch.zeros(n, device=dev).to(torch.float8_e4m3fn)
            s[k + "_scale"] = torch.zeros(n // _BLOCK, device=dev)
    s["step"] = 0
    return s


# ------------------------------------------------------------------- passes

def run(state):
    op = state["case"]["op"]
    if own:
        return {"layer_norm": _own_layer_norm, "linear": _own_linear, "scan": _own_scan,
                "scan_step": _own_scan_step, "adamw": _own_adamw}[op](state)
    with torch.no_grad():
        return {"layer_norm": _plain_layer_norm, "linear": _plain_linear, "scan": _plain_scan,
                "scan_step": _plain_scan_step, "adamw": _plain_adamw}[op](state)


def _own_layer_norm(s):
    from torchwarp_b200 import functional as TF
    if not s["case"]["train"]:
        return {"y": TF.layer_norm(s["x"], s["weight"], s["bias"], eps=_EPS)}
    y = TF.layer_norm(s["x"], s["weight"], s["bias"], eps=_EPS)
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])
    return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}


def _own_linear(s):
    from torchwarp_b200 import functional as TF
    act = None if s["case"]["act"] == "none" else s["case"]["act"]
    y = TF.linear(s["x"], s["weight"], s["bias"], activation=act, residual=s["residual"])
    if not s["case"]["train"]:
        return {"y": y}
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])
    return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}


def _own_scan(s):
    from torchwarp_b200 import functional as TF
    y, last = TF.gated_scan(s["x"], s["gate"], s["state"], lengths=s["lengths"])
    if not s["case"]["train"]:
        return {"y": y, "state": last}
    dx, dg, ds = torch.autograd.grad((y, last), (s["x"], s["gate"], s["state"]),
                                     (s["dy"], s["dstate"]))
    return {"y": y.detach(), "state": last.detach(), "dx": dx, "dgate": dg, "dstate": ds}


def _own_scan_step(s):
    from torchwarp_b200 import functional as TF
    y = TF.gated_scan_step(s["x"], s["gate"], s["state"])
    return {"y": y, "state": s["state"]}


def _own_adamw(s):
    s["optimizer"].step()
    return {"param": s["param"], **s["optimizer"].flat_state(0)}


def _plain_layer_norm(s):
    x, w, dt = s["x"].float(), s["weight"].float(), s["x"].dtype
    xc = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((xc * xc).mean(-1, keepdim=True) + _EPS)
    xhat = xc * rstd
    y = (xhat * w + s["bias"].float()).to(dt)
    if not s["case"]["train"]:
        return {"y": y}
    dy = s["dy"].float()
    q = dy * w
    dx = rstd * (q - q.mean(-1, keepdim=True) - xhat * (q * xhat).mean(-1, keepdim=True))
    return {"y": y, "dx": dx.to(dt), "dweight": (dy * xhat).sum(0).to(dt),
            "dbias": dy.sum(0).to(dt)}


def _plain_act(z, act):
    if act == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z), (z > 0).float()
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "silu":
        f = 1 / (1 + torch.exp(-z))
        return z * f, f * (1 + z * (1 - f))
    if act == "sigmoid":
        f = 1 / (1 + torch.exp(-z))
        return f, f * (1 - f)
    return z, torch.ones_like(z)


def _plain_linear(s):
    x, w, dt = s["x"].float(), s["weight"].float(), s["x"].dtype
    z = x @ w.t() + s["bias"].float()
    y, slope = _plain_act(z, s["case"]["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    if not s["case"]["train"]:
        return {"y": y.to(dt)}
    dz = s["dy"].float() * slope
    return {"y": y.to(dt), "dx": (dz @ w).to(dt), "dweight": (dz.t() @ x).to(dt),
            "dbias": dz.sum(0).to(dt)}


def _plain_recurrence(a, b, first):
    """h_t = a_t h_{t-1} + b_t over dimension 1 from h_{-1} = first: spans double until they
    reach the start."""
    b = torch.cat([b[:, :1] + a[:, :1] * first.unsqueeze(1), b[:, 1:]], 1)
    span, length = 1, a.shape[1]
    while span < length:
        b = torch.cat([b[:, :span], b[:, span:] + a[:, span:] * b[:, :-span]], 1)
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], 1)
        span *= 2
    return b


def _plain_scan(s):
    x, h0, dt = s["x"].float(), s["state"], s["x"].dtype
    f = 1 / (1 + torch.exp(-s["gate"].float()))
    live = None
    if s["lengths"] is not None:  # past its length a sequence keeps its state
        at = torch.arange(x.shape[1], device=x.device)
        live = (at < s["lengths"].unsqueeze(1)).unsqueeze(2)
        f = torch.where(live, f, torch.ones_like(f))
    h = _plain_recurrence(f, (1 - f) * x, h0)
    y = h if live is None else torch.where(live, h, torch.zeros_like(h))
    if not s["case"]["train"]:
        return {"y": y.to(dt), "state": h[:, -1].clone()}
    dy = s["dy"].float()
    if live is not None:
        dy = torch.where(live, dy, torch.zeros_like(dy))
    # adjoints run from the end: lam_t = dy_t + f_{t+1} lam_{t+1}
    back = torch.cat([torch.ones_like(f[:, :1]), f.flip(1)[:, :-1]], 1)
    lam = _plain_recurrence(back, dy.flip(1), s["dstate"]).flip(1)
    before = torch.cat([h0.unsqueeze(1), h[:, :-1]], 1)
    return {"y": y.to(dt), "state": h[:, -1].clone(), "dx": ((1 - f) * lam).to(dt),
            "dgate": (lam * (before - x) * f * (1 - f)).to(dt), "dstate": f[:, 0] * lam[:, 0]}


def _plain_scan_step(s):
    f = 1 / (1 + torch.exp(-s["gate"].float()))
    s["state"].copy_(f * s["state"] + (1 - f) * s["x"].float())
    return {"y": s["state"].to(s["x"].dtype), "state": s["state"]}


def _dither(n, seed, step, device):
    """32 bits for each of n values: an integer hash (lowbias32) of the value's place, the step
    and the seed."""
    key = (seed * 0x9E3779B1 + step * 0x85EBCA77) & 0xFFFFFFFF
    h = torch.arange(n, device=device, dtype=torch.int64) & 0xFFFFFFFF
    h = h ^ key
    h = h ^ (h >> 16)
    h = (h * 0x7FEB352D) & 0xFFFFFFFF
    h = h ^ (h >> 15)
    h = (h * 0x846CA68B) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _to_e4m3(v, u, floor):
    """Blocks of values as e4m3 codes and a scale each; rounding up with the probability u
    gives, and never below the smallest code where `floor` and the value is not zero."""
    scale = v.abs().amax(1, keepdim=True) / 448
    y = v.abs() / torch.where(scale > 0, scale, torch.ones_like(scale))
    exponent = ((y.view(torch.int32) >> 23) - 127).clamp(min=-6)
    ulp = torch.exp2((exponent - 3).float())
    q = torch.floor(y / ulp + u) * ulp
    if floor:
        q = torch.where(y > 0, q.clamp(min=2.0 ** -9), q)
    q = q.clamp(max=448.0) * torch.sign(v)
    return q.to(torch.float8_e4m3fn).view(-1), scale.view(-1)


def _plain_adamw(s):
    (b1, b2), lr = _ADAM["betas"], _ADAM["lr"]
    s["step"] += 1
    g, p = s["grad"].float(), s["param"].float()
    if s["case"]["bits"] == 32:
        m, v = s["exp_avg"], s["exp_avg_sq"]
    else:
        m = (s["exp_avg"].float().view(-1, _BLOCK) * s["exp_avg_scale"].unsqueeze(1)).view(-1)
        r = s["exp_avg_sqrt"].float().view(-1, _BLOCK) * s["exp_avg_sqrt_scale"].unsqueeze(1)
        v = (r * r).view(-1)
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * (g * g)
    denom = torch.sqrt(v) / math.sqrt(1 - b2 ** s["step"]) + _ADAM["eps"]
    p = p * (1 - lr * _ADAM["weight_decay"]) - (lr / (1 - b1 ** s["step"])) * (m / denom)
    s["param"].copy_(p)
    if s["case"]["bits"] == 32:
        s["exp_avg"].copy_(m)
        s["exp_avg_sq"].copy_(v)
        return {k: s[k] for k in ("param", "exp_avg", "exp_avg_sq")}
    h = _dither(m.numel(), s["seed"], s["step"], m.device).view(-1, _BLOCK)
    for k, value, u in (("exp_avg", m, (h & 0xFFFF).float() / 65536),
                        ("exp_avg_sqrt", torch.sqrt(v), (h >> 16).float() / 65536)):
        q, scale = _to_e4m3(value.view(-1, _BLOCK), u, k == "exp_avg_sqrt")
        s[k].copy_(q)
        s[k + "_scale"].copy_(scale)
    return {k: s[k] for k in ("param", "exp_avg", "exp_avg_scale", "exp_avg_sqrt",
                              "exp_avg_sqrt_scale")}


# ------------------------------------------------------------ in 64 bits

def exact(case, seed):
    s = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v
         for k, v in _make(case, seed).items()}
    op = case["op"]
    if op == "layer_norm":
        var, mean = torch.var_mean(s["x"], -1, correction=0, keepdim=True)
        std = torch.sqrt(var + _EPS)
        n = (s["x"] - mean) / std
        out = {"y": n * s["weight"] + s["bias"]}
        if case["train"]:
            q = s["dy"] * s["weight"]
            out["dx"] = (q - q.mean(-1, keepdim=True)
                         - n * torch.mean(q * n, -1, keepdim=True)) / std
            out["dweight"] = torch.einsum("rd,rd->d", s["dy"], n)
            out["dbias"] = s["dy"].sum(0)
        return out
    if op == "linear":
        with torch.enable_grad():
            leaves = [s[k].requires_grad_(True) for k in ("x", "weight", "bias")]
            z = torch.addmm(leaves[2], leaves[0], leaves[1].t())
            y = {"none": lambda t: t, "relu": torch.relu, "silu": torch.nn.functional.silu,
                 "gelu": torch.nn.functional.gelu, "sigmoid": torch.sigmoid}[case["act"]](z)
            if s["residual"] is not None:
                y = y + s["residual"]
            if not case["train"]:
                return {"y": y.detach()}
            grads = torch.autograd.grad(y, leaves, s["dy"])
        return {"y": y.detach(), "dx": grads[0], "dweight": grads[1], "dbias": grads[2]}
    if op == "scan_step":
        f = torch.sigmoid(s["gate"])
        h = torch.lerp(s["x"], s["state"], f)
        return {"y": h, "state": h}
    if op == "scan":
        return _exact_scan(case, s)
    g = s["grad"]
    lr, (b1, b2) = _ADAM["lr"], _ADAM["betas"]
    m, v = (1 - b1) * g, (1 - b2) * g.square()
    p = s["param"] - lr * (_ADAM["weight_decay"] * s["param"]
                           + (m / (1 - b1)) / ((v / (1 - b2)).sqrt() + _ADAM["eps"]))
    if case["bits"] == 32:
        return {"param": p, "exp_avg": m, "exp_avg_sq": v}
    # the rounded states follow a random number's place, which 64 bits do not share; their
    # scales do not
    return {"param": p, "exp_avg": None, "exp_avg_scale": m.view(-1, _BLOCK).abs().amax(1) / 448,
            "exp_avg_sqrt": None,
            "exp_avg_sqrt_scale": v.view(-1, _BLOCK).amax(1).sqrt() / 448}


def _exact_scan(case, s):
    """Frame by frame, then back."""
    x, f, h = s["x"], torch.sigmoid(s["gate"]), s["state"]
    b, t, d = x.shape
    length = s["lengths"] if s["lengths"] is not None else torch.full((b,), t, device=x.device)
    live = (torch.arange(t, device=x.device) < length.unsqueeze(1)).unsqueeze(2)
    f = f.masked_fill(~live, 1.0)
    hs = torch.empty(t + 1, b, d, dtype=torch.float64, device=x.device)
    hs[0] = h
    ft, xt = f.transpose(0, 1).contiguous(), x.transpose(0, 1).contiguous()
    for k in range(t):
        torch.lerp(xt[k], hs[k], ft[k], out=hs[k + 1])
    out = {"y": (hs[1:].transpose(0, 1) * live), "state": hs[t].clone()}
    if not case["train"]:
        return out
    gy = (s["dy"] * live).transpose(0, 1).contiguous()
    lam = torch.empty_like(gy)
    carry = s["dstate"]
    for k in range(t - 1, -1, -1):
        torch.add(gy[k], carry, out=lam[k])
        carry = lam[k] * ft[k]
    out["dx"] = (lam * (1 - ft)).transpose(0, 1)
    out["dgate"] = (lam * (hs[:-1] - xt) * ft * (1 - ft)).transpose(0, 1)
    out["dstate"] = carry
    return out
