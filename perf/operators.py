"""Workloads of the layer norm over rows and of the gated feed-forward block: what they compute, on which sizes.

``own`` False: the operators in plain torch operations (32-bit arithmetic, rounded once at the end); ``own`` True: the
calls a user makes of ``cpm_kernels_b200.torch``.  The three operators:

* ``layernorm_rows(x, eps, weight, bias, rd_mean)``: layer norm of every row (``rd_mean=False``: the RMS form);
* ``gated_linear(x, w_gate, w_up, activation)``: ``act(x w_gate^T) * (x w_up^T)``;
* ``gated_feed_forward(x, w_gate, w_up, w_down, activation)``: the above times ``w_down^T``.

A case with ``train`` returns the output and the gradients of every differentiable input for a given output gradient.
"""
import math

import torch

own = False

EPS = 1e-5
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZES = {"fp16": 2, "bf16": 2, "fp32": 4}


def _ln(name, rows, n, dtype, train, mean, bias):
    return {"name": name, "op": "layernorm_rows", "rows": rows, "n": n, "dtype": dtype, "train": train, "rd_mean": mean, "bias": bias}


def _gated(name, tokens, k, n, dtype, train, act):
    return {"name": name, "op": "gated_linear", "tokens": tokens, "k": k, "n": n, "dtype": dtype, "train": train, "act": act}


def _ff(name, tokens, k, n, dtype, train, act):
    return {"name": name, "op": "gated_feed_forward", "tokens": tokens, "k": k, "n": n, "dtype": dtype, "train": train, "act": act}


def listed():
    return [
        # one token of a decoding step in front of the feed-forward block: launch latency
        _ln("ln_decode_1x4096_fp16", 1, 4096, "fp16", False, False, False),
        # the activations of a 4096-token prefill
        _ln("ln_4096x4096_fp16", 4096, 4096, "fp16", False, True, True),
        # a ragged training batch of a model whose width is odd
        _ln("ln_train_1027x5001_bf16", 1027, 5001, "bf16", True, True, True),
        # a large training batch, RMS form
        _ln("ln_train_16384x4096_bf16", 16384, 4096, "bf16", True, False, False),
        # a small model trained in 32 bits
        _ln("ln_train_8192x1024_fp32", 8192, 1024, "fp32", True, True, True),
        # a batch of decoding sequences, with the second linear done elsewhere (for instance in int8)
        _gated("gated_33x4096x10240_bf16", 33, 4096, 10240, "bf16", False, "silu"),
        # training of a small model, ragged token count
        _gated("gated_train_1000x1024x2816_fp16", 1000, 1024, 2816, "fp16", True, "gelu"),
        # one decoding step, a single sequence
        _ff("ff_decode_1x4096x10240_fp16", 1, 4096, 10240, "fp16", False, "gelu"),
        # a batch of decoding sequences
        _ff("ff_decode_48x4096x10240_bf16", 48, 4096, 10240, "bf16", False, "silu"),
        # prefill
        _ff("ff_4096x4096x10240_fp16", 4096, 4096, 10240, "fp16", False, "gelu"),
        # training of a very small model on a short ragged batch
        _ff("ff_train_201x512x1368_fp16", 201, 512, 1368, "fp16", True, "silu"),
        # a training step of the full-width block
        _ff("ff_train_4096x4096x10240_bf16", 4096, 4096, 10240, "bf16", True, "gelu"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["layernorm_rows", "layernorm_rows", "gated_linear", "gated_feed_forward", "gated_feed_forward"])
    train = rng.random() < 0.5
    if op == "layernorm_rows":
        n = _log(rng, 8, 20000)
        if rng.random() < 0.6:
            n = (n + 7) // 8 * 8                       # most widths are multiples of 8, the others any number
        rows = _log(rng, 1, max(1, 16384 * 4096 // n // 2))
        return {"op": op, "rows": min(rows, 60000), "n": n, "dtype": rng.choice(["fp16", "bf16", "fp32"]), "train": train,
                "rd_mean": rng.random() < 0.5, "bias": rng.random() < 0.5}
    k = _log(rng, 64, 4096) // 8 * 8
    n = _log(rng, 64, 10240) // 8 * 8
    return {"op": op, "tokens": _log(rng, 1, 4096), "k": k, "n": n, "dtype": rng.choice(["fp16", "bf16"]), "train": train,
            "act": rng.choice(["gelu", "silu"])}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(shape, std=1.0, mean=0.0, leaf=case["train"]):
        t = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).add_(mean).to(dtype)
        return t.requires_grad_(leaf)

    state = {"case": case}
    if case["op"] == "layernorm_rows":
        rows, n = case["rows"], case["n"]
        state["x"] = normal((rows, n), 1.5, 0.25)      # a residual stream: some spread, a small common offset
        state["weight"] = normal((n,), 0.1, 1.0)
        state["bias"] = normal((n,), 0.1) if case["bias"] else None
        if case["train"]:
            state["dy"] = normal((rows, n), leaf=False)
        return state
    tokens, k, n = case["tokens"], case["k"], case["n"]
    state["x"] = normal((tokens, k))                   # what a layer norm hands over
    state["w_gate"] = normal((n, k), k ** -0.5)
    state["w_up"] = normal((n, k), k ** -0.5)
    if case["op"] == "gated_feed_forward":
        state["w_down"] = normal((k, n), n ** -0.5)
    if case["train"]:
        state["dy"] = normal((tokens, k if case["op"] == "gated_feed_forward" else n), leaf=False)
    return state


def _plain_layernorm(s):
    case, dtype = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    mean = x.mean(-1, keepdim=True) if case["rd_mean"] else torch.zeros((), device=x.device)
    centred = x - mean
    rstd = 1.0 / ((centred * centred).mean(-1, keepdim=True) + EPS).sqrt()
    xhat = centred * rstd
    y = xhat * w
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if not case["train"]:
        return [y.to(dtype)]
    dy = s["dy"].float()
    gw = dy * w
    dx = gw - xhat * (gw * xhat).mean(-1, keepdim=True)
    if case["rd_mean"]:
        dx = dx - gw.mean(-1, keepdim=True)
    out = [y.to(dtype), (dx * rstd).to(dtype), (dy * xhat).sum(0).to(dtype)]
    if s["bias"] is not None:
        out.append(dy.sum(0).to(dtype))
    return out


def _act_and_slope(g, act):
    """act(g) and act'(g); both activations are g * sigmoid(z(g))."""
    if act == "silu":
        sig = 1.0 / (1.0 + torch.exp(-g))
        return g * sig, sig * (1.0 + g * (1.0 - sig))
    c = math.sqrt(2.0 / math.pi)
    sig = 1.0 / (1.0 + torch.exp(-2.0 * c * (g + 0.044715 * g * g * g)))
    return g * sig, sig + g * sig * (1.0 - sig) * (2.0 * c * (1.0 + 3.0 * 0.044715 * g * g))


def _plain_gated(s):
    case, dtype = s["case"], s["x"].dtype
    x, wg, wu = s["x"].float(), s["w_gate"].float(), s["w_up"].float()
    wd = s["w_down"].float() if "w_down" in s else None
    g, u = x @ wg.t(), x @ wu.t()
    a, slope = _act_and_slope(g, case["act"])
    h = a * u
    y = h if wd is None else h @ wd.t()
    if not case["train"]:
        return [y.to(dtype)]
    dy = s["dy"].float()
    dh = dy if wd is None else dy @ wd
    dg, du = dh * u * slope, dh * a
    out = [y.to(dtype), (dg @ wg + du @ wu).to(dtype), (dg.t() @ x).to(dtype), (du.t() @ x).to(dtype)]
    if wd is not None:
        out.append((dy.t() @ h).to(dtype))
    return out


def run(state):
    case = state["case"]
    if not own:
        with torch.no_grad():
            return _plain_layernorm(state) if case["op"] == "layernorm_rows" else _plain_gated(state)
    import cpm_kernels_b200.torch as ct
    if case["op"] == "layernorm_rows":
        leaves = [t for t in (state["x"], state["weight"], state["bias"]) if t is not None]
        y = ct.layernorm_rows(state["x"], EPS, state["weight"], state["bias"], rd_mean=case["rd_mean"])
    elif case["op"] == "gated_linear":
        leaves = [state["x"], state["w_gate"], state["w_up"]]
        y = ct.gated_linear(*leaves, activation=case["act"])
    else:
        leaves = [state["x"], state["w_gate"], state["w_up"], state["w_down"]]
        y = ct.gated_feed_forward(*leaves, activation=case["act"])
    if not case["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, leaves, state["dy"])]


def exact(case, seed):
    """The definitions in 64 bits, the gradients by automatic differentiation of them."""
    s = prepare(case, seed)
    names = [k for k in ("x", "weight", "bias", "w_gate", "w_up", "w_down") if s.get(k) is not None]
    t = {k: s[k].detach().double().requires_grad_(case["train"]) for k in names}
    if case["op"] == "layernorm_rows":
        x = t["x"]
        if case["rd_mean"]:
            x = x - x.sum(-1, keepdim=True) / case["n"]
        y = x / torch.sqrt(x.square().sum(-1, keepdim=True) / case["n"] + EPS) * t["weight"]
        if "bias" in t:
            y = y + t["bias"]
    else:
        g, u = torch.matmul(t["x"], t["w_gate"].T), torch.matmul(t["x"], t["w_up"].T)
        if case["act"] == "silu":
            a = g * torch.sigmoid(g)
        else:
            a = 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3)))
        y = a * u
        if "w_down" in t:
            y = torch.matmul(y, t["w_down"].T)
    if not case["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, [t[k] for k in names], s["dy"].double())]


def work(case):
    es = SIZES[case["dtype"]]
    if case["op"] == "layernorm_rows":
        rows, n = case["rows"], case["n"]
        vectors = 2 if case["bias"] else 1
        if not case["train"]:
            return {"bytes": es * (2 * rows * n + vectors * n), "flops": 8 * rows * n}
        return {"bytes": es * (4 * rows * n + 2 * vectors * n), "flops": 20 * rows * n}       # x, dy in; y, dx out
    tokens, k, n = case["tokens"], case["k"], case["n"]
    block = case["op"] == "gated_feed_forward"
    weights = (3 if block else 2) * n * k
    out = tokens * (k if block else n)
    flops = 2 * tokens * weights
    if not case["train"]:
        return {"bytes": es * (tokens * k + weights + out), "flops": flops}
    return {"bytes": es * (2 * tokens * k + 2 * weights + 2 * out), "flops": 3 * flops}
