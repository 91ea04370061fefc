"""Layer norm and the gated feed-forward block over stacks of active blocks: the cases that are timed.

A stack ``[blocks, bh, bw, C]`` (or any ``[..., C]``) is a list of rows of ``C`` channels.  Two operators:

* layer norm over the channels: ``y = (x - mean) / sqrt(var + eps) * w + b`` and its backward pass;
* the gated feed-forward block ``y = (act(x Wg^T) * (x Wu^T)) Wd^T`` and its backward pass.

``own`` is false: :func:`run` computes them with elementary torch operations in 32 bits.  ``own`` is true:
it calls ``sbnet_b200``.
"""
import math

import torch

own = False

EPS = 1e-5
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def _case(op, train, rows, channels, hidden=0, act="", type="bf16", wtype="", block=1, blocks=0):
    """``blocks`` > 0: a stack with room for that many blocks of ``block`` rows, of which the first ``rows / block``
    are live; their number is known on the device only (the stack of a pipeline without a host round trip)."""
    return {"op": op, "train": train, "rows": rows, "channels": channels, "hidden": hidden, "act": act, "type": type,
            "wtype": wtype or type, "block": block, "blocks": blocks}


def listed():
    cases = {
        # one position of one sequence, weights kept in 32 bits: nothing but latency
        "norm_token": _case("norm", False, 1, 4096, wtype="f32"),
        # a fifth of the 16x16 blocks of eight 512x512 images, gathered with the count on the device
        "norm_blocks_counted": _case("norm", False, 1638 * 256, 128, type="f16", block=256, blocks=2048),
        # fp32 activations of an odd width: no row but the first starts on a 16-byte boundary
        "norm_train_odd": _case("norm", True, 20011, 1001, type="f32"),
        # the same fifth of the blocks in training, twice the channels, master weights in 32 bits
        "norm_train_blocks": _case("norm", True, 1638 * 256, 256, wtype="f32"),
        # a training batch of wide rows
        "norm_train_wide": _case("norm", True, 8192, 8192),
        # one position: every weight is read for one row
        "ffn_token": _case("ffn", False, 1, 4096, 12288, "silu"),
        # a ragged batch of single positions
        "ffn_decode": _case("ffn", False, 37, 2048, 8192, "gelu", type="f16"),
        # the residual branch on a fifth of the blocks of eight images, count on the device
        "ffn_blocks_counted": _case("ffn", False, 1638 * 256, 128, 512, "silu", type="f16", block=256, blocks=2048),
        # a long prompt through a wide model
        "ffn_prefill": _case("ffn", False, 4096, 4096, 12288, "silu"),
        # the residual branch in training on 400 blocks
        "ffn_train_blocks": _case("ffn", True, 400 * 256, 256, 1024, "silu"),
        # a training batch of a model of ordinary width
        "ffn_train_large": _case("ffn", True, 8192, 2048, 8192, "gelu"),
        # few rows, every size odd
        "ffn_train_odd": _case("ffn", True, 777, 333, 1001, "relu", type="f16"),
    }
    return [dict(c, name=n) for n, c in cases.items()]


def _between(rng, low, high):
    """A whole number, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    train = rng.random() < 0.5
    block, blocks = 1, 0
    if rng.random() < 0.5:
        channels = _between(rng, 24, 8192)
        if rng.random() < 0.5:
            channels = max(8, channels // 8 * 8)
        rows = _between(rng, 1, min(420_000, 64_000_000 // channels))
        type = rng.choice(["f32", "f16", "bf16"])
        hidden, act = 0, ""
        wtype = rng.choice([type, "f32"])
    else:
        channels, hidden = _between(rng, 32, 4096), _between(rng, 64, 12288)
        if rng.random() < 0.7:
            channels, hidden = max(8, channels // 8 * 8), max(8, hidden // 8 * 8)
        # at most the work of the largest listed case of the kind, and no more than 3 GB a temporary
        most = 130_000_000_000 if train else 200_000_000_000
        rows = _between(rng, 1, max(2, min(300_000, most // (channels * hidden), 120_000_000 // max(channels, hidden))))
        type = rng.choice(["f16", "bf16"])
        act = rng.choice(["silu", "gelu", "relu"])
        wtype = type
    if not train and rng.random() < 0.4:
        block = rng.choice([1, 9, 64, 100, 256])
        live = max(1, rows // block)
        rows, blocks = live * block, live + rng.randrange(0, live // 2 + 2)
    return _case("ffn" if hidden else "norm", train, rows, channels, hidden, act, type, wtype, block, blocks)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype, wdtype = _TYPES[case["type"]], _TYPES[case["wtype"]]
    rows, c, f = case["rows"], case["channels"], case["hidden"]
    shape = (case["blocks"], case["block"], c) if case["blocks"] else (rows, c)

    def normal(shape, scale=1.0, shift=0.0, dtype=dtype):
        t = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
        return t.mul_(scale).add_(shift).to(dtype)

    s = {"op": case["op"], "train": case["train"], "act": case["act"]}
    if case["op"] == "norm":
        # activations of a residual stream: a shift of their own and a few channels that stand out
        s["x"] = normal(shape, 1.5, 0.25)
        s["x"][..., :: max(1, c // 4)] *= 4
        s["weight"] = normal((c,), 0.2, 1.0, wdtype)
        s["bias"] = normal((c,), 0.2, 0.0, wdtype)
        leaves = ("x", "weight", "bias")
    else:
        s["x"] = normal(shape)
        s["w_gate"] = normal((f, c), 1 / math.sqrt(c))
        s["w_up"] = normal((f, c), 1 / math.sqrt(c))
        s["w_down"] = normal((c, f), 1 / math.sqrt(f))
        leaves = ("x", "w_gate", "w_up", "w_down")
    if case["train"]:
        s["dy"] = normal(shape)
        for k in leaves:
            s[k].requires_grad_(True)
    if case["blocks"]:
        s["count"] = torch.tensor([rows // case["block"]], dtype=torch.int32, device="cuda")
        s["out"] = torch.zeros(shape, dtype=dtype, device="cuda")
    s["leaves"] = [s[k] for k in leaves]
    return s


# ---- the plain forms ---------------------------------------------------------------------------------

def _rows(t):
    return t.reshape(-1, t.shape[-1]).float()


def _live(s, y):
    """Writes the live blocks of ``y`` into the caller's buffer and leaves the rest of it alone."""
    out = s["out"]
    live = torch.arange(out.shape[0], device=out.device) < s["count"]
    out.copy_(torch.where(live[:, None, None], y.reshape(out.shape), out))
    return out


def _plain_norm(s):
    x, w, b = _rows(s["x"]), s["weight"].float(), s["bias"].float()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = torch.rsqrt((d * d).mean(1, keepdim=True) + EPS)
    xhat = d * rstd
    y = (xhat * w + b).to(s["x"].dtype).reshape(s["x"].shape)
    if not s["train"]:
        return _live(s, y) if "out" in s else y
    g = _rows(s["dy"])
    gw = g * w
    dx = rstd * (gw - gw.mean(1, keepdim=True) - xhat * (gw * xhat).mean(1, keepdim=True))
    dw, db = (g * xhat).sum(0), g.sum(0)
    return y, dx.to(y.dtype).reshape(y.shape), dw.to(s["weight"].dtype), db.to(s["bias"].dtype)


def _act(name, g):
    """The activation and its derivative."""
    if name == "silu":
        sig = 1 / (1 + torch.exp(-g))
        return g * sig, sig * (1 + g * (1 - sig))
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    return g * (g > 0), (g > 0).float()


def _plain_ffn(s):
    dtype = s["x"].dtype
    x, wg, wu, wd = _rows(s["x"]), s["w_gate"].float(), s["w_up"].float(), s["w_down"].float()
    g, u = x @ wg.t(), x @ wu.t()
    a, slope = _act(s["act"], g)
    h = a * u
    y = (h @ wd.t()).to(dtype).reshape(s["x"].shape)
    if not s["train"]:
        return _live(s, y) if "out" in s else y
    dy = _rows(s["dy"])
    dh = dy @ wd
    du, dg = dh * a, dh * u * slope
    dx = dg @ wg + du @ wu
    return (y, dx.to(dtype).reshape(y.shape), (dg.t() @ x).to(dtype), (du.t() @ x).to(dtype), (dy.t() @ h).to(dtype))


# ---- the framework's calls -----------------------------------------------------------------------------

def _own(s):
    from sbnet_b200 import autograd, ops
    if s["op"] == "norm":
        if s["train"]:
            y = autograd.layer_norm(s["x"], s["weight"], s["bias"], EPS)
            return (y.detach(), *torch.autograd.grad(y, s["leaves"], s["dy"]))
        if "out" in s:
            return ops.layer_norm_dyn(s["x"], s["count"], s["weight"], s["bias"], EPS, out=s["out"])
        return ops.layer_norm(s["x"], s["weight"], s["bias"], EPS)
    weights = (s["w_gate"], s["w_up"], s["w_down"])
    if s["train"]:
        y = autograd.gated_ffn(s["x"], *weights, activation=s["act"])
        return (y.detach(), *torch.autograd.grad(y, s["leaves"], s["dy"]))
    if "out" in s:
        return ops.gated_ffn_dyn(s["x"], s["count"], *weights, activation=s["act"], out=s["out"])
    return ops.gated_ffn(s["x"], *weights, activation=s["act"])


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain_norm(state) if state["op"] == "norm" else _plain_ffn(state)


def work(case):
    rows, c, f, e = case["rows"], case["channels"], case["hidden"], _BYTES[case["type"]]
    sides = 4 if case["train"] else 2          # x, y and in training dy, dx
    if case["op"] == "norm":
        weights = (4 if case["train"] else 2) * c * _BYTES[case["wtype"]]
        return {"bytes": sides * rows * c * e + weights, "flops": (20 if case["train"] else 8) * rows * c}
    weights = (6 if case["train"] else 3) * c * f * e
    return {"bytes": sides * rows * c * e + weights, "flops": (18 if case["train"] else 6) * rows * c * f}


def exact(case, seed):
    """The definitions in 64 bits; the gradients by differentiating them."""
    s = prepare(case, seed)
    live = case["rows"] // case["block"] if case["blocks"] else None
    leaves = [t.detach().double().requires_grad_(case["train"]) for t in s["leaves"]]
    x = leaves[0]
    if case["op"] == "norm":
        var, mean = torch.var_mean(x, dim=-1, unbiased=False, keepdim=True)
        y = (x - mean) / torch.sqrt(var + EPS) * leaves[1] + leaves[2]
    else:
        gate, up = torch.matmul(x, leaves[1].mT), torch.matmul(x, leaves[2].mT)
        if case["act"] == "silu":
            gate = gate * torch.sigmoid(gate)
        elif case["act"] == "gelu":
            gate = gate * torch.special.ndtr(gate)
        else:
            gate = torch.clamp(gate, min=0)
        y = torch.matmul(gate * up, leaves[3].mT)
    if case["train"]:
        return (y.detach(), *torch.autograd.grad(y, leaves, s["dy"].double()))
    if live is not None:
        y[live:] = 0
    return y
