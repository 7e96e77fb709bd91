"""Workloads of the operators that train a head on a map: layer norm, gated projections, distillation from the map's routes.

`run` computes them in plain torch operations, or -- with `own` set -- through pink_b200.readout.  `exact` computes the same
from the definitions in 64 bits.
"""
import math

import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
EPS = 1e-5


# ---- cases ---------------------------------------------------------------------------------------------------------------

def _norm(name, **kw):
    return {**dict(op="norm", n=1, D=400, type="float32", affine=True, keep=False, padded=False), **kw, "name": name}


def _norm_grad(name, **kw):
    return {**dict(op="norm_grad", n=1, D=400, type="float32", affine=True, residual=False, padded=False), **kw, "name": name}


def _gated(name, **kw):
    case = dict(op="gated", n=1, K=400, M=10, type="bfloat16", by_input=False, bias=True, activation="silu", keep=False, padded=False)
    return {**case, **kw, "name": name}


def _gated_grad(name, **kw):
    case = dict(op="gated_grad", n=1, K=400, M=10, type="bfloat16", by_input=False, activation="silu", padded=False)
    return {**case, **kw, "name": name}


def _distill(name, **kw):
    case = dict(op="distill", n=1, N=400, k=4, type="float32", teacher="weights", temperature=1.0, scale=1.0, rest=False, mask=False,
                holes=False, padded=False)
    return {**case, **kw, "name": name}


def _distill_grad(name, **kw):
    return {**_distill(name, **kw), "op": "distill_grad"}


def listed():
    return [
        # one image's prototype pixels (90 x 90), normalised as it arrives
        _norm("norm one image", n=1, D=8100),
        # distance regions of 63 x 63 pixels of a survey's images, in front of a head that is being trained
        _norm("norm regions", n=65536, D=3969, type="bfloat16", keep=True),
        # fine-tuning on a few regions of 31 x 31 pixels
        _norm_grad("norm gradient of a few", n=64, D=961, type="float16"),
        # training a head that rebuilds images of 90 x 90 pixels: the gradient of the skip path joins
        _norm_grad("norm gradient images", n=16384, D=8100, type="bfloat16", residual=True),
        # one image through a head whose hidden layer has as many units as the headline map has neurons
        _gated("gated one image", n=1, K=8100, M=2791),
        # a batch of regions through a hidden layer as wide as an image, pre-activations kept for training
        _gated("gated regions", n=8192, K=3969, M=8100, activation="gelu", keep=True),
        # a small head on the 20 x 20 map, weights in rows by input
        _gated_grad("gated gradient 20x20", n=331, K=961, M=400, type="float16", by_input=True, activation="gelu"),
        # training the hidden layer of the headline map's head
        _gated_grad("gated gradient regions", n=4096, K=3969, M=2791),
        # the loss of one image against its four routes on the 2,791-neuron map
        _distill("distill one image", n=1, N=2791, k=4),
        # validation over a survey: the routes' weights leave a rest for the other neurons
        _distill("distill survey", n=65536, N=2791, k=8, type="bfloat16", rest=True),
        # a training step against the logits of the 20 x 20 map, softened; some neurons are left out, some images have no routes
        _distill_grad("distill gradient 20x20", n=4096, N=400, k=8, type="float16", teacher="logits", temperature=2.0, scale=4.0, mask=True,
                      holes=True),
        # a training step of a float32 head on the headline map
        _distill_grad("distill gradient hex 2791", n=16384, N=2791, k=8),
    ]


def _size(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "gated", "gated_grad", "distill", "distill_grad"])
    flag = lambda p=0.5: rng.random() < p
    if op in ("norm", "norm_grad"):
        D = _size(rng, 16, 16384)                        # (of two elements nothing but rounding is left of a gradient)
        common = dict(n=_size(rng, 1, min(65536, (65536 * 3969 if op == "norm" else 16384 * 8100) // D)), D=D, type=rng.choice(sorted(TYPES)),
                      affine=flag(0.8), padded=flag(0.3))
        if common["type"] == "float32":
            common["n"] = (common["n"] + 1) // 2
        case = _norm("", **common, keep=flag()) if op == "norm" else _norm_grad("", **common, residual=flag())
    elif op in ("gated", "gated_grad"):
        K, M = _size(rng, 1, 8192), _size(rng, 1, 8192)
        n = _size(rng, 1, min(8192, (8192 * 3969 * 8100 if op == "gated" else 4096 * 3969 * 2791) // (K * M)))
        common = dict(n=n, K=K, M=M, type=rng.choice(["bfloat16", "float16"]), by_input=flag(), padded=flag(),
                      activation=rng.choice(["none", "relu", "gelu", "silu", "silu", "sigmoid"]))
        case = _gated("", **common, bias=flag(), keep=flag()) if op == "gated" else _gated_grad("", **common)
    else:
        N = _size(rng, 1, 8192)
        n = _size(rng, 1, min(65536, (65536 if op == "distill" else 16384) * 2791 // N))
        teacher = rng.choice(["weights", "weights", "logits"])
        kw = dict(n=n, N=N, k=rng.randint(1, min(N, 16)), type=rng.choice(sorted(TYPES)), teacher=teacher, temperature=rng.choice([1.0, 2.0, 0.7]),
                  scale=rng.choice([1.0, 4.0]), rest=teacher == "weights" and flag(), mask=flag(0.3), holes=flag(0.3), padded=flag(0.3))
        case = (_distill if op == "distill" else _distill_grad)("", **kw)
    return {k_: v for k_, v in case.items() if k_ != "name"}


# ---- inputs --------------------------------------------------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _uniform(g, *shape):
    return torch.rand(shape, generator=g, device="cuda")


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _laid(t, padded):
    """The same matrix; with `padded` in rows of whole 128-byte lines, as the operators lay out what they return."""
    if not padded:
        return t.contiguous()
    line = 128 // t.element_size()
    wide = torch.zeros((t.shape[0], -(-t.shape[1] // line) * line), dtype=t.dtype, device=t.device)
    wide[:, :t.shape[1]] = t
    return wide[:, :t.shape[1]]


def _features(g, n, D):
    """Rows of their own brightness and contrast, as images and hidden layers have them."""
    return _normal(g, n, D) * (0.3 + _uniform(g, n, 1)) + _normal(g, n, 1)


def _teacher(g, case):
    """Scores of a head that has learned something but not all, and the routes of the map that teaches it."""
    n, N, k = case["n"], case["N"], case["k"]
    at, of = _uniform(g, n, 2), _uniform(g, N, 2)
    logits = -2.0 * torch.sqrt(16.0 + 60.0 * ((at[:, None, 0] - of[None, :, 0]) ** 2 + (at[:, None, 1] - of[None, :, 1]) ** 2))
    scores = logits + 1.5 * _normal(g, n, N)
    top = torch.topk(logits, k, dim=1)
    neurons = top.indices.int()
    if case["teacher"] == "logits":
        targets = top.values.contiguous()
    else:
        targets = torch.softmax(logits, 1).gather(1, top.indices)
        if not case["rest"]:
            targets = targets / targets.sum(1, keepdim=True)
    mask = _uniform(g, N) > 0.05 if case["mask"] else None
    if mask is not None:                                 # what stands in the places that are left out does not matter
        scores[:, ~mask] = torch.where(_uniform(g, n, int((~mask).sum())) < 0.5, math.nan, math.inf)
    if case["holes"]:
        gone = (_uniform(g, n, k) < 0.05) | (_uniform(g, n, 1) < 0.02)
        neurons, targets = torch.where(gone, -1, neurons), torch.where(gone, 0.0, targets)
        out = _uniform(g, n, N) < 0.01                   # neurons that the head itself rules out
        scores[out if mask is None else out & mask] = -math.inf
    return _laid(scores.to(TYPES[case["type"]]), case["padded"]), neurons, targets, mask


def prepare(case, seed):
    g, op = _generator(seed), case["op"]
    state, n, dtype = {"case": case}, case["n"], TYPES[case["type"]]
    if op in ("norm", "norm_grad"):
        D = case["D"]
        state["x"] = _laid(_features(g, n, D).to(dtype), case["padded"])
        state["weight"] = 1.0 + 0.2 * _normal(g, D) if case["affine"] else None
        state["bias"] = 0.2 * _normal(g, D) if case["affine"] and op == "norm" else None
        if op == "norm_grad":
            state["dy"] = _laid(_normal(g, n, D).to(dtype), case["padded"])
            state["residual"] = _laid(_normal(g, n, D).to(dtype), case["padded"]) if case["residual"] else None
            mean, rstd = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
            for i in range(0, n, 4096):
                x = state["x"][i:i + 4096].double()
                mean[i:i + 4096] = x.mean(1)
                rstd[i:i + 4096] = (x.var(1, correction=0) + EPS).rsqrt()
            state["mean"], state["rstd"] = mean, rstd
    elif op in ("gated", "gated_grad"):
        K, M = case["K"], case["M"]
        state["x"] = _laid(_normal(g, n, K).to(dtype), case["padded"])
        for name in ("gate", "up"):
            w = _normal(g, M, K) / math.sqrt(K)
            state[name] = _laid((w.t() if case["by_input"] else w).to(dtype), case["padded"])
        if op == "gated":
            state["gate_bias"], state["up_bias"] = (0.5 * _normal(g, M), 0.5 * _normal(g, M)) if case["bias"] else (None, None)
        else:
            for name in ("g", "u", "dy"):
                state[name] = _laid(_normal(g, n, M).to(dtype), case["padded"])
    else:
        state["scores"], state["neurons"], state["targets"], state["mask"] = _teacher(g, case)
        if op == "distill_grad":
            state["dloss"] = 0.5 + _uniform(g, n)
    return state


# ---- the plain form ------------------------------------------------------------------------------------------------------

def _plain_norm(x, weight, bias):
    mean = x.mean(1, keepdim=True)
    away = x - mean
    rstd = 1.0 / torch.sqrt((away * away).mean(1, keepdim=True) + EPS)
    y = away * rstd
    if weight is not None:
        y = y * weight
    if bias is not None:
        y = y + bias
    return y, mean[:, 0], rstd[:, 0]


def _plain_norm_grad(state):
    x, dy, rstd = state["x"].float(), state["dy"].float(), state["rstd"][:, None]
    xhat = (x - state["mean"][:, None]) * rstd
    g = dy if state["weight"] is None else dy * state["weight"]
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    if state["residual"] is not None:
        dx = dx + state["residual"].float()
    return {"dx": dx.to(state["x"].dtype), "dweight": (dy * xhat).sum(0), "dbias": dy.sum(0)}


def _plain_act(z, activation):
    if activation == "relu":
        return torch.clamp(z, min=0.0)
    if activation == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if activation == "silu":
        return z * torch.sigmoid(z)
    if activation == "sigmoid":
        return torch.sigmoid(z)
    return z


def _plain_act_slope(z, activation):
    if activation == "relu":
        return (z > 0).to(z.dtype)
    if activation == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if activation == "silu":
        s = torch.sigmoid(z)
        return s * (1.0 + z * (1.0 - s))
    if activation == "sigmoid":
        s = torch.sigmoid(z)
        return s * (1.0 - s)
    return torch.ones_like(z)


def _plain_gated(state):
    case, dtype = state["case"], state["x"].dtype
    x, gate, up = state["x"].float(), state["gate"].float(), state["up"].float()
    if not case["by_input"]:
        gate, up = gate.t(), up.t()
    g, u = x @ gate, x @ up
    if state["gate_bias"] is not None:
        g, u = g + state["gate_bias"], u + state["up_bias"]
    out = {"h": (_plain_act(g, case["activation"]) * u).to(dtype)}
    if case["keep"]:
        out["g"], out["u"] = g.to(dtype), u.to(dtype)
    return out


def _plain_gated_grad(state):
    case, dtype = state["case"], state["x"].dtype
    x, gate, up = state["x"].float(), state["gate"].float(), state["up"].float()
    g, u, dy = state["g"].float(), state["u"].float(), state["dy"].float()
    dg = dy * u * _plain_act_slope(g, case["activation"])
    du = dy * _plain_act(g, case["activation"])
    if case["by_input"]:
        dx, dgate, dup = dg @ gate.t() + du @ up.t(), x.t() @ dg, x.t() @ du
    else:
        dx, dgate, dup = dg @ gate + du @ up, dg.t() @ x, du.t() @ x
    return {"dx": dx.to(dtype), "dgate": dgate.to(dtype), "dup": dup.to(dtype), "dgate_bias": dg.sum(0), "dup_bias": du.sum(0)}


def _plain_distill(state, grad):
    """loss = scale * (sum of p (log p - log q) over the targets + the rest's), q the softmax of the scores over the temperature."""
    case, scores, neurons, targets, mask = state["case"], state["scores"], state["neurons"], state["targets"], state["mask"]
    n, N = scores.shape
    logits = scores.float() / case["temperature"]
    part = logits != -math.inf
    if mask is not None:
        part = part & mask
    logits = torch.where(part, logits, -math.inf)
    most = logits.amax(1, keepdim=True)
    e = torch.exp(logits - torch.where(most == -math.inf, 0.0, most))
    total = e.sum(1, keepdim=True)
    there = (neurons >= 0) & (neurons < N)
    index = torch.where(there, neurons, 0).long()
    there = there & part.gather(1, index)
    if case["teacher"] == "logits":
        t = targets / case["temperature"]
        there = there & (t > -math.inf)
        t = torch.where(there, t, -math.inf)
        high = t.amax(1, keepdim=True)
        p = torch.exp(t - torch.where(high == -math.inf, 0.0, high))
        p = p / p.sum(1, keepdim=True).clamp(min=1e-30)
    else:
        there = there & (targets > 0)
        p = torch.where(there, targets, 0.0)
    log_q = (logits.gather(1, index) - most) - torch.log(total)
    terms = torch.where(there & (p > 0), p * (torch.log(torch.where(p > 0, p, 1.0)) - torch.where(there, log_q, 0.0)), 0.0)
    loss = terms.sum(1)
    mass = p.sum(1, keepdim=True)
    some = there.any(1)
    if case["rest"]:
        other = torch.cat([part, part[:, :1]], 1).scatter_(1, torch.where(there, index, N), False)[:, :N]
        e_other = torch.where(other, e, 0.0)
        e_rest = e_other.sum(1, keepdim=True)
        r = (1.0 - torch.where(there, targets, 0.0).double().sum(1, keepdim=True)).clamp(min=0.0)
        r = torch.where(e_rest > 0, r, 0.0)
        # r over the rest's q, which are close to one another: 1 / q = 1 + what the targets have over the others' sum
        more = torch.where(there, e.gather(1, index), 0.0).double().sum(1, keepdim=True) / e_rest.clamp(min=1e-30).double()
        ratio = torch.where((r > 0) & (e_rest > 0), r * (1.0 + more), 1.0)
        loss = loss + (r * torch.log(ratio)).float()[:, 0]
        r = r.float()
        mass = mass + r
    out = {"loss": torch.where(some, case["scale"] * loss, 0.0)}
    if grad:
        q = e / total.clamp(min=1e-30)
        d = q * mass
        if case["rest"]:
            d = d - r * e_other / e_rest.clamp(min=1e-30)
        d.scatter_add_(1, index, torch.where(there, -p, 0.0))
        d = d * (state["dloss"][:, None] * (case["scale"] / case["temperature"]))
        out["dscores"] = torch.where(part & some[:, None], d, 0.0).to(scores.dtype)
    return out


def _run_plain(state):
    case, op = state["case"], state["case"]["op"]
    if op == "norm":
        y, mean, rstd = _plain_norm(state["x"].float(), state["weight"], state["bias"])
        out = {"y": y.to(state["x"].dtype)}
        if case["keep"]:
            out["mean"], out["rstd"] = mean, rstd
        return out
    if op == "norm_grad":
        return _plain_norm_grad(state)
    if op == "gated":
        return _plain_gated(state)
    if op == "gated_grad":
        return _plain_gated_grad(state)
    return _plain_distill(state, op == "distill_grad")


# ---- the framework's calls -----------------------------------------------------------------------------------------------

def _run_own(state):
    from pink_b200 import readout
    case, op = state["case"], state["case"]["op"]
    if op == "norm":
        out = readout.layer_norm(state["x"], state["weight"], state["bias"], eps=EPS, keep=case["keep"])
        return dict(zip(("y", "mean", "rstd"), out)) if case["keep"] else {"y": out}
    if op == "norm_grad":
        out = readout.layer_norm_backward(state["dy"], state["x"], state["mean"], state["rstd"], state["weight"], residual=state["residual"])
        return dict(zip(("dx", "dweight", "dbias"), out))
    if op == "gated":
        out = readout.gated(state["x"], state["gate"], state["up"], by_input=case["by_input"], gate_bias=state["gate_bias"],
                            up_bias=state["up_bias"], activation=case["activation"], keep=case["keep"])
        return dict(zip(("h", "g", "u"), out)) if case["keep"] else {"h": out}
    if op == "gated_grad":
        out = readout.gated_backward(state["dy"], state["x"], state["gate"], state["up"], state["g"], state["u"], by_input=case["by_input"],
                                     activation=case["activation"])
        return dict(zip(("dx", "dgate", "dup", "dgate_bias", "dup_bias"), out))
    kw = dict(teacher=case["teacher"], temperature=case["temperature"], scale=case["scale"], rest=case["rest"], mask=state["mask"])
    if op == "distill":
        return {"loss": readout.distill(state["scores"], state["neurons"], state["targets"], **kw)}
    dscores, loss = readout.distill_backward(state["dloss"], state["scores"], state["neurons"], state["targets"], loss=True, **kw)
    return {"loss": loss, "dscores": dscores}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------

def work(case):
    op, n = case["op"], case["n"]
    size = 4 if case["type"] == "float32" else 2
    if op == "norm":
        D = case["D"]
        return {"bytes": 2 * n * D * size + (8 * D if case["affine"] else 0) + (8 * n if case["keep"] else 0), "flops": 8 * n * D}
    if op == "norm_grad":
        D = case["D"]
        return {"bytes": (4 if case["residual"] else 3) * n * D * size + (12 if case["affine"] else 8) * D + 8 * n, "flops": 14 * n * D}
    if op == "gated":
        K, M = case["K"], case["M"]
        return {"bytes": size * (n * K + 2 * K * M + n * M * (3 if case["keep"] else 1)) + (8 * M if case["bias"] else 0), "flops": 4 * n * K * M}
    if op == "gated_grad":
        K, M = case["K"], case["M"]
        return {"bytes": size * (2 * n * K + 4 * K * M + 3 * n * M) + 8 * M, "flops": 8 * n * K * M}
    N, k = case["N"], case["k"]
    return {"bytes": n * N * size * (1 if op == "distill" else 2) + n * (8 * k + (4 if op == "distill" else 8)), "flops": 6 * n * N}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------

def _exact_act(z, activation):
    if activation == "relu":
        return torch.relu(z)
    if activation == "gelu":
        return torch.nn.functional.gelu(z)
    if activation == "silu":
        return torch.nn.functional.silu(z)
    return torch.sigmoid(z) if activation == "sigmoid" else z


def _exact_norm(case, state):
    """The gradients of torch's own layer norm in 64 bits, some rows at a time."""
    D, grad, parts = case["D"], case["op"] == "norm_grad", []
    weight = torch.ones(D, dtype=torch.float64, device="cuda") if state["weight"] is None else state["weight"].double()
    shift = torch.zeros(D, dtype=torch.float64, device="cuda") if state["bias"] is None else state["bias"].double()
    dweight, dbias = torch.zeros_like(weight), torch.zeros_like(weight)
    for i in range(0, case["n"], 8192):
        x = state["x"][i:i + 8192].double()
        if not grad:
            y = torch.nn.functional.layer_norm(x, (D,), weight, shift, EPS)
            parts.append((y, x.mean(1), (x.var(1, correction=0) + EPS).rsqrt()))
            continue
        for t in (x, weight, shift):
            t.requires_grad_(True)
        y = torch.nn.functional.layer_norm(x, (D,), weight, shift, EPS)
        dx, dw, db = torch.autograd.grad(y, (x, weight, shift), state["dy"][i:i + 8192].double())
        parts.append((dx if state["residual"] is None else dx + state["residual"][i:i + 8192].double(),))
        dweight += dw.detach()
        dbias += db.detach()
    whole = [torch.cat(p) for p in zip(*parts)]
    if grad:
        return {"dx": whole[0], "dweight": dweight, "dbias": dbias}
    return {"y": whole[0], "mean": whole[1], "rstd": whole[2]} if case["keep"] else {"y": whole[0]}


def _exact_gated(case, state):
    x, gate, up = (state[k].double() for k in ("x", "gate", "up"))
    if not case["by_input"]:
        gate, up = gate.t(), up.t()                      # [K, M]
    if case["op"] == "gated":
        g = x @ gate if state["gate_bias"] is None else torch.addmm(state["gate_bias"].double(), x, gate)
        u = x @ up if state["up_bias"] is None else torch.addmm(state["up_bias"].double(), x, up)
        out = {"h": _exact_act(g, case["activation"]) * u}
        if case["keep"]:
            out["g"], out["u"] = g, u
        return out
    g, u = state["g"].double().requires_grad_(True), state["u"].double().requires_grad_(True)
    dg, du = torch.autograd.grad(_exact_act(g, case["activation"]) * u, (g, u), state["dy"].double())
    dgate, dup = x.t() @ dg, x.t() @ du
    if not case["by_input"]:
        dgate, dup = dgate.t(), dup.t()
    return {"dx": dg @ gate.t() + du @ up.t(), "dgate": dgate, "dup": dup, "dgate_bias": dg.sum(0), "dup_bias": du.sum(0)}


def _exact_distill(case, state):
    """The targets as a dense distribution over the neurons, the loss as a sum over all of them, its gradient by autograd; some rows at a time."""
    N, T, grad, parts = case["N"], case["temperature"], case["op"] == "distill_grad", []
    for i in range(0, case["n"], 8192):
        s = state["scores"][i:i + 8192].double()
        s = s if state["mask"] is None else s.masked_fill(~state["mask"], -math.inf)
        takes = s != -math.inf
        s = s.masked_fill(~takes, 0.0).requires_grad_(grad)
        log_q = torch.log_softmax((s / T).masked_fill(~takes, -math.inf), 1).masked_fill(~takes, 0.0)
        e, t = state["neurons"][i:i + 8192].long(), state["targets"][i:i + 8192].double()
        e = torch.where((e < 0) | (e >= N), N, e)
        seen = torch.cat([takes, torch.zeros_like(takes[:, :1])], 1).gather(1, e)
        if case["teacher"] == "logits":
            t = torch.nan_to_num(torch.softmax((t / T).masked_fill(~seen, -math.inf), 1), nan=0.0)
        else:
            t = torch.where(seen & (t > 0), t, torch.zeros_like(t))
        p = torch.zeros(s.shape[0], N + 1, dtype=torch.float64, device="cuda").scatter_add_(1, e, t)[:, :N]
        loss = torch.special.xlogy(p, p).sum(1) - (p * log_q).sum(1)
        if case["rest"]:
            others = takes & (p == 0)
            r = torch.where(others.any(1), (1.0 - p.sum(1)).clamp(min=0.0), torch.zeros_like(loss))
            low = torch.where(others, log_q, torch.full_like(log_q, -math.inf))
            low = torch.where(others.any(1, keepdim=True), low, torch.zeros_like(low))
            loss = loss + torch.special.xlogy(r, r) - r * torch.logsumexp(low, 1)
        loss = case["scale"] * torch.where((p > 0).any(1), loss, torch.zeros_like(loss))
        if not grad:
            parts.append((loss,))
            continue
        ds, = torch.autograd.grad(loss, s, state["dloss"][i:i + 8192].double())
        parts.append((loss.detach(), torch.where(takes, ds, torch.zeros_like(ds))))
    whole = [torch.cat(p) for p in zip(*parts)]
    return dict(zip(("loss", "dscores"), whole))


def exact(case, seed):
    state, op = prepare(case, seed), case["op"]
    if op in ("norm", "norm_grad"):
        return _exact_norm(case, state)
    if op in ("gated", "gated_grad"):
        return _exact_gated(case, state)
    return _exact_distill(case, state)
