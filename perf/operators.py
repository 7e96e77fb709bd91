"""Workloads of the read-out operators: routing of images to neurons, read-out of routed neurons, dense product.

`run` computes them in plain torch operations, or -- with `own` set -- through pink_b200.readout.  `exact` computes the same
from the definitions in 64 bits.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
FLT_MAX = float(torch.finfo(torch.float32).max)


# ---- cases ---------------------------------------------------------------------------------------------------------------

def _route(name, **kw):
    case = dict(op="route", n=1, N=400, type="float32", score="softmax", k=4, renormalise=True, slope=-2.0, scale=1.0,
                bias=False, mask=False, groups=1, top_groups=1, group_best=1, balance=False, scores="", holes=False)
    return {**case, **kw, "name": name}


def _route_grad(name, **kw):
    case = dict(op="route_grad", n=1, N=400, type="float32", score="softmax", k=4, renormalise=True, slope=-2.0, scale=1.0,
                mask=False, dscores=False, holes=False)
    return {**case, **kw, "name": name}


def _read_out(name, **kw):
    return {**dict(op="read_out", n=1, N=400, D=10, k=4, type="float32", residual=False, missing=False), **kw, "name": name}


def _read_out_grad(name, **kw):
    return {**dict(op="read_out_grad", n=1, N=400, D=10, k=4, type="float32", missing=False), **kw, "name": name}


def _product(name, **kw):
    case = dict(op="product", n=1, K=400, M=10, type="bfloat16", by_input=False, bias=True, activation="none", residual=False,
                keep=False, padded=False, x="features")
    return {**case, **kw, "name": name}


def _product_grad(name, **kw):
    case = dict(op="product_grad", n=1, K=400, M=10, type="bfloat16", by_input=False, activation="none", padded=False)
    return {**case, **kw, "name": name}


def listed():
    return [
        # one image against the 2,791-neuron hexagonal map of the headline configuration, as it arrives
        _route("route one image", n=1, N=2791, k=4),
        # a night's images on the 20 x 20 map: rows of the map as groups, a bias that evens out the hits, dense scores kept
        _route("route 20x20 by rows", n=4096, N=400, type="bfloat16", score="sigmoid", slope=1.0, k=8, bias=True, mask=True,
               groups=20, top_groups=5, group_best=2, balance=True, scores="bfloat16", holes=True),
        # a survey's distances to the headline map, resident on the GPU
        _route("route hex 2791", n=65536, N=2791, k=8, bias=True, balance=True),
        # training a read-out with dense and routed weights on the headline map
        _route_grad("route gradient dense", n=16384, N=2791, k=8, renormalise=False, dscores=True),
        # training a learned sigmoid router over the 40 x 40 map
        _route_grad("route gradient sigmoid", n=3001, N=1600, type="float16", score="sigmoid", slope=1.0, k=6, scale=2.5, mask=True,
                    holes=True),
        # one image rebuilt from its four best neurons of 90 x 90 pixels
        _read_out("read out one image", n=1, N=2791, D=8100, k=4),
        # residual images of a batch: prediction from eight neurons on top of what is there
        _read_out("read out images", n=2000, N=2791, D=8100, k=8, type="bfloat16", residual=True),
        # labels (ten classes) of the neurons trained from a survey's labelled images
        _read_out_grad("read out labels gradient", n=65536, N=2791, D=10, k=8, missing=True),
        # prototypes of the 20 x 20 map refined by the gradient of rebuilt images
        _read_out_grad("read out images gradient", n=1024, N=400, D=8100, k=4, type="bfloat16"),
        # dense read-out of one image: all responses times the table of prototypes
        _product("product one image", n=1, K=2791, M=8100, by_input=True, bias=False, x="scores"),
        # a batch of them with a correction network's activation, on rows padded as the dense scores are
        _product("product images", n=8192, K=2791, M=8100, activation="sigmoid", residual=True, keep=True, padded=True, x="scores"),
        # training a hidden layer of as many units as the map has neurons on distance regions of 63 x 63 pixels
        _product_grad("product gradient", n=4096, K=3969, M=2791, type="float16", activation="gelu"),
    ]


def _size(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    op = rng.choice(["route", "route_grad", "read_out", "read_out_grad", "product", "product_grad"])
    flag = lambda p=0.5: rng.random() < p
    if op in ("route", "route_grad"):
        groups, N = 1, _size(rng, 1, 8192)
        n = _size(rng, 1, min(65536, (65536 if op == "route" else 16384) * 2791 // N))
        k = rng.randint(1, min(N, 16))
        score = rng.choice(["softmax", "sigmoid"])
        common = dict(n=n, N=N, k=k, score=score, slope=-2.0 if score == "softmax" else 1.0, type=rng.choice(sorted(TYPES)),
                      renormalise=flag(), scale=rng.choice([1.0, 2.5]), mask=flag(0.3), holes=flag(0.3))
        if op == "route_grad":
            return {k_: v for k_, v in _route_grad("", **common, dscores=flag(0.3)).items() if k_ != "name"}
        top_groups = group_best = 1
        if flag(0.4):
            groups = rng.choice([g for g in range(1, min(N, 64) + 1) if N % g == 0])
            top_groups = rng.randint(-(-k * groups // N), groups)
            group_best = rng.choice([1, 2])
        case = _route("", **common, bias=flag(), groups=groups, top_groups=top_groups, group_best=group_best, balance=flag(0.3),
                      scores=rng.choice(["", "", "float32", "bfloat16"]))
    elif op in ("read_out", "read_out_grad"):
        N, D = _size(rng, 1, 4096), _size(rng, 1, 8192)
        n = _size(rng, 1, min(65536, 16_200_000 // D if op == "read_out" else 8_294_400 // D))
        case = (_read_out if op == "read_out" else _read_out_grad)("", n=n, N=N, D=D, k=rng.randint(1, 12), type=rng.choice(sorted(TYPES)),
                                                                    missing=flag(0.3))
        if op == "read_out":
            case["residual"] = flag()
    else:
        K, M = _size(rng, 1, 4096), _size(rng, 1, 8192)
        n = _size(rng, 1, min(8192, (8192 * 2791 * 8100 if op == "product" else 4096 * 3969 * 2791) // (K * M)))
        common = dict(n=n, K=K, M=M, type=rng.choice(["bfloat16", "float16"]), by_input=flag(), padded=flag(),
                      activation=rng.choice(["none", "relu", "gelu", "silu", "sigmoid"]))
        if op == "product":
            case = _product("", **common, bias=flag(), residual=flag(), keep=flag(0.3), x=rng.choice(["scores", "features"]))
        else:
            case = _product_grad("", **common)
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


def _padded(t, padded):
    """The same matrix; with `padded` in rows of a multiple of eight elements, as dense scores are laid out."""
    if not padded:
        return t.contiguous()
    wide = torch.zeros((t.shape[0], -(-t.shape[1] // 8) * 8), dtype=t.dtype, device=t.device)
    wide[:, :t.shape[1]] = t
    return wide[:, :t.shape[1]]


def _values(g, case):
    """Distances of images to the neurons of a map (softmax), or the scores of a learned router (sigmoid)."""
    n, N = case["n"], case["N"]
    if case["score"] == "softmax":
        at, of = _uniform(g, n, 2), _uniform(g, N, 2)
        v = torch.sqrt(16.0 + 60.0 * ((at[:, None, 0] - of[None, :, 0]) ** 2 + (at[:, None, 1] - of[None, :, 1]) ** 2))
        v += 0.3 * _normal(g, n, N)
    else:
        v = _normal(g, n, N) - 1.0
    if case["holes"]:                                    # neurons without an answer, and images that have none at all
        v[_uniform(g, n, N) < 0.01] = math.nan
        v[_uniform(g, n) < 0.02] = math.inf if case["slope"] < 0 else -math.inf
    return v.to(TYPES[case["type"]])


def _mask(g, case):
    if not case["mask"]:
        return None
    return _uniform(g, case["N"]) > 0.05                 # neurons that no image of the training set reached


def _routes(g, n, N, k, missing):
    """Routes as a map gives them: neurons near the best one, some of which are hit far more often than others."""
    centre = (N * _uniform(g, n, 1) ** 2).long()
    neurons = (centre + torch.arange(k, device="cuda") * 7) % N
    weights = torch.softmax(2.0 * _normal(g, n, k), 1)
    if missing:
        gone = _uniform(g, n, k) < 0.02
        neurons, weights = torch.where(gone, -1, neurons), torch.where(gone, 0.0, weights)
    return neurons.int(), weights


def prepare(case, seed):
    g, op = _generator(seed), case["op"]
    state = {"case": case}
    if op in ("route", "route_grad"):
        state["values"], state["mask"] = _values(g, case), _mask(g, case)
        if op == "route":
            state["bias"] = 0.1 * _normal(g, case["N"]) if case["bias"] or case["balance"] else None
        else:
            full = dict(case, groups=1, top_groups=1, group_best=1)
            state["neurons"], state["weights"], _ = _plain_route(state["values"], None, state["mask"], full)
            state["dweights"] = _normal(g, case["n"], case["k"])
            state["dscores"] = _normal(g, case["n"], case["N"]).to(TYPES[case["type"]]) if case["dscores"] else None
    elif op in ("read_out", "read_out_grad"):
        dtype = TYPES[case["type"]]
        state["values"] = _uniform(g, case["N"], case["D"]).to(dtype)
        state["neurons"], state["weights"] = _routes(g, case["n"], case["N"], case["k"], case["missing"])
        if op == "read_out":
            state["residual"] = _normal(g, case["n"], case["D"]).to(dtype) if case["residual"] else None
        else:
            state["dy"] = _normal(g, case["n"], case["D"]).to(dtype)
    else:
        dtype, n, K, M = TYPES[case["type"]], case["n"], case["K"], case["M"]
        if op == "product" and case["x"] == "scores":
            x, w = torch.softmax(3.0 * _normal(g, n, K), 1), _uniform(g, M, K)
        else:
            x, w = _normal(g, n, K), _normal(g, M, K) / math.sqrt(K)
        state["x"] = _padded(x.to(dtype), case["padded"])
        state["w"] = _padded((w.t() if case["by_input"] else w).to(dtype), case["padded"])
        if op == "product":
            state["bias"] = 0.5 * _normal(g, M) if case["bias"] else None
            state["residual"] = _padded(_normal(g, n, M).to(dtype), case["padded"]) if case["residual"] else None
        else:
            state["z"] = _padded(_normal(g, n, M).to(dtype), case["padded"]) if case["activation"] != "none" else None
            state["dy"] = _padded(_normal(g, n, M).to(dtype), case["padded"])
    return state


# ---- the plain form ------------------------------------------------------------------------------------------------------

def _plain_logits(values, mask, case):
    logits = values.float() * case["slope"]
    part = ~torch.isnan(logits) & (logits != -math.inf)
    if mask is not None:
        part &= mask
    return torch.where(part, logits.clamp(max=FLT_MAX), -math.inf), part


def _plain_softmax(logits):
    """Softmax over the finite entries; rows without any are all zero."""
    most = logits.amax(1, keepdim=True)
    e = torch.exp(logits - torch.where(most == -math.inf, 0.0, most))
    return e / e.sum(1, keepdim=True).clamp(min=1e-30)


def _plain_route(values, bias, mask, case):
    n, N, k, G = case["n"], case["N"], case["k"], case["groups"]
    logits, part = _plain_logits(values, mask, case)
    choice = logits
    if bias is not None:
        choice = logits + bias
        choice = torch.where(part & ~torch.isnan(choice), choice.clamp(max=FLT_MAX), -math.inf)
    if G > 1:
        best = torch.sort(choice.view(n, G, N // G), dim=2, descending=True).values
        value = best[:, :, 0]
        if case["group_best"] == 2 and N // G > 1:
            value = torch.where(best[:, :, 1] == -math.inf, value, value + best[:, :, 1])
        order = torch.sort(value, dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        kept = torch.zeros((n, G), dtype=torch.bool, device=values.device).scatter_(1, order, True)
        choice = torch.where(kept[:, :, None].expand(n, G, N // G).reshape(n, N), choice, -math.inf)
    top = torch.sort(choice, dim=1, descending=True, stable=True)
    there = top.values[:, :k] > -math.inf
    index = top.indices[:, :k]
    scores = None
    chosen = torch.where(there, logits.gather(1, index), -math.inf)
    if case["score"] == "softmax":
        if case["renormalise"]:
            weights = _plain_softmax(chosen)
        if not case["renormalise"] or case.get("scores"):
            scores = _plain_softmax(logits)
    else:
        if case["renormalise"]:                          # relative to the largest, so that small ones do not vanish
            low = torch.clamp(chosen, max=0.0)
            most = low.amax(1, keepdim=True)
            s = torch.exp(low - torch.where(most == -math.inf, 0.0, most)) / (1.0 + torch.exp(-chosen.abs()))
            weights = s / s.sum(1, keepdim=True).clamp(min=1e-30)
        if not case["renormalise"] or case.get("scores"):
            scores = torch.sigmoid(logits)
    if not case["renormalise"]:
        weights = scores.gather(1, index)
    weights = torch.where(there, case["scale"] * weights, 0.0)
    return torch.where(there, index, -1).int(), weights, scores


def _plain_route_grad(values, mask, neurons, weights, dweights, dscores, case):
    logits, part = _plain_logits(values, mask, case)
    there = neurons >= 0
    index = torch.where(there, neurons, 0).long()
    g = torch.where(there, dweights, 0.0)
    dlogits = torch.zeros_like(logits)
    dense = torch.zeros_like(logits) if dscores is None else torch.where(part, dscores.float(), 0.0)
    if case["renormalise"]:
        routed = weights * (g - (g * weights).sum(1, keepdim=True) / case["scale"])
        if case["score"] == "sigmoid":
            routed = routed * torch.sigmoid(-logits.gather(1, index))
        dlogits.scatter_add_(1, index, torch.where(there, routed, 0.0))
    else:
        dense.scatter_add_(1, index, case["scale"] * g)
    if dscores is not None or not case["renormalise"]:
        if case["score"] == "softmax":
            p = _plain_softmax(logits)
            dlogits += p * (dense - (p * dense).sum(1, keepdim=True))
        else:
            dlogits += dense * torch.sigmoid(logits) * torch.sigmoid(-logits)
    return torch.where(part, case["slope"] * dlogits, 0.0).to(values.dtype)


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


def _run_plain(state):
    case, op = state["case"], state["case"]["op"]
    if op == "route":
        neurons, weights, scores = _plain_route(state["values"], state["bias"], state["mask"], case)
        out = {"neurons": neurons, "weights": weights}
        if case["scores"]:
            out["scores"] = scores.to(TYPES[case["scores"]])
        if case["balance"]:
            N = case["N"]
            load = torch.bincount(torch.where(neurons < 0, N, neurons).flatten().long(), minlength=N + 1)[:N]
            takes = torch.ones(N, dtype=torch.bool, device="cuda") if state["mask"] is None else state["mask"]
            out["load"] = load.int()
            step = torch.sign(torch.where(takes, load.sum() - load * takes.sum(), 0)).float()
            out["bias"] = state["bias"] + 0.001 * step
        return out
    if op == "route_grad":
        return {"dvalues": _plain_route_grad(state["values"], state["mask"], state["neurons"], state["weights"], state["dweights"],
                                             state["dscores"], case)}
    if op in ("read_out", "read_out_grad"):
        values, neurons, weights = state["values"], state["neurons"], state["weights"]
        there = neurons >= 0
        index, w = torch.where(there, neurons, 0).long(), torch.where(there, weights, 0.0)
        if op == "read_out":
            y = torch.einsum("nk,nkd->nd", w, values[index].float())
            if state["residual"] is not None:
                y = y + state["residual"].float()
            return {"y": y.to(values.dtype)}
        dy = state["dy"].float()
        dweights = torch.where(there, torch.einsum("nd,nkd->nk", dy, values[index].float()), 0.0)
        dvalues = torch.zeros(values.shape, device="cuda")
        dvalues.index_add_(0, index.flatten(), (w[:, :, None] * dy[:, None, :]).flatten(0, 1))
        return {"dvalues": dvalues.to(values.dtype), "dweights": dweights}
    x, w = state["x"].float(), state["w"].float()
    w = w.t() if case["by_input"] else w
    if op == "product":
        z = x @ w.t()
        if state["bias"] is not None:
            z = z + state["bias"]
        y = _plain_act(z, case["activation"])
        if state["residual"] is not None:
            y = y + state["residual"].float()
        out = {"y": y.to(state["x"].dtype)}
        if case["keep"]:
            out["z"] = z.to(state["x"].dtype)
        return out
    dz = state["dy"].float()
    if case["activation"] != "none":
        dz = dz * _plain_act_slope(state["z"].float(), case["activation"])
    dw = x.t() @ dz if case["by_input"] else dz.t() @ x
    return {"dx": (dz @ w).to(state["x"].dtype), "dw": dw.to(state["w"].dtype), "dbias": dz.sum(0)}


# ---- the framework's calls -----------------------------------------------------------------------------------------------

def _run_own(state):
    from pink_b200 import readout
    case, op = state["case"], state["case"]["op"]
    if op == "route":
        load = torch.zeros(case["N"], dtype=torch.int32, device="cuda") if case["balance"] else None
        out = readout.route(state["values"], case["k"], score=case["score"], slope=case["slope"], scale=case["scale"],
                            renormalise=case["renormalise"], bias=state["bias"], mask=state["mask"], groups=case["groups"],
                            top_groups=case["top_groups"], group_best=case["group_best"], load=load,
                            scores=TYPES[case["scores"]] if case["scores"] else None)
        out = dict(zip(("neurons", "weights", "scores"), out))
        if case["balance"]:
            out["load"] = load
            out["bias"] = readout.balance(load, state["bias"], 0.001, mask=state["mask"])
        return out
    if op == "route_grad":
        return {"dvalues": readout.route_backward(state["values"], state["neurons"], state["weights"], state["dweights"],
                                                  score=case["score"], slope=case["slope"], scale=case["scale"],
                                                  renormalise=case["renormalise"], mask=state["mask"], dscores=state["dscores"])}
    if op == "read_out":
        return {"y": readout.read_out(state["values"], state["neurons"], state["weights"], residual=state["residual"])}
    if op == "read_out_grad":
        dvalues, dweights = readout.read_out_backward(state["dy"], state["values"], state["neurons"], state["weights"])
        return {"dvalues": dvalues, "dweights": dweights}
    if op == "product":
        out = readout.product(state["x"], state["w"], by_input=case["by_input"], bias=state["bias"], activation=case["activation"],
                              residual=state["residual"], keep=case["keep"])
        return dict(zip(("y", "z"), out)) if case["keep"] else {"y": out}
    return dict(zip(("dx", "dw", "dbias"), readout.product_backward(state["dy"], state["x"], state["w"], by_input=case["by_input"],
                                                                    z=state["z"], activation=case["activation"])))


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------

def work(case):
    op, n = case["op"], case["n"]
    size = 4 if case["type"] == "float32" else 2
    if op == "route":
        N, k = case["N"], case["k"]
        dense = n * N * (4 if case["scores"] == "float32" else 2) if case["scores"] else 0
        return {"bytes": n * N * size + dense + n * k * 8 + (4 * N if case["bias"] else 0) + (12 * N if case["balance"] else 0),
                "flops": 4 * n * N}
    if op == "route_grad":
        N, k = case["N"], case["k"]
        reads = n * N * size if case["score"] == "softmax" and not case["renormalise"] or case["dscores"] else n * k * size
        return {"bytes": reads + (n * N * size if case["dscores"] else 0) + n * N * size + n * k * 12, "flops": 4 * n * N}
    if op in ("read_out", "read_out_grad"):
        D, k, rows = case["D"], case["k"], min(case["N"], n * case["k"])
        if op == "read_out":
            return {"bytes": rows * D * size + n * k * 8 + n * D * size * (2 if case["residual"] else 1), "flops": 2 * n * k * D}
        return {"bytes": rows * D * size + case["N"] * D * size + n * D * size + n * k * 12, "flops": 4 * n * k * D}
    K, M = case["K"], case["M"]
    if op == "product":
        return {"bytes": size * (n * K + K * M + n * M * (1 + case["residual"] + case["keep"])), "flops": 2 * n * K * M}
    return {"bytes": size * (2 * n * K + 2 * K * M + n * M * (2 if case["activation"] != "none" else 1)) + 4 * M, "flops": 4 * n * K * M}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------

def _f32(t):
    """Rounded to 32 bits where the definition rounds (the choice of neurons is made on such numbers), held in 64."""
    return t.float().double()


def _exact_logits(values, mask, case):
    l = _f32(values.double() * float(np.float32(case["slope"])))
    takes = (l == l) & (l > -math.inf)
    if mask is not None:
        takes = takes & mask
    return torch.where(takes, torch.clamp(l, max=FLT_MAX), torch.full_like(l, -math.inf)), takes


def _exact_pick(c, count):
    """`count` times the largest of every row, the first of equals; -1 where nothing is left."""
    c, picks = c.clone(), []
    place = torch.arange(c.shape[1], device=c.device)
    for _ in range(count):
        most = c.max(1, keepdim=True).values
        first = torch.where(c == most, place, c.shape[1]).min(1, keepdim=True).values
        picks.append(torch.where(most == -math.inf, -1, first))
        c.scatter_(1, first, -math.inf)
    return torch.cat(picks, 1)


def _exact_shares(l):
    """exp(l) over its sum along rows; zeros where the row has none."""
    return torch.nan_to_num(torch.softmax(l, 1), nan=0.0)


def _exact_route(case, state):
    n, N, G, mask = case["n"], case["N"], case["groups"], state["mask"]
    l, takes = _exact_logits(state["values"], mask, case)
    c = l
    if state["bias"] is not None:
        c = torch.clamp(_f32(l + state["bias"].double()), max=FLT_MAX)
        c = torch.where(takes & (c == c), c, torch.full_like(c, -math.inf))
    if G > 1:
        rows = c.reshape(n * G, N // G)
        pair = _exact_pick(rows, min(2, N // G))
        best = torch.where(pair >= 0, rows.gather(1, pair.clamp(min=0)), torch.full_like(pair, 0, dtype=torch.float64))
        value = _f32(best.sum(1)) if case["group_best"] == 2 else best[:, 0]
        value = torch.where(pair[:, 0] >= 0, value, torch.full_like(value, -math.inf)).reshape(n, G)
        groups = _exact_pick(value, case["top_groups"])
        group_of = torch.arange(N, device=c.device) // (N // G)
        kept = torch.zeros(n, G + 1, dtype=torch.bool, device=c.device)
        kept.scatter_(1, torch.where(groups < 0, G, groups), True)
        c = torch.where(kept[:, group_of], c, torch.full_like(c, -math.inf))
    neurons = _exact_pick(c, case["k"])
    there = neurons >= 0
    chosen = torch.where(there, l.gather(1, neurons.clamp(min=0)), torch.full_like(neurons, 0, dtype=torch.float64) - math.inf)
    softmax = case["score"] == "softmax"
    if case["renormalise"]:
        weights = _exact_shares(chosen if softmax else torch.nn.functional.logsigmoid(chosen))
    else:
        weights = _exact_shares(l).gather(1, neurons.clamp(min=0)) if softmax else torch.sigmoid(chosen)
    out = {"neurons": neurons.int(), "weights": torch.where(there, case["scale"] * weights, torch.zeros_like(weights))}
    if case["scores"]:
        out["scores"] = _exact_shares(l) if softmax else torch.sigmoid(l)
    if case["balance"]:
        hits = torch.zeros(N + 1, dtype=torch.int64, device=c.device)
        hits.scatter_add_(0, torch.where(there, neurons, N).reshape(-1), torch.ones(n * case["k"], dtype=torch.int64, device=c.device))
        hits = hits[:N]
        inside = torch.ones(N, dtype=torch.bool, device=c.device) if mask is None else mask
        more = hits.sum() > hits * inside.sum()
        less = hits.sum() < hits * inside.sum()
        out["load"] = hits.int()
        out["bias"] = state["bias"].double() + 0.001 * (more.double() - less.double()) * inside
    return out


def _exact_route_grad(case, state):
    l, takes = _exact_logits(state["values"], state["mask"], case)
    l = torch.where(takes, l, torch.zeros_like(l))
    l.requires_grad_(True)
    neurons, there = state["neurons"].long().clamp(min=0), state["neurons"] >= 0
    log_p = l if case["score"] == "softmax" else torch.nn.functional.logsigmoid(l)
    log_p = torch.where(takes, log_p, torch.full_like(log_p, -1e300))
    p = torch.softmax(log_p, 1) if case["score"] == "softmax" else torch.exp(log_p)
    if case["renormalise"]:
        w = torch.softmax(torch.where(there, log_p.gather(1, neurons), torch.full_like(neurons, 0, dtype=torch.float64) - 1e300), 1)
    else:
        w = p.gather(1, neurons)
    total = (torch.where(there, case["scale"] * w, torch.zeros_like(w)) * state["dweights"].double()).sum()
    if state["dscores"] is not None:
        total = total + (torch.where(takes, p, torch.zeros_like(p)) * state["dscores"].double()).sum()
    total.backward()
    return {"dvalues": torch.where(takes, float(np.float32(case["slope"])) * l.grad, torch.zeros_like(l.grad))}


def _exact_act(z, activation):
    if activation == "relu":
        return torch.relu(z)
    if activation == "gelu":
        return torch.nn.functional.gelu(z)
    if activation == "silu":
        return torch.nn.functional.silu(z)
    return torch.sigmoid(z) if activation == "sigmoid" else z


def exact(case, seed):
    state, op = prepare(case, seed), case["op"]
    if op == "route":
        return _exact_route(case, state)
    if op == "route_grad":
        return _exact_route_grad(case, state)
    if op in ("read_out", "read_out_grad"):
        V, e = state["values"].double(), state["neurons"].long()
        spread = torch.zeros(case["n"], case["N"] + 1, dtype=torch.float64, device="cuda")   # weights as a matrix over the neurons
        e = torch.where(e < 0, case["N"], e)
        spread.scatter_add_(1, e, state["weights"].double())
        spread = spread[:, :case["N"]]
        if op == "read_out":
            y = spread @ V
            return {"y": y if state["residual"] is None else y + state["residual"].double()}
        dy = state["dy"].double()
        inner = torch.cat([dy @ V.t(), torch.zeros(case["n"], 1, dtype=torch.float64, device="cuda")], 1)
        return {"dvalues": spread.t() @ dy, "dweights": inner.gather(1, e)}
    x, w = state["x"].double(), state["w"].double()
    w = w if case["by_input"] else w.t()                 # [K, M]
    if op == "product":
        z = x @ w
        if state["bias"] is not None:
            z = z + state["bias"].double()
        y = _exact_act(z, case["activation"])
        if state["residual"] is not None:
            y = y + state["residual"].double()
        return {"y": y, "z": z} if case["keep"] else {"y": y}
    dz = state["dy"].double()
    if case["activation"] != "none":
        z = state["z"].double().requires_grad_(True)
        _exact_act(z, case["activation"]).backward(dz)
        dz = z.grad
    dw = x.t() @ dz if case["by_input"] else dz.t() @ x
    return {"dx": dz @ w.t(), "dw": dw, "dbias": dz.sum(0)}
