"""The read-out operators against plain implementations in 64 bits.

Tolerances: u = 2^-24 is the unit roundoff of float32.  A float32 sum of m terms in any order is off by at most m u times the sum of
their magnitudes; expf and the other elementary functions by a few units; a result rounded to type t by half of finfo(t).eps."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
FLT_MAX = float(np.finfo(np.float32).max)
TYPES = ["float32", "bfloat16", "float16"]


@pytest.fixture(scope="module")
def R(cuda):
    from pink_b200 import readout
    yield readout
    readout.check_status()


def half_step(torch, dtype):
    return torch.finfo(dtype).eps / 2


def rand(torch, seed, *shape, dtype="float32", scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(shape, generator=g, device="cuda")).to(getattr(torch, dtype))


def within(got, want, bound):
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    off = (got - want).abs()
    worst = (off - bound).max().item() if off.numel() else 0.0
    assert worst <= 0.0, "worst excess %g, largest error %g" % (worst, off.max().item())


# ---- route ---------------------------------------------------------------------------------------------------------------

def ref_logits(torch, values, mask, slope):
    """The definition, row by row, with numpy's float32 rounding."""
    with np.errstate(over="ignore", invalid="ignore"):
        l = (values.float().cpu().numpy() * np.float32(slope)).astype(np.float32)
    takes = ~np.isnan(l) & (l != -np.inf)
    if mask is not None:
        takes &= mask.cpu().numpy().astype(bool)
    return np.where(takes, np.minimum(l, np.float32(FLT_MAX)), -np.inf), takes


def ref_route(torch, values, k, bias=None, mask=None, groups=1, top_groups=None, group_best=1, slope=1.0, score="softmax", scale=1.0, renormalise=True):
    l, takes = ref_logits(torch, values, mask, slope)
    n, N = l.shape
    top_groups = groups if top_groups is None else top_groups
    c = l.copy()
    if bias is not None:
        with np.errstate(over="ignore", invalid="ignore"):
            c = (l + bias.cpu().numpy()[None]).astype(np.float32)
        c = np.where(takes & ~np.isnan(c), np.minimum(c, np.float32(FLT_MAX)), -np.inf)
    neurons = np.full((n, k), -1, np.int64)
    weights = np.zeros((n, k))
    with np.errstate(over="ignore", under="ignore", divide="ignore", invalid="ignore"):
        l64 = l.astype(np.float64)
        if score == "softmax":
            most = l64.max(1, keepdims=True)
            e = np.exp(l64 - np.where(most == -np.inf, 0.0, most))
            total = e.sum(1, keepdims=True)
            p = np.where(total > 0, e / np.where(total > 0, total, 1), 0.0)
        else:
            p = 1.0 / (1.0 + np.exp(-l64))
    for i in range(n):
        ci = c[i].copy()
        if groups > 1:
            value = []
            for g in range(groups):
                m = np.sort(ci[g * (N // groups):(g + 1) * (N // groups)])[::-1]
                v = m[0]
                if group_best == 2 and len(m) > 1 and m[1] != -np.inf:
                    with np.errstate(over="ignore"):
                        v = np.clip(np.float32(m[0]) + np.float32(m[1]), np.float32(-FLT_MAX), np.float32(FLT_MAX))
                value.append(v)
            order = sorted(range(groups), key=lambda g: (-float(value[g]), g))[:top_groups]
            for g in range(groups):
                if g not in order:
                    ci[g * (N // groups):(g + 1) * (N // groups)] = -np.inf
        order = sorted((j for j in range(N) if ci[j] != -np.inf), key=lambda j: (-float(ci[j]), j))[:k]
        neurons[i, :len(order)] = order
        if order:
            if not renormalise:
                weights[i, :len(order)] = p[i, order]
            else:
                logp = l64[i, order] if score == "softmax" else -np.logaddexp(0.0, -l64[i, order])
                e = np.exp(logp - logp.max())
                weights[i, :len(order)] = e / e.sum()
    return neurons, scale * weights, p


def route_tolerance(l, N):
    """Relative: the rounding of l - max (|l - max| <= range of the finite logits that matter, 104: below it exp is zero in float32) in a
    term and in the sum, four units of each of two exponentials, the sum's depth, and six roundings around them."""
    finite = l[np.isfinite(l)]
    span = min(104.0, float(finite.max()) - float(finite.min())) if finite.size else 0.0
    return U * (2 * span + 8 + N / 32 + 16 + 6)


ROUTE_CASES = [
    # n, N, k, type, options
    (1, 1, 1, "float32", {}),
    (3, 2, 2, "float32", dict(score="sigmoid")),
    (5, 31, 4, "bfloat16", dict(slope=-2.0)),
    (7, 32, 32, "float16", dict(renormalise=False)),
    (9, 33, 32, "float32", dict(bias=True, mask=True)),
    (4, 400, 8, "bfloat16", dict(groups=20, top_groups=5, group_best=2, bias=True, mask=True, holes=True)),
    (4, 400, 8, "float32", dict(groups=20, top_groups=1, group_best=1, score="sigmoid", renormalise=False)),
    (6, 255, 3, "float32", dict(groups=255, top_groups=7, group_best=2, holes=True)),
    (6, 256, 5, "float16", dict(groups=256, top_groups=256, score="sigmoid", bias=True)),
    (3, 1000, 17, "float32", dict(bias=True, holes=True, scale=2.5, renormalise=False)),
    (5, 1023, 1, "float32", dict(slope=-0.5, score="sigmoid")),
    (5, 1024, 9, "bfloat16", dict(holes=True)),
    (5, 1025, 9, "float32", dict(holes=True, groups=5, top_groups=2, group_best=2)),
    (3, 2791, 8, "float32", dict(bias=True, slope=-2.0)),
    (2, 4097, 32, "float16", dict(score="sigmoid", scale=0.5)),
    (2, 8192, 6, "float32", dict(groups=64, top_groups=4, group_best=2, mask=True)),
    (2, 8193, 6, "float32", dict(renormalise=False)),
    (2, 32768, 32, "bfloat16", dict(bias=True, groups=256, top_groups=3, group_best=2)),
]


def make_values(torch, seed, n, N, dtype, holes):
    v = rand(torch, seed, n, N, scale=3.0)
    if holes:
        r = torch.rand((n, N), generator=torch.Generator(device="cuda").manual_seed(seed + 1), device="cuda")
        v[r < 0.05] = float("nan")
        v[(r > 0.05) & (r < 0.1)] = float("inf")
        v[(r > 0.1) & (r < 0.15)] = -float("inf")
        v[(r > 0.15) & (r < 0.2)] = 0.0
        v[(r > 0.2) & (r < 0.25)] = -0.0
        v[0] = float("nan")
        if n > 1:
            v[1] = -float("inf")
        if n > 2:
            v[2] = torch.finfo(v.dtype).min
    return v.to(getattr(torch, dtype))


@pytest.mark.parametrize("case", ROUTE_CASES, ids=lambda c: "%dx%d-%d-%s" % c[:4])
@pytest.mark.parametrize("pitch", [0, 3])
def test_route_follows_the_definition(R, cuda, case, pitch):
    torch = cuda
    n, N, k, dtype, o = case
    o = dict(o)
    v = make_values(torch, 11 + N, n, N, dtype, o.pop("holes", False))
    if pitch:                                              # rows at an odd pitch and offset
        wide = torch.full((n, N + pitch + 1), float("nan"), device="cuda", dtype=v.dtype)
        wide[:, 1:N + 1] = v
        v = wide[:, 1:N + 1]
    bias = rand(torch, 5, N) if o.pop("bias", False) else None
    mask = (torch.arange(N, device="cuda") % 7 != 3) if o.pop("mask", False) else None
    load = torch.full((N,), 10, dtype=torch.int32, device="cuda")
    neurons, weights, scores = R.route(v, k, bias=bias, mask=mask, load=load, scores=torch.float32, **o)
    wn, ww, wp = ref_route(torch, v, k, bias, mask, **o)
    assert np.array_equal(neurons.cpu().numpy(), wn)
    assert np.array_equal(load.cpu().numpy(), 10 + np.bincount(wn[wn >= 0], minlength=N))
    l, _ = ref_logits(torch, v, mask, o.get("slope", 1.0))
    tol = route_tolerance(l, N)
    for got, want in ((weights, ww), (scores, wp)):
        got = got.double().cpu().numpy()
        assert np.all(np.abs(got - want) <= tol * want + 2.0 ** -140), np.abs(got - want).max()
    again = R.route(v, k, bias=bias, mask=mask, **o)
    assert torch.equal(again[0], neurons) and torch.equal(again[1], weights)


def test_route_of_equal_values_takes_the_first_neurons(R, cuda):
    torch = cuda
    for N in (5, 40, 700, 3000, 9000):
        v = torch.zeros(3, N, device="cuda")
        v[1] = -0.0
        v[2, ::2] = -0.0                                   # both zeros are equal
        k = min(N, 32)
        neurons, weights = R.route(v, k, slope=-1.0)
        assert torch.equal(neurons.long(), torch.arange(k, device="cuda").expand(3, k))
        assert (weights - 1.0 / k).abs().max().item() <= 4 * U
        neurons, _ = R.route(v, 3, groups=5, top_groups=3, group_best=2)
        assert torch.equal(neurons.long(), torch.arange(3, device="cuda").expand(3, 3) if N > 5 else neurons.long())


def test_route_with_extreme_logits(R, cuda):
    torch = cuda
    v = torch.tensor([[FLT_MAX, FLT_MAX, 1.0, -FLT_MAX], [float("inf"), 0.0, float("inf"), -float("inf")], [-FLT_MAX] * 4,
                      [-1000.0, -1001.0, -2000.0, -1000.0], [1000.0, 999.0, 998.0, 0.0]], device="cuda")
    for score in ("softmax", "sigmoid"):
        neurons, weights = R.route(v, 3, score=score)
        wn, ww, _ = ref_route(torch, v, 3, score=score)
        assert np.array_equal(neurons.cpu().numpy(), wn)
        assert torch.isfinite(weights).all()
        assert np.abs(weights.double().cpu().numpy() - ww).max() <= 300 * U
    # a slope that takes finite values out of range
    neurons, _ = R.route(torch.tensor([[1e30, -1e30, 2e30]], device="cuda"), 3, slope=1e30)
    assert neurons.tolist() == [[0, 2, -1]]


def test_route_with_bias_beyond_range(R, cuda):
    torch = cuda
    v = torch.zeros(2, 6, device="cuda")
    bias = torch.tensor([0.0, float("nan"), -float("inf"), float("inf"), 1.0, FLT_MAX], device="cuda")
    neurons, weights, scores = R.route(v, 6, bias=bias, scores=torch.float32)
    assert neurons.tolist() == [[3, 5, 4, 0, -1, -1]] * 2
    assert (weights[:, :4] - 0.25).abs().max().item() <= 4 * U and (scores - 1 / 6).abs().max().item() <= 4 * U


@pytest.mark.parametrize("N", [40, 700, 2791, 5000])
def test_route_of_infinite_values_under_a_bias(R, cuda, N):
    """+infinity counts as the largest float before the bias: a bias of that size still orders such neurons."""
    torch = cuda
    v = rand(torch, 3, 6, N)
    v[0, ::3] = float("inf")
    v[1, 5], v[2, 7], v[2, 8] = float("inf"), float("inf"), FLT_MAX
    v[3] = float("inf")
    v[4, 1] = -float("inf")
    bias = 0.1 * rand(torch, 4, N)
    bias[3], bias[5], bias[6], bias[7], bias[9], bias[12] = -FLT_MAX, -1e38, float("inf"), -float("inf"), float("nan"), -2e38
    neurons, _ = R.route(v, 32, bias=bias)
    want, _, _ = ref_route(torch, v, 32, bias)
    assert np.array_equal(neurons.cpu().numpy(), want)


def test_route_without_rows_and_without_neurons(R, cuda):
    torch = cuda
    neurons, weights = R.route(torch.empty(0, 7, device="cuda"), 3)
    assert neurons.shape == (0, 3) and weights.shape == (0, 3)
    neurons, weights, scores = R.route(torch.randn(5, 40, device="cuda"), 3, mask=torch.zeros(40, dtype=torch.bool, device="cuda"), scores=torch.bfloat16)
    assert (neurons == -1).all() and (weights == 0).all() and (scores == 0).all()


def test_route_writes_only_its_rows(R, cuda):
    """Dense scores in a wide matrix: the padding and the rows behind the last stay."""
    torch = cuda
    from pink_b200 import capi
    n, N = 5, 37
    v = rand(torch, 3, n, N)
    out = torch.full((n + 2, 48), 7.0, dtype=torch.bfloat16, device="cuda")
    neurons = torch.full((n + 2, 4), 9, dtype=torch.int32, device="cuda")
    weights = torch.full((n + 2, 4), 9.0, device="cuda")
    cfg = capi.RouteConfig(N, 4, capi.SCORE_SIGMOID, 0, 1, 1, 1, 1.0, 1.0)
    capi.check(capi.lib.pink_b200_op_route(C.byref(cfg), n, capi.F32, v.data_ptr(), N, None, None, neurons.data_ptr(), weights.data_ptr(), None,
                                           capi.BF16, out.data_ptr(), 48, torch.cuda.current_stream().cuda_stream))
    assert (out[n:] == 7).all() and (out[:, N:] == 7).all() and (out[:n, :N] < 2).all()
    assert (neurons[n:] == 9).all() and (weights[n:] == 9).all()


def test_balance(R, cuda):
    torch = cuda
    for N, masked in ((1, False), (7, True), (2791, True), (32768, False)):
        load = torch.randint(0, 2 ** 31 - 1 if N > 7 else 4, (N,), dtype=torch.int32, device="cuda", generator=torch.Generator(device="cuda").manual_seed(N))
        mask = torch.arange(N, device="cuda") % 3 != 1 if masked else torch.ones(N, dtype=torch.bool, device="cuda")
        bias = rand(torch, N, N)
        got = R.balance(load, bias, 0.01, mask=mask)
        l = [int(x) for x in load.tolist()]
        m = mask.tolist()
        total, members = sum(a for a, b in zip(l, m) if b), sum(m)
        step = np.array([np.sign(total - members * a) if b else 0 for a, b in zip(l, m)], np.float32)
        want = (bias.cpu().numpy() + np.float32(0.01) * step).astype(np.float32)
        assert np.array_equal(got.cpu().numpy(), want)
        R.balance(load, bias, 0.01, mask=mask, out=bias)
        assert torch.equal(bias, got)


# ---- gradient of a route -------------------------------------------------------------------------------------------------

def ref_route_grad(torch, values, neurons, weights, dweights, score, slope, scale, renormalise, mask, dscores):
    """The formulas in 64 bits, with a bound of the float32 error (before the last rounding) beside every element."""
    l, takes = ref_logits(torch, values, mask, slope)
    n, N = l.shape
    tol = route_tolerance(l, N)
    l = l.astype(np.float64)
    neurons, w, g = neurons.cpu().numpy(), weights.double().cpu().numpy(), dweights.double().cpu().numpy()
    there = (neurons >= 0) & (neurons < N)
    G = np.zeros((n, N)) if dscores is None else np.where(takes, dscores.double().cpu().numpy(), 0.0)
    dl, bound = np.zeros((n, N)), np.zeros((n, N))
    with np.errstate(over="ignore", under="ignore", invalid="ignore"):
        sig, gis = 1 / (1 + np.exp(-l)), 1 / (1 + np.exp(l))
    for i in range(n):
        idx = neurons[i][there[i]]
        gi, wi = g[i][there[i]], w[i][there[i]]
        if renormalise:
            mean, size = (gi * wi).sum() / scale, np.abs(gi * wi).sum() / scale
            f = gis[i][idx] if score == "sigmoid" else 1.0
            np.add.at(dl[i], idx, wi * (gi - mean) * f)
            np.add.at(bound[i], idx, wi * f * (np.abs(gi) + size) * 60 * U)     # sum of up to 32 terms, products, a sigmoid
        else:
            np.add.at(G[i], idx, scale * gi)
    if not renormalise or dscores is not None:
        with np.errstate(over="ignore", under="ignore", invalid="ignore", divide="ignore"):
            if score == "softmax":
                most = l.max(1, keepdims=True)
                e = np.exp(l - np.where(most == -np.inf, 0.0, most))
                p = e / np.maximum(e.sum(1, keepdims=True), 1e-300)
                mean, size = (p * G).sum(1, keepdims=True), (p * np.abs(G)).sum(1, keepdims=True)
                dl += p * (G - mean)
                bound += p * (2 * (np.abs(G) + size) * tol + 8 * U * (np.abs(G) + size))
            else:
                dl += G * sig * gis
                bound += np.abs(G) * sig * gis * 40 * U
    dl, bound = np.where(takes, slope * dl, 0.0), np.where(takes, abs(slope) * bound, 0.0)
    return torch.from_numpy(dl).cuda(), torch.from_numpy(bound).cuda()


GRAD_CASES = [
    (1, 1, 1, "float32", {}), (3, 33, 5, "float32", dict(renormalise=False)), (4, 400, 8, "bfloat16", dict(score="sigmoid", holes=True, mask=True)),
    (5, 255, 32, "float16", dict(renormalise=False, dscores=True, holes=True)), (3, 1000, 6, "float32", dict(score="sigmoid", renormalise=False, scale=2.5)),
    (3, 1025, 6, "float32", dict(dscores=True, mask=True, slope=-2.0)), (2, 2791, 8, "float32", dict(renormalise=False, dscores=True, slope=-2.0)),
    (2, 1600, 4, "float16", dict(score="sigmoid", dscores=True, scale=0.5)), (2, 4099, 4, "bfloat16", dict(renormalise=False)),
    (3, 2791, 8, "bfloat16", dict(holes=True)), (2, 9001, 4, "float16", dict(mask=True, score="sigmoid")), (70, 31, 3, "float32", dict(mask=True)),
    (9, 513, 32, "float16", dict(slope=-0.5)), (2, 9000, 7, "float32", dict(renormalise=False, dscores=True, holes=True)), (2, 32768, 3, "float32", dict(score="sigmoid", dscores=True)),
]


@pytest.mark.parametrize("case", GRAD_CASES, ids=lambda c: "%dx%d-%d-%s" % c[:4])
@pytest.mark.parametrize("pitch", [0, 3])
def test_route_gradient_follows_the_formulas(R, cuda, case, pitch):
    torch = cuda
    n, N, k, dtype, o = case
    o = dict(o)
    v = make_values(torch, 31 + N, n, N, dtype, o.pop("holes", False))
    mask = (torch.arange(N, device="cuda") % 7 != 3) if o.pop("mask", False) else None
    neurons, weights = R.route(v, k, mask=mask, **{q: o[q] for q in o if q != "dscores"})
    g = rand(torch, 8, n, k)
    ds = rand(torch, 9, n, N, dtype=dtype) if o.pop("dscores", False) else None
    if ds is not None:
        ds[0, 0] = float("nan") if torch.isnan(v[0, 0]) else ds[0, 0]      # a masked place's gradient is not looked at
    g[neurons < 0] = float("nan")                          # nor is an absent route's
    if k > 1:
        neurons[0, 1] = neurons[0, 0]                      # the same neuron twice
    if pitch:
        wide = torch.zeros((n, N + pitch), device="cuda", dtype=v.dtype)
        wide[:, :N] = v
        v = wide[:, :N]
    args = dict(score="softmax", slope=1.0, scale=1.0, renormalise=True)
    args.update(o)
    got = R.route_backward(v, neurons, weights, g, mask=mask, dscores=ds, **args)
    want, bound = ref_route_grad(torch, v, neurons, weights, torch.nan_to_num(g), args["score"], args["slope"], args["scale"], args["renormalise"], mask,
                                 None if ds is None else torch.nan_to_num(ds))
    half = half_step(torch, got.dtype)
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps    # below it a result rounds by a fixed step
    within(got, want, bound * (1 + half) + half * want.abs() + tiny)


@pytest.mark.parametrize("score,renormalise", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_route_gradient_against_differences(R, cuda, score, renormalise):
    """Central differences of sum(weights * g) along the values, from the 64-bit definition: with step h they are off by h^2 / 6 times a
    third derivative (at most 6 scale |g| here, all of whose factors are probabilities) and by the 64-bit rounding / h."""
    torch = cuda
    v, g, h = rand(torch, 1, 2, 9), rand(torch, 2, 2, 3), 1e-4
    o = dict(score=score, renormalise=renormalise, slope=-1.5, scale=2.0)
    neurons, weights = R.route(v, 3, **o)
    got = R.route_backward(v, neurons, weights, g, **o).double().cpu().numpy()
    l = v.double().cpu().numpy() * -1.5
    idx, gg = neurons.cpu().numpy(), g.double().cpu().numpy()

    def total(x, i):
        p = np.exp(x) / np.exp(x).sum() if score == "softmax" else 1 / (1 + np.exp(-x))
        w = p[idx[i]]
        return (2.0 * (w / w.sum() if renormalise else w) * gg[i]).sum()
    for i in range(2):
        for j in range(9):
            a, b = l[i].copy(), l[i].copy()
            a[j] += 1.5 * h
            b[j] -= 1.5 * h
            want = -(total(a, i) - total(b, i)) / (2 * h)
            assert abs(got[i, j] - want) <= 200 * U * (1 + np.abs(gg[i]).sum()) + 36 * h * h * np.abs(gg[i]).sum() + 1e-11


# ---- read-out of routed neurons ------------------------------------------------------------------------------------------

READ_OUT_CASES = [(1, 1, 1, 1), (3, 4, 2, 1), (1, 50, 10, 3), (7, 50, 31, 32), (33, 400, 10, 8), (5, 17, 33, 4), (64, 9, 64, 5), (3, 100, 1000, 4), (2, 20, 8100, 8),
                  (9, 30, 2049, 2), (300, 3, 12, 4), (1000, 7, 3, 8), (3000, 50, 10, 4), (1200, 5000, 6, 8),
                  (100, 4096, 40, 5), (100, 4097, 40, 5), (2048, 301, 65, 4), (2049, 301, 65, 4)]


def make_routes(torch, seed, n, N, k):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    neurons = torch.randint(0, N, (n, k), generator=gen, device="cuda", dtype=torch.int32)      # with the same neuron twice
    neurons[torch.rand((n, k), generator=gen, device="cuda") < 0.1] = -1
    if n > 2:
        neurons[1] = -1                                    # an image without routes
        neurons[2, 0] = N                                  # beyond the table
    return neurons, torch.randn((n, k), generator=gen, device="cuda")


def spread(torch, neurons, weights, N):
    """Routes as a matrix over the neurons, and the same of their magnitudes, in 64 bits."""
    n, k = neurons.shape
    ok = (neurons >= 0) & (neurons < N)
    S, A = torch.zeros(n, N, dtype=torch.float64, device="cuda"), torch.zeros(n, N, dtype=torch.float64, device="cuda")
    for j in range(k):
        e = torch.where(ok[:, j], neurons[:, j], 0).long()[:, None]
        w = torch.where(ok[:, j], weights[:, j].double(), 0.0)[:, None]
        S.scatter_add_(1, e, w)
        A.scatter_add_(1, e, w.abs())
    return S, A, ok


def pitched(torch, t, extra, offset=0):
    wide = torch.full((t.shape[0], t.shape[1] + extra + offset), float("nan"), dtype=t.dtype, device="cuda")
    wide[:, offset:offset + t.shape[1]] = t
    return wide[:, offset:offset + t.shape[1]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", READ_OUT_CASES, ids=lambda c: "%d-%d-%d-%d" % c)
def test_read_out_and_its_gradients(R, cuda, case, dtype):
    torch = cuda
    n, N, D, k = case
    V, r = rand(torch, 1, N, D, dtype=dtype), rand(torch, 2, n, D, dtype=dtype)
    neurons, weights = make_routes(torch, 3, n, N, k)
    S, A, ok = spread(torch, neurons, weights, N)
    half, tiny = half_step(torch, V.dtype), torch.finfo(V.dtype).smallest_normal * torch.finfo(V.dtype).eps
    want, size = S @ V.double(), A @ V.double().abs()
    for extra, offset in ((0, 0), (5, 1), (8, 0)):         # aligned and odd pitches
        Vp, rp = pitched(torch, V, extra, offset), pitched(torch, r, extra, offset)
        y = R.read_out(Vp, neurons, weights)
        within(y, want, size * (k + 1) * U * (1 + half) + half * want.abs() + tiny)
        y = R.read_out(Vp, neurons, weights, residual=rp)
        w2 = want + r.double()
        within(y, w2, (size + r.double().abs()) * (k + 2) * U * (1 + half) + half * w2.abs() + tiny)
        dv, dw = R.read_out_backward(rp, Vp, neurons, weights)
        inner, isize = r.double() @ V.double().t(), r.double().abs() @ V.double().abs().t()
        e = torch.where(ok, neurons, 0).long()
        within(dw, torch.where(ok, inner.gather(1, e), 0.0), isize.gather(1, e) * (D + 1) * U)
        wv, vsize = S.t() @ r.double(), A.t() @ r.double().abs()
        within(dv, wv, vsize * (n * k + 1) * U * (1 + half) + half * wv.abs() + tiny)
        again = R.read_out_backward(rp, Vp, neurons, weights)
        assert torch.equal(dv, again[0]) and torch.equal(dw, again[1])


def test_read_out_gradient_of_a_popular_neuron(R, cuda):
    """All images at one neuron: its routes are split over many blocks; the other rows are zero."""
    torch = cuda
    n, N, D, k = 5000, 40, 37, 2
    dy = rand(torch, 4, n, D)
    neurons = torch.full((n, k), 13, dtype=torch.int32, device="cuda")
    neurons[:, 1] = torch.arange(n, device="cuda") % 3
    weights = rand(torch, 5, n, k)
    dv, _ = R.read_out_backward(dy, torch.zeros(N, D, device="cuda"), neurons, weights)
    S, A, _ = spread(torch, neurons, weights, N)
    within(dv, S.t() @ dy.double(), (A.t() @ dy.double().abs()) * (n * k) * U)
    assert (dv[14:] == 0).all()


@pytest.mark.parametrize("D", [4, 200])
def test_read_out_gradient_of_millions_of_routes(R, cuda, D):
    """More routes than 256 chunks of the sort hold, nearly all at three neurons: with ones everywhere the gradients are counts, which
    float32 holds exactly (below 2^24)."""
    torch = cuda
    n, N, k = 1_100_000, 37, 16
    neurons = (torch.arange(n * k, dtype=torch.int32, device="cuda") * 7 % 5).view(n, k)          # 3 and 4 stand for others below
    neurons = torch.where(neurons == 3, 36, torch.where(neurons == 4, -1, neurons)).contiguous()
    neurons[5, 2], neurons[n - 1, k - 1] = 17, 18
    V = torch.arange(N, device="cuda", dtype=torch.float32)[:, None].expand(N, D).contiguous()
    dv, dw = R.read_out_backward(torch.ones(n, D, device="cuda"), V, neurons, torch.ones(n, k, device="cuda"))
    counts = torch.bincount(neurons.flatten().clamp(min=-1).long() + 1, minlength=N + 1)[1:]
    assert counts.max() < 2 ** 24 and (counts > 0).sum() == 6
    assert torch.equal(dv, counts.float()[:, None].expand(N, D))
    assert torch.equal(dw, torch.where(neurons < 0, 0, neurons * D).float())


def test_read_out_in_place_and_without_rows(R, cuda):
    torch = cuda
    V, r = rand(torch, 1, 20, 33), rand(torch, 2, 9, 33)
    neurons, weights = make_routes(torch, 3, 9, 20, 4)
    want = R.read_out(V, neurons, weights, residual=r)
    got = R.read_out(V, neurons, weights, residual=r, out=r)
    assert got is r and torch.equal(want, r)
    none = torch.empty(0, 4, dtype=torch.int32, device="cuda")
    assert R.read_out(V, none, none.float()).shape == (0, 33)
    dv, dw = R.read_out_backward(torch.empty(0, 33, device="cuda"), V, none, none.float())
    assert (dv == 0).all() and dw.shape == (0, 4)


def test_read_out_of_a_table_beyond_32_bits(R, cuda):
    """Element offsets above 2^32 in the table and in the output pitch."""
    torch = cuda
    N, D = 530_000, 8192
    V = torch.empty(N, D, dtype=torch.bfloat16, device="cuda")
    rows = [0, 262_143, 262_144, 524_287, 524_288, N - 1]
    for i, e in enumerate(rows):
        V[e] = float(i + 1)
    neurons = torch.tensor([rows], dtype=torch.int32, device="cuda")
    y = R.read_out(V, neurons, torch.ones(1, len(rows), device="cuda"))
    assert (y == 21).all()


# ---- dense product -------------------------------------------------------------------------------------------------------

ACTS = ["none", "relu", "gelu", "silu", "sigmoid"]


def ref_act(torch, z, act):
    """Activation, its slope and a bound of the slope, in 64 bits."""
    s = torch.sigmoid(z)
    cdf, pdf = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)), torch.exp(-0.5 * z * z) * (2 * np.pi) ** -0.5
    return {"none": (z, torch.ones_like(z)), "relu": (z.clamp(min=0), (z > 0).double()), "gelu": (z * cdf, cdf + z * pdf),
            "silu": (z * s, s * (1 + z * (1 - s))), "sigmoid": (s, s * (1 - s))}[act]


def check_product(R, torch, n, K, M, dtype, by_input, act, bias, residual, extra=0, offset=0, seed=0):
    x, w = rand(torch, seed + 1, n, K, dtype=dtype), rand(torch, seed + 2, M, K, dtype=dtype, scale=K ** -0.5)
    b = rand(torch, seed + 3, M) if bias else None
    r = rand(torch, seed + 4, n, M, dtype=dtype) if residual else None
    wl = w.t().contiguous() if by_input else w
    P = lambda t: None if t is None else pitched(torch, t, extra, offset)
    y, z = R.product(P(x), P(wl), by_input=by_input, bias=b, activation=act, residual=P(r), keep=True)
    half, tiny = half_step(torch, x.dtype), torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    zw = x.double() @ w.double().t()
    # products of 16-bit numbers are exact in float32; the tensor core may cut rather than round its sums: 2 u a term
    ez = (x.double().abs() @ w.double().abs().t()) * (K + 2) * 2 * U
    if b is not None:
        zw = zw + b.double()
        ez = ez + U * zw.abs()
    within(z, zw, ez * (1 + half) + half * zw.abs() + tiny)
    a, _ = ref_act(torch, zw, act)
    ey = 1.13 * ez + 16 * U * (a.abs() + 1e-30)            # no activation here is steeper than 1.13
    if r is not None:
        a = a + r.double()
        ey = ey + U * a.abs()
    within(y, a, ey * (1 + half) + half * a.abs() + tiny)
    # the bound above grows with K; a lost slice or element would show here: rounding alone moves the norm by less than half
    off = (z.double() - zw).norm() / zw.norm().clamp(min=1e-30)
    assert off <= half + 1e-5
    only = R.product(P(x), P(wl), by_input=by_input, bias=b, activation=act, residual=P(r))
    assert torch.equal(only, y)


PRODUCT_SIZES = [(1, 1, 1), (1, 400, 10), (2, 33, 7), (3, 64, 129), (5, 130, 64), (8, 2791, 33), (9, 1, 1), (9, 400, 10), (16, 63, 17), (64, 64, 64), (65, 65, 65), (127, 200, 300),
                 (128, 128, 256), (129, 72, 257), (300, 961, 40), (500, 2791, 10), (1000, 16, 1000), (40, 5000, 24), (257, 321, 513), (4100, 40, 24)]


@pytest.mark.parametrize("size", PRODUCT_SIZES, ids=lambda s: "%d-%d-%d" % s)
@pytest.mark.parametrize("by_input", [False, True])
def test_product_sizes(R, cuda, size, by_input):
    n, K, M = size
    i = n + K + M
    check_product(R, cuda, n, K, M, "bfloat16" if i % 2 else "float16", by_input, ACTS[i % 5], i % 3 != 0, i % 4 < 2)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("pitch", [(0, 0), (8, 0), (3, 1), (4, 0), (4, 4)], ids=str)
def test_product_types_activations_and_pitches(R, cuda, dtype, act, pitch):
    for n, by_input in ((3, True), (3, False), (70, True), (70, False)):
        check_product(R, cuda, n, 100, 44, dtype, by_input, act, True, True, *pitch)


def check_product_backward(R, torch, n, K, M, dtype, by_input, act, extra=0, offset=0, seed=0):
    x, w = rand(torch, seed + 1, n, K, dtype=dtype), rand(torch, seed + 2, M, K, dtype=dtype, scale=K ** -0.5)
    z, dy = rand(torch, seed + 5, n, M, dtype=dtype), rand(torch, seed + 6, n, M, dtype=dtype)
    wl = w.t().contiguous() if by_input else w
    P = lambda t: pitched(torch, t, extra, offset)
    dx, dw, db = R.product_backward(P(dy), P(x), P(wl), by_input=by_input, z=P(z) if act != "none" else None, activation=act)
    half, tiny = half_step(torch, x.dtype), torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    _, slope = ref_act(torch, z.double(), act)
    dz = dy.double() * slope
    edz = 20 * U * dy.double().abs() if act != "none" else torch.zeros_like(dz)       # the slope's terms are at most 1.2
    round_dz = (half * dz.abs() + tiny if act != "none" else 0.0) + edz               # dz enters the products rounded
    if by_input:
        dw = dw.t()
    for got, want, size, err, terms in ((dx, dz @ w.double(), dz.abs() @ w.double().abs(), round_dz @ w.double().abs() if act != "none" else 0.0, M),
                                        (dw, dz.t() @ x.double(), dz.abs().t() @ x.double().abs(), round_dz.t() @ x.double().abs() if act != "none" else 0.0, n)):
        within(got, want, (size * (terms + 2) * 2 * U + err) * (1 + half) + half * want.abs() + tiny)
        off = (got.double() - want).norm() / want.norm().clamp(min=1e-30)
        assert off <= 2 * half + 1e-5                      # one rounding of dz, one of the result
    within(db, dz.sum(0), (dz.abs().sum(0)) * (n + 1) * U + edz.sum(0))


BACKWARD_SIZES = [(1, 1, 1), (1, 400, 10), (3, 10, 70), (9, 65, 33), (64, 64, 64), (129, 72, 257), (300, 961, 40), (1000, 100, 10), (2000, 33, 129), (257, 321, 513), (5000, 24, 16)]


@pytest.mark.parametrize("size", BACKWARD_SIZES, ids=lambda s: "%d-%d-%d" % s)
@pytest.mark.parametrize("by_input", [False, True])
def test_product_gradients(R, cuda, size, by_input):
    n, K, M = size
    i = n + K + M
    check_product_backward(R, cuda, n, K, M, "bfloat16" if i % 2 else "float16", by_input, ACTS[i % 5])


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("pitch", [(0, 0), (8, 0), (3, 1), (4, 4)], ids=str)
def test_product_gradient_activations_and_pitches(R, cuda, act, pitch):
    for by_input in (False, True):
        check_product_backward(R, cuda, 150, 88, 40, "float16", by_input, act, *pitch)


def test_product_gradient_against_differences(R, cuda):
    """Directional differences of sum(y * dy) along a bias step h = 1e-3 in 64 bits: off by h^2 / 6 of a third derivative below 2."""
    torch = cuda
    n, K, M = 12, 16, 8
    x, w, b, dy = rand(torch, 1, n, K, dtype="float16"), rand(torch, 2, M, K, dtype="float16", scale=0.25), rand(torch, 3, M), rand(torch, 4, n, M, dtype="float16")
    for act in ("gelu", "silu", "sigmoid"):
        _, z = R.product(x, w, bias=b, activation=act, keep=True)
        _, _, db = R.product_backward(dy, x, w, z=z, activation=act)
        f = lambda h: (ref_act(torch, z.double() + h, act)[0] * dy.double()).sum(0)
        want = (f(1e-3) - f(-1e-3)) / 2e-3
        within(db, want, dy.double().abs().sum(0) * (1e-6 + 20 * U))


def test_product_in_place_without_rows_and_beyond_its_matrix(R, cuda):
    torch = cuda
    for n in (4, 40):
        x, w, r = rand(torch, 1, n, 64, dtype="bfloat16"), rand(torch, 2, 48, 64, dtype="bfloat16"), rand(torch, 3, n, 48, dtype="bfloat16")
        want = R.product(x, w, residual=r)
        R.product(x, w, residual=r, out=r)
        assert torch.equal(want, r)
        big = torch.full((n + 3, 64), 5.0, dtype=torch.bfloat16, device="cuda")
        R.product(x, w, out=big[:n, 8:56])
        assert (big[n:] == 5).all() and (big[:, :8] == 5).all() and (big[:, 56:] == 5).all()
        assert torch.equal(big[:n, 8:56], R.product(x, w))
    w = rand(torch, 2, 48, 64, dtype="bfloat16")
    none = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    assert R.product(none, w).shape == (0, 48)
    dx, dw, db = R.product_backward(none[:, :48], none, w)
    assert dx.shape == (0, 64) and (dw == 0).all() and (db == 0).all()


def test_product_keeps_infinities_and_nan_in_their_rows(R, cuda):
    torch = cuda
    for n in (5, 50):
        x, w = rand(torch, 1, n, 40, dtype="bfloat16"), rand(torch, 2, 24, 40, dtype="bfloat16")
        x[1, 3], x[2, 5] = float("nan"), float("inf")
        for act in ("none", "relu"):
            y = R.product(x, w, activation=act)
            assert torch.isnan(y[1]).all() and not torch.isfinite(y[2]).all()
            assert torch.isfinite(y[0]).all() and torch.isfinite(y[3:]).all()


def test_offsets_beyond_32_bits(R, cuda):
    """More than 2^32 elements of values, and of a product's result: the rows behind are as the same rows alone."""
    torch = cuda
    n, N = 1_600_000, 2791
    v = torch.empty(n, N, device="cuda", dtype=torch.bfloat16)
    v[-3:] = rand(torch, 1, 3, N, dtype="bfloat16")
    v[:-3] = 0.0
    neurons, weights = R.route(v, 4)
    want = R.route(v[-3:].clone(), 4)
    assert torch.equal(neurons[-3:], want[0]) and torch.equal(weights[-3:], want[1])
    assert torch.equal(neurons[0].cpu(), torch.arange(4, dtype=torch.int32))
    del v, neurons, weights
    n, K, M = 530_000, 16, 8192
    x, w = torch.zeros(n, K, device="cuda", dtype=torch.bfloat16), rand(torch, 2, M, K, dtype="bfloat16")
    x[-3:] = rand(torch, 3, 3, K, dtype="bfloat16")
    x[262_144] = 1.0
    y = R.product(x, w)
    exact = x[-3:].double() @ w.double().t()
    size = x[-3:].double().abs() @ w.double().abs().t()
    half = half_step(torch, torch.bfloat16)
    within(y[-3:], exact, size * (K + 2) * 2 * U * (1 + half) + half * exact.abs() + 2.0 ** -133)
    one = w.double().sum(1)
    within(y[262_144], one, w.double().abs().sum(1) * (K + 2) * 2 * U * (1 + half) + half * one.abs() + 2.0 ** -133)
    assert (y[1000] == 0).all() and (y[262_143] == 0).all()


def test_front_end_between_streams_keeps_its_scratch(R, cuda):
    """Scratch memory freed by the front end right after a call is not reused before the call is done: many calls in a row, one stream."""
    torch = cuda
    V, dy = rand(torch, 1, 50, 300), rand(torch, 2, 2000, 300)
    neurons, weights = make_routes(torch, 3, 2000, 50, 4)
    want = R.read_out_backward(dy, V, neurons, weights)
    got = [R.read_out_backward(dy, V, neurons, weights) for _ in range(20)]
    assert all(torch.equal(a, want[0]) and torch.equal(b, want[1]) for a, b in got)


def test_gradients_asked_for_one_by_one(R, cuda):
    """Each gradient may be left out (NULL): the others are the same bits, the routes' weights the same sums in another order."""
    torch = cuda
    from pink_b200 import capi
    st = torch.cuda.current_stream().cuda_stream
    for n, N, D, k in ((60, 20, 12, 4), (60, 20, 700, 4), (33, 9, 4100, 3)):
        V, dy = rand(torch, 1, N, D), rand(torch, 2, n, D)
        neurons, weights = make_routes(torch, 3, n, N, k)
        dv, dw = R.read_out_backward(dy, V, neurons, weights)
        size = capi.lib.pink_b200_read_out_workspace(N, D, n, k)
        work = torch.empty(size, dtype=torch.uint8, device="cuda")
        got_v, got_w = torch.full_like(dv, 7.0), torch.full_like(dw, 7.0)

        def call(dvalues, dweights, bytes=size):
            return capi.lib.pink_b200_op_read_out_backward(capi.F32, N, D, V.data_ptr(), D, n, k, neurons.data_ptr(), weights.data_ptr(), dy.data_ptr(), D,
                                                           dvalues, D, dweights, work.data_ptr(), bytes, st)
        capi.check(call(got_v.data_ptr(), None))
        capi.check(call(None, got_w.data_ptr(), 0))        # needs no workspace
        capi.check(call(None, None, 0))
        assert torch.equal(got_v, dv)
        inner = dy.double().abs() @ V.double().abs().t()
        ok = (neurons >= 0) & (neurons < N)
        bound = inner.gather(1, torch.where(ok, neurons, 0).long()) * (D + 1) * 2 * U
        assert ((got_w.double() - dw.double()).abs() <= bound).all() and (got_w[~ok] == 0).all()
    n, K, M = 150, 90, 44
    x, w, z, dy = (rand(torch, i, a, b, dtype="float16") for i, (a, b) in enumerate(((n, K), (M, K), (n, M), (n, M))))
    full = R.product_backward(dy, x, w, z=z, activation="silu")
    cfg = capi.ProductConfig(capi.F16, K, M, 0, capi.ACT_SILU, 0, n)
    for chosen in range(8):
        got = [torch.full_like(t, 7.0) for t in full]
        p = [t.data_ptr() if chosen >> i & 1 else None for i, t in enumerate(got)]
        size = C.c_uint64(0)
        args = (C.byref(cfg), dy.data_ptr(), M, x.data_ptr(), K, w.data_ptr(), K, z.data_ptr(), M, p[0], K, p[1], K, p[2])
        capi.check(capi.lib.pink_b200_op_product_backward(*args, None, C.byref(size), 1, st))
        work = torch.empty(max(size.value, 16), dtype=torch.uint8, device="cuda")
        capi.check(capi.lib.pink_b200_op_product_backward(*args, work.data_ptr(), C.byref(size), 0, st))
        for i in range(3):
            assert torch.equal(got[i], full[i]) if chosen >> i & 1 else (got[i] == 7).all()


# ---- together ------------------------------------------------------------------------------------------------------------

def read_out_step(R, state):
    """Routes from distances, their read-out through a head, and every gradient back to the distances."""
    d, V, w, b, dy = state
    neurons, weights, scores = R.route(d, 4, slope=-2.0, scores=V.dtype)
    y = R.read_out(V, neurons, weights)
    out, z = R.product(y, w, bias=b, activation="gelu", residual=y, keep=True)
    dx, dw, db = R.product_backward(dy, y, w, z=z, activation="gelu")
    dense = R.product(scores, V, by_input=True)
    dscores, dV2, _ = R.product_backward(dy, scores, V, by_input=True)
    dV, dweights = R.read_out_backward(dx, V, neurons, weights)
    dd = R.route_backward(d, neurons, weights, dweights, slope=-2.0, dscores=None if d.dtype != dscores.dtype else dscores)
    return [neurons, weights, scores, y, out, z, dx, dw, db, dense, dV2, dV, dweights, dd]


def step_state(torch, seed):
    return [rand(torch, seed, 70, 331).abs(), rand(torch, seed + 1, 331, 40, dtype="bfloat16"), rand(torch, seed + 2, 40, 40, dtype="bfloat16", scale=0.1),
            rand(torch, seed + 3, 40), rand(torch, seed + 4, 70, 40, dtype="bfloat16")]


def test_a_step_of_all_operators_on_another_stream_and_in_a_graph(R, cuda):
    torch = cuda
    state = step_state(torch, 50)
    want = [t.clone() for t in read_out_step(R, state)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = read_out_step(R, state)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = read_out_step(R, state)
    other = step_state(torch, 90)
    for t, o in zip(state, other):
        t.copy_(o)
    expect = [t.clone() for t in read_out_step(R, other)]
    for _ in range(2):
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(held, expect))


def test_two_steps_at_once(R, cuda):
    """Two streams, nothing shared but inputs: scratch memory belongs to each call."""
    torch = cuda
    state = step_state(torch, 7)
    want = [t.clone() for t in read_out_step(R, state)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    results = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                results.append(read_out_step(R, state))
    torch.cuda.synchronize()
    for got in results:
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_dense_read_out_equals_the_routed_one_over_all_neurons(R, cuda):
    """With as many routes as neurons, routed and dense read-out are the same sum; the scores enter the dense one rounded to float16."""
    torch = cuda
    d, V = rand(torch, 1, 50, 30).abs(), rand(torch, 2, 30, 24, dtype="float16")
    neurons, weights, scores = R.route(d, 30, slope=-1.0, scores=torch.float16)
    a, b = R.read_out(V, neurons, weights).double(), R.product(scores, V, by_input=True).double()
    size = scores.double() @ V.double().abs()
    half = half_step(torch, torch.float16)
    assert ((a - b).abs() <= size * (half + 100 * U) * 1.01 + 2 * half * (a.abs() + b.abs()) + 30 * 2.0 ** -24 * V.double().abs().max()).all()


def test_refusals_leave_the_outputs_alone(R, cuda):
    torch = cuda
    from pink_b200 import capi
    x = rand(torch, 1, 4, 16)
    with pytest.raises(capi.PinkError):
        R.route(x, 17)
    with pytest.raises(capi.PinkError):
        R.route(x, 4, groups=3)
    with pytest.raises(ValueError):
        R.route(x, 4, score="tanh")
    with pytest.raises(ValueError):
        R.route(x.t(), 2)                                  # columns, not rows, are contiguous
    with pytest.raises(ValueError):
        R.route(x, 2, bias=torch.zeros(15, device="cuda"))
    with pytest.raises(ValueError):
        R.route(x, 2, bias=torch.zeros(16))
    with pytest.raises(TypeError):
        R.product(x, x)
    h = x.bfloat16()
    with pytest.raises(TypeError):
        R.product(h, h.half())
    with pytest.raises(ValueError):
        R.product_backward(h[:, :4].contiguous(), h, h, activation="gelu")
    with pytest.raises(ValueError):
        R.product(h, h, out=h[:, :3])
