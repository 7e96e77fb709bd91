"""Gated projections and their gradients against plain products in 64 bits (tolerances as for the product in test_gpu_readout.py), and a head
of all the operators, trained against the routes of a map."""
import pytest

from test_gpu_readout import ACTS, U, half_step, pitched, rand, ref_act, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def R(cuda):
    from pink_b200 import readout
    yield readout
    readout.check_status()


def tiny_of(torch, dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def make(torch, n, K, M, dtype, by_input, seed=0):
    x = rand(torch, seed + 1, n, K, dtype=dtype)
    gate, up = (rand(torch, seed + i, M, K, dtype=dtype, scale=K ** -0.5) for i in (2, 3))
    lay = lambda w: w.t().contiguous() if by_input else w
    return x, gate, up, lay(gate), lay(up)


def check_gated(R, torch, n, K, M, dtype, by_input, act, bias, extra=0, offset=0, seed=0):
    x, gate, up, lg, lu = make(torch, n, K, M, dtype, by_input, seed)
    gb, ub = (rand(torch, seed + 4, M), rand(torch, seed + 5, M)) if bias else (None, None)
    P = lambda t: pitched(torch, t, extra, offset)
    o = dict(by_input=by_input, gate_bias=gb, up_bias=ub, activation=act)
    h, g, u = R.gated(P(x), P(lg), P(lu), keep=True, **o)
    half, tiny = half_step(torch, x.dtype), tiny_of(torch, x.dtype)
    want, err = [], []
    for w, b, got in ((gate, gb, g), (up, ub, u)):
        z = x.double() @ w.double().t()
        e = (x.double().abs() @ w.double().abs().t()) * (K + 2) * 2 * U        # (a tensor core may cut its sums: 2 u a term)
        if b is not None:
            z = z + b.double()
            e = e + U * z.abs()
        within(got, z, e * (1 + half) + half * z.abs() + tiny)
        want.append(z)
        err.append(e)
    a, _ = ref_act(torch, want[0], act)
    ea = 1.13 * err[0] + 16 * U * (a.abs() + 1e-30)        # no activation here is steeper than 1.13
    y = a * want[1]
    ey = ea * want[1].abs() + (a.abs() + ea) * err[1] + 2 * U * y.abs()
    within(h, y, ey * (1 + half) + half * y.abs() + tiny)
    # the bounds above grow with K; a lost slice or element would show here: rounding alone moves the norm by less than half
    for got, z in ((g, want[0]), (u, want[1]), (h, y)):
        if z.norm() > 0:
            assert (got.double() - z).norm() / z.norm() <= half + 1e-5
    assert torch.equal(R.gated(P(x), P(lg), P(lu), **o), h)


# few rows, one pair, several tiles, ranges of K, ragged everything
GATED_SIZES = [(1, 1, 1), (1, 400, 10), (2, 33, 7), (3, 64, 129), (4, 4000, 40), (5, 130, 64), (7, 961, 400), (8, 2791, 33), (9, 1, 1), (9, 400, 10), (16, 63, 17), (64, 64, 64), (65, 65, 65),
               (128, 128, 256), (129, 72, 257), (300, 961, 40), (500, 2791, 10), (1000, 16, 1000), (40, 5000, 24), (100, 1000, 10000), (257, 321, 513), (4100, 40, 24), (33, 20000, 33)]


@pytest.mark.parametrize("size", GATED_SIZES, ids=lambda s: "%d-%d-%d" % s)
@pytest.mark.parametrize("by_input", [False, True])
def test_gated_sizes(R, cuda, size, by_input):
    n, K, M = size
    i = n + K + M
    check_gated(R, cuda, n, K, M, "bfloat16" if i % 2 else "float16", by_input, ACTS[i % 5], i % 3 != 0)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("pitch", [(0, 0), (8, 0), (3, 1), (4, 0), (4, 4)], ids=str)
def test_gated_types_activations_and_pitches(R, cuda, dtype, act, pitch):
    for n in (1, 2, 3, 6, 70):
        for by_input in (False, True):
            check_gated(R, cuda, n, 300, 44, dtype, by_input, act, True, *pitch)


# more tiles than pairs of SMs, more K slices than stages
@pytest.mark.parametrize("size", [(3000, 1000, 3300), (2900, 1030, 1701)], ids=lambda s: "%d-%d-%d" % s)
@pytest.mark.parametrize("by_input", [False, True])
def test_gated_of_many_tiles_and_slices(R, cuda, size, by_input):
    check_gated(R, cuda, *size, "bfloat16", by_input, "silu", True)


def check_gated_backward(R, torch, n, K, M, dtype, by_input, act, extra=0, offset=0, seed=0):
    x, gate, up, lg, lu = make(torch, n, K, M, dtype, by_input, seed)
    g, u, dh = (rand(torch, seed + i, n, M, dtype=dtype) for i in (6, 7, 8))
    P = lambda t: pitched(torch, t, extra, offset)
    o = dict(by_input=by_input, activation=act)
    got = R.gated_backward(P(dh), P(x), P(lg), P(lu), P(g), P(u), **o)
    dx, dgate, dup, dgb, dub = got
    half, tiny = half_step(torch, x.dtype), tiny_of(torch, x.dtype)
    a, s = ref_act(torch, g.double(), act)
    d, ud = dh.double(), u.double()
    dg, du = d * ud * s, d * a
    eg, eu = 24 * U * (d * ud).abs(), 24 * U * (d * a).abs() + 1e-30           # (a slope's terms are at most 1.2)
    if by_input:
        dgate, dup = dgate.t(), dup.t()
    rg, ru = eg + half * dg.abs() + tiny, eu + half * du.abs() + tiny          # they enter the products rounded
    gd, pd, xd = gate.double(), up.double(), x.double()
    for result, want, size, err, terms in ((dx, dg @ gd + du @ pd, dg.abs() @ gd.abs() + du.abs() @ pd.abs(), rg @ gd.abs() + ru @ pd.abs(), 2 * M),
                                           (dgate, dg.t() @ xd, dg.abs().t() @ xd.abs(), rg.t() @ xd.abs(), n), (dup, du.t() @ xd, du.abs().t() @ xd.abs(), ru.t() @ xd.abs(), n)):
        within(result, want, (size * (terms + 2) * 2 * U + err) * (1 + half) + half * want.abs() + tiny)
        if want.norm() > 0:
            assert (result.double() - want).norm() / want.norm() <= 2 * half + 1e-5      # one rounding of dg or du, one of the result
    within(dgb, dg.sum(0), dg.abs().sum(0) * (n + 1) * U + eg.sum(0))
    within(dub, du.sum(0), du.abs().sum(0) * (n + 1) * U + eu.sum(0))
    assert all(torch.equal(p, q) for p, q in zip(R.gated_backward(P(dh), P(x), P(lg), P(lu), P(g), P(u), **o), got))


GRADIENT_SIZES = [(1, 1, 1), (1, 400, 10), (3, 10, 70), (9, 65, 33), (64, 64, 64), (129, 72, 257), (300, 961, 40), (1000, 100, 10), (2000, 33, 129), (257, 321, 513), (5000, 24, 16), (20, 130, 4000)]


@pytest.mark.parametrize("size", GRADIENT_SIZES, ids=lambda s: "%d-%d-%d" % s)
@pytest.mark.parametrize("by_input", [False, True])
def test_gated_gradients(R, cuda, size, by_input):
    n, K, M = size
    i = n + K + M
    check_gated_backward(R, cuda, n, K, M, "bfloat16" if i % 2 else "float16", by_input, ACTS[i % 5])


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("pitch", [(0, 0), (8, 0), (3, 1), (4, 4)], ids=str)
def test_gated_gradient_activations_and_pitches(R, cuda, act, pitch):
    for by_input in (False, True):
        check_gated_backward(R, cuda, 150, 88, 40, "float16", by_input, act, *pitch)
        check_gated_backward(R, cuda, 60, 40, 300, "bfloat16", by_input, act, *pitch)


@pytest.mark.parametrize("size", [(3000, 1000, 2300), (2900, 2301, 1030)], ids=lambda s: "%d-%d-%d" % s)
@pytest.mark.parametrize("by_input", [False, True])
def test_gated_gradients_of_many_tiles_and_slices(R, cuda, size, by_input):
    check_gated_backward(R, cuda, *size, "bfloat16", by_input, "silu")
    check_gated_backward(R, cuda, *size, "float16", by_input, "gelu")


@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid", "none"])
@pytest.mark.parametrize("size", [1e-5, 1e-7, 30.0, 2e3])
def test_float16_gradients_keep_what_three_factors_hold(R, cuda, act, size):
    """dh * u * act'(g) far below what float16 holds, or above, in results that it does hold."""
    torch = cuda
    n, K, M = 70, 88, 40
    x, gate, up, _, _ = make(torch, n, K, M, "float16", False)
    scale = 2.0 ** -14 if size > 1 else 200.0
    x, gate, up = (scale * t.float() for t in (x, gate, up))
    x, gate, up = x.half(), gate.half(), up.half()
    g = rand(torch, 6, n, M, dtype="float16", scale=2.0)
    u, dh = rand(torch, 7, n, M, dtype="float16", scale=100.0 if size > 1 else 1e-2), rand(torch, 8, n, M, dtype="float16", scale=size)
    dx, dgate, dup, _, _ = R.gated_backward(dh, x, gate, up, g, u, activation=act)
    a, s = ref_act(torch, g.double(), act)
    dg, du = dh.double() * u.double() * s, dh.double() * a
    peak = max(dg.abs().max(), du.abs().max()).item()
    half, least = 2.0 ** -11, peak * 2.0 ** -14 * 2.0 ** -25       # half of float16's last subnormal step where the peak is 2^14 or more
    rg, ru = half * dg.abs() + 24 * U * (dh.double() * u.double()).abs() + least, half * du.abs() + 24 * U * du.abs() + least
    for got, want, size_, err, terms in ((dx, dg @ gate.double() + du @ up.double(), dg.abs() @ gate.double().abs() + du.abs() @ up.double().abs(),
                                          rg @ gate.double().abs() + ru @ up.double().abs(), 2 * M),
                                         (dgate, dg.t() @ x.double(), dg.abs().t() @ x.double().abs(), rg.t() @ x.double().abs(), n),
                                         (dup, du.t() @ x.double(), du.abs().t() @ x.double().abs(), ru.t() @ x.double().abs(), n)):
        assert want.abs().max() < 65504
        within(got, want, (size_ * (terms + 2) * 2 * U + err) * (1 + half) + half * want.abs() + 2.0 ** -25)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("act", ACTS)
def test_kept_projections_beyond_their_type(R, cuda, act, dtype):
    """A gate that its type holds as -infinity has the limits of act and its slope there; an infinity beside a gradient of zero does nothing."""
    torch = cuda
    n, K, M = 40, 24, 16
    x, gate, up, _, _ = make(torch, n, K, M, dtype, False)
    g, u, dh = (rand(torch, i, n, M, dtype=dtype) for i in (6, 7, 8))
    dh[9, 3] = dh[11, 4] = 0
    g[9, 3], u[11, 4] = float("inf"), -float("inf")
    if act != "none":
        g[3, 2] = -float("inf")
    far = g.clone()
    far[3, 2] = -6e4 if act != "none" else far[3, 2]
    far[9, 3] = 1.0
    near = u.clone()
    near[11, 4] = 1.0
    for got, want in zip(R.gated_backward(dh, x, gate, up, g, u, activation=act), R.gated_backward(dh, x, gate, up, far, near, activation=act)):
        assert torch.isfinite(want).all() and torch.equal(got, want)
    g[5, 6] = float("nan")
    dx, dgate, _, dgb, _ = R.gated_backward(dh, x, gate, up, g, u, activation="silu")
    rows, cols = torch.arange(n) != 5, torch.arange(M) != 6
    assert torch.isnan(dx[5]).all() and torch.isfinite(dx[rows]).all() and torch.isnan(dgate[6]).all() and torch.isfinite(dgate[cols]).all() and torch.isfinite(dgb[cols]).all()
    for t in R.gated_backward(torch.zeros_like(dh), x, gate, up, far, near, activation=act):
        assert (t == 0).all()


@pytest.mark.parametrize("n", [1, 5, 40, 300])
@pytest.mark.parametrize("by_input", [False, True])
def test_what_is_not_finite_stays_in_its_row(R, cuda, n, by_input):
    torch = cuda
    x, _, _, gate, up = make(torch, n, 200, 50, "bfloat16", by_input)
    h = R.gated(x, gate, up, by_input=by_input)
    x[n // 2, 77] = float("nan")
    got = R.gated(x, gate, up, by_input=by_input)
    rows = torch.arange(n) != n // 2
    assert torch.isnan(got[n // 2]).all() and torch.equal(got[rows], h[rows])


def test_gated_of_nothing_and_of_places_behind_the_last(R, cuda):
    torch = cuda
    x, gate, up, _, _ = make(torch, 20, 40, 24, "bfloat16", False)
    none = x[:0]
    assert R.gated(none, gate, up).shape == (0, 24)
    dx, *rest = R.gated_backward(none.new_empty(0, 24), none, gate, up, none.new_empty(0, 24), none.new_empty(0, 24))
    assert dx.shape == (0, 40) and all((t == 0).all() for t in rest) and rest[0].shape == gate.shape
    from pink_b200 import capi
    import ctypes as C
    for n, M in ((3, 24), (11, 21)):
        out = torch.full((20, 30), 7.0, dtype=torch.bfloat16, device="cuda")
        cfg, size = capi.ProductConfig(capi.BF16, 40, M, 0, capi.ACT_SILU, 0, n), C.c_uint64(0)
        args = (x.data_ptr(), 40, gate.data_ptr(), 40, up.data_ptr(), 40, None, None, out.data_ptr(), 30, None, 0, None, 0)
        capi.check(capi.lib.pink_b200_op_gated(cfg, *args, None, size, 1, None))
        work = torch.empty(size.value + 16, dtype=torch.uint8, device="cuda")
        capi.check(capi.lib.pink_b200_op_gated(cfg, *args, work.data_ptr(), size, 0, None))
        assert (out[n:] == 7).all() and (out[:, M:] == 7).all() and torch.equal(out[:n, :M], R.gated(x[:n], gate[:M], up[:M]))


def test_gated_gradient_against_differences(R, cuda):
    """Along the gate's bias in 64 bits, where float16 kept g and u: d sum(h dh) / d bias, central differences of step h = 1e-3, off by
    h^2 / 6 of a third derivative (below 2) times sum |dh u|."""
    torch = cuda
    n, K, M = 12, 16, 8
    x, gate, up, _, _ = make(torch, n, K, M, "float16", False)
    dh, step = rand(torch, 8, n, M, dtype="float16"), 1e-3
    for act in ("gelu", "silu", "sigmoid"):
        _, g, u = R.gated(x, gate, up, activation=act, keep=True)
        _, _, _, dgb, dub = R.gated_backward(dh, x, gate, up, g, u, activation=act)
        f = lambda dz, dv: (ref_act(torch, g.double() + dz, act)[0] * (u.double() + dv) * dh.double()).sum(0)
        slack = (dh.double().abs() * (u.double().abs() + 1)).sum(0) * (2 * step * step / 6 + 30 * U * (n + 2)) + 1e-9
        within(dgb, (f(step, 0) - f(-step, 0)) / (2 * step), slack)
        within(dub, (f(0, step) - f(0, -step)) / (2 * step), slack)


# ---- all of them, as a head is trained -----------------------------------------------------------------------------------------

def head_step(R, p, x, neurons, weights):
    """Losses and gradients of a pre-norm block with a gated hidden layer and scores for the neurons, with the operators."""
    n = x.shape[0]
    y, mean, rstd = R.layer_norm(x, p["w1"], p["b1"], keep=True)
    h, g, u = R.gated(y, p["gate"], p["up"], gate_bias=p["gb"], keep=True)
    t = R.product(h, p["down"], residual=x)
    y2, mean2, rstd2 = R.layer_norm(t, p["w2"], p["b2"], keep=True)
    s = R.product(y2, p["head"], bias=p["hb"])
    ds, loss = R.distill_backward(None, s, neurons, weights, scale=1.0 / n, rest=True, loss=True)
    d = {}
    dy2, d["head"], d["hb"] = R.product_backward(ds, y2, p["head"])
    dt, d["w2"], d["b2"] = R.layer_norm_backward(dy2, t, mean2, rstd2, p["w2"])
    dh, d["down"], _ = R.product_backward(dt, h, p["down"])
    dy, d["gate"], d["up"], d["gb"], _ = R.gated_backward(dh, y, p["gate"], p["up"], g, u)
    d["x"], d["w1"], d["b1"] = R.layer_norm_backward(dy, x, mean, rstd, p["w1"], residual=dt)
    return loss, d


def head_of(torch, D, M, N, dtype):
    r = lambda i, *shape, scale=1.0: rand(torch, i, *shape, scale=scale)
    h = lambda i, *shape: rand(torch, i, *shape, dtype=dtype, scale=shape[-1] ** -0.5)
    return dict(w1=1 + 0.1 * r(1, D), b1=0.1 * r(2, D), gate=h(3, M, D), up=h(4, M, D), gb=0.1 * r(5, M), down=h(6, D, M), w2=1 + 0.1 * r(7, D), b2=0.1 * r(8, D),
                head=h(9, N, D), hb=0.1 * r(10, N))


def exact_head(torch, p, x, neurons, weights):
    F = torch.nn.functional
    q = {k: v.double().requires_grad_(True) for k, v in dict(p, x=x).items()}
    n, D = x.shape
    y = F.layer_norm(q["x"], (D,), q["w1"], q["b1"], 1e-5)
    h = F.silu(y @ q["gate"].t() + q["gb"]) * (y @ q["up"].t())
    t = h @ q["down"].t() + q["x"]
    s = F.layer_norm(t, (D,), q["w2"], q["b2"], 1e-5) @ q["head"].t() + q["hb"]
    lq = torch.log_softmax(s, 1)
    e, w = neurons.long(), weights.double()
    r = 1 - w.sum(1)
    others = torch.ones_like(s, dtype=torch.bool).scatter(1, e, False)
    lr = torch.logsumexp(lq.masked_fill(~others, -float("inf")), 1)
    loss = ((w * (w.log() - lq.gather(1, e))).sum(1) + r * (r.log() - lr)) / n
    grads = torch.autograd.grad(loss.sum(), list(q.values()))
    return loss.detach(), dict(zip(q, grads))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("shape", [(1, 40, 30, 20), (50, 961, 400, 400), (300, 333, 515, 1001)], ids=lambda s: "%d-%d-%d-%d" % s)
def test_a_step_of_a_head_against_64_bits(R, cuda, shape, dtype):
    """Fourteen roundings to 16 bits lie between the input and its gradient, each of half a step of its value, and none of the maps between
    them is longer than 3 (norms, weights of unit rows): relative to its norm no gradient is off by more than 14 * 3 half steps."""
    torch = cuda
    n, D, M, N = shape
    p, x = head_of(torch, D, M, N, dtype), rand(torch, 20, n, D, dtype=dtype)
    neurons, weights = R.route(rand(torch, 21, n, N).abs() * 4, 5, slope=-2.0, renormalise=False)
    loss, d = head_step(R, p, x, neurons, weights)
    want, dwant = exact_head(torch, p, x, neurons, weights)
    limit = 14 * 3 * half_step(torch, x.dtype)
    assert (loss.double() - want).norm() <= limit * want.norm()
    for k in d:
        off = ((d[k].double() - dwant[k]).norm() / dwant[k].norm()).item()
        assert off <= limit, (k, off)


def test_a_step_of_a_head_on_another_stream_and_in_two_graphs(R, cuda):
    """Replays of two graphs of one step on different inputs, in turn, give what the plain calls do: neither has scratch of the other's."""
    torch = cuda
    p = head_of(torch, 200, 120, 300, "bfloat16")
    inputs = []
    for i in range(2):
        x = rand(torch, 30 + i, 90, 200, dtype="bfloat16")
        inputs.append((x,) + tuple(R.route(rand(torch, 40 + i, 90, 300).abs() * 4, 5, slope=-2.0, renormalise=False)))
    want = [head_step(R, p, *i) for i in inputs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        got = [head_step(R, p, *i) for i in inputs]
    side.synchronize()
    for i in inputs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = head_step(R, p, *i)
        graphs.append((graph, out))
    for _ in range(3):
        for graph, _ in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for (loss, d), (sloss, sd), (_, (gloss, gd)) in zip(want, got, graphs):
        assert torch.equal(loss, sloss) and torch.equal(loss, gloss)
        assert all(torch.equal(d[k], sd[k]) and torch.equal(d[k], gd[k]) for k in d)
