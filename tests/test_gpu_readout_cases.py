"""The read-out operators where their larger kernels run, and what the tests of test_gpu_readout.py, whose helpers and tolerances these use,
leave open."""
import threading
import warnings

import numpy as np
import pytest

from test_gpu_readout import ACTS, U, check_product, check_product_backward, half_step, make_routes, make_values, pitched, rand, ref_act, ref_logits, ref_route, \
    ref_route_grad, route_tolerance, spread, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def R(cuda):
    from pink_b200 import readout
    yield readout
    readout.check_status()


# ---- many rows of every width ----------------------------------------------------------------------------------------------

# more than 256 rows: the kernels of batches (one warp a row up to 512 neurons, four up to 4,096, sixteen up to 8,192)
BATCHES = [
    # n, N, k, type, options
    (257, 512, 8, "float32", dict(groups=16, top_groups=4, group_best=2, bias=True, mask=True, holes=True)),
    (260, 513, 8, "float32", dict(bias=True, holes=True)),
    (300, 700, 5, "bfloat16", dict(groups=7, top_groups=3, group_best=2, mask=True, bias=True, holes=True)),
    (257, 1024, 32, "float16", dict(renormalise=False, holes=True)),
    (259, 1600, 6, "float32", dict(score="sigmoid", scale=2.5, mask=True)),
    (258, 2048, 4, "float32", dict(slope=-2.0, renormalise=False, mask=True)),
    (257, 2049, 9, "bfloat16", dict(bias=True, groups=3, top_groups=2, holes=True)),
    (300, 2791, 8, "float32", dict(slope=-2.0, bias=True, holes=True)),
    (261, 4096, 16, "float16", dict(groups=64, top_groups=5, group_best=2, bias=True, mask=True, score="sigmoid", renormalise=False)),
    (40, 4097, 8, "float32", dict(bias=True, mask=True, groups=17, top_groups=4, holes=True)),
]


@pytest.mark.parametrize("case", BATCHES, ids=lambda c: "%dx%d-%d-%s" % c[:4])
def test_routes_of_batches(R, cuda, case):
    torch = cuda
    n, N, k, dtype, o = case
    o = dict(o)
    v = make_values(torch, 101 + N, n, N, dtype, o.pop("holes", False))
    v[3] = 0.25                                            # many equal values: the chosen are taken one after the other
    v[5, : N // 2] = v[5, 0]
    bias = rand(torch, 5, N) if o.pop("bias", False) else None
    mask = (torch.arange(N, device="cuda") % 7 != 3) if o.pop("mask", False) else None
    load = torch.zeros(N, dtype=torch.int32, device="cuda")
    neurons, weights, scores = R.route(v, k, bias=bias, mask=mask, load=load, scores=torch.float32, **o)
    wn, ww, wp = ref_route(torch, v, k, bias, mask, **o)
    assert np.array_equal(neurons.cpu().numpy(), wn)
    assert np.array_equal(load.cpu().numpy(), np.bincount(wn[wn >= 0], minlength=N))
    l, takes = ref_logits(torch, v, mask, o.get("slope", 1.0))
    tol = route_tolerance(l, N)
    for got, want in ((weights, ww), (scores, np.where(takes, wp, 0.0))):
        got = got.double().cpu().numpy()
        assert np.all(np.abs(got - want) <= tol * want + 2.0 ** -140), np.abs(got - want).max()
    # the choice alone is made in fewer passes, with the same result; and a row does not depend on those beside it
    again = R.route(v, k, bias=bias, mask=mask, **o)
    assert torch.equal(again[0], neurons) and torch.equal(again[1], weights)
    few = R.route(v[:7], k, bias=bias, mask=mask, **o)
    assert torch.equal(few[0], neurons[:7])


GRAD_BATCHES = [(257, 512, 4, "float32", dict(renormalise=False, dscores=True, mask=True)), (300, 1600, 6, "float16", dict(score="sigmoid", dscores=True, holes=True)),
                (260, 2791, 8, "float32", dict(dscores=True, slope=-2.0, holes=True)), (65, 5000, 5, "bfloat16", dict(renormalise=False, mask=True)),
                (300, 2791, 8, "float32", dict(mask=True, holes=True))]


@pytest.mark.parametrize("case", GRAD_BATCHES, ids=lambda c: "%dx%d-%d-%s" % c[:4])
def test_route_gradients_of_batches(R, cuda, case):
    torch = cuda
    n, N, k, dtype, o = case
    o = dict(o)
    v = make_values(torch, 131 + N, n, N, dtype, o.pop("holes", False))
    mask = (torch.arange(N, device="cuda") % 7 != 3) if o.pop("mask", False) else None
    ds = rand(torch, 9, n, N, dtype=dtype) if o.pop("dscores", False) else None
    neurons, weights = R.route(v, k, mask=mask, **o)
    g = rand(torch, 8, n, k)
    g[neurons < 0] = float("nan")
    args = dict(score="softmax", slope=1.0, scale=1.0, renormalise=True)
    args.update(o)
    got = R.route_backward(v, neurons, weights, g, mask=mask, dscores=ds, **args)
    want, bound = ref_route_grad(torch, v, neurons, weights, torch.nan_to_num(g), args["score"], args["slope"], args["scale"], args["renormalise"], mask, ds)
    half, tiny = half_step(torch, got.dtype), torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    within(got, want, bound * (1 + half) + half * want.abs() + tiny)


# 300 to 3,000 rows: more tiles than pairs of SMs, so that a pair goes from one to the next, and 16 K slices over at most eight stages; 100
# rows: the kernel of few rows with 16 slices over its stages
@pytest.mark.parametrize("size", [(3000, 1000, 3300), (2900, 1030, 3001), (100, 1000, 10000)], ids=lambda s: "%d-%d-%d" % s)
@pytest.mark.parametrize("by_input", [False, True])
@pytest.mark.parametrize("dtype,act", [("bfloat16", "sigmoid"), ("float16", "gelu")])
def test_products_of_many_tiles_and_slices(R, cuda, size, by_input, dtype, act):
    check_product(R, cuda, *size, dtype, by_input, act, True, True)


@pytest.mark.parametrize("size", [(3000, 1000, 3300), (2900, 3301, 1030)], ids=lambda s: "%d-%d-%d" % s)
@pytest.mark.parametrize("by_input", [False, True])
@pytest.mark.parametrize("dtype,act", [("bfloat16", "silu"), ("float16", "none"), ("float16", "gelu")])
def test_product_gradients_of_many_tiles_and_slices(R, cuda, size, by_input, dtype, act):
    check_product_backward(R, cuda, *size, dtype, by_input, act)


# ---- what the first tests leave open ------------------------------------------------------------------------------------------

def test_groups_of_one_neuron_take_the_first(R, cuda):
    torch = cuda
    neurons, _ = R.route(torch.zeros(3, 5, device="cuda"), 3, groups=5, top_groups=3, group_best=2)
    assert neurons.tolist() == [[0, 1, 2]] * 3


@pytest.mark.parametrize("renormalise", [True, False])
def test_gradients_back_to_float32_distances_through_both_read_outs(R, cuda, renormalise):
    """The routed and the dense read-out of one routing: the dense scores' gradient goes back in float32."""
    torch = cuda
    d, V = rand(torch, 1, 70, 331).abs(), rand(torch, 2, 331, 40, dtype="bfloat16")
    neurons, weights, scores = R.route(d, 4, slope=-2.0, renormalise=renormalise, scores=torch.bfloat16)
    dy = rand(torch, 3, 70, 40, dtype="bfloat16")
    dscores, _, _ = R.product_backward(dy, scores, V, by_input=True)
    _, dweights = R.read_out_backward(dy, V, neurons, weights)
    got = R.route_backward(d, neurons, weights, dweights, slope=-2.0, renormalise=renormalise, dscores=dscores.float())
    want, bound = ref_route_grad(torch, d, neurons, weights, dweights, "softmax", -2.0, 1.0, renormalise, None, dscores.float())
    within(got, want, bound * (1 + U) + U * want.abs() + 2.0 ** -149)


def test_scratch_of_two_streams(R, cuda):
    """Calls that alternate between two streams, each freeing its scratch memory at once: none of them is given the other's."""
    torch = cuda
    V, dy = rand(torch, 1, 50, 300), rand(torch, 2, 2000, 300)
    neurons, weights = make_routes(torch, 3, 2000, 50, 4)
    x, w = rand(torch, 4, 700, 333, dtype="bfloat16"), rand(torch, 5, 90, 333, dtype="bfloat16")
    want = R.read_out_backward(dy, V, neurons, weights) + (R.product(x, w),)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(40):
        with torch.cuda.stream(streams[i % 2]):
            got.append(R.read_out_backward(dy, V, neurons, weights) + (R.product(x, w),))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


# ---- the range of float16 -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("by_input", [False, True])
@pytest.mark.parametrize("pitch", [(0, 0), (3, 1)], ids=str)
@pytest.mark.parametrize("act,z,dout", [("sigmoid", 8.0, 1e-4), ("sigmoid", -9.0, 2e-7), ("silu", 3.0, 1e-7), ("gelu", 1.4, 6e4), ("silu", 2.0, 6.5e4)])
def test_float16_gradients_keep_what_dout_times_slope_holds(R, cuda, by_input, pitch, act, z, dout):
    """dz = dout * act'(z) beyond what float16 holds (here 2^-25 and less, or more than 65,504), in results that it does hold: dz may be
    off by half a step of ITS magnitude, not of the subnormals'."""
    torch = cuda
    n, K, M = 70, 88, 40
    scale = 2.0 ** -12 if dout > 1 else 300.0
    x, w = rand(torch, 1, n, K, dtype="float16", scale=scale), rand(torch, 2, M, K, dtype="float16", scale=scale)
    zz = (z * (1 + 0.01 * rand(torch, 3, n, M))).half()
    dy = (dout * (1 - 0.3 * torch.rand(n, M, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda"))).half()
    P = lambda t: pitched(torch, t, *pitch)
    dx, dw, db = R.product_backward(P(dy), P(x), P(w.t().contiguous() if by_input else w), by_input=by_input, z=P(zz), activation=act)
    _, slope = ref_act(torch, zz.double(), act)
    dz, half, tiny = dy.double() * slope, 2.0 ** -11, 2.0 ** -24
    edz = half * dz.abs() + 20 * U * dy.double().abs() * slope.abs()          # (the slopes here are sums without cancellation)
    for got, want, size, err, terms in ((dx, dz @ w.double(), dz.abs() @ w.double().abs(), edz @ w.double().abs(), M),
                                        (dw.t() if by_input else dw, dz.t() @ x.double(), dz.abs().t() @ x.double().abs(), edz.t() @ x.double().abs(), n)):
        within(got, want, (size * (terms + 2) * 2 * U + err) * (1 + half) + half * want.abs() + tiny / 2)
    within(db, dz.sum(0), edz.sum(0) + dz.abs().sum(0) * (n + 1) * U)


def test_float16_gradients_with_infinities_and_zeros_in_dout(R, cuda):
    """An infinite gradient stays in its row of dx and its column of dw; the others are as without it.  A gradient of zeros gives zeros."""
    torch = cuda
    n, K, M = 33, 24, 16
    x, w, z = rand(torch, 1, n, K, dtype="float16"), rand(torch, 2, M, K, dtype="float16"), rand(torch, 3, n, M, dtype="float16")
    dy = rand(torch, 4, n, M, dtype="float16", scale=1e-4)
    clean = dy.clone()
    clean[5, 3] = 0
    dx0, dw0, _ = R.product_backward(clean, x, w, z=z, activation="silu")
    for bad in (float("inf"), float("nan")):
        dy[5, 3] = bad
        dx, dw, db = R.product_backward(dy, x, w, z=z, activation="silu")
        assert not torch.isfinite(dx[5]).any() and not torch.isfinite(dw[3]).any() and not torch.isfinite(db[3])
        rows, cols = torch.arange(n) != 5, torch.arange(M) != 3
        assert torch.equal(dx[rows], dx0[rows]) and torch.equal(dw[cols], dw0[cols])
    for g in R.product_backward(torch.zeros_like(dy), x, w, z=z, activation="silu"):
        assert (g == 0).all()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("act", ACTS[1:])
def test_slopes_where_z_is_beyond_its_type(R, cuda, act, dtype):
    """A kept z that its type holds as an infinity: the slope there is its limit, 0 or 1 (the forward result is finite on the negative side)."""
    torch = cuda
    n, K, M = 40, 24, 16
    x, w, z, dy = (rand(torch, i, a, b, dtype=dtype) for i, (a, b) in enumerate(((n, K), (M, K), (n, M), (n, M))))
    z[3, 2], z[7, 9] = float("inf"), -float("inf")
    far = z.clone()
    far[3, 2], far[7, 9] = 6e4, -6e4
    for got, want in zip(R.product_backward(dy, x, w, z=z, activation=act), R.product_backward(dy, x, w, z=far, activation=act)):
        assert torch.isfinite(want).all() and torch.equal(got, want)
    z[3, 2] = float("nan")
    dx, dw, _ = R.product_backward(dy, x, w, z=z, activation=act)
    assert act == "relu" or (torch.isnan(dx[3]).all() and torch.isnan(dw[2]).all())


# ---- several threads -------------------------------------------------------------------------------------------------------------

def test_two_threads_with_rows_of_different_sizes(R, cuda):
    """Calls from two threads at once, whose kernels need different amounts of shared memory: neither call may undo what the other has asked
    for between its request and its launch."""
    torch = cuda
    wrong = []

    def work(N, routes):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                v = rand(torch, N, 1, N)
                V, dy = rand(torch, 1, routes, 4), rand(torch, 2, 3000, 4)
                e, w = make_routes(torch, 3, 3000, routes, 4)
                g = rand(torch, 4, 1, 4)
                want = None
                for _ in range(600):
                    neurons, weights = R.route(v, 4)
                    dv = R.route_backward(v, neurons, weights, g, renormalise=False)
                    got = (neurons, weights, dv) + R.read_out_backward(dy, V, e, w)
                    want = want or got
                stream.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(got, want))
        except Exception as err:                           # (an assertion in a thread would be lost)
            wrong.append(err)
    threads = [threading.Thread(target=work, args=a) for a in ((9000, 14000), (32768, 32000), (20000, 20000))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong


@pytest.mark.parametrize("by_input", [False, True])
def test_product_gradient_of_rows_read_often(R, cuda, by_input):
    """dz without an activation, in rows that straddle lines and are read by many tiles: it is copied first, for both products or for one."""
    check_product_backward(R, cuda, 256, 3648, 1032, "bfloat16", by_input, "none")
    check_product_backward(R, cuda, 512, 1030, 8184, "float16", by_input, "none")


# ---- calls that cannot be right ----------------------------------------------------------------------------------------------------

def test_results_that_overlap_what_is_read_are_refused(R, cuda):
    torch = cuda
    h = rand(torch, 1, 40, 64, dtype="bfloat16")
    keep = h.clone()
    w = rand(torch, 2, 64, 64, dtype="bfloat16")
    for out in (h, h.view(-1)[:40 * 32].view(40, 32), h[:, 32:], h[:, :1]):
        with pytest.raises(ValueError, match="overlap"):
            R.product(h, w[:out.shape[1]], out=out)
    with pytest.raises(ValueError, match="overlap"):
        R.product(h[:8], w, out=w[3:11])
    shifted = rand(torch, 5, 41, 64, dtype="bfloat16")
    with pytest.raises(ValueError, match="overlap"):
        R.product(h, w, residual=shifted[:40], out=shifted[1:])
    V, (neurons, weights) = rand(torch, 3, 40, 33), make_routes(torch, 4, 20, 40, 3)
    with pytest.raises(ValueError, match="overlap"):
        R.read_out(V, neurons, weights, out=V[:20])
    assert torch.equal(h, keep)
    # side by side in one matrix is no overlap, nor is a residual that becomes the result
    wide = torch.zeros(40, 104, dtype=torch.bfloat16, device="cuda")
    wide[:, :64] = h
    R.product(wide[:, :64], w[:40], out=wide[:, 64:])
    assert torch.equal(wide[:, 64:], R.product(h, w[:40])) and torch.equal(wide[:, :64], h)
    want = R.product(h, w, residual=keep)
    assert torch.equal(R.product(h, w, residual=keep, out=keep), want)
    rest = torch.zeros(60, 33, device="cuda")
    rest[20:] = V
    assert torch.equal(R.read_out(rest[20:], neurons, weights, out=rest[:20]), R.read_out(V, neurons, weights))


def test_a_result_without_a_graph_is_announced(R, cuda):
    """The operators take no part in autograd: a forward call that torch would be expected to record says that it is not."""
    torch = cuda
    x, w = rand(torch, 1, 9, 16, dtype="bfloat16"), rand(torch, 2, 8, 16, dtype="bfloat16")
    d, V = rand(torch, 3, 9, 8), rand(torch, 4, 8, 5)
    neurons, weights = R.route(d, 2)
    calls = [(lambda t: R.product(t, w), x), (lambda t: R.product(x, t), w), (lambda t: R.product(x, w, bias=t), rand(torch, 5, 8)),
             (lambda t: R.product(x, w, residual=t), rand(torch, 6, 9, 8, dtype="bfloat16")), (lambda t: R.route(t, 2)[1], d),
             (lambda t: R.read_out(t, neurons, weights), V), (lambda t: R.read_out(V, neurons, t), weights),
             (lambda t: R.read_out(V, neurons, weights, residual=t), rand(torch, 7, 9, 5))]
    for call, t in calls:
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            want = call(t)                                 # nothing to say
            with torch.no_grad():
                call(t.clone().requires_grad_())
        with pytest.warns(UserWarning, match="no part in autograd"):
            got = call(t.clone().requires_grad_())
        assert torch.equal(got, want) and not got.requires_grad


# ---- shared memory near its limit without an opt-in -----------------------------------------------------------------------------------

@pytest.mark.parametrize("N", [1359, 1360, 1361, 1362, 1363, 1364, 1365])
def test_small_sorts_around_48_kilobytes(R, cuda, N):
    """Fixed and requested shared memory count together."""
    torch = cuda
    n, D, k = 60, 5, 4
    V, dy = rand(torch, 1, N, D), rand(torch, 2, n, D)
    neurons, weights = make_routes(torch, 3, n, N, k)
    S, A, ok = spread(torch, neurons, weights, N)
    dv, dw = R.read_out_backward(dy, V, neurons, weights)
    within(dv, S.t() @ dy.double(), (A.t() @ dy.double().abs()) * (n * k + 1) * 2 * U)
    e = torch.where(ok, neurons, 0).long()
    within(dw, torch.where(ok, (dy.double() @ V.double().t()).gather(1, e), 0.0), (dy.double().abs() @ V.double().abs().t()).gather(1, e) * (D + 1) * U)


@pytest.mark.parametrize("N,groups", [(12033, 3), (12100, 1), (12160, 64), (12240, 1), (12287, 1), (12288, 1), (12288, 256), (12289, 1)])
def test_long_rows_around_48_kilobytes(R, cuda, N, groups):
    torch = cuda
    v = rand(torch, 1, 2, N)
    o = dict(groups=groups, renormalise=False)
    neurons, weights, scores = R.route(v, 4, scores=torch.float32, **o)
    wn, ww, wp = ref_route(torch, v, 4, **o)
    l, _ = ref_logits(torch, v, None, 1.0)
    tol = route_tolerance(l, N)
    assert np.array_equal(neurons.cpu().numpy(), wn)
    for got, want in ((weights, ww), (scores, wp)):
        assert np.all(np.abs(got.double().cpu().numpy() - want) <= tol * want + 2.0 ** -140)
    g = rand(torch, 2, 2, 4)
    got = R.route_backward(v, neurons, weights, g, renormalise=False)
    want, bound = ref_route_grad(torch, v, neurons, weights, g, "softmax", 1.0, 1.0, False, None, None)
    within(got, want, bound * (1 + U) + U * want.abs() + 2.0 ** -140)
