"""The operators that train a head where their kernels change over and where rows are unlike one another: many rows (the kernels that pass rows through
shared memory), outliers, scores that are not finite, results that are left out or take an argument's place.

References and tolerances are those of test_gpu_head.py and test_gpu_gated.py."""
import ctypes as C

import pytest

from test_gpu_gated import make as make_gated
from test_gpu_head import check_distill, check_norm, check_norm_backward, make_scores, make_targets
from test_gpu_readout import TYPES, U, pitched, rand, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def R(cuda):
    from pink_b200 import readout
    yield readout
    readout.check_status()


def many(torch):
    """Rows from which on norm and distillation pass them through shared memory, and a few more: eight an SM."""
    return 8 * torch.cuda.get_device_properties(0).multi_processor_count + 3


# ---- layer norm --------------------------------------------------------------------------------------------------------------

def with_outliers(torch, n, D, dtype, size):
    """Rows of ordinary elements, of which some have outliers at one, some at four and some at all eight of the places (2 i + 1) D / 16."""
    size = min(size, 6e4) if dtype == "float16" else size
    x, at = rand(torch, 1, n, D), [(2 * i + 1) * D // 16 for i in range(8)]
    for i, p in enumerate(at):
        x[i::16, p] = size
    x[8::16, at] = size
    x[9::16, at[:4]] = -size
    x[10::16, at[::2]] = size
    return x.to(getattr(torch, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [1e3, 1e5, 1e6])
@pytest.mark.parametrize("D", [30, 64, 100, 128, 256, 300, 512, 961, 2791, 8100, 16000])
def test_norm_of_rows_with_outliers(R, cuda, D, size, dtype):
    """An outlier costs the other elements nothing, wherever in its row it stands and whichever kernel takes the row."""
    torch = cuda
    x = with_outliers(torch, 16, D, dtype, size)
    w, b = rand(torch, 2, D), rand(torch, 3, D)
    check_norm(R, torch, x, w, b)
    check_norm_backward(R, torch, x, rand(torch, 4, 16, D, dtype=dtype), w, None)
    check_norm(R, torch, with_outliers(torch, many(torch), D, dtype, size), w, b)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("D", [1, 2, 3])
def test_norm_of_short_rows_near_the_end_of_the_range(R, cuda, D, dtype):
    """A row whose sum is within float32's range: without spread it is the bias."""
    torch = cuda
    x, b = torch.full((5, D), 1e38, dtype=getattr(torch, dtype), device="cuda"), rand(torch, 1, D)
    x[1], x[2] = -x[1], 1.0
    y, mean, rstd = R.layer_norm(x, None, b, keep=True)
    assert torch.equal(y, b.to(y.dtype).expand(5, D)) and torch.equal(mean, x[:, 0].float())
    assert torch.isfinite(rstd).all() and (rstd == rstd[2]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [24, 50, 64, 100, 240])
def test_norm_of_a_row_does_not_depend_on_its_neighbours(R, cuda, D, dtype):
    """Bit for bit, where rows share a warp or a block and one of them lies far from its sampled elements."""
    torch = cuda
    x, far = rand(torch, 1, 40, D, dtype=dtype), with_outliers(torch, 16, D, dtype, 1e4)
    want = R.layer_norm(x, keep=True)
    z = x.clone()
    z[[2, 13, 21, 35]] = far[[8, 0, 8, 9]]
    rest = [i for i in range(40) if i not in (2, 13, 21, 35)]
    for a, b in zip(R.layer_norm(z, keep=True), want):
        assert torch.equal(a[rest], b[rest])
    alone = R.layer_norm(far[8:9], keep=True)
    for a, b in zip(R.layer_norm(z, keep=True), alone):
        assert torch.equal(a[2], b[0]) and torch.equal(a[21], b[0])


# ---- distillation --------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [7, 50, 100, 300, 700, 800, 1300, 1800, 2791, 16389, 20003])
def test_a_score_that_is_not_finite_makes_all_of_its_row_nan(R, cuda, N, dtype):
    """Every element that takes part, whatever its exponential has become; what takes no part stays zero, and so do rows without targets."""
    torch = cuda
    low = torch.finfo(getattr(torch, dtype)).min
    for n in (6, many(torch)):
        s = make_scores(torch, 1, n, N, dtype)
        s[:, N // 2], s[:, N // 3] = low, -200.0
        mask = torch.ones(N, dtype=torch.bool, device="cuda")
        if N > 10:
            mask[5::11] = False
            s[:, 7::13] = -float("inf")
        neurons = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda").repeat(n, 1)
        targets = torch.full((n, 3), 0.25, device="cuda")
        last = n - 1
        neurons[last] = -1
        for bad in (float("inf"), float("nan")):
            for at in (1, N - 1, N // 2, 3):               # a target and others
                if not mask[at]:
                    continue
                z = s.clone()
                z[0, at] = z[n // 2, at] = z[last, at] = bad
                takes = mask & (z[0] != -float("inf"))
                for o in (dict(), dict(rest=True), dict(teacher="logits", temperature=2.0)):
                    want, wloss = R.distill_backward(None, s, neurons, targets, mask=mask, loss=True, **o)
                    d, loss = R.distill_backward(None, z, neurons, targets, mask=mask, loss=True, **o)
                    for i in (0, n // 2):
                        assert torch.isnan(loss[i]) and torch.isnan(d[i][takes]).all() and (d[i][~takes] == 0).all()
                    assert loss[last] == 0 and (d[last] == 0).all()
                    rows = [i for i in range(n) if i not in (0, n // 2, last)]
                    assert torch.equal(d[rows], want[rows]) and torch.equal(loss[rows], wloss[rows])


# chunks a thread: float32 8, 4 (a warp, a block), fewer and 16; 16 bits 8, 6, 4, 2, 1 of the ring, in one warp and in several
MANY_ROWS = [3, 100, 150, 300, 400, 800, 900, 1200, 1300, 1800, 2791, 5000, 8192, 16389, 32768]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", MANY_ROWS)
def test_distill_of_many_rows(R, cuda, N, dtype):
    torch = cuda
    n = many(torch)
    s, dloss, k = make_scores(torch, 1, n, N, dtype, holes=N > 10), rand(torch, 2, n), min(N, 9)
    check_distill(R, torch, s, *make_targets(torch, 3, n, N, k, "weights", True), dloss)
    check_distill(R, torch, s, *make_targets(torch, 4, n, N, min(N, 32), "weights", False), dloss, rest=True, temperature=2.0, scale=4.0)
    check_distill(R, torch, s, *make_targets(torch, 5, n, N, k, "logits", True), dloss, teacher="logits", temperature=0.7)
    check_distill(R, torch, s, *make_targets(torch, 6, n, N, 1, "weights", False), None, rest=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pitch", [(8, 0), (3, 1), (4, 0), (1, 2), (64, 8)], ids=str)
@pytest.mark.parametrize("N", [13, 301, 1000, 2791])
def test_distill_of_many_rows_with_pitches_masks_and_holes(R, cuda, N, pitch, dtype):
    torch = cuda
    n, k = many(torch), 6
    s, dloss = make_scores(torch, 1, n, N, dtype, holes=True), rand(torch, 2, n)
    wide = torch.arange(N + 5, device="cuda") % 7 != 3
    P = lambda t: pitched(torch, t, *pitch)                # (NaN between the rows)
    for at, mask in ((0, wide[:N]), (3, wide[3:N + 3].to(torch.uint8)), (5, None)):
        bad = s.clone()
        if mask is not None:                               # what stands in masked places does not matter
            out = torch.nonzero(mask == 0)[:, 0]
            for i, v in enumerate((float("nan"), float("inf"), -float("inf"), torch.finfo(s.dtype).max)):
                bad[:, out[i::4]] = v
        for o in (dict(rest=True), dict(), dict(teacher="logits", temperature=3.0)):
            neurons, targets = make_targets(torch, 3 + at, n, N, k, o.get("teacher", "weights"), not o.get("rest"))
            d, loss = check_distill(R, torch, bad, neurons, targets, dloss, P, mask=mask, **o)
            assert torch.isfinite(d).all() and torch.isfinite(loss).all() and (mask is None or (d[:, mask == 0] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pitch", [(8, 0), (3, 1), (4, 0), (1, 2), (64, 8)], ids=str)
@pytest.mark.parametrize("D", [140, 333, 2000, 9000])
def test_norm_of_many_rows_with_pitches_and_missing_parameters(R, cuda, D, pitch, dtype):
    torch = cuda
    n = many(torch)
    x, dy, res = (rand(torch, i, n, D, dtype=dtype) for i in (1, 2, 3))
    P = lambda t: pitched(torch, t, *pitch)
    wide = rand(torch, 4, D + 3)
    for w, b in ((None, None), (wide[1:D + 1], None), (None, wide[3:]), (wide[2:D + 2], wide[:D])):
        check_norm(R, torch, x, w, b, P)
    for w, r in ((None, res), (wide[1:D + 1], None)):
        check_norm_backward(R, torch, x, dy, w, r, P)


# ---- results that are left out, and results in an argument's place --------------------------------------------------------------

def norm_backward(R, torch, dy, x, mean, rstd, w, res, dx, ldx, dw, db):
    """The C entry on matrices with dx's own pitch."""
    from pink_b200 import capi
    n, D = x.shape
    size = capi.lib.pink_b200_layer_norm_workspace(R._TYPES[x.dtype], D, n)
    work = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    at = lambda t: None if t is None else t.data_ptr()
    capi.check(capi.lib.pink_b200_op_layer_norm_backward(R._TYPES[x.dtype], D, n, dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), mean.data_ptr(), rstd.data_ptr(),
                                                         at(w), at(res), 0 if res is None else res.stride(0), at(dx), ldx, at(dw), at(db), work.data_ptr(), size,
                                                         torch.cuda.current_stream().cuda_stream))


# eight and 32 lanes a row, through shared memory, two kernels; several rows a block, or a group of lanes
PLACES = [(40000, 30, 0), (20000, 61, 0), (10000, 200, 0), (9999, 100, 3), (1500, 2000, 0), (700, 2001, 0), (700, 2001, 7), (1500, 961, 3), (300, 9000, 0), (40, 17000, 0), (41, 17001, 2)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("place", PLACES, ids=lambda p: "%d-%d-%d" % p)
def test_norm_gradient_in_the_residuals_place(R, cuda, place, dtype):
    """dx may be the residual; and without dx the parameters' gradients are the same."""
    torch = cuda
    n, D, extra = place
    x, dy, res = (pitched(torch, rand(torch, i, n, D, dtype=dtype), extra) for i in (1, 2, 3))
    w = rand(torch, 4, D)
    _, mean, rstd = R.layer_norm(x, keep=True)
    ld = x.stride(0)
    (dx, dw, db), (dw2, db2) = (torch.empty_like(w) for _ in range(3)), (torch.empty_like(w) for _ in range(2))
    dx = torch.full((n, ld), 7.0, dtype=x.dtype, device="cuda")
    norm_backward(R, torch, dy, x, mean, rstd, w, res, dx, ld, dw, db)
    check = R.layer_norm_backward(dy, x, mean, rstd, w, residual=res)
    # (rows elsewhere may go through another kernel: a step of the result's type, and of float32 200 u of terms below 50 in either)
    assert (dx[:, D:] == 7).all()
    within(dx[:, :D], check[0].double(), torch.finfo(x.dtype).eps * check[0].double().abs() + 2 * 200 * U * 50)
    norm_backward(R, torch, dy, x, mean, rstd, w, res, res, ld, dw2, db2)
    assert torch.equal(res, dx[:, :D]) and torch.equal(dw, dw2) and torch.equal(db, db2)
    norm_backward(R, torch, dy, x, mean, rstd, w, None, None, 0, dw2, db2)
    h = (x.double() - mean[:, None].double()) * rstd[:, None].double()
    for a, b, size in ((dw2, check[1], dy.double() * h), (db2, check[2], dy.double())):
        within(a, b.double(), 2 * (n + 200) * U * (size.abs() + dy.double().abs()).sum(0))     # (in another order)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("size", [(1, 40, 24), (40, 33, 70), (300, 128, 72), (700, 1000, 333)], ids=lambda s: "%d-%d-%d" % s)
@pytest.mark.parametrize("by_input", [0, 1])
def test_gated_gradients_that_are_not_asked_for(R, cuda, size, by_input, dtype):
    """Every set of results the C entry may be asked for gives what the whole set does."""
    torch = cuda
    from pink_b200 import capi
    n, K, M = size
    x, _, _, gate, up = make_gated(torch, n, K, M, dtype, bool(by_input))
    g, u, dh = (rand(torch, i, n, M, dtype=dtype) for i in (6, 7, 8))
    want = R.gated_backward(dh, x, gate, up, g, u, by_input=bool(by_input))
    lw, cfg = gate.shape[1], capi.ProductConfig(R._TYPES[x.dtype], K, M, by_input, capi.ACT_SILU, 0, n)
    for asked in range(1, 8):
        dx = torch.zeros(n, K, dtype=x.dtype, device="cuda") if asked & 1 else None
        dgate, dup = (torch.zeros_like(gate), torch.zeros_like(up)) if asked & 2 else (None, None)
        dgb, dub = (torch.zeros(M, device="cuda"), torch.zeros(M, device="cuda")) if asked & 4 else (None, None)
        at = lambda t: None if t is None else t.data_ptr()
        args = (dh.data_ptr(), M, at(x) if asked & 2 else None, K, at(gate) if asked & 1 else None, lw, at(up) if asked & 1 else None, lw, g.data_ptr(), M, u.data_ptr(), M,
                at(dx), K, at(dgate), lw, at(dup), lw, at(dgb), at(dub))
        stream, bytes_ = torch.cuda.current_stream().cuda_stream, C.c_uint64(0)
        capi.check(capi.lib.pink_b200_op_gated_backward(cfg, *args, None, bytes_, 1, stream))
        work = torch.full((max(1, bytes_.value),), 255, dtype=torch.uint8, device="cuda")
        capi.check(capi.lib.pink_b200_op_gated_backward(cfg, *args, work.data_ptr(), bytes_, 0, stream))
        for got, whole in zip((dx, dgate, dup, dgb, dub), want):
            assert got is None or torch.equal(got, whole)


# ---- the ends of what the calls take ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
def test_norm_of_the_longest_rows(R, cuda, dtype):
    torch = cuda
    D = 1 << 24
    x, dy = rand(torch, 1, 2, D, dtype=dtype), rand(torch, 2, 2, D, dtype=dtype)
    w, b = rand(torch, 3, D), rand(torch, 4, D)
    check_norm(R, torch, x, w, b)
    check_norm_backward(R, torch, x, dy, w, None)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [40, 2791])
def test_distill_at_the_ends_of_its_options(R, cuda, N, dtype):
    """The lowest and highest temperature, all targets one neuron, weights that add up to more than 1, infinite logits."""
    torch = cuda
    for n in (5, many(torch)):
        s, dloss = make_scores(torch, 1, n, N, dtype), rand(torch, 2, n)
        routes, logits = make_targets(torch, 3, n, N, 32, "weights", True), make_targets(torch, 4, n, N, 32, "logits", True)
        for T in (0.001, 1000.0):
            check_distill(R, torch, s, *routes, dloss, temperature=T)
            check_distill(R, torch, s, routes[0], 0.7 * routes[1], dloss, temperature=T, rest=True)
            check_distill(R, torch, s, *logits, dloss, temperature=T, teacher="logits")
        check_distill(R, torch, s, routes[0], 3.0 * routes[1], dloss, rest=True)
        one = torch.arange(n, device="cuda", dtype=torch.int32)[:, None].remainder(N).repeat(1, 32)
        check_distill(R, torch, s, one, torch.full((n, 32), 1 / 64, device="cuda"), dloss, rest=True)
        check_distill(R, torch, s, one, logits[1], dloss, teacher="logits")
        far = logits[1].clone()
        far[:, 3] = far[::2, 7] = float("inf")
        far[:, 5] = float("nan")
        check_distill(R, torch, s, logits[0], far, dloss, teacher="logits", temperature=0.7)
