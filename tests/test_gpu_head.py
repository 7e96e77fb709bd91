"""Layer norm and distillation against plain implementations in 64 bits.

Tolerances: u = 2^-24 is the unit roundoff of float32; a sum of m terms, added up in chains of depth d, is off by at most d u times the
sum of their magnitudes (to first order).  The kernels' chains: a thread's elements of a row, then two times five steps across a warp and a block."""
import pytest

from test_gpu_readout import TYPES, U, half_step, make_routes, pitched, rand, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def R(cuda):
    from pink_b200 import readout
    yield readout
    readout.check_status()


def tiny_of(torch, dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


# ---- layer norm ------------------------------------------------------------------------------------------------------------

EPS = 2.0 ** -17                                           # a float32


def depth_of(D):
    """Terms in a chain: up to 32 elements of a thread (long rows: 1,024 threads), ten steps across the threads."""
    return max(32, D // 1024 + 8) + 10


def ref_norm(torch, x, w, b):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = ((d * d).mean(1, keepdim=True) + EPS) ** -0.5
    y = d * rstd
    if w is not None:
        y = y * w.double()
    if b is not None:
        y = y + b.double()
    return y, mean, rstd, d


def check_norm(R, torch, x, w, b, P=lambda t: t):
    """x - mean is off by u of itself and depth u of the row's mean |x - mean| (the mean's own rounding is taken out); rstd by
    depth + 8 u; three roundings follow, and that of the result."""
    n, D = x.shape
    y, mean, rstd = R.layer_norm(P(x), w, b, eps=EPS, keep=True)
    assert torch.equal(R.layer_norm(P(x), w, b, eps=EPS), y) and y.stride(0) % (128 // y.element_size()) == 0
    want, m, s, d = ref_norm(torch, x, w, b)
    k = depth_of(D)
    e = s * ((k + 12 + 4) * U * d.abs() + (k + 2) * U * d.abs().mean(1, keepdim=True))
    if w is not None:
        e = e * w.double().abs()
    e = e + U * want.abs()
    half = half_step(torch, x.dtype)
    within(y, want, e * (1 + half) + half * want.abs() + tiny_of(torch, x.dtype))
    within(mean, m[:, 0], (U * m.abs() + (k + 2) * U * d.abs().mean(1, keepdim=True))[:, 0] + 2.0 ** -149)
    within(rstd, s[:, 0], (k + 8) * U * s[:, 0])
    return mean, rstd


def check_norm_backward(R, torch, x, dy, w, res, P=lambda t: t):
    """Of h: u of itself from each of three roundings, depth u from its mean, depth + 8 u of itself from rstd; of the means depth u of
    those of magnitudes and what h brings; so K = 3 depth + 40 covers the factors below.  Columns: a chain of at most n terms."""
    n, D = x.shape
    _, mean, rstd = R.layer_norm(x, eps=EPS, keep=True)
    dx, dw, db = R.layer_norm_backward(P(dy), P(x), mean, rstd, w, residual=None if res is None else P(res))
    _, _, s, d = ref_norm(torch, x, None, None)
    h, g0 = d * s, dy.double()
    g = g0 if w is None else g0 * w.double()
    c2 = (g * h).mean(1, keepdim=True)
    want = s * (g - g.mean(1, keepdim=True) - h * c2)
    K, mg = 3 * depth_of(D) + 40, g.abs().mean(1, keepdim=True)
    mgh = (g * h).abs().mean(1, keepdim=True)
    e = K * U * s * (g.abs() + mg + (h.abs() + 1) * (mgh + mg))
    if res is not None:
        want = want + res.double()
        e = e + U * want.abs()
    half = half_step(torch, x.dtype)
    within(dx, want, e * (1 + half) + half * want.abs() + tiny_of(torch, x.dtype))
    eh = (depth_of(D) + 12) * U * (h.abs() + 1)
    within(dw, (g0 * h).sum(0), (n + 12) * U * (g0 * h).abs().sum(0) + (g0.abs() * eh).sum(0))
    within(db, g0.sum(0), (n + 12) * U * g0.abs().sum(0))
    only, none, nothing = R.layer_norm_backward(P(dy), P(x), mean, rstd, w, residual=None if res is None else P(res), parameters=False)
    assert torch.equal(only, dx) and none is None and nothing is None
    again = R.layer_norm_backward(P(dy), P(x), mean, rstd, w, residual=None if res is None else P(res))
    assert all(torch.equal(a, b) for a, b in zip(again, (dx, dw, db)))


# a row per eight lanes, per warp, per block of every size, of the last registers, and beyond them
NORM_SIZES = [(1, 1), (3, 2), (5, 7), (70, 8), (33, 33), (40, 64), (300, 65), (9, 255), (17, 256), (2, 257), (7, 512), (5, 513), (11, 961), (3, 1024), (4, 1025), (3, 2791),
              (2, 4097), (5, 8100), (3, 8192), (2, 8193), (2, 16383), (3, 16384), (2, 16385), (1, 40001), (700, 17), (2000, 131), (20, 8201), (4097, 1100), (4099, 2791), (1000, 961), (1300, 300), (1250, 1029), (1200, 8200), (1190, 14001)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", NORM_SIZES, ids=lambda s: "%d-%d" % s)
def test_norm_sizes(R, cuda, size, dtype):
    torch = cuda
    n, D = size
    x, dy, res = (rand(torch, i, n, D, dtype=dtype) for i in (1, 2, 3))
    w, b = rand(torch, 4, D), rand(torch, 5, D)
    check_norm(R, torch, x, w, b)
    check_norm_backward(R, torch, x, dy, w, res if D % 2 else None)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pitch", [(8, 0), (3, 1), (4, 0), (1, 2), (64, 8)], ids=str)
@pytest.mark.parametrize("D", [5, 100, 333, 2000, 9000])
def test_norm_pitches_and_missing_parameters(R, cuda, D, pitch, dtype):
    torch = cuda
    x, dy, res = (rand(torch, i, 7, D, dtype=dtype) for i in (1, 2, 3))
    P = lambda t: pitched(torch, t, *pitch)                # (NaN between the rows)
    wide = rand(torch, 4, D + 3)
    for w, b in ((None, None), (wide[1:D + 1], None), (None, wide[3:]), (wide[2:D + 2], wide[:D])):
        check_norm(R, torch, x, w, b, P)
    for w in (None, wide[1:D + 1]):
        check_norm_backward(R, torch, x, dy, w, res, P)
        check_norm_backward(R, torch, x, dy, w, None, P)


@pytest.mark.parametrize("D", [50, 300, 3000, 20000])
@pytest.mark.parametrize("offset,scale", [(1e4, 1.0), (-3e5, 2.0), (0.0, 1e-6), (1.0, 0.0), (0.0, 1e15)])
def test_norm_of_rows_far_from_zero_and_of_all_sizes(R, cuda, D, offset, scale):
    """What the row's mean loses to rounding does not show; rows without spread are the bias."""
    torch = cuda
    x = offset + rand(torch, 1, 9, D, scale=scale)
    check_norm(R, torch, x, rand(torch, 2, D), rand(torch, 3, D))
    check_norm_backward(R, torch, x, rand(torch, 4, 9, D), rand(torch, 2, D), None)


def test_norm_keeps_what_is_not_finite_in_its_row(R, cuda):
    torch = cuda
    for D in (40, 300, 2791, 17000):
        x, dy = rand(torch, 1, 8, D), rand(torch, 2, 8, D)
        y, mean, rstd = R.layer_norm(x, keep=True)
        dx, _, _ = R.layer_norm_backward(dy, x, mean, rstd)
        for bad in (float("inf"), float("nan")):
            z = x.clone()
            z[3, D // 2] = bad
            got, m, s = R.layer_norm(z, keep=True)
            rows = torch.arange(8) != 3
            assert torch.isnan(got[3]).all() and torch.equal(got[rows], y[rows]) and torch.equal(m[rows], mean[rows])
            gx, gw, gb = R.layer_norm_backward(dy, z, m, s)
            assert torch.isnan(gx[3]).all() and torch.equal(gx[rows], dx[rows]) and torch.isfinite(gb).all()


def test_norm_of_nothing_and_of_rows_behind_the_last(R, cuda):
    torch = cuda
    x = torch.empty(0, 12, device="cuda")
    y, mean, rstd = R.layer_norm(x, keep=True)
    assert y.shape == (0, 12) and mean.shape == (0,)
    dx, dw, db = R.layer_norm_backward(x, x, mean, rstd)
    assert dx.shape == (0, 12) and (dw == 0).all() and (db == 0).all()
    # the C entry writes n rows of dims elements and nothing else
    from pink_b200 import capi
    for dtype in (torch.float32, torch.bfloat16):
        x = rand(torch, 1, 6, 50).to(dtype)
        out = torch.full((6, 57), 7.0, dtype=dtype, device="cuda")
        capi.check(capi.lib.pink_b200_op_layer_norm(R._TYPES[dtype], 50, 4, x.data_ptr(), 50, None, None, 1e-5, out.data_ptr(), 57, None, None, None))
        assert (out[4:] == 7).all() and (out[:, 50:] == 7).all() and torch.equal(out[:4, :50], R.layer_norm(x)[:4])


def test_norm_gradient_against_differences(R, cuda):
    """Directional differences of sum(y dy), step h = 2^-6 in the forward call itself: its results are off by less than 2^-20 each, so
    the quotient by 64 terms * 2^-20 * 2^6 / 2 at most, and by h^2 / 6 of a third derivative (below 30 for rows of this spread)."""
    torch = cuda
    x, dy, v = rand(torch, 1, 4, 64), rand(torch, 2, 4, 64), rand(torch, 3, 4, 64)
    v = v / v.norm()
    w = 1 + 0.1 * rand(torch, 4, 64)
    _, mean, rstd = R.layer_norm(x, w, keep=True)
    dx, _, _ = R.layer_norm_backward(dy, x, mean, rstd, w)
    h = 2.0 ** -6
    f = lambda t: (R.layer_norm(t, w).double() * dy.double()).sum()
    assert abs((f(x + h * v) - f(x - h * v)) / (2 * h) - (dx.double() * v.double()).sum()) <= 64 * 2.0 ** -20 * 2 ** 5 + 30 * h * h / 6


# ---- distillation ------------------------------------------------------------------------------------------------------------

def ref_distill(torch, scores, neurons, targets, dloss, teacher="weights", temperature=1.0, scale=1.0, rest=False, mask=None):
    """Losses and gradients from the definition, with bounds of what float32 loses: every exponential is off by 3 u of its exponent in each
    of two steps and 4 u in each; sums have chains of at most 60 terms; the combinations behind them take fewer than 30 roundings."""
    s = scores.double()
    n, N = s.shape
    T = torch.tensor(temperature, dtype=torch.float32).double().item()
    takes = s != -float("inf")
    if mask is not None:
        takes = takes & mask.bool()
    l = torch.where(takes, s / T, -float("inf"))
    M = l.amax(1, keepdim=True)
    M0 = torch.where(M == -float("inf"), 0.0, M)
    e = torch.exp(l - M0)
    S = e.sum(1, keepdim=True)
    q = torch.nan_to_num(e / S, nan=0.0) if not torch.isnan(s[takes]).any() else e / S
    span = torch.where(takes, M0 - l, 0.0)
    eS = U * (6 * (q * span).sum(1, keepdim=True) + 80)    # relative, of S; the terms' own errors average with their share
    idx = neurons.long()
    inside = (idx >= 0) & (idx < N)
    idx = torch.where(inside, idx, 0)
    there = inside & takes.gather(1, idx)
    if teacher == "weights":
        there = there & (targets > 0)
        p = torch.where(there, targets.double(), 0.0)
        ep = torch.zeros_like(p)
    else:
        there = there & (targets > -float("inf"))
        t = torch.where(there, targets.double().clamp(max=3.4028234663852886e38) / T, -float("inf"))
        high = t.amax(1, keepdim=True)
        high = torch.where(high == -float("inf"), 0.0, high)
        p = torch.exp(t - high)
        p = torch.where(there, p / p.sum(1, keepdim=True), 0.0)
        far = torch.where(there, high - t, 0.0)
        ep = p * U * (3 * far + 3 * (p * far).sum(1, keepdim=True) + 24)
    lq = torch.where(there, (l - M0).gather(1, idx) - torch.log(S), 0.0)
    lp = torch.where(p > 0, torch.log(torch.where(p > 0, p, 1.0)), 0.0)
    loss = torch.where(p > 0, p * (lp - lq), 0.0).sum(1)
    spans = torch.where(there, span.gather(1, idx), 0.0)
    bound = (p * (U * (4 * lp.abs() + 4 * spans + 4 * torch.log(S).abs() + 12) + eS) + ep * (lp.abs() + lq.abs() + 1)).sum(1) + 40 * U * loss.abs()
    listed = torch.zeros(n, N + 1, device="cuda", dtype=torch.float64).scatter_add_(1, torch.where(there, idx, N), p)[:, :N]
    hit = torch.zeros(n, N + 1, device="cuda", dtype=torch.bool).scatter_(1, torch.where(there, idx, N), True)[:, :N]
    mass = p.sum(1, keepdim=True)
    r = torch.zeros_like(mass)
    qr = torch.zeros_like(q)
    if rest:
        other = takes & ~hit
        lo = torch.where(other, l, -float("inf"))
        Mo = lo.amax(1, keepdim=True)
        some = Mo != -float("inf")
        Mo = torch.where(some, Mo, 0.0)
        So = torch.where(some, torch.exp(lo - Mo).sum(1, keepdim=True), 1.0)
        r = torch.where(some, (1 - mass).clamp(min=0), 0.0)
        lr = Mo - M0 + torch.log(So) - torch.log(S)
        qr = torch.where(other, torch.exp(lo - Mo) / So, 0.0)
        logr = torch.log(torch.where(r > 0, r, 1.0))
        apart = (M0 - Mo).abs() + torch.where(hit, (M0 - l).nan_to_num(posinf=0.0), 0.0).amax(1, keepdim=True)
        loss = loss + torch.where(r > 0, r * (logr - lr), 0.0)[:, 0]
        eo = U * (6 * (qr * torch.where(other, Mo - l, 0.0)).sum(1, keepdim=True) + 80)
        # (the quotient's own error, its float32 r and sum of p, and the logarithms')
        bound = bound + (r * (eS + eo + U * (12 * apart + 60 + 4 * logr.abs() + 4 * lr.abs())))[:, 0] + 4 * U
    row = there.any(1)
    by = (dloss.double() * scale / T)[:, None]
    d = by * (q * (mass + r) - listed - r * qr)
    eq = q * (U * (12 * span + 40) + eS)
    eqr = r * qr * U * 200 + r * qr * U * 12 * torch.where(takes, span, 0.0) if rest else 0.0
    ed = by.abs() * (eq * (mass + r) + 10 * U * (q * (mass + r) + listed) + eqr
                     + torch.zeros(n, N + 1, device="cuda", dtype=torch.float64).scatter_add_(1, torch.where(there, idx, N), ep)[:, :N] + 2.0 ** -120)
    zero = torch.zeros(())
    return (torch.where(row, scale * loss, 0.0), scale * bound, torch.where(takes & row[:, None], d, 0.0), ed)


def make_scores(torch, seed, n, N, dtype, holes=False):
    v = rand(torch, seed, n, N, scale=3.0)
    if holes:
        r = torch.rand((n, N), generator=torch.Generator(device="cuda").manual_seed(seed + 1), device="cuda")
        v[r < 0.1] = -float("inf")
        v[(r > 0.1) & (r < 0.15)] = -60.0
    return v.to(getattr(torch, dtype))


def make_targets(torch, seed, n, N, k, teacher, whole):
    """Neurons (in test_gpu_readout's manner: twice, absent, beyond the table) with weights or logits, some of which leave their target out."""
    neurons, t = make_routes(torch, seed, n, N, k)
    if teacher == "logits":
        t = 3 * t
        t[torch.rand(n, k, generator=torch.Generator(device="cuda").manual_seed(seed + 1), device="cuda") < 0.05] = -float("inf")
        return neurons, t
    w = torch.softmax(t, 1) * (1.0 if whole else 0.8)
    w[torch.rand(n, k, generator=torch.Generator(device="cuda").manual_seed(seed + 1), device="cuda") < 0.05] = 0.0
    return neurons, w


def check_distill(R, torch, scores, neurons, targets, dloss=None, P=lambda t: t, **o):
    n, N = scores.shape
    g = torch.ones(n, device="cuda") if dloss is None else dloss
    want, bound, dwant, dbound = ref_distill(torch, scores, neurons, targets, g, **o)
    half, tiny = half_step(torch, scores.dtype), tiny_of(torch, scores.dtype)
    got = R.distill(P(scores), neurons, targets, **o)
    within(got, want, bound + 2.0 ** -126)
    d, loss = R.distill_backward(dloss, P(scores), neurons, targets, loss=True, **o)
    assert torch.equal(loss, got) and torch.equal(R.distill_backward(dloss, P(scores), neurons, targets, **o), d)
    assert d.shape == scores.shape and d.dtype == scores.dtype
    within(d, dwant, dbound * (1 + half) + half * dwant.abs() + tiny)
    return d, loss


DISTILL_SIZES = [(1, 1, 1), (3, 2, 2), (9, 5, 3), (4, 32, 32), (17, 33, 4), (5, 255, 8), (8, 256, 8), (9, 257, 8), (3, 400, 32), (6, 512, 5), (7, 513, 5), (3, 1000, 17), (260, 961, 6),
                 (4, 2791, 8), (3, 4097, 3), (2, 8192, 32), (2, 16384, 9), (2, 16385, 9), (2, 32768, 32), (1030, 1500, 4), (1027, 2791, 8), (1025, 5000, 16), (1024, 17000, 3), (1100, 77, 5), (1024, 900, 8), (2, 16391, 4), (2, 20003, 4), (1050, 3333, 4), (2, 1100, 4), (1, 7, 7), (1033, 16389, 32)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", DISTILL_SIZES, ids=lambda s: "%d-%d-%d" % s)
def test_distill_sizes(R, cuda, size, dtype):
    torch = cuda
    n, N, k = size
    s, dloss = make_scores(torch, 1, n, N, dtype), rand(torch, 2, n)
    check_distill(R, torch, s, *make_targets(torch, 3, n, N, k, "weights", True), dloss)
    check_distill(R, torch, s, *make_targets(torch, 4, n, N, k, "weights", False), dloss, rest=True, temperature=2.0, scale=4.0)
    check_distill(R, torch, s, *make_targets(torch, 5, n, N, k, "logits", True), None, teacher="logits", temperature=0.7)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pitch", [(8, 0), (3, 1), (4, 0), (1, 2), (64, 8)], ids=str)
@pytest.mark.parametrize("N", [40, 301, 1000, 2791])
def test_distill_pitches_masks_and_holes(R, cuda, N, pitch, dtype):
    torch = cuda
    n, k = 12, 6
    s, dloss = make_scores(torch, 1, n, N, dtype, holes=True), rand(torch, 2, n)
    wide = torch.arange(N + 5, device="cuda") % 7 != 3
    P = lambda t: pitched(torch, t, *pitch)
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
@pytest.mark.parametrize("N", [20, 300, 700, 2791, 20000])
def test_distill_rows_that_are_left_out(R, cuda, N, dtype):
    """Without targets a row has neither loss nor gradient, whatever its scores; a row whose neurons all are left out neither."""
    torch = cuda
    s = make_scores(torch, 1, 6, N, dtype)
    neurons, targets = torch.arange(3, device="cuda", dtype=torch.int32).repeat(6, 1), torch.full((6, 3), 0.25, device="cuda")
    want, wloss = R.distill_backward(None, s, neurons, targets, loss=True, rest=True)
    neurons[1], targets[2], s[3], s[4, :3] = -1, 0.0, -float("inf"), -float("inf")
    s[1] = float("nan")
    d, loss = R.distill_backward(None, s, neurons, targets, loss=True, rest=True)
    assert (d[1:5] == 0).all() and (loss[1:5] == 0).all()
    for i in (0, 5):
        assert torch.equal(d[i], want[i]) and loss[i] == wloss[i] and loss[i] != 0
    d, loss = R.distill_backward(None, s, neurons, targets, loss=True, mask=torch.zeros(N, dtype=torch.bool, device="cuda"))
    assert (d == 0).all() and (loss == 0).all()
    # a NaN or +infinity of a neuron that takes part shows
    for bad in (float("nan"), float("inf")):
        s[0, N - 1] = bad
        d, loss = R.distill_backward(None, s, neurons, targets, loss=True)
        assert torch.isnan(loss[0]) and torch.isnan(d[0, :3]).any() and torch.isfinite(loss[5]) and torch.isfinite(d[5]).all()
        s[0, N - 1], s[0, 1] = 0.0, bad                    # of a target too
        d, loss = R.distill_backward(None, s, neurons, targets, loss=True)
        assert torch.isnan(loss[0]) and torch.isnan(d[0]).any()
        s[0, 1] = 0.0


def test_distill_of_extreme_scores(R, cuda):
    """Scores of the type's lowest value take part: alone they share evenly.  Scores far above all others, and targets far below them."""
    torch = cuda
    for N in (50, 400, 2791):
        for dtype in TYPES:
            low = torch.finfo(getattr(torch, dtype)).min
            s = make_scores(torch, 1, 4, N, dtype)
            s[0] = low
            s[1, 5:] = low
            s[2, 7] = 300.0
            s[3, :4] = -200.0
            neurons, targets = torch.tensor([[0, 1, 2, 3]] * 4, device="cuda", dtype=torch.int32), torch.tensor([[0.5, 0.25, 0.125, 0.0625]] * 4, device="cuda")
            for o in (dict(), dict(rest=True)):
                # (the bound of an exponent is u of the difference: of these it is what counts)
                check_distill(R, torch, s, neurons, targets, None, **o)


def test_distill_agrees_with_routes(R, cuda):
    """Scores that are the mapping's own logits: no divergence, and next to no gradient, with the routes' weights, renormalised or not."""
    torch = cuda
    d = rand(torch, 1, 50, 961).abs() * 4
    neurons, weights = R.route(d, 8, slope=-2.0, renormalise=False)
    g, loss = R.distill_backward(None, -2.0 * d, neurons, weights, loss=True, rest=True)
    assert loss.abs().max() <= 200 * U and g.abs().max() <= 200 * U
    few = torch.full_like(d, -float("inf")).scatter(1, neurons.long(), (-2.0 * d).gather(1, neurons.long()))
    neurons, weights = R.route(d, 8, slope=-2.0)
    for t, kw in ((weights, {}), ((-2.0 * d).gather(1, neurons.long()), dict(teacher="logits"))):
        g, loss = R.distill_backward(None, few, neurons, t, loss=True, **kw)
        assert loss.abs().max() <= 200 * U and g.abs().max() <= 200 * U


def test_distill_gradient_against_differences(R, cuda):
    """Directional differences of the summed losses in the forward call, step h = 2^-5 along a unit vector: losses are off by less than 2^-19 each, so
    the quotient by 6 * 2^-19 * 2^5 / 2 * 2, and by h^2 / 6 of a third derivative (below 4: cumulants of a bounded direction)."""
    torch = cuda
    s, v = make_scores(torch, 1, 6, 90, "float32"), rand(torch, 2, 6, 90)
    v = v / v.norm()
    for o in (dict(), dict(rest=True), dict(teacher="logits", temperature=2.0)):
        neurons, targets = make_targets(torch, 3, 6, 90, 7, o.get("teacher", "weights"), not o.get("rest"))
        d = R.distill_backward(None, s, neurons, targets, **o)
        h = 2.0 ** -5
        f = lambda t: R.distill(t, neurons, targets, **o).double().sum()
        assert abs((f(s + h * v) - f(s - h * v)) / (2 * h) - (d.double() * v.double()).sum()) <= 6 * 2.0 ** -19 * 2 ** 5 + 4 * h * h / 6


def test_distill_of_nothing_and_of_rows_behind_the_last(R, cuda):
    torch = cuda
    neurons = torch.empty(0, 4, dtype=torch.int32, device="cuda")
    assert R.distill(torch.empty(0, 12, device="cuda"), neurons, torch.empty(0, 4, device="cuda")).shape == (0,)
    assert R.distill_backward(None, torch.empty(0, 12, device="cuda"), neurons, torch.empty(0, 4, device="cuda")).shape == (0, 12)
    from pink_b200 import capi
    for dtype in (torch.float32, torch.float16):
        for N in (50, 600):
            s = make_scores(torch, 1, 6, N, "float32").to(dtype)
            neurons, targets = make_targets(torch, 3, 6, N, 4, "weights", True)
            out, loss = torch.full((6, N + 7), 7.0, dtype=dtype, device="cuda"), torch.full((6,), 7.0, device="cuda")
            cfg = capi.DistillConfig(N, 4, 0, 0, 1.0, 1.0)
            capi.check(capi.lib.pink_b200_op_distill_backward(cfg, 4, R._TYPES[dtype], s.data_ptr(), N, None, neurons.data_ptr(), targets.data_ptr(), None, out.data_ptr(), N + 7,
                                                              loss.data_ptr(), None))
            assert (out[4:] == 7).all() and (out[:, N:] == 7).all() and (loss[4:] == 7).all()
            assert torch.equal(out[:4, :N], R.distill_backward(None, s, neurons, targets)[:4])


# ---- what the sizes above do not reach ------------------------------------------------------------------------------------------

def test_offsets_beyond_32_bits(R, cuda):
    """Rows 2^22 elements apart, 1,200 of them: the last begins behind element 2^32.  The same results as of rows side by side."""
    torch = cuda
    n, D, far = 1200, 301, 1 << 22
    big = torch.empty(n * far, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(big, (n, D), (far, 1), 5)
    x.copy_(rand(torch, 1, n, D))
    near, dy = x.contiguous(), rand(torch, 2, n, D, dtype="bfloat16")
    want = R.layer_norm(near, keep=True)
    assert all(torch.equal(a, b) for a, b in zip(R.layer_norm(x, keep=True), want))
    for a, b in zip(R.layer_norm_backward(dy, x, *want[1:]), R.layer_norm_backward(dy, near, *want[1:])):
        assert torch.equal(a, b)
    assert torch.equal(R.layer_norm_backward(x, near, *want[1:])[0], R.layer_norm_backward(near, near, *want[1:])[0])
    neurons, targets = make_targets(torch, 3, n, D, 4, "weights", True)
    for m in (n, 50):
        for a, b in zip(R.distill_backward(None, x[-m:], neurons[-m:], targets[-m:], loss=True), R.distill_backward(None, near[-m:], neurons[-m:], targets[-m:], loss=True)):
            assert torch.equal(a, b)
    gate, up = rand(torch, 4, 40, D, dtype="bfloat16"), rand(torch, 5, 40, D, dtype="bfloat16")
    assert torch.equal(R.gated(x, gate, up), R.gated(near, gate, up)) and torch.equal(R.gated(x[-3:], gate, up), R.gated(near[-3:], gate, up))


@pytest.mark.parametrize("dtype", TYPES)
def test_many_rows_give_what_few_give(R, cuda, dtype):
    """Rows do not depend on those beside them, nor -- the choice of neurons, ties and NaN among the scores aside -- on how many there are."""
    torch = cuda
    for D in (40, 700, 2791, 6000):
        x = rand(torch, 1, 1300, D, dtype=dtype)
        x[7], x[1299] = float("nan"), 0.5
        y, mean, rstd = R.layer_norm(x, keep=True)
        half = half_step(torch, x.dtype)
        few, m, s = R.layer_norm(x[1290:], keep=True)
        within(y[1290:].float(), few.double(), 2 * half * few.double().abs() + 40 * U)
        assert torch.isnan(y[7]).all() and torch.isfinite(y[8:]).all() and (y[1299] == 0).all()
        neurons, targets = make_targets(torch, 3, 1300, D, 5, "weights", True)
        d, loss = R.distill_backward(None, x, neurons, targets, loss=True)
        few, l = R.distill_backward(None, x[1290:], neurons[1290:], targets[1290:], loss=True)
        within(loss[1290:], l.double(), 200 * U * (l.double().abs() + 10))
        within(d[1290:], few.double(), 2 * half * few.double().abs() + 200 * U)
        rows = torch.arange(1300, device="cuda") != 7
        assert torch.isfinite(d[rows]).all() and (torch.isnan(loss[7]) or (targets[7] <= 0).all())


def test_two_threads_with_rows_of_different_sizes(R, cuda):
    """Calls from two threads at once, whose kernels need different amounts of shared memory."""
    import threading
    torch = cuda
    wrong = []

    def work(D):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                x, dy = rand(torch, D, 1200, D, dtype="bfloat16"), rand(torch, D + 1, 1200, D, dtype="bfloat16")
                neurons, targets = make_targets(torch, 3, 1200, D, 4, "weights", True)
                want = None
                for _ in range(150):
                    y, mean, rstd = R.layer_norm(x, keep=True)
                    got = (y,) + R.layer_norm_backward(dy, x, mean, rstd) + R.distill_backward(None, x, neurons, targets, loss=True)
                    want = want or got
                stream.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(got, want))
        except Exception as err:                           # (an assertion in a thread would be lost)
            wrong.append(err)
    threads = [threading.Thread(target=work, args=(D,)) for D in (6000, 8100, 5001)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong


def test_a_result_without_a_graph_is_announced(R, cuda):
    torch = cuda
    import warnings
    x, w = rand(torch, 1, 9, 16), rand(torch, 2, 16)
    h, g = rand(torch, 3, 9, 16, dtype="bfloat16"), rand(torch, 4, 8, 16, dtype="bfloat16")
    neurons, targets = torch.zeros(9, 2, dtype=torch.int32, device="cuda"), torch.full((9, 2), 0.5, device="cuda")
    calls = [(lambda t: R.layer_norm(t), x), (lambda t: R.layer_norm(x, t), w), (lambda t: R.layer_norm(x, None, t), w), (lambda t: R.gated(t, g, g), h), (lambda t: R.gated(h, t, g), g),
             (lambda t: R.gated(h, g, t), g), (lambda t: R.distill(t, neurons, targets), x), (lambda t: R.distill(x, neurons, t), targets)]
    for call, t in calls:
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            want = call(t)
        with pytest.warns(UserWarning, match="no part in autograd"):
            got = call(t.clone().requires_grad_())
        assert torch.equal(got, want) and not got.requires_grad


def test_front_end_refuses_what_does_not_fit(R, cuda):
    torch = cuda
    x, v = rand(torch, 1, 6, 16), rand(torch, 2, 16)
    h, g = rand(torch, 3, 6, 16, dtype="bfloat16"), rand(torch, 4, 8, 16, dtype="bfloat16")
    neurons, targets = torch.zeros(6, 2, dtype=torch.int32, device="cuda"), torch.full((6, 2), 0.5, device="cuda")
    from pink_b200.capi import PinkError
    for call, error in ((lambda: R.layer_norm(x, v[:15]), ValueError), (lambda: R.layer_norm(x, v.half()), TypeError), (lambda: R.layer_norm(x, eps=0.0), PinkError),
                        (lambda: R.layer_norm(x.t()), ValueError), (lambda: R.layer_norm(x.double()), TypeError), (lambda: R.layer_norm(x[:, :0]), PinkError),
                        (lambda: R.layer_norm_backward(x, x, v[:5], v[:6]), ValueError), (lambda: R.layer_norm_backward(h, x, v[:6], v[:6]), TypeError),
                        (lambda: R.gated(x, x, x), TypeError), (lambda: R.gated(h, g, g[:7]), ValueError), (lambda: R.gated(h, g, g.half()), TypeError),
                        (lambda: R.gated(h, g, g, activation="tanh"), ValueError), (lambda: R.gated(h, g, g, gate_bias=v), ValueError), (lambda: R.gated(h, g, g, by_input=True), ValueError),
                        (lambda: R.gated_backward(h, h, g, g, h, h), ValueError), (lambda: R.distill(x, neurons.long(), targets), TypeError),
                        (lambda: R.distill(x, neurons, targets[:5]), ValueError), (lambda: R.distill(x, neurons, targets, teacher="labels"), ValueError),
                        (lambda: R.distill(x, neurons, targets, teacher="logits", rest=True), PinkError), (lambda: R.distill(x, neurons, targets, temperature=0.0), PinkError),
                        (lambda: R.distill(x, neurons, targets, mask=torch.ones(15, dtype=torch.bool, device="cuda")), ValueError),
                        (lambda: R.distill_backward(v, x, neurons, targets), ValueError), (lambda: R.distill(x, neurons.cpu(), targets), ValueError)):
        with pytest.raises(error):
            call()
