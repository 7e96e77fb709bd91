"""Mapping with routes and a read-out: the library's own calls of the read-out operators, against the distances that mapping returns
and the definitions in 64 bits."""
import subprocess

import numpy as np
import pytest

from pink_b200 import build as B
from pink_b200 import files
from pink_b200.synthetic import blob_images, mt19937_uniform

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def make(n=150, idim=16, nd=12, ed=7, R=8, N=9, mode=2, seed=5):
    """Images for more than two internal batches, a map, and their engine's arguments."""
    imgs = blob_images(n, idim, 1, seed=seed).reshape(n, 1, idim, idim)
    som = mt19937_uniform(N * nd * nd, seed + 1).reshape(N, 1, nd, nd)
    return imgs, som, (N, 1, idim, nd, ed, R, True, mode)


def reference(dist, k, slope, bias=None, mask=None, score="softmax"):
    """Routes from distances: the choice in float32 as defined, the weights in 64 bits."""
    l = (dist * np.float32(slope)).astype(np.float32)
    c = l if bias is None else (l + bias[None].astype(np.float32)).astype(np.float32)
    if mask is not None:
        c = np.where(mask[None], c, -np.inf)
    n, N = dist.shape
    neurons = np.full((n, k), 0xFFFFFFFF, np.uint32)
    weights = np.zeros((n, k))
    for i in range(n):
        order = sorted((j for j in range(N) if c[i, j] != -np.inf), key=lambda j: (-float(c[i, j]), j))[:k]
        neurons[i, :len(order)] = order
        if order:
            a = l[i, order].astype(np.float64)
            logp = a if score == "softmax" else -np.logaddexp(0, -a)
            e = np.exp(logp - logp.max())
            weights[i, :len(order)] = e / e.sum()
    return neurons, weights


# |l - max| units of 2^-24 in a term and in the sum, four of each of two exponentials, 32 of the sum, six roundings around them
def weight_bound(dist, slope):
    return U * (2 * float(np.ptp(dist)) * abs(slope) + 8 + 32 + 6)


@pytest.mark.parametrize("mode", [0, 1, 2])
def test_map_routes_follows_from_the_distances(cuda, mode):
    from pink_b200 import capi, engine
    imgs, som, args = make(mode=mode)
    N, k = args[0], 4
    values = mt19937_uniform(N * 6, 3).reshape(N, 2, 3)
    with engine.Engine(*args) as e:
        e.set_som(som)
        dist, rot = e.map(imgs)
        before = e.launch_count()
        plain = e.map_routes(imgs, k, distances=True)
        assert e.launch_count() > before and "values" not in plain
        assert np.array_equal(plain["dist"], dist) and np.array_equal(plain["rot"], rot)
        for score, name in ((capi.SCORE_SOFTMAX, "softmax"), (capi.SCORE_SIGMOID, "sigmoid")):
            e.set_values(values)
            got = e.map_routes(imgs, k, score=score, slope=-2.5)
            neurons, weights = reference(dist, k, -2.5, score=name)
            assert np.array_equal(got["neurons"], neurons)
            assert np.abs(got["weights"] - weights).max() <= weight_bound(dist, -2.5)
            assert np.array_equal(got["rotations"], np.take_along_axis(rot, neurons.astype(np.int64), 1))
            # the read-out of the weights that came back: k products and sums
            want = np.einsum("nk,nkab->nab", got["weights"].astype(np.float64), values[neurons].astype(np.float64))
            size = np.einsum("nk,nkab->nab", got["weights"].astype(np.float64), np.abs(values[neurons]).astype(np.float64))
            assert got["values"].shape == (len(imgs), 2, 3)
            assert (np.abs(got["values"] - want) <= size * (k + 1) * U).all()
        e.set_values(None)
        assert "values" not in e.map_routes(imgs[:3], k)
        # one image, several calls, another top_k
        for kk in (1, N):
            got = e.map_routes(imgs[:1], kk)
            assert np.array_equal(got["neurons"], reference(dist[:1], kk, -1.0)[0])


def test_map_routes_with_bias_mask_and_groups(cuda):
    from pink_b200 import engine
    imgs, som, args = make()
    N = args[0]
    bias = np.linspace(-1, 1, N).astype(np.float32)
    mask = np.arange(N) % 4 != 1
    with engine.Engine(*args) as e:
        e.set_som(som)
        dist, rot = e.map(imgs)
        got = e.map_routes(imgs, 8, bias=bias, mask=mask)
        neurons, weights = reference(dist, 8, -1.0, bias, mask)
        assert np.array_equal(got["neurons"], neurons) and np.abs(got["weights"] - weights).max() <= weight_bound(dist, -1.0)
        gone = neurons == 0xFFFFFFFF                       # seven neurons are left
        assert gone[:, 7].all() and (got["rotations"][gone] == 0xFFFFFFFF).all() and (got["weights"][gone] == 0).all()
        got = e.map_routes(imgs, 3, groups=3, top_groups=1)
        rows = got["neurons"] // 3                         # all from the row of the map that holds the best neuron
        assert (rows == rows[:, :1]).all() and np.array_equal(got["neurons"][:, 0], dist.argmin(1))


def test_dense_read_out_of_a_map(cuda):
    """Scores and values enter rounded to bfloat16 (half a step 2^-9 ... 2^-8 relative each), the result leaves so."""
    from pink_b200 import engine
    for D in (5, 64, 300):
        imgs, som, args = make(n=70)
        N = args[0]
        values = mt19937_uniform(N * D, 4).reshape(N, D)
        with engine.Engine(*args) as e:
            e.set_som(som)
            dist, _ = e.map(imgs)
            e.set_values(values, dense=True)
            got = e.map_routes(imgs, 2, slope=-2.0)["values"]
            a = -2.0 * dist.astype(np.float64)
            p = np.exp(a - a.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            half = 2.0 ** -8
            want, size = p @ values.astype(np.float64), p @ np.abs(values).astype(np.float64)
            assert (np.abs(got - want) <= size * (2 * half + half * half + weight_bound(dist, -2.0) * 2 + (N + 2) * 2 * U) * (1 + half) + half * np.abs(want)).all()
            small = e.map_routes(imgs[:3], 2, slope=-2.0)["values"]          # another variant of the product: another order of the same sums
            assert (np.abs(small - want[:3]) <= size[:3] * 3 * half + half * np.abs(want[:3])).all()


def test_group_maps_routes(cuda):
    from pink_b200 import engine
    imgs, som, args = make()
    values = mt19937_uniform(args[0] * 4, 3).reshape(args[0], 4)
    with engine.Engine(*args) as e, engine.Group(*args) as g:
        for x in (e, g):
            x.set_som(som)
            x.set_values(values)
        a, b = e.map_routes(imgs, 3, distances=True), g.map_routes(imgs, 3, distances=True)
        assert sorted(a) == sorted(b) and all(np.array_equal(a[key], b[key]) for key in a)
        g.set_values(None)
        assert "values" not in g.map_routes(imgs, 3)
        assert np.array_equal(g.map(imgs)[0], a["dist"])   # plain mapping as before


def test_map_routes_refusals(cuda):
    from pink_b200 import capi, engine
    imgs, som, args = make(n=4)
    with engine.Engine(*args) as e:
        with pytest.raises(capi.PinkError) as err:
            e.map_routes(imgs, 2)
        assert err.value.code == capi.ESTATE
        e.set_som(som)
        for bad in (dict(top_k=10), dict(top_k=0), dict(top_k=2, groups=2), dict(top_k=2, scale=0.0), dict(top_k=2, score=7)):
            with pytest.raises(capi.PinkError) as err:
                e.map_routes(imgs, **bad)
            assert err.value.code == capi.EINVAL
        with pytest.raises(ValueError):
            e.set_values(np.zeros((8, 3), np.float32))
        with pytest.raises(ValueError):
            e.map_routes(imgs, 2, bias=np.zeros(8))
        e.value_dims, e.value_shape = 3, (3,)              # a read-out without a table
        with pytest.raises(capi.PinkError) as err:
            e.map_routes(imgs, 2)
        assert err.value.code == capi.ESTATE
        e.value_dims = 0
        assert e.map_routes(imgs[:0], 2)["neurons"].shape == (0, 2)
        assert e.map_routes(imgs, 2)["neurons"].shape == (4, 2)


def _run(*args):
    r = subprocess.run([B.CLI] + [str(a) for a in args], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    return r.stdout


def test_command_line_routes_and_read_out(cuda, tmp_path):
    imgs, som, args = make(n=300)
    N, _, idim, nd, ed, R = args[:6]
    path = {name: str(tmp_path / (name + ".bin")) for name in ("data", "som", "map", "map2", "routes", "values", "out", "dense")}
    files.write_data_file(path["data"], imgs.reshape(-1, idim, idim))
    files.write_som_file(path["som"], som.reshape(N, nd, nd), (3, 3))
    values = mt19937_uniform(N * 6, 3).reshape(N, 2, 3)
    files.write_data_file(path["values"], values)
    common = ["--som-width", 3, "--som-height", 3, "--numrot", R, "--neuron-dimension", nd, "--euclidean-distance-dimension", ed,
              "--euclidean-distance-type", "uint8"]
    _run(*common, "--map", path["data"], path["map"], path["som"])
    _run(*common, "--routes", 3, "--route-slope", -2, "--store-routes", path["routes"], "--read-out", path["values"], path["out"], "--map", path["data"],
         path["map2"], path["som"])
    dist, _ = files.read_mapping_file(path["map"])
    assert np.array_equal(dist, files.read_mapping_file(path["map2"])[0])
    neurons, weights, som_dims = files.read_routes_file(path["routes"])
    want, w = reference(dist, 3, -2.0)
    assert som_dims == [3, 3] and np.array_equal(neurons, want.astype(np.int64)) and np.abs(weights - w).max() <= weight_bound(dist, -2.0)
    out, _ = files.read_data_file(path["out"])
    exact = np.einsum("nk,nkab->nab", weights.astype(np.float64), values[neurons].astype(np.float64))
    assert out.shape == (300, 2, 3) and np.abs(out - exact).max() <= 4 * U * np.abs(values).max() * 2
    header = _run("--inspect", path["routes"])
    assert '"file_type": 4' in header and '"entries": 300' in header and '"routes": 3' in header
    _run(*common, "--read-out-all", "--read-out", path["values"], path["dense"], "--map", path["data"], path["map2"], path["som"])
    dense, _ = files.read_data_file(path["dense"])
    assert dense.shape == (300, 2, 3) and np.isfinite(dense).all() and np.abs(dense).max() <= 1.02 * np.abs(values).max()
