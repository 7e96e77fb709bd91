"""Mapping with routes at its edges."""
import subprocess

import numpy as np
import pytest

from pink_b200 import build as B
from pink_b200 import files
from pink_b200.synthetic import mt19937_uniform
from test_gpu_map_routes import U, make, weight_bound

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [5, 150])
def test_dense_read_out_leaves_masked_neurons_out(cuda, n):
    """A masked neuron's values -- NaN, where nothing is known about it -- do not reach the results: those are what zeros there give."""
    from pink_b200 import engine
    imgs, som, args = make(n=n)
    N = args[0]
    for D in (5, 64):
        values = mt19937_uniform(N * D, 4).reshape(N, D).copy()
        values[1], values[5, 2], values[7, 3], values[8, 0] = np.nan, np.inf, -np.inf, 3.4e38      # (3.4e38: an infinity in bfloat16)
        mask = np.ones(N, bool)
        mask[[1, 5, 7, 8]] = False
        with engine.Engine(*args) as e, engine.Group(*args) as g:
            for x in (e, g):
                x.set_som(som)
                x.set_values(np.where(mask[:, None], values, 0.0), dense=True)
                want = x.map_routes(imgs, 2, slope=-2.0, mask=mask)["values"]
                assert np.isfinite(want).all()
                x.set_values(values, dense=True)
                for _ in range(2):
                    assert np.array_equal(x.map_routes(imgs, 2, slope=-2.0, mask=mask)["values"], want)
                # a neuron that takes part brings its values along, before and after
                mask[1] = True
                got = x.map_routes(imgs, 2, slope=-2.0, mask=mask)["values"]
                assert np.isnan(got).all()
                assert np.isnan(x.map_routes(imgs, 2, slope=-2.0)["values"]).all()
                mask[1] = False
                assert np.array_equal(x.map_routes(imgs, 2, slope=-2.0, mask=mask)["values"], want)


def test_dense_mapping_waits_for_its_own_work_only(cuda):
    """The verdict on the mapping's products comes from the context: no other stream's work, nor what it reports, is waited for."""
    torch = cuda
    from pink_b200 import engine
    imgs, som, args = make(n=5)
    values = mt19937_uniform(args[0] * 6, 3).reshape(args[0], 6)
    with engine.Engine(*args) as e:
        e.set_som(som)
        e.set_values(values, dense=True)
        want = e.map_routes(imgs, 2)["values"]
        side, done = torch.cuda.Stream(), torch.cuda.Event()
        with torch.cuda.stream(side):
            torch.cuda._sleep(1_000_000_000)               # about half a second of another's work
            done.record()
        got = e.map_routes(imgs, 2)["values"]
        waited = done.query()
        done.synchronize()
        assert np.array_equal(got, want) and not waited


def test_command_line_keeps_results_where_the_table_is_refused(cuda, tmp_path):
    imgs, som, args = make(n=3)
    N, _, idim, nd, ed, R = args[:6]
    path = {name: str(tmp_path / (name + ".bin")) for name in ("data", "som", "map", "values", "out", "routes")}
    files.write_data_file(path["data"], imgs.reshape(-1, idim, idim))
    files.write_som_file(path["som"], som.reshape(N, nd, nd), (3, 3))
    files.write_data_file(path["values"], np.zeros((N - 1, 2, 3), np.float32))
    for name in ("map", "out", "routes"):
        open(path[name], "w").write("earlier")
    args = ["--som-width", 3, "--som-height", 3, "--numrot", R, "--neuron-dimension", nd, "--euclidean-distance-dimension", ed,
            "--store-routes", path["routes"], "--read-out", path["values"], path["out"], "--map", path["data"], path["map"], path["som"]]
    r = subprocess.run([B.CLI] + [str(a) for a in args], capture_output=True, text=True)
    assert r.returncode == 1 and "one entry per neuron" in r.stderr
    assert all(open(path[name]).read() == "earlier" for name in ("map", "out", "routes"))


def test_command_line_reports_a_data_file_that_ends_too_early(cuda, tmp_path):
    """The reader thread's error reaches the user as a message, from mapping, routed mapping and training alike."""
    imgs, som, args = make(n=700)
    N, _, idim, nd, ed, R = args[:6]
    path = {name: str(tmp_path / (name + ".bin")) for name in ("data", "som", "map", "routes", "trained")}
    files.write_data_file(path["data"], imgs.reshape(-1, idim, idim))
    files.write_som_file(path["som"], som.reshape(N, nd, nd), (3, 3))
    with open(path["data"], "r+b") as f:
        f.truncate(len(open(path["data"], "rb").read()) - 4 * idim * idim * 300)      # the second part of 256 images is incomplete
    common = ["--som-width", 3, "--som-height", 3, "--numrot", R, "--neuron-dimension", nd, "--euclidean-distance-dimension", ed, "--euclidean-distance-type", "uint8"]
    for rest in (["--map", path["data"], path["map"], path["som"]], ["--store-routes", path["routes"], "--map", path["data"], path["map"], path["som"]],
                 ["--input-shuffle-off", "--train", path["data"], path["trained"]]):
        r = subprocess.run([B.CLI] + [str(a) for a in common + rest], capture_output=True, text=True)
        assert r.returncode == 1 and "unexpected end of the data file" in r.stderr, (r.returncode, r.stderr)



def test_command_line_reads_all_neurons_out(cuda, tmp_path):
    """--read-out-all: the softmax of -distance times the values; scores, values and results rounded to bfloat16 (half a step 2^-8 each)."""
    imgs, som, args = make(n=300)
    N, _, idim, nd, ed, R = args[:6]
    path = {name: str(tmp_path / (name + ".bin")) for name in ("data", "som", "map", "values", "dense")}
    files.write_data_file(path["data"], imgs.reshape(-1, idim, idim))
    files.write_som_file(path["som"], som.reshape(N, nd, nd), (3, 3))
    values = mt19937_uniform(N * 6, 3).reshape(N, 2, 3)
    files.write_data_file(path["values"], values)
    args = ["--som-width", 3, "--som-height", 3, "--numrot", R, "--neuron-dimension", nd, "--euclidean-distance-dimension", ed, "--euclidean-distance-type", "uint8",
            "--route-slope", -2, "--read-out-all", "--read-out", path["values"], path["dense"], "--map", path["data"], path["map"], path["som"]]
    r = subprocess.run([B.CLI] + [str(a) for a in args], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    dist, _ = files.read_mapping_file(path["map"])
    got, _ = files.read_data_file(path["dense"])
    a = -2.0 * dist.astype(np.float64)
    p = np.exp(a - a.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    want, size, half = p @ values.reshape(N, 6).astype(np.float64), p @ np.abs(values).reshape(N, 6).astype(np.float64), 2.0 ** -8
    off = np.abs(got.reshape(300, 6) - want)
    assert (off <= size * (2 * half + half * half + weight_bound(dist, -2.0) * 2 + (N + 2) * 2 * U) * (1 + half) + half * np.abs(want)).all()
