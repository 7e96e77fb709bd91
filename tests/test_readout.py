"""Argument checks of the read-out operators, without a GPU: every refusal comes before the first CUDA call."""
import ctypes as C

import pytest

from pink_b200 import capi

ONE = 1 << 20          # stands for a device pointer that a refused call never touches
U64 = C.c_uint64


def route_config(**kw):
    d = dict(n_neurons=12, top_k=3, score=0, renormalise=1, n_groups=1, top_groups=1, group_best=1, slope=-1.0, scale=1.0)
    d.update(kw)
    return capi.RouteConfig(*[d[f] for f, _ in capi.RouteConfig._fields_])


def route(cfg, n=4, type=0, values=ONE, ld=12, neurons=ONE, weights=ONE, stype=0, scores=None, ls=0):
    return capi.lib.pink_b200_op_route(cfg and C.byref(cfg), n, type, values, ld, None, None, neurons, weights, None, stype, scores, ls, None)


@pytest.mark.parametrize("kw,text", [
    (dict(n_neurons=0), b"neurons"), (dict(n_neurons=32769), b"neurons"), (dict(top_k=0), b"top_k"), (dict(top_k=13), b"top_k"),
    (dict(n_neurons=64, top_k=33), b"top_k"), (dict(score=2), b"score"), (dict(renormalise=2), b"renormalise"),
    (dict(slope=float("nan")), b"slope"), (dict(slope=float("inf")), b"slope"), (dict(scale=0.0), b"scale"), (dict(scale=-1.0), b"scale"),
    (dict(scale=float("inf")), b"scale"), (dict(n_groups=0), b"n_groups"), (dict(n_groups=5), b"n_groups"), (dict(n_groups=4, top_groups=0), b"top_groups"),
    (dict(n_groups=4, top_groups=5), b"top_groups"), (dict(n_groups=6, top_groups=1), b"fewer than top_k"), (dict(n_groups=4, group_best=3), b"group_best"),
])
def test_route_refuses_bad_configurations(kw, text):
    assert route(route_config(**kw), ld=40000) == capi.EINVAL
    assert text in capi.lib.pink_b200_last_error()


def test_route_refuses_bad_arguments():
    ok = route_config()
    assert route(None) == capi.EINVAL
    assert route(ok, type=3) == capi.EINVAL
    assert route(ok, ld=11) == capi.EINVAL
    assert route(ok, n=1 << 31) == capi.EINVAL
    assert route(ok, values=None) == capi.EINVAL
    assert route(ok, neurons=None) == capi.EINVAL
    assert route(ok, weights=None) == capi.EINVAL
    assert route(ok, scores=ONE, stype=3, ls=12) == capi.EINVAL
    assert route(ok, scores=ONE, stype=0, ls=11) == capi.EINVAL
    assert route(ok, n=0, values=None, neurons=None, weights=None) == capi.OK
    assert route(route_config(n_groups=257, n_neurons=257), ld=257) == capi.EINVAL


def test_route_backward_refuses_bad_arguments():
    def call(cfg=route_config(), n=4, type=0, ld=12, neurons=ONE, weights=ONE, dweights=ONE, dscores=None, lds=0, out=ONE, ldo=12, values=ONE):
        return capi.lib.pink_b200_op_route_backward(C.byref(cfg), n, type, values, ld, None, neurons, weights, dweights, dscores, lds, out, ldo, None)
    assert call(type=4) == capi.EINVAL and call(ld=3) == capi.EINVAL and call(ldo=11) == capi.EINVAL
    assert call(dscores=ONE, lds=5) == capi.EINVAL
    for missing in ("values", "neurons", "weights", "dweights", "out"):
        assert call(**{missing: None}) == capi.EINVAL
    assert call(cfg=route_config(scale=0.0)) == capi.EINVAL
    assert call(n=0, values=None, out=None) == capi.OK


def test_balance_refuses_bad_arguments():
    f = capi.lib.pink_b200_op_route_balance
    assert f(0, ONE, None, 0.1, ONE, ONE, None) == capi.EINVAL
    assert f(32769, ONE, None, 0.1, ONE, ONE, None) == capi.EINVAL
    assert f(4, ONE, None, float("nan"), ONE, ONE, None) == capi.EINVAL
    assert f(4, None, None, 0.1, ONE, ONE, None) == capi.EINVAL
    assert f(4, ONE, None, 0.1, None, ONE, None) == capi.EINVAL
    assert f(4, ONE, None, 0.1, ONE, None, None) == capi.EINVAL


def test_read_out_refuses_bad_arguments():
    def call(type=0, N=5, D=7, values=ONE, ld=7, n=4, k=2, neurons=ONE, weights=ONE, res=None, lr=0, out=ONE, lo=7):
        return capi.lib.pink_b200_op_read_out(type, N, D, values, ld, n, k, neurons, weights, res, lr, out, lo, None)
    assert call(type=3) == capi.EINVAL and call(N=0) == capi.EINVAL and call(D=0) == capi.EINVAL and call(D=(1 << 24) + 1, ld=1 << 25, lo=1 << 25) == capi.EINVAL
    assert call(k=0) == capi.EINVAL and call(k=33) == capi.EINVAL and call(ld=6) == capi.EINVAL and call(lo=6) == capi.EINVAL
    assert call(res=ONE, lr=6) == capi.EINVAL and call(n=1 << 31) == capi.EINVAL
    for missing in ("values", "neurons", "weights", "out"):
        assert call(**{missing: None}) == capi.EINVAL
    assert call(n=0, values=None, out=None) == capi.OK


def test_read_out_backward_refuses_bad_arguments():
    size = capi.lib.pink_b200_read_out_workspace(5, 7, 4, 2)
    assert size > 0
    assert capi.lib.pink_b200_read_out_workspace(40000, 7, 4, 2) == 0 and capi.lib.pink_b200_read_out_workspace(5, 7, 0, 2) == 0

    def call(N=5, n=4, k=2, ld=7, ldd=7, ldv=7, values=ONE, neurons=ONE, weights=ONE, dout=ONE, dv=ONE, dw=ONE, work=ONE, bytes=size):
        return capi.lib.pink_b200_op_read_out_backward(0, N, 7, values, ld, n, k, neurons, weights, dout, ldd, dv, ldv, dw, work, bytes, None)
    assert call(N=32769) == capi.EINVAL and call(n=1 << 30) == capi.EINVAL and call(ld=6) == capi.EINVAL and call(ldd=6) == capi.EINVAL and call(ldv=6) == capi.EINVAL
    assert call(bytes=size - 1) == capi.EINVAL and call(work=None) == capi.EINVAL and call(work=ONE + 4) == capi.EINVAL
    for missing in ("values", "neurons", "weights", "dout"):
        assert call(**{missing: None}) == capi.EINVAL
    assert call(n=0, dv=None, neurons=None, weights=None, dout=None) == capi.OK


def product_config(**kw):
    d = dict(type=capi.BF16, inputs=24, outputs=10, by_input=0, activation=0, reserved=0, n=40)
    d.update(kw)
    return capi.ProductConfig(*[d[f] for f, _ in capi.ProductConfig._fields_])


def product(cfg, x=ONE, ldx=24, w=ONE, ldw=24, res=None, lr=0, out=ONE, lo=10, z=None, lz=0, work=None, size=None, ask=0):
    return capi.lib.pink_b200_op_product(cfg and C.byref(cfg), x, ldx, w, ldw, None, res, lr, out, lo, z, lz, work, size, ask, None)


def test_product_refuses_bad_arguments():
    ok = product_config()
    assert product(None) == capi.EINVAL
    for kw in (dict(type=capi.F32), dict(type=3), dict(inputs=0), dict(outputs=0), dict(inputs=1 << 31), dict(n=1 << 31), dict(by_input=2),
               dict(activation=5), dict(reserved=1)):
        assert product(product_config(**kw)) == capi.EINVAL, kw
    assert product(ok, ldx=23) == capi.EINVAL and product(ok, ldw=23) == capi.EINVAL and product(ok, lo=9) == capi.EINVAL
    assert product(product_config(by_input=1), ldw=9) == capi.EINVAL
    assert product(ok, res=ONE, lr=9) == capi.EINVAL and product(ok, z=ONE, lz=9) == capi.EINVAL
    assert product(ok, x=None) == capi.EINVAL and product(ok, w=None) == capi.EINVAL and product(ok, out=None) == capi.EINVAL
    assert product(product_config(n=0), x=None, w=None, out=None) == capi.OK
    assert product(product_config(n=1 << 30, outputs=1 << 30, inputs=8), ldx=8, ldw=8, lo=1 << 30) == capi.EINVAL      # more tiles than a grid holds


def test_product_workspace_is_asked_for():
    size = U64(0)
    cfg = product_config(n=4096, inputs=25)                # rows of 25 elements cannot be read in place
    assert product(cfg, ldx=25, ldw=25, size=C.byref(size), ask=1) == capi.OK and size.value >= 2 * 32 * 4096
    assert product(cfg, ldx=25, ldw=25) == capi.EINVAL and b"workspace" in capi.lib.pink_b200_last_error()
    less = U64(size.value - 1)
    assert product(cfg, ldx=25, ldw=25, work=ONE, size=C.byref(less)) == capi.EINVAL
    assert product(cfg, ldx=25, ldw=25, work=ONE + 8, size=C.byref(size)) == capi.EINVAL
    assert product(cfg, ldx=25, ldw=25, ask=1) == capi.EINVAL


def test_product_backward_refuses_bad_arguments():
    def call(cfg=product_config(), d=ONE, ldd=10, x=ONE, w=ONE, z=None, lz=0, dx=ONE, ldx=24, dw=ONE, ldw=24, db=ONE, work=None, size=None, ask=0):
        return capi.lib.pink_b200_op_product_backward(C.byref(cfg), d, ldd, x, 24, w, 24, z, lz, dx, ldx, dw, ldw, db, work, size, ask, None)
    assert call(d=None) == capi.EINVAL and call(x=None) == capi.EINVAL and call(w=None) == capi.EINVAL
    assert call(ldd=9) == capi.EINVAL and call(ldx=23) == capi.EINVAL and call(ldw=23) == capi.EINVAL
    assert call(cfg=product_config(activation=capi.ACT_GELU), z=None, lz=10) == capi.EINVAL
    assert call(cfg=product_config(activation=capi.ACT_GELU), z=ONE, lz=9) == capi.EINVAL
    size = U64(0)
    assert call(size=C.byref(size), ask=1) == capi.OK and size.value > 0
    assert call() == capi.EINVAL                           # needs its workspace


def test_front_end_refuses_what_it_cannot_run():
    torch = pytest.importorskip("torch")
    from pink_b200 import readout as R
    x = torch.zeros(4, 12)
    with pytest.raises(ValueError, match="no CPU form"):
        R.route(x, 2)
    with pytest.raises(ValueError, match="no CPU form"):
        R.product(x.bfloat16(), x.bfloat16())
    with pytest.raises(TypeError):
        R.read_out(torch.zeros(3), x, x)
    with pytest.raises(TypeError):
        R.balance(x, x, 0.1)


def test_command_line_refuses_routes_where_there_are_none():
    import subprocess
    from pink_b200 import build

    def run(*args):
        return subprocess.run([build.CLI] + list(args), capture_output=True, text=True)
    for args, text in (((["--routes", "0"]), "larger than 0"), (["--route-slope", "1"], "must be negative"), (["--route-score", "tanh"], "Unknown route score"),
                       (["--routes", "3", "--train", "a", "b"], "are for --map"), (["--routes", "3", "--map", "a", "b", "c"], "needs --store-routes"),
                       (["--read-out-all", "--store-routes", "r", "--map", "a", "b", "c"], "needs --read-out"),
                       (["--read-out", "v", "--map", "a", "b", "c"], "Missing arguments")):
        r = run(*args)
        assert r.returncode == 1 and text in r.stderr, (args, r.stderr)


def test_routes_file_reader(tmp_path):
    import numpy as np
    from pink_b200 import files
    path = str(tmp_path / "routes.bin")
    pairs = np.array([[(3, 0.75), (1, 0.25)], [(0, 1.0), (-1, 0.0)]], np.dtype([("neuron", np.int32), ("weight", np.float32)]))
    with open(path, "wb") as f:
        np.array([2, 4, 2, 2, 0, 2, 5, 7], np.int32).tofile(f)
        pairs.tofile(f)
    neurons, weights, dims = files.read_routes_file(path)
    assert dims == [5, 7] and neurons.tolist() == [[3, 1], [0, -1]] and weights.tolist() == [[0.75, 0.25], [1.0, 0.0]]


def test_mapping_with_routes_refuses_null_arguments():
    r = capi.RouteResults()
    cfg = route_config()
    assert capi.lib.pink_b200_map_routes(None, C.byref(cfg), ONE, 1, None, None, C.byref(r)) == capi.EINVAL
    assert capi.lib.pink_b200_group_map_routes(None, C.byref(cfg), ONE, 1, None, None, C.byref(r)) == capi.EINVAL
    assert capi.lib.pink_b200_set_values(None, None, 0, 0) == capi.EINVAL
    assert capi.lib.pink_b200_group_set_values(None, None, 0, 0) == capi.EINVAL
