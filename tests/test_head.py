"""Argument checks of the operators that train a head, without a GPU: every refusal comes before the first CUDA call."""
import ctypes as C

import pytest

from pink_b200 import capi

ONE = 1 << 20          # stands for a device pointer that a refused call never touches
INF = float("inf")


def norm(type=0, D=7, n=4, x=ONE, ld=7, w=None, b=None, eps=1e-5, y=ONE, ly=7):
    return capi.lib.pink_b200_op_layer_norm(type, D, n, x, ld, w, b, eps, y, ly, None, None, None)


def test_layer_norm_refuses_bad_arguments():
    for kw, text in ((dict(type=3), b"type"), (dict(D=0), b"elements"), (dict(D=(1 << 24) + 1, ld=1 << 25, ly=1 << 25), b"elements"), (dict(n=1 << 31), b"rows"),
                     (dict(ld=6), b"leading"), (dict(ly=6), b"leading"), (dict(eps=0.0), b"eps"), (dict(eps=-1.0), b"eps"), (dict(eps=INF), b"eps"),
                     (dict(eps=float("nan")), b"eps"), (dict(x=None), b"null"), (dict(y=None), b"null")):
        assert norm(**kw) == capi.EINVAL and text in capi.lib.pink_b200_last_error(), kw
    assert norm(n=0, x=None, y=None) == capi.OK


def test_layer_norm_backward_refuses_bad_arguments():
    size = capi.lib.pink_b200_layer_norm_workspace(0, 7, 4)
    assert size >= 2 * 7 * 4
    for type, D, n in ((3, 7, 4), (0, 0, 4), (0, (1 << 24) + 1, 4), (0, 7, 0), (0, 7, 1 << 31)):
        assert capi.lib.pink_b200_layer_norm_workspace(type, D, n) == 0

    def call(type=0, D=7, n=4, dy=ONE, ldd=7, x=ONE, ld=7, mean=ONE, rstd=ONE, res=None, lr=0, dx=ONE, ldx=7, dw=ONE, db=ONE, work=ONE, bytes=size):
        return capi.lib.pink_b200_op_layer_norm_backward(type, D, n, dy, ldd, x, ld, mean, rstd, None, res, lr, dx, ldx, dw, db, work, bytes, None)
    for kw, text in ((dict(type=3), b"type"), (dict(D=0), b"elements"), (dict(n=1 << 31), b"rows"), (dict(ldd=6), b"leading"), (dict(ld=6), b"leading"), (dict(ldx=6), b"leading"),
                     (dict(res=ONE, lr=6), b"leading"), (dict(dw=None), b"together"), (dict(db=None), b"together"), (dict(dy=None), b"null"),
                     (dict(x=None), b"null"), (dict(mean=None), b"null"), (dict(rstd=None), b"null"), (dict(work=None), b"workspace"), (dict(bytes=0), b"workspace"),
                     (dict(work=ONE + 8), b"aligned")):
        assert call(**kw) == capi.EINVAL and text in capi.lib.pink_b200_last_error(), kw
    assert call(dx=None, dw=None, db=None) == capi.OK        # nothing is asked for
    assert call(n=0, dy=None, x=None, dw=None, db=None, work=None) == capi.OK


def distill_config(**kw):
    d = dict(n_neurons=12, top_k=3, teacher=0, rest=0, temperature=1.0, scale=1.0)
    d.update(kw)
    return capi.DistillConfig(*[d[f] for f, _ in capi.DistillConfig._fields_])


@pytest.mark.parametrize("kw,text", [
    (dict(n_neurons=0), b"neurons"), (dict(n_neurons=32769), b"neurons"), (dict(top_k=0), b"top_k"), (dict(top_k=33), b"top_k"), (dict(teacher=2), b"teacher"),
    (dict(rest=2), b"rest"), (dict(rest=1, teacher=1), b"rest"), (dict(temperature=0.0), b"temperature"), (dict(temperature=-1.0), b"temperature"),
    (dict(temperature=2e3), b"temperature"), (dict(temperature=float("nan")), b"temperature"), (dict(scale=0.0), b"scale"), (dict(scale=INF), b"scale"),
    (dict(scale=float("nan")), b"scale"),
])
def test_distill_refuses_bad_configurations(kw, text):
    cfg = distill_config(**kw)
    assert capi.lib.pink_b200_op_distill(cfg, 4, 0, ONE, 40000, None, ONE, ONE, ONE, None) == capi.EINVAL and text in capi.lib.pink_b200_last_error()
    assert capi.lib.pink_b200_op_distill_backward(cfg, 4, 0, ONE, 40000, None, ONE, ONE, None, ONE, 40000, None, None) == capi.EINVAL


def test_distill_refuses_bad_arguments():
    def forward(cfg=distill_config(), n=4, type=0, s=ONE, ld=12, neurons=ONE, targets=ONE, loss=ONE):
        return capi.lib.pink_b200_op_distill(cfg, n, type, s, ld, None, neurons, targets, loss, None)

    def backward(cfg=distill_config(), n=4, type=0, s=ONE, ld=12, neurons=ONE, targets=ONE, d=ONE, ldd=12):
        return capi.lib.pink_b200_op_distill_backward(cfg, n, type, s, ld, None, neurons, targets, None, d, ldd, None, None)
    for call in (forward, backward):
        for kw in (dict(cfg=None), dict(type=3), dict(ld=11), dict(n=1 << 31), dict(s=None), dict(neurons=None), dict(targets=None)):
            assert call(**kw) == capi.EINVAL, kw
        assert call(n=0, s=None, neurons=None, targets=None) == capi.OK
    assert forward(loss=None) == capi.EINVAL and backward(d=None) == capi.EINVAL and backward(ldd=11) == capi.EINVAL


def test_front_end_refuses_what_it_cannot_run():
    torch = pytest.importorskip("torch")
    from pink_b200 import readout as R
    x, v = torch.zeros(4, 12), torch.zeros(4)
    neurons, targets = torch.zeros(4, 3, dtype=torch.int32), torch.zeros(4, 3)
    for call in (lambda: R.layer_norm(x), lambda: R.layer_norm_backward(x, x, v, v), lambda: R.distill(x, neurons, targets),
                 lambda: R.distill_backward(v, x, neurons, targets)):
        with pytest.raises(ValueError, match="no CPU form"):
            call()
    for call in (lambda: R.layer_norm(v), lambda: R.distill(v, neurons, targets)):
        with pytest.raises(TypeError, match="matrix"):
            call()


def gated_config(**kw):
    d = dict(type=capi.BF16, inputs=24, outputs=10, by_input=0, activation=capi.ACT_SILU, reserved=0, n=40)
    d.update(kw)
    return capi.ProductConfig(*[d[f] for f, _ in capi.ProductConfig._fields_])


def gated(cfg, x=ONE, ldx=24, gate=ONE, ldg=24, up=ONE, ldu=24, h=ONE, lh=10, g=None, lg=0, u=None, lu=0, work=None, size=None, ask=0):
    return capi.lib.pink_b200_op_gated(cfg, x, ldx, gate, ldg, up, ldu, None, None, h, lh, g, lg, u, lu, work, size, ask, None)


def gated_backward(cfg=gated_config(), dh=ONE, ldd=10, x=ONE, gate=ONE, up=ONE, ldw=24, g=ONE, lg=10, u=ONE, lu=10, dx=ONE, ldx=24, dgate=ONE, ldg=24, dup=ONE, ldp=24,
                   dgb=ONE, dub=ONE, work=None, size=None, ask=0):
    return capi.lib.pink_b200_op_gated_backward(cfg, dh, ldd, x, 24, gate, ldw, up, ldw, g, lg, u, lu, dx, ldx, dgate, ldg, dup, ldp, dgb, dub, work, size, ask, None)


def test_gated_refuses_bad_arguments():
    bad = (dict(type=capi.F32), dict(type=3), dict(inputs=0), dict(outputs=0), dict(inputs=1 << 30), dict(outputs=1 << 30), dict(n=1 << 31), dict(by_input=2), dict(activation=5),
           dict(reserved=1))
    for kw in bad:
        assert gated(gated_config(**kw)) == capi.EINVAL and gated_backward(gated_config(**kw)) == capi.EINVAL, kw
    assert gated(None) == capi.EINVAL and gated_backward(None) == capi.EINVAL
    ok = gated_config()
    for kw in (dict(ldx=23), dict(ldg=23), dict(ldu=23), dict(lh=9), dict(g=ONE, lg=9), dict(u=ONE, lu=9), dict(x=None), dict(gate=None), dict(up=None), dict(h=None)):
        assert gated(ok, **kw) == capi.EINVAL, kw
    assert gated(gated_config(by_input=1), ldg=9) == capi.EINVAL and gated(gated_config(by_input=1), ldg=10, ldu=9) == capi.EINVAL
    for kw in (dict(ldd=9), dict(lg=9), dict(lu=9), dict(ldx=23), dict(ldg=23), dict(ldp=23), dict(ldw=23), dict(dh=None), dict(x=None), dict(gate=None), dict(up=None), dict(g=None),
               dict(u=None)):
        assert gated_backward(**kw) == capi.EINVAL, kw
    for kw in (dict(dgate=None), dict(dup=None), dict(dgb=None), dict(dub=None)):
        assert gated_backward(**kw) == capi.EINVAL and b"together" in capi.lib.pink_b200_last_error(), kw
    assert gated(gated_config(n=0), x=None, gate=None, up=None, h=None) == capi.OK
    assert gated_backward(gated_config(n=0), dh=None, dgate=None, dup=None, dgb=None, dub=None) == capi.OK
    assert gated(gated_config(n=1 << 30, outputs=1 << 29, inputs=8), ldx=8, ldg=8, ldu=8, lh=1 << 29) == capi.EINVAL      # more tiles than a grid holds


def test_gated_workspace_is_asked_for():
    size = C.c_uint64(0)
    cfg = gated_config(n=4096, inputs=25)                  # rows of 25 elements cannot be read in place
    lds = dict(ldx=25, ldg=25, ldu=25)
    assert gated(cfg, size=C.byref(size), ask=1, **lds) == capi.OK and size.value >= 2 * 32 * 4096
    assert gated(cfg, **lds) == capi.EINVAL and b"workspace" in capi.lib.pink_b200_last_error()
    assert gated(cfg, work=ONE, size=C.byref(C.c_uint64(size.value - 1)), **lds) == capi.EINVAL
    assert gated(cfg, work=ONE + 8, size=C.byref(size), **lds) == capi.EINVAL
    assert gated(cfg, ask=1, **lds) == capi.EINVAL
    assert gated(gated_config(n=8), size=C.byref(size), ask=1) == capi.OK and size.value == 0      # a few rows need none
    assert gated_backward(size=C.byref(size), ask=1) == capi.OK and size.value >= 2 * 40 * 64 * 2
    assert gated_backward() == capi.EINVAL
    assert gated_backward(dx=None, dgate=None, dup=None, dgb=None, dub=None) == capi.OK      # nothing is asked for
