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
    def call(type=0, D=7, n=4, dy=ONE, ldd=7, x=ONE, ld=7, mean=ONE, rstd=ONE, res=None, lr=0, dx=ONE, ldx=7, dw=ONE, db=ONE, work=None, size=None, ask=0):
        return capi.lib.pink_b200_op_layer_norm_backward(type, D, n, dy, ldd, x, ld, mean, rstd, None, res, lr, dx, ldx, dw, db, work, size, ask, None)
    size = C.c_uint64(0)
    assert call(size=C.byref(size), ask=1) == capi.OK and size.value >= 2 * 7 * 4
    for kw, text in ((dict(type=3), b"type"), (dict(D=0), b"elements"), (dict(n=1 << 31), b"rows"), (dict(ldd=6), b"leading"), (dict(ld=6), b"leading"), (dict(ldx=6), b"leading"),
                     (dict(res=ONE, lr=6), b"leading"), (dict(dw=None), b"together"), (dict(db=None), b"together"), (dict(ask=1), b"null"), (dict(dy=None), b"null"),
                     (dict(x=None), b"null"), (dict(mean=None), b"null"), (dict(rstd=None), b"null"), (dict(), b"workspace"),
                     (dict(work=ONE, size=C.byref(C.c_uint64(size.value - 1))), b"workspace"), (dict(work=ONE + 8, size=C.byref(size)), b"aligned")):
        assert call(**kw) == capi.EINVAL and text in capi.lib.pink_b200_last_error(), kw
    assert call(dx=None, dw=None, db=None) == capi.OK        # nothing is asked for
    assert call(n=0, dy=None, x=None, dw=None, db=None) == capi.OK
    assert call(n=0, size=C.byref(size), ask=1) == capi.OK and size.value == 0


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
