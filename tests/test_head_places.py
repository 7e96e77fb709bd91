"""Results in an argument's place: what the C entries refuse before the first CUDA call."""
from pink_b200 import capi

ONE, TWO = 1 << 20, 1 << 21          # stand for device pointers that a refused call never touches


def call(n=4, dx=TWO, ldx=7, res=TWO, lr=7, work=None):
    return capi.lib.pink_b200_op_layer_norm_backward(capi.F32, 7, n, ONE, 7, ONE, 7, ONE, ONE, None, res, lr, dx, ldx, ONE, ONE, work, 0, None)


def test_dx_in_the_residuals_place_has_its_pitch():
    for kw in (dict(ldx=8), dict(lr=9), dict(ldx=9, lr=8)):
        assert call(**kw) == capi.EINVAL and b"leading dimension" in capi.lib.pink_b200_last_error(), kw
    # the same pitch, another place, a single row or no row: what is missing then is the workspace
    for kw in (dict(), dict(ldx=9, lr=9), dict(dx=ONE << 4, ldx=8), dict(n=1, ldx=8), dict(dx=None, lr=8)):
        assert call(**kw) == capi.EINVAL and b"workspace" in capi.lib.pink_b200_last_error(), kw
