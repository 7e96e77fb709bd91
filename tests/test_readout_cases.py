"""The read-out operators' sources, sizes and refusals that need no GPU."""
import ctypes as C
import glob
import os
import re
import subprocess

import pytest

from pink_b200 import build, capi

ONE = 1 << 20          # stands for a device pointer that is not touched


def test_waits_for_tensor_memory_name_the_registers_they_wait_for():
    """A wait that names no registers orders nothing for the compiler: uses of loaded values could move before it."""
    waits = 0
    for path in glob.glob(os.path.join(build.CSRC, "*.cu*")):
        text = open(path).read()
        for at in re.finditer(r"tcgen05\.wait::ld", text):
            waits += 1
            assert '"+r"(v[0])' in text[at.start():text.index(");", at.start())], path
    assert waits >= 2


def run_pink(*args):
    return subprocess.run([build.CLI] + [str(a) for a in args], capture_output=True, text=True)


def test_command_line_refuses_routes_that_the_library_would(tmp_path):
    """Before any file is touched: the results of an earlier run stay."""
    kept = tmp_path / "result"
    kept.write_text("earlier")
    maps = ["--store-routes", kept, "--map", "data", kept, "som"]
    for args, text in ((["--routes", 33] + maps, "at most 32"), (["--routes", 2000000000] + maps, "at most 32"), (["--route-slope", "-inf"] + maps, "must be finite"),
                       (["--route-slope", "-1e39"] + maps, "must be finite"), (["--route-slope", "nan"] + maps, "must be negative"),
                       (["--som-width", 182, "--som-height", 181] + maps, "at most 32768 neurons")):
        r = run_pink(*args)
        assert r.returncode == 1 and text in r.stderr, (args, r.stderr)
        assert kept.read_text() == "earlier"
    # as many routes as there are neurons are as good as more of them, and a map at the limit is not refused for its size
    for args in (["--som-width", 4, "--som-height", 8, "--routes", 40] + maps, ["--som-width", 128, "--som-height", 256] + maps,
                 ["--som-width", 182, "--som-height", 181, "--map", "data", kept, "som"]):
        r = run_pink(*args)
        assert r.returncode == 1 and "Error opening data" in r.stderr, (args, r.stderr)


@pytest.mark.parametrize("by_input", [0, 1])
def test_product_gradient_asks_for_one_copy_of_dz(by_input):
    """Without an activation, rows that straddle lines and that the products' tiles read 24 times or more: one copy of them serves both
    products.  (By input dz is read 15 times for dw: alone, that pays for no copy.)"""
    n, K, M = 256, 3648, 1032                             # dz: rows of 2,064 bytes; the other operands on whole lines
    cfg = capi.ProductConfig(capi.BF16, K, M, by_input, 0, 0, n)
    ld_w = 1088 if by_input else K

    def size(dx, dw, db=None, activation=0):
        bytes = C.c_uint64(0)
        cfg.activation = activation
        rc = capi.lib.pink_b200_op_product_backward(C.byref(cfg), ONE, M, ONE, K, ONE, ld_w, ONE if activation else None, M, dx, K, dw, ld_w, db, None, C.byref(bytes),
                                                    1, None)
        assert rc == capi.OK
        return bytes.value
    copy, sums = 2 * n * 1088, (n + 31) // 32 * M * 4
    sums = (sums + 255) // 256 * 256
    assert size(ONE, None) == copy and size(None, ONE) == (0 if by_input else copy)
    assert size(ONE, ONE) == copy                          # and not one for each
    assert size(ONE, ONE, activation=capi.ACT_RELU) == copy and size(None, ONE, activation=capi.ACT_RELU) == copy
    assert size(ONE, ONE, ONE) == copy + sums and size(None, None, ONE) == sums


def test_overlap_of_a_result_with_an_argument():
    """Against the shared elements counted one by one: none passes, and where the pitches agree nothing else is refused."""
    import random
    torch = pytest.importorskip("torch")
    from pink_b200 import readout as R
    rng, buf = random.Random(1), torch.zeros(200)

    def places(t):
        return {t.storage_offset() + i * t.stride(0) + j for i in range(t.shape[0]) for j in range(t.shape[1])}
    seen = [0, 0]
    for _ in range(20000):
        (out, lo), (arg, la) = ((torch.as_strided(buf, (rng.randint(1, 6), rng.randint(1, ld)), (ld, 1), rng.randint(0, 60)), ld)
                                for ld in (rng.choice([5, 8, 8, 13]) for _ in range(2)))
        shared = bool(places(out) & places(arg))
        try:
            R._apart(out, "out", out.data_ptr(), lo, (arg, "arg", False), (None, "nothing", False))
            refused = False
        except ValueError:
            refused = True
        assert refused or not shared
        assert not refused or shared or lo != la
        seen[shared] += 1
    assert min(seen) > 5000
    same = torch.zeros(4, 6)
    R._apart(same, "out", same.data_ptr(), 6, (same, "residual", True))
    with pytest.raises(ValueError, match="out overlaps x"):
        R._apart(same, "out", same.data_ptr(), 6, (same, "x", False))
    with pytest.raises(ValueError, match="out overlaps residual"):
        R._apart(same[:3], "out", same.data_ptr(), 6, (same[1:], "residual", True))
