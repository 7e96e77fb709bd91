"""Contexts of different sizes trained from two host threads, one after the other."""
import threading

import numpy as np
import pytest

from pink_b200.synthetic import blob_images, mt19937_uniform

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("step_kernel", [0, 1])
@pytest.mark.parametrize("mode", [0, 1, 2])
def test_another_threads_training_leaves_the_shared_memory_limit(cuda, mode, step_kernel):
    """A small map trained in between, from another thread, does not take away the shared memory that the large neurons' kernels need."""
    from pink_b200 import capi, engine

    def setup(nd, ed, idim, n):
        N = 9
        imgs = blob_images(n, idim, 1, seed=3).reshape(n, 1, idim, idim)
        e = engine.Engine(N, 1, idim, nd, ed, 8, True, mode, options={"step_kernel": step_kernel})
        e.set_som(mt19937_uniform(N * nd * nd, 5).reshape(N, 1, nd, nd))
        e.set_update_factors(engine.update_factors(capi.LAYOUT_CARTESIAN, 3, 3, capi.FUNC_GAUSSIAN, 1.1, 0.2))
        return e, imgs

    def train(e, imgs):
        e.train(imgs)
        e.synchronize()
    large, imgs = setup(90, 63, 64, 6)
    other, _ = setup(90, 63, 64, 6)
    small, few = setup(12, 7, 16, 4)
    try:
        train(large, imgs[:3])
        t = threading.Thread(target=train, args=(small, few))
        t.start()
        t.join()
        train(large, imgs[3:])
        train(other, imgs)
        shape = (9, 1, 90, 90)
        assert np.array_equal(large.get_som(np.zeros(shape, np.float32)), other.get_som(np.zeros(shape, np.float32)))
    finally:
        for e in (large, other, small):
            e.close()
