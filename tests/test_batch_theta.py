"""rbn_rope_kv_store_q8 with a theta below 1: pairs turn by more than a radian per position, and past 2^51 quarter turns there would be
nothing left of the angle in 64 bits."""
import os

import numpy as np
import pytest

from ronn_amd import _lib


@pytest.mark.parametrize("theta,max_blocks,fits", [
    (1e-4, 8, True), (1e-7, 1 << 20, True), (1e-12, 8, True), (1e-12, 1 << 20, False), (1e-20, 8, False), (1e-38, 1, False),
    (1e-45, 1, False), (1.0, 1 << 20, True), (3e38, 1 << 20, True)])
def test_theta_whose_angles_do_not_fit_is_refused(theta, max_blocks, fits):
    if not os.path.exists(_lib.LIB_PATH):
        import __graft_entry__ as g
        g.build()
    lib, p = _lib.load(), 0x10000     # never dereferenced on the host
    t, b = _lib.KvTable(4, max_blocks, 100, p, p, p, p), _lib.KvBatch(64, p, p, p, p, p, p)
    l = _lib.KvLayer(0, 4, 128, 0, p, p, p, p, p, p)
    assert lib.rbn_rope_kv_store_q8(None, p, t, b, l, 8, theta, p) == _lib.RBN_ERR_INVALID
    assert ("context is NULL" if fits else "theta") in lib.rbn_last_error().decode()


@pytest.mark.gpu
@pytest.mark.parametrize("theta", [1e-3, 0.5, 1.0])
def test_small_theta(ctx, theta):
    from test_gpu_batch import Rig
    theta = float(np.float32(theta))                # what the call gets
    rig = Rig(ctx, 4, 2, 64, "i8", rows=2, theta=theta, seed=3)
    for new in ([70, 1], [1, 1], [3, 40]):
        rig.step(new)
        rig.check_cache()
    assert ctx.device_flags() == 0
