"""Group norm of values whose squares, or whose squared deviations, do not fit 32 bits: every route through the kernels gives the
same answer.  The shapes go to the rows of a wave, of a workgroup of 256 and of 1024, to the on-chip kernels of 256 and of 1024
threads, and to two passes with one part a group, several runs of positions, and groups cut into windows."""
import numpy as np
import pytest

import test_gpu_group_norm as base
from sliced_amd import rng

U, NONE, SILU = base.U, base.NONE, base.SILU
SHAPES = [(2, 1, 64, 2), (2, 1, 3000, 1), (2, 1, 5000, 1), (2, 30, 12, 3), (16, 300, 256, 4), (1, 700, 16, 4), (1, 5000, 16, 4), (2, 3, 2600, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
def test_a_mean_whose_square_overflows(hip, shape):
    """Values 10^16 around 10^20: the mean's square does not fit 32 bits, the deviations' do."""
    base.say("norm, large mean", shape)
    x, w, b, dy = base.data(shape, NONE, tag=200, offset=0.0)
    x = (1e20 + 1e16 * x.astype(np.float64)).astype(np.float32)
    out, mean, rstd = hip.group_norm(*shape, x, w, b, act=NONE)
    for got, want, tol, what in zip((out, mean, rstd), *base.forward(shape, x, w, b, NONE, 1e-5), ("out", "mean", "rstd")):
        base.close(got, want, tol, what)
    # and none at all, around a power of two: the sum of 5000 equal values of another number is rounded, and its mean with it,
    # which beside deviations of nothing is all there is; these sums are exact
    same = np.full(x.shape, 2.0 ** 66, np.float32)
    out, mean, rstd = hip.group_norm(*shape, same, w, b, act=NONE)
    assert np.array_equal(out.reshape(x.shape), np.broadcast_to(b, x.shape)) and (mean == same.flat[0]).all()
    assert np.allclose(rstd, 1e-5 ** -0.5, rtol=4 * U)
