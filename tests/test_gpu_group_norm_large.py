"""Group norm of values whose squares, or whose squared deviations, do not fit 32 bits: every route through the kernels gives the
same answer.  The shapes go to the rows of a wave, of a workgroup of 256 and of 1024, to the on-chip kernels of 256 and of 1024
threads, and to two passes with several runs of positions, and with groups cut into windows."""
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


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
def test_deviations_whose_squares_overflow(hip, shape):
    """Deviations near 10^20: the variance is infinite, 1/sqrt(var) zero, the outputs what the biases give, and the gradients zero
    but for the biases'.  A group beside it, of ordinary values, does not notice."""
    base.say("norm, infinite variance", shape)
    n, p, c, g = shape
    x, w, b, dy = base.data(shape, SILU, tag=210, offset=0.0)
    plain = x.copy()
    x[0, :, :c // g] *= np.float32(1e20)                     # the first group of the first sample
    for act in (NONE, SILU):
        out, mean, rstd = hip.group_norm(*shape, x, w, b, act=act)
        (want, wm, wr), (tol, tm, tr) = base.forward(shape, plain, w, b, act, 1e-5)
        big = x[0, :, :c // g].astype(np.float64)
        want[0, :, 0], tol[0, :, 0] = base.act(act, b[:c // g].astype(np.float64)), 6 * U * np.abs(b[:c // g])
        wm[0, 0], tm[0, 0] = big.mean(), base.CHAIN * U * np.abs(big).mean()
        wr[0, 0], tr[0, 0] = 0, 0
        for got, v, t, what in zip((out, mean, rstd), (want, wm, wr), (tol, tm, tr), ("out", "mean", "rstd")):
            base.close(got, v, t, what)
        grads = [np.full(x.size, np.nan, np.float32), np.full(c, np.nan, np.float32), np.full(c, np.nan, np.float32)]
        hip.group_norm_grad(*shape, x, w, b, mean, rstd, dy, *grads, act=act)
        for got, v, t, what in zip(grads, *base.backward(shape, x, w, b, act, mean, rstd, dy), ("x", "weight", "bias")):
            base.close(got, v, t, what)
        assert (grads[0].reshape(x.shape)[0, :, :c // g] == 0).all()
