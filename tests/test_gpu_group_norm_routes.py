"""Group norm against its formula in 64 bits on shapes that take each of its kernels, with the helpers and tolerances of
test_gpu_group_norm.py: the on-chip kernels of 1024 threads and of narrow vectors, wide rows of every kind, rows whose teams take several
each, samples that do not fit the workspace at once, and the activations far from zero."""
import contextlib
import ctypes as C
import math

import numpy as np
import pytest
from scipy.special import erfc

import test_gpu_gated_scan as scan
import test_gpu_group_norm as base
from sliced_amd import rng

U, CHAIN, NONE, SILU, GELU, SEED = base.U, base.CHAIN, base.NONE, base.SILU, base.GELU, base.SEED

ON_CHIP = [(16, 300, 256, 4), (16, 300, 120, 4), (16, 300, 60, 4),     # 1024 threads, vectors of 4, 2 and 1, either direction
           (10, 961, 390, 13),                                         # 1024 threads forward, two passes backward
           (80, 700, 24, 2),                                           # 256 threads forward, 1024 backward
           (2, 50, 36, 6), (3, 20, 18, 3), (3, 40, 10, 2)]             # 256 threads, vectors of 2, 2 and 1
WIDE_ROWS = [(2, 1, 9000, 1), (2, 1, 8002, 1), (2, 1, 4001, 1),        # 1024 threads, four vectors each (backward: two passes)
             (3, 1, 4096, 1), (2, 1, 2050, 1), (2, 1, 1025, 1)]        # 256 threads and four; 1024 and two of narrow ones
SEVERAL_ROWS = [(5000, 1, 512, 1), (3000, 1, 250, 1), (100000, 1, 16, 2), (9000, 1, 390, 13),  # teams of a wave's lanes, folded
                (1100, 1, 1024, 1), (1100, 1, 2048, 1), (700, 1, 4096, 1), (300, 1, 5000, 1),  # of a workgroup, backward
                (4500, 1, 1030, 1), (2100, 1, 4100, 1), (700, 1, 3000, 3)]                     # and forward too


def check(hip, shape, kind, tag=300):
    base.say("group norm", shape, kind)
    x, w, b, dy = base.data(shape, kind, tag=tag)
    out, mean, rstd = hip.group_norm(*shape, x, w, b, act=kind)
    for got, want, tol, what in zip((out, mean, rstd), *base.forward(shape, x, w, b, kind, 1e-5), ("out", "mean", "rstd")):
        base.close(got, want, tol, what)
    outs = [np.full(x.size, np.nan, np.float32), np.full(shape[2], np.nan, np.float32), np.full(shape[2], np.nan, np.float32)]
    hip.group_norm_grad(*shape, x, w, b, mean, rstd, dy, *outs, act=kind)
    for got, want, tol, what in zip(outs, *base.backward(shape, x, w, b, kind, mean, rstd, dy), ("x", "weight", "bias")):
        base.close(got, want, tol, what)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [SILU, GELU])
@pytest.mark.parametrize("shape", ON_CHIP + WIDE_ROWS)
def test_on_chip_and_wide_rows(hip, shape, kind):
    check(hip, shape, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SEVERAL_ROWS)
def test_teams_that_take_several_rows(hip, shape):
    check(hip, shape, SILU)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(5000, 1, 512, 1), (1100, 1, 1024, 1), (300, 1, 5000, 1), (16, 300, 256, 4), (16, 300, 120, 4)])
def test_outputs_over_inputs_and_accumulation(hip, shape):
    """Teams that request their next row while they write this one, and windows of 1024 threads: x_grad over out_grad and out over
    x give the bits of separate arrays; beta = 1 adds to what is there."""
    base.say("group norm in place", shape)
    x, w, b, dy = base.data(shape, SILU, tag=310)
    out, mean, rstd = hip.group_norm(*shape, x, w, b, act=SILU)
    want = [np.zeros(x.size, np.float32), np.zeros(shape[2], np.float32), np.zeros(shape[2], np.float32)]
    hip.group_norm_grad(*shape, x, w, b, mean, rstd, dy, *want, act=SILU)
    old = [rng.normal(k.size, 1.0, tag=320 + i, seed=SEED).astype(np.float32) for i, k in enumerate(want)]
    sums = [o.copy() for o in old]
    hip.group_norm_grad(*shape, x, w, b, mean, rstd, dy, *sums, act=SILU, beta=1.0)
    for got, o, k in zip(sums, old, want):
        assert np.array_equal(got, o + k)
    c = hip.ctx()
    X, W, B, M, R, G = [c.array(a) for a in (x, w, b, mean, rstd, dy)]
    c.call("slhip_group_norm_grad", *shape, SILU, X.ptr, W.ptr, B.ptr, M.ptr, R.ptr, G.ptr, None, None, G.ptr, 0.0)
    assert np.array_equal(G.numpy(), want[0])
    c.call("slhip_group_norm", *shape, SILU, 1e-5, X.ptr, W.ptr, B.ptr, M.ptr, R.ptr, X.ptr)
    assert np.array_equal(X.numpy(), out)
    for k in (X, W, B, M, R, G):
        k.free()


@contextlib.contextmanager
def smaller_workspace(c, size):
    """The context as one whose workspace has `size` bytes: its record of them is the word behind the workspace's address."""
    at, whole = C.c_void_p(), c.lib.slhip_workspace_bytes(c.h)
    c.call("slhip_workspace", C.byref(at))
    words = (C.c_uint64 * 32).from_address(c.h.value)
    k = next(i for i in range(31) if words[i] == at.value and words[i + 1] == whole)
    assert size < whole
    words[k + 1] = size
    try:
        assert c.lib.slhip_workspace_bytes(c.h) == size
        yield
    finally:
        words[k + 1] = whole


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(7, 2500, 16, 4), (5, 3, 2600, 1), (40, 1, 96, 4), (6, 2200, 18, 3)])
def test_samples_that_do_not_fit_the_workspace_at_once(hip, shape):
    """The two-pass kernels over three samples at a time and fewer at the end (and rows whose column sums do not fit, which take them
    too): weights' and biases' gradients add up over the launches, also onto what is there."""
    n, p, ch, g = shape
    x, w, b, dy = base.data(shape, SILU, tag=330)
    from sliced_amd.device import Context
    c = Context(0)
    X, W, B, G = [c.array(a) for a in (x, w, b, dy)]
    M, R, O = c.empty(n * g), c.empty(n * g), c.empty(x.size)
    want, tol = base.forward(shape, x, w, b, SILU, 1e-5)

    def three_samples(call):
        """The smallest workspace that is not refused, times three"""
        size = 8
        while True:
            with smaller_workspace(c, size):
                if call() == 0:
                    break
            size += 8
            assert size < 1 << 20
        base.say("workspace of", 3 * size, "bytes", shape)
        return 3 * size

    def forward():
        return c.lib.slhip_group_norm(c.h, *shape, SILU, 1e-5, X.ptr, W.ptr, B.ptr, M.ptr, R.ptr, O.ptr)

    with smaller_workspace(c, three_samples(forward)):
        assert forward() == 0
        for got, v, t, what in zip((O, M, R), want, tol, ("out", "mean", "rstd")):
            base.close(got.numpy(), v, t, what)
    mean, rstd = M.numpy(), R.numpy()
    want, tol = base.backward(shape, x, w, b, SILU, mean, rstd, dy)
    old = [rng.normal(k, 1.0, tag=340 + i, seed=SEED).astype(np.float32) for i, k in enumerate((x.size, ch, ch))]
    outs = [c.array(o) for o in old]

    def backward(beta=0.0, skip=(), over=False):
        at = [None if i in skip else k.ptr for i, k in enumerate(outs)]
        if over:
            at[0] = G.ptr
        return c.lib.slhip_group_norm_grad(c.h, *shape, SILU, X.ptr, W.ptr, B.ptr, M.ptr, R.ptr, *at, G.ptr, beta)

    with smaller_workspace(c, three_samples(backward)):
        for beta in (0.0, 1.0):
            for k, o in zip(outs, old):
                k.upload(o)
            assert backward(beta) == 0
            for got, o, v, t, what in zip(outs, old, want, tol, ("x", "weight", "bias")):
                v = v + beta * o.reshape(v.shape)
                # (a launch adds to what the one before left: four roundings of the sums at most)
                base.close(got.numpy(), v, t + 4 * U * np.abs(v) + beta * 4 * U * np.abs(o.reshape(v.shape)), (what, beta))
        for only in range(3):
            outs[only].upload(np.full(outs[only].n, np.nan, np.float32))
            assert backward(0.0, skip=[i for i in range(3) if i != only]) == 0
            base.close(outs[only].numpy(), want[only], tol[only] + 4 * U * np.abs(want[only]), only)
        assert backward(0.0, skip=(1, 2), over=True) == 0
        base.close(G.numpy(), want[0], tol[0], "over out_grad")
    for k in [X, W, B, G, M, R, O] + outs:
        k.free()
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("room", [2, 3, 5, 8])
@pytest.mark.parametrize("mode", [scan.LINEAR, scan.SIGMOID])
def test_a_recurrence_split_as_far_as_the_workspace_goes(mode, room):
    """Pairs of states for fewer chunks than the steps would be split into, down to none."""
    from sliced_amd.device import Context
    batch, steps, channels = 2, 9000, 21
    gate, x, h0 = scan.data(mode, batch, steps, channels, tag=110)
    dh = rng.normal(gate.size, 1.0, tag=111, seed=SEED).reshape(gate.shape).astype(np.float32)
    c = Context(0)
    n, s = gate.size, batch * channels
    ins = [c.array(a) for a in (gate, x, h0, dh)]
    h, last, dg, dx, d0 = [c.empty(k) for k in (n, s, n, n, s)]
    with smaller_workspace(c, room * s * 4):
        c.call("slhip_gated_scan", mode, batch, steps, channels, *[k.ptr for k in ins[:3]], h.ptr, last.ptr)
        c.call("slhip_gated_scan_grad", mode, batch, steps, channels, *[k.ptr for k in ins[:3]], h.ptr, dg.ptr, dx.ptr, d0.ptr, ins[3].ptr, None, 0.0)
        got = [k.numpy() for k in (h, last, dg, dx, d0)]
    want, tol = scan.forward(mode, gate, x, h0)
    scan.close(got[0], want, tol, "h")
    assert np.array_equal(got[1].reshape(batch, channels), got[0].reshape(gate.shape)[:, -1])
    for a, v, t, what in zip(got[2:], *scan.backward(mode, gate, x, h0, got[0].reshape(gate.shape), dh, None), ("gate", "x", "h0")):
        scan.close(a, v, t, what)
    for k in ins + [h, last, dg, dx, d0]:
        k.free()
    c.close()


def slope_tolerance(kind, u, off):
    """What 32 bits make of act'(u) where u itself is off by `off`: far out the slope is a constant, and the error goes with
    the exponential that is left of it.  SiLU: |act''| <= (2 + |u|) exp(-|u|); the slope is q (1 + u (1 - q)), eight roundings.  GELU:
    |act''| <= (2 + u^2) f, f = exp(-u^2 / 2) / sqrt(2 pi) the density; the slope is a tail of the distribution and u f, both to 16
    roundings and the exponent's three, of u^2 / 2, in units of itself, the tail to 3e-8 of the fitted polynomial's too."""
    a = np.minimum(np.abs(u), 1e8)
    if kind == SILU:
        near = np.maximum(a - off, 0)
        curve = np.minimum(0.8, (2 + a) * np.exp(-near))
        q, rest = 1 / (1 + np.exp(np.minimum(a, 700))), 1 / (1 + np.exp(-a))
        return curve * off + 8 * U * np.where(u > 0, rest * (1 + a * q), q * (1 + a * rest)) + 1e-37
    near = np.maximum(a - off, 0)
    density = np.exp(-near * near / 2) / math.sqrt(2 * math.pi)
    return np.minimum(0.8, (2 + a * a) * density) * off + (1 + a) * density * (16 + 1.5 * a * a) * U + 3e-8 + 2 * U * (u > 0)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [SILU, GELU])
def test_gradients_of_activations_far_out(hip, kind):
    """Weights from 10^-4 to 10^8 and biases from -30 to 30: slopes next to zero, next to one, and between."""
    shape = (6, 1, 125, 1)
    x, _, _, dy = base.data(shape, kind, tag=350)
    w = (10.0 ** np.linspace(-4, 8, 125)).astype(np.float32)
    b = np.tile(np.linspace(-30, 30, 25), 5).astype(np.float32)
    out, mean, rstd = hip.group_norm(*shape, x, w, b, act=kind)
    outs = [np.zeros(x.size, np.float32), np.zeros(125, np.float32), np.zeros(125, np.float32)]
    hip.group_norm_grad(*shape, x, w, b, mean, rstd, dy, *outs, act=kind)
    with np.errstate(over="ignore"):
        (dx, dw, db), _ = base.backward(shape, x, w, b, kind, mean, rstd, dy)
        hat = (base.split(x, shape) - base.spread(mean, shape)) * base.spread(rstd, shape)
        u = hat * w + b
        g, r = base.split(dy, shape), base.spread(rstd, shape)
        gu = g * base.slope(kind, u)
    off = 3 * U * np.abs(hat * w) + U * np.abs(u)
    tol_g = np.abs(g) * slope_tolerance(kind, u, off) + U * np.abs(gu)
    gx = gu * w
    tol_gx = w * tol_g + U * np.abs(gx)
    means = lambda v: v.mean(axis=3, keepdims=True)  # noqa: E731
    tol_a = means(tol_gx) + CHAIN * U * means(np.abs(gx))
    tol_b = means(tol_gx * np.abs(hat) + 3 * U * np.abs(gx * hat)) + CHAIN * U * means(np.abs(gx * hat))
    tol_x = r * (tol_gx + tol_a + np.abs(hat) * tol_b + 5 * U * (np.abs(gx) + np.abs(means(gx)) + np.abs(hat * means(gx * hat))))
    sums = lambda v: v.sum(axis=(0, 1)).ravel()  # noqa: E731
    tol_w = sums(tol_g * np.abs(hat) + 3 * U * np.abs(gu * hat)) + CHAIN * U * sums(np.abs(gu * hat))
    tol_d = sums(tol_g) + CHAIN * U * sums(np.abs(gu))
    for got, want, tol, what in zip(outs, (dx, dw, db), (tol_x, tol_w, tol_d), ("x", "weight", "bias")):
        base.close(got, want, tol, what)


@pytest.mark.gpu
def test_gelu_below_zero(hip):
    """u Phi(u) from -1 to -12, relative to itself: the exponent -u^2 / 2 of its tail is rounded three times, the fitted polynomial is
    2.6e-7 off, and there are 32 roundings besides."""
    u = -np.linspace(1, 12, 4001).astype(np.float32)
    x, w = np.zeros((1, 1, u.size), np.float32), np.ones(u.size, np.float32)
    out = hip.group_norm(1, 1, u.size, 1, x, w, u, act=GELU)[0].astype(np.float64)
    f = u.astype(np.float64)
    want = f * 0.5 * erfc(-f / math.sqrt(2))
    off = np.abs(out / want - 1)
    base.say("largest relative error", off.max(), "for |u| < 2:", off[f > -2].max())
    assert (off <= 2.6e-7 + (32 + 1.5 * f * f) * U).all(), float((off / (2.6e-7 + (32 + 1.5 * f * f) * U)).max())
