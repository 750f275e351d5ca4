"""Group norm with an activation, forward and backward, through the C ABI against its formula in 64 bits.

Tolerances, u = 2^-24.  A group's mean is a sum of chains of at most CHAIN additions, so it is off by at most
CHAIN u mean|x|, and so is each x - mean, with one more rounding; the variance is a sum of the squares of such
differences, so rstd is off by (CHAIN / 2 + 4) u of itself and by what the mean's error does to it (its square, negligible
beside: a shift of the mean changes the variance by the square of the shift).  From there on every rounding is
counted where it happens; the activations' slopes are at most 1.13, their curvatures at most 0.8."""
import ctypes as C
import math

import numpy as np
import pytest
from scipy.special import erf

from sliced_amd import rng

U = 2.0 ** -24
CHAIN = 160.0    # 128 values of a thread's own run at most in the shapes below, and the joins of threads, waves and workgroups
NONE, RELU, SILU, GELU = range(4)
SEED = 0x51CED


def say(*a):
    print(*a, flush=True)


def act(kind, u):
    if kind == RELU:
        return np.where(u >= 0, u, 0.0)
    if kind == SILU:
        return u / (1 + np.exp(-u))
    if kind == GELU:
        return 0.5 * u * (1 + erf(u / math.sqrt(2)))
    return u


def slope(kind, u):
    if kind == RELU:
        return (u >= 0) * 1.0
    if kind == SILU:
        q = 1 / (1 + np.exp(-u))
        return q * (1 + u * (1 - q))
    if kind == GELU:
        return 0.5 * (1 + erf(u / math.sqrt(2))) + u * np.exp(-u * u / 2) / math.sqrt(2 * math.pi)
    return np.ones_like(u)


def split(x, shape):
    n, p, c, g = shape
    return x.astype(np.float64).reshape(n, p, g, c // g)


def spread(v, shape):
    """[n, g] over the group"""
    return v.astype(np.float64).reshape(shape[0], 1, shape[3], 1)


def channelwise(v, shape, none):
    n, p, c, g = shape
    return np.full((1, 1, g, c // g), none) if v is None else v.astype(np.float64).reshape(1, 1, g, c // g)


def forward(shape, x, w, b, kind, eps):
    xs, ws, bs = split(x, shape), channelwise(w, shape, 1.0), channelwise(b, shape, 0.0)
    mean = xs.mean(axis=(1, 3), keepdims=True)
    d = xs - mean
    rstd = 1 / np.sqrt((d * d).mean(axis=(1, 3), keepdims=True) + eps)
    off = CHAIN * U * np.abs(xs).mean(axis=(1, 3), keepdims=True) + U * np.abs(mean)
    slack = (CHAIN / 2 + 4) * U + 0.5 * (off * rstd) ** 2
    u = d * rstd * ws + bs
    tol_u = np.abs(ws) * (rstd * (off + U * np.abs(d)) + np.abs(d * rstd) * (slack + 2 * U)) + 2 * U * (np.abs(d * rstd * ws) + np.abs(bs))
    out = act(kind, u)
    # (exp, erf and the quotient: 6 roundings of what they act on, 0.5 u (1 + erf) has one of u itself)
    tol = 1.13 * tol_u + 6 * U * np.abs(u)
    return (out, mean[:, 0, :, 0], rstd[:, 0, :, 0]), (tol, off[:, 0, :, 0], (rstd * slack)[:, 0, :, 0])


def backward(shape, x, w, b, kind, mean, rstd, dy):
    """x, weight and bias gradients from the statistics that the forward call left, and their tolerances"""
    xs, ws, bs, g = split(x, shape), channelwise(w, shape, 1.0), channelwise(b, shape, 0.0), split(dy, shape)
    m, r = spread(mean, shape), spread(rstd, shape)
    hat = (xs - m) * r
    u = hat * ws + bs
    tol_u = 3 * U * np.abs(hat * ws) + U * np.abs(u)
    gu = g * slope(kind, u)
    tol_g = np.abs(g) * ((0.8 * tol_u if kind != RELU else 0) + 8 * U * (1 + np.abs(u)) * (kind != NONE)) + U * np.abs(gu)
    gx = gu * ws
    tol_gx = np.abs(ws) * tol_g + U * np.abs(gx)
    means = lambda v: v.mean(axis=(1, 3), keepdims=True)  # noqa: E731
    ga, gb = means(gx), means(gx * hat)
    tol_a = means(tol_gx) + CHAIN * U * means(np.abs(gx))
    tol_b = means(tol_gx * np.abs(hat) + 3 * U * np.abs(gx * hat)) + CHAIN * U * means(np.abs(gx * hat))
    dx = r * (gx - ga - hat * gb)
    tol_x = r * (tol_gx + tol_a + np.abs(hat) * tol_b + 5 * U * (np.abs(gx) + np.abs(ga) + np.abs(hat * gb)))
    sums = lambda v: v.sum(axis=(0, 1)).ravel()  # noqa: E731
    dw, db = sums(gu * hat), sums(gu)
    tol_w = sums(tol_g * np.abs(hat) + 3 * U * np.abs(gu * hat)) + CHAIN * U * sums(np.abs(gu * hat))
    tol_d = sums(tol_g) + CHAIN * U * sums(np.abs(gu))
    return (dx, dw, db), (tol_x, tol_w, tol_d)


def data(shape, kind, tag=0, offset=0.5):
    n, p, c, g = shape
    x = rng.normal(n * p * c, 1.0, tag=tag, seed=SEED).reshape(n, p, c)
    x = (x * np.exp(rng.uniform(c, -0.5, 0.5, tag=tag + 1, seed=SEED)) + offset * rng.normal(c, 1.0, tag=tag + 2, seed=SEED)).astype(np.float32)
    w = rng.uniform(c, 0.5, 1.5, tag=tag + 3, seed=SEED).astype(np.float32)
    b = rng.uniform(c, -0.5, 0.5, tag=tag + 4, seed=SEED).astype(np.float32)
    dy = rng.normal(n * p * c, 1.0, tag=tag + 5, seed=SEED).reshape(n, p, c).astype(np.float32)
    if kind == RELU:  # no gradient where the sign of u is a matter of rounding
        xs = split(x, shape)
        m = xs.mean(axis=(1, 3), keepdims=True)
        u = (xs - m) / np.sqrt(((xs - m) ** 2).mean(axis=(1, 3), keepdims=True) + 1e-5) * channelwise(w, shape, 1.0) + channelwise(b, shape, 0.0)
        dy[np.abs(u).reshape(dy.shape) < 1e-3] = 0
    return x, w, b, dy


def close(got, want, tol, what):
    got = np.asarray(got, np.float64).reshape(want.shape)
    off = np.abs(got - want)
    bad = ~(off <= tol + 1e-37)
    assert not bad.any(), (what, int(bad.sum()), float(np.nanmax(off / (tol + 1e-37))), np.argwhere(bad)[:3].tolist())


# samples, positions, channels, groups
SHAPES = [(1, 1, 8, 1), (1, 1, 1, 1), (4, 1, 64, 4), (64, 1, 512, 8), (7, 1, 390, 13), (3, 1, 1001, 7), (5, 1, 2048, 1), (2, 1, 5000, 1),
          (1, 1, 20000, 1), (1, 1, 9001, 1), (600, 1, 48, 3), (3000, 1, 10, 5), (2, 9, 32, 4), (3, 49, 30, 2), (2, 64, 96, 32), (1, 961, 390, 13),
          (2, 1024, 64, 8), (5, 333, 12, 12), (1, 5000, 16, 4), (1, 2500, 6, 2), (2, 17, 4096, 2), (1, 40, 3000, 1), (30, 25, 7, 7), (1, 1, 4, 4),
          (2, 3, 2600, 1), (1, 16400, 3, 1), (9, 100, 1024, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [NONE, RELU, SILU, GELU])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_backward(hip, shape, kind):
    say("group norm", shape, kind)
    x, w, b, dy = data(shape, kind)
    out, mean, rstd = hip.group_norm(*shape, x, w, b, act=kind)
    for got, want, tol, what in zip((out, mean, rstd), *forward(shape, x, w, b, kind, 1e-5), ("out", "mean", "rstd")):
        close(got, want, tol, what)
    outs = [np.full(x.size, np.nan, np.float32), np.full(shape[2], np.nan, np.float32), np.full(shape[2], np.nan, np.float32)]
    hip.group_norm_grad(*shape, x, w, b, mean, rstd, dy, *outs, act=kind)
    for got, want, tol, what in zip(outs, *backward(shape, x, w, b, kind, mean, rstd, dy), ("x", "weight", "bias")):
        close(got, want, tol, what)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(3, 1, 96, 4), (2, 50, 36, 3), (1, 3000, 10, 2), (2, 4, 2100, 1)])
def test_optional_arguments_and_accumulation(hip, shape):
    say("group norm optional", shape)
    x, w, b, dy = data(shape, SILU, tag=10)
    out, mean, rstd = hip.group_norm(*shape, x, None, None, act=SILU)
    want, tol = forward(shape, x, None, None, SILU, 1e-5)
    close(out, want[0], tol[0], "out")
    c = hip.ctx()
    dx, do = c.array(x), c.empty(x.size)
    c.call("slhip_group_norm", *shape, SILU, 1e-5, dx.ptr, None, None, None, None, do.ptr)        # statistics not kept
    assert np.array_equal(do.numpy(), out)
    c.call("slhip_group_norm", *shape, SILU, 1e-5, dx.ptr, None, None, None, None, dx.ptr)        # in place
    assert np.array_equal(dx.numpy(), out)
    dx.free(), do.free()
    lens = (x.size, shape[2], shape[2])
    want, tol = backward(shape, x, None, None, SILU, mean, rstd, dy)
    for only in range(3):
        outs = [np.full(lens[k], np.nan, np.float32) if k == only else None for k in range(3)]
        hip.group_norm_grad(*shape, x, None, None, mean, rstd, dy, *outs, act=SILU)
        close(outs[only], want[only], tol[only], only)
    old = [rng.normal(n, 1.0, tag=20 + k, seed=SEED).astype(np.float32) for k, n in enumerate(lens)]
    outs = [o.copy() for o in old]
    hip.group_norm_grad(*shape, x, None, None, mean, rstd, dy, *outs, act=SILU, beta=1.0)
    for got, before, v, t in zip(outs, old, want, tol):
        v = v + before.reshape(v.shape)
        close(got, v, t + U * np.abs(v) * 1.01, "beta 1")
    # x_grad over out_grad
    bufs = [c.array(a) for a in (x, mean, rstd, dy)]
    c.call("slhip_group_norm_grad", *shape, SILU, bufs[0].ptr, None, None, bufs[1].ptr, bufs[2].ptr, bufs[3].ptr, None, None, bufs[3].ptr, 0.0)
    close(bufs[3].numpy(), want[0], tol[0], "over out_grad")
    for k in bufs:
        k.free()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 1, 64, 2), (2, 400, 24, 3), (1, 1, 6000, 1)])
def test_groups_far_from_zero_keep_their_variance(hip, shape):
    """A mean a thousand times the deviation, and one value a thousand times the others: the variance is taken from
    differences, so neither costs more than the rounding of x itself."""
    x, w, b, _ = data(shape, NONE, tag=30, offset=0.0)
    far = (x + 1000).astype(np.float32)
    out, mean, rstd = hip.group_norm(*shape, far, w, b)
    for got, want, tol in zip((out, mean, rstd), *forward(shape, far, w, b, NONE, 1e-5)):
        close(got, want, tol, "far")
    x[0, 0, 0] = 1000.0
    out, mean, rstd = hip.group_norm(*shape, x, w, b)
    for got, want, tol in zip((out, mean, rstd), *forward(shape, x, w, b, NONE, 1e-5)):
        close(got, want, tol, "spike")


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 1, 64, 2), (2, 30, 12, 3), (1, 2000, 8, 2)])
def test_constant_groups_and_nan(hip, shape):
    x = np.full(shape[:3], 3.0, np.float32)
    w, b = np.full(shape[2], 2.0, np.float32), np.full(shape[2], 0.25, np.float32)
    out, mean, rstd = hip.group_norm(*shape, x, w, b)
    assert (out == 0.25).all() and (mean == 3).all() and np.allclose(rstd, 1e-5 ** -0.5, rtol=4 * U)
    x = data(shape, NONE, tag=40)[0]
    x[0, 0, 0] = np.nan                                    # one group of one sample
    out, mean, rstd = hip.group_norm(*shape, x, w, b)
    hit = np.isnan(out).reshape(shape[0], shape[1], shape[3], -1)
    assert hit[0, :, 0].all() and hit.sum() == hit[0, :, 0].size and np.isnan(mean).sum() == 1


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [SILU, GELU])
def test_activations_far_out(hip, kind):
    """Weights from 10^-4 to 10^20: where the function is its argument, and where it is next to nothing."""
    shape = (6, 1, 125, 1)
    x, _, b, dy = data(shape, kind, tag=48)
    w = (10.0 ** np.linspace(-4, 20, 125)).astype(np.float32)
    out, mean, rstd = hip.group_norm(*shape, x, w, b, act=kind)
    (want, _, _), (tol, _, _) = forward(shape, x, w, b, kind, 1e-5)
    close(out, want, tol, "forward")
    outs = [np.zeros(x.size, np.float32), np.zeros(125, np.float32), np.zeros(125, np.float32)]
    hip.group_norm_grad(*shape, x, w, b, mean, rstd, dy, *outs, act=kind)
    assert all(np.isfinite(o).all() for o in outs)
    b[3], b[4] = np.inf, np.nan                            # in a bias they stay in their channel
    got = hip.group_norm(*shape, x, w, b, act=kind)[0].reshape(6, 125)
    assert (got[:, 3] == np.inf).all() and np.isnan(got[:, 4]).all()
    assert np.array_equal(np.delete(got, (3, 4), axis=1), np.delete(out.reshape(6, 125), (3, 4), axis=1))


@pytest.mark.gpu
def test_gradients_against_differences(hip):
    shape = (2, 3, 6, 2)
    for kind in (NONE, SILU, GELU):
        x, w, b, dy = data(shape, kind, tag=50)
        out, mean, rstd = hip.group_norm(*shape, x, w, b, act=kind)
        outs = [np.zeros(x.size, np.float32), np.zeros(6, np.float32), np.zeros(6, np.float32)]
        hip.group_norm_grad(*shape, x, w, b, mean, rstd, dy, *outs, act=kind)
        at = [v.astype(np.float64) for v in (x, w, b)]

        def loss():
            return (forward(shape, *at, kind, 1e-5)[0][0] * split(dy, shape)).sum()

        for k in range(3):
            flat = at[k].reshape(-1)
            for i in range(flat.size):
                keep = flat[i]
                flat[i] = keep + 1e-5
                up = loss()
                flat[i] = keep - 1e-5
                down = loss()
                flat[i] = keep
                assert abs((up - down) / 2e-5 - outs[k][i]) <= 2e-5 * (1 + abs(outs[k][i])), (kind, k, i)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(5, 1, 96, 3), (3, 33, 20, 5), (1, 1100, 9, 3)])
def test_float_aligned_operands_and_untouched_surroundings(hip, shape):
    x, w, b, dy = data(shape, GELU, tag=60)
    hip.operands_off_the_vector_grid(True)
    try:
        out, mean, rstd = hip.group_norm(*shape, x, w, b, act=GELU)
        for got, want, tol in zip((out, mean, rstd), *forward(shape, x, w, b, GELU, 1e-5)):
            close(got, want, tol, "forward")
        outs = [np.zeros(x.size, np.float32), np.zeros(shape[2], np.float32), np.zeros(shape[2], np.float32)]
        hip.group_norm_grad(*shape, x, w, b, mean, rstd, dy, *outs, act=GELU)
        for got, want, tol in zip(outs, *backward(shape, x, w, b, GELU, mean, rstd, dy)):
            close(got, want, tol, "backward")
    finally:
        hip.operands_off_the_vector_grid(False)
    c = hip.ctx()
    pools = [c.array(np.full(n + 14, 7.0, np.float32)) for n in (x.size, shape[0] * shape[3], shape[0] * shape[3], shape[2], shape[2])]
    ins = [c.array(a) for a in (x, w, b, dy)]
    at = [p.ptr + 28 for p in pools]
    c.call("slhip_group_norm", *shape, GELU, 1e-5, ins[0].ptr, ins[1].ptr, ins[2].ptr, at[1], at[2], at[0])
    c.call("slhip_group_norm_grad", *shape, GELU, ins[0].ptr, ins[1].ptr, ins[2].ptr, at[1], at[2], at[0], at[3], at[4], ins[3].ptr, 0.0)
    for p in pools:
        got = p.numpy()
        assert (got[:7] == 7).all() and (got[-7:] == 7).all() and not (got[7:-7] == 7).any()
    for k in pools + ins:
        k.free()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(7, 1, 390, 13), (3, 1, 1001, 7), (2, 1, 9000, 1), (2, 9, 32, 4), (5, 333, 12, 12), (1, 5000, 16, 4), (2, 3, 2600, 1)])
def test_outputs_over_inputs_equal_separate_ones(hip, shape):
    x, w, b, dy = data(shape, SILU, tag=63)
    out, mean, rstd = hip.group_norm(*shape, x, w, b, act=SILU)
    want = [np.zeros(x.size, np.float32), np.zeros(shape[2], np.float32), np.zeros(shape[2], np.float32)]
    hip.group_norm_grad(*shape, x, w, b, mean, rstd, dy, *want, act=SILU)
    c = hip.ctx()
    X, W, B, M, R, G = [c.array(a) for a in (x, w, b, mean, rstd, dy)]
    GW, GB = c.empty(shape[2]), c.empty(shape[2])
    c.call("slhip_group_norm_grad", *shape, SILU, X.ptr, W.ptr, B.ptr, M.ptr, R.ptr, G.ptr, GW.ptr, GB.ptr, G.ptr, 0.0)
    for got, k in zip((G, GW, GB), want):
        assert np.array_equal(got.numpy(), k)
    c.call("slhip_group_norm", *shape, SILU, 1e-5, X.ptr, W.ptr, B.ptr, M.ptr, R.ptr, X.ptr)
    for got, k in zip((X, M, R), (out, mean, rstd)):
        assert np.array_equal(got.numpy(), k)
    for k in (X, W, B, M, R, G, GW, GB):
        k.free()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 200000, 4, 1), (1, 3000, 8, 2), (3, 1, 512, 1)])
def test_one_value_far_from_the_rest(hip, shape):
    """A group whose first value is 10^6 standard deviations of the rest away: it is nearly all of the variance, and the sums
    of squares taken around it, or around any other value, must not lose the mean."""
    x = rng.normal(int(np.prod(shape[:3])), 1.0, tag=67, seed=SEED).reshape(shape[:3]).astype(np.float32)
    for n in range(shape[0]):
        x[n, 0, ::shape[2] // shape[3]] = 1e6
    (want, mean, rstd), (tol, tm, tr) = forward(shape, x, None, None, NONE, 1e-5)
    got, m, r = hip.group_norm(*shape, x)
    size = shape[1] * shape[2] // shape[3]
    # the mean is off by a few roundings of the sums' largest terms, 1e6 / size, 1/sqrt(var) by some of itself
    assert np.abs(m.reshape(mean.shape) - mean).max() <= 64 * U * 1e6 / min(size, 512)
    assert np.abs(r.reshape(rstd.shape) / rstd - 1).max() <= 64 * U


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(40, 1, 128, 4), (4, 700, 24, 2), (8, 16, 64, 8)])
def test_recorded_calls_replay_like_the_eager_ones(hip, shape):
    c = hip.ctx()
    x, w, b, dy = data(shape, SILU, tag=70)
    ins = [c.array(a) for a in (x, w, b, dy)]
    outs = [c.empty(n) for n in (x.size, shape[0] * shape[3], shape[0] * shape[3], x.size, shape[2], shape[2])]
    o, m, r, gx, gw, gb = [k.ptr for k in outs]
    c.sync()
    c.call("slhip_graph_begin")
    try:
        c.call("slhip_group_norm", *shape, SILU, 1e-5, ins[0].ptr, ins[1].ptr, ins[2].ptr, m, r, o)
        c.call("slhip_group_norm_grad", *shape, SILU, ins[0].ptr, ins[1].ptr, ins[2].ptr, m, r, gx, gw, gb, ins[3].ptr, 0.0)
    finally:
        graph = C.c_void_p()
        c.call("slhip_graph_end", C.byref(graph))
    for replay in range(3):
        say("replay", replay)
        now = (x + replay * dy).astype(np.float32)
        ins[0].upload(now)
        c.call("slhip_graph_launch", graph)
        got = [k.numpy() for k in outs]
        want = list(hip.group_norm(*shape, now, w, b, act=SILU))
        grads = [np.zeros(x.size, np.float32), np.zeros(shape[2], np.float32), np.zeros(shape[2], np.float32)]
        hip.group_norm_grad(*shape, now, w, b, want[1], want[2], dy, *grads, act=SILU)
        for a, k in zip(got, want + grads):
            assert np.array_equal(a, k), replay
    c.lib.slhip_graph_destroy(graph)
    for k in ins + outs:
        k.free()


def refused(lib, ctx):
    p = C.addressof(C.create_string_buffer(64))
    big = 1 << 62
    call, grad = lib.slhip_group_norm, lib.slhip_group_norm_grad
    assert call(None, 1, 1, 4, 2, 0, 1e-5, p, p, p, p, p, p) == -1
    for bad in ((0, 1, 4, 2, 0), (1, 0, 4, 2, 0), (1, 1, 0, 2, 0), (1, 1, 4, 0, 0), (1, 1, 4, 3, 0), (1, 1, 4, 8, 0), (1, 1, 4, 2, 4), (1, 1, 4, 2, -1),
                (big, 4, 4, 2, 0), (1, big, 4, 2, 0), (2, 1, big, 2, 0)):
        assert call(ctx, *bad, 1e-5, p, p, p, p, p, p) == -1, bad
        assert grad(ctx, *bad, p, p, p, p, p, p, p, p, p, 0.0) == -1, bad
    assert call(ctx, 1, 1, 4, 2, 0, -1e-5, p, p, p, p, p, p) == -1
    assert call(ctx, 1, 1, 4, 2, 0, float("nan"), p, p, p, p, p, p) == -1
    assert call(ctx, 1, 1, 4, 2, 0, 1e-5, None, p, p, p, p, p) == -1
    assert call(ctx, 1, 1, 4, 2, 0, 1e-5, p, p, p, p, p, None) == -1
    for k in (0, 3, 4, 8):
        args = [p] * 9
        args[k] = None
        assert grad(ctx, 1, 1, 4, 2, 0, *args, 0.0) == -1, k
    assert grad(ctx, 1, 1, 4, 2, 0, p, p, p, p, p, None, None, None, p, 0.0) == 0  # nothing asked for
    for bad in ((1, 1, 1 << 31, 1, 0), (1, 1, 1 << 33, 1 << 32, 0)):
        assert call(ctx, *bad, 1e-5, p, None, None, None, None, p + (1 << 40)) == -1, bad
        assert grad(ctx, *bad, p, None, None, p, p, p + (1 << 40), None, None, p, 0.0) == -1, bad
    # x, weight, bias, mean, rstd, out: four floats each; an output over anything but x is refused
    q = [p + 16 * k for k in range(9)]
    for k in (3, 4, 5):
        for other in range(6):
            if other != k and (k, other) != (5, 0):
                args = q[:6]
                args[k] = q[other]
                assert call(ctx, 2, 1, 2, 1, 0, 1e-5, *args) == -4, (k, other)
    assert call(ctx, 2, 1, 2, 1, 0, 1e-5, *q[:5], q[0] + 4) == -4
    for k in (5, 6, 7):
        for other in range(9):
            if other != k and (k, other) != (5, 8):
                args = list(q)
                args[k] = q[other]
                assert grad(ctx, 2, 1, 2, 1, 0, *args, 0.0) == -4, (k, other)
    assert grad(ctx, 2, 1, 2, 1, 0, *q[:5], q[8] + 4, q[6], q[7], q[8], 0.0) == -4


def test_refusals_come_before_anything_touches_the_device():
    from sliced_amd import _lib
    blank = C.create_string_buffer(4096)
    refused(_lib.load(), C.addressof(blank))


@pytest.mark.gpu
def test_refusals(hip):
    refused(hip.ctx().lib, hip.ctx().h)
