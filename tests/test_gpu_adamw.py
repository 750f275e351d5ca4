"""AdamW over many tensors, with its moments in f32 and in 8 bits, through the C ABI.

f32 moments against the formula in 64 bits: with u = 2^-24, m and v round three times each; the update m / (sqrt(v) * root +
eps) * size has the roundings of m, of v (halved by the root), and six of its own.
8-bit moments: m and v before rounding are the 32-bit operations of the formula one by one (no fused ones), so the codes
and scales are compared bit for bit with the same operations in numpy, and the parameters with the 64-bit formula."""
import ctypes as C

import numpy as np
import pytest
import torch

from sliced_amd import rng

U = 2.0 ** -24
SEED = 0x51CED
HYPER = dict(lr=1e-2, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.1)


def say(*a):
    print(*a, flush=True)


def f32(v):
    return float(np.float32(v))


def exact(p, g, m, v, step, lr, beta1, beta2, eps, weight_decay):
    """(p, m, v) in 64 bits and their tolerances"""
    lr, b1, b2, eps, wd = (f32(k) for k in (lr, beta1, beta2, eps, weight_decay))
    p, g, m, v = (a.astype(np.float64) for a in (p, g, m, v))
    tm = 3 * U * (np.abs(b1 * m) + np.abs((1 - b1) * g))
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    root = np.sqrt(v / (1 - b2 ** step))
    size = lr / (1 - b1 ** step)
    up = size * m / (root + eps)
    tp = 2 * U * np.abs(p) + 10 * U * np.abs(up) + np.where(root + eps > 0, size * tm / (root + eps), 0)
    p = p * (1 - lr * wd) - up
    return (p, m, v), (tp + U * np.abs(p), tm, 5 * U * v)


def close(got, want, tol, what):
    off = np.abs(np.asarray(got, np.float64) - want)
    bad = ~(off <= tol + 1e-37)
    assert not bad.any(), (what, int(bad.sum()), float(np.nanmax(off / (tol + 1e-37))), np.argwhere(bad)[:3].tolist())


def tensors(lens, tag=0):
    def make(k, fn):
        return [fn(n, tag + 8 * i + k).astype(np.float32) for i, n in enumerate(lens)]
    p = make(0, lambda n, t: rng.normal(n, 1.0, tag=t, seed=SEED))
    g = make(1, lambda n, t: rng.normal(n, 1.0, tag=t, seed=SEED) * np.exp(rng.uniform(n, -8, 2, tag=t + 4, seed=SEED)))
    m = make(2, lambda n, t: rng.normal(n, 0.3, tag=t, seed=SEED))
    v = make(3, lambda n, t: rng.uniform(n, 0.0, 1.0, tag=t, seed=SEED) ** 4)
    return p, g, m, v


LENS = [[1], [3, 1, 2], [255, 256, 257], [2048], [2047, 2049, 4096, 4097, 8191], [64, 64, 4096, 64, 64, 1], [100003], [5] * 63, [7] * 64, [9] * 65,
        [i % 37 + 1 for i in range(200)], [1 << 20, 3, 70001]]


@pytest.mark.gpu
@pytest.mark.parametrize("lens", LENS, ids=lambda v: "%dx%d" % (len(v), max(v)))
def test_f32_moments(hip, lens):
    say("adamw", len(lens), max(lens))
    p, g, m, v = tensors(lens)
    for step in (1, 2, 1000):
        before = [[a.copy() for a in k] for k in (p, m, v)]
        hip.adamw_step_multi(p, g, m, v, step=step, **HYPER)
        for i in range(len(lens)):
            want, tol = exact(before[0][i], g[i], before[1][i], before[2][i], step, **HYPER)
            for got, w, t, what in zip((p[i], m[i], v[i]), want, tol, "pmv"):
                close(got, w, t, (step, i, what))


@pytest.mark.gpu
def test_first_step_and_hyperparameters(hip):
    """From zero moments the first step is lr * sign(g) and the decay; beta = 0, eps = 0 and weight_decay = 0 are allowed."""
    n = 1000
    p0, g = rng.normal(n, 1.0, tag=1, seed=SEED).astype(np.float32), rng.normal(n, 1.0, tag=2, seed=SEED).astype(np.float32)
    for hyper in (HYPER, dict(HYPER, beta1=0.0), dict(HYPER, beta2=0.0), dict(HYPER, eps=0.0, weight_decay=0.0), dict(HYPER, lr=0.0)):
        p, m, v = [p0.copy()], [np.zeros(n, np.float32)], [np.zeros(n, np.float32)]
        hip.adamw_step_multi(p, [g], m, v, step=1, **hyper)
        want, tol = exact(p0, g, np.zeros(n), np.zeros(n), 1, **hyper)
        close(p[0], want[0], tol[0], hyper)
        lr = f32(hyper["lr"])
        assert np.allclose(p[0] - p0 * (1 - lr * f32(hyper["weight_decay"])), -lr * np.sign(g), atol=1e-5 * lr + 4 * U * np.abs(p0).max())


@pytest.mark.gpu
def test_special_values(hip):
    """An infinite or NaN gradient spoils its own element; zero gradients with zero moments leave p but for the decay."""
    n = 777
    p0 = rng.normal(n, 1.0, tag=3, seed=SEED).astype(np.float32)
    for eight in (False, True):
        p, g = [p0.copy()], [np.zeros(n, np.float32)]
        g[0][[5, 300, 776]] = np.inf, np.nan, -np.inf
        if eight:
            state = [np.zeros(n, np.uint8)], [np.zeros(n, np.uint8)], [np.zeros(8, np.float32)]
            step, calls = hip.adamw8_step_multi, 2
        else:
            state = [np.zeros(n, np.float32)], [np.zeros(n, np.float32)]
            step, calls = hip.adamw_step_multi, 2
        for t in range(calls):
            step(p, g, *state, step=t + 1, **HYPER)
        bad = np.zeros(n, bool)
        bad[[5, 300, 776]] = True
        assert np.isnan(p[0][bad]).all()
        keep = np.float32(1 - f32(0.1) * f32(1e-2))
        assert np.array_equal(p[0][~bad], (p0 * keep * keep)[~bad])
        if eight:
            assert (state[0][0][~bad] == 0).all() and (state[1][0][~bad] == 0).all()
            assert all(c in (0x7f, 0xff) for c in state[0][0][bad]) and list(state[1][0][[5, 776]]) == [0x7c, 0x7c]


# ---------------------------------------------------------------- 8-bit moments
def mix(z):
    with np.errstate(over="ignore"):
        return rng._splitmix64(np.asarray(z, np.uint64))


def random16(n, ordinal, step, seed):
    with np.errstate(over="ignore"):
        key = mix(mix(np.uint64((seed + step) & (2 ** 64 - 1))) + np.uint64(ordinal))
        word = mix(key + np.arange((n + 3) // 4, dtype=np.uint64))
    return ((word[:, None] >> (np.uint64(16) * np.arange(4, dtype=np.uint64))) & np.uint64(0xFFFF)).ravel()[:n].astype(np.uint32)


def blocks(a):
    return np.concatenate([a, np.zeros(-a.size % 256, a.dtype)]).reshape(-1, 256)


def scale_of(x, top):
    e = (np.abs(x).view(np.uint32) >> 23).astype(np.int64)
    e = blocks(np.where(e == 255, 0, e)).max(axis=1)
    return (np.maximum(e - top, 1) << 23).astype(np.uint32).view(np.float32)


def decode(m8, v8, scales):
    n = m8.size
    per = np.repeat(scales.reshape(-1, 2), 256, axis=0)[:n]
    m = torch.from_numpy(m8.copy()).view(torch.float8_e4m3fn).float().numpy()
    v = torch.from_numpy(v8.copy()).view(torch.float8_e5m2).float().numpy()
    return m * per[:, 0], v * per[:, 1]


def encode(m, v, r16):
    sm, sv = scale_of(m, 7), scale_of(v, 14)
    n = m.size
    x = m / np.repeat(sm, 256)[:n]
    y = v / np.repeat(sv, 256)[:n]
    cut = ((y.view(np.uint32) + (r16 << 5)) & ~np.uint32(0x1FFFFF)).view(np.float32)
    y = np.where(y > 0, np.maximum(cut, np.float32(2.0 ** -16)), y).astype(np.float32)
    m8 = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    v8 = torch.from_numpy(y).to(torch.float8_e5m2).view(torch.uint8).numpy()
    return m8, v8, np.stack([sm, sv], axis=1).ravel()


def zeros8(lens):
    return ([np.zeros(n, np.uint8) for n in lens], [np.zeros(n, np.uint8) for n in lens],
            [np.zeros(2 * ((n + 255) // 256), np.float32) for n in lens])


@pytest.mark.gpu
@pytest.mark.parametrize("lens", LENS, ids=lambda v: "%dx%d" % (len(v), max(v)))
def test_8_bit_moments(hip, lens):
    say("adamw8", len(lens), max(lens))
    p, g, _, _ = tensors(lens, tag=20)
    m8, v8, scales = zeros8(lens)
    b1, b2 = np.float32(0.9), np.float32(0.999)
    for step in (1, 2, 3, 500):
        before = [[a.copy() for a in k] for k in (p, m8, v8, scales)]
        hip.adamw8_step_multi(p, g, m8, v8, scales, step=step, seed=SEED, **HYPER)
        for i, n in enumerate(lens):
            m, v = decode(before[1][i], before[2][i], before[3][i])
            want, tol = exact(before[0][i], g[i], m, v, step, **HYPER)
            close(p[i], want[0], tol[0], (step, i, "p"))
            m = m * b1 + g[i] * (np.float32(1) - b1)
            v = v * b2 + (g[i] * (np.float32(1) - b2)) * g[i]
            for got, w, what in zip((m8[i], v8[i], scales[i]), encode(m, v, random16(n, i, step, SEED)), ("m8", "v8", "scales")):
                assert np.array_equal(got, w), (step, i, what, int((got != w).sum()))
        for k in g:
            k *= np.float32(0.5)                      # the largest of a block, and with it its scale, changes


def test_rounding_of_the_8_bit_moments():
    """The oracle's own rounding: m to half a step of E4M3 (2^-4, or 2^-10 of the scale for the smallest), v by less than a
    step of E5M2 and right on average, neither past the format's end, no v that is not zero to zero."""
    n = 1 << 16
    m = (rng.normal(n, 1.0, tag=1, seed=SEED) * np.exp(rng.uniform(n, -6, 3, tag=2, seed=SEED))).astype(np.float32)
    v = (rng.uniform(n, 0, 1, tag=3, seed=SEED) ** 8).astype(np.float32)
    sums = 0.0
    for step in range(8):
        m8, v8, scales = encode(m, v, random16(n, 0, step, SEED))
        dm, dv = decode(m8, v8, scales)
        per = np.repeat(scales.reshape(-1, 2), 256, axis=0).astype(np.float64)
        assert np.isfinite(dm).all() and np.isfinite(dv).all()
        assert (np.abs(dm - m) <= np.maximum(2.0 ** -4 * np.abs(m), 2.0 ** -10 * per[:, 0])).all()
        assert (np.abs(dv.astype(np.float64) - v) <= np.maximum(0.25 * v, 2.0 ** -16 * per[:, 1])).all()
        assert (dv[v > 0] > 0).all() and (np.abs(dm).reshape(-1, 256).max(axis=1) > 0).all()
        sums += dv.astype(np.float64)
    # eight independent roundings of 65536 values, each off by at most a quarter of the value: five deviations
    assert abs(sums.sum() / 8 - v.sum(dtype=np.float64)) <= 5 * 0.25 * np.sqrt((v.astype(np.float64) ** 2).sum() / 8)


@pytest.mark.gpu
def test_8_bit_v_decays_on_average(hip):
    """With no gradient v falls by 0.1 % a step, far less than the spacing of E5M2: 300 steps take it to 0.999^300 = 0.741 on
    average.  64 Ki values that move in steps of at most a quarter: the mean of their relative deviations, each below
    0.25 sqrt(300 * 0.004) = 0.27, is within 5 * 0.27 / 256 of zero."""
    n = 1 << 16
    p, g = [np.zeros(n, np.float32)], [rng.uniform(n, 1.0, 2.0, tag=9, seed=SEED).astype(np.float32)]
    m8, v8, scales = zeros8([n])
    hip.adamw8_step_multi(p, g, m8, v8, scales, step=1, seed=SEED, **HYPER)
    start = decode(m8[0], v8[0], scales[0])[1].astype(np.float64)
    c = hip.ctx()
    bufs = [c.array(a) for a in (p[0], np.zeros(n, np.float32), m8[0].view(np.float32), v8[0].view(np.float32), scales[0])]
    arrays = [(C.c_void_p * 1)(b.ptr) for b in bufs]
    lens = (C.c_size_t * 1)(n)
    for t in range(2, 302):
        c.call("slhip_adamw8_step_multi", 1, *arrays, lens, 1e-2, 0.9, 0.999, 1e-8, 0.1, t, None, SEED)
    v = decode(bufs[2].numpy().view(np.uint8), bufs[3].numpy().view(np.uint8), bufs[4].numpy())[1].astype(np.float64)
    for b in bufs:
        b.free()
    assert abs((v / start).mean() - f32(0.999) ** 300) <= 5 * 0.27 / 256


@pytest.mark.gpu
def test_8_bit_training_follows_the_f32_one(hip):
    """The same problem (a least-squares fit) with both kinds of moments, from the same start: no step of the 8-bit run leaves
    the size of a step of the f32 run by more than the moments' roundings allow (m by 2^-4, v by a quarter, so the step by 25 %)."""
    n = 3000
    g0 = rng.normal(n, 1.0, tag=30, seed=SEED).astype(np.float32)
    a, b = [np.zeros(n, np.float32)], [np.zeros(n, np.float32)]
    m, v = [np.zeros(n, np.float32)], [np.zeros(n, np.float32)]
    state = zeros8([n])
    for t in range(1, 4):
        hip.adamw_step_multi(a, [g0], m, v, lr=1e-2, weight_decay=0.0, step=t)
        before = b[0].copy()
        hip.adamw8_step_multi(b, [g0], *state, lr=1e-2, weight_decay=0.0, step=t, seed=SEED)
        # gradients below 2^-13 of their block's largest are E4M3 subnormals, rounded to as much as twice themselves
        moved = np.abs(b[0] - before)
        assert (moved <= 2.5e-2).all()
        strong = np.abs(g0) > 2.0 ** -6
        assert (np.abs(moved[strong] - 1e-2) <= 0.25e-2).all()


# ---------------------------------------------------------------- counters, recordings, surroundings
@pytest.mark.gpu
@pytest.mark.parametrize("eight", [False, True])
def test_device_counter_and_recording(hip, eight):
    """The counter on the device gives the steps of the counted calls bit for bit, eager and replayed."""
    lens = [700, 3, 2600]
    p, g, m, v = tensors(lens, tag=40)
    if eight:
        m, v, scales = zeros8(lens)
    want = [[a.copy() for a in k] for k in ((p, m, v, scales) if eight else (p, m, v))]
    c = hip.ctx()

    def up(a):
        return c.array(a) if a.dtype == np.float32 else c.array(np.concatenate([a, np.zeros(-a.size % 4, np.uint8)]).view(np.float32))

    dev = [[up(a) for a in k] for k in ((p, g, m, v, scales) if eight else (p, g, m, v))]
    arrays = [(C.c_void_p * 3)(*[b.ptr for b in k]) for k in dev]
    sizes = (C.c_size_t * 3)(*lens)
    counter = c.zeros(2)
    hyper = [HYPER[k] for k in ("lr", "beta1", "beta2", "eps", "weight_decay")]
    name = "slhip_adamw8_step_multi" if eight else "slhip_adamw_step_multi"
    tail = [SEED] if eight else []

    def expect(step):
        if eight:
            hip.adamw8_step_multi(want[0], g, want[1], want[2], want[3], step=step, seed=SEED, **HYPER)
        else:
            hip.adamw_step_multi(want[0], g, want[1], want[2], step=step, **HYPER)
        got = [[b.numpy() for b in k] for i, k in enumerate(dev) if i != 1]
        for i, k in enumerate(got):
            for a, b in zip(k, want[i]):
                a = a.view(np.uint8)[:b.size] if b.dtype == np.uint8 else a
                assert np.array_equal(a, b), (step, i)
        assert counter.numpy().view(np.uint64)[0] == step

    for step in (1, 2):
        c.call(name, 3, *arrays, sizes, *hyper, 0, counter.ptr, *tail)
        expect(step)
    c.sync()
    c.call("slhip_graph_begin")
    try:
        c.call(name, 3, *arrays, sizes, *hyper, 0, counter.ptr, *tail)
    finally:
        graph = C.c_void_p()
        c.call("slhip_graph_end", C.byref(graph))
    for step in (3, 4, 5):
        say("replay", step)
        c.call("slhip_graph_launch", graph)
        expect(step)                                  # reads back and runs eager steps in between
    c.lib.slhip_graph_destroy(graph)
    for k in dev:
        for b in k:
            b.free()
    counter.free()


@pytest.mark.gpu
def test_tensors_side_by_side_and_float_aligned(hip):
    """Tensors that follow each other without a gap, at odd places of one allocation: each is stepped as it would be alone,
    and what lies around them stays as it was."""
    lens, gap = [5, 1, 1030, 258, 4099], 3
    total = sum(lens) + 2 * gap
    p, g, m, v = tensors(lens, tag=60)
    want = [[a.copy() for a in k] for k in (p, m, v)]
    hip.adamw_step_multi(want[0], g, want[1], want[2], step=5, **HYPER)
    c = hip.ctx()
    pools = [c.array(np.concatenate([np.full(gap, 7, np.float32)] + k + [np.full(gap, 7, np.float32)])) for k in (p, g, m, v)]
    starts = np.cumsum([gap] + lens[:-1])
    arrays = [(C.c_void_p * 5)(*[b.ptr + 4 * int(s) for s in starts]) for b in pools]
    c.call("slhip_adamw_step_multi", 5, *arrays, (C.c_size_t * 5)(*lens), *[HYPER[k] for k in ("lr", "beta1", "beta2", "eps", "weight_decay")], 5, None)
    for b, k in zip([pools[0]] + pools[2:], want):
        got = b.numpy()
        assert got.size == total and (got[:gap] == 7).all() and (got[-gap:] == 7).all()
        assert np.array_equal(got[gap:-gap], np.concatenate(k))
    # 8 bits: codes on a 4-byte grid, parameters and gradients anywhere
    m8, v8, scales = zeros8(lens)
    want = [[a.copy() for a in k] for k in (p, m8, v8, scales)]
    hip.adamw8_step_multi(want[0], g, want[1], want[2], want[3], step=5, seed=1, **HYPER)
    pools[0].upload(np.concatenate([np.full(gap, 7, np.float32)] + p + [np.full(gap, 7, np.float32)]))
    codes = [c.array(np.full(3000, 7, np.float32)) for _ in range(2)]
    at = np.cumsum([4] + [(n + 3) // 4 * 4 + 4 for n in lens[:-1]])
    for b in codes:
        host = np.full(12000, 7, np.uint8)
        for s, n in zip(at, lens):
            host[s:s + n] = 0
        b.upload(host.view(np.float32))
    sc = c.zeros(100)
    sat = np.cumsum([1] + [2 * ((n + 255) // 256) + 1 for n in lens[:-1]])
    arrays = arrays[:2] + [(C.c_void_p * 5)(*[b.ptr + int(s) for s in at]) for b in codes] + [(C.c_void_p * 5)(*[sc.ptr + 4 * int(s) for s in sat])]
    c.call("slhip_adamw8_step_multi", 5, *arrays, (C.c_size_t * 5)(*lens), *[HYPER[k] for k in ("lr", "beta1", "beta2", "eps", "weight_decay")], 5, None, 1)
    assert np.array_equal(pools[0].numpy()[gap:-gap], np.concatenate(want[0]))
    for b, k in zip(codes, want[1:3]):
        host, clean = b.numpy().view(np.uint8), np.full(12000, 7, np.uint8)
        for s, a in zip(at, k):
            clean[s:s + a.size] = a
        assert np.array_equal(host, clean)
    host, clean = sc.numpy(), np.zeros(100, np.float32)
    for s, a in zip(sat, want[3]):
        clean[s:s + a.size] = a
    assert np.array_equal(host, clean)
    for b in pools + codes + [sc]:
        b.free()


def refused(lib, ctx):
    room = C.create_string_buffer(1 << 12)
    at = (C.addressof(room) + 63) & ~63
    two = lambda a, b: (C.c_void_p * 2)(a, b)  # noqa: E731
    ok = [two(at, at + 64), two(at + 128, at + 192), two(at + 256, at + 320), two(at + 384, at + 448)]
    scales = two(at + 512, at + 576)
    lens = (C.c_size_t * 2)(16, 16)
    rates = [1e-3, 0.9, 0.999, 1e-8, 0.0]
    f, e = lib.slhip_adamw_step_multi, lib.slhip_adamw8_step_multi

    def both(want, arrays=ok, n=2, lens=lens, rates=rates, step=1, counter=None, sc=scales):
        assert f(ctx, n, *arrays, lens, *rates, step, counter) == want
        assert e(ctx, n, *arrays, sc, lens, *rates, step, counter, 0) == want

    assert f(None, 2, *ok, lens, *rates, 1, None) == -1 and e(None, 2, *ok, scales, lens, *rates, 1, None, 0) == -1
    both(-1, n=0)
    for k in range(4):
        both(-1, arrays=ok[:k] + [None] + ok[k + 1:])
        both(-1, arrays=ok[:k] + [two(at, None)] + ok[k + 1:])
    both(-1, lens=None)
    both(-1, lens=(C.c_size_t * 2)(16, 0))
    both(-1, lens=(C.c_size_t * 2)(16, (1 << 64) - 1))
    nan, inf = float("nan"), float("inf")
    for k, bad in ((0, nan), (0, inf), (1, 1.0), (1, -0.1), (1, nan), (2, 1.0), (2, -0.1), (2, nan), (3, -1e-8), (3, nan), (3, inf), (4, nan)):
        both(-1, rates=rates[:k] + [bad] + rates[k + 1:])
    both(-1, step=0)
    both(-1, step=1, counter=at + 640)
    both(-1, step=0, counter=at + 644)                                  # not on an 8-byte grid
    for k in (0, 2, 3):                                                 # the same tensor twice, and two that share a part
        both(-4, arrays=ok[:k] + [two(at, at)] + ok[k + 1:])
        both(-4, arrays=ok[:k] + [two(at, at + 12)] + ok[k + 1:])
    assert e(ctx, 2, *ok, two(at + 512, at + 516), lens, *rates, 1, None, 0) == -4
    both(-4, arrays=[ok[0], ok[0], ok[2], ok[3]])                       # gradients that are the parameters
    both(-4, arrays=[ok[0], ok[1], ok[3], ok[3]])                       # one set of moments for both
    both(-4, arrays=[ok[0], two(at + 128, at + 260), ok[2], ok[3]])     # a gradient that ends in a moment
    both(-1, arrays=[ok[0], two(at + 128, at + 132), ok[2], ok[3]], rates=[nan] + rates[1:])  # gradients may (it is the rate that is refused)
    assert e(ctx, 2, *ok, two(at + 512, at + 8), lens, *rates, 1, None, 0) == -4              # a scale inside a parameter
    # one parameter twice, further apart than the tensors of a launch
    many = [(C.c_void_p * 70)(*[at + 4 * (70 * k + i) for i in range(70)]) for k in range(5)]
    ones = (C.c_size_t * 70)(*[1] * 70)
    apart = [(C.c_void_p * 70)(*[at + 8 * (70 * k + i) for i in range(70)]) for k in range(5)]
    assert f(ctx, 70, *many[:4], ones, nan, *rates[1:], 1, None) == -1
    assert e(ctx, 70, *apart, ones, nan, *rates[1:], 1, None, 0) == -1
    many[0][69], apart[0][69] = many[0][2], apart[0][2]
    assert f(ctx, 70, *many[:4], ones, *rates, 1, None) == -4
    assert e(ctx, 70, *apart, ones, *rates, 1, None, 0) == -4
    both(-1, n=16385)
    assert e(ctx, 2, *ok[:2], two(at + 257, at + 320), ok[3], scales, lens, *rates, 1, None, 0) == -1
    assert e(ctx, 2, *ok, None, lens, *rates, 1, None, 0) == -1


def test_refusals_come_before_anything_touches_the_device():
    from sliced_amd import _lib
    blank = C.create_string_buffer(4096)
    refused(_lib.load(), C.addressof(blank))


@pytest.mark.gpu
def test_refusals(hip):
    refused(hip.ctx().lib, hip.ctx().h)
