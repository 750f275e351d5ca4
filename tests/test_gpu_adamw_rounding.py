"""The 8-bit second moment of AdamW over the whole of its format: below 2^-14 of a block's scale E5M2 is subnormal, its spacing
2^-16 whatever the value, and the stochastic rounding has to go by that spacing.

The moments before rounding are the 32-bit operations of the formula one by one, so codes and scales are compared bit for bit."""
import ctypes as C

import numpy as np
import pytest
import torch

import test_gpu_adamw as base
from sliced_amd import rng

SEED = base.SEED
HYPER = base.HYPER
SMALLEST, NORMAL = np.float32(2.0 ** -16), np.float32(2.0 ** -14)


def encode(m, v, r16):
    """base.encode with v rounded once, to a spacing of a quarter of its leading bit or of 2^-16: r16 / 2^16 of it is added
    before the rest is cut off"""
    sm, sv = base.scale_of(m, 7), base.scale_of(v, 14)
    x, y = m / np.repeat(sm, 256)[:m.size], v / np.repeat(sv, 256)[:m.size]
    low = np.where(y < NORMAL, NORMAL, np.float32(0))
    cut = (((y + low).view(np.uint32) + (r16 << 5)) & ~np.uint32(0x1FFFFF)).view(np.float32) - low
    y = np.where(v > 0, np.maximum(cut, SMALLEST), y).astype(np.float32)
    code = lambda a, kind: torch.from_numpy(a).to(kind)  # noqa: E731
    v8 = code(y, torch.float8_e5m2)
    assert np.array_equal(v8.float().numpy(), y, equal_nan=True)          # the conversion rounds nothing
    return code(x, torch.float8_e4m3fn).view(torch.uint8).numpy(), v8.view(torch.uint8).numpy(), np.stack([sm, sv], axis=1).ravel()


def gradients(n, tag):
    """Squares over 2^-40 .. 1 of their block's largest, which the first of every 256 holds."""
    g = rng.normal(n, 1.0, tag=tag, seed=SEED) * np.exp2(rng.uniform(n, -20, -4, tag=tag + 1, seed=SEED))
    g[::256] = 1.0
    return g.astype(np.float32)


def test_rounding_is_right_on_average_down_to_the_smallest_value():
    """Each value from one unit of 2^-16 to 2^-12 over 4096 random words that take every 16th place: within the step of the grid that
    does not depend on the word, and as often up as it is far from the lower neighbour (off by at most one word in 4096)."""
    words = np.arange(8, 1 << 16, 16, dtype=np.uint32)
    for y in np.float32(2.0 ** -16) * np.concatenate([np.linspace(1, 16, 61), [1.998, 3.996, 7.99, 15.98]]).astype(np.float32):
        v = np.full(words.size, y, np.float32)
        v[::256] = 2.0 ** 14                                              # (the block's largest, left out below)
        step = max(2.0 ** -16, 2.0 ** (np.floor(np.log2(float(y))) - 2))
        v8 = torch.from_numpy(encode(np.zeros_like(v), v, words)[1]).view(torch.float8_e5m2).double().numpy()
        v8, y = np.delete(v8.reshape(-1, 256), 0, axis=1).ravel(), float(y)
        lower = np.floor(y / step) * step
        assert set(v8) <= {lower, lower + step}
        # each block leaves out one word of 256, evenly spread: the count is off by at most one a block and one
        assert abs((v8 > lower).mean() - (y - lower) / step) <= 17 / v8.size, y / 2.0 ** -16


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[1], [257], [3, 2049, 4096, 1], [9] * 65, [100003]], ids=lambda v: "%dx%d" % (len(v), max(v)))
def test_codes_over_the_whole_format(hip, lens):
    base.say("adamw8 whole format", len(lens), max(lens))
    g = [gradients(n, 100 + 2 * i) for i, n in enumerate(lens)]
    p = [rng.normal(n, 1.0, tag=300 + i, seed=SEED).astype(np.float32) for i, n in enumerate(lens)]
    m8, v8, scales = base.zeros8(lens)
    b1, b2 = np.float32(0.9), np.float32(0.999)
    for step in (1, 2, 3, 500):
        before = [[a.copy() for a in k] for k in (p, m8, v8, scales)]
        hip.adamw8_step_multi(p, g, m8, v8, scales, step=step, seed=SEED, **HYPER)
        for i, n in enumerate(lens):
            m, v = base.decode(before[1][i], before[2][i], before[3][i])
            want, tol = base.exact(before[0][i], g[i], m, v, step, **HYPER)
            base.close(p[i], want[0], tol[0], (step, i, "p"))
            m = m * b1 + g[i] * (np.float32(1) - b1)
            v = v * b2 + (g[i] * (np.float32(1) - b2)) * g[i]
            for got, w, what in zip((m8[i], v8[i], scales[i]), encode(m, v, base.random16(n, i, step, SEED)), ("m8", "v8", "scales")):
                assert np.array_equal(got, w), (step, i, what, int((got != w).sum()))
        for k in g:                                                       # some go on, some stop
            k[1::2] = 0


@pytest.mark.gpu
def test_v_decays_whatever_its_part_of_the_block(hip):
    """Without a gradient v falls to 0.999^300 = 0.741 of itself on average in 300 steps, here for values of 2 to 64 units of
    2^-16 of the scale beside one that stays the block's largest.  With d the grid's spacing at v - a quarter of it, or one
    unit - a step moves v to a neighbour on the grid with variance 0.001 v d at most: the mean of n values after 300 steps is within
    5 sqrt(0.3 v d / n), and the words' 16 bits cost 2^-16 d a step.  What has come down to one unit stays there: it keeps the
    0.26 units that it would have lost."""
    each, sizes = 1 << 14, (2, 3, 4, 6, 8, 16, 64)
    n = each * len(sizes)
    start = np.repeat(np.float32(sizes) * SMALLEST, each)
    start[::256] = 2.0 ** 14
    v8 = torch.from_numpy(start).to(torch.float8_e5m2).view(torch.uint8).numpy()
    g = np.zeros(n, np.float32)
    g[::256] = 1.1 * 2.0 ** 7                                             # keeps v there at 2^14 and above, and its scale at 1
    c = hip.ctx()
    scales = np.ones(2 * (n // 256), np.float32)
    bufs = [c.array(a) for a in (np.zeros(n, np.float32), g, np.zeros(n // 4, np.float32), v8.view(np.float32), scales)]
    arrays, lens = [(C.c_void_p * 1)(b.ptr) for b in bufs], (C.c_size_t * 1)(n)
    for t in range(1, 301):
        c.call("slhip_adamw8_step_multi", 1, *arrays, lens, 1e-2, 0.9, 0.999, 1e-8, 0.1, t, None, SEED)
    v = torch.from_numpy(bufs[3].numpy().view(np.uint8).copy()).view(torch.float8_e5m2).double().numpy()
    per = bufs[4].numpy().reshape(-1, 2)[:, 1]
    for b in bufs:
        b.free()
    assert (per == 1).all()
    v = (v * 65536).reshape(len(sizes), -1, 256)[:, :, 1:].reshape(len(sizes), -1)
    for k, s in enumerate(sizes):
        d = max(1.0, s / 4)
        allowed, want = 5 * np.sqrt(0.3 * s * d / v.shape[1]) + 300 * 2.0 ** -16 * d, s * base.f32(0.999) ** 300
        base.say("v of", s, "units:", v[k].mean(), "expected", want)
        assert -allowed <= v[k].mean() - want <= allowed + (0.26 if s < 4 else 0), s


@pytest.mark.gpu
def test_a_v_that_underflows_beside_the_largest_is_not_zero(hip):
    """Gradients whose squares are 2^330 apart in one block: the small ones' v is zero in units of the scale, and is kept as the
    smallest value all the same."""
    n = 600
    g = np.full(n, 1e-19, np.float32)
    g[[0, 300]] = 3e10
    g[10:20] = 0
    p, (m8, v8, scales) = [np.zeros(n, np.float32)], base.zeros8([n])
    hip.adamw8_step_multi(p, [g], m8, v8, scales, step=1, seed=SEED, **HYPER)
    r1, r2 = np.float32(1) - np.float32(0.9), np.float32(1) - np.float32(0.999)
    v = (g * r2) * g
    assert ((v > 0) == (g > 0)).all() and v[1] / scales[0][1] == 0
    for got, w, what in zip((m8[0], v8[0], scales[0]), encode(g * r1, v, base.random16(n, 0, 1, SEED)), ("m8", "v8", "scales")):
        assert np.array_equal(got, w), what
    assert ((v8[0] > 0) == (g > 0)).all()
