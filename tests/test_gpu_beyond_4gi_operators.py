"""Group norm, the gated recurrence and AdamW over tensors of more than 2^32 elements (16 GiB): every offset on the path has to be 64
bits wide.  As in test_gpu_beyond_4gi.py the operands come from the device generator, whose values the host can recompute at any index,
and results are checked on windows: at the start, either side of element 2^32, at the end.

Needs about 72 GiB of device memory; skipped when the device has less free."""
import ctypes as C
import sys

import numpy as np
import pytest

import test_gpu_adamw as adamw
import test_gpu_adamw_rounding as rounding
from devgen import host_range, host_values
from sliced_amd import rng

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SEED = rng.DEFAULT_SEED
ROWS, COLS = 65553, 65536            # 2^32 + 17 * 2^16 elements
N = ROWS * COLS
TWO32 = 1 << 32
SILU = 2
X, GATE = (0, -1.0, 1.0), (1, 0.1, 0.9)                      # tag, lo, hi of the generated operands


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def big():
    from sliced_amd.device import Context
    rt = C.CDLL("libamdhip64.so.7")
    free, total = C.c_size_t(), C.c_size_t()
    ctx = Context(0)
    assert rt.hipMemGetInfo(C.byref(free), C.byref(total)) == 0
    if free.value < (72 << 30):
        ctx.close()
        pytest.skip("needs 72 GiB of free device memory, %d GiB are free" % (free.value >> 30))
    say("allocating four buffers of", N, "floats")
    bufs = [ctx.uniform(N, X[1], X[2], X[0], SEED), ctx.uniform(N, GATE[1], GATE[2], GATE[0], SEED), ctx.empty(N), ctx.empty(N), ctx.empty(1 << 27)]
    yield [ctx] + bufs
    for b in bufs:
        b.free()
    ctx.close()


def at_rows(t, rows, width, columns):
    """Values of a generated operand at rows x columns of a matrix of that width"""
    return host_values(rows.astype(np.uint64)[:, None] * np.uint64(width) + columns.astype(np.uint64), t[0], t[1], t[2], SEED).astype(np.float64)


def read_rows(buf, first, n, width, columns):
    whole = buf.view(first * width, n * width).numpy().reshape(n, width)
    return whole[:, columns].astype(np.float64)


@pytest.mark.parametrize("channels", [65536, 64])
def test_recurrence(big, channels):
    """Gates of at most 0.9 forget a state within 300 steps to 10^-13 of it: the recurrence run in 64 bits from 300 steps before a window
    (after it, backward) gives its values.  65536 channels in one run of steps each, 64 channels split over workgroups."""
    ctx, x, gate, h, out, _ = big
    steps, cols = N // channels, np.r_[0:16, channels - 16:channels]
    say("recurrence", steps, channels)
    ctx.call("slhip_gated_scan", 0, 1, steps, channels, gate.ptr, x.ptr, None, h.ptr, None)
    n, before = 34, 300
    starts = [0, TWO32 // channels - 20, steps - n]
    states = {}
    for s in starts:
        rows = np.arange(max(s - before, 0), min(s + n, steps))
        a, b, v = at_rows(GATE, rows, channels, cols), at_rows(X, rows, channels, cols), np.zeros(cols.size)
        got = read_rows(h, s, n, channels, cols)
        for k, t in enumerate(rows):
            v = a[k] * v + b[k]
            if t >= s:
                # states are below 10; a step rounds twice, gates of 0.9 keep ten steps' worth
                assert np.abs(got[t - s] - v).max() <= 4 * 10 * 10 * U, (s, t)
        states[s] = got
    say("its gradients")
    for which in ("x", "gate"):
        ctx.call("slhip_gated_scan_grad", 0, 1, steps, channels, gate.ptr, None, None, h.ptr, out.ptr if which == "gate" else None,
                 out.ptr if which == "x" else None, None, x.ptr, None, 0.0)
        for s in starts:
            rows = np.arange(s, min(s + n + before, steps))
            a, d, g = at_rows(GATE, rows, channels, cols), at_rows(X, rows, channels, cols), np.zeros(cols.size)
            got = read_rows(out, s, n, channels, cols)
            for k in range(rows.size - 1, -1, -1):
                v = d[k] + g
                g = a[k] * v
                if k < n and (which == "x" or k > 0):
                    want = v if which == "x" else v * states[s][k - 1]
                    assert np.abs(got[k] - want).max() <= 4 * 10 * 10 * U * (1 if which == "x" else 11), (which, s, k)


@pytest.mark.parametrize("samples,positions,channels,groups", [(1, ROWS, COLS, 512), (ROWS, 1, COLS, 512), (ROWS * 16, 4, 1024, 8)])
def test_group_norm(big, samples, positions, channels, groups):
    """Two passes, rows and the on-chip kernels.  The statistics are those of a uniform distribution on [-1, 1) within six deviations of
    their own, and in the latter two, where a group is small, those of its values; outputs and x gradients follow from them."""
    ctx, x, gate, out, grad, small = big
    say("group norm", samples, positions, channels, groups)
    stats = samples * groups
    mean, rstd = small.view(0, stats), small.view(stats, stats)
    ctx.call("slhip_group_norm", samples, positions, channels, groups, SILU, 1e-5, x.ptr, None, None, mean.ptr, rstd.ptr, out.ptr)
    size, cg = positions * channels // groups, channels // groups
    for row in (0, TWO32 // channels - 3, TWO32 // channels, N // channels - 3):   # three rows of channels each
        rows = np.arange(row, row + 3)
        got = out.view(row * channels, 3 * channels).numpy().reshape(3, groups, cg)
        v = at_rows(X, rows, channels, np.arange(channels)).reshape(3, groups, cg)
        for k, r in enumerate(rows):
            n = int(r) // positions
            m, s = (t.view(n * groups, groups).numpy().astype(np.float64)[:, None] for t in (mean, rstd))
            var = 1 / s ** 2 - 1e-5
            # a uniform value has variance 1/3, its square's deviation from that 4/45
            assert np.abs(m).max() <= 6 * np.sqrt(1 / 3 / size) and np.abs(var - 1 / 3).max() <= 6 * np.sqrt(4 / 45 / size) + 1 / size
            if size <= 1024:
                of = np.arange(n * positions, (n + 1) * positions)
                group = at_rows(X, of, channels, np.arange(channels)).reshape(positions, groups, cg)
                want = group.mean(axis=(0, 2))
                assert np.abs(m[:, 0] - want).max() <= 64 * U and np.abs(var[:, 0] - group.var(axis=(0, 2))).max() <= 128 * U
            u = (v[k] - m) * s
            assert np.abs(got[k] - u / (1 + np.exp(-u))).max() <= 32 * U, (r, k)
    say("its gradients")
    ctx.call("slhip_group_norm_grad", samples, positions, channels, groups, SILU, x.ptr, None, None, mean.ptr, rstd.ptr, grad.ptr, None, None,
             gate.ptr, 0.0)
    for row in (0, TWO32 // channels - 3, TWO32 // channels, N // channels - 3):
        rows = np.arange(row, row + 3)
        got = grad.view(row * channels, 3 * channels).numpy().reshape(3, groups, cg)
        v, dy = (at_rows(t, rows, channels, np.arange(channels)).reshape(3, groups, cg) for t in (X, GATE))
        for k, r in enumerate(rows):
            n = int(r) // positions
            m, s = (t.view(n * groups, groups).numpy().astype(np.float64)[:, None] for t in (mean, rstd))
            hat = (v[k] - m) * s
            q = 1 / (1 + np.exp(-hat))
            g = dy[k] * q * (1 + hat * (1 - q))
            if size <= 1024:
                of = np.arange(n * positions, (n + 1) * positions)
                xs, ds = (at_rows(t, of, channels, np.arange(channels)).reshape(positions, groups, cg) for t in (X, GATE))
                hs = (xs - m) * s
                qs = 1 / (1 + np.exp(-hs))
                gs = ds * qs * (1 + hs * (1 - qs))
                want = s * (g - gs.mean(axis=(0, 2))[:, None] - hat * (gs * hs).mean(axis=(0, 2))[:, None])
                assert np.abs(got[k] - want).max() <= 64 * U, (r, k)
            else:
                # what the sums over 8 million values take off is one pair of numbers for all of a group: two unknowns, fitted
                a = np.stack([np.ones_like(hat), hat], axis=-1)
                off = g - got[k] / s
                fit = np.stack([np.linalg.lstsq(a[i], off[i], rcond=None)[0] for i in range(0, groups, 37)])
                for i, f in zip(range(0, groups, 37), fit):
                    assert np.abs(a[i] @ f - off[i]).max() <= 64 * U, (r, i)
                    # the means of g and g hat for dy uniform on [0.1, 0.9): 0.5 <slope> = 0.25 within a percent, and positive
                    assert abs(f[0] - 0.25) <= 0.01 and 0 < f[1] < 0.5


def test_adamw_f32(big):
    ctx, x, gate, p, m, _ = big
    say("adamw", N)
    ctx.call("slhip_fill", N, 0.5, p.ptr)
    ctx.call("slhip_fill", N, 0.25, m.ptr)
    one = [(C.c_void_p * 1)(b.ptr) for b in (p, x, m, gate)]
    ctx.call("slhip_adamw_step_multi", 1, *one, (C.c_size_t * 1)(N), 1e-2, 0.9, 0.999, 1e-8, 0.1, 7, None)
    for start, n in ((0, 8192), (TWO32 - 4096, 8192), (N - 8192, 8192)):
        g, v = host_range(start, n, *X), host_range(start, n, *GATE)
        want, tol = adamw.exact(np.full(n, 0.5), g, np.full(n, 0.25), v, 7, **adamw.HYPER)
        for buf, w, t, what in zip((p, m, gate), want, tol, "pmv"):
            adamw.close(buf.view(start, n).numpy(), w, t, (start, what))
    ctx.call("slhip_rand_uniform", SEED, GATE[0], GATE[1], GATE[2], N, gate.ptr)


def test_adamw_8_bit(big):
    ctx, x, _, p, state, _ = big
    say("adamw8", N)
    ctx.call("slhip_fill", N, 0.5, p.ptr)
    ctx.call("slhip_fill", N, 0.0, state.ptr)                # the codes of m, those of v behind them, and the scales
    quarter = N // 4
    one = [(C.c_void_p * 1)(a) for a in (p.ptr, x.ptr, state.ptr, state.ptr + N, state.ptr + 2 * N)]
    ctx.call("slhip_adamw8_step_multi", 1, *one, (C.c_size_t * 1)(N), 1e-2, 0.9, 0.999, 1e-8, 0.1, 7, None, SEED)
    r1, r2 = np.float32(1) - np.float32(0.9), np.float32(1) - np.float32(0.999)
    for start, n in ((0, 8192), (TWO32 - 4096, 8192), (N - 8192, 8192)):
        g = host_range(start, n, *X)
        want, tol = adamw.exact(np.full(n, 0.5), g, np.zeros(n), np.zeros(n), 7, **adamw.HYPER)
        adamw.close(p.view(start, n).numpy(), want[0], tol[0], (start, "p"))
        with np.errstate(over="ignore"):
            key = adamw.mix(adamw.mix(np.uint64(SEED + 7)) + np.uint64(0))
            word = adamw.mix(key + np.arange(start // 4, (start + n) // 4, dtype=np.uint64))
        r16 = ((word[:, None] >> (np.uint64(16) * np.arange(4, dtype=np.uint64))) & np.uint64(0xFFFF)).ravel().astype(np.uint32)
        m8, v8, scales = rounding.encode(g * r1, (g * r2) * g, r16)
        assert np.array_equal(state.view(start // 4, n // 4).numpy().view(np.uint8), m8), start
        assert np.array_equal(state.view(quarter + start // 4, n // 4).numpy().view(np.uint8), v8), start
        assert np.array_equal(state.view(2 * quarter + start // 128, n // 128).numpy(), scales), start
