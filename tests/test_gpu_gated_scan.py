"""The gated linear recurrence through the C ABI against the recurrence run step by step in 64 bits, forward and
backward, in both forms.

Tolerances.  With u = 2^-24, a step rounds its coefficients and its multiply-add, and the joins of runs of steps round the
products of gates that a term passes through: k roundings a step, k = 4 for the linear form, 12 for the sigmoid form
(exp to one unit in the last place = 2 u, the sum, the quotient, the product for the small side: 6 u for s and for 1 - s
each).  A term that enters at step s and is read at step t has met (t - s + 1) k of them, so with M_t = |a_t| M_{t-1} + |b_t|
the error of h_t is at most u D_t, D_t = |a_t| D_{t-1} + k M_t - the recurrence itself, run on magnitudes."""
import ctypes as C

import numpy as np
import pytest

from sliced_amd import rng

U = 2.0 ** -24
LINEAR, SIGMOID = 0, 1
K = {LINEAR: 4.0, SIGMOID: 12.0}
SEED = 0x51CED


def say(*a):
    print(*a, flush=True)


def coefficients(mode, gate):
    z = gate.astype(np.float64)
    if mode == LINEAR:
        return z, np.ones_like(z)
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-z)), 1 / (1 + np.exp(z))


def forward(mode, gate, x, h0):
    """(h, tolerance of h) for [batch, steps, channels] arrays"""
    a, rest = coefficients(mode, gate)
    b = rest * x.astype(np.float64)
    h = np.zeros_like(b)
    tol = np.zeros_like(b)
    s = np.zeros_like(b[:, 0]) if h0 is None else h0.astype(np.float64)
    m, d = np.abs(s), np.zeros_like(s)
    for t in range(b.shape[1]):
        s = a[:, t] * s + b[:, t]
        m = np.abs(a[:, t]) * m + np.abs(b[:, t])
        d = np.abs(a[:, t]) * d + K[mode] * m
        h[:, t], tol[:, t] = s, U * d
    return h, tol


def backward(mode, gate, x, h0, h, dh, dl):
    """((gate, x, h0) gradients, their tolerances), from the h that the forward call left"""
    f = np.float64
    a, rest = coefficients(mode, gate)
    h, dh = h.astype(f), dh.astype(f)
    first = np.zeros_like(h[:, 0]) if h0 is None else h0.astype(f)
    g = np.zeros_like(first) if dl is None else dl.astype(f)
    m, e = np.abs(g), np.zeros_like(g)
    dg, dx, tg, tx = (np.zeros_like(h) for _ in range(4))
    for t in range(h.shape[1] - 1, -1, -1):
        before = h[:, t - 1] if t else first
        d = dh[:, t] + g
        md = np.abs(dh[:, t]) + m
        ed = e + K[mode] * md
        if mode == LINEAR:
            dg[:, t], tg[:, t] = d * before, ed * np.abs(before) + np.abs(d * before)
            dx[:, t], tx[:, t] = d, ed
        else:
            xt = x[:, t].astype(f)
            part = a[:, t] * rest[:, t]
            dg[:, t] = d * (before - xt) * part
            # the products' and the difference's roundings, and those of s and 1 - s
            tg[:, t] = (ed * np.abs(before - xt) + md * (16 * np.abs(before - xt) + np.abs(before) + np.abs(xt))) * part
            dx[:, t], tx[:, t] = d * rest[:, t], (ed + 8 * md) * rest[:, t]
        g = a[:, t] * d
        m = np.abs(a[:, t]) * md
        e = np.abs(a[:, t]) * (ed + K[mode] * md)
    return (dg, dx, g), (U * tg, U * tx, U * (e + K[mode] * m))


def data(mode, batch, steps, channels, tag=0, with_h0=True):
    n, s = batch * steps * channels, batch * channels
    slow = np.repeat(rng.uniform(channels, -2, 4, tag=90 + tag, seed=SEED)[None], batch * steps, 0).reshape(batch, steps, channels)
    gate = slow + rng.uniform(n, -2, 2, tag=91 + tag, seed=SEED).reshape(batch, steps, channels)
    if mode == LINEAR:
        gate = 1 / (1 + np.exp(-gate)) * np.where(rng.uniform(n, 0, 1, tag=92 + tag, seed=SEED).reshape(gate.shape) < 0.1, -1, 1)
    gate = gate.astype(np.float32)
    x = rng.normal(n, 1.0, tag=93 + tag, seed=SEED).reshape(batch, steps, channels).astype(np.float32)
    h0 = rng.normal(s, 1.0, tag=94 + tag, seed=SEED).reshape(batch, channels).astype(np.float32) if with_h0 else None
    return gate, x, h0


def close(got, want, tol, what):
    got = np.asarray(got, np.float64).reshape(want.shape)
    off = np.abs(got - want)
    bad = ~(off <= tol + 1e-37)
    assert not bad.any(), (what, int(bad.sum()), float(np.nanmax(off / (tol + 1e-37))), np.argwhere(bad)[:3].tolist())


# one step and two, fewer channels than a vector and more, odd ones, batches, steps around the runs that kernels take
SHAPES = [(1, 1, 1), (1, 1, 2048), (3, 1, 37), (5, 2, 3), (1, 7, 1), (2, 31, 5), (1, 33, 4), (4, 64, 16), (3, 65, 31), (2, 127, 130),
          (1, 129, 67), (2, 257, 33), (1, 1000, 9), (1, 4099, 1), (7, 513, 64), (1, 2048, 260), (33, 40, 100), (1, 9001, 40), (2, 5000, 2),
          (300, 3, 700), (1, 20011, 35), (64, 1030, 4)]


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [LINEAR, SIGMOID])
@pytest.mark.parametrize("batch,steps,channels", SHAPES)
def test_forward_and_backward(hip, batch, steps, channels, mode):
    say("scan", mode, batch, steps, channels)
    gate, x, h0 = data(mode, batch, steps, channels)
    h, last = hip.gated_scan(mode, batch, steps, channels, gate, x, h0)
    want, tol = forward(mode, gate, x, h0)
    close(h, want, tol, "h")
    assert np.array_equal(last, h.reshape(batch, steps, channels)[:, -1].ravel())
    dh = rng.normal(gate.size, 1.0, tag=7, seed=SEED).reshape(gate.shape).astype(np.float32)
    dl = rng.normal(batch * channels, 1.0, tag=8, seed=SEED).reshape(batch, channels).astype(np.float32)
    outs = [np.full(gate.size, np.nan, np.float32), np.full(gate.size, np.nan, np.float32), np.full(batch * channels, np.nan, np.float32)]
    hip.gated_scan_grad(mode, batch, steps, channels, gate, x, h0, h, dh, *outs, h_last_grad=dl)
    grads, tols = backward(mode, gate, x, h0, h.reshape(gate.shape), dh, dl)
    for got, want, tol, what in zip(outs, grads, tols, ("gate", "x", "h0")):
        close(got, want, tol, what)


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [LINEAR, SIGMOID])
@pytest.mark.parametrize("batch,steps,channels", [(2, 70, 12), (1, 3000, 37), (3, 1, 5), (1, 600, 2)])
def test_optional_arguments_and_accumulation(hip, batch, steps, channels, mode):
    """No initial state, no last state, no gradient of it; single gradients; beta = 1 adds to what is there."""
    say("scan optional", mode, batch, steps, channels)
    gate, x, _ = data(mode, batch, steps, channels, tag=10)
    c = hip.ctx()
    bufs = [c.array(gate), c.array(x), c.empty(gate.size)]
    c.call("slhip_gated_scan", mode, batch, steps, channels, bufs[0].ptr, bufs[1].ptr, None, bufs[2].ptr, None)
    h = bufs[2].numpy()
    for b in bufs:
        b.free()
    want, tol = forward(mode, gate, x, None)
    close(h, want, tol, "h")
    dh = rng.normal(gate.size, 1.0, tag=9, seed=SEED).reshape(gate.shape).astype(np.float32)
    grads, tols = backward(mode, gate, x, None, h.reshape(gate.shape), dh, None)
    lens = (gate.size, gate.size, batch * channels)
    for only in range(3):
        outs = [np.full(lens[k], np.nan, np.float32) if k == only else None for k in range(3)]
        hip.gated_scan_grad(mode, batch, steps, channels, gate, x if mode == SIGMOID else None, None, h, dh, *outs)
        close(outs[only], grads[only], tols[only], ("alone", only))
    old = [rng.normal(n, 1.0, tag=11 + k, seed=SEED).astype(np.float32) for k, n in enumerate(lens)]
    outs = [o.copy() for o in old]
    hip.gated_scan_grad(mode, batch, steps, channels, gate, x, None, h, dh, *outs, beta=1.0)
    for got, before, want, tol in zip(outs, old, grads, tols):
        want = want + before.reshape(want.shape)
        close(got, want, tol + U * np.abs(want) * 1.01, "beta 1")


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [LINEAR, SIGMOID])
def test_gradients_against_differences(hip, mode):
    """The gradients of sum(h * dh) + sum(h_last * dl) against central differences of the 64-bit recurrence."""
    batch, steps, channels = 2, 9, 3
    gate, x, h0 = data(mode, batch, steps, channels, tag=20)
    dh = rng.normal(gate.size, 1.0, tag=21, seed=SEED).reshape(gate.shape)
    dl = rng.normal(batch * channels, 1.0, tag=22, seed=SEED).reshape(batch, channels)
    h, _ = hip.gated_scan(mode, batch, steps, channels, gate, x, h0)
    outs = [np.zeros(gate.size, np.float32), np.zeros(gate.size, np.float32), np.zeros(batch * channels, np.float32)]
    hip.gated_scan_grad(mode, batch, steps, channels, gate, x, h0, h, dh, *outs, h_last_grad=dl)

    def loss(*at):
        a, rest = coefficients(mode, at[0])
        s, total = at[2].copy(), 0.0
        for t in range(steps):
            s = a[:, t] * s + rest[:, t] * at[1][:, t]
            total += (s * dh.astype(np.float32).astype(np.float64)[:, t]).sum()
        return total + (s * dl.astype(np.float32).astype(np.float64)).sum()

    at = [v.astype(np.float64) for v in (gate, x, h0)]
    eps = 1e-5
    for k in range(3):
        flat = at[k].reshape(-1)
        for i in range(flat.size):
            keep = flat[i]
            flat[i] = keep + eps
            up = loss(*at)
            flat[i] = keep - eps
            down = loss(*at)
            flat[i] = keep
            # eps^2 of the third derivative and 1e-16 / eps of the difference, and the kernel's own 32 bits
            assert abs((up - down) / (2 * eps) - outs[k][i]) <= 2e-5 * (1 + abs(outs[k][i])), (k, i)


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [LINEAR, SIGMOID])
def test_steps_one_by_one_continue_a_sequence(hip, mode):
    """A sequence in one call, in two calls, and token by token with the state updated in place."""
    batch, steps, channels = 3, 45, 50
    gate, x, h0 = data(mode, batch, steps, channels, tag=30)
    want, tol = forward(mode, gate, x, h0)
    a, last = hip.gated_scan(mode, batch, 30, channels, gate[:, :30], x[:, :30], h0)
    b, _ = hip.gated_scan(mode, batch, 15, channels, gate[:, 30:], x[:, 30:], last)
    close(a.reshape(batch, 30, channels), want[:, :30], tol[:, :30], "first")
    close(b.reshape(batch, 15, channels), want[:, 30:], tol[:, 30:], "second")
    c = hip.ctx()
    state, out = c.array(h0), c.empty(batch * channels)
    for t in range(steps):
        g, v = c.array(gate[:, t]), c.array(x[:, t])
        c.call("slhip_gated_scan", mode, batch, 1, channels, g.ptr, v.ptr, state.ptr, out.ptr, state.ptr)
        got = out.numpy()
        assert np.array_equal(got, state.numpy())
        close(got, want[:, t], tol[:, t], t)
        g.free(), v.free()
    state.free(), out.free()


@pytest.mark.gpu
@pytest.mark.parametrize("batch,steps,channels", [(1, 4000, 24), (1, 3000, 1), (2, 100, 8)])
def test_state_updated_in_place_over_long_sequences(hip, batch, steps, channels):
    """h_last is h0's own array also where the time axis is split over workgroups."""
    gate, x, h0 = data(SIGMOID, batch, steps, channels, tag=40)
    want, tol = forward(SIGMOID, gate, x, h0)
    c = hip.ctx()
    g, v, state, out = c.array(gate), c.array(x), c.array(h0), c.empty(gate.size)
    c.call("slhip_gated_scan", SIGMOID, batch, steps, channels, g.ptr, v.ptr, state.ptr, out.ptr, state.ptr)
    close(out.numpy(), want, tol, "h")
    close(state.numpy(), want[:, -1], tol[:, -1], "state")
    # and h written over x
    c.call("slhip_gated_scan", SIGMOID, batch, steps, channels, g.ptr, v.ptr, None, v.ptr, None)
    want, tol = forward(SIGMOID, gate, x, None)
    close(v.numpy(), want, tol, "over x")
    for b in (g, v, state, out):
        b.free()


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [LINEAR, SIGMOID])
@pytest.mark.parametrize("batch,steps,channels", [(3, 1, 37), (2, 5, 130), (2, 700, 33), (1, 5000, 67)])
def test_outputs_over_inputs_equal_separate_ones(hip, batch, steps, channels, mode):
    gate, x, h0 = data(mode, batch, steps, channels, tag=47)
    want = hip.gated_scan(mode, batch, steps, channels, gate, x, h0)[0]
    same = hip.gated_scan(mode, batch, steps, channels, gate, gate, h0)[0]
    c = hip.ctx()
    for over in range(3):
        if over == 2 and steps > 1:
            continue
        g, v, s = c.array(gate), c.array(x), c.array(h0)
        out = (g, v, s)[over]
        c.call("slhip_gated_scan", mode, batch, steps, channels, g.ptr, v.ptr, s.ptr, out.ptr, None)
        assert np.array_equal(out.numpy(), want), over
        for b in (g, v, s):
            b.free()
    g, s = c.array(gate), c.array(h0)                 # gate, input and output in one
    c.call("slhip_gated_scan", mode, batch, steps, channels, g.ptr, g.ptr, s.ptr, g.ptr, s.ptr)
    assert np.array_equal(g.numpy(), same) and np.array_equal(s.numpy().reshape(batch, channels), same.reshape(batch, steps, channels)[:, -1])
    g.free()
    s.free()


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [LINEAR, SIGMOID])
def test_two_contexts_on_two_streams(hip, mode):
    """A context on a stream of its own and one on the caller's, both busy with split sequences at once: each has its own
    workspace."""
    from sliced_amd.device import Context
    batch, steps, channels = 1, 9000, 40
    runtime = C.CDLL("libamdhip64.so.7")               # (the one the library has loaded)
    stream = C.c_void_p()
    assert runtime.hipStreamCreateWithFlags(C.byref(stream), 1) == 0
    one, two = Context(0), Context(0, stream=stream.value)
    sets = [data(mode, batch, steps, channels, tag=60 + 5 * k) for k in range(2)]
    want = [hip.gated_scan(mode, batch, steps, channels, *s)[0] for s in sets]
    bufs = [[c.array(a) for a in s] + [c.empty(s[0].size)] for c, s in zip((one, two), sets)]
    for _ in range(10):
        for c, b in zip((one, two), bufs):
            c.call("slhip_gated_scan", mode, batch, steps, channels, b[0].ptr, b[1].ptr, b[2].ptr, b[3].ptr, None)
    for c, b, w in zip((one, two), bufs, want):
        c.sync()
        assert np.array_equal(b[3].numpy(), w)
    for c, b in zip((one, two), bufs):
        for k in b:
            k.free()
        c.close()
    assert runtime.hipStreamDestroy(stream) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [50, 5000])
def test_a_closed_gate_starts_a_sequence_anew(hip, steps):
    """gate 0 (linear) and -inf (sigmoid) forget what was before exactly - packed sequences; +inf keeps the state as it is."""
    batch, channels = 1, 20
    cut = steps // 3
    for mode, closed in ((LINEAR, 0.0), (SIGMOID, -np.inf)):
        gate, x, h0 = data(mode, batch, steps, channels, tag=50)
        gate[:, cut] = closed
        h, _ = hip.gated_scan(mode, batch, steps, channels, gate, x, h0)
        other = x.copy()
        other[:, :cut] = rng.normal(cut * channels, 5.0, tag=51, seed=SEED).reshape(1, cut, channels)
        h2, _ = hip.gated_scan(mode, batch, steps, channels, gate, other, h0 * 3)
        assert np.array_equal(h.reshape(x.shape)[:, cut:], h2.reshape(x.shape)[:, cut:])
        assert np.array_equal(h.reshape(x.shape)[:, cut], x[:, cut])
    gate[:] = np.inf
    h, last = hip.gated_scan(SIGMOID, batch, steps, channels, gate, x, h0)
    assert np.array_equal(h.reshape(x.shape), np.repeat(h0[:, None], steps, 1)) and np.array_equal(last, h0.ravel())


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [LINEAR, SIGMOID])
@pytest.mark.parametrize("steps", [20, 3000])
def test_a_nan_stays_in_its_channel_and_behind_its_step(hip, mode, steps):
    channels = 9
    gate, x, h0 = data(mode, 1, steps, channels, tag=60)
    at = steps // 2
    x[0, at, 4] = np.nan
    h, _ = hip.gated_scan(mode, 1, steps, channels, gate, x, h0)
    h = h.reshape(steps, channels)
    assert np.isnan(h[at:, 4]).all() and not np.isnan(h[:at]).any() and not np.isnan(np.delete(h, 4, 1)).any()
    gate[0, at, 2] = np.nan
    h, _ = hip.gated_scan(mode, 1, steps, channels, gate, x, h0)
    h = h.reshape(steps, channels)
    assert np.isnan(h[at:, 2]).all() and not np.isnan(h[:at]).any() and not np.isnan(np.delete(h, [2, 4], 1)).any()


@pytest.mark.gpu
@pytest.mark.parametrize("batch,steps,channels", [(2, 300, 21), (1, 2500, 8), (2, 3, 1)])
def test_float_aligned_operands_and_untouched_surroundings(hip, batch, steps, channels):
    """Every operand 1, 2 or 3 floats into its allocation; what lies around the outputs stays as it was."""
    hip.operands_off_the_vector_grid(True)
    try:
        for mode in (LINEAR, SIGMOID):
            gate, x, h0 = data(mode, batch, steps, channels, tag=70)
            h, _ = hip.gated_scan(mode, batch, steps, channels, gate, x, h0)
            want, tol = forward(mode, gate, x, h0)
            close(h, want, tol, "h")
            outs = [np.zeros(gate.size, np.float32), np.zeros(gate.size, np.float32), np.zeros(batch * channels, np.float32)]
            hip.gated_scan_grad(mode, batch, steps, channels, gate, x, h0, h, x, *outs)
            for got, w, t in zip(outs, *backward(mode, gate, x, h0, h.reshape(x.shape), x, None)):
                close(got, w, t, "grad")
    finally:
        hip.operands_off_the_vector_grid(False)
    c = hip.ctx()
    n = gate.size
    pool = c.empty(n + 14)
    pool.upload(np.full(n + 14, 7.0, np.float32))
    g, v = c.array(gate), c.array(x)
    c.call("slhip_gated_scan", SIGMOID, batch, steps, channels, g.ptr, v.ptr, None, pool.ptr + 4 * 7, None)
    got = pool.numpy()
    assert (got[:7] == 7).all() and (got[-7:] == 7).all() and not (got[7:-7] == 7).any()
    for b in (pool, g, v):
        b.free()


@pytest.mark.gpu
@pytest.mark.parametrize("batch,steps,channels", [(2, 1, 64), (1, 6000, 33), (4, 700, 260)])
def test_recorded_calls_replay_like_the_eager_ones(hip, batch, steps, channels):
    """Forward and backward in one recording, replayed on changing inputs with eager work in between."""
    c = hip.ctx()
    gate, x, h0 = data(SIGMOID, batch, steps, channels, tag=80)
    n, s = gate.size, batch * channels
    g, v, s0 = c.array(gate), c.array(x), c.array(h0)
    h, dg, dx, d0 = c.empty(n), c.empty(n), c.empty(n), c.empty(s)
    c.sync()
    c.call("slhip_graph_begin")
    try:
        c.call("slhip_gated_scan", SIGMOID, batch, steps, channels, g.ptr, v.ptr, s0.ptr, h.ptr, None)
        c.call("slhip_gated_scan_grad", SIGMOID, batch, steps, channels, g.ptr, v.ptr, s0.ptr, h.ptr, dg.ptr, dx.ptr, d0.ptr, v.ptr, None, 0.0)
    finally:
        graph = C.c_void_p()
        c.call("slhip_graph_end", C.byref(graph))
    for replay in range(3):
        say("replay", replay)
        now = rng.normal(n, 1.0, tag=81 + replay, seed=SEED).reshape(x.shape).astype(np.float32)
        v.upload(now)
        c.call("slhip_graph_launch", graph)
        got = [b.numpy() for b in (h, dg, dx, d0)]
        want_h, _ = hip.gated_scan(SIGMOID, batch, steps, channels, gate, now, h0)     # eager work between the replays
        outs = [np.zeros(n, np.float32), np.zeros(n, np.float32), np.zeros(s, np.float32)]
        hip.gated_scan_grad(SIGMOID, batch, steps, channels, gate, now, h0, want_h, now, *outs)
        for a, b in zip(got, [want_h] + outs):
            assert np.array_equal(a, b), replay
    c.lib.slhip_graph_destroy(graph)
    for b in (g, v, s0, h, dg, dx, d0):
        b.free()


def refused(lib, ctx):
    one = C.create_string_buffer(64)
    p = C.addressof(one)
    big = 1 << 62
    call, grad = lib.slhip_gated_scan, lib.slhip_gated_scan_grad
    assert call(None, 0, 1, 1, 1, p, p, None, p, None) == -1
    for bad in ((2, 1, 1, 1), (-1, 1, 1, 1), (0, 0, 1, 1), (0, 1, 0, 1), (0, 1, 1, 0), (0, big, 4, 1), (0, 2, big, 2), (1, 1, 2, big)):
        assert call(ctx, *bad, p, p, None, p, None) == -1, bad
        assert grad(ctx, *bad, p, p, None, p, p, p, p, p, None, 0.0) == -1, bad
    for k in (0, 1, 3):
        args = [p, p, None, p, None]
        args[k] = None
        assert call(ctx, 0, 1, 1, 1, *args) == -1, k
    assert grad(ctx, 0, 1, 1, 1, None, p, None, p, p, p, p, p, None, 0.0) == -1
    assert grad(ctx, 1, 1, 1, 1, p, None, None, p, p, p, p, p, None, 0.0) == -1     # the sigmoid form needs x
    assert grad(ctx, 0, 1, 1, 1, p, None, None, None, p, p, p, p, None, 0.0) == -1
    assert grad(ctx, 0, 1, 1, 1, p, None, None, p, p, p, p, None, None, 0.0) == -1
    assert grad(ctx, 0, 1, 1, 1, p, None, None, p, None, None, None, p, None, 0.0) == 0  # nothing asked for
    # four floats each of gate, x and h, two of the states, and their gradients; outputs over anything else are refused
    q = [p + 16 * k for k in range(9)]
    for out in (q[0] + 4, q[1] - 4, q[2], q[2] + 4):
        assert call(ctx, 0, 1, 2, 2, q[0], q[1], q[2], out, q[4]) == -4, out
    for last in (q[0], q[1] + 12, q[2] + 4, q[3], q[3] + 8):
        assert call(ctx, 0, 1, 2, 2, q[0], q[1], q[2], q[3], last) == -4, last
    assert call(ctx, 0, 1, 1, 4, q[0], q[1], q[2], q[2], q[2]) == -4
    ok = [q[0], q[1], q[2], q[3], q[4], q[5], q[6], q[7], q[8]]
    for k in (4, 5, 6):
        for other in range(9):
            if other != k:
                args = list(ok)
                args[k] = ok[other]
                assert grad(ctx, 1, 1, 2, 2, *args, 0.0) == -4, (k, other)


def test_refusals_come_before_anything_touches_the_device():
    """Every bad argument is answered from the arguments alone: a context that is only zeroed memory will do."""
    from sliced_amd import _lib
    blank = C.create_string_buffer(4096)
    refused(_lib.load(), C.addressof(blank))


@pytest.mark.gpu
def test_refusals(hip):
    refused(hip.ctx().lib, hip.ctx().h)
