"""The example loops' AdamW, step by step, against its formula on the loops' own gradients.

A step of plain descent at a rate of 2^100 leaves -2^100 g where a parameter was (the parameter itself is below the rounding of
that, or g is zero and nothing moves), so the gradient that the tape hands an optimiser at any parameters can be read off one."""
import numpy as np
import pytest

import test_gpu_adamw as base
import test_gpu_adamw_rounding as rounding
from sliced_amd import rng

RATE = 2.0 ** 100
HYPER = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01)


@pytest.mark.gpu
@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("kind", [0, 1])
def test_steps_are_those_of_the_formula(kind, eight, fused):
    from sliced_amd import host
    dims = (kind, 128, 1 if kind == 0 else 20, 32, 1 if kind == 0 else 5)
    x, t = host.mlp_data(kind, dims[1], dims[2], dims[4])
    start = host.mlp_init(kind, *dims[2:])

    def train(params, lr, steps, optimizer):
        params = [p.copy() for p in params]
        host.mlp_train(*dims, x, t, params, lr, steps, 0, fused, fused_loss=fused, optimizer=optimizer)
        return params

    m, v = ([np.zeros(p.size, np.float32) for p in start] for _ in range(2))
    codes = base.zeros8([p.size for p in start])
    b1, b2 = np.float32(0.9), np.float32(0.999)
    at = start
    for step in range(1, 6):
        far = train(at, RATE, 1, "sgd")
        grads = [((a.astype(np.float64) - b) / RATE).astype(np.float32).ravel() for a, b in zip(at, far)]
        assert all(np.isfinite(g).all() for g in grads) and sum(np.count_nonzero(g) for g in grads) > 100
        new = train(start, HYPER["lr"], step, "adamw8" if eight else "adamw")
        for i, (p, g, q) in enumerate(zip(at, grads, new)):
            if eight:
                m[i], v[i] = base.decode(codes[0][i], codes[1][i], codes[2][i])
            want, tol = base.exact(p.ravel(), g, m[i], v[i], step, **HYPER)
            base.close(q.ravel(), want[0], tol[0], (step, i))
            m[i] = m[i] * b1 + g * (np.float32(1) - b1)
            v[i] = v[i] * b2 + (g * (np.float32(1) - b2)) * g
            if eight:
                codes[0][i], codes[1][i], codes[2][i] = rounding.encode(m[i], v[i], base.random16(p.size, i, step, rng.DEFAULT_SEED))
            if step == 1:                                                 # m / sqrt(v) is g / |g|: none stands still (later ones may turn)
                moved = p.ravel() * (1 - 1e-5) - q.ravel().astype(np.float64)
                strong = np.abs(g) > 1e-4
                # eps / |g| of it, and the roundings of p
                assert (np.abs(moved - 1e-3 * np.sign(g))[strong] <= 1e-3 * 2e-4 + 4 * base.U * np.abs(p).max()).all(), i
        at = new
