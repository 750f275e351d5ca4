"""The sigmoid of the gated recurrence and of SiLU where it is next to nothing: exp(-|z|) is a float down to |z| = 103.9, its
last part, from 87.3 on, a subnormal one.

With u = 2^-24 and q = 2^-149, the smallest float: 1/(1 + exp(|z|)) is e / (1 + e), six roundings of itself and, where it is
subnormal, two of up to q / 2 each."""
import numpy as np
import pytest

U, SMALLEST = 2.0 ** -24, 2.0 ** -149


def small_sigmoid(z):
    return 1 / (1 + np.exp(np.abs(z.astype(np.float64))))


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [1, 40])
def test_gates_of_the_recurrence(hip, steps):
    """gate z > 0 takes up 1/(1 + exp(z)) of x: from a state of zero, h_1 is that times x."""
    z = np.linspace(60, 110, 4001).astype(np.float32)
    gate, x = np.full((1, steps, z.size), np.inf, np.float32), np.zeros((1, steps, z.size), np.float32)
    gate[0, 0], x[0, 0] = z, 2.0 ** 100                      # the steps behind it keep the state as it is
    h = hip.gated_scan(1, 1, steps, z.size, gate, x)[0].reshape(steps, z.size).astype(np.float64)
    want = small_sigmoid(z) * 2.0 ** 100
    assert (np.abs(h - want) <= 6 * U * want + 2.0 ** 100 * SMALLEST).all(), np.argwhere(np.abs(h - want) > 6 * U * want + 2.0 ** 100 * SMALLEST)[:3]
    gate[0, 0] = -z                                          # and keeps as little of a state
    h0 = np.full((1, z.size), 2.0 ** 100, np.float32)
    h = hip.gated_scan(1, 1, steps, z.size, gate, np.zeros_like(x), h0)[0].reshape(steps, z.size).astype(np.float64)
    assert (np.abs(h - want) <= 6 * U * want + 2.0 ** 100 * SMALLEST).all()


@pytest.mark.gpu
def test_silu_far_below_zero(hip):
    """SiLU(u) = u / (1 + exp(-u)) and its slope for u from -60 to -110, as the biases of a group whose values are all equal."""
    u = -np.linspace(60, 110, 4001).astype(np.float32)
    c = u.size
    x, w = np.zeros((1, 1, c), np.float32), np.ones(c, np.float32)
    out, mean, rstd = hip.group_norm(1, 1, c, 1, x, w, u, act=2)
    q, f = small_sigmoid(u), u.astype(np.float64)
    tol = 8 * U * np.abs(f * q) + (1 + np.abs(f)) * SMALLEST
    assert (np.abs(out - f * q) <= tol).all()
    grads = [np.zeros(c, np.float32), np.zeros(c, np.float32), np.zeros(c, np.float32)]
    hip.group_norm_grad(1, 1, c, 1, x, w, u, mean, rstd, np.full(c, 2.0 ** 100, np.float32), *grads, act=2)
    slope = q * (1 + f * (1 - q))
    # (the bracket is 1 + u with three roundings of u; times q)
    assert (np.abs(grads[2] - slope * 2.0 ** 100) <= 2.0 ** 100 * (14 * U * np.abs(f * q) + (2 + np.abs(f)) * SMALLEST)).all()
