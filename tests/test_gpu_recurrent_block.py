"""Group norm, the gated recurrence and AdamW together, on the tape: a recurrent block

    n = silu(group_norm(x));  z = n Wz + bz;  v = n Wv + bv;  h = gated_scan(z, v);  y = group_norm(h) Wo + bo;  L = mse(y, t)

trained the way the example loops train, against the same graph in 64-bit torch on the CPU.

Tolerance of a gradient: the graph in 32-bit torch makes the same roundings in another order, a few thousand of them on the longest
path here (sums of 192 products, 24 steps of a recurrence, their gradients); what 32 bits cost is measured on it, and the kernels
may be four times as far from the 64-bit graph in the 2-norm, or 64 units of 2^-24."""
import numpy as np
import pytest
import torch

from sliced_amd import rng

SEED = 0x51CED
U = 2.0 ** -24
B, T, D, H, G = 4, 24, 24, 32, 4          # sequences, steps, width, channels of the recurrence, groups
NAMES = ("w1", "b1", "wz", "bz", "wv", "bv", "w2", "b2", "wo", "bo")


def inputs():
    n = lambda k, *s: rng.normal(int(np.prod(s)), 1.0, tag=k, seed=SEED).reshape(s).astype(np.float32)  # noqa: E731
    p = {"w1": 1 + 0.2 * n(1, D), "b1": 0.2 * n(2, D), "wz": 0.3 * n(3, D, H), "bz": 1 + 0.2 * n(4, H), "wv": 0.3 * n(5, D, H), "bv": 0.1 * n(6, H),
         "w2": 1 + 0.2 * n(7, H), "b2": 0.1 * n(8, H), "wo": 0.3 * n(9, H, D), "bo": 0.1 * n(10, D)}
    return {k: v.astype(np.float32) for k, v in p.items()}, n(11, B * T, D), n(12, B * T, D)


def torch_norm(x, w, b):
    g = x.reshape(x.shape[0], G, -1)
    m = g.mean(dim=2, keepdim=True)
    r = 1 / torch.sqrt(((g - m) ** 2).mean(dim=2, keepdim=True) + 1e-5)
    return ((g - m) * r).reshape(x.shape) * w + b


def torch_loss(p, x, t):
    u = torch_norm(x, p["w1"], p["b1"])
    n = u * torch.sigmoid(u)
    z, v = n @ p["wz"] + p["bz"], n @ p["wv"] + p["bv"]
    s = torch.sigmoid(z).reshape(B, T, H)
    v = v.reshape(B, T, H)
    h, out = torch.zeros(B, H, dtype=x.dtype), []
    for k in range(T):
        h = s[:, k] * h + (1 - s[:, k]) * v[:, k]
        out.append(h)
    h = torch.stack(out, dim=1).reshape(B * T, H)
    y = torch_norm(h, p["w2"], p["b2"]) @ p["wo"] + p["bo"]
    return ((y - t) ** 2).mean()


def torch_grads(p, x, t, dtype):
    q = {k: torch.tensor(v, dtype=dtype, requires_grad=True) for k, v in p.items()}
    xs = torch.tensor(x, dtype=dtype, requires_grad=True)
    loss = torch_loss(q, xs, torch.tensor(t, dtype=dtype))
    loss.backward()
    return loss.item(), dict({k: v.grad.numpy().astype(np.float64) for k, v in q.items()}, x=xs.grad.numpy().astype(np.float64))


def device_loss(d, q, x, t):
    from sliced_amd import host
    n = d.group_norm(B * T, 1, D, G, x, q["w1"], q["b1"], act=host.ACT_SILU)
    z = d.linear(B * T, D, H, n, q["wz"], q["bz"], False)
    v = d.linear(B * T, D, H, n, q["wv"], q["bv"], False)
    h = d.gated_scan(host.SCAN_SIGMOID, B, T, H, z, v)
    y = d.linear(B * T, H, D, d.group_norm(B * T, 1, H, G, h, q["w2"], q["b2"]), q["wo"], q["bo"], False)
    return d.mse_loss(y, t)


@pytest.mark.gpu
def test_block_gradients():
    from sliced_amd import host
    p, x, t = inputs()
    loss, want = torch_grads(p, x, t, torch.float64)
    _, rough = torch_grads(p, x, t, torch.float32)
    with host.HIP(0, cached=False) as d:
        # the tape's matrix products overwrite their operands' gradients as the reference's CPU device does; n has two readers
        d.set_grad_policy(gemm_beta=1.0)
        q = {k: d.buffer(v) for k, v in p.items()}
        xs, ts = d.buffer(x), d.buffer(t)
        out = device_loss(d, q, xs, ts)
        assert abs(out.read()[0] - loss) <= 64 * U * loss
        out.backward()
        q["x"] = xs
        for k, w in want.items():
            got = q[k].grad().read().astype(np.float64).reshape(w.shape)
            size = np.linalg.norm(w)
            off, allowed = np.linalg.norm(got - w) / size, max(4 * np.linalg.norm(rough[k] - w) / size, 64 * U)
            print("gradient of %-2s off by %.2e, allowed %.2e" % (k, off, allowed), flush=True)
            assert off <= allowed, k


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [False, True])
def test_block_trains_eagerly_and_recorded_alike(eight):
    """Six AdamW steps through the C++ optimiser: the steps run eagerly give the parameters of the steps recorded once and
    replayed, bit for bit, and (f32 moments) those of torch's AdamW in 64 bits."""
    from sliced_amd import host
    p, x, t = inputs()
    ends = []
    for recorded in (False, True):
        with host.HIP(0, cached=True) as d:
            d.set_grad_policy(gemm_beta=1.0)
            q = {k: d.buffer(v) for k, v in p.items()}
            xs, ts = d.buffer(x).no_grad(), d.buffer(t).no_grad()
            opt = d.adamw([q[k] for k in NAMES], lr=1e-2, weight_decay=0.1, eight=eight)

            def step():
                d.begin_iteration()
                d.zero_grad()
                device_loss(d, q, xs, ts).backward()
                opt.step()

            step()
            step()
            if recorded:
                for _ in range(4):                    # record_end() runs what was recorded once
                    d.record_begin()
                    step()
                    assert d.record_end() > 10
            else:
                for _ in range(4):
                    step()
            ends.append({k: q[k].read() for k in NAMES})
            opt.close()
    for k in NAMES:
        assert np.array_equal(ends[0][k], ends[1][k]), k
    ref = {k: torch.tensor(v, dtype=torch.float64, requires_grad=True) for k, v in p.items()}
    torch_opt = torch.optim.AdamW(ref.values(), lr=float(np.float32(1e-2)), betas=(float(np.float32(0.9)), float(np.float32(0.999))), eps=1e-8,
                                  weight_decay=float(np.float32(0.1)))
    for _ in range(6):
        torch_opt.zero_grad()
        torch_loss(ref, torch.tensor(x, dtype=torch.float64), torch.tensor(t, dtype=torch.float64)).backward()
        torch_opt.step()
    if eight:
        return                                        # (its moments are rounded on purpose; what a step may differ by is tested with the step)
    for k in NAMES:
        # a step moves an element by at most 1e-2 * 1.1 in these six; a gradient near zero may be off by as much as it is
        # large, which moves such an element by a part of that: all but one in a hundred agree to 1e-4 of a step each
        off = np.abs(ends[0][k].astype(np.float64) - ref[k].detach().numpy().ravel())
        assert np.mean(off <= 6 * 1e-6) >= 0.99 and off.max() <= 6 * 1.1e-2, (k, float(off.max()))


@pytest.mark.gpu
def test_serving_step_continues_a_prefix():
    """The recurrence over a prefix, then token by token through gated_scan_step, equals the whole sequence."""
    from sliced_amd import host
    g = rng.normal(B * T * H, 1.0, tag=50, seed=SEED).reshape(B, T, H).astype(np.float32)
    v = rng.normal(B * T * H, 1.0, tag=51, seed=SEED).reshape(B, T, H).astype(np.float32)
    with host.HIP(0, cached=False) as d:
        d.enable_tape(False)
        want = d.gated_scan(host.SCAN_SIGMOID, B, T, H, d.buffer(g), d.buffer(v)).read().reshape(B, T, H)
        head = d.gated_scan(host.SCAN_SIGMOID, B, T - 5, H, d.buffer(g[:, :-5]), d.buffer(v[:, :-5])).read().reshape(B, T - 5, H)
        state = d.buffer(head[:, -1])
        for k in range(T - 5, T):
            d.gated_scan_step(host.SCAN_SIGMOID, B, H, d.buffer(g[:, k]), d.buffer(v[:, k]), state)
            # states are averages of v: two roundings of coefficients and sums in each of 24 steps
            assert np.abs(state.read().reshape(B, H) - want[:, k]).max() <= 24 * 12 * U * np.abs(v).max()
        with pytest.raises(host.HostError):
            d.gated_scan_step(host.SCAN_SIGMOID, B, H, state, d.buffer(v[:, 0]), state)


@pytest.mark.gpu
def test_shared_and_missing_operands_on_the_tape():
    """The gate is the input itself, weight and bias are one buffer, and there are none: gradients are the sums of both terms."""
    from sliced_amd import host
    x = rng.normal(6 * 10, 1.0, tag=60, seed=SEED).astype(np.float32)
    w = rng.uniform(10, 0.5, 1.5, tag=61, seed=SEED).astype(np.float32)
    with host.HIP(0, cached=False) as d:
        bx, bw = d.buffer(x), d.buffer(w)
        n = d.group_norm(6, 1, 10, 2, bx, bw, bw)
        d.gated_scan(host.SCAN_SIGMOID, 2, 3, 10, n, n).backward()
        got = bx.grad().read(), bw.grad().read(), n.grad().read()
        n2 = d.group_norm(6, 1, 10, 2, bx)
        d.zero_grad()
        n2.backward()
        plain = bx.grad().read()
    xs, ws = (torch.tensor(v, dtype=torch.float64, requires_grad=True) for v in (x, w))
    g = xs.reshape(6, 2, 5)
    m = g.mean(dim=2, keepdim=True)
    hat = ((g - m) / torch.sqrt(((g - m) ** 2).mean(dim=2, keepdim=True) + 1e-5)).reshape(6, 10)
    n = hat * ws + ws
    n.retain_grad()
    s = torch.sigmoid(n).reshape(2, 3, 10)
    v, h, total = n.reshape(2, 3, 10), 0, 0
    for k in range(3):
        h = s[:, k] * h + (1 - s[:, k]) * v[:, k]
        total = total + h.sum()
    total.backward()
    for a, b in zip(got, (xs.grad, ws.grad, n.grad)):
        b = b.numpy().ravel()
        assert np.abs(a - b).max() <= 200 * U * np.abs(b).max()
    # the sum of a group's normalised values is zero whatever x is: its gradient is rounding, of terms of size rstd
    assert np.abs(plain).max() <= 64 * U * 10


@pytest.mark.gpu
@pytest.mark.parametrize("optimizer", ["adamw", "adamw8"])
@pytest.mark.parametrize("kind", [0, 1])
def test_example_loops_train_by_adamw(kind, optimizer):
    """The example loops with AdamW: eager, fused and replayed steps start from the same loss and stay together."""
    from sliced_amd import host
    dims = dict(kind=kind, batch=128, d_in=1 if kind == 0 else 20, d_h=32, d_out=1 if kind == 0 else 5)
    x, t = host.mlp_data(dims["kind"], dims["batch"], dims["d_in"], dims["d_out"])
    runs = []
    for fused, graph in ((False, False), (True, False), (True, True)):
        params = host.mlp_init(dims["kind"], dims["d_in"], dims["d_h"], dims["d_out"])
        losses, _ = host.mlp_train(dims["kind"], dims["batch"], dims["d_in"], dims["d_h"], dims["d_out"], x, t, params, 1e-3, 8, 0, fused,
                                   graph=graph, fused_loss=fused, optimizer=optimizer)
        runs.append((losses, params))
    assert np.array_equal(runs[1][0], runs[2][0]) and all(np.array_equal(a, b) for a, b in zip(runs[1][1], runs[2][1]))
    assert abs(runs[0][0][0] - runs[1][0][0]) <= 64 * U * abs(runs[0][0][0])
    assert all(np.isfinite(l).all() for l, _ in runs)
    # eight steps move no parameter by more than the sum of their lengths (|m / sqrt(v)| is at most 1 / sqrt(1 - b1) early on)
    start = host.mlp_init(dims["kind"], dims["d_in"], dims["d_h"], dims["d_out"])
    for a, b in zip(runs[0][1], start):
        assert np.abs(a - b).max() <= 8 * 1e-3 * 4


@pytest.mark.gpu
def test_adamw_errors_on_the_tape():
    from sliced_amd import host
    with host.HIP(0, cached=False) as d:
        a, b = d.buffer([1.0, 2.0]), d.buffer([3.0, 4.0])
        opt = d.adamw([a, b])
        with pytest.raises(host.HostError):           # no gradient yet
            opt.step()
        opt.close()
        with pytest.raises(host.HostError):
            opt.step()
        left = d.adamw([b])                           # closed with the device
        d.add(a, b).backward()
        twice = d.adamw([a, a])
        with pytest.raises(host.HostError, match="overlap"):
            twice.step()
        twice.close()
        with pytest.raises(host.HostError):
            d.gated_scan(host.SCAN_LINEAR, 1, 2, 2, a, b)
        with pytest.raises(host.HostError):
            d.group_norm(1, 1, 2, 3, a)
        with pytest.raises(host.HostError):
            host.mlp_train(0, 8, 1, 4, 1, np.zeros(8, np.float32), np.zeros(8, np.float32), host.mlp_init(0, 1, 4, 1), 1e-3, 1, whole_step=True,
                           optimizer="adamw")
    left.close()
    with pytest.raises(host.HostError):
        left.step()
