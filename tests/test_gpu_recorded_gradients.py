"""Recorded steps add up their gradients like eager ones: zero_grad() only marks gradients of 2^20 floats and more, and what a
recording finds marked belongs before it, not into every replay."""
import ctypes as C

import numpy as np
import pytest

from sliced_amd import rng

SEED = 0x51CED
B, T, D = 4, 513, 520                                        # 1 067 040 elements


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["gated_scan", "group_norm", "square"])
def test_replays_add_to_gradients_that_were_zeroed_before_the_recording(op):
    from sliced_amd import _lib, host
    x = rng.normal(B * T * D, 1.0, tag=1, seed=SEED).astype(np.float32)
    g = rng.normal(B * T * D, 1.0, tag=2, seed=SEED).astype(np.float32)
    w = rng.uniform(D, 0.5, 1.5, tag=3, seed=SEED).astype(np.float32)
    lib = _lib.load()
    ends = []
    for recorded in (False, True):
        with host.HIP(0, cached=True) as d:
            bx, bg, bw = d.buffer(x), d.buffer(g), d.buffer(w)

            def step():
                d.begin_iteration()
                if op == "gated_scan":
                    d.gated_scan(host.SCAN_SIGMOID, B, T, D, bg, bx).backward()
                elif op == "group_norm":
                    d.group_norm(B * T, 1, D, 4, bx, bw, act=host.ACT_SILU).backward()
                else:
                    d.square(bx).backward()

            step()
            d.zero_grad()
            if recorded:
                ctx, graph = d.ctx_handle(), C.c_void_p()
                d.record_begin()
                step()
                assert lib.slhip_graph_end(ctx, C.byref(graph)) == 0
                for _ in range(3):
                    assert lib.slhip_graph_launch(ctx, graph) == 0
                    assert lib.slhip_sync(ctx) == 0
                assert lib.slhip_graph_destroy(graph) == 0
            else:
                for _ in range(3):
                    step()
            ends.append([b.grad().read() for b in ([bx, bg] if op == "gated_scan" else [bx, bw] if op == "group_norm" else [bx])])
    for a, b in zip(*ends):
        assert np.array_equal(a, b) and np.abs(a).max() > 0
