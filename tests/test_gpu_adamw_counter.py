"""The step counter on the device is one of the arrays that an AdamW call writes: it may share memory with none of them."""
import ctypes as C

import pytest


def refused(lib, ctx, count):
    room = C.create_string_buffer(1 << 16)
    at = (C.addressof(room) + 63) & ~63
    lens = (C.c_size_t * count)(*[16] * count)
    kinds = [[at + (k * count + i) * 64 for i in range(count)] for k in range(5)]       # 64 bytes each, nothing between them
    arrays = [(C.c_void_p * count)(*k) for k in kinds]
    behind = at + 5 * count * 64
    nan, rates = float("nan"), [0.9, 0.999, 1e-8, 0.0]

    def f32(counter, lr=1e-3):
        return lib.slhip_adamw_step_multi(ctx, count, *arrays[:4], lens, lr, *rates, 0, counter)

    def eight(counter, lr=1e-3):
        return lib.slhip_adamw8_step_multi(ctx, count, *arrays, lens, lr, *rates, 0, counter, 0)

    for i in (0, count // 2, count - 1):
        for kind in range(4):                                # parameters, gradients, moments: first and last eight bytes
            assert f32(kinds[kind][i]) == -4 and f32(kinds[kind][i] + 56) == -4, (kind, i)
        for kind, used in ((0, 64), (1, 64), (2, 16), (3, 16), (4, 8)):
            assert eight(kinds[kind][i]) == -4 and eight(kinds[kind][i] + used - 8) == -4, (kind, i)
        for kind, used in ((2, 16), (3, 16), (4, 8)):        # behind what is there of it (it is the rate that is refused)
            assert eight(kinds[kind][i] + used, nan) == -1, (kind, i)
    assert f32(behind, nan) == -1 and eight(behind, nan) == -1


@pytest.mark.parametrize("count", [1, 64, 65, 150])
def test_refused_before_anything_touches_the_device(count):
    from sliced_amd import _lib
    blank = C.create_string_buffer(4096)
    refused(_lib.load(), C.addressof(blank), count)


@pytest.mark.gpu
def test_refused(hip):
    refused(hip.ctx().lib, hip.ctx().h, 70)
