"""Waits of kernels that call the engine: none is without a bound, and a call that
gives up leaves the ring as it was."""
import numpy as np
import pytest
import torch

import accl_amd as A
import accl_amd._core as core

SEGMENT = 8192  # floats of a segment of the demo kernel

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(),
                                           reason="no HIP GPU")]


@pytest.mark.parametrize("demo", ["demo_vadd_put", "demo_vadd_devicecall"])
def test_needs_a_gpu_engine(demo):
    a = A.ACCL(nranks=1, rank=0, backend="emu", job=f"waits_{demo}",
               heap_bytes=1 << 20)
    try:
        s = a.create_buffer(16, A.DataType.float32)
        args = (s, 16, 0) if demo == "demo_vadd_put" else (s, s, 16, 0)
        with pytest.raises(RuntimeError, match="gpu backend only"):
            getattr(core, demo)(a._a, *args)
    finally:
        a.close()


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="no HIP GPU")
def test_refuses_ranks_and_counts_that_are_not_there():
    """On the host: neither call launches anything."""
    a = A.ACCL(nranks=1, rank=0, backend="gpu", heap_bytes=64 << 20)
    try:
        s, t = (a.create_buffer(n, A.DataType.float32) for n in (16, 8))
        for call in (lambda: core.demo_vadd_put(a._a, s, 16, 1),
                     lambda: core.demo_vadd_put(a._a, s, 17, 0),
                     lambda: core.demo_vadd_devicecall(a._a, s, s, 16, 1),
                     lambda: core.demo_vadd_devicecall(a._a, s, t, 9, 0),
                     lambda: core.demo_vadd_devicecall(a._a, t, s, 9, 0)):
            with pytest.raises(RuntimeError, match="no such rank"):
                call()
    finally:
        a.close()


@pytest.mark.parametrize("rooms", [1, 4])
@pytest.mark.parametrize("wait_ms", [0, 20])
class TestPush:
    pytestmark = gpu

    def test_gives_up_where_nobody_pops(self, rooms, wait_ms):
        a = A.ACCL(nranks=1, rank=0, backend="gpu", heap_bytes=64 << 20,
                   n_stream=rooms)
        try:
            cnt = (rooms + 2) * SEGMENT - 100
            s = a.create_buffer(cnt, A.DataType.float32)
            x = np.arange(cnt, dtype=np.float32)
            s.write(x)
            buf = np.zeros(cnt, np.float32)
            for tag in (7, 8):
                with pytest.raises(RuntimeError, match="TIMEOUT"):
                    core.demo_vadd_put(a._a, s, cnt, 0, tag, 1.0, wait_ms)
                for i in range(rooms):
                    n, got = a.pop_stream(0, buf)
                    assert n == SEGMENT * 4 and got == tag
                    assert np.array_equal(
                        buf[:SEGMENT], x[i * SEGMENT:(i + 1) * SEGMENT] + 1)
            # what fits goes through
            core.demo_vadd_put(a._a, s, 100, 0, 9, 2.0, wait_ms)
            n, got = a.pop_stream(0, buf)
            assert n == 400 and got == 9
            assert np.array_equal(buf[:100], x[:100] + 2)
        finally:
            a.close()
