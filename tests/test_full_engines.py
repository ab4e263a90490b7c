"""Two engines of the default size on one GPU."""
import numpy as np
import pytest
import torch

import accl_amd as A
from emu_util import pattern, rd, run_ranks

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(),
                                 reason="no HIP GPU")]


def _collectives(a, rank, n):
    # from what one wave copies to tiles for every wave of a fleet
    for cnt in (1000, 200_000, 60 << 20):
        s, d = (a.create_buffer(cnt, A.DataType.float32) for _ in range(2))
        s.write(pattern(cnt, rank, seed=cnt))
        a.allreduce(s, d, cnt, A.ReduceFunction.SUM)
        want = sum(pattern(cnt, r, seed=cnt) for r in range(n))
        assert np.array_equal(rd(d, cnt), want)
        g = a.create_buffer(cnt * n, A.DataType.float32)
        a.allgather(s, g, cnt)
        assert np.array_equal(rd(g, cnt * n), np.concatenate(
            [pattern(cnt, r, seed=cnt) for r in range(n)]))
    a.barrier()


def test_two_full_engines(monkeypatch):
    monkeypatch.setenv("ACCL_ENGINE_WGS", "684")
    run_ranks(_collectives, 2, backend="gpu", timeout=90)
