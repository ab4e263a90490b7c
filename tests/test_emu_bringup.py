"""Bring-up of emulator ranks that find each other's arenas half made."""
import multiprocessing as mp
import os
import time

import numpy as np

import accl_amd as A


def _rank(rank, job, late, q):
    time.sleep(late)
    a = A.ACCL(nranks=2, rank=rank, backend="emu", job=job,
               heap_bytes=1 << 20)
    s, d = (a.create_buffer(100, A.DataType.float32) for _ in range(2))
    s.write(np.full(100, rank + 1, np.float32))
    a.allreduce(s, d, 100, A.ReduceFunction.SUM)
    out = np.zeros(100, np.float32)
    d.read(out)
    a.barrier()
    a.close()
    q.put((rank, bool((out == 3).all())))


def test_arena_without_its_size_yet():
    """A peer's arena has its name before it has its size: a rank that looks then
    waits, and does not read memory that is not there."""
    from accl_amd.accl import emu_job_name
    job = f"bringup{os.getpid()}"
    early = f"/dev/shm/{emu_job_name(job)}_r1"
    with open(early, "wb"):
        pass
    ctx = mp.get_context("fork")
    q = ctx.Queue()
    ps = [ctx.Process(target=_rank, args=(r, job, 0.5 * r, q))
          for r in range(2)]
    try:
        for p in ps:
            p.start()
        for p in ps:
            p.join(timeout=25)
        assert [p.exitcode for p in ps] == [0, 0]
        assert sorted(q.get(timeout=5) for _ in ps) == [(0, True), (1, True)]
    finally:
        for p in ps:
            if p.is_alive():
                p.terminate()
                p.join(timeout=5)
        if os.path.exists(early):
            os.unlink(early)
