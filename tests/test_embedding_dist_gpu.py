"""The tensor operators over the "accl" backend between two GPU engines that share
one card: sparse gradients through all_reduce, and a sequence-parallel block that
gathers 8-bit activations."""
import multiprocessing as mp
import os
import traceback

import pytest
import torch

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(),
                                 reason="no HIP GPU")]


def _sparse(rows, ids, values):
    return torch.sparse_coo_tensor(
        torch.tensor([ids], dtype=torch.int64, device="cuda"), values,
        (rows, *values.shape[1:]))


def _all_reduce_sparse(dist, rank, world):
    # one rank names a row twice, ranks differ in length, rows overlap
    def part(r):
        ids = [[3, 9, 3], [0, 9, 7, 5, 1]][r]
        g = torch.Generator().manual_seed(r)
        return ids, torch.randint(-8, 8, (len(ids), 6), generator=g).float()
    want = torch.zeros(10, 6)
    for r in range(world):
        ids, values = part(r)
        want.index_add_(0, torch.tensor(ids), values)
    ids, values = part(rank)
    t = _sparse(10, ids, values.cuda())
    dist.all_reduce(t)
    assert t.is_coalesced()
    assert t._indices().tolist() == [[0, 1, 3, 5, 7, 9]]
    assert torch.equal(t.to_dense().cpu(), want)  # small integers: exact
    t = _sparse(10, ids, values.bfloat16().reshape(-1, 2, 3).cuda())
    dist.all_reduce(t, op=dist.ReduceOp.AVG)
    assert t.dtype == torch.bfloat16 and t.shape == (10, 2, 3)
    assert torch.equal(t.to_dense().float().cpu().reshape(10, 6), want / 2)
    # one rank, or all of them, without a row
    none = torch.zeros(0, 6, device="cuda")
    t = _sparse(10, [], none) if rank else _sparse(10, ids, values.cuda())
    dist.all_reduce(t)
    ids, values = part(0)
    want = torch.zeros(10, 6).index_add_(0, torch.tensor(ids), values)
    assert torch.equal(t.to_dense().cpu(), want)
    t = _sparse(10, [], none)
    dist.all_reduce(t)
    assert t._nnz() == 0
    # more rows than a rank of the sort takes at once
    n = 3000 + 500 * rank
    ids = torch.arange(n, device="cuda") * 7 % 2000
    t = torch.sparse_coo_tensor(ids[None], torch.ones(n, 40, device="cuda"),
                                (2000, 40))
    dist.all_reduce(t)
    want = sum(torch.bincount(torch.arange(3000 + 500 * r) * 7 % 2000,
                              minlength=2000) for r in range(world))
    assert torch.equal(t.to_dense().cpu(),
                       want.float()[:, None].expand(2000, 40))


def _sequence_parallel(dist, rank, world):
    """Each rank holds half of a sequence; the results and gradients are
    those of the whole sequence on one rank."""
    from accl_amd import torch_ops as ops
    g = torch.Generator().manual_seed(2)
    x = torch.randn(8, 3, 40, generator=g).cuda()
    w = (torch.randn(2 * 24, 40, generator=g) * 0.2).cuda()
    up = torch.randn(8, 3, 24, generator=g).cuda()

    def step(part, group):
        part = part.clone().requires_grad_()
        weight = w.clone().requires_grad_()
        y = ops.act8_swiglu(ops.act8_linear(part, weight, group=group))
        y.backward(up)
        return y.detach(), part.grad, weight.grad
    y, d_x, d_w = step(x[4 * rank:4 * rank + 4], dist.group.WORLD)
    y1, d_x1, d_w1 = step(x, None)
    assert torch.equal(y, y1)
    assert torch.equal(d_w, d_w1)  # the gathered codes are those of the whole
    # both ranks compute the same product here, and their sum is scattered
    assert torch.equal(d_x, world * d_x1[4 * rank:4 * rank + 4])


def _main(fn, rank, world, port, q):
    try:
        os.environ["MASTER_ADDR"] = "127.0.0.1"
        os.environ["MASTER_PORT"] = str(port)
        os.environ.setdefault("ACCL_ENGINE_WGS", "64")  # 2 engines, 1 GPU
        import torch.distributed as dist

        import accl_amd.torch_backend  # noqa: F401  (registers "accl")
        dist.init_process_group("accl", rank=rank, world_size=world)
        fn(dist, rank, world)
        dist.barrier()
        dist.destroy_process_group()
        q.put((rank, None))
    except Exception:
        q.put((rank, traceback.format_exc()))


@pytest.mark.parametrize("fn", [_all_reduce_sparse, _sequence_parallel],
                         ids=["all_reduce_sparse", "sequence_parallel"])
def test_two_engines_of_one_gpu(fn):
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = 31000 + os.getpid() % 200 + 200 * (fn is _sequence_parallel)
    ps = [ctx.Process(target=_main, args=(fn, r, 2, port, q))
          for r in range(2)]
    for p in ps:
        p.start()
    errs = []
    try:
        for _ in ps:
            rank, err = q.get(timeout=90)
            if err:
                errs.append(f"rank {rank}:\n{err}")
    finally:
        for p in ps:
            p.join(timeout=15)
            if p.is_alive():
                p.terminate()
                errs.append("rank hung")
    assert not errs, "\n".join(errs)
