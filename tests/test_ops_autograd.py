"""Derivatives of accl_amd.torch_ops where they are easily lost: tokens far from
a shard, tensors without elements, forward mode, captures."""
import pytest
import torch

from accl_amd import torch_ops as ops

# Other tests fork this process: a pool of threads, which a fork does not
# take along, must not have been started by then.
torch.set_num_threads(1)

_NEEDS = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(),
                                              reason="no HIP GPU")]
DEVICES = ["cpu", pytest.param("cuda", marks=_NEEDS)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens", [3, 300, 5000])
@pytest.mark.parametrize("first", [2 ** 32 + 5, 2 ** 31, -2 ** 31, 2 ** 62])
def test_shard_far_from_the_tokens(device, index, tokens, first):
    """No token of a 32-bit type is in such a shard, though a difference in 32
    bits would be: zeros, and no gradient, dense or sparse."""
    ids = torch.arange(tokens, device=device, dtype=index).remainder(8) + 5
    w = torch.ones(64, 3, device=device)
    for sparse in (False, True):
        leaf = w.clone().requires_grad_()
        out = ops.embedding(ids, leaf, first_row=first, sparse=sparse)
        assert not out.any()
        out.backward(torch.ones_like(out))
        assert leaf.grad.is_sparse == sparse
        assert not leaf.grad.to_dense().any()
        if sparse:
            assert leaf.grad._nnz() == 0


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("tokens", [4, 300, 5000])
@pytest.mark.parametrize("first", [2 ** 40, -7, 1000])
def test_sparse_gradient_of_a_shard(device, tokens, first):
    """The touched rows, counted from the shard's first."""
    ids = torch.arange(tokens, device=device).remainder(20) * 3 + first - 6
    up = torch.ones(tokens, 5, device=device)
    leaf = torch.zeros(31, 5, device=device).requires_grad_()
    ops.embedding(ids, leaf, 2.0, first, sparse=True).backward(up)
    at = (ids - first).cpu()
    here = at[(at >= 0) & (at < 31)]
    want = torch.bincount(here, minlength=31).float() * 2
    assert leaf.grad._indices()[0].tolist() == here.unique().tolist()
    assert torch.equal(leaf.grad.to_dense().cpu(), want[:, None].expand(31, 5))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("sparse", [False, True])
@pytest.mark.parametrize("shape", [(3,), (2, 3), (0,), (0, 3), ()])
@pytest.mark.parametrize("rows,width", [(10, 0), (0, 4), (10, 4)])
def test_embedding_without_elements(device, sparse, shape, rows, width):
    weight = torch.ones(rows, width, device=device).requires_grad_()
    ids = torch.ones(shape, dtype=torch.int64, device=device)
    out = ops.embedding(ids, weight, sparse=sparse)
    assert out.shape == (*shape, width)
    out.backward(torch.ones_like(out))
    want = torch.zeros(rows, width)
    want[1:2] = ids.numel()
    assert torch.equal(weight.grad.to_dense().cpu(), want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lead", [(5,), (2, 3), (0,), (0, 3), ()])
@pytest.mark.parametrize("outputs,width", [(24, 0), (0, 40), (0, 0), (24, 40)])
def test_linear_without_elements(device, lead, outputs, width):
    x = torch.ones(*lead, width, device=device).requires_grad_()
    w = torch.ones(outputs, width, device=device).requires_grad_()
    with torch.no_grad():
        assert ops.act8_linear(x, w).shape == (*lead, outputs)
    y = ops.act8_linear(x, w)
    assert y.shape == (*lead, outputs) and (y == width).all()
    y.backward(torch.ones_like(y))
    assert x.grad.shape == x.shape and (x.grad == outputs).all()
    assert w.grad.shape == w.shape
    assert (w.grad == torch.Size(lead).numel()).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lead", [(5,), (0,), (0, 3)])
@pytest.mark.parametrize("width", [0, 6])
def test_swiglu_without_elements(device, lead, width):
    x = torch.ones(*lead, 2 * width, device=device).requires_grad_()
    y = ops.act8_swiglu(x)
    assert y.shape == (*lead, width)
    y.backward(torch.ones_like(y))
    assert x.grad.shape == x.shape and x.grad.isfinite().all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("trained", [False, True])
def test_forward_mode_is_refused(device, trained):
    """A result without a tangent would read as a derivative of zero."""
    import torch.autograd.forward_ad as fwd
    ids = torch.tensor([1, 2], device=device)
    x = torch.ones(2, 8, device=device).requires_grad_(trained)
    kept = ops.act8_pack(torch.ones(2, 8, device=device))
    two = ops.act8_swiglu_forward(torch.ones(2, 8, device=device))[1]
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: ops.embedding(ids, dual),
                     lambda: ops.embedding(ids, dual, sparse=True),
                     lambda: ops.embedding_grad(dual, ids, 4),
                     lambda: ops.sum_rows(ids, dual, 4),
                     lambda: ops.act8_pack(dual),
                     lambda: ops.act8_weight_grad(dual, kept),
                     lambda: ops.act8_swiglu(dual),
                     lambda: ops.act8_swiglu_forward(dual),
                     lambda: ops.act8_swiglu_grad(dual[:, :4], two)):
            with pytest.raises(RuntimeError, match="forward"):
                call()
        out = torch.zeros(4, 8, device=device)
        with pytest.raises(RuntimeError, match="forward"):
            ops.embedding_grad(x.detach(), ids, 4,
                               out=fwd.make_dual(out, torch.ones_like(out)))
        # tensors without a tangent are as ever
        assert ops.embedding(ids, x).shape == (2, 8)
        ops.act8_swiglu(x)
    ops.embedding(ids, dual)


@pytest.mark.parametrize("device", DEVICES)
def test_forward_mode_of_the_product(device):
    """With operands that are not trained act8_linear is torch's product, and
    has its tangent."""
    import torch.autograd.forward_ad as fwd
    x, w = torch.ones(2, 8, device=device), torch.ones(3, 8, device=device)
    with fwd.dual_level():
        y = ops.act8_linear(fwd.make_dual(x, 2 * x), w)
        assert (fwd.unpack_dual(y).tangent == 16).all()
        with pytest.raises(RuntimeError):
            ops.act8_linear(fwd.make_dual(x, 2 * x),
                            w.clone().requires_grad_())


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="no HIP GPU")
@pytest.mark.parametrize("operator", ["embedding", "linear"])
@pytest.mark.parametrize("held", [False, True])
def test_capture_after_steps_on_a_side_stream(operator, held):
    """Eager steps on a side stream, whose results still live, then a capture of
    forward and backward pass on another one, replayed over new inputs. With
    `held` the parameter's accumulator is kept as DDP keeps it."""
    g = torch.Generator().manual_seed(0)
    w = torch.randn(50, 64, generator=g).cuda().requires_grad_()
    x = torch.randn(10, 64, generator=g).cuda()
    ids = torch.randint(0, 50, (10,), generator=g).cuda()

    def step(weight):
        y = ops.embedding(ids, weight, 2.0) if operator == "embedding" else \
            ops.act8_linear(x, weight)
        y.backward(y.detach())
        return y
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        if held:
            kept = w.view_as(w).grad_fn.next_functions[0][0]
        for _ in range(3):
            w.grad = None
            alive = step(w)
    torch.cuda.current_stream().wait_stream(side)
    w.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step(w)
    for seed in range(3):
        g.manual_seed(seed)
        with torch.no_grad():
            x.copy_(torch.randn(10, 64, generator=g).cuda())
            ids.copy_(torch.randint(0, 50, (10,), generator=g).cuda())
        graph.replay()
        torch.cuda.synchronize()
        leaf = w.detach().requires_grad_()
        assert torch.equal(step(leaf), y)
        assert torch.equal(leaf.grad, w.grad)
    assert alive.shape == y.shape and (not held or kept is not None)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_out_between_the_columns_of_an_operand(device, dtype):
    """Columns of one buffer, side by side: rows of out lie between rows of the
    operand, and share no element with them."""
    g = torch.Generator().manual_seed(0)
    room = torch.randn(40, 48, generator=g).to(dtype).to(device)
    grad, out = room[:24, :19], room[:, 19:38]
    ids = torch.arange(24, device=device).remainder(7)
    want = ops.embedding_grad(grad.clone(), ids, 40, out=out.clone())
    before = room.clone()
    assert ops.embedding_grad(grad, ids, 40, out=out) is out
    assert torch.equal(out, want)
    assert torch.equal(room[:, :19], before[:, :19])
    assert torch.equal(room[:, 38:], before[:, 38:])
    # behind the columns of out, and round the end of a row
    ops.embedding_grad(room[:24, 29:48], ids, 40, out=room[:, 5:24])
    ops.embedding_grad(room.view(-1)[43:43 + 48 * 24].view(24, 48)[:, :8], ids,
                       40, out=room[:, 3:11])
    kept = ops.act8_pack(torch.ones(40, 19, device=device, dtype=dtype))
    ops.act8_weight_grad(room[:, :24], kept, out=room[:24, 24:43])


@pytest.mark.parametrize("device", DEVICES)
def test_out_that_shares_elements(device):
    room = torch.zeros(40, 48, device=device)
    ids = torch.arange(24, device=device).remainder(7)
    flat = room.view(-1)
    for grad, out in [
            (room[:24, :19], room[:, 18:37]),
            (room[:24, 20:39], room[:, 20:39]),
            (room[:24, 20:39], room[:, 2:21]),
            # a row that goes on at the beginning of the next
            (flat[40:40 + 48 * 24].view(24, 48)[:, :9], room[:, :9]),
            (room[:24, :9], flat[40:40 + 48 * 39].view(39, 48)[:, :9]),
            # rows of another distance
            (flat[19:19 + 24 * 19].view(24, 19), room[:, 19:38]),
            (room.t()[:24, :19], room[:, 19:38])]:
        with pytest.raises(ValueError, match="shares"):
            ops.embedding_grad(grad, ids[:len(grad)], out.size(0), out=out)
    with pytest.raises(ValueError, match="shares"):
        ops.embedding_grad(torch.zeros(480, 5, device=device),
                           room.view(torch.int32).view(-1)[:480],
                           40, out=room[:, 7:12])


@pytest.mark.parametrize("device", DEVICES)
def test_gated_unit_of_large_gates(device):
    """Both directions of gates far from zero, where the logistic function is a
    power of e or one less such a power: off by 7 units of 2^-24, and by one for
    each product behind it (two, and two more that the codes leave exact)."""
    # multiples of 2^-1 below 127 of them: what is kept is exact
    gate = torch.arange(-126, 127).remainder(127).sub(63).mul(0.5)
    gate = torch.cat([gate, -gate]).clamp(-60, 60).view(-1, 1).expand(-1, 32)
    gate = gate.contiguous()
    gate[:, 0] = 63.5  # the group's unit
    up = torch.ones_like(gate)
    x = torch.cat([gate, up], 1)
    y, kept = ops.act8_swiglu_forward(x.to(device))
    assert torch.equal(ops.act8_unpack(kept).cpu(), x)
    d = ops.act8_swiglu_grad(torch.ones_like(y), kept)
    wide = gate.double()
    sig = 1 / (1 + torch.exp(-wide))
    exact = wide * sig
    unit = 2.0 ** -24
    assert ((y.cpu().double() - exact).abs() <= 9 * unit * exact.abs()).all()
    assert ((d[:, 32:].cpu().double() - exact).abs()
            <= 9 * unit * exact.abs()).all()
