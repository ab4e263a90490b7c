"""Types of accl_amd.torch_ops' 8-bit activations: kept values that float16 does
not hold, and products under autocast."""
import pytest
import torch

from accl_amd import torch_ops as ops

# Other tests fork this process: a pool of threads, which a fork does not
# take along, must not have been started by then.
torch.set_num_threads(1)

DEVICES = ["cpu", pytest.param("cuda", marks=[
    pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(),
                                        reason="no HIP GPU")])]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows", [1, 70, 200])
@pytest.mark.parametrize("width", [3, 32, 71])
def test_codes_that_float16_does_not_hold(device, rows, width):
    """A group whose values would overflow gives NaN, as one with an infinity
    does, and leaves its neighbours alone. The largest exponent of values that
    came from float16 is exact."""
    groups = -(-width // 32)
    codes = torch.full((rows, width), 2, dtype=torch.int8)
    exps = torch.full((rows, groups), 9, dtype=torch.int8)
    grad = torch.full((rows, 5), 2.0 ** -10, dtype=torch.float16)
    want = torch.full((5, width), float(rows))
    kept = ops.Act8(codes.to(device), exps.to(device), torch.float16)
    got = ops.act8_weight_grad(grad.to(device), kept, dtype=torch.float32)
    assert torch.equal(got.cpu(), want)
    for e in (10, 60, 121):
        exps[rows // 2, groups - 1] = e
        kept = ops.Act8(codes.to(device), exps.to(device), torch.float16)
        got = ops.act8_weight_grad(grad.to(device), kept,
                                   dtype=torch.float32).cpu()
        bad = 32 * (groups - 1)
        assert got[:, bad:].isnan().all()
        assert torch.equal(got[:, :bad], want[:, :bad])
    # the other types hold them
    kept = ops.Act8(codes.to(device), exps.to(device), torch.bfloat16)
    got = ops.act8_weight_grad(grad.bfloat16().to(device), kept,
                               dtype=torch.float32).cpu()
    assert got.isfinite().all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("needs", ["x", "weight", "both"])
@pytest.mark.parametrize("inside", [False, True])
def test_linear_under_autocast(device, dtype, needs, inside):
    """As with both operands cast by hand, forward and backward, wherever the
    backward pass runs."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(6, 40, generator=g).to(device)
    w = torch.randn(24, 40, generator=g).to(device)
    up = torch.randn(6, 24, generator=g).to(dtype).to(device)
    x.requires_grad_(needs != "weight")
    w.requires_grad_(needs != "x")
    leaves = [t for t in (x, w) if t.requires_grad]
    want = ops.act8_linear(x.to(dtype), w.to(dtype))
    want_d = torch.autograd.grad(want, leaves, up)
    with torch.autocast(device, dtype):
        y = ops.act8_linear(x, w)
        assert y.dtype == dtype and torch.equal(y, want)
        if inside:
            d = torch.autograd.grad(y, leaves, up)
    if not inside:
        d = torch.autograd.grad(y, leaves, up)
    for got, right in zip(d, want_d):
        assert got.dtype == torch.float32 and torch.equal(got, right)
    with torch.autocast(device, dtype), torch.no_grad():
        assert torch.equal(ops.act8_linear(x, w), want)


@pytest.mark.parametrize("device", DEVICES)
def test_linear_keeps_its_types_in_the_backward_pass(device):
    """A forward pass outside of autocast: the backward pass inside of it has
    products of the same types."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(6, 40, generator=g).to(device).requires_grad_()
    w = torch.randn(24, 40, generator=g).to(device).requires_grad_()
    up = torch.randn(6, 24, generator=g).to(device)
    want = torch.autograd.grad(ops.act8_linear(x, w), (x, w), up)
    y = ops.act8_linear(x, w)
    with torch.autocast(device, torch.bfloat16):
        got = torch.autograd.grad(y, (x, w), up)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("device", DEVICES)
def test_linear_under_autocast_takes_operands_of_two_types(device):
    x = torch.ones(3, 40, device=device)
    w = torch.ones(5, 40, device=device, dtype=torch.bfloat16)
    with pytest.raises(TypeError):
        ops.act8_linear(x, w)
    with torch.autocast(device, torch.bfloat16):
        assert (ops.act8_linear(x, w) == 40).all()


@pytest.mark.parametrize("device", DEVICES)
def test_what_float16_does_not_hold_is_seen_under_autocast(device):
    x = torch.ones(3, 40, device=device)
    x[1, 35] = 1e6
    w = torch.ones(5, 40, device=device).requires_grad_()
    with torch.autocast(device, torch.float16):
        y = ops.act8_linear(x, w)
    d, = torch.autograd.grad(y, w, torch.ones_like(y))
    assert d[:, 32:].isnan().all() and (d[:, :32] == 3).all()
