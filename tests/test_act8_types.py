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
