"""Tensor operators that stand next to the collectives in a training job.

Two families, for tensors on a GPU (hand-written HIP kernels on the caller's
current stream) and, for ranks of the CPU emulator, for tensors in host
memory:

* the embedding of a vocabulary, whole or sharded over ranks, and its gradient
  summed by sorted tokens, dense or as the rows that were touched.
  ``sum_rows`` is also what reduces sparse gradients in the "accl" backend of
  torch.distributed;
* activations kept in 8 bits between the forward and the backward pass (the
  reference keeps to 16-bit casts on the wire, kernels/plugins/hp_compression/
  hp_compression.cpp:72-144): packing, the weight gradient of a projection
  straight from the codes, and a gated unit that keeps its inputs that way.

Values are float32, bfloat16 or float16, sums are held in 32 bits, and every
result is rounded once. No function waits for the GPU or keeps anything
between calls: results and workspaces come from torch's allocator, so calls
can run on several streams at once and be captured into graphs (forward and
backward pass; a capture over a parameter whose gradient belongs to the default
stream is refused). A gradient has the same bits in every run.

A persistent engine may be live on the same GPU: its kernels leave these room.
But they never end, and hold two of the four hardware queues that HIP deals a
process's streams out to, so keep to the default stream beside an engine: work
on a side stream may wait until the engine is closed, whoever launches it. What
waits for the whole device (torch.cuda.synchronize, empty_cache) does wait.
"""
import contextlib

import torch
from torch.autograd import forward_ad

from . import _core
from .accl import DataType, _torch_dtype_map

__all__ = [
    "Act8", "act8_linear", "act8_pack", "act8_swiglu", "act8_swiglu_forward",
    "act8_swiglu_grad", "act8_unpack", "act8_weight_grad", "embedding",
    "embedding_grad", "sum_rows",
]

GROUP = 32  # values that share an exponent

_VALUES = (torch.float32, torch.bfloat16, torch.float16)
_CODE = {t: int(d) for d, t in _torch_dtype_map().items()}


# ------------------------------------------------------------------ checks
def _value(name, t, tangent=False):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: a tensor is needed, not {type(t).__name__}")
    if t.layout is not torch.strided:
        raise TypeError(f"{name}: a dense tensor is needed, not {t.layout}")
    if t.dtype not in _VALUES:
        raise TypeError(f"{name}: float32, bfloat16 or float16 are supported, "
                        f"not {t.dtype}")
    # without a tangent a result would read as a derivative of zero
    if not tangent and forward_ad._current_level >= 0 and \
            forward_ad.unpack_dual(t).tangent is not None:
        raise RuntimeError(f"{name}: forward-mode derivatives are not "
                           f"supported")
    return t


def _ids(ids):
    if not isinstance(ids, torch.Tensor):
        raise TypeError(f"ids: a tensor is needed, not {type(ids).__name__}")
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"ids: int64 or int32 are supported, not {ids.dtype}")
    return ids


def _together(first, *others):
    """The device index that all operands share (-1: host memory)."""
    on_gpu, index = first.is_cuda, first.get_device()
    if not on_gpu and not first.is_cpu:
        raise ValueError(f"operands on {first.device} are not supported")
    for t in others:
        if t.get_device() != index or t.is_cuda != on_gpu or \
                t.is_cpu == on_gpu:
            raise ValueError(f"operands on {first.device} and {t.device}")
    return index


def _matrix(t):
    """t as a matrix of its last axis, also where that has no elements."""
    return t.reshape(t.shape[:-1].numel(), t.size(-1))


def _rows(t, width):
    """t as [rows, width] with neighbouring columns, and the distance of its
    rows: a view where its strides allow one, else a copy."""
    if t.dim() == 2 and t.is_contiguous():
        return t, width
    if t.dim() != 2 or (t.stride(1) != 1 and width > 1) or t.stride(0) < width:
        t = _matrix(t)
        if (width > 1 and t.stride(1) != 1) or \
                (t.size(0) > 1 and t.stride(0) < width):
            t = t.contiguous()
    return t, t.stride(0)


def _run(index, op, *operands):
    """op on the current stream of device `index` (host memory: -1)."""
    if index < 0:
        op(-1, *operands)
    elif torch._C._cuda_getDevice() == index:
        op(torch._C._cuda_getCurrentRawStream(index), *operands)
    else:
        with torch.cuda.device(index):
            op(torch._C._cuda_getCurrentRawStream(index), *operands)


def _workspace(n, device):
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def _range(t):
    """First and last byte address of t's elements."""
    at = t.data_ptr()
    return at, at + t.element_size() * (
        1 + sum((n - 1) * d for n, d in zip(t.shape, t.stride()))) - 1


def _side_by_side(a, b):
    """Whether rows of a and b, equally far apart, take different columns of one
    buffer."""
    if a.dim() != 2 or b.dim() != 2:
        return False
    row = a.stride(0) * a.element_size()
    a_width, b_width = (t.size(1) * t.element_size() for t in (a, b))
    if b.stride(0) * b.element_size() != row or max(a_width, b_width) > row or \
            any(t.size(1) > 1 and t.stride(1) != 1 for t in (a, b)):
        return False
    return a_width <= (b.data_ptr() - a.data_ptr()) % row <= row - b_width


def _apart(name, out, *operands):
    """An `out` that shares memory with an operand would be read and written
    at once."""
    if out.numel():
        first, last = _range(out)
        for t in operands:
            if t.numel():
                a, b = _range(t)
                if a <= last and first <= b and not _side_by_side(out, t):
                    raise ValueError(
                        f"{name}: out shares its memory with an operand")


def _capturable(y):
    """Marks the gradient accumulators that y's graph holds with the stream
    they were first met on, and refuses a capture over one of the default
    stream: a backward pass that is captured there ends the process, since the
    default stream cannot take part in a capture. One of another stream can,
    as after the usual steps on a side stream before a capture."""
    if y.is_cuda:
        stream = torch._C._cuda_getCurrentRawStream(y.device.index)
        capturing = torch.cuda.is_current_stream_capturing()
        for node, _ in y.grad_fn.next_functions:
            if node is not None and \
                    node.name() == "torch::autograd::AccumulateGrad":
                made = node.metadata.setdefault("accl_stream", stream)
                if capturing and made == 0:
                    raise RuntimeError(
                        "accl_amd: the gradient of a parameter of this call "
                        "belongs to the default stream, since an eager graph "
                        "of it is alive, or DDP or a hook keeps it so. Drop "
                        "the graph's results before the capture, run eager "
                        "steps (and construct DDP) on a side stream, or "
                        "capture with parameter.detach().requires_grad_()")
    return y


def _out(name, out, shape, index):
    _value("out", out)
    if tuple(out.shape) != tuple(shape):
        raise ValueError(f"{name}: out has shape {tuple(out.shape)}, "
                         f"{tuple(shape)} is needed")
    if _together(out) != index:
        raise ValueError(f"{name}: out is on {out.device}")
    if out.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name}: out requires grad")
    if out.numel() and ((shape[1] > 1 and out.stride(1) != 1) or
                        (shape[0] > 1 and out.stride(0) < shape[1])):
        raise ValueError(f"{name}: the columns of out have to be neighbours, "
                         f"and its rows apart")
    return out


# ------------------------------------------------------------------ embedding
def _lookup(ids, weight, scale, first_row):
    rows, width = weight.shape
    index = _together(weight, ids)
    ids = ids.contiguous()
    table, stride = _rows(weight, width)
    out = weight.new_empty((*ids.shape, width))
    if out.numel():
        dt = _CODE[weight.dtype]
        _run(index, _core.ops_lookup, ids.data_ptr(), _CODE[ids.dtype],
             ids.numel(), first_row, rows, width, scale, table.data_ptr(),
             stride, dt, out.data_ptr(), width, dt)
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, first_row, sparse):
        ctx.save_for_backward(ids)
        ctx.of = (tuple(weight.shape), weight.dtype, scale, first_row, sparse)
        return _lookup(ids, weight, scale, first_row)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        ids, = ctx.saved_tensors
        (rows, width), dtype, scale, first_row, sparse = ctx.of
        if not sparse:
            return (None, embedding_grad(grad, ids, rows, scale, first_row,
                                         dtype=dtype), None, None, None)
        found, sums, count = _sum_rows(
            ids.reshape(-1), _matrix(grad), rows, scale, first_row)
        n = int(count)
        return (None, torch.sparse_coo_tensor(
            found[:n].long()[None], sums[:n].to(dtype), (rows, width),
            is_coalesced=True), None, None, None)


def embedding(ids, weight, scale=1.0, first_row=0, sparse=False):
    """``scale * weight[ids - first_row]``, and zeros for every token whose
    row is not among this weight's.

    ids: int64 or int32, of any shape. weight: [rows, width], the rows
    ``first_row ..`` of the vocabulary: a rank's shard, whose results add up
    to the whole embedding in an all-reduce. A token that no rank holds (-1,
    say) gives zeros and gets no gradient.

    Differentiable in weight; with ``sparse`` its gradient is a coalesced
    sparse tensor of the touched rows, whose number the host waits for (so a
    graph cannot capture that backward pass). DDP expects such gradients from
    parameters of a torch.nn.Embedding with ``sparse=True``, or a subclass.
    """
    _ids(ids)
    _value("weight", weight)
    if weight.dim() != 2:
        raise ValueError(f"weight: [rows, width] is needed, not "
                         f"{tuple(weight.shape)}")
    scale, first_row = float(scale), int(first_row)
    if weight.requires_grad and torch.is_grad_enabled():
        return _capturable(_Embedding.apply(ids, weight, scale, first_row,
                                            bool(sparse)))
    return _lookup(ids, weight, scale, first_row)


def embedding_grad(grad, ids, rows, scale=1.0, first_row=0, out=None,
                   dtype=None):
    """Gradient of :func:`embedding` with respect to its weight: row r of the
    result is ``scale`` times the sum of ``grad`` over the tokens whose
    ``ids - first_row`` is r.

    grad: [*ids.shape, width]. Without `out` the result is a new tensor
    [rows, width] of type `dtype` (grad's if not given). With `out` the sums
    are added to it, and rows that no token names are left as they are; each
    touched row is rounded once to out's type.
    """
    _ids(ids)
    _value("grad", grad)
    rows, scale, first_row = int(rows), float(scale), int(first_row)
    if rows < 0:
        raise ValueError(f"rows: {rows}")
    if grad.dim() != ids.dim() + 1 or grad.shape[:-1] != ids.shape:
        raise ValueError(f"grad of shape {tuple(grad.shape)} for ids of shape "
                         f"{tuple(ids.shape)}")
    width = grad.size(-1)
    index = _together(grad, ids)
    if out is None:
        dtype = grad.dtype if dtype is None else dtype
        if dtype not in _VALUES:
            raise TypeError(f"dtype: {dtype} is not supported")
        total = grad.new_empty((rows, width), dtype=dtype)
    else:
        if dtype is not None and dtype != out.dtype:
            raise TypeError(f"embedding_grad: out is {out.dtype}, not {dtype}")
        total = _out("embedding_grad", out, (rows, width), index)
        _apart("embedding_grad", out, grad, ids)
    if total.numel():
        ids = ids.contiguous()
        values, stride = _rows(grad, width)
        n = ids.numel()
        size = 0 if index < 0 else _core.ops_gradient_workspace(
            n, rows, width, False)
        ws = _workspace(size, grad.device)
        _run(index, _core.ops_gradient, ids.data_ptr(), _CODE[ids.dtype], n,
             first_row, rows, width, scale, values.data_ptr(), stride,
             _CODE[grad.dtype], total.data_ptr(), total.stride(0),
             _CODE[total.dtype], out is not None,
             ws.data_ptr() if size else 0, size)
    return total


def sum_rows(ids, values, rows, scale=1.0):
    """The rows of a sparse gradient, each once: ``(ids, sums, count)``.

    ids: [n], which row each row of values [n, width] belongs to; ids outside
    ``0 .. rows - 1`` are dropped. The first ``count`` entries of the result
    are the distinct ids in ascending order and ``scale`` times the sum of
    their values; behind them, up to n, stand -1 and zeros, so that shapes
    do not depend on the data and a result can be an operand again. count is
    a tensor of one int64.
    """
    _ids(ids)
    _value("values", values)
    rows, scale = int(rows), float(scale)
    if rows < 0:
        raise ValueError(f"rows: {rows}")
    if ids.dim() != 1 or values.dim() != 2 or values.size(0) != ids.size(0):
        raise ValueError(f"ids [n] and values [n, width] are needed, not "
                         f"{tuple(ids.shape)} and {tuple(values.shape)}")
    return _sum_rows(ids, values, rows, scale, 0)


def _sum_rows(ids, values, rows, scale, first_row):
    """sum_rows of ``ids - first_row``, which may have more bits than ids."""
    n, width = values.shape
    index = _together(values, ids)
    ids = ids.contiguous()
    values, stride = _rows(values, width)
    found = torch.empty_like(ids)
    sums = values.new_empty((n, width))
    count = ids.new_empty(1, dtype=torch.int64)
    size = 0 if index < 0 else _core.ops_gradient_workspace(
        n, rows, width, True)
    ws = _workspace(size, ids.device)
    _run(index, _core.ops_sum_rows, ids.data_ptr(), _CODE[ids.dtype], n,
         first_row, rows, width, scale, values.data_ptr(), stride,
         _CODE[values.dtype], sums.data_ptr(), width, _CODE[sums.dtype],
         found.data_ptr(), count.data_ptr(), ws.data_ptr() if size else 0,
         size)
    return found, sums, count


# ------------------------------------------------------------------ 8 bits
class Act8:
    """Activations kept in 8 bits.

    A row consists of `sections` equal parts, each of groups of 32 neighbouring
    values (the last group of a part may be shorter). A group shares 2**e with
    ``e = max(floor(log2(largest magnitude)) - 6, -126)``; a value is held as
    its multiple of 2**e, rounded to the nearest, ties to even, within
    -127..127. A group that holds an infinity or a NaN has e = -128 and codes
    of zero, and stands for NaN.

    codes: int8 [*, width]; exponents: int8 [*, groups]; dtype: of the values
    that were packed. Those of float16 have exponents of at most 9;
    :func:`act8_weight_grad` takes a group beyond that as one that holds none.
    Both tensors are plain data: they can be sliced along rows, moved, or
    gathered over ranks at half the bytes of the values.
    """

    __slots__ = ("codes", "exponents", "dtype", "sections")

    def __init__(self, codes, exponents, dtype, sections=1):
        for name, t in (("codes", codes), ("exponents", exponents)):
            if not isinstance(t, torch.Tensor) or t.dtype != torch.int8 or \
                    t.layout is not torch.strided or t.dim() < 1:
                raise TypeError(f"{name}: a dense int8 tensor of at least one "
                                f"dimension is needed")
        if dtype not in _VALUES:
            raise TypeError(f"dtype: {dtype} is not supported")
        width = codes.size(-1)
        if sections < 1 or width % sections:
            raise ValueError(f"{width} values in {sections} sections")
        groups = sections * -(-(width // sections) // GROUP)
        if exponents.shape != (*codes.shape[:-1], groups):
            raise ValueError(f"exponents of shape {tuple(exponents.shape)} for "
                             f"codes of shape {tuple(codes.shape)}: {groups} "
                             f"groups are needed")
        _together(codes, exponents)
        self.codes, self.exponents = codes, exponents
        self.dtype, self.sections = dtype, sections

    @property
    def shape(self):
        return self.codes.shape

    @property
    def nbytes(self):
        return self.codes.numel() + self.exponents.numel()

    def _flat(self):
        """Addresses and distances of the rows of the codes and exponents, and
        the tensors that hold them."""
        codes, codes_stride = _rows(self.codes, self.codes.shape[-1])
        exps, exps_stride = _rows(self.exponents, self.exponents.shape[-1])
        return (codes.data_ptr(), codes_stride, exps.data_ptr(),
                exps_stride), (codes, exps)


def _new_act8(x, sections):
    """Room for x in 8 bits."""
    *lead, width = x.shape
    kept = object.__new__(Act8)
    kept.codes = torch.empty_like(x, dtype=torch.int8,
                                  memory_format=torch.contiguous_format)
    kept.exponents = x.new_empty(
        (*lead, sections * -(-(width // sections) // GROUP)),
        dtype=torch.int8)
    kept.dtype, kept.sections = x.dtype, sections
    return kept


def act8_pack(x, sections=1):
    """x, of one dimension or more, as :class:`Act8`."""
    _value("x", x)
    if x.dim() < 1:
        raise ValueError("x: at least one dimension is needed")
    sections = int(sections)
    width = x.shape[-1]
    if sections < 1 or width % sections:
        raise ValueError(f"{width} values in {sections} sections")
    index = _together(x)
    kept = _new_act8(x, sections)
    n = x.numel()
    if n:
        rows, stride = _rows(x, width)
        _run(index, _core.ops_act8_pack, rows.data_ptr(), stride,
             _CODE[x.dtype], n // width, width // sections, sections,
             kept.codes.data_ptr(), width, kept.exponents.data_ptr(),
             kept.exponents.shape[-1])
    return kept


def _kept(name, kept):
    if not isinstance(kept, Act8):
        raise TypeError(f"{name}: an Act8 is needed, not "
                        f"{type(kept).__name__}")
    return kept


def act8_unpack(kept, dtype=None):
    """The values that `kept` stands for, in `dtype` (kept.dtype if not
    given): exact in float32 and bfloat16, and in kept.dtype."""
    _kept("kept", kept)
    dtype = kept.dtype if dtype is None else dtype
    if dtype not in _VALUES:
        raise TypeError(f"dtype: {dtype} is not supported")
    x = torch.empty_like(kept.codes, dtype=dtype,
                         memory_format=torch.contiguous_format)
    n = x.numel()
    if n:
        width = x.shape[-1]
        flat, _held = kept._flat()
        _run(_together(x), _core.ops_act8_unpack, x.data_ptr(), width,
             _CODE[dtype], n // width, width // kept.sections, kept.sections,
             *flat)
    return x


def act8_weight_grad(grad, kept, out=None, dtype=None):
    """Weight gradient of ``y = x @ weight.t()`` from y's gradient and the x
    that was kept: ``grad.t() @ x``, [outputs, width].

    grad: [*, outputs] of the type that was kept. Without `out` the result is
    a new tensor of type `dtype` (grad's if not given); with `out` it is added
    to what that holds. Products are exact and summed in 32 bits. On a GPU,
    outputs are fewer than 2**24.
    """
    _value("grad", grad)
    _kept("kept", kept)
    if grad.dtype != kept.dtype:
        raise TypeError(f"grad is {grad.dtype}, {kept.dtype} was kept")
    if kept.sections != 1:
        raise ValueError("act8_weight_grad: one section is needed")
    if grad.dim() < 1 or grad.shape[:-1] != kept.shape[:-1]:
        raise ValueError(f"grad of shape {tuple(grad.shape)} for activations "
                         f"of shape {tuple(kept.shape)}")
    index = _together(grad, kept.codes)
    outputs, width = grad.size(-1), kept.shape[-1]
    if out is None:
        dtype = grad.dtype if dtype is None else dtype
        if dtype not in _VALUES:
            raise TypeError(f"dtype: {dtype} is not supported")
        total = grad.new_empty((outputs, width), dtype=dtype)
    else:
        if dtype is not None and dtype != out.dtype:
            raise TypeError(f"act8_weight_grad: out is {out.dtype}, not "
                            f"{dtype}")
        total = _out("act8_weight_grad", out, (outputs, width), index)
        _apart("act8_weight_grad", out, grad, kept.codes, kept.exponents)
    if total.numel():
        g, stride = _rows(grad, outputs)
        flat, _held = kept._flat()
        of = (g.data_ptr(), stride, _CODE[g.dtype], grad.numel() // outputs,
              outputs, width)
        size = 0 if index < 0 else _core.ops_act8_weight_grad_workspace(*of)
        ws = _workspace(size, grad.device)
        _run(index, _core.ops_act8_weight_grad, *of, *flat, total.data_ptr(),
             total.stride(0), _CODE[total.dtype], out is not None,
             ws.data_ptr() if size else 0, size)
    return total


def act8_swiglu_forward(x):
    """``(y, kept)`` of the gated unit ``y = silu(gate) * up``: x is
    [*, 2 * width], gate its first half and up its second, and kept is x in
    8 bits, in two sections, for :func:`act8_swiglu_grad`."""
    _value("x", x)
    if x.dim() < 1 or x.size(-1) % 2:
        raise ValueError(f"x of shape {tuple(x.shape)}: an even number of "
                         f"columns is needed")
    index = _together(x)
    kept = _new_act8(x, 2)
    width = x.size(-1) // 2
    y = x.new_empty((*x.shape[:-1], width))
    if y.numel():
        rows, stride = _rows(x, 2 * width)
        _run(index, _core.ops_act8_swiglu, rows.data_ptr(), stride,
             _CODE[x.dtype], y.numel() // width, width, kept.codes.data_ptr(),
             2 * width, kept.exponents.data_ptr(), kept.exponents.shape[-1],
             y.data_ptr(), width)
    return y, kept


def act8_swiglu_grad(grad, kept):
    """Gradient of the gated unit with respect to its x, [*, 2 * width], from
    y's gradient [*, width] and what :func:`act8_swiglu_forward` kept."""
    _value("grad", grad)
    _kept("kept", kept)
    if grad.dtype != kept.dtype:
        raise TypeError(f"grad is {grad.dtype}, {kept.dtype} was kept")
    if kept.sections != 2:
        raise ValueError("act8_swiglu_grad: two sections are needed")
    if grad.dim() < 1 or \
            (*grad.shape[:-1], 2 * grad.size(-1)) != tuple(kept.shape):
        raise ValueError(f"grad of shape {tuple(grad.shape)} for activations "
                         f"of shape {tuple(kept.shape)}")
    index = _together(grad, kept.codes)
    d = grad.new_empty(kept.shape)
    if d.numel():
        width = grad.size(-1)
        g, stride = _rows(grad, width)
        flat, _held = kept._flat()
        _run(index, _core.ops_act8_swiglu_grad, d.data_ptr(), 2 * width,
             _CODE[d.dtype], grad.numel() // width, width, *flat,
             g.data_ptr(), stride)
    return d


class _SwiGLU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        y, kept = act8_swiglu_forward(x)
        ctx.save_for_backward(kept.codes, kept.exponents)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        kept = Act8(*ctx.saved_tensors, grad.dtype, 2)
        return act8_swiglu_grad(grad, kept)


def act8_swiglu(x):
    """``silu(gate) * up`` of x's two halves, differentiable; what stays in
    memory for the backward pass is x in 8 bits."""
    _value("x", x)
    if x.requires_grad and torch.is_grad_enabled():
        return _capturable(_SwiGLU.apply(x))
    return act8_swiglu_forward(x)[0]


def _gathered(t, group):
    """The ranks' t, one after the other along the first dimension."""
    import torch.distributed as dist
    t = t.contiguous()
    whole = torch.empty((t.size(0) * dist.get_world_size(group),
                         *t.shape[1:]), dtype=t.dtype, device=t.device)
    dist.all_gather_into_tensor(whole, t, group=group)
    return whole


def _own_types(device):
    """Products of operands whose type is settled, whatever autocast asks."""
    return torch.autocast(device.type, enabled=False) \
        if torch.is_autocast_enabled(device.type) else contextlib.nullcontext()


def _product(x, weight, group):
    whole = x if group is None else _gathered(x, group)
    y = _matrix(whole) @ weight.t()
    return y.view(*whole.shape[:-1], weight.size(0))


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, group):
        # only a trained weight needs x again
        if ctx.needs_input_grad[1]:
            kept = act8_pack(x)
            ctx.save_for_backward(weight, kept.codes, kept.exponents)
        else:
            ctx.save_for_backward(weight)
        ctx.of = (x.dtype, group)
        return _product(x, weight, group)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        weight, *kept = ctx.saved_tensors
        dtype, group = ctx.of
        d_x = d_weight = None
        if ctx.needs_input_grad[0]:
            with _own_types(grad.device):
                d_x = (_matrix(grad) @ weight).view(
                    *grad.shape[:-1], weight.size(1))
            if group is not None:
                import torch.distributed as dist
                whole = d_x
                n = dist.get_world_size(group)
                d_x = torch.empty((whole.size(0) // n, *whole.shape[1:]),
                                  dtype=whole.dtype, device=whole.device)
                dist.reduce_scatter_tensor(d_x, whole, group=group)
        if ctx.needs_input_grad[1]:
            if group is not None:
                kept = [_gathered(t, group) for t in kept]
            d_weight = act8_weight_grad(grad, Act8(*kept, dtype))
        return d_x, d_weight, None


def act8_linear(x, weight, group=None):
    """``x @ weight.t()``, differentiable, with x kept in 8 bits for weight's
    gradient. x: [*, width], weight: [outputs, width], of one type; under
    autocast both are cast to its type first, as for a product of torch's.

    With a process group, x is this rank's part of a sequence (the same shape
    on every rank, at least two dimensions, split along the first): it is
    gathered before the product, x's gradient is reduced and scattered, and
    what the backward pass gathers again are the 8-bit codes.
    """
    _value("x", x, tangent=True)
    _value("weight", weight, tangent=True)
    if torch.is_autocast_enabled(x.device.type):
        dtype = torch.get_autocast_dtype(x.device.type)
        x, weight = x.to(dtype), weight.to(dtype)
    if weight.dtype != x.dtype:
        raise TypeError(f"x is {x.dtype}, weight {weight.dtype}")
    if weight.dim() != 2 or x.dim() < 1 or x.size(-1) != weight.size(1):
        raise ValueError(f"x of shape {tuple(x.shape)} for a weight of shape "
                         f"{tuple(weight.shape)}")
    if group is not None and x.dim() < 2:
        raise ValueError("act8_linear: with a group, x needs two dimensions")
    _together(x, weight)
    with _own_types(x.device):
        if torch.is_grad_enabled() and (x.requires_grad or
                                        weight.requires_grad):
            return _capturable(_Linear.apply(x, weight, group))
        return _product(x, weight, group)
