"""Operators on rows of features: a table looked up by id (a latent per keyframe, a vector per token) with the table's gradient, and
layer norm over a row with its backward pass -- host side of `csrc/embedding.hip` and `csrc/layer_norm.hip`.

A row is the last axis of a tensor (f16, bf16 or f32): channels-last activations as `nerfslam.conv` keeps them are rows of C channels.
Inputs may be slices of wider tensors or expanded along the leading axes, as long as the last axis is dense and the leading ones
collapse to one stride; outputs are fresh dense tensors.  Sums are f32, every output is rounded once.  The backward functions are
explicit, as the trainer's are: nothing here records on torch's autograd tape.  Launches go to torch's current stream of the tensors'
device, nothing synchronises, and every call has its own workspace, so calls may be captured into HIP graphs and run on several streams.
"""
import functools

import torch

from ._lib import NerfSlamHipError, check, lib, require_cuda

_DT = {torch.float16: 1, torch.float32: 2, torch.bfloat16: 3}


def _fail(op, what):
    raise NerfSlamHipError(f"{op}: {what}")


def _same_device(op, first, *others):
    device = first.device
    for t in others:
        if t is not None and t.device != device:
            require_cuda(first, *others)
            _fail(op, "all tensors have to be on one device")
    require_cuda(first)
    return device


def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(name, what, device, *args):
    """the entry point `name` on the current stream of `device`"""
    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            return _call(name, what, device, *args)
    # (the stream's handle without building torch's Stream object: 0.1 us instead of 3.4, of calls that take 3 us on the device)
    check(getattr(lib(), name)(*args, torch._C._cuda_getCurrentRawStream(device.index)), what)


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(name, n, *args):
    """what a size query of the library answers: a function of sizes alone"""
    return getattr(lib(), name)(n, *args)


def _rows_of(op, name, t):
    """(number of rows, distance of two rows in elements) of a tensor whose last axis is the row"""
    if t.dtype not in _DT:
        _fail(op, f"{name} is {t.dtype}: float16, bfloat16 or float32 are supported")
    if t.dim() < 1:
        _fail(op, f"{name} needs at least one axis")
    cols = t.shape[-1]
    if cols > 65536:
        _fail(op, f"{name} has rows of {cols} elements: at most 65536 are supported")
    if cols and t.is_contiguous():
        return t.numel() // cols, cols
    n = 1
    for s in t.shape[:-1]:
        n *= s
    if n * cols == 0:
        return n, cols
    if cols > 1 and t.stride(-1) != 1:
        _fail(op, f"the last axis of {name} must be contiguous")
    stride, inner = None, 1                 # collapse the leading axes, innermost first; axes of size 1 have no stride to mind
    for size, st in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size == 1:
            continue
        if stride is None:
            stride = st
        elif st != stride * inner:
            _fail(op, f"the rows of {name} are not a constant stride apart: pass {name}.contiguous()")
        inner *= size
    return n, cols if stride is None else stride


def _ids(op, ids):
    if ids.dtype not in (torch.int32, torch.int64):
        _fail(op, f"ids are {ids.dtype}: int32 or int64 are supported")
    if not ids.is_contiguous():
        _fail(op, "ids must be contiguous")
    return int(ids.dtype == torch.int64)


def embedding(table, ids, scale=1.0):
    """table [rows, D], ids (any shape, int32 / int64) -> ids.shape + (D,) in the table's dtype: scale * table[ids].  An id outside
    [0, rows), e.g. -1 for a padded place, gives a row of zeros."""
    if table.dim() != 2:
        _fail("embedding", "the table is a [rows, D] tensor")
    rows, stride = _rows_of("embedding", "table", table)
    is64 = _ids("embedding", ids)
    device = _same_device("embedding", table, ids)
    cols = table.shape[1]
    out = table.new_empty((*ids.shape, cols))
    if out.numel():
        _call("ns_embedding_forward", "embedding_forward", device, _ptr(table), stride, _ptr(ids), is64, _ptr(out),
              _DT[table.dtype], ids.numel(), rows, cols, float(scale))
    return out


def embedding_backward(dout, ids, rows, scale=1.0, dtype=None):
    """gradient of `embedding` for its table: dout ids.shape + (D,) -> [rows, D] of `dtype` (None: float32; or dout's own),
    grad[r] = scale * sum of dout over the places with id r; zero where there is none.  Places whose id is outside [0, rows) are left
    out.  The order of the sums follows from the ids alone: the same inputs give the same bits."""
    op = "embedding_backward"
    dtype = torch.float32 if dtype is None else dtype
    if dout.dim() != ids.dim() + 1 or tuple(dout.shape[:-1]) != tuple(ids.shape):
        _fail(op, f"dout {tuple(dout.shape)} does not match ids {tuple(ids.shape)} + (D,)")
    n, stride = _rows_of(op, "dout", dout)
    if dtype not in (torch.float32, dout.dtype):
        _fail(op, f"a gradient in {dtype} of a {dout.dtype} dout: float32 or dout's own dtype are supported")
    is64 = _ids(op, ids)
    rows, cols = int(rows), dout.shape[-1]
    if rows < 0:
        _fail(op, f"{rows} rows")
    device = _same_device(op, dout, ids)
    grad = torch.empty((rows, cols), dtype=dtype, device=device)
    if grad.numel():
        nbytes = _workspace_bytes("ns_embedding_backward_workspace_bytes", n, rows, cols, _DT[dout.dtype])
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
        _call("ns_embedding_backward", op, device, _ptr(dout), stride, _DT[dout.dtype], _ptr(ids), is64, _ptr(grad), _DT[dtype],
              n, rows, cols, float(scale), _ptr(ws), nbytes)
    return grad


def _weight(op, x, name, t):
    if t.dtype != x.dtype and t.dtype != torch.float32:
        _fail(op, f"{name} is {t.dtype}: {x.dtype} (as x) or float32 are supported")
    if t.dim() != 1 or t.shape[0] != x.shape[-1] or not t.is_contiguous():
        _fail(op, f"{name} must be a contiguous [{x.shape[-1]}] tensor")
    return t.dtype


def _weights(op, x, weight, bias):
    """the dtype of weight and bias, each may be None"""
    wdtype = torch.float32
    if weight is not None:
        wdtype = _weight(op, x, "weight", weight)
    if bias is not None:
        bdtype = _weight(op, x, "bias", bias)
        if weight is not None and bdtype != wdtype:
            _fail(op, "weight and bias have to be of one dtype")
        wdtype = bdtype
    return wdtype


def layer_norm(x, weight=None, bias=None, eps=1e-5, stats=False):
    """(x - mean) * rstd * weight + bias over the last axis (at most 16384 wide), rstd = 1 / sqrt(var + eps) with the biased variance;
    weight / bias [D] in x's dtype or float32, each may be None; eps positive.  Sums of squares are f32: rows of values beyond about 1e17 overflow
    them.  stats=True: (y, mean, rstd), the latter two float32 of x.shape[:-1] -- what `layer_norm_backward` takes."""
    op = "layer_norm"
    n, stride = _rows_of(op, "x", x)
    wdtype = _weights(op, x, weight, bias)
    device = _same_device(op, x, weight, bias)
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    mean = rstd = None
    if stats:
        mean = torch.empty(x.shape[:-1], dtype=torch.float32, device=device)
        rstd = torch.empty_like(mean)
    _call("ns_layer_norm_forward", "layer_norm_forward", device, _ptr(x), stride, _ptr(weight), _ptr(bias), _DT[wdtype], _ptr(y),
          _ptr(mean), _ptr(rstd), _DT[x.dtype], n, x.shape[-1], float(eps))
    return (y, mean, rstd) if stats else y


def layer_norm_backward(dout, x, mean, rstd, weight=None, bias=None):
    """gradients of `layer_norm` from the upstream gradient dout (x's shape and dtype) and what the forward pass saved:
    (dx, dweight, dbias) -- dx in x's dtype, the other two in the weight's or the bias'.  A weight alone gives both (dbias takes no further
    pass); a bias alone, of which only dtype and shape count, (dx, None, dbias); neither (dx, None, None)."""
    op = "layer_norm_backward"
    n, stride = _rows_of(op, "x", x)
    if dout.dtype != x.dtype or dout.shape != x.shape:
        _fail(op, f"dout {tuple(dout.shape)} {dout.dtype} does not match x {tuple(x.shape)} {x.dtype}")
    _, dstride = _rows_of(op, "dout", dout)
    for name, t in (("mean", mean), ("rstd", rstd)):
        if t.dtype != torch.float32 or t.shape != x.shape[:-1] or not t.is_contiguous():
            _fail(op, f"{name} must be a contiguous float32 {tuple(x.shape[:-1])} tensor")
    wdtype = _weights(op, x, weight, bias)
    device = _same_device(op, x, dout, mean, rstd, weight, bias)
    cols = x.shape[-1]
    dx = torch.empty_like(x, memory_format=torch.contiguous_format)
    dw = db = ws = None
    nbytes = 0
    if weight is not None or bias is not None:
        db = torch.empty_like(bias if weight is None else weight)
        dw = None if weight is None else torch.empty_like(weight)
        nbytes = _workspace_bytes("ns_layer_norm_backward_workspace_bytes", n, cols, _DT[x.dtype])
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    _call("ns_layer_norm_backward", op, device, _ptr(dout), dstride, _ptr(x), stride, _ptr(mean), _ptr(rstd), _ptr(weight),
          _DT[wdtype], _ptr(dx), _ptr(dw), _ptr(db), _DT[x.dtype], n, cols, _ptr(ws), nbytes)
    return dx, dw, db
