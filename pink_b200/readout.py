"""Read-out of a map on torch tensors: routes of images to neurons, read-out of routed neurons, dense product, and their gradients.

The functions marshal arguments for the pink_b200_op_* entries of the C ABI (include/pink_b200.h defines every result) and
allocate what they return.  They run on the tensors' device and on its current torch stream, do not synchronise, and can be
captured into a CUDA graph.  Matrices may have any row pitch; their rows must be contiguous.  Like the rest of the library
they have no CPU form.  Gradients are explicit functions: nothing here takes part in autograd, and a call whose arguments
require a gradient warns that its result has no graph.

A read-out of the routed neurons, and its gradients:

    neurons, weights = route(distances, 4, slope=-1.0)
    y = read_out(values, neurons, weights)
    dvalues, dweights = read_out_backward(dy, values, neurons, weights)
    ddistances = route_backward(distances, neurons, weights, dweights, slope=-1.0)
"""
import ctypes as C
import warnings

import torch

from . import capi

_TYPES = {torch.float32: capi.F32, torch.bfloat16: capi.BF16, torch.float16: capi.F16}
_SCORES = {"softmax": capi.SCORE_SOFTMAX, "sigmoid": capi.SCORE_SIGMOID}
_ACTIVATIONS = {"none": capi.ACT_NONE, "relu": capi.ACT_RELU, "gelu": capi.ACT_GELU, "silu": capi.ACT_SILU, "sigmoid": capi.ACT_SIGMOID}


def _refuse(t, name, shape, dtypes, index):
    """Says what is wrong with an argument that is not a tensor of this shape, one of these types and this device."""
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a torch tensor" % name)
    if t.get_device() != index:
        raise ValueError("%s is on %s, expected cuda:%d" % (name, t.device, index))
    if t.dtype not in dtypes:
        raise TypeError("%s has type %s, expected %s" % (name, t.dtype, " or ".join(str(d) for d in dtypes)))
    raise ValueError("%s has shape %s, expected %s" % (name, tuple(t.shape), tuple(shape)))


def _matrix(t, name, shape, dtypes, index):
    """Pointer and leading dimension of a matrix whose rows are contiguous."""
    if not isinstance(t, torch.Tensor) or t.shape != shape or t.dtype not in dtypes or t.get_device() != index:
        _refuse(t, name, shape, dtypes, index)
    rows, cols = shape
    ld, step = t.stride()
    if step != 1 and cols > 1:
        raise ValueError("the rows of %s must be contiguous" % name)
    if rows <= 1:
        ld = cols
    elif ld < cols:
        raise ValueError("the rows of %s overlap" % name)
    return t.data_ptr(), ld


def _table(t, name, shape, dtypes, index):
    """Pointer of a tensor without gaps."""
    if not isinstance(t, torch.Tensor) or t.shape != shape or t.dtype not in dtypes or t.get_device() != index:
        _refuse(t, name, shape, dtypes, index)
    if not t.is_contiguous():
        raise ValueError("%s must be contiguous" % name)
    return t.data_ptr()


def _apart(out, name, p, ld, *others):
    """Refuses a result that shares elements with an argument, of which it would be both read and written in an order that nothing sets.
    Side by side in the rows of one matrix they share none.  An argument of the same place and pitch that is marked so may become the result."""
    rows, cols = out.shape
    size = out.element_size()
    end = p + ((rows - 1) * ld + cols) * size
    for t, what, may_be in others:
        if t is None or rows == 0 or t.numel() == 0:
            continue
        q, (r, c) = t.data_ptr(), t.shape
        step = t.stride(0) if r > 1 else c
        if end <= q or q + ((r - 1) * step + c) * size <= p or (may_be and p == q and (rows <= 1 or step == ld)):
            continue
        pitch = step if rows <= 1 else ld                  # (a single row goes with any pitch)
        if (r <= 1 or step == pitch) and (q - p) % size == 0:
            at = (q - p) // size % pitch                   # the argument's first column, counted from the result's
            if cols <= at and at + c <= pitch:
                continue
        raise ValueError("%s overlaps %s" % (name, what))


def _two_d(t, name):
    """Device index and shape of the matrix that sets them for a call."""
    if not isinstance(t, torch.Tensor) or t.dim() != 2:
        raise TypeError("%s must be a matrix" % name)
    index = t.get_device()
    if index < 0:
        raise ValueError("%s must be on a GPU: there is no CPU form" % name)
    return index, t.shape


def _new(t, shape, dtype):
    """A new contiguous matrix on t's device (empty_strided: 1.5 us where empty takes 2.4)."""
    return torch.empty_strided(shape, (shape[1], 1), dtype=dtype, device=t.device)


def _new_vector(t, size, dtype):
    return torch.empty_strided((size,), (1,), dtype=dtype, device=t.device)


def _unrecorded(*tensors):
    """Says that a result has no graph where torch's own operators would have given it one."""
    for t in tensors:
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            warnings.warn("the read-out operators take no part in autograd: this result has no graph, although an argument requires a gradient "
                          "(call the *_backward functions, and these under torch.no_grad())", stacklevel=3)
            return


def _of(table, key, what):
    if key not in table:
        raise ValueError("unknown %s %r; known: %s" % (what, key, ", ".join(table)))
    return table[key]


def _call(index, entry, *args):
    """Runs a C entry on device `index` and its current stream."""
    if index == torch.cuda.current_device():
        rc = entry(*args, _current_stream(index))
    else:
        with torch.cuda.device(index):
            rc = entry(*args, _current_stream(index))
    if rc:
        capi.check(rc)


def _current_stream(index):
    return torch.cuda.current_stream(index).cuda_stream


if hasattr(torch._C, "_cuda_getCurrentRawStream"):
    _current_stream = torch._C._cuda_getCurrentRawStream       # the same handle without a Stream object: 0.1 instead of 2.2 us


_ANY = tuple(_TYPES)
_FLOAT = (torch.float32,)
_INT = (torch.int32,)
_BYTE = (torch.bool, torch.uint8)


def route(values, top_k, *, score="softmax", slope=1.0, scale=1.0, renormalise=True, bias=None, mask=None, groups=1, top_groups=None,
          group_best=1, load=None, scores=None):
    """The top_k neurons of every row of `values` ([n, N] distances or learned scores) and their weights.

    logit = slope * value (negative slope for distances); score: "softmax" over the neurons, or "sigmoid" of each.  bias ([N]
    float32) is added to the logit, not to the score, and shifts the choice only; mask ([N] bool) leaves neurons out; NaN and -infinity leave single entries out.  groups > 1:
    neurons come from the top_groups groups of N / groups consecutive neurons with the best member (group_best=1) or pair (2).
    renormalise: the weights of a row add up to `scale`.  load ([N] int32): counters that the choices are added to.
    Returns (neurons [n, top_k] int32, -1 where there is none; weights [n, top_k] float32) and, with scores=dtype, the scores
    of all neurons [n, N] in rows padded for product()."""
    index, shape = _two_d(values, "values")
    n, N = shape
    p, ld = _matrix(values, "values", shape, _ANY, index)
    cfg = capi.RouteConfig(N, top_k, _of(_SCORES, score, "score"), 1 if renormalise else 0, groups, groups if top_groups is None else top_groups,
                           group_best, slope, scale)
    pb = None if bias is None else _table(bias, "bias", (N,), _FLOAT, index)
    pm = None if mask is None else _table(mask, "mask", (N,), _BYTE, index)
    pl = None if load is None else _table(load, "load", (N,), _INT, index)
    _unrecorded(values)
    neurons, weights = _new(values, (n, top_k), torch.int32), _new(values, (n, top_k), torch.float32)
    dense, ps, st, ls = None, None, 0, 0
    if scores is not None:
        st, ls = _of(_TYPES, scores, "type of the scores"), (N + 63) // 64 * 64
        dense = _new(values, (n, ls), scores)[:, :N]         # rows that product() reads in place and at full speed
        ps = dense.data_ptr()
    _call(index, capi.lib.pink_b200_op_route, cfg, n, _TYPES[values.dtype], p, ld, pb, pm, neurons.data_ptr(), weights.data_ptr(), pl, st, ps, ls)
    return (neurons, weights) if dense is None else (neurons, weights, dense)


def route_backward(values, neurons, weights, dweights, *, score="softmax", slope=1.0, scale=1.0, renormalise=True, mask=None, dscores=None):
    """Gradient of route() with respect to its values, from those of its weights and (dscores, [n, N]) of its dense scores."""
    index, shape = _two_d(values, "values")
    n, N = shape
    p, ld = _matrix(values, "values", shape, _ANY, index)
    k = _two_d(neurons, "neurons")[1][1]
    pn, pw = _table(neurons, "neurons", (n, k), _INT, index), _table(weights, "weights", (n, k), _FLOAT, index)
    pd = _table(dweights, "dweights", (n, k), _FLOAT, index)
    cfg = capi.RouteConfig(N, k, _of(_SCORES, score, "score"), 1 if renormalise else 0, 1, 1, 1, slope, scale)
    pm = None if mask is None else _table(mask, "mask", (N,), _BYTE, index)
    ps, ls = (None, 0) if dscores is None else _matrix(dscores, "dscores", shape, (values.dtype,), index)
    out = _new(values, shape, values.dtype)
    _call(index, capi.lib.pink_b200_op_route_backward, cfg, n, _TYPES[values.dtype], p, ld, pm, pn, pw, pd, ps, ls, out.data_ptr(), N)
    return out


def balance(load, bias, rate, *, mask=None, out=None):
    """bias + rate * sign(mean load - load): one step of the choice bias towards even loads.  out may be bias itself."""
    if not isinstance(load, torch.Tensor) or load.dim() != 1 or load.get_device() < 0:
        raise TypeError("load must be a vector on a GPU")
    index, N = load.get_device(), load.shape[0]
    if out is None:
        out = _new_vector(load, N, torch.float32)
    pm = None if mask is None else _table(mask, "mask", (N,), _BYTE, index)
    _call(index, capi.lib.pink_b200_op_route_balance, N, _table(load, "load", (N,), _INT, index), pm, rate, _table(bias, "bias", (N,), _FLOAT, index),
          _table(out, "out", (N,), _FLOAT, index))
    return out


def _routes(neurons, weights, index):
    n, k = shape = _two_d(neurons, "neurons")[1]
    return n, k, _table(neurons, "neurons", shape, _INT, index), _table(weights, "weights", shape, _FLOAT, index)


def read_out(values, neurons, weights, *, residual=None, out=None):
    """sum over the routes of weight * values[neuron] (+ residual): values [N, D], neurons / weights [n, k] as route() gives them.

    out may be the residual; otherwise it shares no element with the arguments."""
    index, shape = _two_d(values, "values")
    N, D = shape
    p, ld = _matrix(values, "values", shape, _ANY, index)
    n, k, pn, pw = _routes(neurons, weights, index)
    own = (values.dtype,)
    pr, lr = (None, 0) if residual is None else _matrix(residual, "residual", (n, D), own, index)
    _unrecorded(values, weights, residual)
    if out is None:
        out = _new(values, (n, D), values.dtype)
        po, lo = out.data_ptr(), D
    else:
        po, lo = _matrix(out, "out", (n, D), own, index)
        _apart(out, "out", po, lo, (values, "values", False), (residual, "residual", True))
    _call(index, capi.lib.pink_b200_op_read_out, _TYPES[values.dtype], N, D, p, ld, n, k, pn, pw, pr, lr, po, lo)
    return out


def read_out_backward(dy, values, neurons, weights):
    """Gradients (dvalues [N, D], dweights [n, k]) of read_out() from that of its result."""
    index, shape = _two_d(values, "values")
    N, D = shape
    p, ld = _matrix(values, "values", shape, _ANY, index)
    n, k, pn, pw = _routes(neurons, weights, index)
    pd, ldd = _matrix(dy, "dy", (n, D), (values.dtype,), index)
    dvalues, dweights = _new(values, shape, values.dtype), _new(values, (n, k), torch.float32)
    size = capi.lib.pink_b200_read_out_workspace(N, D, n, k)
    work = _new_vector(values, size, torch.uint8)
    _call(index, capi.lib.pink_b200_op_read_out_backward, _TYPES[values.dtype], N, D, p, ld, n, k, pn, pw, pd, ldd, dvalues.data_ptr(), D,
          dweights.data_ptr(), work.data_ptr(), size)
    return dvalues, dweights


_HALF = (torch.bfloat16, torch.float16)
_FEW_ROWS = 8          # up to as many rows the product needs no workspace


def _sized_call(x, index, ask, entry, *args):
    """A product entry: asks for its workspace (where it may need one), allocates it, runs it."""
    if not ask:
        return _call(index, entry, *args, None, None, 0)
    size = C.c_uint64(0)
    _call(index, entry, *args, None, size, 1)                # (on the same device: the plan depends on its number of SMs)
    work = _new_vector(x, size.value, torch.uint8) if size.value else None
    _call(index, entry, *args, None if work is None else work.data_ptr(), size, 0)


def _product_shapes(x, w, by_input, activation):
    index, shape = _two_d(x, "x")
    _, wshape = _two_d(w, "w")
    n, K = shape
    M = wshape[1] if by_input else wshape[0]
    px, ldx = _matrix(x, "x", shape, _HALF, index)
    pw, ldw = _matrix(w, "w", (K, M) if by_input else (M, K), (x.dtype,), index)
    cfg = capi.ProductConfig(_TYPES[x.dtype], K, M, 1 if by_input else 0, _of(_ACTIVATIONS, activation, "activation"), 0, n)
    return index, n, K, M, px, ldx, pw, ldw, cfg


def product(x, w, *, by_input=False, bias=None, activation="none", residual=None, keep=False, out=None):
    """act(x w^T + bias) + residual on the tensor cores: x [n, K] and w [M, K] (by_input: [K, M]) bfloat16 or float16, bias [M] float32.

    keep=True also returns z = x w^T + bias, which product_backward() needs where there is an activation.  out may be the residual;
    otherwise it shares no element with the arguments."""
    index, n, K, M, px, ldx, pw, ldw, cfg = _product_shapes(x, w, by_input, activation)
    own = (x.dtype,)
    pb = None if bias is None else _table(bias, "bias", (M,), _FLOAT, index)
    pr, lr = (None, 0) if residual is None else _matrix(residual, "residual", (n, M), own, index)
    _unrecorded(x, w, bias, residual)
    if out is None:
        out = _new(x, (n, M), x.dtype)
        po, lo = out.data_ptr(), M
    else:
        po, lo = _matrix(out, "out", (n, M), own, index)
        _apart(out, "out", po, lo, (x, "x", False), (w, "w", False), (residual, "residual", True))
    z = _new(x, (n, M), x.dtype) if keep else None
    _sized_call(x, index, n > _FEW_ROWS, capi.lib.pink_b200_op_product, cfg, px, ldx, pw, ldw, pb, pr, lr, po, lo, z.data_ptr() if keep else None, M)
    return (out, z) if keep else out


def product_backward(dy, x, w, *, by_input=False, z=None, activation="none"):
    """Gradients (dx, dw, dbias) of product() from that of its result; the residual's is dy itself."""
    index, n, K, M, px, ldx, pw, ldw, cfg = _product_shapes(x, w, by_input, activation)
    own = (x.dtype,)
    pd, ldd = _matrix(dy, "dy", (n, M), own, index)
    if activation != "none" and z is None:
        raise ValueError("the gradient of an activation needs z: product(..., keep=True)")
    pz, lz = (None, 0) if activation == "none" else _matrix(z, "z", (n, M), own, index)
    dx, dw = _new(x, (n, K), x.dtype), _new(x, w.shape, x.dtype)
    dbias = _new_vector(x, M, torch.float32)
    _sized_call(x, index, True, capi.lib.pink_b200_op_product_backward, cfg, pd, ldd, px, ldx, pw, ldw, pz, lz, dx.data_ptr(), K, dw.data_ptr(), w.shape[1],
                dbias.data_ptr())
    return dx, dw, dbias


def check_status():
    """Waits for the current device and raises if a bounded device-side wait of a product expired."""
    capi.check(capi.lib.pink_b200_op_status())
