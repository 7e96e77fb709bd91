"""Read-out of a map on torch tensors: routes of images to neurons, read-out of routed neurons, dense product, and their gradients.

The functions marshal arguments for the pink_b200_op_* entries of the C ABI (include/pink_b200.h defines every result) and
allocate what they return.  They run on the tensors' device and on its current torch stream, do not synchronise, and can be
captured into a CUDA graph.  Matrices may have any row pitch; their rows must be contiguous.  Like the rest of the library
they have no CPU form.  Gradients are explicit functions: nothing here takes part in autograd.

A read-out of the routed neurons, and its gradients:

    neurons, weights = route(distances, 4, slope=-1.0)
    y = read_out(values, neurons, weights)
    dvalues, dweights = read_out_backward(dy, values, neurons, weights)
    ddistances = route_backward(distances, neurons, weights, dweights, slope=-1.0)
"""
import ctypes as C

import torch

from . import capi

_TYPES = {torch.float32: capi.F32, torch.bfloat16: capi.BF16, torch.float16: capi.F16}
_SCORES = {"softmax": capi.SCORE_SOFTMAX, "sigmoid": capi.SCORE_SIGMOID}
_ACTIVATIONS = {"none": capi.ACT_NONE, "relu": capi.ACT_RELU, "gelu": capi.ACT_GELU, "silu": capi.ACT_SILU, "sigmoid": capi.ACT_SIGMOID}


def _check(t, name, shape, dtypes, device):
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a torch tensor" % name)
    if t.device != device:
        raise ValueError("%s is on %s, expected %s" % (name, t.device, device))
    if t.dtype not in dtypes:
        raise TypeError("%s has type %s, expected %s" % (name, t.dtype, " or ".join(str(d) for d in dtypes)))
    if tuple(t.shape) != shape:
        raise ValueError("%s has shape %s, expected %s" % (name, tuple(t.shape), shape))


def _matrix(t, name, shape, dtypes, device):
    """Pointer and leading dimension of a matrix whose rows are contiguous."""
    _check(t, name, shape, dtypes, device)
    rows, cols = t.shape
    if cols > 1 and t.stride(1) != 1:
        raise ValueError("the rows of %s must be contiguous" % name)
    ld = t.stride(0) if rows > 1 else cols
    if ld < cols:
        raise ValueError("the rows of %s overlap" % name)
    return t.data_ptr(), ld


def _vector(t, name, size, dtypes, device):
    if t is None:
        return None
    _check(t, name, (size,), dtypes, device)
    if not t.is_contiguous():
        raise ValueError("%s must be contiguous" % name)
    return t.data_ptr()


def _table(t, name, shape, dtypes, device):
    _check(t, name, shape, dtypes, device)
    if not t.is_contiguous():
        raise ValueError("%s must be contiguous" % name)
    return t.data_ptr()


def _two_d(t, name):
    if not isinstance(t, torch.Tensor) or t.dim() != 2:
        raise TypeError("%s must be a matrix" % name)
    if t.device.type != "cuda":
        raise ValueError("%s must be on a GPU: there is no CPU form" % name)
    return t.device


def _of(table, key, what):
    if key not in table:
        raise ValueError("unknown %s %r; known: %s" % (what, key, ", ".join(table)))
    return table[key]


def _call(device, entry, *args):
    """Runs a C entry on `device` and its current stream."""
    index = device.index
    stream = _current_stream(index)
    if index == torch.cuda.current_device():
        rc = entry(*args, stream)
    else:
        with torch.cuda.device(index):
            rc = entry(*args, stream)
    if rc:
        capi.check(rc)


def _padded(n, cols, dtype, device):
    """An n x cols matrix in rows of a multiple of 64 elements, which the dense product reads in place and at full speed."""
    return torch.empty((n, (cols + 63) // 64 * 64), dtype=dtype, device=device)[:, :cols]


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
    float32) shifts the choice only; mask ([N] bool) leaves neurons out; NaN and -infinity leave single entries out.  groups > 1:
    neurons come from the top_groups groups of N / groups consecutive neurons with the best member (group_best=1) or pair (2).
    renormalise: the weights of a row add up to `scale`.  load ([N] int32): counters that the choices are added to.
    Returns (neurons [n, top_k] int32, -1 where there is none; weights [n, top_k] float32) and, with scores=dtype, the scores
    of all neurons [n, N] in rows padded for product()."""
    device = _two_d(values, "values")
    n, N = values.shape
    p, ld = _matrix(values, "values", (n, N), _ANY, device)
    cfg = capi.RouteConfig(N, top_k, _of(_SCORES, score, "score"), int(bool(renormalise)), groups,
                           groups if top_groups is None else top_groups, group_best, slope, scale)
    pb, pm, pl = _vector(bias, "bias", N, _FLOAT, device), _vector(mask, "mask", N, _BYTE, device), _vector(load, "load", N, _INT, device)
    neurons = torch.empty((n, top_k), dtype=torch.int32, device=device)
    weights = torch.empty((n, top_k), dtype=torch.float32, device=device)
    dense, ps, st, ls = None, None, 0, 0
    if scores is not None:
        st = _of(_TYPES, scores, "type of the scores")
        dense = _padded(n, N, scores, device)
        ps, ls = dense.data_ptr(), (N + 63) // 64 * 64
    _call(device, capi.lib.pink_b200_op_route, C.byref(cfg), n, _TYPES[values.dtype], p, ld, pb, pm, neurons.data_ptr(), weights.data_ptr(), pl,
          st, ps, ls)
    return (neurons, weights) if dense is None else (neurons, weights, dense)


def route_backward(values, neurons, weights, dweights, *, score="softmax", slope=1.0, scale=1.0, renormalise=True, mask=None, dscores=None):
    """Gradient of route() with respect to its values, from those of its weights and (dscores, [n, N]) of its dense scores."""
    device = _two_d(values, "values")
    n, N = values.shape
    p, ld = _matrix(values, "values", (n, N), _ANY, device)
    _two_d(neurons, "neurons")
    k = neurons.shape[1]
    pn, pw = _table(neurons, "neurons", (n, k), _INT, device), _table(weights, "weights", (n, k), _FLOAT, device)
    pd = _table(dweights, "dweights", (n, k), _FLOAT, device)
    cfg = capi.RouteConfig(N, k, _of(_SCORES, score, "score"), int(bool(renormalise)), 1, 1, 1, slope, scale)
    ps, ls = (None, 0) if dscores is None else _matrix(dscores, "dscores", (n, N), (values.dtype,), device)
    out = torch.empty((n, N), dtype=values.dtype, device=device)
    _call(device, capi.lib.pink_b200_op_route_backward, C.byref(cfg), n, _TYPES[values.dtype], p, ld,
          _vector(mask, "mask", N, _BYTE, device), pn, pw, pd, ps, ls, out.data_ptr(), N)
    return out


def balance(load, bias, rate, *, mask=None, out=None):
    """bias + rate * sign(mean load - load): one step of the choice bias towards even loads.  out may be bias itself."""
    if not isinstance(load, torch.Tensor) or load.device.type != "cuda" or load.dim() != 1:
        raise TypeError("load must be a vector on a GPU")
    device, N = load.device, load.shape[0]
    if out is None:
        out = torch.empty(N, dtype=torch.float32, device=device)
    _call(device, capi.lib.pink_b200_op_route_balance, N, _vector(load, "load", N, _INT, device), _vector(mask, "mask", N, _BYTE, device), rate,
          _vector(bias, "bias", N, _FLOAT, device), _vector(out, "out", N, _FLOAT, device))
    return out


def read_out(values, neurons, weights, *, residual=None, out=None):
    """sum over the routes of weight * values[neuron] (+ residual): values [N, D], neurons / weights [n, k] as route() gives them."""
    device = _two_d(values, "values")
    N, D = values.shape
    p, ld = _matrix(values, "values", (N, D), _ANY, device)
    _two_d(neurons, "neurons")
    n, k = neurons.shape
    pn, pw = _table(neurons, "neurons", (n, k), _INT, device), _table(weights, "weights", (n, k), _FLOAT, device)
    pr, lr = (None, 0) if residual is None else _matrix(residual, "residual", (n, D), (values.dtype,), device)
    if out is None:
        out = torch.empty((n, D), dtype=values.dtype, device=device)
    po, lo = _matrix(out, "out", (n, D), (values.dtype,), device)
    _call(device, capi.lib.pink_b200_op_read_out, _TYPES[values.dtype], N, D, p, ld, n, k, pn, pw, pr, lr, po, lo)
    return out


def read_out_backward(dy, values, neurons, weights):
    """Gradients (dvalues [N, D], dweights [n, k]) of read_out() from that of its result."""
    device = _two_d(values, "values")
    N, D = values.shape
    p, ld = _matrix(values, "values", (N, D), _ANY, device)
    _two_d(neurons, "neurons")
    n, k = neurons.shape
    pn, pw = _table(neurons, "neurons", (n, k), _INT, device), _table(weights, "weights", (n, k), _FLOAT, device)
    pd, ldd = _matrix(dy, "dy", (n, D), (values.dtype,), device)
    dvalues = torch.empty((N, D), dtype=values.dtype, device=device)
    dweights = torch.empty((n, k), dtype=torch.float32, device=device)
    size = capi.lib.pink_b200_read_out_workspace(N, D, n, k)
    work = torch.empty(size, dtype=torch.uint8, device=device)
    _call(device, capi.lib.pink_b200_op_read_out_backward, _TYPES[values.dtype], N, D, p, ld, n, k, pn, pw, pd, ldd, dvalues.data_ptr(), D,
          dweights.data_ptr(), work.data_ptr(), size)
    return dvalues, dweights


_HALF = (torch.bfloat16, torch.float16)
_FEW_ROWS = 8          # up to as many rows the product needs no workspace


def _sized_call(device, ask, entry, *args):
    """A product entry: asks for its workspace (where it may need one), allocates it, runs it."""
    size = C.c_uint64(0)
    if ask:
        capi.check(entry(*args, None, C.byref(size), 1, None))
    work = torch.empty(size.value, dtype=torch.uint8, device=device) if size.value else None
    _call(device, entry, *args, None if work is None else work.data_ptr(), C.byref(size), 0)


def _product_shapes(x, w, by_input, activation):
    device = _two_d(x, "x")
    _two_d(w, "w")
    n, K = x.shape
    M = w.shape[1] if by_input else w.shape[0]
    px, ldx = _matrix(x, "x", (n, K), _HALF, device)
    pw, ldw = _matrix(w, "w", (K, M) if by_input else (M, K), (x.dtype,), device)
    cfg = capi.ProductConfig(_TYPES[x.dtype], K, M, int(bool(by_input)), _of(_ACTIVATIONS, activation, "activation"), 0, n)
    return device, n, K, M, px, ldx, pw, ldw, cfg


def product(x, w, *, by_input=False, bias=None, activation="none", residual=None, keep=False, out=None):
    """act(x w^T + bias) + residual on the tensor cores: x [n, K] and w [M, K] (by_input: [K, M]) bfloat16 or float16, bias [M] float32.

    keep=True also returns z = x w^T + bias, which product_backward() needs where there is an activation."""
    device, n, K, M, px, ldx, pw, ldw, cfg = _product_shapes(x, w, by_input, activation)
    pb = _vector(bias, "bias", M, _FLOAT, device)
    pr, lr = (None, 0) if residual is None else _matrix(residual, "residual", (n, M), (x.dtype,), device)
    if out is None:
        out = torch.empty((n, M), dtype=x.dtype, device=device)
    po, lo = _matrix(out, "out", (n, M), (x.dtype,), device)
    z = torch.empty((n, M), dtype=x.dtype, device=device) if keep else None
    _sized_call(device, n > _FEW_ROWS, capi.lib.pink_b200_op_product, C.byref(cfg), px, ldx, pw, ldw, pb, pr, lr, po, lo, z.data_ptr() if keep else None, M)
    return (out, z) if keep else out


def product_backward(dy, x, w, *, by_input=False, z=None, activation="none"):
    """Gradients (dx, dw, dbias) of product() from that of its result; the residual's is dy itself."""
    device, n, K, M, px, ldx, pw, ldw, cfg = _product_shapes(x, w, by_input, activation)
    pd, ldd = _matrix(dy, "dy", (n, M), (x.dtype,), device)
    if activation != "none" and z is None:
        raise ValueError("the gradient of an activation needs z: product(..., keep=True)")
    pz, lz = (None, 0) if activation == "none" else _matrix(z, "z", (n, M), (x.dtype,), device)
    dx = torch.empty((n, K), dtype=x.dtype, device=device)
    dw = torch.empty(w.shape, dtype=x.dtype, device=device)
    dbias = torch.empty(M, dtype=torch.float32, device=device)
    _sized_call(device, True, capi.lib.pink_b200_op_product_backward, C.byref(cfg), pd, ldd, px, ldx, pw, ldw, pz, lz, dx.data_ptr(), K,
                dw.data_ptr(), dw.shape[1], dbias.data_ptr())
    return dx, dw, dbias


def check_status():
    """Waits for the current device and raises if a bounded device-side wait of a product expired."""
    capi.check(capi.lib.pink_b200_op_status())
