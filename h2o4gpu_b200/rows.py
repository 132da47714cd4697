"""Row operators on device tensors, beside the engine: what a layer of experts does around a k-means model that routes
its rows.

    norm = layer_norm(x, weight, bias)                  # rows of one length: distances then compare directions
    routes = nearest(handle, 2)                         # a ResidentKMeans: its nearest clusters and their weights
    routes = route(scores, 2, scale)                    # or the same from any scores
    plan = sort_rows(routes.ids, k, align=128)          # places of the rows sorted by cluster
    xs = dispatch(norm.y, plan)                         # the sorted rows, for the experts
    y = combine(expert_rows, plan, routes.weights)      # and back

and the gradients of each (``layer_norm_grad``, ``route_grad``, ``dispatch_grad``, ``combine_grad``).  Thin Python over
section 5 of include/h2o4gpu_kmeans.h: tensors are torch CUDA tensors (float32, float16 or bfloat16; ids int32), work is
enqueued on the current stream of their device, nothing waits (``nearest`` does, as every call on a handle), nothing is
kept between calls.  Outputs are new tensors of the caller's allocator.  Gradients are explicit functions: no call here
records anything for autograd.  There is no CPU implementation.
"""
import ctypes
from typing import NamedTuple

import torch

from .libs import lib_kmeans as _lk

_CODES = {torch.float32: 0, torch.float16: 2, torch.bfloat16: 11}
_OVER = {"chosen": 0, "all": 1}


class LayerNorm(NamedTuple):
    """Normed rows, and the float32 mean and 1 / sqrt(variance + eps) of each row, which the gradient takes."""
    y: torch.Tensor
    mean: torch.Tensor
    rstd: torch.Tensor


class LayerNormGrad(NamedTuple):
    """Gradients of the rows (their type), the weight and the bias (float32 sums over the rows; None if not asked for)."""
    dx: torch.Tensor
    dweight: torch.Tensor
    dbias: torch.Tensor


class Routes(NamedTuple):
    """Chosen clusters of each row, best first (int32, -1: none), their float32 weights, and per row the best score
    and the sum that the weights were divided by."""
    ids: torch.Tensor
    weights: torch.Tensor
    best: torch.Tensor
    total: torch.Tensor


class SortedRows(NamedTuple):
    """Places of rows sorted by cluster (all int32): where each cluster's group starts (k + 1), its entries (k), the place
    of every entry (rows x n, -1: none), and the entry at every place (-1: padding)."""
    offsets: torch.Tensor
    counts: torch.Tensor
    slot: torch.Tensor
    source: torch.Tensor


class CombineGrad(NamedTuple):
    """Gradients of the sorted rows and of the weights."""
    drows: torch.Tensor
    dweights: torch.Tensor


def _call(name, device, *args):
    """One C call with `device` current, on its current stream."""
    fn = getattr(_lk.cdll(), name)
    index = device.index
    if torch.cuda.current_device() == index:
        _lk.check(fn(*args, torch.cuda.current_stream(index).cuda_stream))
    else:
        with torch.cuda.device(index):
            _lk.check(fn(*args, torch.cuda.current_stream(index).cuda_stream))


def _code(name, t):
    code = _CODES.get(t.dtype)
    if code is None:
        raise ValueError("%s must be float32, float16 or bfloat16, not %s" % (name, t.dtype))
    return code


def _on(name, t, device=None, dtype=None, shape=None):
    """`t` as a CUDA tensor (on `device`, of `dtype` and `shape` where they are given)."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError("%s must be a CUDA tensor" % name)
    if device is not None and t.device != device:
        raise ValueError("%s is on %s, not on %s" % (name, t.device, device))
    if dtype is not None and t.dtype != dtype:
        raise ValueError("%s must be %s, not %s" % (name, dtype, t.dtype))
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError("%s has shape %s, not %s" % (name, tuple(t.shape), tuple(shape)))
    return t


def _block(name, t, device=None, dtype=None, shape=None):
    """`t` as a two-dimensional tensor whose rows have their elements side by side; its row stride."""
    _on(name, t, device, dtype, shape)
    if t.dim() != 2:
        raise ValueError("%s must be two-dimensional" % name)
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError("%s: the elements of a row must lie side by side" % name)
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _vector(name, t, device, dtype, shape):
    _on(name, t, device, dtype, shape)
    if not t.is_contiguous():
        raise ValueError("%s must be contiguous" % name)
    return t.data_ptr()


def _out(name, out, like, rows, cols, exact=True):
    """The caller's output, or a new one of `like`'s type and device; and its row stride."""
    if out is None:
        return torch.empty((rows, cols), dtype=like.dtype, device=like.device), cols
    stride = _block(name, out, like.device, like.dtype)
    if out.shape[1] != cols or out.shape[0] < rows or (exact and out.shape[0] != rows):
        raise ValueError("%s has shape %s, not (%d, %d)" % (name, tuple(out.shape), rows, cols))
    return out, stride


def _over(over):
    if over not in _OVER:
        raise ValueError("over must be 'chosen' or 'all', not %r" % (over,))
    return _OVER[over]


# ---- layer norm ------------------------------------------------------------------------------------------------------

def _params(x, weight, bias):
    """Pointers of weight and bias, and the code of their type."""
    given = [t for t in (weight, bias) if t is not None]
    if not given:
        return None, None, 0
    if any(t.dtype not in (torch.float32, x.dtype) or t.dtype != given[0].dtype for t in given):
        raise ValueError("weight and bias must be float32, or both of the rows' type")
    shape = (x.shape[1],)
    return (None if weight is None else _vector("weight", weight, x.device, None, shape),
            None if bias is None else _vector("bias", bias, x.device, None, shape), _CODES[given[0].dtype])


def layer_norm(x, weight=None, bias=None, eps=1e-5, out=None):
    """(x - mean) / sqrt(variance + eps) * weight + bias of each row of x (rows, cols); weight and bias (cols, float32
    or x's type) may be left out.  `out` may be x."""
    stride, code = _block("x", x), _code("x", x)
    rows, cols = x.shape
    w, b, pcode = _params(x, weight, bias)
    y, ystride = _out("out", out, x, rows, cols)
    mean = torch.empty(rows, dtype=torch.float32, device=x.device)
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
    _call("kmeans_layer_norm", x.device, code, x.data_ptr(), stride, rows, cols, w, b, pcode, eps, y.data_ptr(), ystride,
          mean.data_ptr(), rstd.data_ptr())
    return LayerNorm(y, mean, rstd)


def layer_norm_grad(dy, x, mean, rstd, weight=None, params=True):
    """Gradient of :func:`layer_norm`: dx, and with `params` the float32 gradients of weight and bias."""
    stride, code = _block("x", x), _code("x", x)
    rows, cols = x.shape
    dev = x.device
    dstride = _block("dy", dy, dev, x.dtype, x.shape)
    m = _vector("mean", mean, dev, torch.float32, (rows,))
    r = _vector("rstd", rstd, dev, torch.float32, (rows,))
    w, _, pcode = _params(x, weight, None)
    dx = torch.empty((rows, cols), dtype=x.dtype, device=dev)
    dweight = dbias = ws = None
    size = ctypes.c_size_t(0)
    if params:
        dweight = torch.empty(cols, dtype=torch.float32, device=dev)
        dbias = torch.empty(cols, dtype=torch.float32, device=dev)
        with torch.cuda.device(dev):
            _lk.check(_lk.cdll().kmeans_layer_norm_grad_workspace(rows, cols, ctypes.byref(size)))
        ws = torch.empty(size.value, dtype=torch.uint8, device=dev)
    _call("kmeans_layer_norm_grad", dev, code, dy.data_ptr(), dstride, x.data_ptr(), stride, m, r, rows, cols, w, pcode,
          dx.data_ptr(), cols, None if dweight is None else dweight.data_ptr(), None if dbias is None else dbias.data_ptr(),
          None if ws is None else ws.data_ptr(), size.value)
    return LayerNormGrad(dx, dweight, dbias)


# ---- routing ---------------------------------------------------------------------------------------------------------

def _scores(name, t):
    _on(name, t)
    if t.dim() != 2:
        raise ValueError("%s must be two-dimensional" % name)
    return _code(name, t)


def route(scores, n, scale=-1.0, over="chosen"):
    """The n best of the clusters of each row and their weights, from scores (rows, k) in any strides: distances as
    ``transform`` lays them out (cluster after cluster), a linear router's logits (row after row).

    scale > 0: larger scores are better, scale < 0: smaller ones (distances; -1 / temperature).  The weights are a softmax
    of scale * score over the chosen clusters, or over all of them (`over`).  Ties go to the lowest cluster; NaN and infinitely
    bad scores are never chosen."""
    code = _scores("scores", scores)
    rows, k = scores.shape
    dev = scores.device
    ids = torch.empty((rows, n), dtype=torch.int32, device=dev)
    weights = torch.empty((rows, n), dtype=torch.float32, device=dev)
    best = torch.empty(rows, dtype=torch.float32, device=dev)
    total = torch.empty(rows, dtype=torch.float32, device=dev)
    _call("kmeans_route", dev, code, scores.data_ptr(), scores.stride(0), scores.stride(1), rows, k, n, scale, _over(over),
          ids.data_ptr(), weights.data_ptr(), best.data_ptr(), total.data_ptr())
    return Routes(ids, weights, best, total)


def route_grad(dweights, scores, routes, scale=-1.0, over="chosen"):
    """Gradient of the scores, of their type and in their order of dimensions, from that of the weights; `routes`, `scale`
    and `over` as :func:`route` returned and took them."""
    code = _scores("scores", scores)
    rows, k = scores.shape
    dev = scores.device
    if routes.ids.dim() != 2:
        raise ValueError("routes.ids must be two-dimensional")
    shape = (rows, routes.ids.shape[1])
    args = (_vector("routes.ids", routes.ids, dev, torch.int32, shape),
            _vector("routes.weights", routes.weights, dev, torch.float32, shape),
            _vector("routes.best", routes.best, dev, torch.float32, (rows,)),
            _vector("routes.total", routes.total, dev, torch.float32, (rows,)))
    if scores.stride(0) < scores.stride(1):
        out = torch.empty((k, rows), dtype=scores.dtype, device=dev).t()
        drs, dcs = 1, rows
    else:
        out = torch.empty((rows, k), dtype=scores.dtype, device=dev)
        drs, dcs = k, 1
    _call("kmeans_route_grad", dev, code, _vector("dweights", dweights, dev, torch.float32, shape), scores.data_ptr(),
          scores.stride(0), scores.stride(1), rows, k, shape[1], scale, _over(over), *args, out.data_ptr(), drs, dcs)
    return out


def nearest(handle, n, scale=-1.0, over="chosen", local=0):
    """:func:`route` on the distances of a ``ResidentKMeans`` handle's shard `local` to its centroids, which never leave the
    device: the n nearest clusters of every row.  float32 handles."""
    device, rows = handle.shard_device(local), handle.shard_rows(local)
    dev = torch.device("cuda", device)
    ids = torch.empty((rows, n), dtype=torch.int32, device=dev)
    weights = torch.empty((rows, n), dtype=torch.float32, device=dev)
    best = torch.empty(rows, dtype=torch.float32, device=dev)
    total = torch.empty(rows, dtype=torch.float32, device=dev)
    torch.cuda.current_stream(dev).synchronize()      # the handle's stream is another one
    handle.nearest(ids.data_ptr(), weights.data_ptr(), best.data_ptr(), total.data_ptr(), n, scale, _over(over), local)
    return Routes(ids, weights, best, total)


# ---- rows sorted by cluster and back ---------------------------------------------------------------------------------

def sort_rows(ids, k, align=1):
    """Places of rows sorted by cluster: ids (rows,) or (rows, n) int32, outside [0, k) for entries that go nowhere.  Groups
    start on multiples of `align`; entries of a group keep their order."""
    if isinstance(ids, torch.Tensor) and ids.dim() == 1:
        ids = ids.unsqueeze(1)
    stride = _block("ids", ids, None, torch.int32)
    rows, n = ids.shape
    dev = ids.device
    capacity, size = ctypes.c_size_t(0), ctypes.c_size_t(0)
    with torch.cuda.device(dev):
        _lk.check(_lk.cdll().kmeans_sort_rows_sizes(rows, n, k, align, ctypes.byref(capacity), ctypes.byref(size)))
    offsets = torch.empty(k + 1, dtype=torch.int32, device=dev)
    counts = torch.empty(k, dtype=torch.int32, device=dev)
    slot = torch.empty((rows, n), dtype=torch.int32, device=dev)
    source = torch.empty(capacity.value, dtype=torch.int32, device=dev)
    ws = torch.empty(size.value, dtype=torch.uint8, device=dev)
    _call("kmeans_sort_rows", dev, ids.data_ptr(), stride, rows, n, k, align, offsets.data_ptr(), counts.data_ptr(),
          slot.data_ptr(), source.data_ptr(), ws.data_ptr(), size.value)
    return SortedRows(offsets, counts, slot, source)


def _plan(plan, dev):
    if plan.slot.dim() != 2 or plan.source.dim() != 1:
        raise ValueError("plan.slot must be two-dimensional and plan.source one-dimensional")
    return (_vector("plan.slot", plan.slot, dev, torch.int32, plan.slot.shape),
            _vector("plan.source", plan.source, dev, torch.int32, plan.source.shape),
            plan.slot.shape[0], plan.slot.shape[1], plan.source.shape[0])


def dispatch(x, plan, out=None):
    """Rows of x (rows, cols) at the places of `plan` (places, cols); padding becomes zero rows.  `out` may have more
    rows than the plan has places: those behind stay as they are."""
    stride, code = _block("x", x), _code("x", x)
    slot, source, rows, n, capacity = _plan(plan, x.device)
    cols = x.shape[1]
    if x.shape[0] != rows:
        raise ValueError("x has %d rows, the plan %d" % (x.shape[0], rows))
    y, ystride = _out("out", out, x, capacity, cols, exact=False)
    _call("kmeans_dispatch", x.device, code, x.data_ptr(), stride, rows, cols, n, slot, source, capacity, y.data_ptr(), ystride)
    return y


def _sorted_block(name, t, capacity):
    stride, code = _block(name, t), _code(name, t)
    if t.shape[0] < capacity:
        raise ValueError("%s has %d rows, the plan %d places" % (name, t.shape[0], capacity))
    return stride, code


def dispatch_grad(drows, plan, out=None):
    """Gradient of :func:`dispatch`: each row's sum over its places."""
    return combine(drows, plan, None, out)


def combine(rows, plan, weights=None, out=None):
    """Sum of each row's entries of the sorted `rows` (places, cols), with weights (rows, n) float32 or without; entries
    that went nowhere add nothing."""
    _on("rows", rows)
    slot, _, t, n, capacity = _plan(plan, rows.device)
    stride, code = _sorted_block("rows", rows, capacity)
    cols = rows.shape[1]
    w = None if weights is None else _vector("weights", weights, rows.device, torch.float32, (t, n))
    y, ystride = _out("out", out, rows, t, cols)
    _call("kmeans_combine", rows.device, code, rows.data_ptr(), stride, capacity, cols, slot, w, t, n, y.data_ptr(), ystride)
    return y


def combine_grad(dy, rows, plan, weights):
    """Gradients of :func:`combine` for the sorted rows (zero rows at padding) and the weights."""
    _on("rows", rows)
    dev = rows.device
    slot, source, t, n, capacity = _plan(plan, dev)
    stride, code = _sorted_block("rows", rows, capacity)
    cols = rows.shape[1]
    dstride = _block("dy", dy, dev, rows.dtype, (t, cols))
    w = _vector("weights", weights, dev, torch.float32, (t, n))
    drows = torch.empty((capacity, cols), dtype=rows.dtype, device=dev)
    dweights = torch.empty((t, n), dtype=torch.float32, device=dev)
    _call("kmeans_combine_grad", dev, code, dy.data_ptr(), dstride, rows.data_ptr(), stride, capacity, cols, slot, source, w, t, n,
          drows.data_ptr(), cols, dweights.data_ptr())
    return CombineGrad(drows, dweights)
