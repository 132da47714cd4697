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


class _Library(object):
    """The C functions as attributes, each looked up once."""

    def __getattr__(self, name):
        fn = getattr(_lk.cdll(), name)
        setattr(self, name, fn)
        return fn


_lib = _Library()
# The current device and its current stream without the objects that torch.cuda makes for them (1.5 us a call).
_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(fn, index, *args):
    """One C call with device `index` current, on its current stream."""
    if _device() == index:
        rc = fn(*args, _stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _stream(index))
    if rc:
        _lk.check(rc)


def _sizes(fn, index, *args):
    """A C call that only asks about device `index`."""
    if _device() == index:
        rc = fn(*args)
    else:
        with torch.cuda.device(index):
            rc = fn(*args)
    if rc:
        _lk.check(rc)


def _refuse(name, t, device=None, dtype=None, shape=None):
    """Raises what is wrong with a tensor that should be on `device`, of `dtype` and `shape` (where they are given)."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError("%s must be a CUDA tensor" % name)
    if device is not None and t.device != device:
        raise ValueError("%s is on %s, not on %s" % (name, t.device, device))
    if dtype is not None and t.dtype != dtype:
        raise ValueError("%s must be %s, not %s" % (name, dtype, t.dtype))
    if dtype is None and t.dtype not in _CODES:
        raise ValueError("%s must be float32, float16 or bfloat16, not %s" % (name, t.dtype))
    if shape is not None and t.shape != shape:
        raise ValueError("%s has shape %s, not %s" % (name, tuple(t.shape), tuple(shape)))
    raise ValueError("%s: the elements must lie side by side" % name)


def _rows(name, t):
    """(rows, cols, row stride, type code) of a two-dimensional tensor whose rows have their elements side by side."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in _CODES:
        _refuse(name, t)
    if t.dim() != 2:
        raise ValueError("%s must be two-dimensional" % name)
    rows, cols = t.shape
    stride, inner = t.stride()
    if inner != 1 and cols > 1:
        raise ValueError("%s: the elements of a row must lie side by side" % name)
    return rows, cols, stride if rows > 1 else cols, _CODES[t.dtype]


def _same_rows(name, t, like, shape):
    """Row stride of such a tensor that has `shape` and is `like` another in type and device."""
    if not isinstance(t, torch.Tensor) or t.dtype != like.dtype or t.device != like.device or t.shape != shape:
        _refuse(name, t, like.device, like.dtype, shape)
    stride, inner = t.stride()
    if inner != 1 and shape[1] > 1:
        raise ValueError("%s: the elements of a row must lie side by side" % name)
    return stride if shape[0] > 1 else shape[1]


def _flat(name, t, device, dtype, shape):
    """Address of a contiguous tensor of this type and shape."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.device != device or t.shape != shape or not t.is_contiguous():
        _refuse(name, t, device, dtype, shape)
    return t.data_ptr()


def _out(out, like, rows, cols, exact=True):
    """The caller's output, or a new one of `like`'s type and device; and its row stride."""
    if out is None:
        return like.new_empty((rows, cols)), cols
    have = out.shape[0] if isinstance(out, torch.Tensor) and out.dim() == 2 else rows
    return out, _same_rows("out", out, like, (rows if exact or have < rows else have, cols))


def _over(over):
    if over not in _OVER:
        raise ValueError("over must be 'chosen' or 'all', not %r" % (over,))
    return _OVER[over]


# ---- layer norm ------------------------------------------------------------------------------------------------------

def _param(name, t, x, cols):
    """Address and type code of a weight or bias."""
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.float32, x.dtype):
        raise ValueError("%s must be float32 or of the rows' type" % name)
    return _flat(name, t, x.device, t.dtype, (cols,)), _CODES[t.dtype]


def layer_norm(x, weight=None, bias=None, eps=1e-5, out=None):
    """(x - mean) / sqrt(variance + eps) * weight + bias of each row of x (rows, cols); weight and bias (cols, float32
    or x's type, both the same) may be left out.  `out` may be x."""
    rows, cols, stride, code = _rows("x", x)
    w = b = None
    pcode = 0
    if weight is not None:
        w, pcode = _param("weight", weight, x, cols)
    if bias is not None:
        b, bcode = _param("bias", bias, x, cols)
        if weight is not None and bcode != pcode:
            raise ValueError("weight and bias must be of one type")
        pcode = bcode
    y, ystride = _out(out, x, rows, cols)
    mean = x.new_empty(rows, dtype=torch.float32)
    rstd = torch.empty_like(mean)
    _call(_lib.kmeans_layer_norm, x.get_device(), code, x.data_ptr(), stride, rows, cols, w, b, pcode, eps, y.data_ptr(), ystride,
          mean.data_ptr(), rstd.data_ptr())
    return LayerNorm(y, mean, rstd)


def layer_norm_grad(dy, x, mean, rstd, weight=None, params=True):
    """Gradient of :func:`layer_norm`: dx, and with `params` the float32 gradients of weight and bias."""
    rows, cols, stride, code = _rows("x", x)
    dev, index = x.device, x.get_device()
    dstride = _same_rows("dy", dy, x, x.shape)
    m = _flat("mean", mean, dev, torch.float32, (rows,))
    r = _flat("rstd", rstd, dev, torch.float32, (rows,))
    w, pcode = (None, 0) if weight is None else _param("weight", weight, x, cols)
    dx = x.new_empty((rows, cols))
    dweight = dbias = ws = None
    size = ctypes.c_size_t(0)
    if params:
        dweight = x.new_empty(cols, dtype=torch.float32)
        dbias = torch.empty_like(dweight)
        _sizes(_lib.kmeans_layer_norm_grad_workspace, index, rows, cols, ctypes.byref(size))
        ws = x.new_empty(size.value, dtype=torch.uint8)
    _call(_lib.kmeans_layer_norm_grad, index, code, dy.data_ptr(), dstride, x.data_ptr(), stride, m, r, rows, cols, w, pcode,
          dx.data_ptr(), cols, dweight.data_ptr() if params else None, dbias.data_ptr() if params else None,
          ws.data_ptr() if params else None, size.value)
    return LayerNormGrad(dx, dweight, dbias)


# ---- routing ---------------------------------------------------------------------------------------------------------

def _scores(scores):
    """(rows, clusters, their strides, type code) of two-dimensional scores in any strides."""
    if not isinstance(scores, torch.Tensor) or not scores.is_cuda or scores.dtype not in _CODES:
        _refuse("scores", scores)
    if scores.dim() != 2:
        raise ValueError("scores must be two-dimensional")
    return (*scores.shape, *scores.stride(), _CODES[scores.dtype])


def _routes(rows, n, like):
    ids = like.new_empty((rows, n), dtype=torch.int32)
    weights = like.new_empty((rows, n), dtype=torch.float32)
    best = like.new_empty(rows, dtype=torch.float32)
    return Routes(ids, weights, best, torch.empty_like(best))


def route(scores, n, scale=-1.0, over="chosen"):
    """The n best of the clusters of each row and their weights, from scores (rows, k) in any strides: distances as
    ``transform`` lays them out (cluster after cluster), a linear router's logits (row after row).

    scale > 0: larger scores are better, scale < 0: smaller ones (distances; -1 / temperature).  The weights are a softmax
    of scale * score over the chosen clusters, or over all of them (`over`).  Ties go to the lowest cluster; NaN and infinitely
    bad scores are never chosen."""
    rows, k, rs, cs, code = _scores(scores)
    flag = _over(over)
    out = _routes(rows, n, scores)
    ids, weights, best, total = out
    _call(_lib.kmeans_route, scores.get_device(), code, scores.data_ptr(), rs, cs, rows, k, n, scale, flag, ids.data_ptr(),
          weights.data_ptr(), best.data_ptr(), total.data_ptr())
    return out


def route_grad(dweights, scores, routes, scale=-1.0, over="chosen"):
    """Gradient of the scores, of their type and in their order of dimensions, from that of the weights; `routes`, `scale`
    and `over` as :func:`route` returned and took them."""
    rows, k, rs, cs, code = _scores(scores)
    flag = _over(over)
    ids, weights, best, total = routes
    if ids.dim() != 2:
        raise ValueError("routes.ids must be two-dimensional")
    dev, n = scores.device, ids.shape[1]
    f32, shape = torch.float32, (rows, n)
    args = (_flat("routes.ids", ids, dev, torch.int32, shape), _flat("routes.weights", weights, dev, f32, shape),
            _flat("routes.best", best, dev, f32, (rows,)), _flat("routes.total", total, dev, f32, (rows,)))
    if rs < cs:
        out = scores.new_empty((k, rows)).t()
        drs, dcs = 1, rows
    else:
        out = scores.new_empty((rows, k))
        drs, dcs = k, 1
    _call(_lib.kmeans_route_grad, scores.get_device(), code, _flat("dweights", dweights, dev, f32, shape), scores.data_ptr(), rs, cs,
          rows, k, n, scale, flag, *args, out.data_ptr(), drs, dcs)
    return out


def nearest(handle, n, scale=-1.0, over="chosen", local=0):
    """:func:`route` on the distances of a ``ResidentKMeans`` handle's shard `local` to its centroids, which never leave the
    device: the n nearest clusters of every row.  float32 handles."""
    dev = torch.device("cuda", handle.shard_device(local))
    out = _routes(handle.shard_rows(local), n, torch.empty(0, device=dev))
    torch.cuda.current_stream(dev).synchronize()      # the handle's stream is another one
    handle.nearest(*[t.data_ptr() for t in out], n, scale, _over(over), local)
    return out


# ---- rows sorted by cluster and back ---------------------------------------------------------------------------------

def sort_rows(ids, k, align=1):
    """Places of rows sorted by cluster: ids (rows,) or (rows, n) int32, outside [0, k) for entries that go nowhere.  Groups
    start on multiples of `align`; entries of a group keep their order."""
    if not isinstance(ids, torch.Tensor) or not ids.is_cuda or ids.dtype != torch.int32:
        _refuse("ids", ids, None, torch.int32)
    if ids.dim() == 1:
        ids = ids.unsqueeze(1)
    if ids.dim() != 2:
        raise ValueError("ids must be one- or two-dimensional")
    rows, n = ids.shape
    stride, inner = ids.stride()
    if inner != 1 and n > 1:
        raise ValueError("ids: the elements of a row must lie side by side")
    index = ids.get_device()
    capacity, size = ctypes.c_size_t(0), ctypes.c_size_t(0)
    _sizes(_lib.kmeans_sort_rows_sizes, index, rows, n, k, align, ctypes.byref(capacity), ctypes.byref(size))
    offsets = ids.new_empty(k + 1)
    counts = ids.new_empty(k)
    slot = ids.new_empty((rows, n))
    source = ids.new_empty(capacity.value)
    ws = ids.new_empty(size.value, dtype=torch.uint8) if size.value else None
    _call(_lib.kmeans_sort_rows, index, ids.data_ptr(), stride if rows > 1 else n, rows, n, k, align, offsets.data_ptr(),
          counts.data_ptr(), slot.data_ptr(), source.data_ptr(), None if ws is None else ws.data_ptr(), size.value)
    return SortedRows(offsets, counts, slot, source)


def _plan(plan, dev):
    """(address of slot, address of source, rows, entries a row, places)"""
    slot, source = plan.slot, plan.source
    if slot.dim() != 2 or source.dim() != 1:
        raise ValueError("plan.slot must be two-dimensional and plan.source one-dimensional")
    rows, n = slot.shape
    return (_flat("plan.slot", slot, dev, torch.int32, slot.shape), _flat("plan.source", source, dev, torch.int32, source.shape),
            rows, n, source.shape[0])


def dispatch(x, plan, out=None):
    """Rows of x (rows, cols) at the places of `plan` (places, cols); padding becomes zero rows.  `out` may have more
    rows than the plan has places: those behind stay as they are."""
    have, cols, stride, code = _rows("x", x)
    slot, source, rows, n, capacity = _plan(plan, x.device)
    if have != rows:
        raise ValueError("x has %d rows, the plan %d" % (have, rows))
    y, ystride = _out(out, x, capacity, cols, exact=False)
    _call(_lib.kmeans_dispatch, x.get_device(), code, x.data_ptr(), stride, rows, cols, n, slot, source, capacity, y.data_ptr(),
          ystride)
    return y


def dispatch_grad(drows, plan, out=None):
    """Gradient of :func:`dispatch`: each row's sum over its places."""
    return combine(drows, plan, None, out)


def combine(rows, plan, weights=None, out=None):
    """Sum of each row's entries of the sorted `rows` (places, cols), with weights (rows, n) float32 or without; entries
    that went nowhere add nothing."""
    have, cols, stride, code = _rows("rows", rows)
    slot, _, t, n, capacity = _plan(plan, rows.device)
    if have < capacity:
        raise ValueError("rows has %d rows, the plan %d places" % (have, capacity))
    w = None if weights is None else _flat("weights", weights, rows.device, torch.float32, (t, n))
    y, ystride = _out(out, rows, t, cols)
    _call(_lib.kmeans_combine, rows.get_device(), code, rows.data_ptr(), stride, capacity, cols, slot, w, t, n, y.data_ptr(), ystride)
    return y


def combine_grad(dy, rows, plan, weights):
    """Gradients of :func:`combine` for the sorted rows (zero rows at padding) and the weights."""
    have, cols, stride, code = _rows("rows", rows)
    slot, source, t, n, capacity = _plan(plan, rows.device)
    if have < capacity:
        raise ValueError("rows has %d rows, the plan %d places" % (have, capacity))
    dstride = _same_rows("dy", dy, rows, (t, cols))
    w = _flat("weights", weights, rows.device, torch.float32, (t, n))
    drows = rows.new_empty((capacity, cols))
    dweights = torch.empty_like(weights)
    _call(_lib.kmeans_combine_grad, rows.get_device(), code, dy.data_ptr(), dstride, rows.data_ptr(), stride, capacity, cols, slot,
          source, w, t, n, drows.data_ptr(), cols, dweights.data_ptr())
    return CombineGrad(drows, dweights)
