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
records anything for autograd, and one whose inputs require gradients while autograd records says so in a warning (call it
under ``torch.no_grad()`` or on detached tensors).  There is no CPU implementation.
"""
import ctypes
import warnings
from typing import NamedTuple

import torch

from .libs import lib_kmeans as _lk

_CODES = {torch.float32: 0, torch.float16: 2, torch.bfloat16: 11}
_OVER = {"chosen": 0, "all": 1}
_FEW_ROWS = 256           # rows whose gradient's workspace need not be asked for
_SORT_ONE_CTA = 2048      # entries below which kmeans_sort_rows needs no workspace
_SORT_KNOWN = 16384       # k and align up to which the places of so few entries need not be asked for
_INT = 0x7fffffff         # ctypes would cut what is more down to a C int without a word


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


def _refuse(name, t, index=None, dtype=None, shape=None):
    """Raises what is wrong with a tensor that should be on device `index`, of `dtype` and `shape` (where they are given)."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError("%s must be a CUDA tensor" % name)
    if t.is_neg():
        raise ValueError("%s is a view whose sign torch keeps apart: take its resolve_neg()" % name)
    if index is not None and t.get_device() != index:
        raise ValueError("%s is on %s, not on cuda:%d" % (name, t.device, index))
    if dtype is not None and t.dtype != dtype:
        raise ValueError("%s must be %s, not %s" % (name, dtype, t.dtype))
    if dtype is None and t.dtype not in _CODES:
        raise ValueError("%s must be float32, float16 or bfloat16, not %s" % (name, t.dtype))
    if shape is not None and t.shape != shape:
        raise ValueError("%s has shape %s, not %s" % (name, tuple(t.shape), tuple(shape)))
    if shape is None and t.dim() != 2:
        raise ValueError("%s must be two-dimensional" % name)
    raise ValueError("%s: the elements must lie side by side" % name)


# The checks below ask a tensor for as little as they can: they are a good part of a small call's time.

def _rows(name, t):
    """(rows, cols, row stride, type code, device) of a two-dimensional tensor whose rows have their elements side by side."""
    try:
        code, index = _CODES[t.dtype], t.get_device()
        rows, cols = t.shape
        stride, inner = t.stride()
    except (AttributeError, KeyError, ValueError):
        _refuse(name, t)
    if index < 0 or (inner != 1 and (cols > 1 or t.is_neg())):
        _refuse(name, t)
    return rows, cols, stride if rows > 1 else cols, code, index


def _same_rows(name, t, like, index, shape):
    """Row stride of such a tensor that has `shape`, `like`'s type and its device."""
    if not isinstance(t, torch.Tensor) or t.dtype is not like.dtype or t.get_device() != index or t.shape != shape:
        _refuse(name, t, index, like.dtype, shape)
    stride, inner = t.stride()
    if inner != 1 and (shape[1] > 1 or t.is_neg()):
        _refuse(name, t, index, like.dtype, shape)
    return stride if shape[0] > 1 else shape[1]


def _flat(name, t, index, dtype, shape):
    """Address of a contiguous tensor of this type and shape on this device."""
    try:
        if t.dtype is dtype and t.get_device() == index and t.shape == shape and t.is_contiguous():
            return t.data_ptr()
    except AttributeError:
        pass
    _refuse(name, t, index, dtype, shape)


def _per_entry(name, t, index, dtype, shape):
    """A tensor of this type and shape on this device in any strides, as one whose elements lie side by side: routes and weights that were
    sorted from scores lying cluster after cluster lie so too, a gradient may be one number for all.  The caller keeps it until its call is made."""
    try:
        if t.dtype is dtype and t.get_device() == index and t.shape == shape:
            return t if t.is_contiguous() else t.contiguous()
    except AttributeError:
        pass
    _refuse(name, t, index, dtype, shape)


def _overlap(out, rows, t, t_rows):
    """Whether the first `rows` rows of `out` share memory with the first `t_rows` of `t` (of the same type and as many columns); False too
    for rows in two different strides, which are not looked at."""
    cols, size = t.shape[1], t.element_size()
    s, ts = (out.stride(0) if rows > 1 else 0), (t.stride(0) if t_rows > 1 else 0)
    at = (t.data_ptr() - out.data_ptr()) // size
    if not rows or not t_rows or at >= (rows - 1) * s + cols or at + (t_rows - 1) * ts + cols <= 0:
        return False
    if s and ts and s != ts:
        return False
    step = s or ts
    return not step or not cols <= at % step <= step - cols      # columns side by side in rows of one stride


def _out(out, like, index, rows, cols, exact=True, read=None, in_place=False):
    """The caller's output, or a new one of `like`'s type and device; and its row stride.  `read`: rows of `like` that the call reads."""
    if out is None:
        return like.new_empty((rows, cols)), cols
    have = out.shape[0] if isinstance(out, torch.Tensor) and out.dim() == 2 else rows
    stride = _same_rows("out", out, like, index, (rows if exact or have < rows else have, cols))
    read = like.shape[0] if read is None else read
    same = in_place and out.data_ptr() == like.data_ptr() and (rows < 2 or stride == like.stride(0))
    if not same and _overlap(out, rows, like, read):
        raise ValueError("out shares memory with the rows that are read")
    return out, stride


def _unrecorded(name):
    """Warns that a call, some of whose inputs require gradients, cuts autograd's record."""
    if torch.is_grad_enabled():
        warnings.warn("%s records nothing for autograd: its result has no gradient, take %s_grad" % (name, name), stacklevel=3)


def _over(over):
    if over not in _OVER:
        raise ValueError("over must be 'chosen' or 'all', not %r" % (over,))
    return _OVER[over]


# ---- layer norm ------------------------------------------------------------------------------------------------------

def _param(name, t, x, index, cols):
    """Address and type code of a weight or bias."""
    dtype = getattr(t, "dtype", None)
    if dtype is not x.dtype and dtype is not torch.float32:
        raise ValueError("%s must be float32 or of the rows' type" % name)
    return _flat(name, t, index, dtype, (cols,)), _CODES[dtype]


def layer_norm(x, weight=None, bias=None, eps=1e-5, out=None):
    """(x - mean) / sqrt(variance + eps) * weight + bias of each row of x (rows, cols); weight and bias (cols, float32
    or x's type, both the same) may be left out.  `out` may be x."""
    rows, cols, stride, code, index = _rows("x", x)
    w = b = None
    pcode = 0
    if weight is not None:
        w, pcode = _param("weight", weight, x, index, cols)
    if bias is not None:
        b, bcode = _param("bias", bias, x, index, cols)
        if weight is not None and bcode != pcode:
            raise ValueError("weight and bias must be of one type")
        pcode = bcode
    if out is None and stride == cols:
        y, ystride = torch.empty_like(x), cols
    else:
        y, ystride = _out(out, x, index, rows, cols, in_place=True)
    mean = x.new_empty(rows, dtype=torch.float32)
    rstd = torch.empty_like(mean)
    if x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad):
        _unrecorded("layer_norm")
    _call(_lib.kmeans_layer_norm, index, code, x.data_ptr(), stride, rows, cols, w, b, pcode, eps, y.data_ptr(), ystride,
          mean.data_ptr(), rstd.data_ptr())
    return LayerNorm(y, mean, rstd)


def layer_norm_grad(dy, x, mean, rstd, weight=None, params=True):
    """Gradient of :func:`layer_norm`: dx, and with `params` the float32 gradients of weight and bias."""
    rows, cols, stride, code, index = _rows("x", x)
    dstride = _same_rows("dy", dy, x, index, x.shape)
    m = _flat("mean", mean, index, torch.float32, (rows,))
    r = _flat("rstd", rstd, index, torch.float32, (rows,))
    w, pcode = (None, 0) if weight is None else _param("weight", weight, x, index, cols)
    dx = torch.empty_like(x) if stride == cols else x.new_empty((rows, cols))
    if not params:
        _call(_lib.kmeans_layer_norm_grad, index, code, dy.data_ptr(), dstride, x.data_ptr(), stride, m, r, rows, cols, w, pcode,
              dx.data_ptr(), cols, None, None, None, 0)
        return LayerNormGrad(dx, None, None)
    dweight = x.new_empty(cols, dtype=torch.float32)
    dbias = torch.empty_like(dweight)
    work = 8 * rows * cols      # a partial sum for every row is always enough
    if rows > _FEW_ROWS:
        size = ctypes.c_size_t(0)
        _sizes(_lib.kmeans_layer_norm_grad_workspace, index, rows, cols, ctypes.byref(size))
        work = size.value
    ws = x.new_empty(work, dtype=torch.uint8)
    _call(_lib.kmeans_layer_norm_grad, index, code, dy.data_ptr(), dstride, x.data_ptr(), stride, m, r, rows, cols, w, pcode,
          dx.data_ptr(), cols, dweight.data_ptr(), dbias.data_ptr(), ws.data_ptr(), work)
    return LayerNormGrad(dx, dweight, dbias)


# ---- routing ---------------------------------------------------------------------------------------------------------

def _scores(scores):
    """(rows, clusters, their strides, type code, device) of two-dimensional scores in any strides."""
    try:
        code, index = _CODES[scores.dtype], scores.get_device()
        rows, k = scores.shape
        rs, cs = scores.stride()
    except (AttributeError, KeyError, ValueError):
        _refuse("scores", scores)
    if index < 0 or scores.is_neg():
        _refuse("scores", scores)
    if k > _INT:
        raise ValueError("scores of %d clusters are too many" % k)
    return rows, k, rs, cs, code, index


def _routes(rows, n, like):
    ids = like.new_empty((rows, n), dtype=torch.int32)
    weights = torch.empty_like(ids, dtype=torch.float32)
    best = like.new_empty(rows, dtype=torch.float32)
    return Routes(ids, weights, best, torch.empty_like(best))


def route(scores, n, scale=-1.0, over="chosen"):
    """The n best of the clusters of each row and their weights, from scores (rows, k) in any strides: distances as
    ``transform`` lays them out (cluster after cluster), a linear router's logits (row after row).

    scale > 0: larger scores are better, scale < 0: smaller ones (distances; -1 / temperature).  The weights are a softmax
    of scale * score over the chosen clusters, or over all of them (`over`).  Ties go to the lowest cluster; NaN and infinitely
    bad scores are never chosen."""
    rows, k, rs, cs, code, index = _scores(scores)
    flag = _over(over)
    if not 0 < n <= k:
        raise ValueError("a row takes 1 to %d clusters, not %s" % (k, n))
    out = _routes(rows, n, scores)
    ids, weights, best, total = out
    if scores.requires_grad:
        _unrecorded("route")
    _call(_lib.kmeans_route, index, code, scores.data_ptr(), rs, cs, rows, k, n, scale, flag, ids.data_ptr(),
          weights.data_ptr(), best.data_ptr(), total.data_ptr())
    return out


def _no_scores(ids, k, dtype, over):
    """What :func:`_scores` gives, of scores that are not at hand: as if they lay row after row."""
    if over != "chosen":
        raise ValueError("weights over all clusters: their gradient needs the scores")
    if dtype not in _CODES:
        raise ValueError("dtype must be float32, float16 or bfloat16, not %s" % dtype)
    if not isinstance(ids, torch.Tensor) or not ids.is_cuda or ids.dim() != 2:
        _refuse("routes.ids", ids, None, torch.int32)
    if k is None or not 0 < k <= _INT:
        raise ValueError("without scores, k is the number of clusters, not %s" % k)
    return ids.shape[0], k, k, 1, _CODES[dtype], ids.get_device()


def route_grad(dweights, scores, routes, scale=-1.0, over="chosen", k=None, dtype=torch.float32):
    """Gradient of the scores, of their type and in their order of dimensions, from that of the weights; `routes`, `scale`
    and `over` as :func:`route` returned and took them.  Routes and `dweights` may lie in any strides (others than side by side are
    copied).  Over the chosen clusters no score is read: `scores` may be None (behind :func:`nearest`, whose distances nobody
    has), the gradient then is (rows, `k`) of `dtype`, row after row.  With scores, `k` and `dtype` are theirs."""
    ids, weights, best, total = (None,) * 4 if routes is None else routes
    if scores is None:
        rows, k, rs, cs, code, index = _no_scores(ids, k, dtype, over)
    else:
        rows, k, rs, cs, code, index = _scores(scores)
        dtype = scores.dtype
    flag = _over(over)
    if not isinstance(ids, torch.Tensor) or ids.dim() != 2:
        raise ValueError("routes.ids must be a two-dimensional tensor")
    n, f32 = ids.shape[1], torch.float32
    if n > k:
        raise ValueError("routes of %d clusters a row, scores of %d" % (n, k))
    shape = (rows, n)
    dweights = _per_entry("dweights", dweights, index, f32, shape)
    ids, weights = _per_entry("routes.ids", ids, index, torch.int32, shape), _per_entry("routes.weights", weights, index, f32, shape)
    best, total = _per_entry("routes.best", best, index, f32, (rows,)), _per_entry("routes.total", total, index, f32, (rows,))
    if rs < cs:
        out = dweights.new_empty((k, rows), dtype=dtype).t()
        drs, dcs = 1, rows
    else:
        out = dweights.new_empty((rows, k), dtype=dtype)
        drs, dcs = k, 1
    _call(_lib.kmeans_route_grad, index, code, dweights.data_ptr(), None if scores is None else scores.data_ptr(), rs, cs, rows, k, n,
          scale, flag, ids.data_ptr(), weights.data_ptr(), best.data_ptr(), total.data_ptr(), out.data_ptr(), drs, dcs)
    return out


def nearest(handle, n, scale=-1.0, over="chosen", local=0):
    """:func:`route` on the distances of a ``ResidentKMeans`` handle's shard `local` to its centroids, which never leave the
    device: the n nearest clusters of every row.  float32 handles."""
    if n > _INT:
        raise ValueError("%d clusters a row are too many" % n)
    dev = torch.device("cuda", handle.shard_device(local))
    out = _routes(handle.shard_rows(local), n, torch.empty(0, device=dev))
    torch.cuda.current_stream(dev).synchronize()      # the handle's stream is another one
    handle.nearest(*[t.data_ptr() for t in out], n, scale, _over(over), local)
    return out


# ---- rows sorted by cluster and back ---------------------------------------------------------------------------------

def sort_rows(ids, k, align=1):
    """Places of rows sorted by cluster: ids (rows,) or (rows, n) int32, outside [0, k) for entries that go nowhere.  Groups
    start on multiples of `align`; entries of a group keep their order."""
    if not isinstance(ids, torch.Tensor) or not ids.is_cuda or ids.dtype is not torch.int32:
        _refuse("ids", ids, None, torch.int32)
    if ids.dim() == 1:
        ids = ids.unsqueeze(1)
    if ids.dim() != 2:
        raise ValueError("ids must be one- or two-dimensional")
    rows, n = ids.shape
    stride, inner = ids.stride()
    if inner != 1 and n > 1:
        raise ValueError("ids: the elements of a row must lie side by side")
    if not 0 < k <= _INT or not 0 < align <= _INT or n > _INT:
        raise ValueError("k, align and the entries of a row are 1 to %d, not %s, %s and %d" % (_INT, k, align, n))
    index, entries = ids.get_device(), rows * n
    places, work = entries + min(k, entries) * (align - 1), 0
    if entries >= _SORT_ONE_CTA or k > _SORT_KNOWN or align > _SORT_KNOWN:
        capacity, size = ctypes.c_size_t(0), ctypes.c_size_t(0)
        _sizes(_lib.kmeans_sort_rows_sizes, index, rows, n, k, align, ctypes.byref(capacity), ctypes.byref(size))
        places, work = capacity.value, size.value
    offsets = ids.new_empty(k + 1)
    counts = ids.new_empty(k)
    slot = ids.new_empty((rows, n))
    source = ids.new_empty(places)
    ws = ids.new_empty(work, dtype=torch.uint8) if work else None
    _call(_lib.kmeans_sort_rows, index, ids.data_ptr(), stride if rows > 1 else n, rows, n, k, align, offsets.data_ptr(),
          counts.data_ptr(), slot.data_ptr(), source.data_ptr(), ws.data_ptr() if work else None, work)
    return SortedRows(offsets, counts, slot, source)


def _plan(plan, index):
    """(address of slot, address of source, rows, entries a row, places)"""
    slot, source = plan.slot, plan.source
    try:
        rows, n = slot.shape
        places, = source.shape
    except ValueError:
        raise ValueError("plan.slot must be two-dimensional and plan.source one-dimensional") from None
    if n > _INT:
        raise ValueError("a plan of %d entries a row has too many" % n)
    return (_flat("plan.slot", slot, index, torch.int32, slot.shape), _flat("plan.source", source, index, torch.int32, source.shape),
            rows, n, places)


def dispatch(x, plan, out=None):
    """Rows of x (rows, cols) at the places of `plan` (places, cols); padding becomes zero rows.  `out` may have more
    rows than the plan has places: those behind stay as they are."""
    have, cols, stride, code, index = _rows("x", x)
    slot, source, rows, n, places = _plan(plan, index)
    if have != rows:
        raise ValueError("x has %d rows, the plan %d" % (have, rows))
    y, ystride = _out(out, x, index, places, cols, exact=False)
    if x.requires_grad:
        _unrecorded("dispatch")
    _call(_lib.kmeans_dispatch, index, code, x.data_ptr(), stride, rows, cols, n, slot, source, places, y.data_ptr(), ystride)
    return y


def dispatch_grad(drows, plan, out=None):
    """Gradient of :func:`dispatch`: each row's sum over its places."""
    return combine(drows, plan, None, out)


def combine(rows, plan, weights=None, out=None):
    """Sum of each row's entries of the sorted `rows` (places, cols), with weights (rows, n) float32 in any strides or without;
    entries that went nowhere add nothing."""
    have, cols, stride, code, index = _rows("rows", rows)
    slot, _, t, n, places = _plan(plan, index)
    if have < places:
        raise ValueError("rows has %d rows, the plan %d places" % (have, places))
    if weights is not None:
        weights = _per_entry("weights", weights, index, torch.float32, (t, n))
    w = None if weights is None else weights.data_ptr()
    y, ystride = _out(out, rows, index, t, cols, read=places)
    if rows.requires_grad or (weights is not None and weights.requires_grad):
        _unrecorded("combine")
    _call(_lib.kmeans_combine, index, code, rows.data_ptr(), stride, places, cols, slot, w, t, n, y.data_ptr(), ystride)
    return y


def combine_grad(dy, rows, plan, weights):
    """Gradients of :func:`combine` for the sorted rows (zero rows at padding) and the weights."""
    have, cols, stride, code, index = _rows("rows", rows)
    slot, source, t, n, places = _plan(plan, index)
    if have < places:
        raise ValueError("rows has %d rows, the plan %d places" % (have, places))
    dstride = _same_rows("dy", dy, rows, index, (t, cols))
    weights = _per_entry("weights", weights, index, torch.float32, (t, n))
    drows = rows.new_empty((places, cols))
    dweights = torch.empty_like(weights)
    _call(_lib.kmeans_combine_grad, index, code, dy.data_ptr(), dstride, rows.data_ptr(), stride, places, cols, slot, source,
          weights.data_ptr(), t, n, drows.data_ptr(), cols, dweights.data_ptr())
    return CombineGrad(drows, dweights)
