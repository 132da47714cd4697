"""The row operators (h2o4gpu_b200.rows) against their definitions in float64, their refusals, and a run of them together.

Tolerances count roundings.  U = 2^-24 is half a float32 step; a value stored in type t is off by at most `half(t)` of itself.  A sum of
m terms whose partial sums pass through at most L additions is off by at most L U times the sum of the terms' magnitudes; the kernels'
lanes add at most cols / 32 terms each and join 32 lanes and 32 warps in 10 steps, so L = cols / 32 + 12 covers every variant.
"""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

U = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
gpu = pytest.mark.gpu


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Below the smallest normal number the steps no longer shrink with the value (float16: 2^-24 below 2^-14): half of one."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def rows_module(built_lib):
    from h2o4gpu_b200 import rows
    return rows


def randn(shape, seed, dtype=torch.float32, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g, dtype=torch.float64) * scale + shift).to(dtype).cuda()


def within(got, want, tol):
    got, want = got.double().cpu(), want.double().cpu()
    tol = torch.as_tensor(tol, dtype=torch.float64).cpu()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), "%d of %d off, worst %g times the tolerance" % (
        int(bad.sum()), bad.numel(), float(((got - want).abs() / tol.clamp_min(1e-300)).nan_to_num(1e9).max()))


# ---- layer norm ------------------------------------------------------------------------------------------------------

def norm_reference(x, w, b, eps):
    """y, mean, rstd in float64, and how far y, mean and rstd (relative) may be off."""
    xd = x.double()
    d = x.shape[1]
    mean = xd.mean(1)
    xc = xd - mean[:, None]
    rstd = 1.0 / torch.sqrt((xc * xc).mean(1) + eps)
    wd = torch.ones(d, dtype=torch.float64, device=x.device) if w is None else w.double()
    bd = torch.zeros(d, dtype=torch.float64, device=x.device) if b is None else b.double()
    depth = d / 32 + 12
    dmean = depth * U * xd.abs().mean(1) + U * mean.abs()
    # the squares of (x - mean) are off by twice the mean's error beside |x - mean| (whose average is below the deviation), their
    # sum by its additions; the root halves that, the square root and the division add four roundings
    drstd = 0.5 * ((depth + 4) * U + 2 * (dmean + U * xd.abs().amax(1)) * rstd + (dmean * rstd) ** 2) + 4 * U
    xh = xc * rstd[:, None]
    y = xh * wd + bd
    tol = ((dmean + U * xd.abs().amax(1)) * rstd)[:, None] * wd.abs() + (drstd[:, None] + 4 * U) * (xh * wd).abs() + 2 * U * bd.abs()
    return y, mean, rstd, tol + half(x.dtype) * (y.abs() + tol) + tiny(x.dtype) + 1e-30, dmean, drstd * rstd


NORM_SHAPES = [(1, 1), (1, 4096), (3, 7), (5, 1023), (33, 784), (2, 8192), (257, 64), (130, 130), (2, 20000), (1, 70001), (1200, 40)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", NORM_SHAPES, ids=str)
def test_layer_norm(built_lib, shape, dtype):
    R = rows_module(built_lib)
    x = randn(shape, 1, dtype, 2.0, 0.7)
    for params in (None, torch.float32, dtype):
        w = None if params is None else randn(shape[1], 2, params, 0.2, 1.0)
        b = None if params is None else randn(shape[1], 3, params, 0.3)
        out = R.layer_norm(x, w, b)
        y, mean, rstd, tol, dmean, drstd = norm_reference(x, w, b, 1e-5)
        assert out.y.dtype == dtype and out.mean.dtype == torch.float32
        within(out.y, y, tol)
        within(out.mean, mean, dmean + 1e-30)
        within(out.rstd, rstd, drstd)


@gpu
def test_layer_norm_weight_or_bias_alone_and_far_from_zero(built_lib):
    R = rows_module(built_lib)
    x = randn((17, 500), 4, torch.float32, 1.0, 1000.0)      # the mean is a thousand deviations away
    w, b = randn(500, 5), randn(500, 6)
    for w_, b_ in ((w, None), (None, b), (w, b)):
        y, _, _, tol, _, _ = norm_reference(x, w_, b_, 0.25)
        within(R.layer_norm(x, w_, b_, eps=0.25).y, y, tol)
    x[3] = 2.5                                                # a constant row: its norm is the bias
    got = R.layer_norm(x, w, b).y
    assert torch.equal(got[3], b)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_layer_norm_strides_and_alignment(built_lib, dtype):
    R = rows_module(built_lib)
    wide = randn((40, 1100), 7, dtype)
    flat = randn(40 * 513 + 3, 8, dtype)
    w, b = randn(1025, 9, dtype, 0.1, 1.0), randn(1025, 10, dtype)
    views = [wide[:, :1024], wide[:, 1:1025], wide[:, 3:515], wide[::3, 8:520], wide[:1].expand(6, 1100),
             flat[1:1 + 40 * 513].view(40, 513), flat[2:2 + 40 * 512].view(40, 512), wide[5:6]]
    for x in views:
        d = x.shape[1]
        for ww, bb in ((w[:d], b[:d]), (w[1:1 + d], b[1:1 + d])) if d < 1025 else ((None, None),):
            y, _, _, tol, _, _ = norm_reference(x, ww, bb, 1e-5)
            got = R.layer_norm(x, ww, bb)
            within(got.y, y, tol)
            frame = torch.full((x.shape[0] + 2, d + 9), 7.0, dtype=dtype, device="cuda")
            for off in (0, 1, 8):
                frame.fill_(7.0)
                o = frame[1:-1, off:off + d]
                assert R.layer_norm(x, ww, bb, out=o).y.data_ptr() == o.data_ptr()
                assert torch.equal(o, got.y)
                frame[1:-1, off:off + d] = 7.0
                assert bool((frame == 7.0).all())            # nothing beside the rows was written


@gpu
def test_layer_norm_in_place_and_rows_that_are_not_finite(built_lib):
    R = rows_module(built_lib)
    for shape in ((64, 768), (3, 30000), (9, 33)):
        x = randn(shape, 11, torch.bfloat16)
        want = R.layer_norm(x).y
        x[1, 5], x[2, 7] = float("inf"), float("nan")
        y = R.layer_norm(x, out=x).y
        keep = [i for i in range(shape[0]) if i not in (1, 2)]
        assert y.data_ptr() == x.data_ptr()
        assert torch.equal(y[keep], want[keep]) and bool(y[1].isnan().all()) and bool(y[2].isnan().all())


def norm_grad_reference(dy, x, mean, rstd, w):
    dyd, xd = dy.double(), x.double()
    m, r = mean.double()[:, None], rstd.double()[:, None]
    wd = torch.ones(x.shape[1], dtype=torch.float64, device=x.device) if w is None else w.double()
    xh, g = (xd - m) * r, dyd * wd
    m1, m2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    dx = r * (g - m1 - xh * m2)
    depth = x.shape[1] / 32 + 12
    # xh: a difference, a product; g: a product; the two means: their additions; the result: five operations
    axh = xh.abs() + U * (xd.abs() + m.abs()) * r
    tol = U * r * (8 * g.abs() + (depth + 8) * g.abs().mean(1, keepdim=True) + (depth + 12) * axh * (g.abs() * axh).mean(1, keepdim=True))
    tol = tol + r * (U * (xd.abs() + m.abs()) * r) * m2.abs()
    t = x.shape[0]
    dw, db = (dyd * xh).sum(0), dyd.sum(0)
    tw = U * (((t + 16) * dyd.abs() * xh.abs()) + dyd.abs() * (xd.abs() + m.abs()) * r).sum(0)
    return dx, dw, db, tol + half(x.dtype) * (dx.abs() + tol) + tiny(x.dtype) + 1e-30, tw + 1e-30, U * (t + 4) * dyd.abs().sum(0) + 1e-30


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", NORM_SHAPES, ids=str)
def test_layer_norm_grad(built_lib, shape, dtype):
    R = rows_module(built_lib)
    x, dy = randn(shape, 12, dtype, 2.0, 0.7), randn(shape, 13, dtype)
    for params in (None, torch.float32, dtype):
        w = None if params is None else randn(shape[1], 14, params, 0.2, 1.0)
        f = R.layer_norm(x, w)
        got = R.layer_norm_grad(dy, x, f.mean, f.rstd, w)
        dx, dw, db, tol, tw, tb = norm_grad_reference(dy, x, f.mean, f.rstd, w)
        within(got.dx, dx, tol)
        within(got.dweight, dw, tw)
        within(got.dbias, db, tb)
        again = R.layer_norm_grad(dy, x, f.mean, f.rstd, w)
        assert all(torch.equal(a, b) for a, b in zip(got, again))            # sums in a fixed order
        alone = R.layer_norm_grad(dy, x, f.mean, f.rstd, w, params=False)
        assert torch.equal(alone.dx, got.dx) and alone.dweight is None and alone.dbias is None


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_layer_norm_grad_strides(built_lib, dtype):
    R = rows_module(built_lib)
    a, b = randn((50, 1100), 15, dtype), randn((50, 1100), 16, dtype)
    w = randn(1100, 17, dtype, 0.2, 1.0)
    for d, xo, go, wo in ((1024, 0, 0, 0), (1024, 1, 0, 1), (513, 3, 2, 0), (512, 8, 16, 3), (1023, 0, 0, 0)):
        x, dy, ww = a[:, xo:xo + d], b[:, go:go + d], w[wo:wo + d]
        f = R.layer_norm(x, ww)
        for g in (dy, dy[:1].expand(50, d)):
            got = R.layer_norm_grad(g, x, f.mean, f.rstd, ww)
            dx, dw, db, tol, tw, tb = norm_grad_reference(g, x, f.mean, f.rstd, ww)
            within(got.dx, dx, tol)
            within(got.dweight, dw, tw)
            within(got.dbias, db, tb)


@gpu
def test_layer_norm_gradient_against_differences(built_lib):
    """Central differences of the float64 formula: the gradient's formula itself."""
    R = rows_module(built_lib)
    x, w, b, dy = randn((4, 24), 18), randn(24, 19, scale=0.2, shift=1.0), randn(24, 20), randn((4, 24), 21)
    f = R.layer_norm(x, w, b)
    got = R.layer_norm_grad(dy, x, f.mean, f.rstd, w)

    def loss(x_, w_, b_):
        return float((norm_reference(x_, w_, b_, 1e-5)[0] * dy.double()).sum())

    h = 1e-5
    for t, g, at in ((x, got.dx, [(0, 0), (1, 7), (3, 23)]), (w, got.dweight, [(0,), (11,)]), (b, got.dbias, [(5,), (23,)])):
        for i in at:
            args = [x.double(), w.double(), b.double()]
            which = [k for k, v in enumerate((x, w, b)) if v is t][0]
            hi, lo = args[which].clone(), args[which].clone()
            hi[i] += h
            lo[i] -= h
            up = list(args)
            up[which] = hi
            down = list(args)
            down[which] = lo
            num = (loss(*up) - loss(*down)) / (2 * h)
            # truncation h^2 times a third derivative of order ten, cancellation 1e-15 * |loss| / h, float32 roundings of the kernel
            assert abs(num - float(g[i])) <= 1e-8 + 1e-9 + 64 * U * (1 + abs(num)) * 8


# ---- routing ---------------------------------------------------------------------------------------------------------

HUGE = float(np.finfo(np.float32).max)


def route_reference(scores, n, scale, over):
    s = scores.float().cpu().numpy().astype(np.float64)
    up = 1.0 if scale > 0 else -1.0
    q = np.where(np.isnan(s), -np.inf, s * up)
    q = np.minimum(q, HUGE)
    t, k = q.shape
    ids = np.argsort(-q, axis=1, kind="stable")[:, :n]
    top = np.take_along_axis(q, ids, 1)
    there = top > -np.inf
    best = np.where(there[:, :1], top[:, :1], 0.0)
    a = abs(float(np.float32(scale)))
    arg = np.where(there, a * (top - best), 0.0)
    z = np.where(there, np.exp(arg), 0.0)
    allarg = np.where(q > -np.inf, a * (q - best), -np.inf)
    pool = np.exp(allarg) if over == "all" else z
    poolarg = np.where(np.isfinite(allarg), allarg, 0.0) if over == "all" else arg
    total = pool.sum(1, keepdims=True)
    safe = np.where(total > 0, total, 1.0)
    # an argument is off by two roundings of itself, exp by two units in the last place, the sum by its additions
    dpool = ((2 * np.abs(poolarg) + 4) * pool).sum(1, keepdims=True) / safe + pool.shape[1] / 32 + 12
    rel = U * (2 * np.abs(arg) + 4 + dpool + 2)
    return dict(ids=np.where(there, ids, -1), weights=np.where(there, z / safe, 0.0), best=up * best[:, 0], total=total[:, 0],
                wtol=rel * z / safe + 2.0 ** -126, ttol=(U * (dpool + 1) * total + 2.0 ** -126)[:, 0], q=q, a=a, safe=safe,
                base=best, dpool=dpool)


def check_route(R, scores, n, scale, over):
    got = R.route(scores, n, scale, over)
    ref = route_reference(scores, n, scale, over)
    assert np.array_equal(got.ids.cpu().numpy(), ref["ids"])
    within(got.weights, torch.from_numpy(ref["weights"]), torch.from_numpy(ref["wtol"]))
    assert np.array_equal(got.best.double().cpu().numpy(), ref["best"])
    within(got.total, torch.from_numpy(ref["total"]), torch.from_numpy(ref["ttol"]))
    return got, ref


def make_scores(rows, k, dtype, seed, masked=True, low=None):
    s = randn((rows, k), seed, torch.float32, 2.0)
    if masked:
        g = torch.Generator().manual_seed(seed + 1)
        s[torch.rand((rows, k), generator=g).cuda() < 0.1] = float("-inf") if low is None else low
        s[torch.rand((rows, k), generator=g).cuda() < 0.02] = float("nan")
        s[rows // 2:: 7] = float("-inf")
    return s.to(dtype)


ROUTE_SHAPES = [(1, 1, 1), (1, 8, 2), (5, 8, 8), (70, 33, 5), (300, 100, 4), (129, 1000, 8), (9, 4096, 32), (33, 300, 1), (2, 65, 32),
                (1000, 16, 2), (40, 2047, 7), (3, 20000, 3), (65, 256, 16)]


@gpu
@pytest.mark.parametrize("over", ["chosen", "all"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", ROUTE_SHAPES, ids=str)
def test_route(built_lib, shape, dtype, over):
    R = rows_module(built_lib)
    rows, k, n = shape
    s = make_scores(rows, k, dtype, 30)
    check_route(R, s, n, 1.0, over)                                   # row after row
    check_route(R, s.t().contiguous().t(), n, 1.0, over)              # cluster after cluster
    check_route(R, -s, n, -0.7, over)                                 # distances
    check_route(R, (-s).t().contiguous().t(), n, -0.7, over)


@gpu
def test_route_other_strides(built_lib):
    R = rows_module(built_lib)
    wide = make_scores(60, 130, torch.float32, 31)
    for s in (wide[:, 1:100], wide[::2, ::3], wide[5:6], wide[:, 7:8], wide[:1].expand(20, 130), wide.t()[3:40], wide[:, 5:6].expand(60, 9)):
        for over in ("chosen", "all"):
            check_route(R, s, min(3, s.shape[1]), 1.0, over)
    half_ = make_scores(50, 203, torch.bfloat16, 32)
    for s in (half_[:, 1:], half_[:, 3:100], half_.t()[1:]):
        check_route(R, s, 4, 1.0, "all")


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_route_ties_masks_and_infinities(built_lib, dtype):
    R = rows_module(built_lib)
    low, inf, nan = torch.finfo(dtype).min, float("inf"), float("nan")
    s = torch.zeros((12, 40), dtype=dtype, device="cuda")
    s[1] = low                               # all masked by the lowest value: still a score, uniform weights
    s[2] = -inf                              # nothing can be taken
    s[3] = nan
    s[4, :38] = -inf                         # two left for three places
    s[5, 10:] = low
    s[6, 7] = s[6, 21] = inf                 # two infinitely good ones share
    s[7, ::2] = -0.0                         # the two zeros tie
    s[8, 5] = torch.finfo(dtype).max
    s[9] = torch.arange(40, dtype=torch.float32).to(dtype).cuda()
    s[10] = nan
    s[10, 39] = low
    for v in (s, s.t().contiguous().t()):
        for over in ("chosen", "all"):
            got, _ = check_route(R, v, 3, 1.0, over)
            assert got.ids[0].tolist() == [0, 1, 2] and got.ids[1].tolist() == [0, 1, 2] and got.ids[7].tolist() == [0, 1, 2]
            assert got.ids[2].tolist() == [-1] * 3 and got.weights[2].tolist() == [0.0] * 3 and float(got.total[2]) == 0.0
            assert got.ids[3].tolist() == [-1] * 3
            assert got.ids[4].tolist() == [38, 39, -1] and got.weights[4].tolist() == [0.5, 0.5, 0.0]
            assert got.ids[6].tolist() == [7, 21, 0] and got.weights[6].tolist() == [0.5, 0.5, 0.0]
            assert got.ids[10].tolist() == [39, -1, -1] and got.weights[10].tolist() == [1.0, 0.0, 0.0]
            check_route(R, -v, 3, -1e30, over)                         # differences that overflow: all weight on the best


@gpu
@pytest.mark.parametrize("n", [1, 2, 8, 12])
@pytest.mark.parametrize("k", [40, 300, 640, 701, 1500, 5000])
def test_route_of_many_equal_scores(built_lib, k, n):
    """More scores reach the bound than any list holds, in every kernel: equal ones, masks, infinities, two levels."""
    R = rows_module(built_lib)
    for dtype in (torch.float32, torch.bfloat16):
        s = torch.zeros((70, k), dtype=dtype, device="cuda")
        s[1:70:9] = torch.finfo(dtype).min
        s[2:70:9, : k // 2] = 1.0
        s[3:70:9, ::3] = float("inf")
        s[4:70:9] = float("nan")
        s[5:70:9, : k - 3] = float("-inf")
        s[6:70:9] = torch.arange(k, device="cuda").to(dtype)
        s[7:70:9] = (torch.arange(k, device="cuda") % 5).to(dtype)
        s[8:70:9] = -torch.arange(k, device="cuda").to(dtype)
        for v in (s, s.t().contiguous().t(), torch.cat([s, s], 1)[:, 1:k + 1][:, :k], torch.cat([s, s], 0).t().contiguous().t()[1:]):
            for over in ("chosen", "all"):
                check_route(R, v, n, 0.5, over)
                check_route(R, -v, n, -0.5, over)


@gpu
@pytest.mark.parametrize("over", ["chosen", "all"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", ROUTE_SHAPES, ids=str)
def test_route_grad(built_lib, shape, dtype, over):
    R = rows_module(built_lib)
    rows, k, n = shape
    base = make_scores(rows, k, dtype, 33)
    dw = randn((rows, n), 34)
    for s, scale in ((base, 1.0), ((-base).t().contiguous().t(), -0.7)):
        got, ref = check_route(R, s, n, scale, over)
        g = dw.double().cpu().numpy()
        ids, w = ref["ids"], got.weights.double().cpu().numpy()
        g = np.where(ids >= 0, g, 0.0)
        c = (w * g).sum(1, keepdims=True)
        dc = (n + 8) * U * np.abs(w * g).sum(1, keepdims=True)
        G = np.zeros((rows, k + 1))
        W = np.zeros((rows, k + 1))
        np.put_along_axis(G, np.where(ids >= 0, ids, k), g, 1)
        np.put_along_axis(W, np.where(ids >= 0, ids, k), w, 1)
        G, W = G[:, :k], W[:, :k]
        if over == "chosen":
            p, drel = W, 0.0
        else:
            arg = ref["a"] * (ref["q"] - ref["base"])
            tot = got.total.double().cpu().numpy()[:, None]
            p = np.where(np.isfinite(ref["q"]) & (tot > 0), np.exp(arg) / np.where(tot > 0, tot, 1.0), 0.0)
            drel = U * (2 * np.where(np.isfinite(arg), np.abs(arg), 0.0) + 6)
        want = scale * p * (G - c)
        taken = np.zeros((rows, k + 1), bool)
        np.put_along_axis(taken, np.where(ids >= 0, ids, k), True, 1)
        if over == "chosen":
            want = np.where(taken[:, :k], want, 0.0)
        tol = abs(scale) * p * ((drel + 6 * U) * np.abs(G - c) + dc + U * np.abs(G)) + 2.0 ** -126
        tol = tol + half(dtype) * (np.abs(want) + tol) + tiny(dtype)
        ds = R.route_grad(dw, s, got, scale, over)
        assert ds.dtype == dtype and ds.shape == s.shape
        if min(rows, k) > 1:
            assert (ds.stride(0) < ds.stride(1)) == (s.stride(0) < s.stride(1))
        within(ds, torch.from_numpy(want), torch.from_numpy(tol))


@gpu
@pytest.mark.parametrize("over", ["chosen", "all"])
def test_route_gradient_against_differences(built_lib, over):
    R = rows_module(built_lib)
    s, dw = randn((3, 9), 35), randn((3, 4), 36)
    got = R.route(s, 4, -0.6, over)
    ds = R.route_grad(dw, s, got, -0.6, over)
    ids = got.ids.long().cpu()

    def loss(v):
        z = torch.exp(float(np.float32(-0.6)) * v)
        pick = torch.gather(z, 1, ids)
        w = pick / (z if over == "all" else pick).sum(1, keepdim=True)
        return float((w * dw.double().cpu()).sum())

    h = 1e-5
    base = s.double().cpu()
    for i in range(3):
        for e in range(9):
            hi, lo = base.clone(), base.clone()
            hi[i, e] += h
            lo[i, e] -= h
            # truncation h^2, cancellation 1e-15 / h, and a few float32 roundings of values below 4
            assert abs((loss(hi) - loss(lo)) / (2 * h) - float(ds[i, e])) <= 1e-9 + 1e-9 + 64 * U * 4


# ---- sorted rows -----------------------------------------------------------------------------------------------------

def sort_reference(ids, k, align):
    ids = ids.cpu().numpy()
    if ids.ndim == 1:
        ids = ids[:, None]
    flat = ids.reshape(-1).astype(np.int64)
    n_entries = flat.size
    cap = n_entries + min(k, n_entries) * (align - 1)
    offsets, counts = np.zeros(k + 1, np.int64), np.zeros(k, np.int64)
    slot, source = np.full(n_entries, -1, np.int64), np.full(cap, -1, np.int64)
    at = 0
    for e in range(k):
        mine = np.flatnonzero(flat == e)
        offsets[e], counts[e] = at, mine.size
        slot[mine] = at + np.arange(mine.size)
        source[at:at + mine.size] = mine
        at += -(-mine.size // align) * align
    offsets[k] = at
    return offsets, counts, slot.reshape(ids.shape), source


def make_ids(rows, n, k, seed, drop=0.1):
    g = np.random.default_rng(seed)
    p = np.exp(g.standard_normal(k))
    ids = g.choice(k, size=(rows, n), p=p / p.sum()).astype(np.int32)
    ids[g.random((rows, n)) < drop] = -1
    if rows > 4:
        ids[1, 0], ids[2, 0] = k, 2 ** 31 - 1            # beyond the clusters: nowhere as well
        ids[3] = ids[3, 0]                               # the same cluster twice
    return torch.from_numpy(ids).cuda()


SORT_SHAPES = [(1, 1, 1, 1), (1, 2, 8, 1), (16, 2, 8, 16), (100, 3, 7, 128), (5000, 1, 100, 1), (3000, 8, 64, 16), (777, 2, 1000, 1),
               (2000, 4, 4096, 2), (500, 2, 16384, 3), (40000, 2, 3, 128), (30, 1, 600, 1), (9000, 5, 300, 1)]


@gpu
@pytest.mark.parametrize("shape", SORT_SHAPES, ids=str)
def test_sort_rows(built_lib, shape):
    R = rows_module(built_lib)
    rows, n, k, align = shape
    for drop in (0.0, 0.2, 1.0):
        ids = make_ids(rows, n, k, 40, drop)
        plan = R.sort_rows(ids, k, align)
        for got, want in zip(plan, sort_reference(ids, k, align)):
            assert got.dtype == torch.int32 and np.array_equal(got.cpu().numpy(), want)


@gpu
def test_sort_rows_of_labels_and_strided_ids(built_lib):
    R = rows_module(built_lib)
    ids = make_ids(700, 6, 20, 41)
    for v in (ids[:, 0].contiguous(), ids[:, 0], ids[:, 1:4], ids[::3, 2:5], ids[:1].expand(50, 6)):
        for got, want in zip(R.sort_rows(v, 20, 4), sort_reference(v, 20, 4)):
            assert np.array_equal(got.cpu().numpy(), want)


MOVE_SHAPES = [(1, 1, 1, 1, 1), (1, 2, 8, 1024, 1), (16, 2, 8, 1023, 1), (100, 3, 7, 784, 16), (257, 8, 64, 64, 1), (300, 1, 20, 33, 4),
               (50, 4, 4096, 130, 1), (37, 2, 5, 4100, 2), (64, 33, 40, 96, 1), (9, 2, 3, 20000, 1), (130, 5, 12, 1021, 1)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", MOVE_SHAPES, ids=str)
def test_dispatch_and_combine(built_lib, shape, dtype):
    R = rows_module(built_lib)
    rows, n, k, d, align = shape
    for drop in (0.0, 0.3, 1.0):
        ids = make_ids(rows, n, k, 42, drop)
        plan = R.sort_rows(ids, k, align)
        src, slot = plan.source.long(), plan.slot.long()
        x = randn((rows, d), 43, dtype)
        got = R.dispatch(x, plan)
        want = torch.where(src[:, None] >= 0, x[src.clamp(min=0) // n], torch.zeros((), dtype=dtype, device="cuda"))
        assert torch.equal(got, want)

        e = randn((src.shape[0], d), 44, dtype)
        e[src < 0] = float("nan")                                   # padding rows are never read
        w = randn((rows, n), 45)
        w[slot < 0] = float("nan")                                  # nor are weights of entries that go nowhere
        picked = torch.where(slot[:, :, None] >= 0, e.double()[slot.clamp(min=0)], 0.0)
        wz = torch.where(slot >= 0, w, 0.0).double()
        for weights, ww in ((w, wz), (None, (slot >= 0).double())):
            y = (picked * ww[:, :, None]).sum(1)
            tol = (n + 1) * U * (picked * ww[:, :, None]).abs().sum(1)
            out = R.combine(e, plan, weights)
            within(out, y, tol + half(dtype) * (y.abs() + tol) + tiny(dtype))
            if weights is None:
                assert torch.equal(R.dispatch_grad(e, plan), out)

        dy = randn((rows, d), 46, dtype)
        drows, dweights = R.combine_grad(dy, e, plan, w)
        g = torch.where(src[:, None] >= 0, dy.double()[src.clamp(min=0) // n] * wz.reshape(-1)[src.clamp(min=0)][:, None], 0.0)
        within(drows, g, (half(dtype) + 2 * U) * g.abs() + tiny(dtype))
        dots = (picked * dy.double()[:, None, :]).sum(2)
        within(dweights, dots, (d / 32 + 12) * U * (picked * dy.double()[:, None, :]).abs().sum(2) + 1e-30)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_dispatch_and_combine_strides(built_lib, dtype):
    R = rows_module(built_lib)
    rows, n, k, align = 61, 3, 9, 4
    ids = make_ids(rows, n, k, 47, 0.1)
    plan = R.sort_rows(ids, k, align)
    cap = plan.source.shape[0]
    w = randn((rows, n), 48)
    x, e, dy = randn((rows, 700), 49, dtype), randn((cap + 3, 700), 50, dtype), randn((rows, 700), 51, dtype)
    frame = torch.full((cap + 5, 720), 5.0, dtype=dtype, device="cuda")
    for d, xo, eo, oo in ((512, 0, 0, 0), (512, 1, 0, 0), (512, 0, 3, 8), (333, 1, 2, 3), (640, 8, 16, 1), (100, 2, 2, 2)):
        xs, es, gs = x[:, xo:xo + d], e[:, eo:eo + d], dy[:, xo:xo + d]
        plain = R.dispatch(xs.contiguous(), plan)
        frame.fill_(5.0)
        out = frame[1:, oo:oo + d]
        assert torch.equal(R.dispatch(xs, plan, out=out)[:cap], plain)
        frame[1:1 + cap, oo:oo + d] = 5.0
        assert bool((frame == 5.0).all())                           # rows behind the places and columns beside stay as they were
        assert torch.equal(R.dispatch(xs, plan), plain)
        y = R.combine(es[:cap].contiguous(), plan, w)
        assert torch.equal(R.combine(es, plan, w), y)
        frame.fill_(5.0)
        R.combine(es, plan, w, out=frame[2:2 + rows, oo:oo + d])
        assert torch.equal(frame[2:2 + rows, oo:oo + d], y)
        frame[2:2 + rows, oo:oo + d] = 5.0
        assert bool((frame == 5.0).all())
        a, b = R.combine_grad(gs, es, plan, w), R.combine_grad(gs.contiguous(), es[:cap].contiguous(), plan, w)
        assert torch.equal(a.drows, b.drows)
        bound = (d / 32 + 12) * U * (e.double().abs().max() * gs.double().abs().sum(1, keepdim=True))
        within(a.dweights, b.dweights, 2 * bound.expand(rows, n))
        one = dy[:1, xo:xo + d].expand(rows, d)                     # a gradient that every row shares
        assert torch.equal(R.combine_grad(one, es, plan, w).drows, R.combine_grad(one.contiguous(), es, plan, w).drows)


@gpu
def test_combine_gradient_against_differences(built_lib):
    R = rows_module(built_lib)
    ids = make_ids(6, 2, 3, 52, 0.2)
    plan = R.sort_rows(ids, 3, 2)
    e, w, dy = randn((plan.source.shape[0], 5), 53), randn((6, 2), 54), randn((6, 5), 55)
    got = R.combine_grad(dy, e, plan, w)
    slot = plan.slot.long()

    def loss(e_, w_):
        picked = torch.where(slot[:, :, None] >= 0, e_[slot.clamp(min=0)], 0.0)
        return float(((picked * w_[:, :, None]).sum(1) * dy.double()).sum())

    h = 1e-4                                                        # the loss is linear in each: no truncation
    for t, g in ((0, got.drows), (1, got.dweights)):
        args = [e.double(), w.double()]
        for i in [(r, c) for r in range(args[t].shape[0]) for c in range(args[t].shape[1])]:
            hi, lo = [v.clone() for v in args], [v.clone() for v in args]
            hi[t][i] += h
            lo[t][i] -= h
            assert abs((loss(*hi) - loss(*lo)) / (2 * h) - float(g[i])) <= 1e-10 + 32 * U * 16


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_rows_at_the_edges_of_their_memory(built_lib, dtype):
    """Rows that start and end anywhere within 16 bytes, in memory that NaN surrounds: nothing beside them counts, nothing beside the
    outputs is written."""
    R = rows_module(built_lib)
    for d in (1, 2, 3, 5, 7, 8, 9, 15, 17, 31, 33, 255, 257, 1025, 2049):
        for start in (0, 1, 3, 7):
            for rows in (1, 2, 5):
                def at(seed, count):
                    buf = torch.full((count * d + 32,), float("nan"), dtype=dtype, device="cuda")
                    view = buf[8 + start:8 + start + count * d].view(count, d)
                    view.copy_(randn((count, d), seed, dtype))
                    return view
                def clean(view):
                    base = torch.full((view.shape[0] * d + 32,), 9.0, dtype=dtype, device="cuda")
                    return base, base[8 + (start * 3) % 8:][:view.shape[0] * d].view(view.shape)
                x, dy = at(180, rows), at(181, rows)
                f = R.layer_norm(x)
                y, _, _, tol, _, _ = norm_reference(x, None, None, 1e-5)
                within(f.y, y, tol)
                base, o = clean(x)
                R.layer_norm(x, out=o)
                assert torch.equal(o, f.y)
                o.fill_(9.0)
                assert bool((base == 9.0).all())
                g = R.layer_norm_grad(dy, x, f.mean, f.rstd)
                dx, dw, db, tol, tw, tb = norm_grad_reference(dy, x, f.mean, f.rstd, None)
                within(g.dx, dx, tol)
                within(g.dweight, dw, tw)
                n = 2
                ids = torch.arange(rows * n, device="cuda", dtype=torch.int32).view(rows, n) % 3
                plan = R.sort_rows(ids, 3)
                e = at(182, rows * n)
                w = randn((rows, n), 183)
                slot = plan.slot.long()
                base, o = clean(e)
                R.dispatch(x, plan, out=o)
                assert torch.equal(o[slot], x[:, None, :].expand(rows, n, d))
                o.fill_(9.0)
                assert bool((base == 9.0).all())
                picked = e.double()[slot] * w.double()[:, :, None]
                base, o = clean(x)
                R.combine(e, plan, w, out=o)
                tol = (n + 1) * U * picked.abs().sum(1)
                within(o, picked.sum(1), tol + half(dtype) * (picked.sum(1).abs() + tol) + tiny(dtype))
                o.fill_(9.0)
                assert bool((base == 9.0).all())
                drows, dwt = R.combine_grad(dy, e, plan, w)
                want = dy.double()[:, None, :] * w.double()[:, :, None]
                within(drows[slot], want, (half(dtype) + 2 * U) * want.abs() + tiny(dtype))
                dots = e.double()[slot] * dy.double()[:, None, :]
                within(dwt, dots.sum(2), (d / 32 + 12) * U * dots.abs().sum(2) + 1e-30)
                if d > 1:
                    sc = at(184, rows)
                    got, _ = check_route(R, sc, min(2, d), 1.0, "all")
                    ds = R.route_grad(torch.ones_like(got.weights), sc, got, 1.0, "all")
                    assert bool(ds.isfinite().all())


@gpu
def test_places_that_no_plan_gives_are_skipped(built_lib):
    R = rows_module(built_lib)
    slot = torch.tensor([[0, 5], [2 ** 31 - 1, -7], [1, 99]], dtype=torch.int32, device="cuda")
    source = torch.tensor([0, 4, -1, -1], dtype=torch.int32, device="cuda")
    plan = R.SortedRows(None, None, slot, source)
    x = randn((3, 40), 56)
    frame = torch.full((12, 40), 3.0, device="cuda")
    got = R.dispatch(x, plan, out=frame)
    assert torch.equal(got[0], x[0]) and torch.equal(got[1], x[2]) and bool((got[2:4] == 0).all()) and bool((got[4:] == 3).all())
    y = R.combine(frame[:4], plan)
    assert torch.equal(y[0], x[0]) and bool((y[1] == 0).all()) and torch.equal(y[2], x[2])
    drows, dw = R.combine_grad(x, frame[:4], plan, torch.ones((3, 2), device="cuda"))
    assert torch.equal(drows[0], x[0]) and torch.equal(drows[1], x[2]) and bool((drows[2:] == 0).all())
    assert dw[1].tolist() == [0.0, 0.0] and float(dw[0, 1]) == 0.0 and float(dw[2, 1]) == 0.0


# ---- how they are called ---------------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_no_rows(built_lib, dtype):
    R = rows_module(built_lib)
    x = torch.empty((0, 64), dtype=dtype, device="cuda")
    f = R.layer_norm(x)
    assert f.y.shape == (0, 64)
    g = R.layer_norm_grad(x, x, f.mean, f.rstd)
    assert bool((g.dweight == 0).all()) and bool((g.dbias == 0).all())
    s = torch.empty((0, 9), dtype=dtype, device="cuda")
    r = R.route(s, 2)
    assert r.ids.shape == (0, 2) and R.route_grad(r.weights, s, r).shape == (0, 9)
    plan = R.sort_rows(r.ids, 9, 8)
    assert plan.offsets.tolist() == [0] * 10 and plan.counts.tolist() == [0] * 9 and plan.source.shape == (0,)
    xs = R.dispatch(x, plan)
    assert xs.shape == (0, 64) and R.combine(xs, plan, r.weights).shape == (0, 64)
    assert R.combine_grad(x, xs, plan, r.weights).drows.shape == (0, 64)


def a_layer(R, x, w, b, s, dy):
    """Every operator once, as one pass of a layer and its gradient use them; all results."""
    f = R.layer_norm(x, w, b)
    r = R.route(s, 2, 1.0, "all")
    plan = R.sort_rows(r.ids, s.shape[1], 8)
    xs = R.dispatch(f.y, plan)
    y = R.combine(xs, plan, r.weights)
    g = R.combine_grad(dy, xs, plan, r.weights)
    ds = R.route_grad(g.dweights, s, r, 1.0, "all")
    n = R.layer_norm_grad(R.dispatch_grad(g.drows, plan), x, f.mean, f.rstd, w)
    return (*f, *r, *plan, xs, y, *g, ds, *n)


def layer_inputs(seed, rows=3000, d=200, k=12):
    return (randn((rows, d), seed, torch.bfloat16), randn(d, seed + 1, scale=0.1, shift=1.0), randn(d, seed + 2),
            make_scores(rows, k, torch.float32, seed + 3), randn((rows, d), seed + 4, torch.bfloat16))


@gpu
def test_layer_on_other_streams_at_once(built_lib):
    R = rows_module(built_lib)
    inputs = [layer_inputs(60), layer_inputs(70)]
    want = [a_layer(R, *v) for v in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(a_layer(R, *inputs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))


@gpu
def test_layer_captured_in_two_graphs(built_lib):
    """Two captured layers replayed one after the other and at once: each has outputs and workspaces of its own."""
    R = rows_module(built_lib)
    inputs = [layer_inputs(80), layer_inputs(90)]
    fresh = [layer_inputs(100), layer_inputs(110)]
    a_layer(R, *inputs[0])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for v in inputs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(a_layer(R, *v))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for values in (inputs, fresh):
        for v, f in zip(inputs, values):
            for a, b in zip(v, f):
                a.copy_(b)
        torch.cuda.synchronize()
        for _ in range(3):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        for v, out in zip(values, outs):
            assert all(torch.equal(a, b) for a, b in zip(out, a_layer(R, *v)))
            torch.cuda.synchronize()


@gpu
def test_captured_without_a_call_before(built_lib):
    """A process whose first calls of the operators are captured ones."""
    import subprocess
    import sys
    code = """
import sys
sys.path[:0] = [%r, %r]
import torch
from h2o4gpu_b200 import rows as R
from test_rows import a_layer, layer_inputs
v = layer_inputs(60)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = a_layer(R, *v)
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, a_layer(R, *v)))
print("as captured")
"""
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code % (root, os.path.join(root, "tests"))], capture_output=True, text=True, timeout=300,
                       cwd=root)
    assert r.returncode == 0 and "as captured" in r.stdout, r.stderr[-2000:]


@gpu
def test_more_than_32_bits_of_elements(built_lib):
    """Rows behind the 2^31st and 2^32nd byte and element come out as they do by themselves."""
    R = rows_module(built_lib)
    rows, d = 270_001, 8192                                   # 2.2e9 elements, 4.4 GB
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB of free memory")
    x = torch.empty((rows, d), dtype=torch.bfloat16, device="cuda")
    x[:] = randn((1, d), 160, torch.bfloat16)
    pick = torch.tensor([0, 131_071, 131_072, 262_143, 262_144, 262_145, 270_000], device="cuda")
    x[pick] = randn((7, d), 161, torch.bfloat16)
    small = x[pick]
    y = R.layer_norm(x)
    want = R.layer_norm(small)
    assert torch.equal(y.y[pick], want.y) and torch.equal(y.mean[pick], want.mean)
    g = R.layer_norm_grad(x, x, y.mean, y.rstd, params=False).dx[pick]
    assert torch.equal(g, R.layer_norm_grad(small, small, want.mean, want.rstd, params=False).dx)
    del y, g
    ids = (torch.arange(rows, device="cuda", dtype=torch.int32) % 3).unsqueeze(1)
    plan = R.sort_rows(ids, 3)
    xs = R.dispatch(x, plan)
    assert torch.equal(xs[plan.slot[pick, 0].long()], small)
    assert torch.equal(R.dispatch_grad(xs, plan)[pick], small)
    w = torch.ones((rows, 1), device="cuda")
    dx, dw = R.combine_grad(x, xs, plan, w)
    assert torch.equal(dx[plan.slot[pick, 0].long()], small)
    square = (small.double() ** 2).sum(1)
    within(dw[pick, 0], square, (d / 32 + 12) * U * square)
    del xs, dx, x
    torch.cuda.empty_cache()
    k = 9000
    s = torch.full((250_000, k), -5.0, dtype=torch.float16, device="cuda")        # 2.25e9 scores
    best = torch.tensor([0, 119_304, 238_609, 249_999], device="cuda")
    s[best, torch.tensor([5, 8999, 0, 77], device="cuda")] = 3.0
    for v in (s, s.view(k, 250_000).t()):
        if v is not s:
            s.fill_(-5.0)
            v[best, torch.tensor([5, 8999, 0, 77], device="cuda")] = 3.0
        r = R.route(v, 1, 1.0)
        assert r.ids[best, 0].tolist() == [5, 8999, 0, 77] and int((r.ids != 0).sum()) == 3
        ds = R.route_grad(torch.ones_like(r.weights), v, r, 1.0)
        assert ds.stride() == v.stride() and not bool(ds[best].any())            # one chosen: its weight is one whatever the score
        del ds, r
        r2 = R.route(v, 2, 1.0, "all")
        assert r2.ids[best, 0].tolist() == [5, 8999, 0, 77]
        ds = R.route_grad(torch.ones_like(r2.weights), v, r2, 1.0, "all")
        few = R.route_grad(torch.ones((4, 2), device="cuda"), v[best].contiguous(),
                           R.Routes(*[t[best].contiguous() for t in r2]), 1.0, "all")
        # the same float32 value, but for a few roundings, rounded once on either side
        assert bool(((ds[best] - few).float().abs() <= 4 * half(torch.float16) * few.float().abs() + 2 * tiny(torch.float16)).all())
        del ds, r2


@gpu
def test_route_with_the_largest_scales(built_lib):
    R = rows_module(built_lib)
    s = make_scores(40, 200, torch.float32, 170, masked=False)
    s[:, 7] = s[:, 3]
    for scale in (HUGE, -HUGE, 2.0 ** -126):
        for n in (1, 4, 12):
            for over in ("chosen", "all"):
                for v in (s, s.t().contiguous().t()):
                    check_route(R, v, n, scale, over)


@gpu
def test_layer_on_another_device_than_the_current_one(built_lib):
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two devices")
    R = rows_module(built_lib)
    v = layer_inputs(120)
    want = a_layer(R, *v)
    got = a_layer(R, *[t.to("cuda:1") for t in v])
    assert torch.cuda.current_device() == 0
    assert all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(got, want))


@gpu
@pytest.mark.parametrize("shape", [(5000, 64, 100, 4), (777, 50, 12, 3), (3000, 128, 300, 8)], ids=str)
@pytest.mark.parametrize("batch_rows", [None, 256])
def test_nearest_equals_transform_and_route(built_lib, monkeypatch, shape, batch_rows):
    """The handle's own path: the same distances as transform gives, the same choice as route makes of them."""
    from h2o4gpu_b200 import ResidentKMeans
    R = rows_module(built_lib)
    if batch_rows:
        monkeypatch.setenv("H2O4GPU_KM_TRANSFORM_BATCH_ROWS", str(batch_rows))
    rows, d, k, n = shape
    X = randn((rows, d), 130, torch.float32, 3.0)
    h = ResidentKMeans()
    with pytest.raises(RuntimeError):
        R.nearest(h, n)                                            # nothing attached
    h.attach_device(0, X.data_ptr(), rows, d)
    h.set_centroids(X[torch.randperm(rows, generator=torch.Generator().manual_seed(1))[:k]].cpu().numpy())
    D = torch.from_numpy(np.ascontiguousarray(h.transform().T)).cuda().t()
    for over in ("chosen", "all"):
        # (the blocks lie otherwise than D: the sums' order may differ, each is as near the definition as route's)
        got, ref = R.nearest(h, n, -0.02, over), route_reference(D, n, -0.02, over)
        assert np.array_equal(got.ids.cpu().numpy(), ref["ids"]) and np.array_equal(got.best.double().cpu().numpy(), ref["best"])
        within(got.weights, torch.from_numpy(ref["weights"]), torch.from_numpy(ref["wtol"]))
        within(got.total, torch.from_numpy(ref["total"]), torch.from_numpy(ref["ttol"]))
    h.assign()
    labels = torch.from_numpy(h.labels()).cuda()
    near = R.nearest(h, 1).ids[:, 0]
    far = torch.cdist(X.double(), torch.from_numpy(h.centroids()).cuda().double()) ** 2
    two = torch.topk(far, 2, dim=1, largest=False).values
    clear = (two[:, 1] - two[:, 0]) > 1e-4 * (X.double() ** 2).sum(1)
    assert torch.equal(near[clear], labels[clear]) and clear.float().mean() > 0.9
    for bad in (0, k + 1):
        with pytest.raises(RuntimeError):
            R.nearest(h, bad)
    h.close()
    h64 = ResidentKMeans(dtype=np.float64)
    h64.upload(X[:100].double().cpu().numpy())
    h64.set_centroids(X[:4].double().cpu().numpy())
    with pytest.raises(RuntimeError, match="float32 handles"):
        R.nearest(h64, 2)
    h64.close()


@gpu
def test_a_layer_of_experts_behind_a_fitted_model(built_lib):
    """As they are used: rows are normed, a k-means model fitted on them routes them, each cluster's expert sees its rows, and the
    results come back; then the gradients.  Against float64 autograd on the same choice of clusters."""
    from h2o4gpu_b200 import ResidentKMeans
    R = rows_module(built_lib)
    rows, d, k, n, tau = 1500, 48, 6, 2, 40.0
    x = randn((rows, d), 140, torch.float32, 1.0) * torch.exp(randn((rows, 1), 141))     # lengths that differ
    w, b = randn(d, 142, scale=0.1, shift=1.0), randn(d, 143, scale=0.1)
    E = randn((k, d, d), 144, scale=d ** -0.5)
    dy = randn((rows, d), 145)
    f = R.layer_norm(x, w, b)
    torch.cuda.synchronize()
    h = ResidentKMeans()
    h.attach_device(0, f.y.data_ptr(), rows, d)
    h.fit(f.y[:k].cpu().numpy(), 5)
    C = torch.from_numpy(h.centroids()).cuda()
    r = R.nearest(h, n, -1.0 / tau)
    h.close()
    plan = R.sort_rows(r.ids, k, 16)
    xs = R.dispatch(f.y, plan)
    starts = plan.offsets.tolist()
    out = torch.zeros_like(xs)
    for e in range(k):
        out[starts[e]:starts[e + 1]] = xs[starts[e]:starts[e + 1]].double().matmul(E[e].double()).float()
    y = R.combine(out, plan, r.weights)

    dout, dweights = R.combine_grad(dy, out, plan, r.weights)
    dxs = torch.zeros_like(xs)
    for e in range(k):
        dxs[starts[e]:starts[e + 1]] = dout[starts[e]:starts[e + 1]].double().matmul(E[e].double().t()).float()
    dist = torch.cdist(f.y.double(), C.double()).square().float()
    routes = R.Routes(r.ids, r.weights, r.best, r.total)
    dd = R.route_grad(dweights, dist, routes, -1.0 / tau).double()
    dfy = R.dispatch_grad(dxs, plan).double() + 2 * (dd.sum(1, keepdim=True) * f.y.double() - dd @ C.double())
    g = R.layer_norm_grad(dfy.float(), x, f.mean, f.rstd, w)

    xd, wd, bd = (t.double().requires_grad_() for t in (x, w, b))
    norm = (xd - xd.mean(1, keepdim=True)) / torch.sqrt(xd.var(1, correction=0, keepdim=True) + 1e-5) * wd + bd
    d2 = (norm[:, None, :] - C.double()[None]).square().sum(2)
    logit = torch.gather(-d2 / tau, 1, r.ids.long())
    weights = torch.softmax(logit, 1)
    each = torch.einsum("td,edf->tef", norm, E.double())
    want = (torch.gather(each, 1, r.ids.long()[:, :, None].expand(-1, -1, d)) * weights[:, :, None]).sum(1)
    want.backward(dy.double())
    # a chain of some ten float32 sums of up to 48 terms, each off by at most 48 + 12 roundings of its terms' magnitudes, which are
    # below 2.5 times the largest result: 1500 roundings; over 1500 rows of either sign the magnitudes add up to sqrt(1500) < 40
    # times the result
    for got, ref, times in ((y, want.detach(), 1), (g.dx, xd.grad, 1), (g.dweight, wd.grad, 40), (g.dbias, bd.grad, 40)):
        assert float((got.double() - ref).abs().max()) <= times * 1500 * U * float(ref.abs().max())


# ---- refusals --------------------------------------------------------------------------------------------------------

def test_python_refuses_what_is_not_on_a_gpu(built_lib):
    R = rows_module(built_lib)
    x, ids = torch.zeros((4, 8)), torch.zeros((4, 2), dtype=torch.int32)
    plan = R.SortedRows(ids[0], ids[0], ids, ids.view(-1))
    for call in (lambda: R.layer_norm(x), lambda: R.layer_norm_grad(x, x, x[0], x[0]), lambda: R.route(x, 2),
                 lambda: R.route_grad(x, x, None), lambda: R.sort_rows(ids, 3), lambda: R.dispatch(x, plan),
                 lambda: R.combine(x, plan), lambda: R.combine_grad(x, x, plan, x), lambda: R.sort_rows([1, 2], 3)):
        with pytest.raises(ValueError, match="must be a CUDA tensor"):
            call()


def test_c_refuses_bad_arguments_before_any_device_call(built_lib):
    """KM_EINVAL without a GPU, for pointers that are never dereferenced."""
    from h2o4gpu_b200.libs import lib_kmeans
    lib = lib_kmeans.cdll()
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4097)
    size = ctypes.c_size_t()
    nan = float("nan")

    def norm(dtype=0, x=p, xs=8, rows=4, cols=8, w=None, b=None, pd=0, eps=1e-5, y=p, ys=8, mean=p, rstd=p):
        return lib.kmeans_layer_norm(dtype, x, xs, rows, cols, w, b, pd, eps, y, ys, mean, rstd, None)

    def norm_grad(dtype=0, dy=p, x=p, rows=4, cols=8, w=None, pd=0, dx=p, dxs=8, dw=p, db=p, ws=p, wb=1 << 30, mean=p):
        return lib.kmeans_layer_norm_grad(dtype, dy, 8, x, 8, mean, p, rows, cols, w, pd, dx, dxs, dw, db, ws, wb, None)

    def route(dtype=0, s=p, rs=8, cs=1, rows=4, k=8, n=2, scale=1.0, ids=p, w=p, best=p, total=p):
        return lib.kmeans_route(dtype, s, rs, cs, rows, k, n, scale, 0, ids, w, best, total, None)

    def route_grad(dtype=0, dw=p, s=p, k=8, n=2, scale=1.0, over=1, ids=p, ds=p, drs=8, dcs=1, best=p):
        return lib.kmeans_route_grad(dtype, dw, s, 8, 1, 4, k, n, scale, over, ids, p, best, p, ds, drs, dcs, None)

    def sort(ids=p, stride=2, rows=4, n=2, k=8, align=1, off=p, cnt=p, slot=p, src=p):
        return lib.kmeans_sort_rows(ids, stride, rows, n, k, align, off, cnt, slot, src, p, 1 << 20, None)

    def dispatch(dtype=0, x=p, xs=8, rows=4, cols=8, n=2, slot=p, src=p, cap=8, out=p, os_=8):
        return lib.kmeans_dispatch(dtype, x, xs, rows, cols, n, slot, src, cap, out, os_, None)

    def combine(dtype=0, e=p, es=8, cap=8, cols=8, slot=p, w=p, rows=4, n=2, y=p, ys=8):
        return lib.kmeans_combine(dtype, e, es, cap, cols, slot, w, rows, n, y, ys, None)

    def combine_grad(dtype=0, dy=p, e=p, cap=8, cols=8, slot=p, src=p, w=p, rows=4, n=2, de=p, des=8, dw=p):
        return lib.kmeans_combine_grad(dtype, dy, 8, e, 8, cap, cols, slot, src, w, rows, n, de, des, dw, None)

    big = 1 << 40
    bad = [norm(dtype=1), norm(dtype=3), norm(dtype=99), norm(x=None), norm(x=odd), norm(xs=-1), norm(cols=0), norm(ys=7), norm(y=None),
           norm(w=p, pd=2), norm(w=odd), norm(eps=-1.0), norm(eps=nan), norm(eps=float("inf")), norm(eps=1e300), norm(rows=big), norm(cols=big),
           norm(mean=odd), norm(xs=big),
           norm_grad(dtype=1), norm_grad(dy=None), norm_grad(dw=None), norm_grad(dx=odd), norm_grad(dxs=4), norm_grad(mean=None),
           norm_grad(rows=big), norm_grad(w=p, pd=11),
           lib.kmeans_layer_norm_grad_workspace(4, 0, ctypes.byref(size)), lib.kmeans_layer_norm_grad_workspace(4, 8, None),
           route(dtype=4), route(s=None), route(rs=-1), route(n=0), route(n=9), route(n=33, k=100), route(k=0), route(scale=0.0),
           route(scale=nan), route(ids=None), route(w=odd), route(best=None), route(total=None), route(rows=big),
           route_grad(dw=None), route_grad(s=None), route_grad(best=None), route_grad(ds=None), route_grad(drs=7), route_grad(drs=2, dcs=8),
           route_grad(drs=1, dcs=3), route_grad(n=0), route_grad(scale=float("inf")),
           sort(ids=None), sort(stride=-1), sort(n=0), sort(k=0), sort(k=16385), sort(align=0), sort(rows=1 << 30), sort(align=1 << 30),
           sort(off=None), sort(cnt=None), sort(slot=None), sort(src=odd),
           lib.kmeans_sort_rows_sizes(4, 2, 8, 0, ctypes.byref(size), ctypes.byref(size)),
           lib.kmeans_sort_rows_sizes(4, 2, 8, 1, None, ctypes.byref(size)),
           dispatch(dtype=7), dispatch(x=None), dispatch(xs=-8), dispatch(cols=0), dispatch(n=0), dispatch(slot=None), dispatch(src=None),
           dispatch(cap=big), dispatch(out=None), dispatch(os_=7), dispatch(rows=1 << 30, n=4),
           combine(dtype=8), combine(e=None), combine(cap=big), combine(slot=odd), combine(w=odd), combine(y=None), combine(ys=3), combine(n=0),
           combine_grad(dtype=9), combine_grad(dy=None), combine_grad(e=None), combine_grad(src=None), combine_grad(w=None),
           combine_grad(de=None), combine_grad(des=2), combine_grad(dw=None)]
    assert [i for i, rc in enumerate(bad) if rc != -1] == []
    assert lib.kmeans_nearest_resident(None, 0, 1, 1.0, 0, p, p, p, p) == -1
    # sizes need no device while one CTA or none does the work
    assert lib.kmeans_sort_rows_sizes(0, 2, 8, 4, ctypes.byref(size), ctypes.byref(ctypes.c_size_t())) == 0 and size.value == 0
    # no rows: nothing to do, nothing is asked of a device
    assert norm(rows=0, x=None, y=None) == 0 and route(rows=0, s=None) == 0 and dispatch(rows=0, cap=0, x=None, out=None) == 0


def test_bfloat16_is_not_a_matrix_type_of_the_engine(built_lib):
    from h2o4gpu_b200 import engine
    assert 11 not in engine.DTYPE_CODES.values()


@gpu
def test_python_refuses_bad_arguments(built_lib):
    R = rows_module(built_lib)
    x = randn((6, 8), 150)
    ids = torch.zeros((6, 2), dtype=torch.int32, device="cuda")
    plan = R.sort_rows(ids, 3)
    f = R.layer_norm(x)
    w = randn(8, 151)
    r = R.route(x, 2)
    e = R.dispatch(x, plan)
    wt = torch.ones((6, 2), device="cuda")
    bad = [lambda: R.layer_norm(x[0]), lambda: R.layer_norm(x.double()), lambda: R.layer_norm(x.t()), lambda: R.layer_norm(x, w[:7]),
           lambda: R.layer_norm(x, w.half()), lambda: R.layer_norm(x.half(), w, w.half()), lambda: R.layer_norm(x, w.cpu()),
           lambda: R.layer_norm(x, out=x[:5]), lambda: R.layer_norm(x, out=x.half()), lambda: R.layer_norm(x, eps=-1.0),
           lambda: R.layer_norm(x, randn(16, 1)[::2]), lambda: R.layer_norm(x, out=x[:1].expand(6, 8)),
           lambda: R.layer_norm_grad(x.half(), x, f.mean, f.rstd), lambda: R.layer_norm_grad(x[:5], x, f.mean, f.rstd),
           lambda: R.layer_norm_grad(x, x, f.mean[:5], f.rstd), lambda: R.layer_norm_grad(x, x, f.mean.half(), f.rstd),
           lambda: R.route(x.double(), 2), lambda: R.route(x, 9), lambda: R.route(x, 0), lambda: R.route(x, 2, 0.0),
           lambda: R.route(x, 2, float("nan")), lambda: R.route(x, 2, 1.0, "some"), lambda: R.route(x[0], 2),
           lambda: R.route_grad(wt[:, :1], x, r), lambda: R.route_grad(wt.half(), x, r), lambda: R.route_grad(wt, x[:5], r),
           lambda: R.sort_rows(ids.long(), 3), lambda: R.sort_rows(ids, 0), lambda: R.sort_rows(ids, 20000), lambda: R.sort_rows(ids, 3, 0),
           lambda: R.sort_rows(ids.t(), 3),
           lambda: R.dispatch(x[:5], plan), lambda: R.dispatch(x, plan, out=e[:11]), lambda: R.dispatch(x, plan, out=e.half()),
           lambda: R.combine(e[:11], plan), lambda: R.combine(e, plan, wt[:5]), lambda: R.combine(e, plan, wt.half()),
           lambda: R.combine(e.double(), plan), lambda: R.combine_grad(x.half(), e, plan, wt), lambda: R.combine_grad(x, e, plan, wt.t())]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError)):
            call()
            pytest.fail("call %d was not refused" % i)
