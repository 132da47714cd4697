"""Calls of the row operators (h2o4gpu_b200.rows) that their documentation allows and that need care.  References and tolerances as in
test_rows.py."""
import ctypes
import os
import subprocess
import warnings

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_rows import DTYPES, HUGE, U, check_route, half, make_ids, make_scores, randn, rows_module, tiny, within  # noqa: E402

gpu = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def by_column(t):
    """The same values, the first dimension's side by side."""
    return t.t().contiguous().t()


# ---- routes and weights in the strides of the scores they came from ----------------------------------------------------

@gpu
@pytest.mark.parametrize("over", ["chosen", "all"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_route_grad_of_routes_that_lie_as_the_scores_do(built_lib, dtype, over):
    """Sorting column-major scores gives column-major ids and weights: the same gradient, bit by bit, as from dense ones."""
    R = rows_module(built_lib)
    for rows, k, n in ((70, 33, 5), (1, 8, 2), (300, 100, 4)):
        base = make_scores(rows, k, dtype, 200)
        dw = randn((rows, n), 201)
        for s in (base, by_column(base)):
            r = R.route(s, n, 1.0, over)
            want = R.route_grad(dw, s, r, 1.0, over)
            both = torch.stack([r.best, r.total], 1)          # one of two statistics side by side
            turned = R.Routes(by_column(r.ids), by_column(r.weights), both[:, 0], both[:, 1])
            got = R.route_grad(by_column(dw), s, turned, 1.0, over)
            assert got.stride() == want.stride() and torch.equal(got, want)
            wide = torch.zeros((rows, n + 3), device="cuda")
            wide[:, 1:n + 1] = dw
            assert torch.equal(R.route_grad(wide[:, 1:n + 1], s, turned, 1.0, over), want)
            one = torch.full((1, 1), 0.5, device="cuda")       # a gradient that all entries share
            assert torch.equal(R.route_grad(one.expand(rows, n), s, r, 1.0, over), R.route_grad(torch.full_like(dw, 0.5), s, r, 1.0, over))


@gpu
def test_combine_with_weights_in_other_strides(built_lib):
    R = rows_module(built_lib)
    rows, n, k, d = 100, 3, 7, 64
    plan = R.sort_rows(make_ids(rows, n, k, 202), k, 4)
    e, w, dy = randn((plan.source.shape[0], d), 203), randn((rows, n), 204), randn((rows, d), 205)
    assert torch.equal(R.combine(e, plan, by_column(w)), R.combine(e, plan, w))
    got, want = R.combine_grad(dy, e, plan, by_column(w)), R.combine_grad(dy, e, plan, w)
    assert torch.equal(got.drows, want.drows) and torch.equal(got.dweights, want.dweights)
    one = torch.full((1, 1), 0.25, device="cuda").expand(rows, n)
    assert torch.equal(R.combine(e, plan, one), R.combine(e, plan, one.contiguous()))


# ---- nothing is read behind the last row -----------------------------------------------------------------------------

ROWS_OF_A_CTA = """
#include <cstdio>
#include <vector>
#include "km_rows_move.cuh"
using namespace km::rows;
int main() {
  for (int rows = 1; rows < 14000; rows += rows < 70 ? 1 : 997)
    for (int words : {1, 16, 32, 33, 64, 100, 5000})
      for (int sms : {1, 148}) {
        const int warps = combine_grad_warps(rows, words, sms), per_cta = kCombineGradThreads / 32 / warps;
        const int blocks = (rows + per_cta - 1) / per_cta;      // as kmeans_combine_grad launches them
        std::vector<int> seen(rows, 0);
        for (int b = 0; b < blocks; ++b)
          for (int y = 0; y < per_cta; ++y) {
            const int t = combine_grad_row(b, per_cta, y, rows);
            if (t < -1 || t >= rows) { printf("row %d of %d is addressed\\n", t, rows); return 1; }
            if (t >= 0) ++seen[t];
          }
        for (int n : seen)
          if (n != 1) { printf("a row of %d is taken %d times\\n", rows, n); return 1; }
      }
  printf("every row once\\n");
  return 0;
}
"""


def test_combine_grad_addresses_only_rows_that_are_there(tmp_path):
    """The rows of the last CTA's threads, on the host: behind the last row nothing is addressed (the values read there would not be used, so
    no result shows it)."""
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    src, exe = tmp_path / "rows.cu", tmp_path / "rows"
    src.write_text(ROWS_OF_A_CTA)
    subprocess.check_call([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "--expt-relaxed-constexpr",
                           "-I", os.path.join(ROOT, "h2o4gpu_b200", "csrc"), "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(src),
                           "-ldl"])
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout == "every row once\n", r.stdout


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_combine_grad_of_rows_that_do_not_fill_a_cta(built_lib, dtype):
    """Rows of dy far apart, one to seven of them: results as from rows side by side."""
    R = rows_module(built_lib)
    n, k = 4, 6
    for rows, d in [(r, c) for r in range(1, 8) for c in (64, 256, 400, 1024)]:      # one, two and four warps a row
        plan = R.sort_rows(make_ids(rows, n, k, 206), k, 2)
        e, w, dy = randn((plan.source.shape[0], d), 207, dtype), randn((rows, n), 208), randn((rows, d), 209, dtype)
        apart = torch.zeros((rows, 50, d), dtype=dtype, device="cuda")
        apart[:, 0] = dy
        got, want = R.combine_grad(apart[:, 0], e, plan, w), R.combine_grad(dy, e, plan, w)
        assert torch.equal(got.drows, want.drows) and torch.equal(got.dweights, want.dweights)


# ---- layer norm's gradient of rows far from zero -----------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("shape", [(5, 64), (5, 500), (6, 784), (5, 1021), (3, 4096), (4, 8100), (3, 9000)], ids=str)
def test_layer_norm_grad_far_from_zero(built_lib, shape):
    """Rows whose mean is thousands of deviations away: x - mean loses nothing there (the difference of two near numbers is exact), so the
    gradient is off by the roundings of the small numbers alone."""
    R = rows_module(built_lib)
    rows, d = shape
    x = randn(shape, 220, torch.float32, 1.0, 5000.0)
    x[1] -= 9000.0
    w, dy = randn(d, 221, scale=0.1, shift=1.0), randn(shape, 222)
    f = R.layer_norm(x)
    for weight in (w, None):
        got = R.layer_norm_grad(dy, x, f.mean, f.rstd, weight)
        r = f.rstd.double()[:, None]
        xh = (x.double() - f.mean.double()[:, None]) * r
        dyd = dy.double()
        g = dyd if weight is None else dyd * w.double()
        m1, m2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
        dx = r * (g - m1 - xh * m2)
        # xh: a difference and a product; g: a product; each mean: its additions and two products; the result: five operations
        depth = d / 32 + 12
        tol = U * r * (8 * g.abs() + (depth + 8) * g.abs().mean(1, keepdim=True) + (depth + 14) * xh.abs() * (g * xh).abs().mean(1, keepdim=True))
        within(got.dx, dx, tol + U * dx.abs())
        within(got.dweight, (dyd * xh).sum(0), U * (rows + 18) * (dyd * xh).abs().sum(0))
        within(got.dbias, dyd.sum(0), U * (rows + 4) * dyd.abs().sum(0))


# ---- backward from the engine's own routes, whose scores nobody has ----------------------------------------------------

@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_route_grad_without_scores(built_lib, dtype):
    """Over the chosen no score is read: the same gradient without them, bit by bit."""
    R = rows_module(built_lib)
    for rows, k, n in ((70, 33, 5), (1, 8, 2), (300, 100, 4), (50, 1000, 32)):
        s, dw = make_scores(rows, k, dtype, 250), randn((rows, n), 251)
        r = R.route(s, n, 0.5)
        assert torch.equal(R.route_grad(dw, None, r, 0.5, k=k, dtype=dtype), R.route_grad(dw, s, r, 0.5))
    for bad in (lambda: R.route_grad(dw, None, r, 0.5), lambda: R.route_grad(dw, None, r, 0.5, "all", k=k),
                lambda: R.route_grad(dw, None, r, 0.5, k=n - 1), lambda: R.route_grad(dw, None, r, 0.5, k=k, dtype=torch.float64),
                lambda: R.route_grad(dw[:3], None, r, 0.5, k=k), lambda: R.route_grad(dw, None, None, 0.5, k=k),
                lambda: R.route_grad(dw, s, None, 0.5)):
        with pytest.raises(ValueError):
            bad()


@gpu
def test_route_grad_behind_nearest(built_lib):
    """A handle's nearest clusters, and the gradient of its distances from that of their weights."""
    from h2o4gpu_b200 import ResidentKMeans
    R = rows_module(built_lib)
    rows, d, k, n = 900, 24, 9, 3
    X = randn((rows, d), 252)
    h = ResidentKMeans()
    h.attach_device(0, X.data_ptr(), rows, d)
    h.set_centroids(X[:k].cpu().numpy())
    r = R.nearest(h, n, -0.1)
    D = torch.from_numpy(h.transform()).cuda()
    h.close()
    dw = randn((rows, n), 253)
    got = R.route_grad(dw, None, r, -0.1, k=k)
    assert got.shape == (rows, k) and got.dtype == torch.float32
    # D lies cluster after cluster, where another kernel adds up c in another order: each of the two is off by at most n + 8 roundings of
    # sum |w g|, two of |g| (the difference), and four of the result
    w, g = r.weights.double(), dw.double()
    size = 0.1 * w * ((n + 12) * (w * g).abs().sum(1, keepdim=True) + 6 * g.abs())
    tol = torch.zeros((rows, k), dtype=torch.float64, device="cuda").scatter_(1, r.ids.long(), 2 * U * size)
    within(got, R.route_grad(dw, D, r, -0.1), tol)


# ---- routing's gradient where masks and limits meet --------------------------------------------------------------------

def check_route_grad(R, s, dw, n, scale, over):
    """route_grad of what route gives for `s`, against  scale p (g - c)  in float64."""
    dtype = s.dtype
    rows, k = s.shape
    got, ref = check_route(R, s, n, scale, over)
    ids, w = ref["ids"], got.weights.double().cpu().numpy()
    g = np.where(ids >= 0, dw.double().cpu().numpy(), 0.0)
    c = (w * g).sum(1, keepdims=True)
    dc = (n + 8) * U * np.abs(w * g).sum(1, keepdims=True)
    G, W = np.zeros((rows, k + 1)), np.zeros((rows, k + 1))
    np.put_along_axis(G, np.where(ids >= 0, ids, k), g, 1)
    np.put_along_axis(W, np.where(ids >= 0, ids, k), w, 1)
    G, W = G[:, :k], W[:, :k]
    open_ = ref["q"] > -np.inf
    if over == "chosen":
        p, drel = W, 0.0
    else:
        # exp's argument is off by two roundings of itself, exp by two units in the last place, then a division
        arg = np.where(open_, ref["a"] * (np.where(open_, ref["q"], 0.0) - ref["base"]), -np.inf)
        total = got.total.double().cpu().numpy()[:, None]
        p = np.where(open_ & (total > 0), np.exp(arg) / np.where(total > 0, total, 1.0), 0.0)
        drel = U * (2 * np.where(open_, np.abs(arg), 0.0) + 6)
    want = scale * p * (G - c)
    # beside the result's own roundings, what the smallest exponentials lose below 2^-126
    tol = abs(scale) * (p * ((drel + 6 * U) * np.abs(G - c) + dc + U * np.abs(G)) + 2.0 ** -126 * (p > 0) * np.abs(G - c)) + 2.0 ** -126
    tol = tol + half(dtype) * (np.abs(want) + tol) + tiny(dtype)
    ds = R.route_grad(dw, s, got, scale, over)
    within(ds, torch.from_numpy(want), torch.from_numpy(tol))
    assert not bool(ds.cpu()[torch.from_numpy(~open_)].any())        # a cluster that cannot be taken has no gradient
    return ds


def masked_scores(dtype, k=40):
    """Scores of large quality better: rows that masks of the lowest value, infinities and NaN leave little of."""
    low, inf, nan = torch.finfo(dtype).min, float("inf"), float("nan")
    s = torch.zeros((14, k), dtype=dtype, device="cuda")
    s[1] = low
    s[2] = -inf
    s[3] = nan
    s[4, :k - 2] = -inf
    s[5, 10:] = low
    s[6, 7] = s[6, 21] = inf
    s[7, ::2] = -0.0
    s[8, 5] = torch.finfo(dtype).max
    s[9] = torch.arange(k, dtype=torch.float32).to(dtype).cuda()
    s[10] = nan
    s[10, k - 1] = low
    s[11] = -inf                       # one mask by the lowest value, another by -inf, nothing open
    s[11, 3:9] = low
    s[12, ::3] = low
    s[12, 1::3] = -inf
    s[12, 2::3] = nan
    s[13] = -inf                       # the lowest value beside infinities of both signs
    s[13, 4] = inf
    s[13, 6:11] = low
    return s


@gpu
@pytest.mark.parametrize("over", ["chosen", "all"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("k", [40, 41, 1003])
def test_route_grad_ties_masks_and_infinities(built_lib, k, dtype, over):
    R = rows_module(built_lib)
    s = masked_scores(dtype, k)
    dw = randn((s.shape[0], 3), 210)
    for v in (s, by_column(s)):
        up, down = check_route_grad(R, v, dw, 3, 1.0, over), check_route_grad(R, -v, dw, 3, -1.0, over)
        assert torch.equal(up, -down)


@gpu
@pytest.mark.parametrize("over", ["chosen", "all"])
@pytest.mark.parametrize("k", [40, 41, 200])
def test_route_grad_with_the_largest_scales(built_lib, k, over):
    """The scale times the weights' gradient is beyond float32, the gradient of clusters without weight is zero all the same."""
    R = rows_module(built_lib)
    s = make_scores(20, k, torch.float32, 211, masked=False)
    s[:, 7] = s[:, 3]
    s[1::2, 5:30:3] = float("-inf")
    for shift in (0.0, 3.0):
        dw = randn((20, 4), 212, scale=2.0, shift=shift)
        for scale in (HUGE / 2, -HUGE / 2, 2.0 ** -126):
            for v in (s, by_column(s)):
                check_route_grad(R, v if scale > 0 else -v, dw, 4, scale, over)


# ---- sizes that an int does not hold -----------------------------------------------------------------------------------

def test_c_refuses_more_columns_than_an_int_holds(built_lib):
    """KM_EINVAL before any device call, for pointers that are never dereferenced."""
    from h2o4gpu_b200.libs import lib_kmeans
    lib = lib_kmeans.cdll()
    p, size = ctypes.c_void_p(4096), ctypes.c_size_t()
    most, most_grad = 0x7fff0000, 0x3fff0000

    def norm(cols):
        return lib.kmeans_layer_norm(2, p, cols, 1, cols, None, None, 0, 1e-5, p, cols, p, p, None)

    def norm_grad(cols):
        return lib.kmeans_layer_norm_grad(2, p, cols, p, cols, p, p, 1, cols, None, 0, p, cols, p, p, p, 1 << 50, None)

    def moves(cols):
        return [lib.kmeans_dispatch(2, p, cols, 1, cols, 1, p, p, 1, p, cols, None),
                lib.kmeans_combine(2, p, cols, 1, cols, p, p, 1, 1, p, cols, None),
                lib.kmeans_combine_grad(2, p, cols, p, cols, 1, cols, p, p, p, 1, 1, p, cols, p, None)]

    for cols in (most + 1, 0x7fffffff, 1 << 31, (1 << 32) + 8):
        assert norm(cols) == -1 and norm_grad(cols) == -1 and moves(cols) == [-1, -1, -1], cols
    for cols in (most_grad + 1, 1 << 30, 1_200_000_000):
        assert norm_grad(cols) == -1 and lib.kmeans_layer_norm_grad_workspace(1, cols, ctypes.byref(size)) == -1, cols


@gpu
def test_python_refuses_sizes_that_a_c_int_cuts(built_lib):
    """2^32 + 8 clusters would arrive as 8; and what is refused allocates nothing first."""
    R = rows_module(built_lib)
    from h2o4gpu_b200 import ResidentKMeans
    x = randn((6, 8), 230)
    wide = torch.zeros((1, 1), device="cuda").expand(1, (1 << 32) + 8)
    ids = torch.zeros((6, 2), dtype=torch.int32, device="cuda")
    r = R.route(x, 2)
    one = R.Routes(r.ids[:1], r.weights[:1], r.best[:1], r.total[:1])
    h = ResidentKMeans()
    bad = [lambda: R.route(wide, 2), lambda: R.route(x, (1 << 32) + 2), lambda: R.route(x, 1 << 20),
           lambda: R.route_grad(one.weights, wide, one), lambda: R.nearest(h, (1 << 32) + 1),
           lambda: R.sort_rows(ids, (1 << 32) + 3), lambda: R.sort_rows(ids, 3, (1 << 32) + 1), lambda: R.sort_rows(ids, 1 << 30),
           lambda: R.sort_rows(ids, 3, 1 << 30), lambda: R.sort_rows(ids, -3), lambda: R.sort_rows(ids, 3, -1)]
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError)):
            call()
            pytest.fail("call %d was not refused" % i)
    assert torch.cuda.max_memory_allocated() - before < 1 << 20
    h.close()
    # the largest of what is taken
    plan = R.sort_rows(ids, 16384, 16384)
    assert plan.offsets[1:].tolist() == [16384] * 16384 and plan.slot.view(-1).tolist() == list(range(12))
    plan = R.sort_rows(ids[:1], 3, 1 << 20)
    assert plan.offsets.tolist() == [0, 1 << 20, 1 << 20, 1 << 20] and plan.source[:2].tolist() == [0, 1]


# ---- a handle that got no memory ---------------------------------------------------------------------------------------

@gpu
def test_nearest_after_a_failed_attach_or_upload(built_lib):
    """The outputs have the rows that the engine works on: a failed attach leaves the old matrix, a failed upload none."""
    from h2o4gpu_b200 import ResidentKMeans
    from h2o4gpu_b200.libs import lib_kmeans
    R = rows_module(built_lib)
    lib = lib_kmeans.cdll()
    few, many = randn((300, 16), 240), randn((200_000, 16), 241)
    h = ResidentKMeans()
    h.attach_device(0, few.data_ptr(), 300, 16)
    h.set_centroids(few[:7].cpu().numpy())
    h.assign()
    want, labels = R.nearest(h, 3), h.labels()

    def fails(call):
        lib.kmeans_selftest_alloc_limit(1000)
        try:
            with pytest.raises(RuntimeError):
                call()
        finally:
            lib.kmeans_selftest_alloc_limit(-1)

    fails(lambda: h.attach_device(0, many.data_ptr(), 200_000, 16))
    assert all(torch.equal(a, b) for a, b in zip(R.nearest(h, 3), want)) and np.array_equal(h.labels(), labels)
    with pytest.raises(RuntimeError):
        h.upload(np.empty((0, 16), np.float32))      # refused: nothing has changed
    assert all(torch.equal(a, b) for a, b in zip(R.nearest(h, 3), want)) and np.array_equal(h.labels(), labels)
    fails(lambda: h.upload(many.cpu().numpy()))
    for call in (lambda: R.nearest(h, 3), h.transform, h.labels, lambda: h.fit(few[:7].cpu().numpy(), 2), h.assign):
        with pytest.raises(RuntimeError, match="no data"):
            call()
    h.upload(few.cpu().numpy())
    h.set_centroids(few[:7].cpu().numpy())
    assert all(torch.equal(a, b) for a, b in zip(R.nearest(h, 3), want))
    h.attach_device(0, many.data_ptr(), 200_000, 16)
    assert R.nearest(h, 3).ids.shape == (200_000, 3)
    h.close()


def test_route_grad_without_scores_refuses_what_is_not_on_a_gpu(built_lib):
    R = rows_module(built_lib)
    ids = torch.zeros((4, 2), dtype=torch.int32)
    with pytest.raises(ValueError, match="must be a CUDA tensor"):
        R.route_grad(ids.float(), None, R.Routes(ids, ids.float(), ids[:, 0].float(), ids[:, 0].float()), k=3)
    with pytest.raises(ValueError, match="needs the scores"):
        R.route_grad(ids.float(), None, R.Routes(ids, ids.float(), ids[:, 0].float(), ids[:, 0].float()), over="all", k=3)


@gpu
def test_a_call_that_cuts_autograd_warns(built_lib):
    R = rows_module(built_lib)
    x, s, w, wt = randn((6, 8), 260), randn((6, 5), 261), randn(8, 262), randn((6, 2), 263)
    plan = R.sort_rows(torch.zeros((6, 2), dtype=torch.int32, device="cuda"), 3)
    e = R.dispatch(x, plan)

    def leaf(t):
        return t.clone().requires_grad_()

    calls = {"layer_norm": (lambda f: R.layer_norm(f(x))[0], lambda f: R.layer_norm(x, f(w))[0], lambda f: R.layer_norm(x, w, f(w))[0]),
             "route": (lambda f: R.route(f(s), 2)[1],), "dispatch": (lambda f: R.dispatch(f(x), plan),),
             "combine": (lambda f: R.combine(f(e), plan, wt), lambda f: R.combine(e, plan, f(wt)), lambda f: R.dispatch_grad(f(e), plan))}
    for name, some in calls.items():
        for call in some:
            with pytest.warns(UserWarning, match=name + " records nothing for autograd.*" + name + "_grad"):
                got = call(leaf)
            with warnings.catch_warnings():
                warnings.simplefilter("error")
                want = call(lambda t: t)
                with torch.no_grad():
                    again = call(leaf)
            assert torch.equal(got, want) and torch.equal(again, want) and not got.requires_grad


@gpu
def test_views_whose_sign_is_kept_apart_are_refused(built_lib):
    """The imaginary part of a conjugate: its memory holds the other sign."""
    R = rows_module(built_lib)
    z = torch.complex(randn((6, 5), 270), randn((6, 5), 271))
    s = z.conj().imag
    assert s.is_neg()
    r = R.route(s.resolve_neg(), 2)
    for call in (lambda: R.route(s, 2), lambda: R.route_grad(r.weights, s, r), lambda: R.layer_norm(s[:, :1]),
                 lambda: R.layer_norm(z.imag[:, :1], out=s[:, :1])):
        with pytest.raises(ValueError, match="resolve_neg"):
            call()
    check_route(R, s.resolve_neg(), 2, 1.0, "all")
    check_route(R, z.imag, 2, 1.0, "all")                      # every second element


@gpu
def test_outputs_on_the_memory_of_their_inputs(built_lib):
    """Rows are read while others are written: an output that shares memory with them is refused, but for the norm in place; parts of one
    buffer beside each other are not."""
    R = rows_module(built_lib)
    buf = randn((64, 40), 280)
    plan = R.sort_rows(torch.arange(16, device="cuda", dtype=torch.int32).view(8, 2) % 3, 3)       # 16 places for 8 rows
    x, e = buf[:8, :16], buf[:16, :16]
    for call in (lambda: R.layer_norm(x, out=buf[1:9, :16]), lambda: R.layer_norm(x, out=buf[:8, 4:20]), lambda: R.layer_norm(buf[:1, :16], out=buf[:1, 15:31]),
                 lambda: R.layer_norm(buf.view(-1)[:128].view(8, 16), out=buf.view(-1)[16:144].view(8, 16)),
                 lambda: R.dispatch(x, plan, out=buf[:16, :16]), lambda: R.dispatch(x, plan, out=buf[7:23, :16]),
                 lambda: R.dispatch(x, plan, out=buf[:, :16]), lambda: R.combine(e, plan, out=x), lambda: R.combine(e, plan, out=buf[15:23, :16]),
                 lambda: R.dispatch_grad(e, plan, out=x), lambda: R.dispatch(buf[3:4, 8:24].expand(8, 16), plan, out=buf[:16, :16])):
        with pytest.raises(ValueError, match="shares memory"):
            call()
    want = R.layer_norm(x).y
    keep = buf.clone()
    for out in (buf[8:16, :16], buf[:8, 16:32], buf[1:9, 20:36], buf[:8, 24:40], buf[20:28, 3:19], x):
        assert torch.equal(R.layer_norm(x, out=out).y, want)
        buf.copy_(keep)
    want = R.dispatch(x, plan)
    for out in (buf[8:24, :16], buf[:16, 16:32], buf[8:, :16], buf[:, 24:]):
        assert torch.equal(R.dispatch(x, plan, out=out)[:16], want)
        buf.copy_(keep)
    for rows, out in ((e, buf[16:24, :16]), (buf[:, :16], buf[16:24, :16]), (e, buf[:8, 16:32]), (buf[::2, :16], buf[1:17:2, :16])):
        assert torch.equal(R.combine(rows, plan, out=out), R.combine(rows.clone(), plan))
        buf.copy_(keep)


def test_overlap_rule_against_sets_of_addresses(built_lib):
    from h2o4gpu_b200.rows import _overlap
    rng = np.random.default_rng(1)
    buf = torch.zeros(400)
    seen = [0, 0]
    for _ in range(4000):
        cols = int(rng.integers(1, 9))

        def view(zero):
            rows, step = int(rng.integers(1, 6)), int(rng.choice([0, cols, cols + 1, cols + 5, 2 * cols, 20]))
            return buf.as_strided((rows if step or zero else 1, cols), (max(step, cols) if step else 0, 1), int(rng.integers(0, 120)))

        a, b = view(False), view(True)
        sa, sb = a.stride(0) * (a.shape[0] > 1), b.stride(0) * (b.shape[0] > 1)
        places = [{t.storage_offset() + i * t.stride(0) + j for i in range(t.shape[0]) for j in range(cols)} for t in (a, b)]
        shared = bool(places[0] & places[1])
        if not (sa and sb and sa != sb):
            assert _overlap(a, a.shape[0], b, b.shape[0]) == shared
            seen[shared] += 1
        else:
            assert not _overlap(a, a.shape[0], b, b.shape[0])
    assert min(seen) > 300
