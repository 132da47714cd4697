"""Calls of the row operators (h2o4gpu_b200.rows) that their documentation allows and that need care.  References and tolerances as in
test_rows.py."""
import os
import subprocess

import pytest

torch = pytest.importorskip("torch")

from test_rows import DTYPES, make_ids, make_scores, randn, rows_module  # noqa: E402

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
    n, k, d = 4, 6, 64
    for rows in range(1, 8):
        plan = R.sort_rows(make_ids(rows, n, k, 206), k, 2)
        e, w, dy = randn((plan.source.shape[0], d), 207, dtype), randn((rows, n), 208), randn((rows, d), 209, dtype)
        apart = torch.zeros((rows, 50, d), dtype=dtype, device="cuda")
        apart[:, 0] = dy
        got, want = R.combine_grad(apart[:, 0], e, plan, w), R.combine_grad(dy, e, plan, w)
        assert torch.equal(got.drows, want.drows) and torch.equal(got.dweights, want.dweights)
