"""Calls of the row operators (h2o4gpu_b200.rows) that their documentation allows and that need care.  References and tolerances as in
test_rows.py."""
import pytest

torch = pytest.importorskip("torch")

from test_rows import DTYPES, make_ids, make_scores, randn, rows_module  # noqa: E402

gpu = pytest.mark.gpu


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
