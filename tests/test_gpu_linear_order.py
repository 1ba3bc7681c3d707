"""4-bit linear and expert calls one behind another: streams, grids that start early, host threads."""

import pytest
import torch

from conftest import pkg
from test_gpu_linear import assert_within, expected_experts, make_weight, make_x, routing_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [200, 1500])
@pytest.mark.parametrize("gated", [False, True])
def test_a_call_behind_one_without_rows(cuda, gated, rows):
    """A grid whose experts hold no row has no work and still ends only after the grid before it:
    the next call writes the same workspace.  Repeated; every result is the first one's bits."""
    n, k, n_experts = 2304, 704, 4
    ws = [make_weight((n_experts, n, k), torch.bfloat16, cuda, seed=i) for i in range(1 + gated)]
    q = [pkg.Q4Weight(*w) for w in ws]
    r = routing_of((torch.arange(rows, device=cuda) % n_experts)[:, None], n_experts)
    none = r._replace(offsets=torch.zeros_like(r.offsets))
    xs = [make_x(rows, k, torch.bfloat16, cuda, seed=s) for s in range(2)]
    f = lambda x, r, out=None: (pkg.expert_swiglu(x, *q, r, out=out) if gated else  # noqa: E731
                                pkg.expert_matmul(x, q[0], r, gather=True, out=out))
    want = f(xs[0], r)
    assert_within(want, *expected_experts(xs[0], ws, r, True))
    untouched = torch.full_like(want, 3.0)
    for _ in range(50):
        f(xs[1], none, untouched)
        assert torch.equal(f(xs[0], r), want)
    assert bool((untouched == 3.0).all())
