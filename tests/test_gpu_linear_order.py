"""4-bit linear and expert calls one behind another: streams, grids that start early, host threads."""

import threading

import pytest
import torch

from conftest import pkg
from test_gpu_linear import assert_within, check_route, expected_experts, make_weight, make_x, routing_of

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


def test_routing_from_several_host_threads(cuda):
    """Calls whose sort kernels need 51 to 172 KB of shared memory, from four threads at once: no launch
    may depend on the size another thread has just asked for."""
    cases = [(4200, 1024, 32), (2000, 256, 8), (1000, 1024, 1), (3000, 128, 2)]
    logits = [make_x(t, e, torch.float32, cuda, seed=e + t) for t, e, _ in cases]
    want = [pkg.route_experts(z, k) for z, (_, _, k) in zip(logits, cases)]
    for z, (_, _, k) in zip(logits, cases):
        check_route(z, k, True)
    torch.cuda.synchronize(cuda)
    errors = []

    def work(z, k, ref):
        try:
            side = torch.cuda.Stream(cuda)
            with torch.cuda.stream(side):
                for _ in range(1500):
                    got = pkg.route_experts(z, k)
            side.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, ref))
        except BaseException as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(z, c[2], w)) for z, c, w in zip(logits, cases, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]
