"""The 4-bit linear layers where their forms meet: the precision of each type, the calls on both
sides of a change of kernel, experts far from the mean, the bounded waits, and the example."""

import sys

import pytest
import torch

from conftest import ROOT, pkg
from test_gpu_linear import (assert_within, dense, expected, expected_experts, make_weight, make_x, routing_of)

pytestmark = pytest.mark.gpu

TIMEOUT = 4  # AM_STATUS_TIMEOUT


def trained_weight(n, k, dtype, dev, seed):
    """Normal weights in the cache's format (the framework's own quantization)."""
    g = torch.Generator(device="cpu").manual_seed(seed)
    return pkg.quantize((torch.randn(n, k, generator=g) * k ** -0.5).to(dtype).to(dev))


@pytest.mark.parametrize("rows", [3, 20, 50, 100, 600])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_error_stays_near_the_rounding_of_the_output(cuda, dtype, gated, rows):
    """Root mean square errors against 64 bits.  Rounding the exact result once costs 2.1e-4 in fp16
    and 1.7e-3 in bf16.  A weight rounded once to fp16 adds 1.8e-4 of a product, one of two parts
    1.0e-4: sqrt(1 + (1.8 / 2.1)^2) = 1.32 plain and sqrt(1 + 2 (1.0 / 2.1)^2) = 1.21 gated in
    fp16, 1.02 in bf16.  (silu steepens the gate's error by up to 1.1.)"""
    n, k = 8192, 1024
    ws = [trained_weight(n, k, dtype, cuda, seed=s) for s in range(2 if gated else 1)]
    x = make_x(rows, k, dtype, cuda)
    q = [pkg.Q4Weight(*w) for w in ws]
    got = (pkg.quantized_swiglu(x, *q) if gated else pkg.quantized_matmul(x, *q)).double()
    y = x.double() @ dense(ws[0]).mT
    if gated:
        y = y * torch.sigmoid(y) * (x.double() @ dense(ws[1]).mT)
    once = float((y.to(dtype).double() - y).norm())
    assert float((got - y).norm()) <= {torch.float16: 1.4, torch.bfloat16: 1.05}[dtype] * once


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [4, 5, 8, 9])
def test_large_gated_pairs_of_a_few_tokens(cuda, rows, dtype):
    """Pairs on both sides of the size and the tokens at which the tiles take over."""
    for n, k in ((7000, 4096), (6600, 4160)):
        ws = [make_weight((n, k), dtype, cuda, seed=i) for i in range(2)]
        x = make_x(rows, k, dtype, cuda)
        assert_within(pkg.quantized_swiglu(x, *[pkg.Q4Weight(*w) for w in ws]), *expected(x, ws))


@pytest.mark.parametrize("rows,n_experts", [(1, 64), (32, 64), (33, 64), (96, 48), (97, 48), (128, 64)])
def test_experts_far_from_the_mean(cuda, rows, n_experts):
    """All rows at one expert, at the first and the last, and one each: an expert with more rows
    than an item holds takes several items."""
    n, k = 208, 320
    ws = [make_weight((n_experts, n, k), torch.bfloat16, cuda, seed=i) for i in range(2)]
    q = [pkg.Q4Weight(*w) for w in ws]
    x = make_x(rows, k, torch.bfloat16, cuda)
    i = torch.arange(rows, device=cuda)
    for chosen in (torch.full_like(i, n_experts // 2), (i % 2) * (n_experts - 1), i % n_experts):
        r = routing_of(chosen[:, None], n_experts)
        assert_within(pkg.expert_swiglu(x, *q, r), *expected_experts(x, ws, r, True), "gated")
        assert_within(pkg.expert_matmul(x, q[0], r, gather=True), *expected_experts(x, ws[:1], r, True), "plain")


@pytest.mark.parametrize("tokens,gated", [(40, False), (120, True), (150, False), (1200, True), (1200, False)])
def test_wait_timeout_is_flagged_and_recovers(cuda, monkeypatch, tokens, gated):
    """The tiles of one SM (split over a cluster and not) and of pairs of SMs with every wait giving up
    at once: the call returns with AM_STATUS_TIMEOUT and the next one is right."""
    n, k = 2176 if gated else 4352, 640  # (17 row tiles either way)
    ws = [make_weight((4, n, k), torch.float16, cuda, seed=i) for i in range(2 if gated else 1)]
    q = [pkg.Q4Weight(*w) for w in ws]
    r = routing_of((torch.arange(tokens, device=cuda) % 4)[:, None], 4)
    x = make_x(tokens, k, torch.float16, cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    f = lambda: (pkg.expert_swiglu(x, *q, r, status=status) if gated else  # noqa: E731
                 pkg.expert_matmul(x, q[0], r, gather=True, status=status))
    monkeypatch.setenv("AM_Q4_TEST_WAIT_LIMIT_NS", "0")
    f()
    torch.cuda.synchronize(cuda)
    assert int(status.item()) & TIMEOUT
    monkeypatch.delenv("AM_Q4_TEST_WAIT_LIMIT_NS")
    status.zero_()
    assert_within(f(), *expected_experts(x, ws, r, True))
    assert int(status.item()) == 0


def test_combine_of_no_rows(cuda):
    """Without a row every position is out of range: the residual comes back, flagged."""
    y = torch.empty(0, 64, dtype=torch.float16, device=cuda)
    w = torch.ones(3, 2, device=cuda)
    res = make_x(3, 64, torch.float16, cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = pkg.combine_experts(y, w, torch.zeros(3, 2, dtype=torch.int32, device=cuda), residual=res, status=status)
    assert torch.equal(out, res) and int(status) == pkg._lib.STATUS_BAD_POSITION


def test_example_expert_decoder_layer(cuda):
    """The layer around the cache against dense float32 products: intermediate tensors are rounded to
    bf16 on both sides (2^-8 each), a dozen of them."""
    sys.path.insert(0, str(ROOT / "examples"))
    try:
        import expert_decoder_layer as example
    finally:
        sys.path.pop(0)
    r = example.run(agents=3, prefill=37, steps=3, device=str(cuda))
    assert r["error"] <= 12 * 2.0 ** -8
