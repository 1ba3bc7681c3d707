"""4-bit linear layers and expert layers against their definitions in 64 bits.

The bound of an output is derived from the arithmetic: a weight enters its product rounded to
fp16 (relative 2^-11), products and sums are fp32 (a relative 2^-13 of the absolute sum covers
the longest sums here), and the result is rounded once to the output type (half an ulp).  With
S = sum |w| |x| that is (2^-11 + 2^-13) S + u |y|; through silu(g) * u the two sums' bounds enter
by |silu'| <= 1.1 and |silu(g)|.
"""

import pytest
import torch

from conftest import pkg

pytestmark = pytest.mark.gpu
GROUP = 64
SUM_REL = 2.0 ** -11 + 2.0 ** -13
OUT_REL = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = 2.0 ** -24  # smallest fp16 number: outputs below it round to a multiple of it


def make_weight(shape, dtype, dev, seed=0, spread=0.0, scale=0.02):
    """Random codes, scales and biases of both signs (spread: log2 spread of the scales)."""
    g = torch.Generator(device="cpu").manual_seed(seed)
    *lead, n, k = shape
    codes = torch.randint(-2 ** 31, 2 ** 31, (*lead, n, k // 8), generator=g, dtype=torch.int64).to(torch.int32)
    s = scale * (0.5 + torch.rand(*lead, n, k // GROUP, generator=g))
    s = s * torch.exp2(spread * (torch.rand(s.shape, generator=g) - 0.5))
    s = torch.where(torch.rand(s.shape, generator=g) < 0.5, s, -s)
    b = -7.5 * s * (1 + 0.2 * torch.randn(s.shape, generator=g))
    return codes.to(dev), s.to(dtype).to(dev), b.to(dtype).to(dev)


def dense(w):
    codes, s, b = w
    n = torch.stack([(codes.long() >> (4 * i)) & 15 for i in range(8)], -1).flatten(-2).double()
    return n * s.double().repeat_interleave(GROUP, -1) + b.double().repeat_interleave(GROUP, -1)


def make_x(m, k, dtype, dev, seed=1):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return torch.randn(m, k, generator=g).to(dtype).to(dev)


def product(x, w):
    """-> (y, bound of the fp32 sum's error)."""
    x, w = x.double(), dense(w)
    return x @ w.mT, SUM_REL * (x.abs() @ w.abs().mT)


def expected(x, ws):
    y, e = product(x, ws[0])
    if len(ws) == 2:
        u, eu = product(x, ws[1])
        s = y * torch.sigmoid(y)
        y, e = s * u, 1.1 * e * (u.abs() + eu) + s.abs() * eu + 2.0 ** -20 * (s * u).abs()
    return y, e


def assert_within(got, want, bound, what=""):
    assert got.shape == want.shape, what
    u = OUT_REL[got.dtype]
    tol = bound + u * (want.abs() + bound) + TINY
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst "
                           f"{float((err / tol).nan_to_num(1e30).max()):.2f} x the bound at "
                           f"{torch.nonzero(bad)[0].tolist()}")


def run(x, ws, dtype=None):
    q = [pkg.Q4Weight(*w) for w in ws]
    return pkg.quantized_swiglu(x, *q) if len(q) == 2 else pkg.quantized_matmul(x, *q)


SHAPES = [(1, 64), (7, 128), (16, 64), (40, 192), (130, 320), (257, 704), (512, 2880), (300, 4096)]
TOKENS = [1, 2, 3, 5, 8, 9, 15, 16, 17, 24, 32, 33, 48, 64, 65, 100, 128, 129, 200, 256, 257, 515]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("n,k", SHAPES)
def test_linear_every_token_count(cuda, n, k, gated, dtype):
    ws = [make_weight((n, k), dtype, cuda, seed=i) for i in range(1 + gated)]
    q = [pkg.Q4Weight(*w) for w in ws]
    for m in TOKENS:
        x = make_x(m, k, dtype, cuda, seed=m)
        got = pkg.quantized_swiglu(x, *q) if gated else pkg.quantized_matmul(x, *q)
        assert_within(got, *expected(x, ws), f"{m} tokens {n}x{k}")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k,gated", [(1, 4096, 4096, False), (3, 5000, 14336, False), (8, 9001, 1024, True),
                                         (20, 2049, 4096, True), (96, 4096, 4096, False),
                                         (700, 1537, 2880, True), (1500, 2304, 1024, False),
                                         (2048, 2049, 320, False), (2300, 1030, 192, True),
                                         (1000, 4097, 1024, False), (4096, 2048, 64, True),
                                         (2100, 2304, 2880, True), (3333, 1100, 448, True)])
def test_linear_larger(cuda, m, n, k, gated, dtype):
    ws = [make_weight((n, k), dtype, cuda, seed=i) for i in range(1 + gated)]
    x = make_x(m, k, dtype, cuda)
    assert_within(run(x, ws), *expected(x, ws))


@pytest.mark.parametrize("m", [0, 1, 40, 150])
def test_linear_leading_dims_and_strides(cuda, m):
    w = make_weight((48, 256), torch.bfloat16, cuda)
    q = pkg.Q4Weight(*w)
    x = make_x(3 * max(m, 1), 512, torch.bfloat16, cuda).view(3, max(m, 1), 512)[:, :m]
    for view in (x[..., :256], x[..., 256:], x[..., 1:257], x[..., ::2], x.transpose(0, 1)[..., 8:264]):
        got = pkg.quantized_matmul(view, q)
        assert got.shape == (*view.shape[:-1], 48)
        assert_within(got, *expected(view, [w]), str(view.stride()))
    out = torch.empty(3, m, 48, dtype=torch.bfloat16, device=cuda)
    assert pkg.quantized_matmul(x[..., :256], q, out=out) is out
    assert_within(out, *expected(x[..., :256], [w]))


def test_weight_from_unaligned_and_strided_tensors(cuda):
    codes, s, b = make_weight((40, 256), torch.float16, cuda)
    flat = torch.empty(codes.numel() + 1, dtype=torch.int32, device=cuda)
    flat[1:] = codes.flatten()
    wide = torch.stack([s, b], -1)
    q = pkg.Q4Weight(flat[1:].view(codes.shape), wide[..., 0], wide[..., 1])
    x = make_x(5, 256, torch.float16, cuda)
    assert_within(pkg.quantized_matmul(x, q), *expected(x, [(codes, s, b)]))


@pytest.mark.parametrize("m", [1, 12, 40, 160])
@pytest.mark.parametrize("scale,spread", [(1e-6, 0.0), (1e-6, 16.0), (30.0, 0.0), (1e3, 12.0), (1e-20, 4.0),
                                          (1e8, 0.0)])
def test_linear_weights_of_every_magnitude(cuda, m, scale, spread):
    """bf16 weights from 1e-20 to 1e9, with scales 2^spread apart within a row (a group far below
    its row's largest keeps its value to 2^-24 of that)."""
    w = make_weight((72, 640), torch.bfloat16, cuda, spread=spread, scale=scale)
    x = make_x(m, 640, torch.bfloat16, cuda)
    want, bound = expected(x, [w])
    row = dense(w).abs().amax(-1)
    bound = bound + 2.0 ** -24 * row * x.double().abs().sum(-1, keepdim=True)
    got = pkg.quantized_matmul(x, pkg.Q4Weight(*w))
    err = (got.double() - want).abs()
    tol = bound + OUT_REL[torch.bfloat16] * (want.abs() + bound) + 1e-38
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("m", [1, 12, 40, 160])
def test_linear_activations_of_every_magnitude(cuda, m):
    """bf16 tokens scaled from 1e-30 to 1e30, a zero token, and outliers of 2^12 in a token: each
    token as exact as by itself."""
    w = make_weight((72, 640), torch.bfloat16, cuda)
    x = make_x(m, 640, torch.bfloat16, cuda).float()
    x *= torch.tensor([1.0, 1e-30, 1e30, 0.0, 1e5, 1e-5], device=cuda)[torch.arange(m, device=cuda) % 6, None]
    x[:, 17] *= 4096.0
    x = x.to(torch.bfloat16)
    want, bound = expected(x, [w])
    got = pkg.quantized_matmul(x, pkg.Q4Weight(*w))
    err = (got.double() - want).abs()
    tol = bound + OUT_REL[torch.bfloat16] * (want.abs() + bound) + 1e-38
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m", [3, 40, 150])
def test_linear_zero_scales_and_nonfinite_tokens(cuda, m, dtype):
    """Groups and rows with scale (and bias) zero; a token with an infinity or NaN has no finite
    outputs in rows it reaches and leaves the other tokens alone."""
    codes, s, b = make_weight((70, 256), dtype, cuda)
    s[3], b[3] = 0, 0
    s[5, 1], b[9] = 0, 0
    x = make_x(m, 256, dtype, cuda)
    clean = x.clone()
    q = pkg.Q4Weight(codes, s, b)
    want, bound = expected(clean, [(codes, s, b)])
    assert_within(pkg.quantized_matmul(clean, q), want, bound)
    x[0, 7], x[2, 11] = float("inf"), float("nan")
    got = pkg.quantized_matmul(x, q)
    keep = torch.ones(m, dtype=torch.bool, device=cuda)
    keep[[0, 2]] = False
    assert_within(got[keep], want[keep], bound[keep])
    assert not torch.isfinite(got[2]).any()
    live = dense((codes, s, b))[:, 7] != 0
    assert not torch.isfinite(got[0][live]).any()


def test_linear_on_a_side_stream_and_in_a_graph(cuda):
    for m in (1, 30, 200):
        ws = [make_weight((520, 1024), torch.bfloat16, cuda, seed=i) for i in range(2)]
        q = [pkg.Q4Weight(*w) for w in ws]
        x = make_x(m, 1024, torch.bfloat16, cuda)
        want = expected(x, ws)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            got = pkg.quantized_swiglu(x, *q)
        side.synchronize()
        assert_within(got, *want)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = pkg.quantized_swiglu(x, *q)
        x.copy_(make_x(m, 1024, torch.bfloat16, cuda, seed=77))
        g.replay()
        torch.cuda.synchronize()
        assert_within(got, *expected(x, ws))


def test_linear_repeats_bit_for_bit(cuda):
    for m in (1, 7, 60, 300):
        q = pkg.Q4Weight(*make_weight((1030, 2048), torch.float16, cuda))
        x = make_x(m, 2048, torch.float16, cuda)
        first = pkg.quantized_matmul(x, q)
        for _ in range(3):
            assert torch.equal(first, pkg.quantized_matmul(x, q))


# ----------------------------------------------------------------------------- experts


def routing_of(experts, n_experts):
    """ExpertRouting of chosen experts [tokens, top_k] (plain tensor operations)."""
    flat = experts.flatten().long()
    order = torch.argsort(flat, stable=True)
    pos = torch.empty_like(order)
    pos[order] = torch.arange(order.numel(), device=flat.device)
    off = torch.searchsorted(flat[order], torch.arange(n_experts + 1, device=flat.device))
    w = torch.full(experts.shape, 1.0 / experts.shape[1], device=flat.device)
    i32 = lambda t: t.to(torch.int32)  # noqa: E731
    return pkg.ExpertRouting(i32(experts), w, i32(off), i32(order), i32(pos.view(experts.shape)))


def choose(kind, tokens, n_experts, top_k, dev):
    g = torch.Generator(device="cpu").manual_seed(tokens * 131 + n_experts)
    score = torch.rand(tokens, n_experts, generator=g)
    if kind == "skewed":  # most tokens on the first experts, many experts empty
        score += 2.0 * (torch.arange(n_experts) < max(top_k, n_experts // 4))
    if kind == "one":
        score += 2.0 * (torch.arange(n_experts) >= n_experts - top_k)
    return score.topk(top_k, dim=-1).indices.to(dev)


def expected_experts(x, ws, r, gather):
    order, off = r.order.long(), r.offsets.tolist()
    rows = order.numel()
    y = torch.zeros(rows, ws[0][0].shape[1], dtype=torch.float64, device=x.device)
    e = torch.zeros_like(y)
    top_k = r.experts.shape[1]
    for i in range(len(off) - 1):
        if off[i] < off[i + 1]:
            sl = slice(off[i], off[i + 1])
            y[sl], e[sl] = expected(x[order[sl] // top_k] if gather else x[sl], [[p[i] for p in w] for w in ws])
    return y, e


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", ["even", "skewed", "one"])
@pytest.mark.parametrize("tokens,n_experts,top_k,n,k", [
    (1, 8, 2, 96, 128), (1, 64, 6, 200, 256), (3, 5, 5, 33, 192), (16, 64, 6, 176, 256), (40, 16, 1, 130, 320),
    (100, 32, 4, 260, 704), (256, 8, 2, 129, 448), (600, 4, 2, 300, 384), (513, 1, 1, 80, 128)])
def test_experts(cuda, tokens, n_experts, top_k, n, k, kind, dtype):
    ws = [make_weight((n_experts, n, k), dtype, cuda, seed=i) for i in range(2)]
    q = [pkg.Q4Weight(*w) for w in ws]
    r = routing_of(choose(kind, tokens, n_experts, top_k, cuda), n_experts)
    x = make_x(tokens, k, dtype, cuda)
    assert_within(pkg.expert_swiglu(x, *q, r), *expected_experts(x, ws, r, True), "gated, gathered")
    assert_within(pkg.expert_matmul(x, q[0], r, gather=True), *expected_experts(x, ws[:1], r, True), "gathered")
    xs = make_x(tokens * top_k, k, dtype, cuda, seed=9)
    assert_within(pkg.expert_matmul(xs, q[0], r), *expected_experts(xs, ws[:1], r, False), "sorted")
    assert_within(pkg.expert_swiglu(xs, *q, r, gather=False), *expected_experts(xs, ws, r, False),
                  "gated, sorted")


def test_experts_wide(cuda):
    """Shapes of the expert layers served here: 64 experts of 1408 x 2048, 32 of 2880 x 2880."""
    for tokens, e, k, n, d in ((1, 64, 6, 1408, 2048), (33, 64, 6, 2048, 1408), (150, 32, 4, 2880, 2880)):
        ws = [make_weight((e, n, d), torch.bfloat16, cuda, seed=i) for i in range(2)]
        q = [pkg.Q4Weight(*w) for w in ws]
        r = routing_of(choose("skewed", tokens, e, k, cuda), e)
        x = make_x(tokens, d, torch.bfloat16, cuda)
        assert_within(pkg.expert_swiglu(x, *q, r), *expected_experts(x, ws, r, True))
        assert_within(pkg.expert_matmul(x, q[1], r, gather=True), *expected_experts(x, ws[1:], r, True))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", ["even", "skewed", "one"])
def test_experts_many_rows(cuda, kind, dtype):
    """Hundreds of rows an expert: tiles of pairs of SMs with items of every size."""
    for tokens, e, k, n, d in ((3000, 3, 2, 800, 320), (4000, 8, 1, 1200, 704)):
        ws = [make_weight((e, n, d), dtype, cuda, seed=i) for i in range(2)]
        q = [pkg.Q4Weight(*w) for w in ws]
        r = routing_of(choose(kind, tokens, e, k, cuda), e)
        x = make_x(tokens, d, dtype, cuda)
        assert_within(pkg.expert_swiglu(x, *q, r), *expected_experts(x, ws, r, True))
        assert_within(pkg.expert_matmul(x, q[1], r, gather=True), *expected_experts(x, ws[1:], r, True))


def test_experts_without_tokens(cuda):
    q = pkg.Q4Weight(*make_weight((4, 32, 64), torch.float16, cuda))
    r = routing_of(torch.zeros(0, 2, dtype=torch.int64, device=cuda), 4)
    assert pkg.expert_matmul(torch.empty(0, 64, dtype=torch.float16, device=cuda), q, r).shape == (0, 32)


@pytest.mark.parametrize("tokens", [6, 90, 700])
def test_experts_with_bad_indices(cuda, tokens):
    """Order entries outside x read as zero rows and are flagged; offsets past the rows are
    clamped, and rows that no expert holds stay as they were."""
    n_experts, top_k = 4, 2
    w = make_weight((n_experts, 72, 256), torch.bfloat16, cuda)
    q = pkg.Q4Weight(*w)
    r = routing_of(choose("even", tokens, n_experts, top_k, cuda), n_experts)
    x = make_x(tokens, 256, torch.bfloat16, cuda)
    want, bound = expected_experts(x, [w], r, True)
    order = r.order.clone()
    order[1], order[-2] = tokens * top_k, -5
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    got = pkg.expert_matmul(x, q, r._replace(order=order), gather=True, status=status)
    assert int(status) == pkg._lib.STATUS_BAD_POSITION
    want[[1, -2]], bound[[1, -2]] = 0, 0
    assert_within(got, want, bound)
    off = r.offsets.clone()
    last = int(off[-2])
    off[-1] = last
    out = torch.full((tokens * top_k, 72), 5.0, dtype=torch.bfloat16, device=cuda)
    pkg.expert_matmul(x, q, r._replace(offsets=off), gather=True, out=out)
    assert bool((out[last:] == 5.0).all())
    off[-1] = 10 ** 9
    want, bound = expected_experts(x, [w], r, True)
    assert_within(pkg.expert_matmul(x, q, r._replace(offsets=off), gather=True), want, bound)


# ----------------------------------------------------------------------------- routing, combine


def expected_route(logits, top_k, normalize):
    z = torch.where(torch.isnan(logits), -torch.inf, logits.double())
    idx = torch.argsort(z, dim=-1, descending=True, stable=True)[:, :top_k]
    chosen = torch.gather(z, 1, idx)
    top = z.amax(-1, keepdim=True)

    def e(v):
        return torch.where(v == top, 1.0, torch.exp(v - top)).nan_to_num(0.0)

    w = e(chosen) / e(chosen if normalize else z).sum(-1, keepdim=True)
    return idx, torch.where(top == -torch.inf, 0.0, w)


def check_route(logits, top_k, normalize):
    tokens, n_experts = logits.shape
    r = pkg.route_experts(logits, top_k, normalize=normalize)
    idx, w = expected_route(logits, top_k, normalize)
    assert torch.equal(r.experts.long(), idx)
    # softmax in fp32: expf and the division are within a few ulp, the sum of n terms within n/2
    assert float((r.weights.double() - w).abs().max() if tokens else 0.0) <= (8 + n_experts / 32) * 2.0 ** -24
    ref = routing_of(idx, n_experts)
    for got, want, what in ((r.offsets, ref.offsets, "offsets"), (r.order, ref.order, "order"),
                            (r.positions, ref.positions, "positions")):
        assert torch.equal(got, want), what


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,n_experts,top_k", [(0, 8, 2), (1, 1, 1), (1, 64, 6), (2, 4, 4), (7, 33, 8),
                                                    (31, 32, 1), (100, 128, 8), (257, 256, 4), (1000, 60, 5),
                                                    (4097, 32, 4), (9000, 8, 2), (300, 1024, 32),
                                                    (20001, 64, 6)])
def test_route(cuda, tokens, n_experts, top_k, dtype, normalize):
    g = torch.Generator(device="cpu").manual_seed(tokens + n_experts)
    logits = torch.randn(tokens, n_experts, generator=g).to(dtype).to(cuda)
    check_route(logits, top_k, normalize)


@pytest.mark.parametrize("normalize", [True, False])
def test_route_ties_infinities_and_strides(cuda, normalize):
    g = torch.Generator(device="cpu").manual_seed(3)
    z = torch.randint(-2, 3, (400, 40), generator=g).float().to(cuda)  # many equal logits
    check_route(z, 8, normalize)
    z[3] = -torch.inf                      # nothing to choose: the lowest indices, weights 0
    z[4, 5:] = -torch.inf                  # fewer finite logits than slots
    z[5, 7] = torch.inf
    z[6, [2, 9]] = torch.inf               # infinite logits share the weight
    z[7, 3:30] = torch.nan                 # NaN is never chosen before a number
    z[8] = torch.nan
    z[9] = torch.finfo(torch.float32).min  # the type's lowest value is an ordinary logit
    z[10, ::2] = torch.finfo(torch.float32).min
    z[11] = 0.0
    z[12] = torch.where(torch.arange(40, device=cuda) % 2 == 0, 0.0, -0.0)
    z[13] = torch.finfo(torch.float32).max
    check_route(z, 8, normalize)
    wide = torch.zeros(400, 96, device=cuda)
    wide[:, 8:48] = z
    check_route(wide[:, 8:48], 8, normalize)
    check_route(z.t().contiguous().t(), 8, normalize)
    check_route(torch.zeros(5000, 16, device=cuda), 3, normalize)  # every token the same experts


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,top_k,width", [(0, 2, 64), (1, 1, 1), (1, 6, 2048), (3, 2, 7), (16, 6, 2048),
                                                (65, 8, 345), (500, 4, 2880), (2000, 3, 130), (37, 32, 256)])
def test_combine(cuda, tokens, top_k, width, dtype):
    g = torch.Generator(device="cpu").manual_seed(tokens + width)
    y = torch.randn(tokens * top_k, width, generator=g).to(dtype).to(cuda)
    res = torch.randn(tokens, width, generator=g).to(dtype).to(cuda)
    w = torch.rand(tokens, top_k, generator=g).to(cuda)
    pos = torch.randperm(tokens * top_k, generator=g).to(torch.int32).view(tokens, top_k).to(cuda)
    terms = w.double()[..., None] * y.double()[pos.long()]
    want, bound = terms.sum(1), 2.0 ** -23 * (top_k + 1) * terms.abs().sum(1)
    assert_within(pkg.combine_experts(y, w, pos), want, bound)
    assert_within(pkg.combine_experts(y, w, pos, residual=res), want + res.double(),
                  bound + 2.0 ** -23 * res.double().abs())


def test_combine_strides_and_bad_positions(cuda):
    g = torch.Generator(device="cpu").manual_seed(5)
    for lo in (0, 1, 8):
        y = torch.randn(40, 300, generator=g).bfloat16().to(cuda)[:, lo:lo + 200]
        res = torch.randn(10, 400, generator=g).bfloat16().to(cuda)[:, lo:lo + 200]
        w = torch.rand(10, 4, generator=g).to(cuda)
        pos = torch.randint(0, 40, (10, 4), generator=g).to(torch.int32).to(cuda)  # repeats are allowed
        pos[2, 1], pos[3, 0] = 40, -1
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        got = pkg.combine_experts(y, w, pos, residual=res, status=status)
        assert int(status) == pkg._lib.STATUS_BAD_POSITION
        ok = (pos >= 0) & (pos < 40)
        terms = (w.double() * ok)[..., None] * y.double()[pos.long().clamp(0, 39)]
        assert_within(got, terms.sum(1) + res.double(), 2.0 ** -22 * (terms.abs().sum(1) + res.double().abs()) * 4)


def test_expert_layer_end_to_end(cuda):
    """route -> gated -> down -> combine, against the layer written per token."""
    tokens, e, k, d, inner = 70, 16, 4, 256, 192
    dtype = torch.bfloat16
    g, u = (make_weight((e, inner, d), dtype, cuda, seed=i) for i in range(2))
    dn = make_weight((e, d, inner), dtype, cuda, seed=2)
    x = make_x(tokens, d, dtype, cuda)
    logits = make_x(tokens, e, torch.float32, cuda, seed=4)
    r = pkg.route_experts(logits, k)
    h = pkg.expert_swiglu(x, pkg.Q4Weight(*g), pkg.Q4Weight(*u), r)
    y = pkg.expert_matmul(h, pkg.Q4Weight(*dn), r)
    out = pkg.combine_experts(y, r.weights, r.positions, residual=x)
    wg, wu, wd = dense(g), dense(u), dense(dn)
    idx, w = expected_route(logits, k, True)
    want = x.double().clone()
    size = x.double().abs()
    for j in range(k):
        gj = torch.einsum("td,tid->ti", x.double(), wg[idx[:, j]])
        uj = torch.einsum("td,tid->ti", x.double(), wu[idx[:, j]])
        hj = gj * torch.sigmoid(gj) * uj
        want += w[:, j:j + 1] * torch.einsum("ti,tdi->td", hj, wd[idx[:, j]])
        size += w[:, j:j + 1] * torch.einsum("ti,tdi->td", hj.abs(), wd[idx[:, j]].abs())
    # h and y are rounded to bf16 (2^-8 each) on the way, and h's own sums carry their bounds
    assert bool(((out.double() - want).abs() <= 2.0 ** -6 * size + 2.0 ** -7).all())


# ----------------------------------------------------------------------------- refusals


def test_refusals(cuda):
    w = make_weight((32, 128), torch.bfloat16, cuda)
    q = pkg.Q4Weight(*w)
    qe = pkg.Q4Weight(*make_weight((4, 32, 128), torch.bfloat16, cuda))
    x = make_x(4, 128, torch.bfloat16, cuda)
    r = routing_of(choose("even", 4, 4, 2, cuda), 4)
    with pytest.raises(TypeError):
        pkg.quantized_matmul(x.half(), q)
    with pytest.raises(ValueError):
        pkg.quantized_matmul(x[:, :64], q)
    with pytest.raises(ValueError):
        pkg.quantized_matmul(x.cpu(), q)
    with pytest.raises(ValueError):
        pkg.quantized_matmul(x, qe)
    with pytest.raises(ValueError):
        pkg.expert_matmul(x, q, r, gather=True)
    with pytest.raises(ValueError):
        pkg.expert_matmul(x, qe, r)  # 4 rows, the routing has 8
    with pytest.raises(ValueError):
        pkg.expert_matmul(x, qe, r._replace(offsets=r.offsets[:-1]), gather=True)
    with pytest.raises(ValueError):
        pkg.expert_matmul(x, qe, r._replace(order=r.order.long()), gather=True)
    with pytest.raises(ValueError):
        pkg.quantized_swiglu(x, q, pkg.Q4Weight(*make_weight((48, 128), torch.bfloat16, cuda)))
    with pytest.raises(ValueError):
        pkg.quantized_matmul(x, q, out=torch.empty(4, 33, dtype=torch.bfloat16, device=cuda))
    with pytest.raises(RuntimeError):
        pkg.quantized_matmul(x.clone().requires_grad_(), q)
    with torch.no_grad():
        pkg.quantized_matmul(x.clone().requires_grad_(), q)
    with pytest.raises(ValueError):
        pkg.Q4Weight(w[0], w[1][:, :1], w[2])
    with pytest.raises(TypeError):
        pkg.Q4Weight(w[0], w[1], w[2].half())
    with pytest.raises(TypeError):
        pkg.Q4Weight(w[0].long(), w[1], w[2])
    with pytest.raises(NotImplementedError):
        pkg.Q4Weight(*w, group_size=32)
    for logits, k in ((x, 0), (x, 200), (x[0], 2), (torch.zeros(2, 1100, device=cuda), 2),
                      (torch.zeros(2, 64, device=cuda), 40)):
        with pytest.raises(ValueError):
            pkg.route_experts(logits, k)
    with pytest.raises(TypeError):
        pkg.route_experts(torch.zeros(2, 8, dtype=torch.float64, device=cuda), 2)
    y, wt, pos = x, torch.ones(2, 2, device=cuda), torch.zeros(2, 2, dtype=torch.int32, device=cuda)
    with pytest.raises(ValueError):
        pkg.combine_experts(y, wt.half(), pos)
    with pytest.raises(ValueError):
        pkg.combine_experts(y, wt, pos.long())
    with pytest.raises(TypeError):
        pkg.combine_experts(y.float(), wt, pos)
    with pytest.raises(ValueError):
        pkg.combine_experts(y, wt, pos, residual=y)
