"""4-bit linear and expert calls at the edges of what they take: many inputs, unusual rows, infinities."""

import pytest
import torch

from conftest import pkg
from test_gpu_linear import (GROUP, assert_within, dense, expected, expected_experts, make_weight, make_x, product,
                             routing_of, run)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,k", [(1, 49216), (4, 53248), (5, 14336), (8, 14336), (5, 49152), (5, 49216),
                                      (8, 49152), (8, 53248), (9, 53248), (3, 69632), (2, 139264), (1, 278528)])
def test_many_inputs(cuda, tokens, k):
    """Few tokens of more inputs than a CTA, a cluster of 4 or 8, or the few-token kernel holds."""
    w = make_weight((48, k), torch.bfloat16, cuda)
    x = make_x(tokens, k, torch.bfloat16, cuda)
    assert_within(run(x, [w]), *expected(x, [w]))


@pytest.mark.parametrize("tokens,k", [(2, 139264), (4, 69632), (8, 14336), (5, 32768), (5, 32832), (8, 53248)])
def test_many_inputs_gated(cuda, tokens, k):
    ws = [make_weight((40, k), torch.float16, cuda, seed=i, scale=0.002) for i in range(2)]
    x = make_x(tokens, k, torch.float16, cuda)
    assert_within(run(x, ws), *expected(x, ws))


def test_many_inputs_of_experts(cuda):
    n_experts, k = 3, 139264
    ws = [make_weight((n_experts, 24, k), torch.float16, cuda, seed=i, scale=0.002) for i in range(2)]
    q = [pkg.Q4Weight(*w) for w in ws]
    for tokens in (1, 3, 6):
        r = routing_of((torch.arange(tokens, device=cuda) % n_experts)[:, None], n_experts)
        x = make_x(tokens, k, torch.float16, cuda)
        assert_within(pkg.expert_swiglu(x, *q, r), *expected_experts(x, ws, r, True))
        assert_within(pkg.expert_matmul(x, q[0], r, gather=True), *expected_experts(x, ws[:1], r, True))


@pytest.mark.parametrize("tokens", [2, 8, 40, 300])
def test_rows_that_share_memory(cuda, tokens):
    """A broadcast token (row stride 0) and overlapping windows of one sequence (row stride 64)."""
    w, up = (make_weight((48, 256), torch.bfloat16, cuda, seed=i) for i in range(2))
    experts = make_weight((3, 48, 256), torch.bfloat16, cuda)
    r = routing_of((torch.arange(tokens, device=cuda) % 3)[:, None], 3)
    flat = make_x(1, 256 + 64 * tokens, torch.bfloat16, cuda).flatten()
    for x in (flat[:256].expand(tokens, -1), flat.as_strided((tokens, 256), (64, 1)), flat[64:320].expand(2, tokens, -1)):
        assert_within(run(x, [w]), *expected(x, [w]), str(x.stride()))
        assert_within(run(x, [w, up]), *expected(x, [w, up]), str(x.stride()))
        if x.dim() == 2:
            got = pkg.expert_matmul(x, pkg.Q4Weight(*experts), r, gather=True)
            assert_within(got, *expected_experts(x, [experts], r, True), str(x.stride()))


@pytest.mark.parametrize("tokens,n,gated", [(40, 512, False), (40, 40960, False), (100, 600, True), (600, 8448, True),
                                            (1500, 4352, False)])
def test_a_linear_call_reports_waits_that_ran_out(cuda, monkeypatch, tokens, n, gated):
    """Tiles of one SM (split over a cluster and not) and of pairs of SMs whose waits give up at once say so
    in the caller's status word; the next call is right and leaves it alone."""
    ws = [make_weight((n, 640), torch.float16, cuda, seed=i) for i in range(1 + gated)]
    q = [pkg.Q4Weight(*w) for w in ws]
    x = make_x(tokens, 640, torch.float16, cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    f = lambda: (pkg.quantized_swiglu if gated else pkg.quantized_matmul)(x, *q, status=status)  # noqa: E731
    monkeypatch.setenv("AM_Q4_TEST_WAIT_LIMIT_NS", "0")
    f()
    torch.cuda.synchronize(cuda)
    assert int(status.item()) == pkg._lib.STATUS_TIMEOUT
    monkeypatch.delenv("AM_Q4_TEST_WAIT_LIMIT_NS")
    status.zero_()
    assert_within(f(), *expected(x, ws))
    assert int(status.item()) == 0
    for bad in (status.long(), status.cpu(), status[:0]):
        with pytest.raises(ValueError):
            pkg.quantized_matmul(x, q[0], status=bad)


@pytest.mark.parametrize("tokens", [20, 40, 100])
@pytest.mark.parametrize("gated", [False, True])
def test_a_split_tile_that_gave_up_stores_nothing(cuda, monkeypatch, tokens, gated):
    """Clusters of 8, 4 and 2 that split the inputs: no unfinished sum reaches the output."""
    for n in (256, 2048, 8192):
        ws = [make_weight((n, 2048), torch.bfloat16, cuda, seed=i) for i in range(1 + gated)]
        q = [pkg.Q4Weight(*w) for w in ws]
        x = make_x(tokens, 2048, torch.bfloat16, cuda)
        out = torch.empty(tokens, n, dtype=torch.bfloat16, device=cuda)
        f = lambda: (pkg.quantized_swiglu if gated else pkg.quantized_matmul)(x, *q, out=out)  # noqa: E731
        assert_within(f(), *expected(x, ws))
        out.fill_(7.0)
        monkeypatch.setenv("AM_Q4_TEST_WAIT_LIMIT_NS", "0")
        f()
        torch.cuda.synchronize(cuda)
        monkeypatch.delenv("AM_Q4_TEST_WAIT_LIMIT_NS")
        assert bool((out == 7.0).all())
        assert_within(f(), *expected(x, ws))


@pytest.mark.parametrize("tokens", [1, 4, 8, 40])
def test_an_output_on_the_memory_of_the_input_is_refused(cuda, tokens):
    k = 256
    w = make_weight((k, k), torch.bfloat16, cuda)
    q = pkg.Q4Weight(*w)
    qe = pkg.Q4Weight(*make_weight((1, k, k), torch.bfloat16, cuda))
    r = routing_of(torch.zeros(tokens, 1, dtype=torch.int64, device=cuda), 1)
    buf = make_x(2 * tokens + 1, k, torch.bfloat16, cuda)
    x = buf[:tokens]
    for out in (x, buf[tokens - 1:2 * tokens - 1], buf.flatten()[8:8 + x.numel()].view(tokens, k)):
        for call in (lambda: pkg.quantized_matmul(x, q, out=out), lambda: pkg.quantized_swiglu(x, q, q, out=out),
                     lambda: pkg.expert_matmul(x, qe, r, out=out)):
            with pytest.raises(ValueError, match="shares memory"):
                call()
    want = expected(x, [w])
    assert_within(pkg.quantized_matmul(x, q, out=buf[tokens:2 * tokens]), *want)  # right behind x
    wide = make_x(2, 4 * k, torch.bfloat16, cuda)
    gap = wide.flatten()[k:2 * k].view(1, k)  # between two rows of a strided x
    assert_within(pkg.quantized_matmul(wide[:1, :k], q, out=gap), *expected(wide[:1, :k], [w]))
    every_other = make_x(tokens, 2 * k, torch.bfloat16, cuda)[:, ::2]  # copied: an output on it is no matter
    want = expected(every_other, [w])
    out = every_other._base.flatten()[:tokens * k].view(tokens, k) if every_other._base is not None else None
    assert_within(pkg.quantized_matmul(every_other, q, out=out), *want)


def test_a_combination_onto_its_inputs(cuda):
    y = make_x(12, 64, torch.float16, cuda)
    w = torch.rand(6, 2, device=cuda)
    pos = torch.arange(12, dtype=torch.int32, device=cuda).view(6, 2)
    res = make_x(7, 64, torch.float16, cuda, seed=3)
    want = pkg.combine_experts(y, w, pos, residual=res[:6])
    with pytest.raises(ValueError, match="shares memory with y"):
        pkg.combine_experts(y, w, pos, out=y[3:9])
    with pytest.raises(ValueError, match="residual"):
        pkg.combine_experts(y, w, pos, residual=res[:6], out=res[1:])
    assert torch.equal(pkg.combine_experts(y, w, pos, residual=res[:6], out=res[:6]), want)


def spread_weight(n, k, dtype, dev, r, seed=0):
    """A weight whose first group's scales and biases are 2^r times the others'."""
    codes, s, b = make_weight((n, k), torch.float32, dev, seed=seed, scale=0.25)
    f = torch.full((k // GROUP,), 2.0 ** -r, device=dev)
    f[0] = 1.0
    return codes, (s * f).to(dtype), (b * f).to(dtype)


SPREADS = [(torch.float16, 6), (torch.float16, 10), (torch.float16, 14), (torch.float16, 18),
           (torch.bfloat16, 8), (torch.bfloat16, 14), (torch.bfloat16, 20), (torch.bfloat16, 24)]


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("dtype,r", SPREADS)
def test_groups_far_below_their_rows_largest(cuda, dtype, r, gated):
    """Activations of zero at a row's largest group leave the small groups alone to count.  Few tokens
    multiply them exactly; the tiles round a weight to 11 bits or to 2^-14 of the row's largest scale
    (two parts: 2^-12), which is more than their few bits below 2^-10 of it."""
    n, k = 72, 320
    ws = [spread_weight(n, k, dtype, cuda, r, seed=i) for i in range(1 + gated)]
    q = [pkg.Q4Weight(*w) for w in ws]
    for tokens in (1, 2, 4, 7, 8, 9, 40, 150, 600):
        x = (make_x(tokens, k, torch.float32, cuda, seed=tokens) * 2.0 ** min(r, 12)).to(dtype)  # (fp16: finite)
        x[:, :GROUP] = 0
        tiles = tokens > 8
        largest = torch.stack([w[1].double().abs().amax(-1).maximum(w[2].double().abs().amax(-1) / 16) for w in ws])
        floor = largest * (0.0 if not tiles else 2.0 ** -12 if gated and dtype == torch.float16 else 2.0 ** -14)
        size = x.double().abs().sum(-1, keepdim=True)
        y, e = product(x, ws[0])
        e = e + floor[0] * size
        if gated:
            u, eu = product(x, ws[1])
            eu = eu + floor[1] * size
            s = y * torch.sigmoid(y)
            y, e = s * u, 1.1 * e * (u.abs() + eu) + s.abs() * eu + 2.0 ** -20 * (s * u).abs()
        got = pkg.quantized_swiglu(x, *q) if gated else pkg.quantized_matmul(x, *q)
        assert_within(got, y, e, f"{tokens} tokens, 2^-{r}")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("ratio", [0.0, 1.0, 16.0, 64.0, 1024.0])
def test_biases_of_every_size_beside_their_scales(cuda, dtype, ratio):
    """Rows that are all scale, and rows that are nearly all bias (weights far from zero)."""
    codes, s, _ = make_weight((72, 320), torch.float32, cuda, scale=2.0 ** -10)
    g = torch.Generator(device="cpu").manual_seed(9)
    b = s * ratio * (0.5 + torch.rand(s.shape, generator=g).to(cuda))
    w = codes, s.to(dtype), b.to(dtype)
    for tokens in (1, 5, 12, 200):
        x = make_x(tokens, 320, dtype, cuda)
        assert_within(run(x, [w]), *expected(x, [w]), f"{tokens} tokens, bias / scale {ratio}")


def formula(x, ws):
    """The layer as it is defined, infinities and NaN with it: sums in 64 bits over the tokens' own values."""
    y = x.double() @ dense(ws[0]).mT
    return y / (1 + torch.exp(-y)) * (x.double() @ dense(ws[1]).mT) if len(ws) == 2 else y


def put_nonfinite(x):
    """Tokens with one infinity, two of both signs, a NaN, and one of each at the ends."""
    inf, k = float("inf"), x.shape[1]
    at = [(0, [(7, inf)]), (1, [(k - 1, -inf)]), (2, [(64, inf), (65, -inf)]), (4, [(3, float("nan"))]),
          (5, [(0, -inf), (k - 2, -inf)]), (x.shape[0] - 1, [(100, inf)])]
    for row, values in at:
        for col, v in values if row < x.shape[0] else ():
            x[row, col] = v
    return ~torch.isfinite(x).all(-1)


def assert_same_kind(got, want):
    same = (got.double() == want) | (torch.isnan(got) & torch.isnan(want))
    assert bool(same.all()), f"{int((~same).sum())} of {same.numel()} differ: {got[~same][:4]} for {want[~same][:4]}"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("tokens,n,k", [(1, 130, 320), (2, 130, 14336), (4, 130, 320), (8, 300, 14336), (20, 130, 704),
                                        (40, 4100, 320), (60, 40000, 320), (150, 1030, 1344), (700, 8450, 320)])
def test_infinities_and_nan_as_the_formula_has_them(cuda, tokens, n, k, gated, dtype):
    """A token with infinite or NaN activations gives the infinities and NaN of the formula in every
    kernel (few tokens, tiles split and whole, pairs); the other tokens do not notice.  Some
    weights are zero."""
    ws = [make_weight((n, k), dtype, cuda, seed=i) for i in range(1 + gated)]
    for _, s, b in ws:
        s[3], b[3] = 0, 0
        s[5, 1], b[5, 1] = 0, 0
        b[7] = -3 * s[7]
    x = make_x(tokens, k, dtype, cuda)
    clean = x.clone()
    bad = put_nonfinite(x)
    got = run(x, ws)
    assert_same_kind(got[bad], formula(x[bad], ws))
    want, bound = expected(clean[~bad], ws)
    assert_within(got[~bad], want, bound)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens", [6, 60, 2400])
def test_infinities_and_nan_through_experts(cuda, tokens, dtype):
    n_experts, n, k = 6, 700, 320
    ws = [make_weight((n_experts, n, k), dtype, cuda, seed=i) for i in range(2)]
    q = [pkg.Q4Weight(*w) for w in ws]
    r = routing_of((torch.arange(tokens, device=cuda) % n_experts)[:, None], n_experts)
    x = make_x(tokens, k, dtype, cuda)
    bad = put_nonfinite(x)
    for many in (1, 2):
        got = pkg.expert_swiglu(x, *q, r) if many == 2 else pkg.expert_matmul(x, q[0], r, gather=True)
        for t in torch.nonzero(bad)[:, 0].tolist():
            e = int(r.experts[t, 0])
            want = formula(x[t:t + 1], [[p[e] for p in w] for w in ws[:many]])
            assert_same_kind(got[r.positions[t].long()], want)
        keep = ~bad[r.order.long()]
        want, bound = expected_experts(x.masked_fill(bad[:, None], 0), ws[:many], r, True)
        assert_within(got[keep], want[keep], bound[keep])


@pytest.mark.parametrize("tokens", [8, 100, 1024])
def test_tokens_of_nothing_but_nan_or_infinity(cuda, tokens):
    """Every token: all NaN, all infinite, or finite (the calls end in ordinary time)."""
    ws = [make_weight((2304, 1024), torch.float16, cuda, seed=i) for i in range(2)]
    x = make_x(tokens, 1024, torch.float16, cuda)
    x[0::3] = float("nan")
    x[1::3] = float("inf")
    got = run(x, ws)
    bad = ~torch.isfinite(x).all(-1)
    assert_same_kind(got[bad], formula(x[bad], ws))
    want, bound = expected(x[~bad], ws)
    assert_within(got[~bad], want, bound)


@pytest.mark.parametrize("tokens", [6, 90, 700])
def test_order_entries_of_rows_that_no_expert_holds(cuda, tokens):
    """Offsets that leave rows out at both ends, whose order entries point nowhere: no status bit, the
    rows stay as they were, the others are right."""
    n_experts, top_k = 4, 2
    ws = [make_weight((n_experts, 72, 256), torch.bfloat16, cuda, seed=i) for i in range(2)]
    q = [pkg.Q4Weight(*w) for w in ws]
    r = routing_of(torch.stack([torch.arange(tokens, device=cuda) % n_experts,
                                (torch.arange(tokens, device=cuda) + 1) % n_experts], 1), n_experts)
    x = make_x(tokens, 256, torch.bfloat16, cuda)
    off, order = r.offsets.clone(), r.order.clone()
    lo, hi = int(off[1]), int(off[-2])
    off[0], off[-1] = lo, hi
    order[:lo], order[hi:] = -1, 10 ** 9
    r2 = r._replace(offsets=off, order=order)
    for many in (1, 2):
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        out = torch.full((2 * tokens, 72), 5.0, dtype=torch.bfloat16, device=cuda)
        if many == 2:
            pkg.expert_swiglu(x, *q, r2, out=out, status=status)
        else:
            pkg.expert_matmul(x, q[0], r2, gather=True, out=out, status=status)
        want, bound = expected_experts(x, ws[:many], r, True)
        assert_within(out[lo:hi], want[lo:hi], bound[lo:hi])
        assert bool((out[:lo] == 5.0).all()) and bool((out[hi:] == 5.0).all())
        assert int(status) == 0


def test_a_combination_of_two_billion_tokens(cuda):
    """As many tokens as the interface can count (the walk over them passes 31 bits)."""
    tokens = 2 ** 31 - 1
    if torch.cuda.mem_get_info(cuda)[0] < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    y = torch.full((3, 1), 1.5, dtype=torch.float16, device=cuda)
    w = torch.full((1, 1), 2.0, device=cuda).expand(tokens, 1).contiguous()
    pos = torch.ones(tokens, 1, dtype=torch.int32, device=cuda)
    pos[-1] = 7  # out of range: adds nothing
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = pkg.combine_experts(y, w, pos, status=status)
    assert bool((out[:-1] == 3.0).all()) and float(out[-1]) == 0.0
    assert int(status) == pkg._lib.STATUS_BAD_POSITION
    del y, w, pos, out
    torch.cuda.empty_cache()
