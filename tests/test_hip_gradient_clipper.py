"""Global gradient norm and clipping against the definition in 64 bits.

Tolerances: squares and their sums are doubles; n terms in any order are off by at most n 2^-53 relative
(n <= 2^24 here), the root halves that.  A clipped element is one product in double, rounded
once to its type (for float16 and bfloat16 by way of float32: 2^-24 more), half a step of that type
and half its smallest subnormal; the factor carries the norm's error."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float64, torch.float16, torch.bfloat16]
SMALLEST = {torch.float32: 2.0**-149, torch.float64: 2.0**-1074, torch.float16: 2.0**-24, torch.bfloat16: 2.0**-133}


def _norm(grads):
    return math.sqrt(math.fsum(float((g.double().cpu() ** 2).sum()) for g in grads))


def _check(norm, clipped, grads, max_norm):
    want = _norm(grads)
    assert norm.dtype == torch.float64 and norm.shape == ()
    assert abs(float(norm) - want) <= 2.0**-28 * want
    factor = max_norm / want if want > max_norm else 1.0
    for got, g in zip(clipped, grads):
        assert got.dtype == g.dtype and got.shape == g.shape
        exact = g.double().cpu() * factor
        slack = (torch.finfo(g.dtype).eps / 2 + (2.0**-23 if g.dtype != torch.float64 else 2.0**-28)) * exact.abs()
        assert torch.all((got.double().cpu() - exact).abs() <= slack + SMALLEST[g.dtype])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("sizes", [[1], [3], [0, 5, 0], [64] * 40, [4095, 4096, 4097, 1], [8192, 100003, 2, 65536]],
                         ids=str)
@pytest.mark.parametrize("max_norm", [0.01, 1e6])
def test_follows_the_definition(sizes, dtype, max_norm):
    from bayesiannetwork_amd.optimizers import HipGradientClipper

    gen = torch.Generator().manual_seed(len(sizes))
    grads = [torch.randn((n,), generator=gen).to(dtype).cuda() for n in sizes]
    before = [g.clone() for g in grads]
    out = [torch.full_like(g, 9.0) for g in grads]
    clipper = HipGradientClipper(grads, out=out)
    norm = clipper.clip(max_norm)
    _check(norm, out, before, max_norm)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))  # the gradients stay
    assert torch.equal(clipper.norm(), norm)
    if max_norm > 1:
        assert all(torch.equal(a, b) for a, b in zip(out, before))
    in_place = HipGradientClipper(grads)
    assert torch.equal(in_place.clip(max_norm), norm)
    assert all(torch.equal(a, b) for a, b in zip(grads, out))


def test_types_and_places_mixed():
    """Types side by side, slices of one buffer at odd places, gaps that stay as they were."""
    from bayesiannetwork_amd.optimizers import HipGradientClipper

    gen = torch.Generator().manual_seed(6)
    flat = torch.randn((70001,), generator=gen).cuda()
    half = torch.randn((40003,), generator=gen).half().cuda()
    grads = [flat[1:9], flat[9:5000], half[1:20001], flat[5003:70001], half[20001:20002],
             torch.randn((50, 3), generator=gen).double().cuda(), torch.randn((9, 9), generator=gen).bfloat16().cuda(),
             flat[5000:5001], half[20010:]]
    copies = [g.clone() for g in grads]
    kept = (flat.clone(), half.clone())
    norm = HipGradientClipper(grads).clip(0.5)
    _check(norm, grads, copies, 0.5)
    assert torch.equal(flat[0], kept[0][0]) and torch.equal(flat[5001:5003], kept[0][5001:5003])
    assert torch.equal(half[0], kept[1][0]) and torch.equal(half[20002:20010], kept[1][20002:20010])


def test_tables_of_a_network_and_no_dependence_on_the_cut():
    """785 tables, apart and as slices of one buffer: the same norm to rounding, and the same bits from
    call to call."""
    from bayesiannetwork_amd.optimizers import HipGradientClipper

    gen = torch.Generator().manual_seed(8)
    flat = torch.randn((784 * 20 + 10,), generator=gen).cuda()
    slices = list(torch.split(flat, [20] * 784 + [10]))
    apart = [s.clone() for s in slices]
    a, b = HipGradientClipper(slices), HipGradientClipper(apart)
    first = b.norm()
    assert all(torch.equal(first, b.norm()) for _ in range(5))
    assert abs(float(a.norm()) - float(first)) <= 1e-13 * float(first)
    _check(a.clip(1.0), slices, apart, 1.0)


def test_values_that_are_no_numbers_and_extremes():
    from bayesiannetwork_amd.optimizers import HipGradientClipper

    inf, nan = float("inf"), float("nan")
    grads = [torch.tensor([1.0, nan, 2.0]).cuda(), torch.ones(5).half().cuda()]
    assert math.isnan(float(HipGradientClipper(grads).clip(1.0)))
    assert all(torch.isnan(g).all() for g in grads)
    grads = [torch.tensor([1.0, -inf]).cuda(), torch.ones(5).cuda()]
    assert float(HipGradientClipper(grads).clip(1.0)) == inf
    assert torch.isnan(grads[0][1]) and float(grads[0][0]) == 0 and (grads[1] == 0).all()
    big = [torch.full((4,), 3e38).cuda()]  # the squares overflow float32
    copies = [big[0].clone()]
    _check(HipGradientClipper(big).clip(1.0), big, copies, 1.0)
    tiny = [torch.full((4,), 1e-40).cuda(), torch.zeros(3).cuda()]
    copies = [t.clone() for t in tiny]
    _check(HipGradientClipper(tiny).clip(1.0), tiny, copies, 1.0)
    zero = [torch.zeros(3).cuda()]
    assert float(HipGradientClipper(zero).clip(1.0)) == 0 and (zero[0] == 0).all()
    empty = [torch.zeros(0).cuda()]
    assert float(HipGradientClipper(empty).clip(1.0)) == 0


def test_refusals():
    from bayesiannetwork_amd.optimizers import HipGradientClipper

    g = torch.zeros((4, 4), device="cuda")
    for call, error in [
        (lambda: HipGradientClipper([g, g]), RuntimeError),
        (lambda: HipGradientClipper([g[:, :2]]), ValueError),
        (lambda: HipGradientClipper([g.t()]), ValueError),
        (lambda: HipGradientClipper([g], out=[g.double()]), ValueError),
        (lambda: HipGradientClipper([g], out=[]), ValueError),
        (lambda: HipGradientClipper([g[:2]], out=[g[1:3]]), RuntimeError),
        (lambda: HipGradientClipper([g, g.cpu()]), ValueError),
        (lambda: HipGradientClipper([g]).clip(0.0), ValueError),
        (lambda: HipGradientClipper([g]).clip(float("inf")), ValueError),
        (lambda: HipGradientClipper([g]).clip(float("nan")), ValueError),
    ]:
        with pytest.raises(error):
            call()


def test_captured():
    from bayesiannetwork_amd.optimizers import HipGradientClipper

    gen = torch.Generator().manual_seed(3)
    grads = [torch.randn((n,), generator=gen).cuda() for n in (7, 30000, 1)]
    out = [torch.empty_like(g) for g in grads]
    clipper = HipGradientClipper(grads, out=out)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        clipper.clip(2.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        norm = clipper.clip(2.0)
    for _ in range(4):
        for g in grads:
            g.copy_(torch.randn(g.shape, generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        kept = [o.clone() for o in out]
        assert torch.equal(clipper.clip(2.0), norm)
        assert all(torch.equal(a, b) for a, b in zip(kept, out))
        _check(norm, kept, grads, 2.0)


def test_learning_a_conditional_model():
    """The operators together, as a discriminative step uses them: log-likelihood of the observed
    states under a linear model of each node's states, its gradient through autograd, the global norm
    clipped, an update, and draws from the updated rows."""
    from bayesiannetwork_amd.optimizers import HipGradientClipper, states_log_likelihood
    from bayesiannetwork_amd.samplers import draw_states

    gen = torch.Generator().manual_seed(12)
    features = torch.randn((500, 6), generator=gen, dtype=torch.float64)
    states = [torch.randint(0, n, (500,), generator=gen) for n in (3, 7)]
    weights = [torch.randn((6, n), generator=gen, dtype=torch.float64) for n in (3, 7)]

    device = [w.cuda().requires_grad_(True) for w in weights]
    loss = -sum(states_log_likelihood(features.cuda() @ w, s.cuda()).mean() for w, s in zip(device, states))
    loss.backward()
    want = []
    for w, s in zip(weights, states):
        p = torch.softmax(features @ w, dim=1)
        p[torch.arange(500), s] -= 1.0
        want.append(features.t() @ p / 500)
    for d, g in zip(device, want):
        assert torch.allclose(d.grad.cpu(), g, rtol=1e-12, atol=1e-14)
    norm = HipGradientClipper([d.grad for d in device]).clip(0.1)
    assert abs(float(norm) - _norm(want)) < 1e-12
    factor = min(1.0, 0.1 / _norm(want))
    for d, g in zip(device, want):
        assert torch.allclose(d.grad.cpu(), g * factor, rtol=1e-12, atol=1e-14)
    with torch.no_grad():
        for d in device:
            d -= d.grad
    rows = features.cuda() @ device[1].detach()
    u = torch.rand((500,), generator=gen, dtype=torch.float64)
    got = draw_states(rows, u.cuda(), top_p=0.9)
    assert int(got.min()) >= 0 and int(got.max()) < 7
    upto = torch.cumsum(torch.softmax(rows.cpu(), dim=1), dim=1)
    plain = draw_states(rows, u.cuda())
    assert torch.equal(plain.cpu().long(), (upto <= u[:, None] * upto[:, -1:]).sum(dim=1))


def test_a_backward_pass_that_needs_unclipped_gradients_raises():
    from bayesiannetwork_amd.optimizers import HipGradientClipper

    x = torch.randn((50,), generator=torch.Generator().manual_seed(1)).cuda()
    for make in (lambda: x.clone(), lambda: x.clone()[3:40], lambda: torch.split(x.clone(), [20, 30])[1]):
        g = make()
        factor = torch.ones_like(g, requires_grad=True)
        product = factor * g  # keeps g
        clipper = HipGradientClipper([g])
        clipper.norm()
        product.sum().backward(retain_graph=True)
        assert torch.equal(factor.grad, g)
        clipper.clip(1e9)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            product.sum().backward()
    # clipped copies elsewhere: the gradients stay as they are, the copies' buffer is the one that changes
    grads = [x.clone(), x.clone()]
    flat = torch.empty((100,), device="cuda")
    versions = [g._version for g in grads] + [flat._version]
    HipGradientClipper(grads, out=list(torch.split(flat, [50, 50]))).clip(1.0)
    assert [g._version for g in grads] == versions[:2] and flat._version > versions[2]
    with torch.inference_mode():
        HipGradientClipper([x.clone()]).clip(1.0)


@pytest.mark.parametrize("size", [1e200, 1e154, 1e-160, 1e-200, 1e-306, 1e300])
@pytest.mark.parametrize("others", [False, True], ids=["float64", "mixed"])
@pytest.mark.parametrize("max_norm", [1.0, 1e-3, 1e-280, 1e250])
def test_float64_gradients_whose_squares_leave_the_range(size, others, max_norm):
    """Expected from exact integers (every double is one times 2^-1074).  64 squares and their sum, whose scaling by
    a power of two is exact, are off by 66 2^-53 at most, the root by half of that and its own rounding: 2^-47; an
    element by that, three roundings and half the smallest subnormal."""
    from fractions import Fraction

    from bayesiannetwork_amd.optimizers import HipGradientClipper

    gen = torch.Generator().manual_seed(5)
    big = torch.rand((64,), generator=gen, dtype=torch.float64) * size
    grads = [big.cuda()]
    if others:  # what other types hold next to them does not count, unless it is all there is
        grads += [torch.zeros((5,)).cuda() if size < 1 else torch.ones((5,)).cuda(), torch.zeros((3,)).bfloat16().cuda()]
    unit = Fraction(1, 2**1074)
    total = sum((Fraction(float(v)) / unit) ** 2 for g in grads for v in g.double().cpu())
    norm_units = math.isqrt(int(total))  # of 2^-1074: 18 digits at the least
    exact_norm = Fraction(norm_units) * unit
    out = [torch.empty_like(g) for g in grads]
    clipper = HipGradientClipper(grads, out=out)
    norm = clipper.clip(max_norm)
    assert torch.equal(norm, clipper.norm())
    assert abs(Fraction(float(norm)) - exact_norm) <= exact_norm * Fraction(2.0**-47) + unit
    factor = min(Fraction(1), Fraction(max_norm) / exact_norm)
    for v, o in zip(big.tolist(), out[0].cpu().tolist()):
        want = Fraction(v) * factor
        assert abs(Fraction(o) - want) <= want * (Fraction(2.0**-47) + Fraction(2.0**-51)) + unit


def test_a_clipper_that_goes_while_a_graph_is_captured():
    from bayesiannetwork_amd.optimizers import HipGradientClipper

    gen = torch.Generator().manual_seed(4)
    grads = [torch.randn((n,), generator=gen).cuda() for n in (7, 30000)]
    out = [torch.empty_like(g) for g in grads]
    clipper, other = HipGradientClipper(grads, out=out), HipGradientClipper([g.clone() for g in grads])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        clipper.clip(2.0)
        other.clip(2.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        del other
        norm = clipper.clip(2.0)
    for _ in range(3):
        for g in grads:
            g.copy_(torch.randn(g.shape, generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        _check(norm, out, grads, 2.0)
