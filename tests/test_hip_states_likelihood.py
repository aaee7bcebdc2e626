"""Log-likelihoods of rows' states and their gradients against the definition in 64 bits.

Tolerances.  Values are carried in float32 (float64 for float64 logits); with eps = 2^-24 for one float32
rounding (2^-53 for double):
 * log-likelihood: every term exp(x - max) is off by eps (|x - max| log2(e) + 2) relative - the
   argument's roundings, the exponential's last bit - which weights e^-|x - max| keep below 3 eps
   of the sum; the sum of n terms in a tree of at most depth d adds d eps, where a lane adds at most
   n / 64 terms one after the other.  log(sum) and the differences are taken in double and rounded once:
   |error| <= (n / 64 + 16) eps + eps |ll|, with n / 64 at most 512 for the lengths here.
 * gradient: the same relative error of a softmax value p, plus that of its exponential's argument, whose
   roundings grow with |x - L| <= 40: (n / 64 + 16 + 60 + 4) eps p, then one rounding of the weight's product
   and one to the stored type (half a step, and half the smallest subnormal)."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float64, torch.float16, torch.bfloat16]
SMALLEST = {torch.float32: 2.0**-149, torch.float64: 2.0**-1074, torch.float16: 2.0**-24, torch.bfloat16: 2.0**-133}


def _definition(x, states, weights, counts):
    """ll and gradient in float64, row by row; columns beyond a row's states are 0."""
    x = x.double()
    ll = torch.zeros((x.shape[0],), dtype=torch.float64)
    gradient = torch.zeros_like(x)
    p_all = torch.zeros_like(x)
    for r in range(x.shape[0]):
        n = max(0, min(int(counts[r]), x.shape[1]))
        s = int(states[r])
        if not 0 <= s < n:
            continue
        row = x[r, :n]
        if torch.isnan(row).any() or torch.isposinf(row).any():
            ll[r] = float("nan")
            gradient[r, :n] = float("nan")
            continue
        if torch.isneginf(row).all():
            ll[r] = -float("inf")
            continue
        # the largest logit goes first: next to one of 3e38 a double keeps nothing of log(sum)
        row = row - row.max()
        total = torch.logsumexp(row, dim=0)
        ll[r] = row[s] - total
        p = torch.exp(row - total)
        p_all[r, :n] = p
        gradient[r, :n] = -weights[r].double() * p
        gradient[r, s] += weights[r].double()
    return ll, gradient, p_all


def _check(ll, gradient, x, states, weights, counts):
    dtype, n = x.dtype, x.shape[1]
    eps = 2.0**-53 if dtype == torch.float64 else 2.0**-24
    want_ll, want, p = _definition(x, states, weights, counts)
    want_ll = want_ll.to(ll.dtype).double()  # one below the type's range is -inf in it
    assert ll.dtype == (torch.float64 if dtype == torch.float64 else torch.float32)
    depth = n / 64 + 16
    got = ll.detach().cpu().double()
    same = (got == want_ll) | (torch.isnan(got) & torch.isnan(want_ll))
    assert torch.all(same | ((got - want_ll).abs() <= depth * eps + eps * want_ll.abs()))
    if gradient is None:
        return
    assert gradient.dtype == dtype and gradient.shape == x.shape
    got = gradient.cpu().double()
    slack = weights.double().abs()[:, None] * (depth + 64) * eps * p + (torch.finfo(dtype).eps / 2 + 2 * eps) * want.abs() + SMALLEST[dtype]
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    bad = ~(same | ((got - want).abs() <= slack))
    assert not bad.any(), (bad.nonzero()[:5], got[bad][:5], want[bad][:5])


def _inputs(rows, n, dtype, seed, ragged):
    gen = torch.Generator().manual_seed(seed)
    x = (3.0 * torch.randn((rows, n), generator=gen)).to(dtype)
    states = torch.randint(0, n, (rows,), generator=gen)
    states[0] = -1  # not observed
    if rows > 2:
        states[1], states[2] = n + 4, 0
    weights = (torch.rand((rows,), generator=gen, dtype=torch.float64) - 0.3).to(
        torch.float64 if dtype == torch.float64 else torch.float32)
    counts = torch.full((rows,), n)
    if ragged:
        counts = torch.randint(0, n + 3, (rows,), generator=gen)
        for r in range(rows):
            x[r, int(counts[r]):] = [float("nan"), float("inf"), -1.0][r % 3]
    return x, states, weights, counts


@pytest.mark.parametrize("ragged", [False, True], ids=["full", "ragged"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 8, 9, 16, 31, 64, 65, 127, 256, 257, 511, 1000, 1024, 1025, 2048, 2049,
                               4096, 4097, 8191, 32768])
def test_follows_the_definition(n, dtype, ragged):
    from bayesiannetwork_amd.optimizers import states_log_likelihood, states_log_likelihood_and_gradient

    rows = 33 if n < 3000 else 7
    x, states, weights, counts = _inputs(rows, n, dtype, n, ragged)
    given = dict(num_states=counts.cuda()) if ragged else {}
    dx, ds, dw = x.cuda(), states.cuda(), weights.cuda()
    ll, gradient = states_log_likelihood_and_gradient(dx, ds, dw, **given)
    _check(ll, gradient, x, states, weights, counts)
    _check(states_log_likelihood(dx, ds.int(), **given), None, x, states, weights, counts)
    leaf = dx.clone().requires_grad_(True)
    again = states_log_likelihood(leaf, ds, **given)
    (backward,) = torch.autograd.grad(again, leaf, grad_outputs=dw)
    _check(again, backward, x, states, weights, counts)
    # in place of the logits
    ll_in, same = states_log_likelihood_and_gradient(dx, ds, dw, out=dx, **given)
    assert same is dx and torch.equal(dx.nan_to_num(7.0), gradient.nan_to_num(7.0))
    assert torch.equal(ll_in.nan_to_num(7.0), ll.nan_to_num(7.0))


@pytest.mark.parametrize("n", [65536, 65537, 70001, 131072, 140003])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_rows_that_no_block_holds(n, dtype):
    from bayesiannetwork_amd.optimizers import states_log_likelihood, states_log_likelihood_and_gradient

    x, states, weights, counts = _inputs(3, n, dtype, n, False)
    states[0], states[1] = n - 1, -7
    dx, ds, dw = x.cuda(), states.cuda(), weights.cuda()
    ll, gradient = states_log_likelihood_and_gradient(dx, ds, dw)
    _check(ll, gradient, x, states, weights, counts)
    leaf = dx.clone().requires_grad_(True)
    again = states_log_likelihood(leaf, ds)
    (backward,) = torch.autograd.grad(again, leaf, grad_outputs=dw)
    _check(again, backward, x, states, weights, counts)
    states_log_likelihood_and_gradient(dx, ds, dw, out=dx)
    assert torch.equal(dx, gradient)


@pytest.mark.parametrize("n", [5, 100, 3000])
def test_masks_and_values_that_are_no_numbers(n):
    from bayesiannetwork_amd.optimizers import states_log_likelihood, states_log_likelihood_and_gradient

    inf, low = float("inf"), torch.finfo(torch.float32).min
    x = torch.zeros((10, n))
    x[0] = -inf
    x[1, 1:] = -inf
    x[2, 1:] = -inf
    x[3, 2] = float("nan")
    x[4, 2] = inf
    x[5] = low
    x[6] = low
    x[6, 3] = 0.5
    x[7] = torch.finfo(torch.float32).max
    x[7, 1] = low
    x[8] = float("nan")
    x[9] = float("nan")
    states = torch.tensor([1, 0, 1, 0, 0, 2, 3, 1, 0, -1])
    weights = torch.linspace(0.5, 2.0, 10)
    ll, gradient = states_log_likelihood_and_gradient(x.cuda(), states.cuda(), weights.cuda())
    _check(ll, gradient, x, states, weights, torch.full((10,), n))
    assert ll.cpu()[0] == -inf and ll.cpu()[2] == -inf and ll.cpu()[1] == 0 and torch.isnan(ll.cpu()[[3, 4, 8]]).all()
    assert (gradient.cpu()[9] == 0).all() and ll.cpu()[9] == 0
    leaf = x.cuda().requires_grad_(True)
    again = states_log_likelihood(leaf, states.cuda())
    (backward,) = torch.autograd.grad(again, leaf, grad_outputs=weights.cuda())
    _check(again, backward, x, states, weights, torch.full((10,), n))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n", [13, 900, 5000])
def test_rows_anywhere_in_a_buffer(n, dtype):
    """Odd strides and first elements on both sides, one row read by all (stride 0), uint8 states, one
    weight for all rows; what lies between the gradient's rows stays as it was."""
    from bayesiannetwork_amd.optimizers import states_log_likelihood, states_log_likelihood_and_gradient

    gen = torch.Generator().manual_seed(n)
    buffer = torch.randn((9, n + 7), generator=gen).to(dtype).cuda()
    states = torch.randint(0, min(n, 256), (9,), generator=gen, dtype=torch.uint8).cuda()
    for first in (0, 1, 5):
        view = buffer[:, first : first + n]
        target = torch.full((9, n + 3), 42.0, dtype=dtype, device="cuda")
        ll, _ = states_log_likelihood_and_gradient(view, states, out=target[:, 2 : 2 + n])
        ll_copy, gradient = states_log_likelihood_and_gradient(view.contiguous(), states.long())
        assert torch.equal(ll, ll_copy) and torch.equal(target[:, 2 : 2 + n], gradient)
        assert (target[:, :2] == 42.0).all() and (target[:, 2 + n :] == 42.0).all()
    one = buffer[:1, :n].expand(9, n)
    leaf = one.contiguous().requires_grad_(True)
    ll = states_log_likelihood(leaf, states)
    ll.sum().backward()  # the weights come as one expanded number
    _, gradient = states_log_likelihood_and_gradient(one, states)
    weights = torch.ones((9,), dtype=ll.dtype)
    _check(ll, leaf.grad, one.cpu(), states.cpu(), weights, torch.full((9,), n))
    _check(ll, gradient, one.cpu(), states.cpu(), weights, torch.full((9,), n))
    shared = buffer[:1, :n].clone().requires_grad_(True)  # a broadcast input: the rows' gradients add up
    states_log_likelihood(shared.expand(9, n), states).sum().backward()
    assert shared.grad.shape == (1, n)


def test_gradient_against_differences():
    """Central differences in float64 with step h: truncation h^2 |f'''| / 6 <= 0.1 h^2, rounding
    2^-52 |f| / h with |f| <= 20: below 1e-8 at h = 1e-5."""
    from bayesiannetwork_amd.optimizers import states_log_likelihood

    gen = torch.Generator().manual_seed(2)
    x = torch.randn((4, 9), generator=gen, dtype=torch.float64).cuda()
    states = torch.tensor([0, 8, 3, -1]).cuda()
    leaf = x.clone().requires_grad_(True)
    states_log_likelihood(leaf, states).sum().backward()
    h = 1e-5
    for i in range(9):
        up, down = x.clone(), x.clone()
        up[:, i] += h
        down[:, i] -= h
        slope = (states_log_likelihood(up, states) - states_log_likelihood(down, states)) / (2 * h)
        assert float((slope - leaf.grad[:, i]).abs().max()) < 1e-8


def test_refusals():
    from bayesiannetwork_amd.optimizers import states_log_likelihood, states_log_likelihood_and_gradient

    x, s = torch.zeros((3, 4), device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    w = torch.ones(3, device="cuda")
    for call, error in [
        (lambda: states_log_likelihood(x.t(), s), ValueError),
        (lambda: states_log_likelihood(x, s[:2]), ValueError),
        (lambda: states_log_likelihood(x, s.cpu()), ValueError),
        (lambda: states_log_likelihood(x, w), TypeError),
        (lambda: states_log_likelihood(x, s, num_states=w), TypeError),
        (lambda: states_log_likelihood_and_gradient(x, s, w.double()), TypeError),
        (lambda: states_log_likelihood_and_gradient(x, s, w[:1]), ValueError),
        (lambda: states_log_likelihood_and_gradient(x, s, out=x.double()), ValueError),
        (lambda: states_log_likelihood_and_gradient(x, s, out=x.t()), ValueError),
        (lambda: states_log_likelihood_and_gradient(x, s, out=x[:1].expand(3, 4)), RuntimeError),
        (lambda: states_log_likelihood_and_gradient(x[:2], s[:2], out=x[1:]), RuntimeError),
        (lambda: states_log_likelihood_and_gradient(x, s, out=torch.zeros((3, 4), device="cuda", requires_grad=True)),
         ValueError),
    ]:
        with pytest.raises(error):
            call()
    leaf = x.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(states_log_likelihood(leaf, s).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()  # once differentiable
    assert states_log_likelihood(x[:0], s[:0]).shape == (0,)
    assert states_log_likelihood_and_gradient(x[:0], s[:0])[1].shape == (0, 4)


def test_backward_captured_while_an_eager_graph_lives():
    """Forward and backward of one leaf captured into a graph and replayed with new logits, with another
    eager result of the same kind still waiting for its backward."""
    from bayesiannetwork_amd.optimizers import states_log_likelihood

    gen = torch.Generator().manual_seed(14)
    x = torch.randn((50, 33), generator=gen).cuda()
    states = torch.randint(0, 33, (50,), generator=gen).cuda()
    weights = torch.rand((50,), generator=gen).cuda()
    other = x.clone().requires_grad_(True)
    waiting = states_log_likelihood(other, states)  # its backward comes last
    leaf = x.clone().requires_grad_(True)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.autograd.grad(states_log_likelihood(leaf, states), leaf, grad_outputs=weights)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ll = states_log_likelihood(leaf, states)
        (gradient,) = torch.autograd.grad(ll, leaf, grad_outputs=weights)
    for _ in range(3):
        with torch.no_grad():
            leaf.copy_(torch.randn((50, 33), generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        eager = leaf.detach().clone().requires_grad_(True)
        want = states_log_likelihood(eager, states)
        (want_gradient,) = torch.autograd.grad(want, eager, grad_outputs=weights)
        assert torch.equal(ll, want) and torch.equal(gradient, want_gradient)
    (late,) = torch.autograd.grad(waiting, other, grad_outputs=weights)
    again = x.clone().requires_grad_(True)
    (want,) = torch.autograd.grad(states_log_likelihood(again, states), again, grad_outputs=weights)
    assert torch.equal(late, want)


@pytest.mark.parametrize("n", [10, 3001, 70001])
def test_captured_and_on_another_stream(n):
    from bayesiannetwork_amd.optimizers import states_log_likelihood_and_gradient

    gen = torch.Generator().manual_seed(4)
    x, states = torch.randn((8, n), generator=gen).cuda(), torch.randint(0, n, (8,), generator=gen).cuda()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        states_log_likelihood_and_gradient(x, states)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ll, gradient = states_log_likelihood_and_gradient(x, states)
    for _ in range(3):
        x.copy_(torch.randn((8, n), generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        want_ll, want = states_log_likelihood_and_gradient(x, states)
        assert torch.equal(ll, want_ll) and torch.equal(gradient, want)


@pytest.mark.parametrize("n", [6, 300, 5000])
def test_a_backward_pass_that_needs_overwritten_logits_raises(n):
    """The gradient written over logits that an earlier result, or the operation that made them, has kept."""
    from bayesiannetwork_amd.optimizers import states_log_likelihood, states_log_likelihood_and_gradient

    gen = torch.Generator().manual_seed(n)
    x, states = torch.randn((4, n), generator=gen).cuda(), torch.randint(0, n, (4,), generator=gen).cuda()
    leaf = x.clone().requires_grad_(True)
    ll = states_log_likelihood(leaf, states)
    states_log_likelihood_and_gradient(leaf.detach(), states, out=leaf.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        ll.sum().backward()
    leaf = x.clone().requires_grad_(True)
    y = torch.tanh(leaf)  # keeps its result
    _, gradient = states_log_likelihood_and_gradient(y.detach(), states, out=y.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(gradient)
    # a gradient of its own memory disturbs nothing
    leaf = x.clone().requires_grad_(True)
    ll = states_log_likelihood(leaf, states)
    version = leaf._version
    out = torch.empty_like(x)
    states_log_likelihood_and_gradient(leaf.detach(), states)
    states_log_likelihood_and_gradient(leaf.detach(), states, out=out)
    ll.sum().backward()
    assert leaf._version == version
    _check(ll, leaf.grad, x.cpu(), states.cpu(), torch.ones((4,)), torch.full((4,), n))
    with torch.inference_mode():
        states_log_likelihood_and_gradient(x.clone(), states, out=torch.empty_like(x))


def test_logits_with_a_tangent_are_refused():
    from torch.autograd import forward_ad

    from bayesiannetwork_amd.optimizers import states_log_likelihood

    x, states = torch.randn((3, 4), generator=torch.Generator().manual_seed(0)).cuda(), torch.tensor([0, 1, 2]).cuda()
    want = states_log_likelihood(x, states)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: states_log_likelihood(dual, states),
                     lambda: states_log_likelihood(dual.clone().requires_grad_(True), states)):
            with pytest.raises(NotImplementedError):
                call()
        with torch.no_grad(), pytest.raises(NotImplementedError):
            states_log_likelihood(dual, states)
        assert torch.equal(states_log_likelihood(x, states), want)  # no tangent
        assert torch.equal(states_log_likelihood(forward_ad.unpack_dual(dual).primal, states), want)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n", [1, 13, 900, 5000])
def test_gradients_in_columns_between_the_logits(n, dtype):
    from bayesiannetwork_amd.optimizers import states_log_likelihood_and_gradient

    gen = torch.Generator().manual_seed(n)
    x = torch.randn((9, n), generator=gen).to(dtype)
    states = torch.randint(0, n, (9,), generator=gen).cuda()
    ll, gradient = states_log_likelihood_and_gradient(x.cuda(), states)
    for first, second in ((0, n), (n, 0), (1, n + 3), (n + 2, 2)):
        buffer = torch.full((9, 2 * n + 5), 42.0, dtype=dtype, device="cuda")
        logits, out = buffer[:, first : first + n], buffer[:, second : second + n]
        logits.copy_(x)
        got, _ = states_log_likelihood_and_gradient(logits, states, out=out)
        assert torch.equal(got, ll) and torch.equal(out, gradient) and torch.equal(logits.cpu(), x)
        out.fill_(0.0)
        logits.fill_(0.0)
        assert float((buffer == 42.0).sum()) == 9 * 5
    if n > 1:
        buffer = torch.zeros((9, 2 * n + 5), dtype=dtype, device="cuda")
        for first, second in ((0, n - 1), (n, 1), (n + 4, 5)):
            with pytest.raises(RuntimeError, match="lies over"):
                states_log_likelihood_and_gradient(buffer[:, first : first + n], states, out=buffer[:, second : second + n])


def _check_on_gpu(ll, gradient, x, states, weights, counts):
    """The definition over many rows at once, in float64 on the GPU, with the tolerances above."""
    dtype, (rows, n) = x.dtype, x.shape
    eps = 2.0**-53 if dtype == torch.float64 else 2.0**-24
    inside = torch.arange(n, device="cuda")[None, :] < counts[:, None]
    wide = torch.where(inside, x.double(), -float("inf"))
    seen = (states >= 0) & (states < counts)
    row, target = torch.arange(rows, device="cuda"), torch.where(seen, states, 0)
    best = wide.max(dim=1, keepdim=True).values
    wide = torch.where(seen[:, None], wide - best, 0.0)
    total = torch.logsumexp(wide, dim=1)
    want_ll = torch.where(seen, wide[row, target] - total, 0.0)
    depth = n / 64 + 16
    assert torch.all((ll.detach().double() - want_ll).abs() <= depth * eps + eps * want_ll.abs())
    p = torch.where(seen[:, None], torch.exp(wide - total[:, None]), 0.0)
    want = -p
    want[row, target] += seen.double()
    want *= weights.double()[:, None]
    slack = weights.double().abs()[:, None] * (depth + 64) * eps * p + (torch.finfo(dtype).eps / 2 + 2 * eps) * want.abs()
    assert torch.all((gradient.double() - want).abs() <= slack + SMALLEST[dtype])


# Rows beyond which a group of lanes takes several of them (by the bytes of a row), and the rows a block takes one after
# the other; the last groups and turns are not full.
@pytest.mark.parametrize("ragged", [False, True], ids=["full", "ragged"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,bytes_of_a_row", [
    (262147, 30), (262149, 60), (131079, 125), (65541, 256), (32771, 500), (16389, 1000), (16389, 2000), (8201, 4000),
    (2307, 10000), (1801, 30000), (601, 50000), (601, 130000), (601, 200000)])
def test_many_rows(rows, bytes_of_a_row, dtype, ragged):
    from bayesiannetwork_amd.optimizers import states_log_likelihood, states_log_likelihood_and_gradient

    n = bytes_of_a_row * 8 // torch.finfo(dtype).bits
    gen = torch.Generator(device="cuda").manual_seed(rows + n)
    x = (3.0 * torch.randn((rows, n), generator=gen, device="cuda")).to(dtype)
    states = torch.randint(-1, n, (rows,), generator=gen, device="cuda")
    weights = torch.rand((rows,), generator=gen, device="cuda", dtype=torch.float64) - 0.3
    weights = weights if dtype == torch.float64 else weights.float()
    counts = torch.randint(0, n + 1, (rows,), generator=gen, device="cuda") if ragged else torch.full((rows,), n, device="cuda")
    if ragged:
        x.masked_fill_(torch.arange(n, device="cuda")[None, :] >= counts[:, None], float("nan"))
    given = dict(num_states=counts) if ragged else {}
    ll, gradient = states_log_likelihood_and_gradient(x, states, weights, **given)
    _check_on_gpu(ll, gradient, x, states, weights, counts)
    leaf = x.clone().requires_grad_(True)
    again = states_log_likelihood(leaf, states, **given)
    (backward,) = torch.autograd.grad(again, leaf, grad_outputs=weights)
    _check_on_gpu(again, backward, x, states, weights, counts)
    states_log_likelihood_and_gradient(x, states, weights, out=x, **given)
    assert torch.equal(x, gradient)


def test_backward_of_more_packs_than_32_bits_count():
    """8200 rows of 2^22 states, all the same logits: 4.3e9 packs of 16 bytes.  The pass is elementwise, so each row is,
    bit for bit, what a call for that row alone gives."""
    from bayesiannetwork_amd.optimizers import states_log_likelihood

    rows, n = 8200, 1 << 22
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("needs 69 GB for the gradient")
    gen = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn((1, n), generator=gen, device="cuda").half()
    states = torch.randint(0, n, (rows,), generator=gen, device="cuda")
    weights = torch.rand((rows,), generator=gen, device="cuda") + 0.5
    leaf = x.expand(rows, n).requires_grad_(True)
    (gradient,) = torch.autograd.grad(states_log_likelihood(leaf, states), leaf, grad_outputs=weights)
    assert gradient.shape == (rows, n)
    for r in (0, 1, 4095, 4096, 8190, 8191, 8192, 8199):
        one = x.clone().requires_grad_(True)
        (want,) = torch.autograd.grad(states_log_likelihood(one, states[r : r + 1]), one, grad_outputs=weights[r : r + 1])
        assert torch.equal(gradient[r], want[0]), r
    del gradient
    torch.cuda.empty_cache()
