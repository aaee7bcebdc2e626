"""Draws from rows of logits against the definition in 64 bits, at the lengths where the kernels change
hands, with ties, masks, padding and every filter.

The states have to be equal.  Both sides sum in double (the kept set's borders partly in integers
of 2^-38 of a weight or finer), so they can only differ where a border lies within 1e-10 of the target;
the oracle says how far its borders are.  A row that is nearer than that (among a million states some
weights are below 1e-10 of the sum) is not compared, unless all its sums are exact (equal weights)."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float64, torch.float16, torch.bfloat16]


def _oracle(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(state, distance of the nearest border that decided it, relative to the sums)"""
    x = np.asarray(x, dtype=np.float64)
    n = x.size
    if n == 0 or np.isnan(x).any() or np.isposinf(x).any() or np.isneginf(x).all() or not 0 <= u <= 1:
        return -1, 1.0
    if temperature == 0:
        return int(np.argmax(x)), 1.0
    w = np.exp((x - x.max()) / temperature)
    order = np.argsort(-x, kind="stable")
    margin = 1.0
    if 0 < top_k < n:
        order = order[:top_k]
    if top_p < 1:
        upto = np.cumsum(w[order])
        before = np.concatenate([[0.0], upto[:-1]])
        margin = min(margin, np.abs(upto / upto[-1] - top_p).min())
        order = order[before < top_p * upto[-1]] if top_p > 0 else order[:1]
    if min_p > 0:
        margin = min(margin, np.abs(w[order] - min(min_p, 1.0)).min() if min_p < 1 else 1.0)
        order = order[w[order] >= min(min_p, 1.0)]
    order = np.sort(order)
    upto = np.cumsum(w[order])
    target = u * upto[-1]
    margin = min(margin, np.abs(upto[:-1] - target).min() / upto[-1] if order.size > 1 else 1.0)
    at = np.searchsorted(upto, target, side="right")
    if at == order.size:
        at = np.flatnonzero(w[order])[-1]
    return int(order[at]), margin


def _check(got, rows, uniforms, settings, exact_sums=False):
    got = got.cpu().numpy()
    undecided = 0
    for r, x in enumerate(rows):
        want, margin = _oracle(x, float(uniforms[r]), **{k: v[r] if hasattr(v, "__len__") else v
                                                         for k, v in settings.items()})
        if margin <= 1e-10 and not exact_sums:
            undecided += 1
            continue
        assert got[r] == want, (r, got[r], want, margin)
    assert undecided <= len(rows) // 4


SETTINGS = {
    "none": {},
    "greedy": dict(temperature=0.0),
    "cold": dict(temperature=0.3),
    "top_k": dict(top_k=5),
    "top_k 300": dict(top_k=300, temperature=2.0),
    "top_p": dict(temperature=1.5, top_p=0.9),
    "top_p small": dict(top_p=0.05),
    "min_p": dict(min_p=0.1),
    "all": dict(temperature=1.2, top_k=40, top_p=0.8, min_p=0.02),
}


@pytest.mark.parametrize("setting", SETTINGS, ids=list(SETTINGS))
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("states", [1, 2, 3, 8, 9, 17, 33, 64, 65, 200, 513, 1024, 1025, 2048, 2049, 4099, 16384, 16385,
                                    20001])
def test_follows_the_definition(states, dtype, setting):
    from bayesiannetwork_amd.samplers import draw_states

    gen = torch.Generator().manual_seed(states)
    rows = 37 if states < 2000 else 5
    x = (2.5 * torch.randn((rows, states), generator=gen)).to(dtype)
    u = torch.rand((rows,), generator=gen, dtype=torch.float64)
    got = draw_states(x.cuda(), u.cuda(), **SETTINGS[setting])
    assert got.shape == (rows,) and got.dtype == torch.int32
    _check(got, x.double().numpy(), u.numpy(), SETTINGS[setting])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("states", [11, 64, 700, 6001])
def test_settings_and_lengths_of_every_row(states, dtype):
    """One call with greedy, unfiltered and filtered rows, rows of 0 states to all of them, settings
    beyond their range (off), in a buffer whose padding holds NaN and infinities."""
    from bayesiannetwork_amd.samplers import draw_states

    gen = torch.Generator().manual_seed(7 * states)
    rows = 60
    x = (2.0 * torch.randn((rows, states), generator=gen)).to(dtype)
    u = torch.rand((rows,), generator=gen, dtype=torch.float32)
    counts = torch.randint(0, states + 1, (rows,), generator=gen)
    counts[:4] = torch.tensor([0, 1, states, states + 5])  # more than the row: all of it
    padded = x.clone()
    for r in range(rows):
        padded[r, int(counts[r]):] = [float("nan"), float("inf"), 3.0][r % 3]
    pick = lambda values: torch.tensor([values[int(i)] for i in torch.randint(0, len(values), (rows,), generator=gen)])
    settings = dict(temperature=pick([0.0, 0.7, 1.0, 1.9]).double(), top_k=pick([0, 1, 7, 50, 10**12, -3]),
                    top_p=pick([1.0, 0.9, 0.35, 1.7]).double(), min_p=pick([0.0, 0.05, -1.0]).double())
    got = draw_states(padded.cuda(), u.cuda(), num_states=counts.cuda(), **{k: v.cuda() for k, v in settings.items()})
    plain = {k: v.numpy() for k, v in settings.items()}
    _check(got, [x[r, : int(counts[r])].double().numpy() for r in range(rows)], u.double().numpy(), plain)


@pytest.mark.parametrize("states", [10, 64, 300, 5000])
def test_equal_logits_are_taken_by_index(states):
    """All weights are 1 and all sums exact: the borders themselves are tested.  Half the states lie on one
    key, the other half far below."""
    from bayesiannetwork_amd.samplers import draw_states

    x = torch.full((1, states), -200.0)
    x[0, 1::2] = 3.0  # the weight of the others is exp(-203): none of them moves a sum
    top = states // 2
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 1.0], dtype=torch.float64)
    rows = x.expand(u.numel(), states)  # row stride 0
    for settings in (dict(), dict(top_k=3), dict(top_k=top), dict(top_p=0.5), dict(top_p=0.5, top_k=4), dict(min_p=1.0)):
        got = draw_states(rows.cuda(), u.cuda(), **settings)
        _check(got, rows.double().numpy(), u.numpy(), settings, exact_sums=True)
    assert draw_states(rows.cuda(), u.cuda(), top_k=1).cpu().tolist() == [1] * 5
    assert draw_states(rows.cuda(), u.cuda(), temperature=0.0).cpu().tolist() == [1] * 5


@pytest.mark.parametrize("states", [5, 40, 300, 3000])
@pytest.mark.parametrize("settings", [dict(), dict(top_k=2), dict(top_p=0.9), dict(temperature=0.0)], ids=str)
def test_masks_and_values_that_are_no_numbers(states, settings):
    from bayesiannetwork_amd.samplers import draw_states

    inf, low = float("inf"), torch.finfo(torch.float32).min
    rows = torch.zeros((9, states))
    rows[0] = -inf  # nothing possible
    rows[1] = -inf
    rows[1, states - 1] = -4.0  # one state possible
    rows[2, 2] = float("nan")
    rows[3, 0] = inf
    rows[4] = low  # masked with the type's lowest value: equal weights
    rows[5] = low
    rows[5, 3] = 1.0
    rows[6, ::2] = -0.0  # one key with 0
    rows[7, 1:] = -inf
    rows[8] = torch.finfo(torch.float32).max
    rows[8, 1] = low  # the difference overflows float32
    u = torch.full((9,), 0.625, dtype=torch.float64)
    got = draw_states(rows.cuda(), u.cuda(), **settings)
    _check(got, rows.double().numpy(), u.numpy(), settings, exact_sums=True)
    assert got[:4].cpu().tolist() == [-1, states - 1, -1, -1]


def test_uniform_numbers_and_settings_of_a_row_that_cannot_be_drawn():
    from bayesiannetwork_amd.samplers import draw_states

    nan, inf = float("nan"), float("inf")
    x = torch.zeros((6, 8), device="cuda")
    u = torch.tensor([nan, -0.1, 1.1, 0.0, 1.0, 0.5], device="cuda")
    assert draw_states(x, u).cpu().tolist() == [-1, -1, -1, 0, 7, 4]
    u = torch.full((6,), 0.99, device="cuda")
    t = torch.tensor([nan, -1.0, inf, 0.0, 1.0, 1e-300], device="cuda", dtype=torch.float64)
    assert draw_states(x, u, temperature=t).cpu().tolist() == [-1, -1, -1, 0, 7, 7]
    p = torch.tensor([nan, 0.0, -2.0, 0.25, 1.0, 9.0], device="cuda")
    assert draw_states(x, u, top_p=p).cpu().tolist() == [7, 0, 0, 1, 7, 7]
    m = torch.tensor([nan, 0.0, 5.0, 1.0, -1.0, 0.5], device="cuda")
    assert draw_states(x, u, min_p=m).cpu().tolist() == [7] * 6


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("states", [13, 1500])
def test_rows_anywhere_in_a_buffer(states, dtype):
    """Odd row strides and first elements: the same states as from a copy."""
    from bayesiannetwork_amd.samplers import draw_states

    gen = torch.Generator().manual_seed(3)
    buffer = torch.randn((21, states + 7), generator=gen).to(dtype).cuda()
    u = torch.rand((21,), generator=gen).cuda()
    for first in (0, 1, 3, 6):
        view = buffer[:, first : first + states]
        for settings in (dict(), dict(top_p=0.8), dict(top_k=9)):
            assert torch.equal(draw_states(view, u, **settings), draw_states(view.contiguous(), u, **settings))
    assert torch.equal(draw_states(view, u[::2].repeat_interleave(2)[:21]),
                       draw_states(view, torch.stack([u[::2].repeat_interleave(2)[:21]] * 2, dim=1)[:, 0]))


def test_refusals():
    from bayesiannetwork_amd.samplers import draw_states

    x, u = torch.zeros((3, 4), device="cuda"), torch.zeros(3, device="cuda")
    for call, error in [
        (lambda: draw_states(x.t(), u), ValueError),
        (lambda: draw_states(x, u[:2]), ValueError),
        (lambda: draw_states(x, u.half()), TypeError),
        (lambda: draw_states(x, u.cpu()), ValueError),
        (lambda: draw_states(x, u, temperature=-1), ValueError),
        (lambda: draw_states(x, u, top_p=0.0), ValueError),
        (lambda: draw_states(x, u, min_p=1.5), ValueError),
        (lambda: draw_states(x, u, top_k=-1), ValueError),
        (lambda: draw_states(x, u, top_k=2.5), ValueError),
        (lambda: draw_states(x, u, top_k=u), TypeError),
        (lambda: draw_states(x, u, temperature=u[:1]), ValueError),
        (lambda: draw_states(x, u, num_states=u), TypeError),
    ]:
        with pytest.raises(error):
            call()
    assert draw_states(x[:0], u[:0]).shape == (0,)


def test_long_rows_of_flat_and_peaked_distributions():
    """A flat row keeps most of its states, a peaked one few: 131 072 states in bfloat16 (many ties) and
    100 003 in float32."""
    from bayesiannetwork_amd.samplers import draw_states

    gen = torch.Generator().manual_seed(5)
    for states, dtype in ((131072, torch.bfloat16), (100003, torch.float32)):
        x = torch.randn((6, states), generator=gen)
        x[:2] *= 0.01
        x[2:4] *= 6.0
        x = x.to(dtype)
        u = torch.rand((6,), generator=gen, dtype=torch.float64)
        for settings in (dict(), dict(top_p=0.97), dict(top_k=5000), dict(top_k=20000, top_p=0.5, min_p=1e-4)):
            _check(draw_states(x.cuda(), u.cuda(), **settings), x.double().numpy(), u.numpy(), settings)


@pytest.mark.parametrize("states,dtype", [(2000, torch.float32), (3001, torch.float16), (9000, torch.bfloat16),
                                          (60001, torch.float64), (300007, torch.float16), (1200001, torch.float32)],
                         ids=str)
def test_rows_that_keep_many_states(states, dtype):
    """Filters that leave most of a flat row: the threshold lies among thousands of states, on keys that many
    share (float16, bfloat16) or that are nearly all different; some rows end inside their ties."""
    from bayesiannetwork_amd.samplers import draw_states

    gen = torch.Generator().manual_seed(states)
    rows = 4
    x = torch.randn((rows, states), generator=gen)
    x[0] = torch.round(x[0] * 2) / 2  # a dozen keys
    x[1] *= 0.05
    x[2] *= 3
    x = x.to(dtype)
    u = torch.rand((rows,), generator=gen, dtype=torch.float64)
    for settings in (dict(top_p=0.93), dict(top_k=states // 3), dict(top_k=states - 7, temperature=0.8),
                     dict(top_k=states // 2, top_p=0.6), dict(min_p=0.01), dict(top_p=0.9, min_p=0.05),
                     dict(top_k=states // 2, top_p=0.7, min_p=0.02), dict(top_p=0.999999)):
        _check(draw_states(x.cuda(), u.cuda(), **settings), x.double().numpy(), u.numpy(), settings)


def test_many_long_rows_that_keep_many_states():
    """More rows than are shared between blocks, each with settings of its own that leave a flat row nearly
    whole."""
    from bayesiannetwork_amd.samplers import draw_states

    gen = torch.Generator().manual_seed(77)
    rows, states = 530, 16400
    x = torch.randn((rows, states), generator=gen).bfloat16()
    u = torch.rand((rows,), generator=gen, dtype=torch.float64)
    settings = dict(top_p=0.8 + 0.15 * torch.rand((rows,), generator=gen, dtype=torch.float64),
                    top_k=torch.where(torch.arange(rows) % 5 == 0, 9000, 0))
    got = draw_states(x.cuda(), u.cuda(), **{k: v.cuda() for k, v in settings.items()})
    _check(got, x.double().numpy(), u.numpy(), {k: v.numpy() for k, v in settings.items()})


@pytest.mark.parametrize("states", [64, 5000, 40000])
def test_two_streams_at_once(states):
    from bayesiannetwork_amd.samplers import draw_states

    gen = torch.Generator().manual_seed(states)
    inputs = [(torch.randn((200, states), generator=gen).cuda(), torch.rand((200,), generator=gen).cuda())
              for _ in range(2)]
    want = [draw_states(x, u, top_p=0.9) for x, u in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for k, (x, u) in enumerate(inputs):
            with torch.cuda.stream(streams[k]):
                got[k].append(draw_states(x, u, top_p=0.9))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(g, want[k]) for g in got[k])


def test_frequencies_of_a_posterior():
    """Draws from a machine's posterior follow it (chi-square, alpha = 0.001)."""
    from scipy import stats

    from bayesiannetwork_amd.samplers import draw_states

    p = torch.tensor([0.05, 0.1, 0.0, 0.4, 0.45], dtype=torch.float64)
    n = 200_000
    u = torch.rand((n,), generator=torch.Generator().manual_seed(9), dtype=torch.float32)
    got = draw_states(p.log().float().cuda().expand(n, 5), u.cuda()).cpu().long()
    counts = torch.bincount(got, minlength=5).double()
    assert counts[2] == 0
    keep = p > 0
    _, level = stats.chisquare(counts[keep].numpy(), (p[keep] / p[keep].sum() * n).numpy())
    assert level > 0.001


@pytest.mark.parametrize("states", [10, 300, 40000])
def test_captured_and_on_another_stream(states):
    """Two graphs and eager calls, replayed in turn with new inputs: each replay equals an eager call."""
    from bayesiannetwork_amd.samplers import draw_states

    gen = torch.Generator().manual_seed(1)
    x = torch.randn((16, states), generator=gen).cuda()
    u = torch.rand((16,), generator=gen).cuda()
    settings = dict(top_k=20, top_p=0.9)
    draw_states(x, u, **settings)
    graphs = []
    for kwargs in (settings, dict(temperature=0.5)):
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            draw_states(x, u, **kwargs)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = draw_states(x, u, **kwargs)
        graphs.append((graph, out, kwargs))
    for step in range(4):
        x.copy_(torch.randn((16, states), generator=gen))
        u.copy_(torch.rand((16,), generator=gen))
        for graph, out, kwargs in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, draw_states(x, u, **kwargs))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16], ids=str)
@pytest.mark.parametrize("states", [3, 5, 16, 64, 300, 1500, 5000, 40000])
def test_borders_that_single_precision_does_not_resolve(states, dtype):
    """Uniform numbers, shares and smallest weights 2e-9 to either side of a border of the row's own: closer than
    sums of floats can tell (6e-8), twenty times farther than sums of doubles need."""
    from bayesiannetwork_amd.samplers import draw_states

    gen = torch.Generator().manual_seed(11 * states)
    rows = 24
    x = (2.0 * torch.randn((rows, states), generator=gen)).to(dtype)
    side = torch.where(torch.arange(rows) % 2 == 0, 2e-9, -2e-9).double()
    w = torch.softmax(x.double(), dim=1)
    place = torch.randint(0, states - 1, (rows,), generator=gen)
    u = (w.cumsum(1)[torch.arange(rows), place] + side).clamp(0.0, 1.0)
    _check(draw_states(x.cuda(), u.cuda()), x.double().numpy(), u.numpy(), {})

    place = torch.randint(0, min(states - 1, 40), (rows,), generator=gen)
    p = torch.sort(w, dim=1, descending=True).values.cumsum(1)[torch.arange(rows), place] + side
    u = torch.ones((rows,), dtype=torch.float64)  # the last kept state tells where the kept ones end
    u[::3] = torch.rand((8,), generator=gen, dtype=torch.float64)
    got = draw_states(x.cuda(), u.cuda(), top_p=p.cuda())
    _check(got, x.double().numpy(), u.numpy(), dict(top_p=p.numpy()))

    least = torch.sort(w / w.max(1, keepdim=True).values, dim=1, descending=True).values
    m = least[torch.arange(rows), torch.clamp(place, max=3)].clamp(min=0.1) + side
    got = draw_states(x.cuda(), u.cuda(), min_p=m.cuda())
    _check(got, x.double().numpy(), u.numpy(), dict(min_p=m.numpy()))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("states", [2100, 20000])
def test_rows_of_a_few_states_in_a_long_tensor(states, dtype):
    """Rows shorter than 16 bytes of logits, and some that end just behind a piece of 16 or 64 states."""
    from bayesiannetwork_amd.samplers import draw_states

    gen = torch.Generator().manual_seed(states)
    counts = torch.tensor([1, 2, 3, 4, 5, 6, 7, 8, 9, 15, 16, 17, 63, 64, 65, 66, 1025, 2049])
    rows = counts.numel()
    x = torch.randn((rows, states), generator=gen).to(dtype)
    u = torch.rand((rows,), generator=gen, dtype=torch.float64)
    padded = x.clone()
    for r in range(rows):
        padded[r, int(counts[r]):] = float("nan")
    for settings in (dict(), dict(top_k=2), dict(top_p=0.8), dict(top_k=3, top_p=0.9), dict(min_p=0.3), dict(temperature=0.0)):
        got = draw_states(padded.cuda(), u.cuda(), num_states=counts.cuda(), **settings)
        _check(got, [x[r, : int(counts[r])].double().numpy() for r in range(rows)], u.numpy(), settings)


@pytest.mark.parametrize("tied", [900, 2500, 6000])
def test_ties_around_the_threshold_side_by_side(tied):
    """A share's threshold among states on one key that lie next to each other: the blocks that share a row find
    nearly all of them in one block's part, or in two."""
    from bayesiannetwork_amd.samplers import draw_states

    gen = torch.Generator().manual_seed(tied)
    rows, states = 5, 131072
    x = torch.randn((rows, states), generator=gen)
    x[:, 5000 : 5000 + tied] = 1.25
    w = torch.softmax(x.double(), dim=1)
    above, on = torch.where(x > 1.25, w, 0.0).sum(1), torch.where(x == 1.25, w, 0.0).sum(1)
    p = above + on * torch.tensor([0.0004, 0.25, 0.5, 0.75, 0.9996], dtype=torch.float64)
    u = torch.tensor([1.0, 0.3, 1.0, 0.8, 0.041], dtype=torch.float64)
    got = draw_states(x.cuda(), u.cuda(), top_p=p.cuda()).cpu().tolist()
    # a quarter of 900 ties is 225 of them: where a border lies on the share itself, the sums' roundings decide, and the
    # states of both neighbours are right
    for r in range(rows):
        row = x[r].double().numpy()
        assert got[r] in {_oracle(row, float(u[r]), top_p=float(p[r]) + d)[0] for d in (-1e-10, 0.0, 1e-10)}, r


@pytest.mark.parametrize("states", [40, 3000, 16384, 60001])
def test_top_k_of_all_of_a_row(states):
    """A top-k that is no less than the row's states (all of them, or of those that a padded row has) leaves top-p
    alone at work."""
    from bayesiannetwork_amd.samplers import draw_states

    gen = torch.Generator().manual_seed(3 * states)
    rows = 6
    x = torch.randn((rows, states), generator=gen)
    u = torch.rand((rows,), generator=gen, dtype=torch.float64)
    counts = torch.tensor([states, states // 2, states // 2 + 1, states - 1, 7 * states // 8, 3])
    for top_k in (states // 2, states - 1, states, states + 1, 10**9):
        settings = dict(top_k=top_k, top_p=0.9)
        _check(draw_states(x.cuda(), u.cuda(), **settings), x.double().numpy(), u.numpy(), settings)
        got = draw_states(x.cuda(), u.cuda(), num_states=counts.cuda(), **settings)
        _check(got, [x[r, : int(counts[r])].double().numpy() for r in range(rows)], u.numpy(), settings)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16], ids=str)
@pytest.mark.parametrize("states", [2049, 9000, 70001])
def test_small_top_k_of_rows_with_many_states_around_it(states, dtype):
    """Sorted rows (the largest states side by side, so that the pieces they are in say little), a few levels that
    hundreds of states share, and flat rows, at the largest top-k of that kind and one beyond it."""
    from bayesiannetwork_amd.samplers import draw_states

    gen = torch.Generator().manual_seed(13 * states)
    rows = 8
    x = torch.randn((rows, states), generator=gen)
    x[0:2] = torch.sort(x[0:2], dim=1, descending=True).values
    x[2] = torch.sort(x[2]).values
    x[3:5] = torch.round(x[3:5])
    x[5] = 0.25
    x[6, : states // 2] = -float("inf")
    x = x.to(dtype)
    u = torch.rand((rows,), generator=gen, dtype=torch.float64)
    u[4:6] = torch.tensor([1.0, 1.0])
    for settings in (dict(top_k=1), dict(top_k=50), dict(top_k=256), dict(top_k=257), dict(top_k=256, top_p=0.7),
                     dict(top_k=200, min_p=0.4), dict(top_k=250, top_p=0.9, min_p=0.3, temperature=3.0)):
        got = draw_states(x.cuda(), u.cuda(), **settings)
        _check(got, x.double().numpy(), u.numpy(), settings, exact_sums=False)


@pytest.mark.parametrize("dtype,states", [(torch.bfloat16, 131072), (torch.float32, 50000), (torch.float64, 12000)], ids=str)
@pytest.mark.parametrize("rows", [12, 520])
def test_a_share_that_min_p_does_not_leave(dtype, states, rows):
    """More than 512 states are left by min-p, and together they hold less than top-p's share of the row: all of them
    are kept, and finding that out takes no longer than finding a threshold (a search through keys that no state has
    would take a hundred times as long)."""
    from bayesiannetwork_amd.samplers import draw_states

    gen = torch.Generator().manual_seed(states + rows)
    x = (-torch.randint(0, 256, (rows, states), generator=gen) / 64.0).to(dtype)
    u = torch.rand((rows,), generator=gen, dtype=torch.float64)
    settings = dict(top_p=0.95, min_p=0.1)
    dx, du = x.cuda(), u.cuda()
    w = torch.exp(dx[:12].double() - dx[:12].double().max(1, keepdim=True).values)
    assert ((w >= 0.1).sum(1) > 512).all() and (torch.where(w >= 0.1, w, 0.0).sum(1) < 0.95 * w.sum(1)).all()
    got = draw_states(dx, du, **settings)
    _check(got[:12], x[:12].double().numpy(), u.numpy(), settings)

    def shortest(**kwargs):
        times = []
        for _ in range(6):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            draw_states(dx, du, **kwargs)
            end.record()
            torch.cuda.synchronize()
            times.append(start.elapsed_time(end))
        return min(times)

    assert shortest(**settings) < 10 * shortest(top_p=0.95)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64], ids=str)
@pytest.mark.parametrize("states,tail", [(1 << 24, [-26.625]), (1 << 20, [-30.0]), ((1 << 20) + 3, [-28.5, -28.75, -29.0]),
                                         (70001, [-22.0, -22.5]), (16000, [-18.0])], ids=str)
def test_a_tail_that_only_counts_together(states, tail, dtype):
    """One state of weight 1, and a tail in which every state is next to nothing but top-p's threshold lies: 0.5 states
    behind the k-th of a key that hundreds of thousands share.  Weights, sums and the expected state in closed form
    (a running sum of the tail would round more of it away): a border is off by about 2^-53 of the row where the
    weights are, against half a state, 2^-45 of it at the least."""
    from bayesiannetwork_amd.samplers import draw_states

    keys = torch.tensor(tail, dtype=dtype)
    levels = np.arange(states) % len(tail)
    levels[0] = -1
    x = keys[torch.from_numpy(levels).clamp(min=0)]
    x[0] = 0.0
    w = np.exp(keys.double().numpy())
    sizes = np.array([(levels == k).sum() for k in range(len(tail))])
    total = 1.0 + float((sizes * w).sum())
    end = len(tail) // 2  # the key on which the share ends
    kept = int(sizes[end] * 0.37)
    p = (1.0 + float((sizes[:end] * w[:end]).sum()) + (kept + 0.5) * w[end]) / total
    assert 0.5 * w[end] > 100 * 2.0**-53 and p < 1.0
    numbers = [np.cumsum(levels == k) for k in range(len(tail))]  # states of each key up to an index
    upto = 1.0 + sum(numbers[k] * w[k] for k in range(end)) + np.minimum(numbers[end], kept + 1) * w[end]
    drawn = np.flatnonzero(np.diff(upto, prepend=0.0) > 0)
    picks = drawn[[1, len(drawn) // 7, len(drawn) // 2, len(drawn) - 2, len(drawn) - 1]]
    before = np.concatenate([[0.0], upto])[picks]
    u = np.append((before + upto[picks]) / 2 / upto[-1], 1.0)
    want = np.append(picks, drawn[-1])
    got = draw_states(x.cuda()[None].expand(len(u), states), torch.from_numpy(u).cuda(), top_p=float(p))
    assert got.cpu().tolist() == want.tolist()


@pytest.mark.parametrize("states", [12000, 40000])
@pytest.mark.parametrize("temperature", [1e-100, 1e-40, 1e-31, 1.0, 1e31, 1e45, 1e200], ids=str)
def test_temperatures_beyond_single_precision(states, temperature):
    """Rows that keep many states, with logits as large or small as the temperature: a few levels, 8192 states on
    the highest one (in one row these and nothing else within reach), and levels all over."""
    from bayesiannetwork_amd.samplers import draw_states

    gen = torch.Generator().manual_seed(states)
    x = torch.full((4, states), -1.0, dtype=torch.float64)
    x[0, torch.randperm(states, generator=gen)[:8192]] = 0.0
    x[1] = -torch.randint(0, 3, (states,), generator=gen).double()
    x[2] = torch.randn((states,), generator=gen, dtype=torch.float64)
    x[3] = 3.0 * torch.randn((states,), generator=gen, dtype=torch.float64)
    x *= temperature
    x[0, x[0] < 0] = -float("inf")
    u = torch.tensor([1.0, 0.7, 1.0, 0.3], dtype=torch.float64)
    for settings in (dict(top_p=0.5), dict(top_p=0.9), dict(top_k=states // 4, top_p=0.6), dict(min_p=0.2)):
        settings["temperature"] = temperature
        # the row of one level has exact sums
        got = draw_states(x.cuda(), u.cuda(), **settings)
        _check(got, x.numpy(), u.numpy(), settings, exact_sums=True)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("states", [16, 37, 64, 250, 1000, 2048, 2500, 20000])
def test_a_last_row_that_ends_its_buffer(states, dtype):
    """Through the C ABI: the buffer ends with the last row's own states, whose padding does not exist; and rows whose
    lengths run through all places of a pack."""
    import ctypes

    from bayesiannetwork_amd.inference_machines.hip_spa import _native

    gen = torch.Generator().manual_seed(states)
    lib = _native.load()
    for last in (1, 3, 7, 9, 16, states - 1):
        counts = torch.tensor([min(n, states) for n in (1, 2, 5, 8, 11, 14, 17, 20, 23, 30, 65, 66, states)] + [last])
        rows = counts.numel()
        x = torch.randn((rows, states), generator=gen).to(dtype)
        u = torch.rand((rows,), generator=gen, dtype=torch.float64)
        flat = x.flatten()[: (rows - 1) * states + last].cuda()
        dc, du = counts.cuda(), u.cuda()
        need = lib.bn_draw_states_workspace_bytes(_native.DTYPE_CODES[dtype], rows, states)
        workspace = torch.empty((max(need, 1),), dtype=torch.uint8, device="cuda")
        for settings in (dict(), dict(top_p=0.8), dict(top_k=3, temperature=2.0), dict(temperature=0.0)):
            filters = _native.DrawFilters(1.0, 0, 1.0, 0.0)
            for k, v in settings.items():
                setattr(filters, k, v)
            out = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
            _native.launch(flat.device, lib.bn_draw_states, _native.DTYPE_CODES[dtype], flat.data_ptr(), rows, states, states,
                           dc.data_ptr(), 1, du.data_ptr(), ctypes.byref(filters), workspace.data_ptr(), out.data_ptr())
            _check(out, [x[r, : int(counts[r])].double().numpy() for r in range(rows)], u.numpy(), settings)


def _oracle_on_gpu(x, u, counts, temperature, top_k, top_p, min_p):
    """_oracle for many rows at once, in float64 on the GPU; settings are numbers."""
    rows, n = x.shape
    place = torch.arange(n, device="cuda")[None, :]
    x = torch.where(place < counts[:, None], x.double(), -float("inf"))
    w = torch.exp((x - x.max(1, keepdim=True).values) / temperature)
    by_key, order = torch.sort(x, dim=1, descending=True, stable=True)
    sorted_w = torch.gather(w, 1, order)
    top = torch.where(place < (top_k or n), sorted_w, 0.0)
    upto = top.cumsum(1)
    total = upto[:, -1:]
    kept = (place < (top_k or n)) & (upto - top < top_p * total) if top_p < 1 else place < torch.full_like(counts, top_k or n)[:, None]
    margin = torch.ones((rows,), device="cuda", dtype=torch.float64)
    if top_p < 1:
        margin = torch.minimum(margin, (upto / total - top_p).abs().min(1).values)
    if min_p > 0:
        margin = torch.minimum(margin, (sorted_w - min_p).abs().min(1).values)
    kept &= sorted_w >= min_p
    w = torch.where(torch.zeros_like(kept).scatter_(1, order, kept), w, 0.0)
    upto = w.cumsum(1)
    target = u.double()[:, None] * upto[:, -1:]
    margin = torch.minimum(margin, ((upto - target).abs() / upto[:, -1:]).min(1).values)
    state = (upto <= target).sum(1)
    return torch.where(counts > 0, state, -1), margin


# 16 states per lane, in groups of 1 to 64 lanes: from these numbers of rows on
@pytest.mark.parametrize("ragged", [False, True], ids=["full", "ragged"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,states", [(262147, 5), (262145, 16), (131075, 17), (131073, 32), (65537, 50), (65539, 64),
                                         (32769, 100), (32771, 128), (16387, 130), (16385, 256), (5003, 300), (3001, 1024)])
def test_many_rows(rows, states, dtype, ragged):
    from bayesiannetwork_amd.samplers import draw_states

    gen = torch.Generator(device="cuda").manual_seed(rows + states)
    x = (2.0 * torch.randn((rows, states), generator=gen, device="cuda")).to(dtype)
    u = torch.rand((rows,), generator=gen, device="cuda", dtype=torch.float64) * 0.999
    counts = torch.randint(0, states + 1, (rows,), generator=gen, device="cuda") if ragged else torch.full((rows,), states, device="cuda")
    padded = x.masked_fill(torch.arange(states, device="cuda")[None, :] >= counts[:, None], float("nan"))
    for settings in (dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), dict(temperature=0.8, top_k=4, top_p=1.0, min_p=0.0),
                     dict(temperature=1.3, top_k=0, top_p=0.9, min_p=0.0), dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.05),
                     dict(temperature=1.1, top_k=9, top_p=0.85, min_p=0.03)):
        want, margin = _oracle_on_gpu(x, u, counts, **settings)
        got = draw_states(padded, u, **({**settings, "num_states": counts} if ragged else settings))
        decided = (margin > 1e-10) | (counts == 0)
        assert decided.double().mean() > 0.99
        assert torch.equal(got[decided].long(), want[decided])
