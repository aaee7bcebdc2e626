"""Cases of the row operators on logits (draws, log-likelihood with its gradient) and of gradient
clipping: their inputs, one pass through each in plain torch operations or through this package, and
their values in 64 bits.

A case is a dict of plain values; ``op`` names the operator:

* ``draw``      - ``samplers.draw_states``: one state per row of logits at a given uniform number
* ``evaluate``  - ``optimizers.states_log_likelihood`` without a gradient
* ``backward``  - the same through autograd, with the gradient of the logits
* ``step``      - ``optimizers.states_log_likelihood_and_gradient``: both in one call
* ``clip``      - ``optimizers.HipGradientClipper``: global norm over many tensors, clipped copies
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "float64": torch.float64, "float16": torch.float16, "bfloat16": torch.bfloat16}


def listed():
    return [
        # one latent class per observation from the posterior of the 10-class model (60 000 observations)
        dict(name="draw class posteriors", op="draw", rows=60000, states=10, dtype="float32", filters="none",
             ragged=False),
        # one state of a 64-state node per observation, the improbable tail cut off, rows of nodes with fewer states padded
        dict(name="draw 64-state rows, top-p", op="draw", rows=131072, states=64, dtype="float32", filters="top_p",
             ragged=True),
        # one request's next state from a large vocabulary: latency
        dict(name="draw one long row", op="draw", rows=1, states=32000, dtype="bfloat16", filters="all", ragged=False),
        # a serving batch, every request with settings of its own (some greedy, some unfiltered)
        dict(name="draw a serving batch", op="draw", rows=256, states=131072, dtype="bfloat16", filters="per_row",
             ragged=False),
        # a medium batch of an odd vocabulary, nucleus only: the whole row's mass is needed
        dict(name="draw odd rows, top-p", op="draw", rows=48, states=50003, dtype="float16", filters="top_p",
             ragged=False),
        # held-out score of a classifier of 10 classes
        dict(name="evaluate 10 classes", op="evaluate", rows=60000, states=10, dtype="float32", ragged=False),
        # gradient of a 64-state conditional through autograd, some rows unobserved
        dict(name="backward 64 states", op="backward", rows=131072, states=64, dtype="float32", ragged=True),
        # training step over a large vocabulary: log-likelihood and gradient in one call
        dict(name="step large vocabulary", op="step", rows=4096, states=64000, dtype="bfloat16", ragged=False),
        # a smaller training step of odd width in full precision
        dict(name="step odd width", op="step", rows=1000, states=5003, dtype="float32", ragged=False),
        # gradients of the 784-leaf model's tables, one small tensor per node
        dict(name="clip 785 tables", op="clip", layout="tables", count=784, elements=20, dtype="float32"),
        # layers of mixed sizes, matrices in half precision and vectors in full
        dict(name="clip mixed layers", op="clip", layout="mixed", count=96, elements=400003, dtype="bfloat16"),
        # few large tensors, larger than any cache
        dict(name="clip large", op="clip", layout="even", count=8, elements=16777216, dtype="float32"),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["draw", "draw", "draw", "evaluate", "backward", "step", "clip"])
    if op == "clip":
        layout = rng.choice(["tables", "mixed", "even"])
        count = _log_uniform(rng, 1, 1000)
        elements = _log_uniform(rng, 2, min(16777216, 40000000 // count))
        return dict(op=op, layout=layout, count=count, elements=elements,
                    dtype=rng.choice(["float32", "float32", "bfloat16", "float16", "float64"]))
    states = _log_uniform(rng, 2, 131072)
    rows = _log_uniform(rng, 1, min(131072, 25000000 // states))
    case = dict(op=op, rows=rows, states=states,
                dtype=rng.choice(["float32", "float32", "bfloat16", "bfloat16", "float16", "float64"]),
                ragged=rng.random() < 0.3)
    if op == "draw":
        case["filters"] = rng.choice(["none", "top_k", "top_p", "min_p", "all", "per_row"])
    return case


# ---- inputs -------------------------------------------------------------------------------------


def _logits(gen, rows, states, dtype):
    """Rows of logits: a broad bulk and, in long rows, some favoured states well above it."""
    x = torch.randn((rows, states), generator=gen, device="cuda", dtype=torch.float32).mul_(2.0)
    if states > 256:
        boost = torch.rand((rows, states), generator=gen, device="cuda", dtype=torch.float32)
        x += boost.pow_(400.0).mul_(12.0)
    return x.to(dtype)


def _filters(kind, rows, gen):
    """The keyword arguments of a draw: numbers for the whole call, or one setting per row."""
    if kind == "none":
        return {}
    if kind == "top_k":
        return dict(temperature=0.9, top_k=40)
    if kind == "top_p":
        return dict(temperature=0.8, top_p=0.95)
    if kind == "min_p":
        return dict(temperature=1.1, min_p=0.05)
    if kind == "all":
        return dict(temperature=0.7, top_k=50, top_p=0.95, min_p=0.02)
    pick = torch.rand((4, rows), generator=gen, device="cuda", dtype=torch.float64)
    value = torch.rand((4, rows), generator=gen, device="cuda", dtype=torch.float64)
    zero = torch.zeros_like(value[0])
    return dict(
        temperature=torch.where(pick[0] < 0.1, zero, 0.5 + value[0]),  # 0: greedy
        top_k=torch.where(pick[1] < 0.4, zero, 1 + 200 * value[1]).long(),  # 0: off
        top_p=torch.where(pick[2] < 0.3, zero + 1.0, 0.5 + 0.49 * value[2]),  # 1: off
        min_p=torch.where(pick[3] < 0.6, zero, 0.1 * value[3]),  # 0: off
    )


def _clip_shapes(case):
    """Sizes and types of a case's tensors."""
    count, elements, dtype = case["count"], case["elements"], case["dtype"]
    if case["layout"] == "tables":  # one table per node, and the root's
        return [(elements, dtype)] * count + [(max(elements // 2, 1), dtype)]
    if case["layout"] == "even":
        return [(elements, dtype)] * count
    out = []
    for i in range(count):  # matrices of different sizes, every third one a vector in full precision
        if i % 3 == 2:
            out.append((max(elements // 997, 1), "float32"))
        else:
            out.append((max(elements >> (i % 4), 1), dtype))
    return out


def _by_type(grads):
    """(type, places of its tensors) for every type among the gradients, in order of appearance."""
    places = {}
    for i, g in enumerate(grads):
        places.setdefault(g.dtype, []).append(i)
    return list(places.items())


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    state = {"op": op}
    if op == "clip":
        grads = []
        for i, (size, dtype) in enumerate(_clip_shapes(case)):
            g = torch.randn((size,), generator=gen, device="cuda", dtype=torch.float32).mul_(0.02 * (1 + i % 5))
            grads.append(g.to(DTYPES[dtype]))
        state["grads"] = grads
        state["max_norm"] = 1.0
        if own:
            from bayesiannetwork_amd.optimizers import HipGradientClipper

            # the clipped copies are slices of one buffer per type, what an update reads
            state["flat"], out = {}, [None] * len(grads)
            for dtype, members in _by_type(grads):
                sizes = [grads[i].numel() for i in members]
                state["flat"][dtype] = torch.empty((sum(sizes),), device="cuda", dtype=dtype)
                for i, piece in zip(members, torch.split(state["flat"][dtype], sizes)):
                    out[i] = piece
            state["clipper"] = HipGradientClipper(grads, out=out)
        return state
    rows, states, dtype = case["rows"], case["states"], DTYPES[case["dtype"]]
    state["logits"] = _logits(gen, rows, states, dtype)
    state["num_states"] = None
    if case["ragged"]:
        low = max(states // 2, 1)
        state["num_states"] = torch.randint(low, states + 1, (rows,), generator=gen, device="cuda")
    if op == "draw":
        state["uniforms"] = torch.rand((rows,), generator=gen, device="cuda", dtype=torch.float32)
        state["filters"] = _filters(case["filters"], rows, gen)
        return state
    state["states"] = torch.randint(0, states, (rows,), generator=gen, device="cuda")  # beyond a short row: unobserved
    kind = torch.float64 if dtype == torch.float64 else torch.float32
    state["weights"] = torch.rand((rows,), generator=gen, device="cuda", dtype=kind) + 0.5
    if op == "backward":
        state["logits"].requires_grad_(True)
    return state


# ---- the plain form -----------------------------------------------------------------------------


def _column(value, rows):
    if isinstance(value, torch.Tensor):
        return value[:, None]
    return torch.full((rows, 1), value, device="cuda", dtype=torch.float64)


def _plain_draw(logits, uniforms, num_states, filters):
    # in 64 bits: the sums run over whole rows, and a state's border decides an index
    rows, states = logits.shape
    place = torch.arange(states, device="cuda")[None, :]
    x = logits.double()
    if num_states is not None:
        x = x.masked_fill(place >= num_states[:, None], -math.inf)
    u = uniforms.double()[:, None]
    temperature = _column(filters.get("temperature", 1.0), rows)
    top_k = _column(filters.get("top_k", 0), rows).long()
    top_p = _column(filters.get("top_p", 1.0), rows)
    min_p = _column(filters.get("min_p", 0.0), rows)

    best = x.max(dim=1, keepdim=True).values
    greedy = temperature == 0
    scale = torch.where(greedy, torch.ones_like(temperature), temperature)
    ordered, order = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((ordered - best) / scale)
    k = torch.where(top_k <= 0, states, top_k)
    w_top = torch.where(place < k, w, 0.0)
    before = torch.cumsum(w_top, dim=1)
    total = before[:, -1:].clone()
    before = torch.cat([torch.zeros_like(total), before[:, :-1]], dim=1)
    kept = (place < k) & ((before < top_p * total) | (top_p >= 1)) & (w >= min_p)
    kept = torch.zeros_like(kept).scatter_(1, order, kept)
    w = torch.where(kept, torch.exp((x - best) / scale), 0.0)
    upto = torch.cumsum(w, dim=1)
    index = (upto <= u * upto[:, -1:]).sum(dim=1)
    last = torch.where(w > 0, place, -1).max(dim=1).values
    index = torch.where(index >= states, last, index)
    first = torch.where(x == best, place, states).min(dim=1).values
    return torch.where(greedy[:, 0], first, index).to(torch.int32)


def _plain_likelihood(logits, states, num_states, weights):
    """Log-likelihood of each row's state and, with weights, the gradient of their weighted sum."""
    rows, width = logits.shape
    x = logits.float() if logits.dtype != torch.float64 else logits
    place = torch.arange(width, device="cuda")[None, :]
    seen = torch.full_like(states, width) if num_states is None else num_states
    seen = (states >= 0) & (states < seen)
    if num_states is not None:
        x = x.masked_fill(place >= num_states[:, None], -math.inf)
    best = x.max(dim=1, keepdim=True).values
    w = torch.exp(x - best)
    total = w.sum(dim=1, keepdim=True)
    target = torch.where(seen, states, 0)[:, None]
    ll = (x.gather(1, target) - best - torch.log(total))[:, 0]
    ll = torch.where(seen, ll, 0.0)
    if weights is None:
        return ll
    hit = (place == target).to(x.dtype)
    gradient = torch.where(seen, weights, 0.0)[:, None] * (hit - w / total)
    return ll, gradient.to(logits.dtype)


def _plain_clip(grads, max_norm):
    # in 64 bits: a sum over all elements
    square = torch.zeros((), device="cuda", dtype=torch.float64)
    for g in grads:
        square = square + (g.double() * g.double()).sum()
    norm = torch.sqrt(square)
    factor = torch.where(norm > max_norm, max_norm / norm, 1.0)
    clipped = [(g.double() * factor).to(g.dtype) for g in grads]
    return norm, [torch.cat([clipped[i] for i in members]) for _, members in _by_type(grads)]


def run(state):
    op = state["op"]
    if op == "clip":
        if own:
            return state["clipper"].clip(state["max_norm"]), list(state["flat"].values())
        return _plain_clip(state["grads"], state["max_norm"])
    logits, num_states = state["logits"], state["num_states"]
    if op == "draw":
        if own:
            from bayesiannetwork_amd.samplers import draw_states

            return draw_states(logits, state["uniforms"], num_states=num_states, **state["filters"])
        return _plain_draw(logits, state["uniforms"], num_states, state["filters"])
    states, weights = state["states"], state["weights"]
    if own:
        from bayesiannetwork_amd.optimizers import states_log_likelihood, states_log_likelihood_and_gradient

        if op == "evaluate":
            return states_log_likelihood(logits, states, num_states=num_states)
        if op == "step":
            return states_log_likelihood_and_gradient(logits, states, weights, num_states=num_states)
        ll = states_log_likelihood(logits, states, num_states=num_states)
        (gradient,) = torch.autograd.grad(ll, logits, grad_outputs=weights)
        return ll.detach(), gradient
    return _plain_likelihood(logits.detach(), states, num_states, None if op == "evaluate" else weights)


# ---- what a pass cannot do without, and its values in 64 bits ------------------------------------


def work(case):
    size = {"float32": 4, "float64": 8, "float16": 2, "bfloat16": 2}
    if case["op"] == "clip":
        shapes = _clip_shapes(case)
        return {"bytes": sum(2 * n * size[t] for n, t in shapes) + 8, "flops": sum(3 * n for n, _ in shapes)}
    rows, elements = case["rows"], case["rows"] * case["states"]
    data = elements * size[case["dtype"]]
    per_row = 8 if case["ragged"] else 0
    if case["op"] == "draw":
        per_row += 4 + 4 + (32 if case["filters"] == "per_row" else 0)
        return {"bytes": data + rows * per_row, "flops": 4 * elements}
    out = 8 if case["dtype"] == "float64" else 4
    per_row += 8 + out
    if case["op"] == "evaluate":
        return {"bytes": data + rows * per_row, "flops": 4 * elements}
    return {"bytes": 2 * data + rows * (per_row + out), "flops": 7 * elements}


def _exact_draw(state):
    """Row by row on the host: the kept states are found by walking the sorted row, the draw by walking
    the kept states in their own order."""
    logits = state["logits"].double().cpu().numpy()
    uniforms = state["uniforms"].double().cpu().numpy()
    rows, states = logits.shape
    counts = np.full((rows,), states) if state["num_states"] is None else state["num_states"].cpu().numpy()
    given = state["filters"]

    def setting(name, default):
        value = given.get(name, default)
        return value.cpu().numpy() if isinstance(value, torch.Tensor) else np.full((rows,), value)

    temperature, top_k = setting("temperature", 1.0), setting("top_k", 0)
    top_p, min_p = setting("top_p", 1.0), setting("min_p", 0.0)
    out = np.empty((rows,), np.int32)
    for r in range(rows):
        x = logits[r, : counts[r]]
        if temperature[r] == 0:
            out[r] = int(np.argmax(x))
            continue
        w = np.exp((x - x.max()) / temperature[r])
        if top_k[r] > 0 or top_p[r] < 1 or min_p[r] > 0:
            order = np.argsort(-x, kind="stable")
            if top_k[r] > 0:
                order = order[: top_k[r]]
            upto = np.cumsum(w[order])
            keep = order.size
            if top_p[r] < 1:
                keep = int(np.searchsorted(upto, top_p[r] * upto[-1], side="left")) + 1
            order = order[: min(keep, order.size)]
            order = np.sort(order[w[order] >= min_p[r]])
        else:
            order = np.arange(x.size)
        upto = np.cumsum(w[order])
        at = int(np.searchsorted(upto, uniforms[r] * upto[-1], side="right"))
        if at == order.size:
            at = int(np.flatnonzero(w[order])[-1])
        out[r] = order[at]
    return torch.from_numpy(out)


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "clip":
        squares = [float(torch.dot(g.double().flatten(), g.double().flatten())) for g in state["grads"]]
        norm = math.sqrt(math.fsum(squares))
        factor = min(1.0, state["max_norm"] / norm) if norm > 0 else 1.0
        flat = [torch.cat([state["grads"][i] for i in members]) for _, members in _by_type(state["grads"])]
        return torch.tensor(norm, dtype=torch.float64), [g.double() * factor for g in flat]
    if op == "draw":
        return _exact_draw(state)
    x = state["logits"].detach().double()
    rows, width = x.shape
    counts = torch.full((rows,), width, device="cuda") if state["num_states"] is None else state["num_states"]
    inside = torch.arange(width, device="cuda")[None, :] < counts[:, None]
    x = torch.where(inside, x, -math.inf)
    log_total = torch.logsumexp(x, dim=1)
    row = torch.arange(rows, device="cuda")
    seen = state["states"] < counts
    target = torch.where(seen, state["states"], 0)
    ll = torch.where(seen, x[row, target] - log_total, 0.0)
    if op == "evaluate":
        return ll
    gradient = torch.exp(x - log_total[:, None]).neg_()
    gradient[row, target] += 1.0
    gradient *= torch.where(seen, state["weights"].double(), 0.0)[:, None]
    return ll, gradient
