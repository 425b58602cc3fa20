"""What a network of layers needs besides them to be trained, as programs call it.

``op`` names the operator and ``direction`` what is asked of it.

* ``gated``: the first half of a gated feed-forward block, by group (an expert per token, a block per element): both
  projections of a row by the matrices of its group, the activation of the one, times the other. ``forward``, or
  ``gradients``: its vector-Jacobian product. The order of the rows by group is in hand before the call.
* ``loss``: a linear layer to a vocabulary and the cross entropy of its softmax with the row's target, for tokens or for
  elements that were masked; rows without a target are padding. ``forward``: the losses and the logarithms of the
  softmax's sums, or ``training``: the losses, and the gradients of both operands.
* ``clip``: the norm of all gradients of a network together. ``forward``: the norm alone, or ``clipped``: the gradients
  as well, scaled so that their norm is at most ``max_norm``.

``run`` makes the calls of the ``mops_amd`` package where ``own`` is true, and the same mathematics in elementary torch
operations in 32 bits where it is not.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def _gated(direction, dtype, rows, groups, k, l, activation, skew, padded, ordered):
    return {
        "op": "gated", "direction": direction, "dtype": dtype, "rows": rows, "groups": groups, "k": k, "l": l,
        "activation": activation, "skew": skew, "padded": padded, "ordered": ordered,
    }  # fmt: skip


def _loss(direction, dtype, rows, vocabulary, k, skew, padded):
    return {
        "op": "loss", "direction": direction, "dtype": dtype, "rows": rows, "vocabulary": vocabulary, "k": k,
        "skew": skew, "padded": padded,
    }  # fmt: skip


def _clip(direction, dtype, blocks, width, hidden, table_rows, single, reached):
    return {
        "op": "clip", "direction": direction, "dtype": dtype, "blocks": blocks, "width": width, "hidden": hidden,
        "table_rows": table_rows, "single": single, "reached": reached,
    }  # fmt: skip


def listed():
    def case(name, sizes):
        return {"name": name, **sizes}

    return [
        # 24 single tokens, each to one of 16 experts: the experts' matrices are read and little is computed
        case("gated experts, single tokens", _gated("forward", "bfloat16", 24, 16, 2048, 1408, "silu", 0.5, 0.0, True)),
        # one small structure of four elements: nothing but the cost of a call
        case("gated elements, small structure", _gated("forward", "float32", 600, 4, 128, 128, "silu", 1.0, 0.0, True)),
        # a prompt or a step of training through 32 experts of uneven load
        case("gated experts, many tokens", _gated("forward", "bfloat16", 16384, 32, 2048, 1408, "silu", 0.5, 0.0, True)),
        # the backward pass of experts of odd width, with rows that are padding
        case("gated experts, gradients", _gated("gradients", "bfloat16", 20011, 24, 1280, 1000, "gelu", 0.5, 0.01, True)),
        # the backward pass of a block per element, rows already in the order of their element
        case("gated elements, gradients", _gated("gradients", "float32", 100000, 7, 256, 256, "silu", 1.0, 0.0, False)),
        # the next token of each of 64 sequences is scored: the vocabulary's table is read and little is computed
        case("loss of single tokens", _loss("forward", "bfloat16", 64, 50000, 2048, 1.0, 0.0)),
        # texts are scored: an odd vocabulary, a fifth of the places is padding
        case("loss of texts", _loss("forward", "float16", 4001, 32003, 1000, 1.0, 0.2)),
        # the end of a step of training on text: a large vocabulary, tokens as frequent as words are
        case("loss of tokens, training", _loss("training", "bfloat16", 8192, 100003, 2048, 1.0, 0.0)),
        # the end of a step of training on structures: the elements of the atoms that were masked are learned
        case("loss of masked elements, training", _loss("training", "float32", 200000, 94, 128, 1.5, 0.85)),
        # the gradients of a small network of structures: nothing but the cost of a call
        case("clip of a small network", _clip("clipped", "float32", 3, 128, 256, 94, False, True)),
        # the gradients of a network of text
        case("clip of a large network", _clip("clipped", "bfloat16", 10, 2048, 5632, 50000, False, True)),
        # the norm that is watched, matrices in 16 bits and norms' weights in 32
        case("norm of a large network", _clip("forward", "bfloat16", 10, 1280, 4001, 32003, True, False)),
    ]


def draw(rng):
    def size(low, high):
        return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5)))))))

    dtype = rng.choice(["float32", "bfloat16", "float16"])
    op = rng.choice(["gated", "loss", "clip"])
    if op == "gated":
        direction = rng.choice(["forward", "gradients"])
        rows, groups, k, l = size(1, 65536), size(1, 64), size(1, 4096), size(1, 4096)
        # (the matrices of all groups within half a gigabyte, and no more work than a step's)
        groups = max(1, min(groups, (1 << 26) // (k * l)))
        passes = 3 if direction == "gradients" else 1
        rows = max(1, min(rows, (1 << 38) // (2 * passes * k * l), (1 << 27) // max(k, l)))
        if dtype == "float32":
            rows = max(1, min(rows, (1 << 36) // (2 * passes * k * l)))
        activation, skew = rng.choice(["silu", "gelu", "sigmoid"]), rng.choice([0.0, 0.5, 1.0])
        return _gated(direction, dtype, rows, groups, k, l, activation, skew, rng.choice([0.0, 0.05]), rng.random() < 0.7)
    if op == "loss":
        direction = rng.choice(["forward", "training"])
        rows, vocabulary, k = size(1, 200000), size(2, 150000), size(1, 4096)
        k = min(k, (1 << 28) // vocabulary)
        rows = max(1, min(rows, (1 << 29) // vocabulary, (1 << 40) // (vocabulary * k), (1 << 27) // k))
        if dtype == "float32":
            rows = max(1, min(rows, (1 << 37) // (vocabulary * k)))
        return _loss(direction, dtype, rows, vocabulary, k, rng.choice([0.0, 1.0, 1.5]), rng.choice([0.0, 0.2, 0.85]))
    blocks, width, hidden, table_rows = rng.randint(1, 10), size(1, 2048), size(1, 5632), size(1, 100000)
    table_rows = min(table_rows, (1 << 26) // width)
    direction, single, reached = rng.choice(["forward", "clipped"]), rng.random() < 0.3, rng.random() < 0.7
    return _clip(direction, dtype, blocks, width, hidden, table_rows, single, reached)


def _indices(case, count, seed):
    """One value in [0, count) per row, the v-th most frequent as often as (v + 1)^-skew; -1: padding."""
    rng = np.random.default_rng(seed)
    weights = np.arange(1, count + 1, dtype=np.float64) ** -case["skew"]
    weights = weights[rng.permutation(count)]
    cumulated = np.cumsum(weights)
    index = np.searchsorted(cumulated / cumulated[-1], rng.random(case["rows"]), side="right")
    index = np.minimum(index, count - 1).astype(np.int32)
    if case["padded"] > 0:
        index[rng.random(case["rows"]) < case["padded"]] = -1
    return index


def _shapes(case):
    """The parameters of a network: a table, and per block the projections of attention, the matrices of a gated
    feed-forward block, two weights of norms."""
    width, hidden = case["width"], case["hidden"]
    block = [(width, 3 * width), (width, width), (width, 2 * hidden), (hidden, width), (width,), (width,)]
    return [(case["table_rows"], width)] + block * case["blocks"] + [(width,)]


def prepare(case, seed):
    device = torch.device("cuda")
    dtype = DTYPES[case["dtype"]]
    generator = torch.Generator(device=device)
    generator.manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=dtype):
        values = torch.randn(shape, generator=generator, device=device, dtype=torch.float32)
        return (values * scale).to(dtype)

    state = {"case": case}
    if case["op"] == "gated":
        index = _indices(case, case["groups"], seed)
        by_group = np.where(index < 0, case["groups"], index)
        order = np.argsort(by_group, kind="stable").astype(np.int32)
        offsets = np.searchsorted(by_group[order], np.arange(case["groups"] + 1)).astype(np.int32)
        state["order"] = torch.from_numpy(order).to(device) if case["ordered"] else None
        state["offsets"] = torch.from_numpy(offsets).to(device)
        state["boundaries"] = offsets.tolist()
        state["A"] = normal(case["rows"], case["k"])
        state["W"] = normal(case["groups"], case["k"], 2 * case["l"], scale=1.5 * case["k"] ** -0.5)
        if case["direction"] == "gradients":
            state["grad_output"] = normal(case["rows"], case["l"])
    elif case["op"] == "loss":
        state["targets"] = torch.from_numpy(_indices(case, case["vocabulary"], seed)).to(device)
        state["A"] = normal(case["rows"], case["k"])
        state["W"] = normal(case["vocabulary"], case["k"], scale=2.0 * case["k"] ** -0.5)
        if case["direction"] == "training":
            # (the mean over the rows, with weights; in float16 the loss is scaled up, so that gradients are numbers)
            weights = torch.rand(case["rows"], generator=generator, device=device, dtype=torch.float32) + 0.5
            state["grad_losses"] = weights * ((1024.0 if case["dtype"] == "float16" else 1.0) / case["rows"])
    else:
        gradients = []
        for i, shape in enumerate(_shapes(case)):
            of_norm = case["single"] and len(shape) == 1
            scale = 10.0 ** -(1 + i % 3)
            gradients.append(normal(*shape, scale=scale, dtype=torch.float32 if of_norm else dtype))
        state["gradients"] = gradients
        squares = sum(g.numel() * 100.0 ** -(1 + i % 3) for i, g in enumerate(gradients))
        state["max_norm"] = math.sqrt(squares) * (0.3 if case["reached"] else 3.0)
    return state


# ------------------------------------------------------------ plain forms ----
def _activation(name, x):
    """act(x) and its derivative."""
    if name == "gelu":
        normal = 0.5 * (1 + torch.erf(x * math.sqrt(0.5)))
        return x * normal, normal + x * torch.exp(-0.5 * x * x) * (1 / math.sqrt(2 * math.pi))
    sigmoid = 1 / (1 + torch.exp(-x))
    if name == "sigmoid":
        return sigmoid, sigmoid * (1 - sigmoid)
    return x * sigmoid, sigmoid * (1 + x * (1 - sigmoid))


def _plain_gated(s):
    A, W, order, ends = s["A"], s["W"], s["order"], s["boundaries"]
    columns = W.shape[2] // 2
    gradients = s["case"]["direction"] == "gradients"
    if gradients:
        grad_A = torch.zeros(A.shape, dtype=torch.float32, device=A.device)
        grad_W = torch.zeros(W.shape, dtype=torch.float32, device=A.device)
    else:
        output = torch.zeros(A.shape[0], columns, dtype=torch.float32, device=A.device)
    for group in range(W.shape[0]):
        first, last = ends[group], ends[group + 1]
        if first == last:
            continue
        rows = slice(first, last) if order is None else order[first:last]
        a = A[rows].float()
        w = W[group].float()
        both = a @ w
        gate, up = both[:, :columns], both[:, columns:]
        value, slope = _activation(s["case"]["activation"], gate)
        if gradients:
            g = s["grad_output"][rows].float()
            both = torch.cat([g * up * slope, g * value], 1)
            grad_A[rows] = both @ w.t()
            grad_W[group] = a.t() @ both
        else:
            output[rows] = value * up
    if gradients:
        return grad_A.to(A.dtype), grad_W.to(A.dtype)
    return output.to(A.dtype)


def _plain_loss(s):
    A, W, targets = s["A"].float(), s["W"].float(), s["targets"].long()
    kept = targets >= 0
    column = torch.where(kept, targets, 0)[:, None]
    logits = A @ W.t()
    most = logits.max(1, keepdim=True).values
    powers = torch.exp(logits - most)
    sums = powers.sum(1, keepdim=True)
    log_sums = (torch.log(sums) + most).squeeze(1)
    losses = torch.where(kept, log_sums - logits.gather(1, column).squeeze(1), 0.0)
    if s["case"]["direction"] == "forward":
        return losses, torch.where(kept, log_sums, 0.0)
    del logits
    grad = powers.div_(sums)
    grad.scatter_add_(1, column, torch.full(column.shape, -1.0, device=A.device))
    grad *= torch.where(kept, s["grad_losses"], 0.0)[:, None]
    return losses, (grad @ W).to(s["A"].dtype), (grad.t() @ A).to(s["W"].dtype)


def _plain_clip(s):
    squares = torch.stack([g.float().square().sum(dtype=torch.float64) for g in s["gradients"]])
    norm = torch.sqrt(squares.sum())
    if s["case"]["direction"] == "forward":
        return norm.float()
    factor = torch.clamp(s["max_norm"] / norm, max=1.0).float()
    return [(g.float() * factor).to(g.dtype) for g in s["gradients"]], norm.float()


# --------------------------------------------------- the package's own calls ----
def _own(s):
    import mops_amd

    case = s["case"]
    if case["op"] == "gated":
        inputs = (s["A"], s["W"], s["offsets"], s["order"], case["activation"])
        if case["direction"] == "forward":
            return mops_amd.gated_grouped_product(*inputs)
        return mops_amd.gated_grouped_product_vjp(s["grad_output"], *inputs)
    if case["op"] == "loss":
        losses, log_sums = mops_amd.linear_cross_entropy(s["A"], s["W"], s["targets"])
        if case["direction"] == "forward":
            return losses, log_sums
        grads = mops_amd.linear_cross_entropy_vjp(s["grad_losses"], None, s["A"], s["W"], s["targets"], log_sums)
        return (losses, *grads)
    if case["direction"] == "forward":
        return mops_amd.gradient_norm(s["gradients"])
    return mops_amd.clip_gradients(s["gradients"], s["max_norm"])


PLAIN = {"gated": _plain_gated, "loss": _plain_loss, "clip": _plain_clip}


def run(state):
    return _own(state) if own else PLAIN[state["case"]["op"]](state)


def work(case):
    width = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "gated":
        rows, k, l = case["rows"], case["k"], case["l"]
        used = min(rows, case["groups"]) * 2 * k * l
        index = 4 * rows if case["ordered"] else 0
        if case["direction"] == "forward":
            return {"bytes": (rows * (k + l) + used) * width + index, "flops": 4 * rows * k * l}
        # (the projections, which are not kept, and two products)
        bytes_moved = (rows * (2 * k + l) + used + case["groups"] * 2 * k * l) * width + index
        return {"bytes": bytes_moved, "flops": 12 * rows * k * l}
    if case["op"] == "loss":
        rows, vocabulary, k = case["rows"], case["vocabulary"], case["k"]
        kept = max(1, round(rows * (1 - case["padded"])))
        if case["direction"] == "forward":
            return {"bytes": (kept + vocabulary) * k * width + 12 * rows, "flops": 2 * kept * vocabulary * k}
        bytes_moved = (kept + rows + 2 * vocabulary) * k * width + 12 * rows
        return {"bytes": bytes_moved, "flops": 6 * kept * vocabulary * k}
    count = sum(math.prod(shape) for shape in _shapes(case))
    passes = 1 if case["direction"] == "forward" else 2
    return {"bytes": passes * count * width, "flops": (passes + 1) * count}


# ------------------------------------------------------ values in 64 bits ----
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "gated":
        return _exact_gated(case, s)
    if case["op"] == "loss":
        return _exact_loss(case, s)
    norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(g.double()) for g in s["gradients"]]))
    if case["direction"] == "forward":
        return norm
    factor = s["max_norm"] / max(norm.item(), s["max_norm"])
    return [g.double() * factor for g in s["gradients"]], norm


def _exact_gated(case, s):
    A, W, l = s["A"].double(), s["W"].double(), case["l"]
    gradients = case["direction"] == "gradients"
    results = [torch.zeros_like(A), torch.zeros_like(W)] if gradients else [A.new_zeros(case["rows"], l)]
    places = torch.arange(case["rows"], device=A.device) if s["order"] is None else s["order"].long()
    for g in range(case["groups"]):
        rows = places[s["boundaries"][g] : s["boundaries"][g + 1]]
        a = A[rows]
        gate, up = torch.matmul(a, W[g, :, :l].contiguous()), torch.matmul(a, W[g, :, l:].contiguous())
        # x / (1 + e^-x), x times the normal distribution's integral, 1 / (1 + e^-x): value and derivative
        if case["activation"] == "gelu":
            below = torch.special.ndtr(gate)
            value = gate * below
            slope = below + gate * torch.exp(-gate * gate / 2) / math.sqrt(2 * math.pi)
        else:
            below, above = torch.sigmoid(gate), torch.sigmoid(-gate)
            value = below if case["activation"] == "sigmoid" else gate * below
            slope = below * above if case["activation"] == "sigmoid" else below + gate * below * above
        if not gradients:
            results[0][rows] = value * up
            continue
        cotangent = s["grad_output"][rows].double()
        on_gate, on_up = cotangent * up * slope, cotangent * value
        results[0][rows] = torch.matmul(on_gate, W[g, :, :l].t().contiguous()) + torch.matmul(
            on_up, W[g, :, l:].t().contiguous()
        )
        turned = a.t().contiguous()
        results[1][g, :, :l] = torch.matmul(turned, on_gate)
        results[1][g, :, l:] = torch.matmul(turned, on_up)
    return tuple(results) if gradients else results[0]


def _exact_loss(case, s):
    rows = (s["targets"] >= 0).nonzero().squeeze(1)
    A, W, targets = s["A"][rows].double(), s["W"].double(), s["targets"][rows].long()
    losses = torch.zeros(case["rows"], dtype=torch.float64, device=A.device)
    log_sums = torch.zeros_like(losses)
    grad_A = torch.zeros(case["rows"], case["k"], dtype=torch.float64, device=A.device)
    grad_W = torch.zeros_like(W)
    turned = W.t().contiguous()
    for first in range(0, rows.shape[0], 4096):
        part = slice(first, first + 4096)
        logits = torch.matmul(A[part], turned)
        total = torch.logsumexp(logits, 1)
        at = targets[part][:, None]
        losses[rows[part]] = total - logits.gather(1, at).squeeze(1)
        log_sums[rows[part]] = total
        if case["direction"] == "training":
            probability = torch.exp(logits - total[:, None])
            probability.scatter_(1, at, probability.gather(1, at) - 1)
            probability *= s["grad_losses"][rows[part]].double()[:, None]
            grad_A[rows[part]] = torch.matmul(probability, W)
            grad_W += torch.matmul(probability.t().contiguous(), A[part])
    return (losses, log_sums) if case["direction"] == "forward" else (losses, grad_A, grad_W)
