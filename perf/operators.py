"""The operators of a network's layers around the sums over edges, as programs call them.

``op`` names the operator and ``direction`` what is asked of it: ``forward``, the operator alone, or ``gradients``,
its vector-Jacobian product.

* ``embedding``: the rows of a table that an index names, times a constant (the element of each atom, the token of
  each position); gradient with respect to the table.
* ``grouped``: every row times the matrix of its group (a linear layer per element, an expert per token). The order
  of the rows by group is the plan that a program makes once per batch and uses in every layer; it is in hand before
  the call.
* ``update``: the residual update around a block: norm of the block's output, gate, residual scale, and the norm in
  front of the next block.

``run`` makes the calls of the ``mops_amd`` package where ``own`` is true, and the same mathematics in elementary torch
operations in 32 bits where it is not.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
EPSILON = 1e-6


def _embedding(direction, dtype, rows, table_rows, columns, skew, padded):
    return {
        "op": "embedding", "direction": direction, "dtype": dtype, "rows": rows, "table_rows": table_rows,
        "columns": columns, "skew": skew, "padded": padded,
    }  # fmt: skip


def _grouped(direction, dtype, rows, groups, k, l, skew, padded, ordered):
    return {
        "op": "grouped", "direction": direction, "dtype": dtype, "rows": rows, "groups": groups, "k": k, "l": l,
        "skew": skew, "padded": padded, "ordered": ordered,
    }  # fmt: skip


def _update(direction, dtype, rows, columns, gate_rows):
    return {
        "op": "update", "direction": direction, "dtype": dtype, "rows": rows, "columns": columns,
        "gate_rows": gate_rows,
    }  # fmt: skip


def listed():
    def case(name, sizes):
        return {"name": name, **sizes}

    return [
        # one token of each of 64 sequences that are being continued: nothing but the cost of a call
        case("embedding of single tokens", _embedding("forward", "bfloat16", 64, 50000, 2048, 1.0, 0.0)),
        # a batch of structures, 94 elements, most atoms of a few of them; padded to a fixed number of atoms
        case("embedding of elements, gradients", _embedding("gradients", "float32", 200000, 94, 128, 1.5, 0.02)),
        # a step of training on text: a large vocabulary, tokens as frequent as words are
        case("embedding of tokens, gradients", _embedding("gradients", "bfloat16", 32768, 100003, 2048, 1.0, 0.0)),
        # 24 single tokens, each to one of 16 experts: the matrices of the experts are read and little is computed
        case("experts, single tokens", _grouped("forward", "bfloat16", 24, 16, 2048, 1408, 0.5, 0.0, True)),
        # one small structure of four elements: nothing but the cost of a call
        case("elements, small structure", _grouped("forward", "float32", 600, 4, 128, 128, 1.0, 0.0, True)),
        # a prompt or a step of training through 32 experts of uneven load
        case("experts, many tokens", _grouped("forward", "bfloat16", 32768, 32, 2048, 4096, 0.5, 0.0, True)),
        # the backward pass of experts of odd width, with rows that are padding
        case("experts, gradients", _grouped("gradients", "bfloat16", 20011, 24, 1280, 1000, 0.5, 0.01, True)),
        # the backward pass of a linear layer per element, rows already in the order of their element
        case("elements, gradients", _grouped("gradients", "float32", 100000, 7, 256, 256, 1.0, 0.0, False)),
        # single tokens of eight sequences
        case("update of single tokens", _update("forward", "bfloat16", 8, 4096, 1)),
        # a prompt or a step of training, every token with a gate of its own
        case("update of many tokens", _update("forward", "bfloat16", 16384, 4096, 16384)),
        # its backward pass
        case("update of many tokens, gradients", _update("gradients", "bfloat16", 16384, 4096, 16384)),
        # a batch of structures, features of ordinary width, one learned gate for all atoms
        case("update of atoms, gradients", _update("gradients", "float32", 50021, 384, 1)),
    ]


def draw(rng):
    def size(low, high):
        return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5)))))))

    dtype = rng.choice(["float32", "bfloat16", "float16"])
    direction = rng.choice(["forward", "gradients"])
    op = rng.choice(["embedding", "grouped", "update"])
    if op == "embedding":
        rows, columns = size(1, 200000), size(1, 4096)
        rows = min(rows, (1 << 27) // columns)
        table_rows = min(size(2, 200000), (1 << 28) // columns)
        skew, padded = rng.choice([0.0, 1.0, 1.5]), rng.choice([0.0, 0.05])
        return _embedding(direction, dtype, rows, table_rows, columns, skew, padded)
    if op == "grouped":
        rows, groups, k, l = size(1, 100000), size(1, 64), size(1, 4096), size(1, 4096)
        # (the matrices of all groups within half a gigabyte, and no more work than the largest listed case)
        groups = max(1, min(groups, (1 << 27) // (k * l)))
        passes = 2 if direction == "gradients" else 1
        rows = max(1, min(rows, (1 << 38) // (passes * k * l), (1 << 27) // max(k, l)))
        if dtype == "float32":
            rows = max(1, min(rows, (1 << 35) // (passes * k * l)))
        skew, padded, ordered = rng.choice([0.0, 0.5, 1.0]), rng.choice([0.0, 0.05]), rng.random() < 0.7
        return _grouped(direction, dtype, rows, groups, k, l, skew, padded, ordered)
    rows, columns = size(1, 65536), size(1, 8192)
    rows = min(rows, (1 << 26) // columns)
    return _update(direction, dtype, rows, columns, rng.choice([1, rows]))


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


def prepare(case, seed):
    device = torch.device("cuda")
    dtype = DTYPES[case["dtype"]]
    generator = torch.Generator(device=device)
    generator.manual_seed(seed)

    def normal(*shape, scale=1.0, mean=0.0):
        values = torch.randn(shape, generator=generator, device=device, dtype=torch.float32)
        return (values * scale + mean).to(dtype)

    state = {"case": case}
    if case["op"] == "embedding":
        index = _indices(case, case["table_rows"], seed)
        state["indices"] = torch.from_numpy(index).to(device)
        state["table"] = normal(case["table_rows"], case["columns"], scale=0.02)
        state["scale"] = math.sqrt(case["columns"])
        if case["direction"] == "gradients":
            state["grad_output"] = normal(case["rows"], case["columns"])
    elif case["op"] == "grouped":
        index = _indices(case, case["groups"], seed)
        by_group = np.where(index < 0, case["groups"], index)
        order = np.argsort(by_group, kind="stable").astype(np.int32)
        offsets = np.searchsorted(by_group[order], np.arange(case["groups"] + 1)).astype(np.int32)
        state["order"] = torch.from_numpy(order).to(device) if case["ordered"] else None
        state["offsets"] = torch.from_numpy(offsets).to(device)
        state["boundaries"] = offsets.tolist()
        state["A"] = normal(case["rows"], case["k"])
        state["W"] = normal(case["groups"], case["k"], case["l"], scale=case["k"] ** -0.5)
        if case["direction"] == "gradients":
            state["grad_output"] = normal(case["rows"], case["l"])
    else:
        rows, columns = case["rows"], case["columns"]
        state["residual"] = normal(rows, columns, scale=2.0)
        state["block"] = normal(rows, columns, scale=0.5)
        state["gate"] = torch.sigmoid(normal(case["gate_rows"], columns).float()).to(dtype)
        state["weight_block"] = normal(columns, scale=0.1, mean=1.0)
        state["weight_next"] = normal(columns, scale=0.1, mean=1.0)
        state["residual_scale"] = 0.25
        if case["direction"] == "gradients":
            state["grad_state"] = normal(rows, columns)
            state["grad_next"] = normal(rows, columns)
    return state


# ------------------------------------------------------------ plain forms ----
def _plain_embedding(s):
    dtype = s["table"].dtype
    inside = (s["indices"] >= 0) & (s["indices"] < s["table"].shape[0])
    if s["case"]["direction"] == "forward":
        rows = s["table"][torch.where(inside, s["indices"], 0)].float() * s["scale"]
        return torch.where(inside[:, None], rows, 0.0).to(dtype)
    columns = s["table"].shape[1]
    # (a last row that takes the padding, which is left out at the end)
    gradient = torch.zeros(s["table"].shape[0] + 1, columns, dtype=torch.float32, device=s["table"].device)
    gradient.index_add_(0, torch.where(inside, s["indices"], s["table"].shape[0]), s["grad_output"].float())
    return (gradient[:-1] * s["scale"]).to(dtype)


def _plain_grouped(s):
    A, W, order, ends = s["A"], s["W"], s["order"], s["boundaries"]
    gradients = s["case"]["direction"] == "gradients"
    if gradients:
        grad_A = torch.zeros(A.shape, dtype=torch.float32, device=A.device)
        grad_W = torch.zeros(W.shape, dtype=torch.float32, device=A.device)
    else:
        output = torch.zeros(A.shape[0], W.shape[2], dtype=torch.float32, device=A.device)
    for group in range(W.shape[0]):
        first, last = ends[group], ends[group + 1]
        if first == last:
            continue
        rows = slice(first, last) if order is None else order[first:last]
        a = A[rows].float()
        w = W[group].float()
        if gradients:
            g = s["grad_output"][rows].float()
            grad_A[rows] = g @ w.t()
            grad_W[group] = a.t() @ g
        else:
            output[rows] = a @ w
    if gradients:
        return grad_A.to(A.dtype), grad_W.to(A.dtype)
    return output.to(A.dtype)


def _plain_update(s):
    dtype = s["residual"].dtype
    residual, block, gate = s["residual"].float(), s["block"].float(), s["gate"].float()
    weight_block, weight_next, scale = s["weight_block"].float(), s["weight_next"].float(), s["residual_scale"]
    inverse_block = torch.rsqrt((block * block).mean(1, keepdim=True) + EPSILON)
    unit = block * inverse_block
    inner = unit * weight_block
    state = residual + scale * gate * inner
    inverse_state = torch.rsqrt((state * state).mean(1, keepdim=True) + EPSILON)
    unit_state = state * inverse_state
    if s["case"]["direction"] == "forward":
        return state.to(dtype), (unit_state * weight_next).to(dtype)
    grad_next = s["grad_next"].float()
    h = grad_next * weight_next
    along = (h * unit_state).mean(1, keepdim=True)
    grad_state = s["grad_state"].float() + inverse_state * (h - unit_state * along)
    grad_gate = scale * grad_state * inner
    if gate.shape[0] == 1 and residual.shape[0] != 1:
        grad_gate = grad_gate.sum(0, keepdim=True)
    through = scale * grad_state * gate
    k = through * weight_block
    grad_block = inverse_block * (k - unit * (k * unit).mean(1, keepdim=True))
    grads = (grad_state, grad_block, grad_gate, (through * unit).sum(0), (grad_next * unit_state).sum(0))
    return tuple(g.to(dtype) for g in grads)


# --------------------------------------------------- the package's own calls ----
def _own(s):
    import mops_amd

    forward = s["case"]["direction"] == "forward"
    if s["case"]["op"] == "embedding":
        if forward:
            return mops_amd.scaled_embedding(s["table"], s["indices"], s["scale"])
        return mops_amd.scaled_embedding_vjp(s["grad_output"], s["table"], s["indices"], s["scale"])
    if s["case"]["op"] == "grouped":
        if forward:
            return mops_amd.grouped_matrix_product(s["A"], s["W"], s["offsets"], s["order"])
        return mops_amd.grouped_matrix_product_vjp(s["grad_output"], s["A"], s["W"], s["offsets"], s["order"])
    inputs = [s[name] for name in ("residual", "block", "gate", "weight_block", "weight_next")]
    if forward:
        return mops_amd.gated_residual_norm(*inputs, s["residual_scale"], EPSILON)
    return mops_amd.gated_residual_norm_vjp(s["grad_state"], s["grad_next"], *inputs, s["residual_scale"], EPSILON)


PLAIN = {"embedding": _plain_embedding, "grouped": _plain_grouped, "update": _plain_update}


def run(state):
    return _own(state) if own else PLAIN[state["case"]["op"]](state)


def work(case):
    width = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "embedding":
        rows, columns, table = case["rows"], case["columns"], case["table_rows"]
        if case["direction"] == "forward":
            # (a row of the table that several rows name is read once)
            return {"bytes": (rows + min(rows, table)) * columns * width + 4 * rows, "flops": rows * columns}
        return {"bytes": (rows + table) * columns * width + 4 * rows, "flops": rows * columns}
    if case["op"] == "grouped":
        rows, k, l = case["rows"], case["k"], case["l"]
        used = min(rows, case["groups"]) * k * l
        index = 4 * rows if case["ordered"] else 0
        if case["direction"] == "forward":
            return {"bytes": (rows * (k + l) + used) * width + index, "flops": 2 * rows * k * l}
        bytes_moved = (rows * (2 * k + l) + used + case["groups"] * k * l) * width + index
        return {"bytes": bytes_moved, "flops": 4 * rows * k * l}
    rows, columns = case["rows"], case["columns"]
    gate = case["gate_rows"]
    if case["direction"] == "forward":
        return {"bytes": (4 * rows + gate + 2) * columns * width, "flops": 11 * rows * columns}
    return {"bytes": (6 * rows + 2 * gate + 4) * columns * width, "flops": 35 * rows * columns}


# ------------------------------------------------------ values in 64 bits ----
def exact(case, seed):
    s = prepare(case, seed)
    wide = {name: t.double() for name, t in s.items() if torch.is_tensor(t) and t.is_floating_point()}
    gradients = case["direction"] == "gradients"
    if case["op"] == "embedding":
        index = s["indices"].long()
        kept = (index >= 0).nonzero().squeeze(1)
        if gradients:
            result = torch.zeros_like(wide["table"])
            result.index_put_((index[kept],), wide["grad_output"][kept] * s["scale"], accumulate=True)
            return result
        result = torch.zeros(case["rows"], case["columns"], dtype=torch.float64, device=index.device)
        result[kept] = torch.index_select(wide["table"], 0, index[kept]) * s["scale"]
        return result
    if case["op"] == "grouped":
        A, W = wide["A"], wide["W"]
        group = torch.full((case["rows"],), -1, dtype=torch.long)
        for g in range(case["groups"]):
            positions = torch.arange(s["boundaries"][g], s["boundaries"][g + 1])
            group[positions if s["order"] is None else s["order"].cpu().long()[positions]] = g
        group = group.to(A.device)
        if not gradients:
            result = torch.zeros(case["rows"], case["l"], dtype=torch.float64, device=A.device)
            for g in range(case["groups"]):
                mask = group == g
                result[mask] = torch.matmul(A[mask], W[g])
            return result
        grad_A, grad_W = torch.zeros_like(A), torch.zeros_like(W)
        for g in range(case["groups"]):
            mask = group == g
            cotangent = wide["grad_output"][mask]
            grad_A[mask] = torch.matmul(W[g], cotangent.t().contiguous()).t()
            grad_W[g] = torch.matmul(A[mask].t().contiguous(), cotangent)
        return grad_A, grad_W
    columns = case["columns"]
    gate = wide["gate"].expand(case["rows"], columns)
    norm_block = torch.sqrt(torch.sum(wide["block"] ** 2, 1, keepdim=True) / columns + EPSILON)
    direction = wide["block"] / norm_block
    state = wide["residual"] + s["residual_scale"] * gate * direction * wide["weight_block"]
    norm_state = torch.sqrt(torch.sum(state**2, 1, keepdim=True) / columns + EPSILON)
    if not gradients:
        return state, state / norm_state * wide["weight_next"]
    onto_next = wide["grad_next"] * wide["weight_next"]
    # d(state_j / norm) / d state_i = (delta_ij - state_i state_j / (columns norm^2)) / norm
    projected = torch.sum(onto_next * state, 1, keepdim=True) / (columns * norm_state**2)
    total = wide["grad_state"] + (onto_next - state * projected) / norm_state
    onto_unit = s["residual_scale"] * total * gate * wide["weight_block"]
    projected = torch.sum(onto_unit * wide["block"], 1, keepdim=True) / (columns * norm_block**2)
    grad_block = (onto_unit - wide["block"] * projected) / norm_block
    grad_gate = s["residual_scale"] * total * direction * wide["weight_block"]
    if case["gate_rows"] == 1:
        grad_gate = torch.sum(grad_gate, 0, keepdim=True)
    grad_weight_block = torch.sum(s["residual_scale"] * total * gate * direction, 0)
    return total, grad_block, grad_gate, grad_weight_block, torch.sum(wide["grad_next"] * state / norm_state, 0)
