"""A small network over atoms, trained for a few steps: the sums over edges and the layers around them together.

Every atom has an element, every edge a pair of atoms and a few radial functions. An element's embedding is the first
state of its atoms; a layer sends the states along the edges (``outer_product_scatter_add_with_weights``), maps what
arrives by a matrix of the atom's element (``grouped_matrix_product``) and adds it to the state, with its two norms and
a learned gate (``gated_residual_norm``). The energy is a last product with a column per element, summed over atoms.
One plan (``order_by_group``) serves all layers.

    python examples/element_network.py
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import mops_amd.torch  # noqa: E402,F401  (registers torch.ops.mops.*)

ATOMS, ELEMENTS, EDGES, RADIAL, CHANNELS, LAYERS = 2000, 5, 30000, 8, 32, 2


def structure(device, dtype=torch.float32, seed=0):
    """Atoms of a few elements (-1: padding), edges sorted by receiver, radial functions, and an energy per structure."""
    generator = torch.Generator().manual_seed(seed)
    elements = torch.randint(0, ELEMENTS, (ATOMS,), generator=generator, dtype=torch.int32)
    elements[-20:] = -1
    receivers = torch.randint(0, ATOMS, (EDGES,), generator=generator, dtype=torch.int32).sort().values
    senders = torch.randint(0, ATOMS, (EDGES,), generator=generator, dtype=torch.int32)
    radial = torch.rand(EDGES, RADIAL, generator=generator, dtype=torch.float64)
    return {
        "elements": elements.to(device), "receivers": receivers.to(device), "senders": senders.to(device),
        "radial": radial.to(device, dtype), "energy": torch.tensor(7.0, device=device, dtype=dtype),
    }  # fmt: skip


def parameters(device, dtype=torch.float32, seed=1):
    generator = torch.Generator().manual_seed(seed)

    def normal(*shape, scale=1.0, mean=0.0):
        values = torch.randn(shape, generator=generator, dtype=torch.float64) * scale + mean
        return values.to(device, dtype).requires_grad_(True)

    result = {"table": normal(ELEMENTS, CHANNELS, scale=CHANNELS**-0.5)}
    for layer in range(LAYERS):
        width = RADIAL * CHANNELS
        result[f"edge{layer}"] = normal(RADIAL, CHANNELS, scale=RADIAL**-0.5)
        result[f"W{layer}"] = normal(ELEMENTS, width, CHANNELS, scale=width**-0.5)
        result[f"gate{layer}"] = normal(1, CHANNELS, scale=0.1, mean=0.5)
        result[f"weight_block{layer}"] = normal(CHANNELS, scale=0.1, mean=1.0)
        result[f"weight_next{layer}"] = normal(CHANNELS, scale=0.1, mean=1.0)
    result["readout"] = normal(ELEMENTS, CHANNELS, 1, scale=CHANNELS**-0.5)
    return result


def energy(p, s, ops=torch.ops.mops):
    """The energy of a structure; ``ops``: where the operators come from."""
    order, offsets = ops.order_by_group(s["elements"], ELEMENTS)
    state = ops.scaled_embedding(p["table"], s["elements"], CHANNELS**0.5)
    features = state
    for layer in range(LAYERS):
        edges = s["radial"] @ p[f"edge{layer}"]
        message = ops.outer_product_scatter_add_with_weights(
            s["radial"], edges, features, s["senders"], s["receivers"]
        ).reshape(ATOMS, RADIAL * CHANNELS)
        block = ops.grouped_matrix_product(message, p[f"W{layer}"], offsets, order)
        state, features = ops.gated_residual_norm(
            state, block, p[f"gate{layer}"], p[f"weight_block{layer}"], p[f"weight_next{layer}"], 0.5, 1e-6
        )
    return ops.grouped_matrix_product(features, p["readout"], offsets, order).sum() / ATOMS


def train(steps=20, device="cuda"):
    """Loss of every step."""
    s, p = structure(device), parameters(device)
    optimizer = torch.optim.Adam(list(p.values()), lr=0.02)
    losses = []
    for _ in range(steps):
        optimizer.zero_grad()
        loss = (energy(p, s) - s["energy"]) ** 2
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
    return losses


if __name__ == "__main__":
    for step, loss in enumerate(train()):
        print(f"step {step:2d}: loss {loss:.4f}")
