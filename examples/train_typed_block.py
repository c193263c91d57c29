"""Trains a typed feed-forward block on a synthetic heterogeneous graph.

Nodes have types and are sorted by type.  Each node's features are averaged
over its neighbours (the library's sparse product), then pass the block

    n = layer_norm(x)                      x: a node's features and its neighbours' mean
    a = gelu(n W1[type] + b1[type])
    y = x + a W2[type] + b2[type]

and the loss is the mean squared distance of y from a target.  The forward
pass keeps what the backward pass needs in 8 bits: the normalised rows, the
pre-activation and the activation (``--full`` keeps them as they are).

    python examples/train_typed_block.py [--nodes 20000] [--width 256] [--types 6] [--steps 30] [--full]
"""
from __future__ import annotations

import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import tinygnn_b200 as tg  # noqa: E402


class TypedBlock:
    """x + typed_linear(gelu(typed_linear(layer_norm(x)))), with its backward
    pass.  ``save8``: the saved activations are 8-bit copies."""

    def __init__(self, types: int, width: int, hidden: int, dtype=torch.bfloat16, save8: bool = True, seed: int = 0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        init = lambda k, n: (torch.randn(types, k, n, device="cuda", generator=g) / math.sqrt(k))  # noqa: E731
        self.dtype, self.save8 = dtype, save8
        self.params = {  # fp32 masters
            "gamma": torch.ones(width, device="cuda"), "beta": torch.zeros(width, device="cuda"),
            "w1": init(width, hidden), "b1": torch.zeros(types, hidden, device="cuda"),
            "w2": init(hidden, width) * 0.1, "b2": torch.zeros(types, width, device="cuda")}

    def forward(self, x: torch.Tensor, offsets: torch.Tensor):
        """(y, what the backward pass needs)."""
        p = self.params
        w1, w2 = p["w1"].to(self.dtype), p["w2"].to(self.dtype)
        if self.save8:
            n, stats, h = tg.layer_norm(x, p["gamma"], p["beta"], save8=True)
            a, z = tg.typed_linear(n, w1, offsets, p["b1"], "gelu", save8=True)
            n_kept, a_kept = tg.save8(n), tg.save8(a)
        else:
            n, stats = tg.layer_norm(x, p["gamma"], p["beta"])
            z = tg.typed_linear(n, w1, offsets, p["b1"])
            a = tg.activation_save8(z, "gelu")[0]
            h, n_kept, a_kept = x, n, a
        y = x + tg.typed_linear(a, w2, offsets, p["b2"])
        return y, (h, stats, n_kept, z, a_kept, w1, w2, offsets)

    def backward(self, dy: torch.Tensor, kept):
        """(dx, gradients by name); weight gradients in fp32."""
        h, stats, n, z, a, w1, w2, offsets = kept
        grads = {}
        da, grads["w2"], grads["b2"] = tg.typed_linear_backward(dy, a, w2, offsets, dtype=torch.float32)
        dz = tg.activation_backward(da, z, "gelu")
        dn, grads["w1"], grads["b1"] = tg.typed_linear_backward(dz, n, w1, offsets, dtype=torch.float32)
        dx, grads["gamma"], grads["beta"] = tg.layer_norm_backward(dn, h, stats, self.params["gamma"])
        return dx + dy, grads

    def step(self, grads, rate: float) -> None:
        for name, g in grads.items():
            self.params[name].sub_(rate * g)


def kept_bytes(kept) -> int:
    """Bytes of the saved activations (the weights and offsets are not counted)."""
    size = lambda t: t.nbytes if isinstance(t, tg.Saved8) else t.numel() * t.element_size()  # noqa: E731
    return sum(size(t) for t in kept[:5])


def graph(nodes: int, degree: int, seed: int) -> tg.CSR:
    """A random graph, every row scaled to a mean."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    src = torch.randint(nodes, (nodes * degree,), device="cuda", generator=g, dtype=torch.int32)
    dst = torch.randint(nodes, (nodes * degree,), device="cuda", generator=g, dtype=torch.int32)
    A = tg.edge_list_to_csr(src, dst, nodes)
    lengths = (A.row_ptr[1:] - A.row_ptr[:-1]).clamp(min=1)
    A.values = torch.repeat_interleave(1.0 / lengths.float(), (A.row_ptr[1:] - A.row_ptr[:-1]).long())
    return A


def train(nodes=20000, width=256, types=6, steps=30, save8=True, seed=0, rate=0.5, report=print):
    """The losses of `steps` steps."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    cuts = torch.sort(torch.randint(nodes + 1, (types - 1,), device="cuda", generator=g))[0]
    offsets = torch.cat([torch.zeros(1, device="cuda"), cuts, torch.full((1,), nodes, device="cuda")]).int()
    tg.check_row_offsets(offsets, nodes)
    features = torch.randn(nodes, width, device="cuda", generator=g)
    x = (features + tg.spmm(graph(nodes, 8, seed), features)).to(torch.bfloat16)
    # a target that depends on the type: what each type's block has to learn
    sizes = (offsets[1:] - offsets[:-1]).long()
    mix = torch.randn(types, width, device="cuda", generator=g)
    target = x.float() + torch.tanh(x.float() * torch.repeat_interleave(mix, sizes, 0))

    block = TypedBlock(types, width, 2 * width, save8=save8, seed=seed)
    losses = []
    for i in range(steps):
        y, kept = block.forward(x, offsets)
        off = y.float() - target
        losses.append((off * off).mean())
        dy = (off * (2.0 / width)).to(torch.bfloat16)
        _, grads = block.backward(dy, kept)
        block.step(grads, rate * types / nodes)
        if report and (i % 10 == 0 or i == steps - 1):
            report(f"step {i}: loss {losses[-1].item():.4f}, saved activations {kept_bytes(kept) / 2**20:.1f} MiB")
    return [v.item() for v in losses]


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--nodes", type=int, default=20000)
    ap.add_argument("--width", type=int, default=256)
    ap.add_argument("--types", type=int, default=6)
    ap.add_argument("--steps", type=int, default=30)
    ap.add_argument("--full", action="store_true", help="keep the activations as they are")
    a = ap.parse_args()
    train(a.nodes, a.width, a.types, a.steps, save8=not a.full)
