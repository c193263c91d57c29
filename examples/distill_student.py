"""Distills a graph network into a student without message passing.

A two-layer GCN (here with fixed random weights) labels the nodes of a batch of
graphs.  Its best classes of each node, with their log probabilities, are kept
(``label_log_probs`` with ``top``), and a student sees the nodes' own features
alone:

    h = gelu(group_norm(x W1 + b1))        statistics over each graph's nodes
    z = h W2 + b2

Its loss at each node is ``mix`` times the distillation loss against the
teacher's best classes and 1 - mix times the cross entropy of the node's label
(where it has one), less a little of the entropy.

    python examples/distill_student.py [--graphs 64] [--nodes 20000] [--classes 41] [--top 5] [--steps 30]
"""
from __future__ import annotations

import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import tinygnn_b200 as tg  # noqa: E402
from tinygnn_b200 import synth  # noqa: E402


class Student:
    """Linear, group norm with GELU, linear, with its backward pass."""

    def __init__(self, features: int, hidden: int, classes: int, groups: int, dtype=torch.bfloat16, seed: int = 0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        init = lambda k, n: (torch.randn(1, k, n, device="cuda", generator=g) / math.sqrt(k))  # noqa: E731
        self.groups, self.dtype = groups, dtype
        self.params = {  # fp32 masters
            "w1": init(features, hidden), "b1": torch.zeros(1, hidden, device="cuda"),
            "gamma": torch.ones(hidden, device="cuda"), "beta": torch.zeros(hidden, device="cuda"),
            "w2": init(hidden, classes), "b2": torch.zeros(1, classes, device="cuda")}

    def forward(self, x: torch.Tensor, graphs: torch.Tensor):
        """(logits, what the backward pass needs); graphs: the graphs' row offsets."""
        p = self.params
        all_rows = torch.tensor([0, x.shape[0]], dtype=torch.int32, device="cuda")
        w1, w2 = p["w1"].to(self.dtype), p["w2"].to(self.dtype)
        a = tg.typed_linear(x, w1, all_rows, p["b1"])
        h, stats = tg.group_norm(a, p["gamma"], p["beta"], self.groups, graphs, "gelu")
        z = tg.typed_linear(h, w2, all_rows, p["b2"])
        return z, (x, a, h, stats, w1, w2, all_rows, graphs)

    def backward(self, dz: torch.Tensor, kept):
        """Gradients by name; weight gradients in fp32."""
        x, a, h, stats, w1, w2, all_rows, graphs = kept
        p, grads = self.params, {}
        dh, grads["w2"], grads["b2"] = tg.typed_linear_backward(dz, h, w2, all_rows, torch.float32)
        da, grads["gamma"], grads["beta"] = tg.group_norm_backward(dh, a, stats, p["gamma"], p["beta"], self.groups, graphs, "gelu")
        grads["w1"], grads["b1"] = tg.typed_linear_grad_weight(x, da, all_rows, torch.float32)
        return grads


def loss_and_gradient(z, labels, top_classes, top_log_probs, mix: float = 0.7, temperature: float = 2.0, entropy: float = 0.01):
    """(mean loss, dlogits) of a student's logits; labels outside the classes count as none."""
    rows = z.shape[0]
    weight = torch.full((rows,), mix / rows, device=z.device)
    distill, dz = tg.distill_loss(z, top_classes, top_log_probs, temperature, weight)
    log_probs, h, stats = tg.label_log_probs(z, labels)
    dlog = torch.full((rows,), (mix - 1) / rows, device=z.device)
    dent = torch.full((rows,), -entropy / rows, device=z.device)
    dz = dz + tg.label_log_probs_backward(dlog, z, labels, stats, dent, h)
    return (mix * distill - (1 - mix) * log_probs - entropy * h).mean(), dz


def batch(graphs: int, nodes: int, features: int, seed: int):
    """(adjacency of all graphs, its diagonal blocks; features; the graphs' row offsets)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    cuts = torch.randint(0, nodes + 1, (graphs - 1,), device="cuda", generator=g).sort().values
    ends = torch.tensor([0, nodes], device="cuda")
    offsets = torch.cat([ends[:1], cuts, ends[1:]]).to(torch.int32)
    of = torch.searchsorted(offsets[1:].long(), torch.arange(nodes, device="cuda"), right=True)   # a node's graph
    first, size = offsets[:-1].long()[of], (offsets[1:] - offsets[:-1]).long()[of]
    src = torch.arange(nodes, device="cuda").repeat_interleave(8)
    dst = first[src] + (torch.rand(src.shape[0], device="cuda", generator=g) * size[src]).long().clamp(max=nodes)
    dst = torch.minimum(dst, first[src] + size[src] - 1)
    adj = tg.edge_list_to_csr(src.to(torch.int32), dst.to(torch.int32), nodes)
    return adj, synth.normal_rows(0, nodes, features, seed + 1, 0, "cuda"), tg.check_row_offsets(offsets, nodes)


def train(graphs: int = 64, nodes: int = 20000, features: int = 96, hidden: int = 128, classes: int = 41, top: int = 5,
          steps: int = 30, lr: float = 0.5, dtype=torch.bfloat16, seed: int = 0, report=print):
    adj, x, offsets = batch(graphs, nodes, features, seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 7)
    w = [torch.randn(a, b, device="cuda", generator=g) * 2.0 / math.sqrt(a) for a, b in ((features, hidden), (hidden, classes))]
    norm = tg.gcn_norm(adj)
    teacher = tg.gcn_layer(norm, tg.gcn_layer(norm, x, w[0], None, "relu"), w[1], None, None)
    labels = teacher.argmax(1)
    labels[torch.rand(nodes, device="cuda", generator=g) < 0.5] = -1      # half of the nodes have one
    best = tg.label_log_probs(teacher, labels, top)[3:]
    student, rows = Student(features, hidden, classes, 8, dtype, seed), x.to(dtype)
    losses = []
    for step in range(steps):
        z, kept = student.forward(rows, offsets)
        loss, dz = loss_and_gradient(z, labels, best[1], best[0])
        for name, grad in student.backward(dz, kept).items():
            student.params[name] -= lr * grad.view_as(student.params[name])
        losses.append(float(loss))
        if report and (step % 10 == 0 or step == steps - 1):
            report(f"step {step:4d}  loss {losses[-1]:.5f}")
    return losses


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, value in (("graphs", 64), ("nodes", 20000), ("classes", 41), ("top", 5), ("steps", 30)):
        ap.add_argument(f"--{name}", type=int, default=value)
    train(**vars(ap.parse_args()))
