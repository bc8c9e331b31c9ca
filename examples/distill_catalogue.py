"""A graph network that classifies nodes over a large catalogue, and a smaller
one distilled from its top logits.

    python examples/distill_catalogue.py [--nodes N] [--classes V] [--epochs E]

Both are GCN_BCSR bodies with a LinearHead over the classes; no step keeps
the [nodes, classes] logits.  The teacher is trained on the labels, its best
`--top` classes of every training node are listed once, and the student
learns from the labels and the lists together.  The graph and labels are
synthetic: a node's class is that of its community's nearest prototype.
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from graph_rws_amd import synth  # noqa: E402
from graph_rws_amd.data import BCSRGraph  # noqa: E402
from graph_rws_amd.helper import evaluate_head, train_epoch_head  # noqa: E402
from graph_rws_amd.layers import LinearHead  # noqa: E402
from graph_rws_amd.models import GCN_BCSR  # noqa: E402


def dataset(nodes: int, classes: int, width: int, device):
    """A community graph whose features hold a noisy code of the node's class."""
    g = synth.sbm(nodes, max(2, nodes // 2000), 0.8, 16 * nodes, seed=1, device=device)
    graph = BCSRGraph.from_csr(g.row_ptr, g.col_idx, g.values, nodes, nodes, tile_cols=16, device=device,
                               values_dtype=torch.bfloat16)
    gen = torch.Generator(device=device)
    gen.manual_seed(2)
    labels = torch.randint(0, classes, (nodes,), generator=gen, device=device)
    codes = torch.randn(classes, width, generator=gen, device=device)
    features = codes[labels] + 0.5 * torch.randn(nodes, width, generator=gen, device=device)
    chosen = torch.rand(nodes, generator=gen, device=device) < 0.7
    return graph, features, labels, chosen.nonzero()[:, 0], (~chosen).nonzero()[:, 0]


def build(width: int, hidden: int, classes: int, device):
    body = GCN_BCSR(width, hidden, hidden, 2, dropout=0.0, use_checkpoint=False).to(device)
    head = LinearHead(hidden, classes).to(device)
    return body, head, torch.optim.Adam([*body.parameters(), *head.parameters()], lr=5e-3)


def train(name, parts, data, epochs, device, teacher=None):
    body, head, optimizer = parts
    graph, features, labels, train_idx, eval_idx = data
    graphs = body._ensure_graph_list(graph)
    for epoch in range(epochs):
        begin = time.perf_counter()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            loss, acc = train_epoch_head(body, head, graphs, features, labels, train_idx, optimizer, device,
                                         teacher=teacher)
        if epoch % 10 == 0 or epoch == epochs - 1:
            print(f"{name} epoch {epoch}: loss {loss:.3f}, accuracy {float(acc):.3f}, "
                  f"{1e3 * (time.perf_counter() - begin):.1f} ms", flush=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss, acc = evaluate_head(body, head, graph, features, labels, eval_idx)
    print(f"{name}: held-out loss {loss:.3f}, accuracy {acc:.3f}", flush=True)
    return loss, acc


def main():
    p = argparse.ArgumentParser()
    p.add_argument("--nodes", type=int, default=20000)
    p.add_argument("--classes", type=int, default=20011)
    p.add_argument("--width", type=int, default=128)
    p.add_argument("--epochs", type=int, default=40)
    p.add_argument("--top", type=int, default=32)
    a = p.parse_args()
    device = torch.device("cuda", 0)
    torch.manual_seed(0)
    data = dataset(a.nodes, a.classes, a.width, device)
    graph, features, _, train_idx, _ = data
    teacher = build(a.width, 256, a.classes, device)
    train("teacher", teacher, data, a.epochs, device)
    body, head, _ = teacher
    body.eval()
    with torch.autocast("cuda", dtype=torch.bfloat16), torch.no_grad():
        hidden = body.inference(graph, features)
        lists = head.top(hidden[train_idx], a.top)
    train("student", build(a.width, 64, a.classes, device), data, a.epochs, device, teacher=lists)


if __name__ == "__main__":
    main()
