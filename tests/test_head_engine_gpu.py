"""LinearHead and train_epoch_head: the fused losses on a graph model, against
the same step from torch's own ops on kept logits.

The fused step's f32 sums differ from torch's by their order and the split
f32 products: gradients agree to 1e-4 of their largest magnitude (the bound
of the fused epilogues' tests), losses to 1e-5."""
import copy

import pytest
import torch
import torch.nn.functional as F

from graph_rws_amd import synth
from graph_rws_amd.data import BCSRGraph
from graph_rws_amd.helper import evaluate_head, train_epoch_head
from graph_rws_amd.layers import LinearHead
from graph_rws_amd.models import GCN_BCSR

pytestmark = pytest.mark.gpu


def _problem(dev, nodes=1500, width=40, hidden=48, classes=777):
    torch.manual_seed(7)
    g = synth.chung_lu(nodes, 6 * nodes, 2.3, seed=4)
    graph = BCSRGraph.from_csr(g.row_ptr, g.col_idx, g.values, nodes, nodes, tile_cols=16, device=dev)
    features = torch.randn(nodes, width, device=dev)
    labels = torch.randint(0, classes, (nodes,), device=dev)
    idx = (torch.rand(nodes, device=dev) < 0.6).nonzero()[:, 0]
    model = GCN_BCSR(width, hidden, hidden, 2, dropout=0.0, use_checkpoint=False).to(dev)
    head = LinearHead(hidden, classes).to(dev)
    return graph, features, labels, idx, model, head


@pytest.mark.parametrize("distilled", [False, True])
def test_step_matches_torch_ops(cuda_device, distilled):
    graph, features, labels, idx, model, head = _problem(cuda_device)
    teacher = None
    if distilled:
        teacher = LinearHead(48, 777).to(cuda_device).top(torch.randn(idx.numel(), 48, device=cuda_device), 9,
                                                          rows_at_once=100)
    twin, twin_head = copy.deepcopy(model), copy.deepcopy(head)
    params = [*model.parameters(), *head.parameters()]
    loss, acc = train_epoch_head(model, head, model._ensure_graph_list(graph), features, labels, idx,
                                 torch.optim.SGD(params, lr=0.0), cuda_device, teacher=teacher, temperature=2.0)
    logits = twin_head(twin(twin._ensure_graph_list(graph), features)[idx])
    want = F.cross_entropy(logits, labels[idx])
    hits = int((logits.argmax(1) == labels[idx]).sum())
    if distilled:
        values, classes = teacher
        q = torch.softmax(values / 2.0, 1)
        logp = torch.log_softmax(logits / 2.0, 1).gather(1, classes.long())
        want = 0.5 * want + 0.5 * 4.0 * (q * (q.log() - logp)).sum(1).mean()
    twins = [*twin.parameters(), *twin_head.parameters()]
    grads = torch.autograd.grad(want, twins)
    torch.nn.utils.clip_grad_norm_(twins, 1.0)
    assert abs(loss - float(want.detach())) <= 1e-5 * abs(float(want.detach()))
    assert round(float(acc) * idx.numel()) == hits
    norm = torch.sqrt(sum((g.double() ** 2).sum() for g in grads))
    scale = min(1.0, 1.0 / (float(norm) + 1e-6))
    for p, g in zip(params, grads):
        assert float((p.grad - scale * g).abs().max()) <= 1e-4 * float((scale * g).abs().max())


def test_training_and_evaluation(cuda_device):
    """A few epochs under autocast lower the loss; evaluation agrees with the
    kept logits."""
    graph, features, labels, idx, model, head = _problem(cuda_device)
    opt = torch.optim.Adam([*model.parameters(), *head.parameters()], lr=1e-2)
    graphs = model._ensure_graph_list(graph)
    losses = []
    for _ in range(12):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            loss, _ = train_epoch_head(model, head, graphs, features, labels, idx, opt, cuda_device)
        losses.append(loss)
    assert losses[-1] < 0.9 * losses[0]
    loss, acc = evaluate_head(model, head, graph, features, labels, idx)
    logits = head(model.inference(graph, features)[idx])
    assert abs(loss - float(F.cross_entropy(logits, labels[idx]))) <= 1e-5 * loss
    assert abs(acc - float((logits.argmax(1) == labels[idx]).float().mean())) <= 1.5 / idx.numel()


def test_head_top_in_batches(cuda_device):
    head = LinearHead(32, 500).to(cuda_device)
    x = torch.randn(70, 32, device=cuda_device)
    values, classes = head.top(x, 6, rows_at_once=16)
    v, c = torch.sort(torch.cat([head(x[i:i + 16]) for i in range(0, 70, 16)]).detach(), dim=1, descending=True,
                      stable=True)
    assert torch.equal(values, v[:, :6]) and torch.equal(classes.long(), c[:, :6])


@pytest.mark.parametrize("kind", ["repeated", "shuffled", "mask"])
def test_step_with_other_indices(cuda_device, kind):
    """Rows listed twice, in any order, or a mask train as torch's ops do."""
    graph, features, labels, idx, model, head = _problem(cuda_device)
    if kind == "repeated":
        idx = torch.cat([idx, idx[::3], idx[:5]])
    elif kind == "shuffled":
        idx = idx[torch.randperm(idx.numel(), device=cuda_device)]
    else:
        idx = torch.zeros(features.shape[0], dtype=torch.bool, device=cuda_device).index_fill(0, idx, True)
    at = idx.nonzero()[:, 0] if kind == "mask" else idx
    n = at.numel()
    values, classes = LinearHead(48, 777).to(cuda_device).top(torch.randn(n, 48, device=cuda_device), 9)
    twin, twin_head = copy.deepcopy(model), copy.deepcopy(head)
    params = [*model.parameters(), *head.parameters()]
    loss, acc = train_epoch_head(model, head, model._ensure_graph_list(graph), features, labels, idx,
                                 torch.optim.SGD(params, lr=0.0), cuda_device, teacher=(values, classes))
    logits = twin_head(twin(twin._ensure_graph_list(graph), features)[at])
    q = torch.softmax(values / 2.0, 1)
    logp = torch.log_softmax(logits / 2.0, 1).gather(1, classes.long())
    want = 0.5 * F.cross_entropy(logits, labels[at]) + 0.5 * 4.0 * (q * (q.log() - logp)).sum(1).mean()
    twins = [*twin.parameters(), *twin_head.parameters()]
    grads = torch.autograd.grad(want, twins)
    assert abs(loss - float(want.detach())) <= 1e-5 * abs(float(want.detach()))
    assert round(float(acc) * n) == int((logits.argmax(1) == labels[at]).sum())
    norm = torch.sqrt(sum((g.double() ** 2).sum() for g in grads))
    scale = min(1.0, 1.0 / (float(norm) + 1e-6))
    for p, g in zip(params, grads):
        assert float((p.grad - scale * g).abs().max()) <= 1e-4 * float((scale * g).abs().max())
    loss, acc = evaluate_head(model, head, graph, features, labels, idx)
    logits = head(model.inference(graph, features)[at])
    assert abs(loss - float(F.cross_entropy(logits, labels[at]))) <= 1e-5 * loss
