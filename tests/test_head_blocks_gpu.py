"""The fused classifier losses (csrc/head.hip) where a call is cut up: blocks
of rows, pieces of the classes, runs of the sums, both tiles.  Every test
says which cuts it is there for and checks that the call has them.

Bounds as in test_head_gpu, formed per element from the 64-bit reference."""
import ctypes

import pytest
import torch

from graph_rws_amd.core import _lib as L
from graph_rws_amd.core import ops
from graph_rws_amd.layers import linear_cross_entropy, linear_distill
from test_head_gpu import _inputs, _onehot, _Ref, _teacher

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def plan(backward, h, w, n, k=0):
    """{blocks, rows, pieces, classes, few, tile, dw_tile, dw_runs, dh_tile, dh_runs} of a call."""
    view = L.HeadView(h.data_ptr(), w.data_ptr(), None, None, None if k else 8, 8 if k else None, 8 if k else None,
                      h.stride(0), w.stride(0), h.shape[0], n, h.shape[1], w.shape[0], L.dtype_code(h.dtype), k, 0, 1.0)
    out = (ctypes.c_int64 * 10)()
    L.call("grws_head_plan", ctypes.byref(view), backward, out)
    return dict(zip(("blocks", "rows", "pieces", "classes", "few", "tile", "dw_tile", "dw_runs", "dh_tile", "dh_runs"),
                    out))


def _check(dev, dt, n, width, classes, seed, nodes=None, k=0, scale=1.0):
    """A step of a call against 64 bits; returns the inputs."""
    h, w, b, labels = _inputs(dev, n, width, classes, dt, seed, nodes=nodes, bias=True)
    rows = torch.randperm(nodes, device=dev)[:n] if nodes else None
    params = [x.requires_grad_(True) for x in (h, w, b)]
    if k:
        # distinct classes: _Ref's entropy is that of the summed probabilities
        index = (torch.randint(0, classes, (n, 1), device=dev) + torch.arange(k, device=dev) * 7) % classes
        index[1::6] = -1
        teacher = torch.randn(n, k, device=dev) * 3
        loss, counts = linear_distill(h, w, index, teacher, bias=b, rows=rows, temperature=2.0)
        target, live = _teacher(index, teacher, classes, 2.0)
        ref = _Ref(h.detach(), w.detach(), b.detach(), rows, target, live, 2.0)
        assert counts.tolist() == [ref.count, 0]
    else:
        labels[1::6] = -100
        loss, counts = linear_cross_entropy(h, w, labels, bias=b, rows=rows)
        ref = _Ref(h.detach(), w.detach(), b.detach(), rows, *_onehot(labels, classes))
        assert counts.tolist()[1:] == [ref.count, 0]
    grads = torch.autograd.grad(loss, params, torch.tensor(scale, device=dev))
    ref.check_loss(loss)
    ref.check_grads(*grads, scale / ref.count)


@pytest.mark.parametrize("dt,n,width,classes,nodes,k", [
    (torch.bfloat16, 130000, 24, 4300, None, 0), (torch.float16, 130000, 24, 4300, 140000, 0),
    (torch.float32, 60000, 24, 4300, None, 0), (torch.float32, 60000, 24, 9000, 70000, 0),
    (torch.float32, 50001, 24, 4300, None, 3), (torch.bfloat16, 1100003, 16, 47, None, 0),
    (torch.float16, 1100003, 16, 47, 1200000, 2), (torch.float32, 1100003, 16, 47, None, 2)])
def test_blocks_of_rows(cuda_device, dt, n, width, classes, nodes, k):
    print(f"case blocks {dt} {n}x{width}x{classes} rows of {nodes} k={k}", flush=True)
    h = torch.empty(nodes or n, width, device=cuda_device, dtype=dt)
    p = plan(1, h, torch.empty(classes, width, device=cuda_device, dtype=dt), n, k)
    assert p["blocks"] > 1 and (p["pieces"] > 1) == (classes == 9000) and n % p["rows"]
    _check(cuda_device, dt, n, width, classes, 4, nodes, k, 4096.0)


@pytest.mark.parametrize("kind", ["labels", "lists"])
def test_blocks_of_rows_forward(cuda_device, kind):
    """Row losses of several blocks, and the mean, against 64 bits."""
    n, width, classes, dt = 70001, 16, 66000, torch.bfloat16
    h, w, b, labels = _inputs(cuda_device, n, width, classes, dt, 4, bias=True)
    assert plan(0, h, w, n)["blocks"] == 2
    labels[::9] = -100
    index = torch.randint(0, classes, (n, 2), device=cuda_device)
    index[::9] = -1
    teacher = torch.randn(n, 2, device=cuda_device)
    if kind == "labels":
        row, counts = linear_cross_entropy(h, w, labels, bias=b, reduction="none")
        mean, again = linear_cross_entropy(h, w, labels, bias=b)
    else:
        row, counts = linear_distill(h, w, index, teacher, bias=b, reduction="none")
        mean, again = linear_distill(h, w, index, teacher, bias=b)
    assert torch.equal(counts, again)
    hits = 0
    for i in range(0, n, 10000):
        z = h[i:i + 10000].double() @ w.double().t() + b.double()
        logp = torch.log_softmax(z, 1)
        if kind == "labels":
            y = labels[i:i + 10000]
            live = y >= 0
            ref = -logp.gather(1, y.clamp(min=0)[:, None])[:, 0]
            hits += int(((z.argmax(1) == y) & live).sum())
        else:
            q = torch.softmax(teacher[i:i + 10000].double(), 1)
            live = index[i:i + 10000, 0] >= 0
            ref = (q * (q.log() - logp.gather(1, index[i:i + 10000].clamp(min=0)))).sum(1)
        # logits off by 24 2^-23 of 16 products' magnitudes (20 at most), twice
        assert float((row[i:i + 10000].double() - torch.where(live, ref, 0.0)).abs().max()) <= 2e-4
    assert int(counts[-2]) == int((labels >= 0).sum()) and int(counts[-1]) == 0
    if kind == "labels":
        assert abs(int(counts[0]) - hits) <= 2  # logits closer than their rounding
    assert abs(float(mean) - float(row.double().sum()) / int(counts[-2])) <= 1e-6 * float(mean)


def test_blocks_of_rows_and_repeated_rows(cuda_device):
    """A row listed in two blocks; a factor per row; the last block short."""
    n, width, classes, dt = 130000, 16, 4300, torch.bfloat16
    h, w, b, labels = _inputs(cuda_device, n, width, classes, dt, 4, nodes=n + 9, bias=True)
    assert plan(1, h, w, n)["blocks"] == 2
    rows = torch.randperm(n + 9, device=cuda_device)[:n]
    rows[n - 1] = rows[3]
    factors = torch.randn(n, device=cuda_device)
    out = []
    for r in (rows, None):
        params = [x.detach().requires_grad_(True) for x in (h if r is not None else h[rows], w, b)]
        loss, _ = linear_cross_entropy(params[0], params[1], labels, bias=params[2], rows=r, reduction="none")
        out.append([loss.detach(), *torch.autograd.grad(loss, params, factors)])
    (loss, dh, dw, db), (loss2, dx, dw2, db2) = out
    assert torch.equal(loss, loss2) and torch.equal(dw, dw2) and torch.equal(db, db2)
    assert torch.isnan(dh).any(1).nonzero()[:, 0].tolist() == [int(rows[3])]
    want = torch.zeros_like(dh)
    want[rows] = dx
    dh[rows[3]] = want[rows[3]]
    assert torch.equal(dh, want)


@pytest.mark.parametrize("dt,n,width,classes", [
    (torch.bfloat16, 66000, 16, 9300), (torch.float16, 66000, 16, 9300),  # pieces, runs
    (torch.bfloat16, 66000, 256, 9300),  # pieces of one run: the last adds and writes
    (torch.float32, 40000, 256, 6000)])
def test_pieces_of_classes(cuda_device, dt, n, width, classes):
    """G of all the classes passes its bound: the hidden gradient is added up
    over the pieces."""
    print(f"case pieces {dt} {n}x{width}x{classes}", flush=True)
    p = plan(1, torch.empty(n, width, device=cuda_device, dtype=dt),
             torch.empty(classes, width, device=cuda_device, dtype=dt), n)
    assert p["blocks"] == 1 and p["pieces"] > 1, p
    assert (p["dh_runs"] == 1 and p["dh_tile"] == 256) or width != 256 or dt == torch.float32, p
    _check(cuda_device, dt, n, width, classes, 5, scale=4096.0)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("k", [0, 4])
def test_large_tiles_of_one_run(cuda_device, dt, k):
    """256-tiles of both gradients, each all of its sum (f32: of two pieces,
    which the hidden gradient adds up, and two runs of the weight gradient)."""
    n, width, classes = 16384 - 5, 1000, 16384 - 3
    print(f"case tiles {dt} k={k}", flush=True)
    p = plan(1, torch.empty(n, width, device=cuda_device, dtype=dt),
             torch.empty(classes, width, device=cuda_device, dtype=dt), n, k)
    assert (p["tile"], p["dw_tile"], p["dh_tile"], p["dh_runs"]) == (256, 256, 256, 1), p
    assert p["dw_runs"] == p["pieces"] == (2 if dt == torch.float32 else 1), p
    _check(cuda_device, dt, n, width, classes, 6, k=k, scale=4096.0)


@pytest.mark.parametrize("n", [1, 40, 300])
def test_pieces_of_packed_weight(cuda_device, n):
    """f32 weight in several packed pieces, forward and backward (few rows
    read it as it lies, but take the same pieces backward)."""
    width, classes, dt = 1030, 50000, torch.float32
    h, w = torch.empty(n, width, device=cuda_device), torch.empty(classes, width, device=cuda_device)
    f, b = plan(0, h, w, n), plan(1, h, w, n)
    assert b["pieces"] > 1 and f["few"] == b["few"] == (n <= 128) and (n <= 128 or f["pieces"] > 1), (f, b)
    _check(cuda_device, dt, n, width, classes, 7)
    _check(cuda_device, dt, n, width, classes, 8, nodes=2 * n, k=4)


@pytest.mark.parametrize("n", [20, 300])
def test_pieces_of_unaligned_weight(cuda_device, n):
    """The same of a 16-bit weight whose rows are not 16-byte aligned."""
    width, classes, dt = 1030, 140000, torch.bfloat16
    h, w = (torch.empty(x, width, device=cuda_device, dtype=dt) for x in (n, classes))
    f, b = plan(0, h, w, n), plan(1, h, w, n)
    assert b["pieces"] > 1 and f["few"] == (n <= 32) and (n <= 32 or f["pieces"] > 1), (f, b)
    _check(cuda_device, dt, n, width, classes, 9)
