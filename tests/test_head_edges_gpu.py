"""Edges of the fused classifier losses (csrc/head.hip): upstream gradients,
exact comparisons, extreme logits, layouts.

Where two calls have to agree they agree bit for bit; other tolerances are
stated at the test."""
import math

import numpy as np
import pytest
import torch

from graph_rws_amd.core import ops
from graph_rws_amd.layers import linear_cross_entropy, linear_distill

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _inputs(dev, n, width, classes, dt, seed, nodes=None):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    h = torch.randn(nodes or n, width, generator=g, device=dev).to(dt)
    w = (torch.randn(classes, width, generator=g, device=dev) * 2 / math.sqrt(width)).to(dt)
    b = torch.randn(classes, generator=g, device=dev).to(dt)
    labels = torch.randint(0, classes, (n,), generator=g, device=dev)
    lists = torch.stack([torch.randperm(classes, generator=g, device=dev)[:5] for _ in range(n)]).int()
    teacher = torch.randn(n, 5, generator=g, device=dev)
    return h, w, b, labels, lists, teacher


def _row_grads(kind, h, w, b, target, factors):
    """Row losses and the gradients of their sum weighted by factors."""
    params = [x.detach().requires_grad_(True) for x in (h, w, b)]
    if kind == "labels":
        loss, _ = linear_cross_entropy(params[0], params[1], target, bias=params[2], reduction="none")
    else:
        loss, _ = linear_distill(params[0], params[1], *target, bias=params[2], temperature=2.0, reduction="none")
    return [loss.detach(), *torch.autograd.grad(loss, params, factors)]


# 9 rows: the kernels of few rows; 200: the products
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("n", [9, 200])
@pytest.mark.parametrize("kind", ["labels", "lists"])
def test_factors_of_rows_that_do_not_count(cuda_device, dt, n, kind):
    """Whatever the upstream gradient holds at a row that does not count, the
    gradients are those of a zero there."""
    print(f"case dead factors {dt} {n} {kind}", flush=True)
    h, w, b, labels, lists, teacher = _inputs(cuda_device, n, 40, 300, dt, 5)
    labels[::4] = -100
    lists[::4] = -1
    target = labels if kind == "labels" else (lists, teacher)
    factors = torch.randn(n, device=cuda_device)
    factors[::4] = 0
    want = _row_grads(kind, h, w, b, target, factors)
    assert all(bool(torch.isfinite(x).all()) for x in want)
    for bad in (math.nan, math.inf, -math.inf, 3e38):
        factors[::4] = bad
        for x, y in zip(want, _row_grads(kind, h, w, b, target, factors)):
            assert torch.equal(x, y), bad


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("n", [9, 200])
@pytest.mark.parametrize("kind", ["labels", "lists"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_bad_factor_stays_in_its_row(cuda_device, dt, n, kind, bad):
    """An upstream gradient that is not finite spoils its own row of the
    hidden gradient and no other."""
    print(f"case bad factor {dt} {n} {kind} {bad}", flush=True)
    h, w, b, labels, lists, teacher = _inputs(cuda_device, n, 40, 300, dt, 6)
    target = labels if kind == "labels" else (lists, teacher)
    factors = torch.randn(n, device=cuda_device)
    factors[3] = 0
    want = _row_grads(kind, h, w, b, target, factors)[1]
    factors[3] = bad
    got = _row_grads(kind, h, w, b, target, factors)[1]
    assert not bool(torch.isfinite(got[3]).any())
    got[3] = want[3]
    assert torch.equal(got, want)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("n", [9, 200, 5000])
@pytest.mark.parametrize("per_row", [False, True])
def test_rows_that_do_not_count_get_zero(cuda_device, dt, n, per_row):
    """An infinite upstream gradient (an overflowed loss scale) leaves zeros
    in the hidden rows without a target, as F.cross_entropy does."""
    h, w, b, labels, _, _ = _inputs(cuda_device, n, 40, 300, dt, 7)
    labels[::4] = -100
    h.requires_grad_(True)
    loss, _ = linear_cross_entropy(h, w, labels, bias=b, reduction="none" if per_row else "mean")
    up = torch.full_like(loss, math.inf)
    dh = torch.autograd.grad(loss, [h], up)[0]
    assert not bool(dh[::4].any()), dh[::4]


# logits 1.5 + j 2^-23 of these j and j + 1 are one float when both are
# multiplied by log2 e and rounded
def _merged():
    x = (1.5 + np.arange(200) * 2.0 ** -23).astype(np.float32)
    y = x * np.float32(1.4426950408889634)
    j = int(np.nonzero(y[1:] == y[:-1])[0][0])
    assert x[j] != x[j + 1]
    return j


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("n", [9, 200])
@pytest.mark.parametrize("other", [1, 31, 40, 127, 200, 600])
def test_hits_of_neighbouring_floats(cuda_device, dt, n, other):
    """A logit one ulp above the label's is larger, wherever it lies; the
    logits 1.5 + j 2^-23 are exact in every operand type."""
    j = _merged()
    h = torch.tensor([[1.0, 2.0 ** -11]], device=cuda_device).expand(n, 2).contiguous().to(dt)
    w = torch.zeros(700, 2, device=cuda_device)
    w[0, 0] = w[other, 0] = 1.5
    w[0, 1], w[other, 1] = j * 2.0 ** -12, (j + 1) * 2.0 ** -12
    assert torch.equal(w, w.to(dt).float())
    labels = torch.zeros(n, dtype=torch.int64, device=cuda_device)
    labels[1::3] = other
    labels[2::3] = 5
    _, counts = linear_cross_entropy(h, w.to(dt), labels)
    assert counts.tolist() == [len(range(1, n, 3)), n, 0]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("n", [9, 200])
def test_a_strip_of_lowest_logits(cuda_device, dt, n):
    """Classes masked with the type's lowest value, a whole run of them, are
    nothing beside the others."""
    h, w, b, labels, _, _ = _inputs(cuda_device, n, 40, 600, dt, 3)
    b[130:520] = torch.finfo(dt).min
    labels = labels % 100
    loss, counts = linear_cross_entropy(h, w, labels, bias=b, reduction="none")
    z = h.double() @ w.double().t() + b.double()
    ref = torch.nn.functional.cross_entropy(z, labels, reduction="none")
    assert float((loss - ref).abs().max()) <= 1e-4
    assert int(counts[0]) == int((z.argmax(1) == labels).sum())


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("n", [9, 200])
def test_loss_of_confident_rows(cuda_device, dt, n):
    """The loss of a row whose label stands 8 above the rest is
    log(1 + (V - 1) e^-8) to 4e-6 of itself (exp2 and log2 at 2^-21 and their
    sums), whatever the size of the logits; those are exact."""
    classes = 400
    w = torch.zeros(classes, 2, device=cuda_device)
    w[:, 0], w[:, 1] = 1.0, 0.0
    w[7, 1] = 8.0
    for base in (0.0, 30.0, -100.0, 200.0):
        h = torch.tensor([[base, 1.0]], device=cuda_device).expand(n, 2).contiguous()
        labels = torch.full((n,), 7, dtype=torch.int64, device=cuda_device)
        want = math.log1p((classes - 1) * math.exp(-8.0))
        loss, _ = linear_cross_entropy(h.to(dt), w.to(dt), labels)
        assert abs(float(loss) - want) <= 4e-6 * want, (base, float(loss), want)
        index = torch.tensor([[7]], dtype=torch.int32, device=cuda_device).expand(n, 1)
        kd, _ = linear_distill(h.to(dt), w.to(dt), index, torch.zeros(n, 1, device=cuda_device))
        assert abs(float(kd) - want) <= 4e-6 * want, (base, float(kd), want)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("n", [9, 200])
def test_lowest_logits(cuda_device, dt, n):
    """Logits of the type's lowest value: rows with nothing else are uniform,
    and a label there costs what it does in F.cross_entropy."""
    classes, low = 500, torch.finfo(dt).min
    h = torch.zeros(n, 8, device=cuda_device, dtype=dt).requires_grad_(True)
    w = torch.ones(classes, 8, device=cuda_device, dtype=dt).requires_grad_(True)
    b = torch.full((classes,), low, device=cuda_device, dtype=dt).requires_grad_(True)
    labels = torch.arange(n, device=cuda_device) % classes
    loss, _ = linear_cross_entropy(h, w, labels, bias=b, reduction="none")
    assert float((loss - math.log(classes)).abs().max()) <= 1e-5
    db = torch.autograd.grad(loss.sum(), [b])[0].double()
    want = n / classes - torch.bincount(labels, minlength=classes).double()
    assert float((db - want).abs().max()) <= 0.01
    b = b.detach().clone()
    b[250:] = 0
    loss, counts = linear_cross_entropy(h, w, labels, bias=b, reduction="none")
    ref = torch.nn.functional.cross_entropy(h.detach().float() @ w.detach().float().t() + b.float(), labels,
                                            reduction="none")
    assert float((loss / ref - 1).abs().max()) <= 1e-6
    assert counts.tolist() == [0, n, 0]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("n", [9, 200])
def test_infinite_operands(cuda_device, dt, n):
    """An infinity in an operand gives the logits that it gives elsewhere:
    +-inf where it meets a number, NaN where it meets a zero."""
    classes, width = 300, 24
    h, w, b, labels, _, _ = _inputs(cuda_device, n, width, classes, dt, 8)
    h = h.abs() + 0.25
    w[5, 3] = -math.inf  # a masked class
    labels[:] = labels % 100 + 50
    labels[1] = 5
    loss, counts = linear_cross_entropy(h, w, labels, bias=b, reduction="none")
    z = (h.double() @ w.double().t()) + b.double()
    ref = torch.nn.functional.cross_entropy(z, labels, reduction="none")
    assert bool(torch.isinf(ref[1])) and torch.equal(torch.isinf(loss), torch.isinf(ref))
    live = torch.isfinite(ref)
    assert float((loss[live].double() - ref[live]).abs().max()) <= 1e-4
    h[2, 3] = 0.0  # 0 x inf
    h[3, 0] = math.inf
    loss, _ = linear_cross_entropy(h, w, labels, bias=b, reduction="none")
    assert bool(torch.isnan(loss[2])) and bool(torch.isnan(loss[3]))
    keep = [0, 4, 5, 6, 7, 8]
    assert float((loss[keep].double() - ref[keep]).abs().max()) <= 1e-4


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("n", [9, 200])
@pytest.mark.parametrize("kind", ["labels", "lists"])
def test_infinite_weight_and_rows_that_do_not_count(cuda_device, dt, n, kind):
    """A class masked by a weight of -inf has a probability of zero in the
    rows that count and no gradient from the others (whose zeros times an
    infinity are none of it)."""
    h, w, b, labels, lists, teacher = _inputs(cuda_device, n, 24, 300, dt, 8)
    h = h.abs() + 0.25
    w[5, 3] = -math.inf
    labels[:] = labels % 100 + 50
    lists[:] = lists % 100 + 50
    labels[::4] = -100
    lists[::4] = -1
    target = labels if kind == "labels" else (lists, teacher)
    _, _, dw, db = _row_grads(kind, h, w, b, target, torch.ones(n, device=cuda_device))
    assert bool(torch.isfinite(dw).all()) and bool(torch.isfinite(db).all())
    assert not bool(dw[5].any()) and float(db[5]) == 0


@pytest.mark.parametrize("kind", ["labels", "lists"])
def test_no_second_derivative(cuda_device, kind):
    """A second derivative is refused, not left out."""
    h, w, b, labels, lists, teacher = _inputs(cuda_device, 30, 16, 60, torch.float32, 9)
    h.requires_grad_(True)
    w.requires_grad_(kind == "labels")
    if kind == "labels":
        loss, _ = linear_cross_entropy(h, w, labels, bias=b)
    else:
        loss, _ = linear_distill(h, w, lists, teacher, bias=None)
    g = torch.autograd.grad(loss, [h], create_graph=True)[0]
    assert g.requires_grad
    with pytest.raises(RuntimeError, match="second"):
        torch.autograd.grad((g ** 2).sum() + (h ** 2).sum(), [h])


@pytest.mark.parametrize("dt", DTYPES)
def test_rows_far_apart(cuda_device, dt):
    """Rows more than 2^21 elements apart."""
    pitch = (1 << 21) + 24
    wide = torch.randn(6 * pitch, device=cuda_device).to(dt)
    h, w = wide.as_strided((6, 32), (pitch, 1)), wide.as_strided((5, 32), (pitch, 1), 64)
    labels = torch.arange(6, device=cuda_device) % 5
    out = []
    for x, y in ((h, w), (h.contiguous(), w.contiguous())):
        x, y = x.detach().requires_grad_(True), y.detach().requires_grad_(True)
        loss, _ = linear_cross_entropy(x, y, labels)
        out.append((loss.detach(), *torch.autograd.grad(loss, [x, y])))
    for x, y in zip(*out):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("n,width", [(9, 40), (200, 40), (6000, 300)])
def test_repeated_rows(cuda_device, dt, n, width):
    """A row listed twice: losses and the other gradients count both, its own
    hidden gradient is NaN and no other row's is."""
    print(f"case repeated {dt} {n}x{width}", flush=True)
    classes, nodes = 300, 7000
    h, w, b, labels, _, _ = _inputs(cuda_device, n, width, classes, dt, 3, nodes=nodes)
    rows = torch.randperm(nodes, device=cuda_device)[:n]
    labels[::5] = -100
    single = rows.clone()
    rows[5], rows[7] = rows[1], rows[1]
    rows[6] = rows[0]  # one of the two does not count
    out = []
    for r in (rows, None):
        x = h if r is not None else h[rows]
        params = [t.detach().requires_grad_(True) for t in (x, w, b)]
        loss, counts = linear_cross_entropy(params[0], params[1], labels, bias=params[2], rows=r)
        out.append([loss.detach(), counts, *torch.autograd.grad(loss, params)])
    (loss, counts, dh, dw, db), (loss2, counts2, dx, dw2, db2) = out
    assert torch.equal(loss, loss2) and torch.equal(counts, counts2)
    assert torch.equal(dw, dw2) and torch.equal(db, db2)
    nan = torch.isnan(dh).any(1)
    assert sorted(nan.nonzero()[:, 0].tolist()) == sorted({int(rows[1]), int(rows[0])})
    assert bool(torch.isnan(dh[nan]).all())
    want = torch.zeros_like(dh)
    want[rows] = dx
    assert torch.equal(dh[~nan], want[~nan])
    assert single.unique().numel() == n


@pytest.mark.parametrize("dt", DTYPES)
def test_bias_gradient_of_lists(cuda_device, dt):
    """A uniform student of 2,048 classes, each of which 6 of 4,096 rows list
    with a probability of 1/3: the bias gradient 4,096 / 2,048 - 6 / 3 is 0,
    to 2^-21 of the two probabilities' sums of 2 and the fp32 sums' rounding
    (128 terms one after the other, 2^-24 of at most 4 each)."""
    n, classes = 4096, 2048
    h = torch.randn(n, 16, device=cuda_device).to(dt)
    w = torch.zeros(classes, 16, device=cuda_device).to(dt)
    b = torch.zeros(classes, device=cuda_device, dtype=dt).requires_grad_(True)
    index = (torch.arange(n, device=cuda_device)[:, None] * 3 + torch.arange(3, device=cuda_device)) % classes
    loss, _ = linear_distill(h, w, index, torch.zeros(n, 3, device=cuda_device), bias=b, reduction="none")
    db = torch.autograd.grad(loss.sum(), [b])[0].float()
    assert float(db.abs().max()) <= 4 * 2.0 ** -21 + 128 * 4 * 2.0 ** -24


@pytest.mark.parametrize("n", [9, 200])
@pytest.mark.parametrize("dt", DTYPES)
def test_bias_gradient_of_a_spoiled_list(cuda_device, dt, n):
    """A NaN among a list's logits is seen in its classes' bias gradients."""
    h, w, b, _, lists, teacher = _inputs(cuda_device, n, 24, 2000, dt, 8)
    teacher[3, 1] = math.nan
    b.requires_grad_(True)
    loss, _ = linear_distill(h, w, lists, teacher, bias=b)
    db = torch.autograd.grad(loss, [b])[0]
    assert bool(torch.isnan(loss)) and bool(torch.isnan(db[lists[3].long()]).all())
    other = torch.ones(2000, dtype=torch.bool, device=cuda_device)
    other[lists[3].long()] = False
    assert bool(torch.isfinite(db[other]).all())


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("n", [9, 200])
@pytest.mark.parametrize("kind", ["labels", "lists"])
def test_saved_statistics(cuda_device, dt, n, kind):
    """lse as the header has it, within the buffer it asks for, and a second
    backward of the same forward has the same bits."""
    h, w, b, labels, lists, teacher = _inputs(cuda_device, n, 40, 300, dt, 5)
    labels[::4] = -100
    lists[::4] = -1
    t = 1.0 if kind == "labels" else 2.0
    call = (ops.HeadCall(h, w, b, None, labels) if kind == "labels"
            else ops.HeadCall(h, w, b, None, None, lists, teacher, t))
    loss, counts, saved = ops.head_fwd(call, True)
    assert saved.numel() == n * (2 if kind == "labels" else 16)
    z = (h.double() @ w.double().t() + b.double()) / t * math.log2(math.e)
    live = torch.ones(n, dtype=torch.bool, device=cuda_device)
    live[::4] = False
    assert bool((saved[:n][~live] == math.inf).all())
    want = torch.logsumexp(z * math.log(2), 1) / math.log(2)
    # 48 2^-23 of the summed magnitudes (20 at most), and lse's own rounding
    assert float((saved[:n][live].double() - want[live]).abs().max()) <= 2e-4
    up = torch.randn(n, device=cuda_device)
    first = ops.head_bwd(call, saved, counts, up)
    for x, y in zip(first, ops.head_bwd(call, saved, counts, up)):
        assert torch.equal(x, y)
