"""The fused classifier losses (csrc/head.hip) on whole numbers whose sums are
exact in f32: what the kernels compute from operands split into planes is then
the number itself, and a plane or a product of two planes left out is seen.

A 21-bit number takes three bf16 planes, a 12-bit one two; 200 rows go through
the products, 9 through the kernels of few rows."""
import pytest
import torch

from graph_rws_amd.layers import linear_cross_entropy, linear_distill

pytestmark = pytest.mark.gpu


def _ints(gen, shape, bits):
    return torch.randint(0, 1 << bits, shape, generator=gen, device=gen.device).float()


@pytest.mark.parametrize("n", [9, 200])
@pytest.mark.parametrize("hbits,wbits", [(21, 3), (12, 12), (3, 21)])
def test_f32_logits(cuda_device, n, hbits, wbits):
    """A row's hidden has one entry, so a logit is one product; the largest
    logit stands so far above that the loss is its distance from the label's
    (or, for rows whose two largest are near, off by log 2 and less)."""
    gen = torch.Generator(device=cuda_device)
    gen.manual_seed(n + hbits)
    classes, width = 300, 16
    h = torch.zeros(n, width, device=cuda_device)
    at = torch.arange(n, device=cuda_device)
    h[at, at % width] = _ints(gen, (n,), hbits) + 1
    w = _ints(gen, (classes, width), wbits)
    labels = torch.randint(0, classes, (n,), generator=gen, device=cuda_device)
    loss, _ = linear_cross_entropy(h, w, labels, reduction="none")
    z = h.double() @ w.double().t()
    assert float(z.max()) <= 1 << 24
    top = z.topk(2, dim=1).values
    ref = torch.nn.functional.cross_entropy(z, labels, reduction="none")
    clear = top[:, 0] - top[:, 1] >= 100
    if wbits > 3:
        assert int(clear.sum()) > n // 2
    assert torch.equal(loss[clear].double(), ref[clear])
    assert float((loss.double() - ref).abs().max()) <= 0.5  # an ulp of 2^22


def _one_class(dev, classes, bias_dt):
    """A bias that gives class 0 all of the probability: exactly one, as its
    logit is 0 (times log2 e it is not rounded)."""
    b = torch.full((classes,), -1000.0, device=dev, dtype=bias_dt)
    b[0] = 0
    return b


@pytest.mark.parametrize("n", [9, 200])
@pytest.mark.parametrize("fbits,wbits", [(21, 2), (11, 12), (2, 21)])
def test_f32_hidden_gradient(cuda_device, n, fbits, wbits):
    """G is +f at class 0 and -f at the label, f the row's factor (a power of
    two the largest), so d_hidden = f (w_0 - w_label)."""
    gen = torch.Generator(device=cuda_device)
    gen.manual_seed(n + fbits)
    classes, width = 300, 24
    w = _ints(gen, (classes, width), wbits)
    h = torch.zeros(n, width, device=cuda_device, requires_grad=True)
    labels = torch.randint(1, classes, (n,), generator=gen, device=cuda_device)
    f = _ints(gen, (n,), fbits)
    f[0] = 1 << fbits
    loss, _ = linear_cross_entropy(h, w, labels, bias=_one_class(cuda_device, classes, torch.float32),
                                   reduction="none")
    dh = torch.autograd.grad(loss, [h], f)[0]
    assert torch.equal(dh.double(), f.double()[:, None] * (w[:1].double() - w[labels].double()))


@pytest.mark.parametrize("n", [9, 200])
@pytest.mark.parametrize("fbits,hbits", [(19, 2), (10, 11), (2, 19)])
def test_f32_weight_gradient(cuda_device, n, fbits, hbits):
    """Six rows count: d_weight is -f h at their labels, the sum at class 0."""
    gen = torch.Generator(device=cuda_device)
    gen.manual_seed(n + fbits)
    classes, width = 300, 24
    w = torch.zeros(classes, width, device=cuda_device, requires_grad=True)
    h = _ints(gen, (n, width), hbits)
    labels = torch.full((n,), -100, device=cuda_device)
    live = torch.randperm(n, generator=gen, device=cuda_device)[:6]
    labels[live] = torch.arange(50, 56, device=cuda_device)
    f = torch.zeros(n, device=cuda_device)
    f[live] = _ints(gen, (6,), fbits)
    f[live[0]] = 1 << fbits
    loss, _ = linear_cross_entropy(h, w, labels, bias=_one_class(cuda_device, classes, torch.float32),
                                   reduction="none")
    dw = torch.autograd.grad(loss, [w], f)[0]
    g = f[live].double()[:, None] * h[live].double()
    want = torch.zeros(classes, width, dtype=torch.float64, device=cuda_device)
    want[50:56] = -g
    want[0] = g.sum(0)
    assert torch.equal(dw.double(), want)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [9, 200])
def test_second_plane_in_the_weight_gradient(cuda_device, dt, n):
    """Up to 1,024 classes 16-bit G keeps what its rounding left over: rows
    whose factors f and -(f - 3) cancel leave 3 h at class 0, for an odd f of
    15 bits."""
    classes, width = 1000, 24
    h = torch.ones(n, width, device=cuda_device, dtype=dt)
    w = torch.zeros(classes, width, device=cuda_device, dtype=dt, requires_grad=True)
    bias = _one_class(cuda_device, classes, dt)
    for f in (32767, 21847, 17001, 29123):
        labels = torch.full((n,), -100, device=cuda_device)
        labels[2], labels[5], labels[7] = 40, 41, 0
        factors = torch.zeros(n, device=cuda_device)
        factors[2], factors[5], factors[7] = f, 3 - f, 1 << 15  # the last: the largest, with no gradient at all
        loss, _ = linear_cross_entropy(h, w, labels, bias=bias, reduction="none")
        dw = torch.autograd.grad(loss, [w], factors)[0].float()
        assert bool((dw[0] == 3).all()), (f, float(dw[0, 0]))


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [9, 200])
def test_second_plane_in_the_hidden_gradient(cuda_device, dt, n):
    """Teachers with 1/4 and 3/4 of two classes, a student with all on a
    third: G is 4 g, -g and -3 g, whose sum over a weight of ones is zero (to
    the probabilities' 2^-22 of 2^15); rounded to one plane it is not."""
    classes, width = 1000, 24
    w = torch.ones(classes, width, device=cuda_device, dtype=dt)
    h = torch.zeros(n, width, device=cuda_device, dtype=dt, requires_grad=True)
    index = torch.tensor([[17, 400]], device=cuda_device).expand(n, 2)
    teacher = torch.tensor([[0.0, 3.0]], device=cuda_device).log().clamp(min=0).expand(n, 2).contiguous()
    factors = 4.0 * torch.arange(5001, 5001 + n, device=cuda_device)
    factors[1] = 1 << 15
    loss, _ = linear_distill(h, w, index, teacher, bias=_one_class(cuda_device, classes, dt), reduction="none")
    dh = torch.autograd.grad(loss, [h], factors)[0].float()
    assert float(dh.abs().max()) <= 2.0 ** -6
