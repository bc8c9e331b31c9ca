"""Fused classifier losses (csrc/head.hip: linear_cross_entropy,
linear_distill) against the definitions in 64 bits.

Tolerances are bounds, formed per element from the reference.  With u a
rounding of the operands' type (2^-23 for f32, 2^-11 f16, 2^-8 bf16):
  * a logit is an fp32 sum of D products, each step off by 2^-23 of the sum
    of magnitudes at most (f32 operands, split in three, leave out another
    2^-21): dz = (D + 8) 2^-23 sum |h||w| + 2^-22 |z|;
  * exp2 and log2 are good to 2^-21, so a loss is off by 2 max dz + 2^-19
    (plus 2^-21 of its largest term), a probability by
    e = 2 max dz / T + 2^-19 of itself;
  * dz is formed in fp32 and rounded once to the operands' type (f16: with
    2^15 in front, so 2^-40 at least), hence off by u |g| + e p; sums add
    their length times 2^-23, and the result is rounded once."""
import math

import pytest
import torch

from graph_rws_amd.core import ops
from graph_rws_amd.layers import linear_cross_entropy, linear_distill

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
U = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 1e-30, torch.float16: 2.0 ** -24, torch.bfloat16: 1e-30}


def _inputs(dev, n, width, classes, dt, seed, nodes=None, bias=False, scale=1.0):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    h = (torch.randn(nodes or n, width, generator=g, device=dev) * scale).to(dt)
    w = (torch.randn(classes, width, generator=g, device=dev) * 2 / math.sqrt(width)).to(dt)
    b = torch.randn(classes, generator=g, device=dev).to(dt) if bias else None
    labels = torch.randint(0, classes, (n,), generator=g, device=dev)
    return h, w, b, labels


class _Ref:
    """Loss, gradients and their bounds in 64 bits.  target [n, classes]:
    the rows' target distribution, live [n]."""

    def __init__(self, h, w, b, rows, target, live, temperature=1.0):
        self.dt, self.b = h.dtype, b
        t = temperature
        self.hid = h.shape
        self.rows = rows if rows is not None else torch.arange(target.shape[0], device=h.device)
        x = h.double()[self.rows]
        x[~live] = 0
        wd = w.double()
        D, V, n = w.shape[1], w.shape[0], target.shape[0]
        z = x @ wd.t()
        mag = x.abs() @ wd.abs().t()
        if b is not None:
            z = z + b.double()
            mag = mag + b.double().abs().nan_to_num(posinf=0.0)
        zz = z.nan_to_num(neginf=0.0)
        dz = ((D + 8) * 2.0 ** -23 * mag + 2.0 ** -22 * zz.abs()).amax(1, keepdim=True)
        logp = torch.log_softmax(z / t, 1)
        p = logp.exp()
        part = torch.where(target > 0, target * (target.clamp(min=1e-300).log() - logp), 0.0)
        self.row = torch.where(live, part.sum(1) * t * t, 0.0)
        big = torch.where(target > 0, logp.abs() + target.clamp(min=1e-300).log().abs(), 0.0).amax(1)
        self.row_tol = t * t * (2 * dz[:, 0] / t + 2.0 ** -19 + 2.0 ** -20 * (big + zz.abs().amax(1) / t))
        self.count = int(live.sum())
        g = (p - target) * t
        e = 2 * dz / t + 2.0 ** -19
        u = U[self.dt]
        dg = u * g.abs() + t * (e * p + (2.0 ** -20) * target) + (2.0 ** -40 * t if self.dt == torch.float16 else 0.0)
        dead = ~live
        g[dead], dg[dead], p[dead] = 0, 0, 0
        self.g, self.dg, self.x, self.w = g, dg, x, wd

    def check_loss(self, loss, row_loss=None):
        if row_loss is not None:
            d = (row_loss.double() - self.row).abs()
            assert bool((d <= self.row_tol).all()), f"row loss off by {float((d - self.row_tol).max())} over its bound"
        if loss is not None:
            ref, tol = float(self.row.sum()) / self.count, float(self.row_tol.mean()) + 1e-7 * float(self.row.mean())
            assert abs(float(loss) - ref) <= tol * 2, (float(loss), ref, tol)

    def check_grads(self, dh, dw, db, scale):
        """scale: a factor, or [n] factors."""
        s = scale if isinstance(scale, torch.Tensor) else torch.full((self.g.shape[0],), float(scale),
                                                                    dtype=torch.float64, device=self.g.device)
        g, dg = self.g * s[:, None], self.dg * s.abs()[:, None]
        if isinstance(scale, torch.Tensor):  # rows are scaled to the largest before the rounding
            dg = dg + s.abs().max() * (2.0 ** -40 if self.dt == torch.float16 else 0.0)
        u, tiny = U[self.dt], TINY[self.dt]
        n, V = g.shape

        def close(got, ref, tol, what):
            d = (got.double() - ref).abs()
            tol = tol + u * (ref.abs() + tol) + tiny
            worst = float((d / tol).max())
            assert worst <= 1.0, f"{what}: {worst} of the bound"

        if dh is not None:
            ref = torch.zeros(self.hid, dtype=torch.float64, device=g.device)
            tol = torch.zeros_like(ref)
            ref[self.rows] = g @ self.w
            tol[self.rows] = dg @ self.w.abs() + (V + 8) * 2.0 ** -23 * (g.abs() @ self.w.abs())
            close(dh, ref, tol, "d_hidden")
        if dw is not None:
            a = self.x.abs()
            close(dw, g.t() @ self.x, dg.t() @ a + (n + 8) * 2.0 ** -23 * (g.abs().t() @ a), "d_weight")
        if db is not None:
            close(db, g.sum(0), dg.sum(0) + (n + 8) * 2.0 ** -23 * g.abs().sum(0), "d_bias")


def _onehot(labels, classes):
    live = labels != -100
    t = torch.zeros(labels.numel(), classes, dtype=torch.float64, device=labels.device)
    t[live.nonzero()[:, 0], labels[live]] = 1.0
    return t, live


def _teacher(index, logits, classes, temperature):
    n, k = index.shape
    has = (index >= 0) & (logits != -math.inf)
    live = has.any(1)
    q = torch.softmax((logits.double() / temperature).masked_fill(~has, -math.inf), 1).nan_to_num(0.0)
    t = torch.zeros(n, classes, dtype=torch.float64, device=index.device)
    t.scatter_add_(1, index.long().clamp(min=0), torch.where(has, q, 0.0))
    return t, live


def _hits(ref_z, labels, live):
    return int(((ref_z.argmax(1) == labels) & live).sum())


SHAPES = [(1, 16, 47), (1, 8, 1), (2, 1, 2), (5, 13, 257), (17, 64, 128), (64, 250, 129), (130, 96, 300),
          (129, 256, 172), (300, 1433, 7), (257, 40, 1003), (1024, 256, 172), (4099, 72, 4099)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("bias", [False, True])
def test_cross_entropy(cuda_device, dt, shape, bias):
    print(f"case ce {dt} {shape} bias={bias}", flush=True)
    n, width, classes = shape
    h, w, b, labels = _inputs(cuda_device, n, width, classes, dt, n + classes, bias=bias)
    if n > 2:
        labels[::5] = -100
    params = [t.requires_grad_(True) for t in (h, w, b) if t is not None]
    loss, counts = linear_cross_entropy(h, w, labels, bias=b)
    assert loss.dtype == torch.float32 and loss.dim() == 0
    grads = torch.autograd.grad(loss, params, torch.tensor(256.0, device=cuda_device))
    ref = _Ref(h.detach(), w.detach(), b.detach() if bias else None, None, *_onehot(labels, classes))
    assert counts.tolist()[1:] == [ref.count, 0]
    ref.check_loss(loss)
    assert all(g.dtype == dt for g in grads)
    ref.check_grads(grads[0], grads[1], grads[2] if bias else None, 256.0 / ref.count)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("shape", [(1, 16, 47, 5), (3, 9, 12, 12), (33, 250, 1003, 64), (130, 64, 300, 1),
                                   (1024, 256, 47, 5), (515, 520, 2049, 100), (4099, 72, 4099, 7)])
@pytest.mark.parametrize("temperature", [1.0, 2.5])
def test_distill(cuda_device, dt, shape, temperature):
    print(f"case distill {dt} {shape} T={temperature}", flush=True)
    n, width, classes, k = shape
    h, w, b, _ = _inputs(cuda_device, n, width, classes, dt, n + k, bias=n % 2 == 1)
    teacher = torch.randn(n, classes, device=cuda_device) * 3
    values, index = ops.top_logits(teacher, k)
    if n > 2:  # shorter lists, an empty one, a listed -inf
        index[::3, k // 2:] = -1
        index[1] = -1
        values[2, 0] = -math.inf
    params = [t.requires_grad_(True) for t in (h, w, b) if t is not None]
    loss, counts = linear_distill(h, w, index, values, bias=b, temperature=temperature)
    grads = torch.autograd.grad(loss, params, torch.tensor(256.0, device=cuda_device))
    ref = _Ref(h.detach(), w.detach(), b.detach() if b is not None else None, None,
               *_teacher(index, values, classes, temperature), temperature)
    assert counts.tolist() == [ref.count, 0]
    ref.check_loss(loss)
    ref.check_grads(grads[0], grads[1], grads[2] if b is not None else None, 256.0 / ref.count)


@pytest.mark.parametrize("dt", DTYPES)
def test_rows_and_row_losses(cuda_device, dt):
    """reduction "none" over chosen rows, each row's gradient with its own
    factor; rows that are not chosen get zero."""
    n, nodes, width, classes = 301, 700, 136, 517
    h, w, b, labels = _inputs(cuda_device, n, width, classes, dt, 3, nodes=nodes, bias=True)
    rows = torch.randperm(nodes, device=cuda_device)[:n]
    labels[7:40] = -100
    h.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)
    loss, counts = linear_cross_entropy(h, w, labels, bias=b, rows=rows, reduction="none")
    assert loss.shape == (n,)
    factors = torch.randn(n, device=cuda_device) * 10
    factors[5] = 0
    grads = torch.autograd.grad(loss, [h, w, b], factors)
    ref = _Ref(h.detach(), w.detach(), b.detach(), rows, *_onehot(labels, classes))
    ref.check_loss(None, loss)
    assert bool((loss[7:40] == 0).all())
    ref.check_grads(*grads, factors.double())
    other = torch.ones(nodes, dtype=torch.bool, device=cuda_device)
    other[rows] = False
    assert not bool(grads[0][other].any())


def test_hits_and_ties(cuda_device):
    """A hit is a label that is the first of the largest logits: equal rows
    of the weight give equal logits, in one strip of classes and across."""
    n, width, classes = 64, 32, 700
    for dt in DTYPES:
        h, w, _, labels = _inputs(cuda_device, n, width, classes, dt, 11)
        w[5] = w[600] = w[9]
        h[:] = w[9] * 8
        labels[:] = 9
        labels[0], labels[1], labels[2] = 5, 600, -100
        _, counts = linear_cross_entropy(h, w, labels)
        assert counts.tolist() == [1, n - 1, 0]
        w[5] = 0
        _, counts = linear_cross_entropy(h, w, labels)
        assert counts.tolist() == [n - 3, n - 1, 0]


@pytest.mark.parametrize("dt", DTYPES)
def test_hits_match_argmax(cuda_device, dt):
    h, w, _, labels = _inputs(cuda_device, 500, 64, 3001, dt, 5)
    z = h.double() @ w.double().t()
    labels[::2] = z.argmax(1)[::2]
    top2 = z.topk(2, dim=1).values
    clear = top2[:, 0] - top2[:, 1] > 1e-3
    labels[~clear] = -100
    _, counts = linear_cross_entropy(h, w, labels)
    assert int(counts[0]) == _hits(z, labels, clear)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("n", [1, 7, 16, 17, 32, 33, 64, 65, 100, 128])
@pytest.mark.parametrize("width", [24, 131, 512])
def test_few_rows(cuda_device, dt, n, width):
    """Row counts around the small kernel's tiles, aligned widths and not,
    with and without every row counting, labels and lists."""
    print(f"case few {dt} {n}x{width}", flush=True)
    classes = 1533
    h, w, b, labels = _inputs(cuda_device, n, width, classes, dt, n + width, nodes=n + 3, bias=True)
    rows = torch.randperm(n + 3, device=cuda_device)[:n]
    labels[1::6] = -100
    params = [x.requires_grad_(True) for x in (h, w, b)]
    loss, counts = linear_cross_entropy(h, w, labels, bias=b, rows=rows, reduction="none")
    factors = torch.rand(n, device=cuda_device) + 0.5
    grads = torch.autograd.grad(loss, params, factors)
    ref = _Ref(h.detach(), w.detach(), b.detach(), rows, *_onehot(labels, classes))
    assert counts.tolist()[1:] == [ref.count, 0]
    ref.check_loss(None, loss)
    ref.check_grads(*grads, factors.double())
    values, index = ops.top_logits(torch.randn(n, classes, device=cuda_device) * 3, 6)
    index[1::6] = -1
    loss, counts = linear_distill(h, w, index, values, bias=b, rows=rows, temperature=2.0)
    grads = torch.autograd.grad(loss, params)
    ref = _Ref(h.detach(), w.detach(), b.detach(), rows, *_teacher(index, values, classes, 2.0), 2.0)
    assert counts.tolist() == [ref.count, 0]
    ref.check_loss(loss)
    ref.check_grads(*grads, 1.0 / ref.count)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_pieces(cuda_device, dt):
    """More rows than one piece of the gradient's scratch takes at all the
    classes: several pieces, with the hidden gradient added up over them."""
    n, width, classes = 40000, 16, 4500
    h, w, b, labels = _inputs(cuda_device, n, width, classes, dt, 21, bias=True)
    labels[::7] = -100
    h.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)
    loss, _ = linear_cross_entropy(h, w, labels, bias=b)
    grads = torch.autograd.grad(loss, [h, w, b], torch.tensor(4096.0, device=cuda_device))
    ref = _Ref(h.detach(), w.detach(), b.detach(), None, *_onehot(labels, classes))
    ref.check_loss(loss)
    ref.check_grads(*grads, 4096.0 / ref.count)


@pytest.mark.parametrize("dt", DTYPES)
def test_rows_that_do_not_count_reach_nothing(cuda_device, dt):
    """NaN and infinities in rows without a target stay out of the loss and
    of every gradient."""
    n, width, classes = 200, 64, 333
    h, w, _, labels = _inputs(cuda_device, n, width, classes, dt, 2)
    labels[::4] = -100
    clean = h.clone()
    h[0], h[4], h[8] = math.nan, math.inf, -math.inf
    out = []
    for x in (clean, h):
        x, wt = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        loss, _ = linear_cross_entropy(x, wt, labels)
        out.append((loss.detach(), *torch.autograd.grad(loss, [x, wt])))
    for a, b in zip(*out):
        assert torch.equal(a, b) and bool(torch.isfinite(a).all())
    assert not bool(out[1][1][::4].any())


def test_nothing_counts(cuda_device):
    for dt in DTYPES:
        h, w, _, labels = _inputs(cuda_device, 6, 16, 40, dt, 1)
        h.requires_grad_(True), w.requires_grad_(True)
        labels[:] = -100
        loss, counts = linear_cross_entropy(h, w, labels)
        assert bool(torch.isnan(loss)) and counts.tolist() == [0, 0, 0]
        assert not any(bool(g.any()) for g in torch.autograd.grad(loss, [h, w]))
        index = torch.full((6, 3), -1, dtype=torch.int32, device=cuda_device)
        loss, counts = linear_distill(h, w, index, torch.zeros(6, 3, device=cuda_device))
        assert bool(torch.isnan(loss)) and counts.tolist() == [0, 0]
        assert not any(bool(g.any()) for g in torch.autograd.grad(loss, [h, w]))
        # no rows at all
        loss, counts = linear_cross_entropy(h, w, labels[:0])
        assert bool(torch.isnan(loss)) and counts.tolist() == [0, 0, 0]
        assert not any(bool(g.any()) for g in torch.autograd.grad(loss, [h, w]))
        loss, _ = linear_cross_entropy(h, w, labels[:0], reduction="none")
        assert loss.shape == (0,)


def test_bad_targets(cuda_device):
    """A label, class index or row id out of range: NaN and the flag, as
    cross_entropy_rows has it; the row reaches no gradient."""
    h, w, _, labels = _inputs(cuda_device, 10, 24, 50, torch.float32, 1)
    h.requires_grad_(True)
    for bad in (50, -1, -101, 2 ** 40):
        lab = labels.clone()
        lab[3] = bad
        loss, counts = linear_cross_entropy(h, w, lab)
        assert bool(torch.isnan(loss)) and counts.tolist()[1:] == [9, 1]
        assert not bool(torch.autograd.grad(loss, [h])[0][3].any())
        rl, _ = linear_cross_entropy(h, w, lab, reduction="none")
        assert bool(torch.isnan(rl[3])) and int(torch.isnan(rl).sum()) == 1
    rows = torch.arange(10, device=cuda_device)
    rows[2] = 10
    loss, counts = linear_cross_entropy(h, w, labels, rows=rows)
    assert bool(torch.isnan(loss)) and counts.tolist()[1:] == [9, 1]
    for bad in (50, -2, 2 ** 33):
        index = torch.randint(0, 50, (10, 4), device=cuda_device)
        index[6, 2] = bad
        loss, counts = linear_distill(h, w, index, torch.randn(10, 4, device=cuda_device))
        assert bool(torch.isnan(loss)) and counts.tolist() == [9, 1]


def test_masked_classes(cuda_device):
    """A bias of -inf takes a class out: probability and gradient zero; a
    target there costs infinity; a teacher's probability of zero there, nothing."""
    n, width, classes = 20, 32, 300
    h, w, b, labels = _inputs(cuda_device, n, width, classes, torch.float32, 4, bias=True)
    b[128:256] = -math.inf  # a whole strip of classes
    b[3] = torch.finfo(torch.float32).min
    labels = labels % 100 + 4
    h.requires_grad_(True), w.requires_grad_(True)
    loss, _ = linear_cross_entropy(h, w, labels, bias=b)
    dh, dw = torch.autograd.grad(loss, [h, w])
    keep = torch.ones(classes, dtype=torch.bool, device=cuda_device)
    keep[128:256] = False
    keep[3] = False
    z = (h.detach().double() @ w.detach().double().t() + b.double()).masked_fill(~keep, -math.inf)
    assert abs(float(loss) - float(torch.nn.functional.cross_entropy(z, labels))) <= 1e-5
    assert not bool(dw[~keep].any()) and bool(torch.isfinite(dh).all())
    labels[0] = 130
    rl, _ = linear_cross_entropy(h, w, labels, bias=b, reduction="none")
    assert float(rl[0]) == math.inf and bool(torch.isfinite(rl[1:]).all())
    index = torch.tensor([[5, 130]], dtype=torch.int32, device=cuda_device).expand(n, 2)
    t = torch.tensor([[1.0, -math.inf]], device=cuda_device).expand(n, 2)
    rl, _ = linear_distill(h, w, index, t, bias=b, reduction="none")
    assert bool(torch.isfinite(rl).all())


def test_repeated_teacher_class(cuda_device):
    """A class listed twice counts with both probabilities."""
    h, w, _, _ = _inputs(cuda_device, 50, 40, 90, torch.float32, 9)
    index = torch.randint(0, 90, (50, 6), device=cuda_device, dtype=torch.int32)
    index[:, 3] = index[:, 0]
    index[:, 5] = index[:, 0]
    t = torch.randn(50, 6, device=cuda_device)
    t[::2, 0] = -math.inf
    h.requires_grad_(True), w.requires_grad_(True)
    loss, _ = linear_distill(h, w, index, t, temperature=2.0)
    grads = torch.autograd.grad(loss, [h, w])
    has = t != -math.inf
    q = torch.softmax(t.double().masked_fill(~has, -math.inf) / 2, 1)
    hd, wd = h.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
    logp = torch.log_softmax(hd @ wd.t() / 2, 1).gather(1, index.long())
    ref = (torch.where(has, q * (q.clamp(min=1e-300).log() - logp), 0.0)).sum() * 4 / 50
    want = torch.autograd.grad(ref, [hd, wd])
    assert abs(float(loss) - float(ref)) <= 1e-5 * float(ref)
    for a, r in zip(grads, want):
        assert float((a.double() - r).abs().max()) <= 1e-5 * float(r.abs().max())


@pytest.mark.parametrize("dt", DTYPES)
def test_strides(cuda_device, dt):
    """Row pitches, misaligned starts and transposed operands give what
    contiguous copies give, bit for bit."""
    n, width, classes = 70, 56, 333
    wide = torch.randn(n, 3 * width + 5, device=cuda_device).to(dt)
    table = torch.randn(classes, width + 8, device=cuda_device).to(dt)
    labels = torch.randint(0, classes, (2 * n,), device=cuda_device)[::2]
    hs = [wide[:, 3:3 + width], wide[:, 8:8 + width], wide.t()[:n, :width] if n <= width else wide[:, :width],
          torch.randn(width, n, device=cuda_device).to(dt).t(), wide[:1, :width].expand(n, width)]
    ws = [table[:, :width], table[:, 1:1 + width], torch.randn(width, classes, device=cuda_device).to(dt).t()]
    for h in hs:
        for w in ws:
            out = []
            for a, b in ((h, w), (h.contiguous(), w.contiguous())):
                a, b = a.detach().requires_grad_(True), b.detach().requires_grad_(True)
                loss, _ = linear_cross_entropy(a, b, labels)
                out.append((loss.detach(), *torch.autograd.grad(loss, [a, b])))
            for x, y in zip(*out):
                assert torch.equal(x, y)


def test_differences(cuda_device):
    """Gradients against central differences of the loss along random
    directions: the step 2^-6 leaves its square times a third derivative (at
    most 1 for unit directions here), the f32 losses 2^-22 / 2^-6 each."""
    n, width, classes = 40, 24, 120
    h, w, b, labels = _inputs(cuda_device, n, width, classes, torch.float32, 8, bias=True)
    index = torch.stack([torch.randperm(classes, device=cuda_device)[:5] for _ in range(n)])
    t = torch.randn(n, 5, device=cuda_device)
    calls = [lambda *p: linear_cross_entropy(p[0], p[1], labels, bias=p[2])[0],
             lambda *p: linear_distill(p[0], p[1], index, t, bias=p[2], temperature=2.0)[0]]
    eps = 2.0 ** -6
    for call in calls:
        params = [x.detach().requires_grad_(True) for x in (h, w, b)]
        grads = torch.autograd.grad(call(*params), params)
        for which in range(3):
            d = torch.randn_like(params[which])
            d /= d.norm()
            up = [p.detach() + (eps * d if i == which else 0) for i, p in enumerate(params)]
            down = [p.detach() - (eps * d if i == which else 0) for i, p in enumerate(params)]
            slope = (float(call(*up)) - float(call(*down))) / (2 * eps)
            assert abs(slope - float((grads[which] * d).sum())) <= eps ** 2 + 8 * 2.0 ** -22 / eps


def test_same_bits_streams_and_capture(cuda_device):
    """Two calls, a call on another stream and replays of a captured call
    give the same bits."""
    h, w, b, labels = _inputs(cuda_device, 700, 200, 1500, torch.bfloat16, 6, bias=True)
    values, index = ops.top_logits(torch.randn(700, 1500, device=cuda_device), 9)
    params = [x.requires_grad_(True) for x in (h, w, b)]

    def both():
        a, _ = linear_cross_entropy(h, w, labels, bias=b)
        c, _ = linear_distill(h, w, index, values, bias=b, temperature=2.0)
        return [a.detach(), c.detach(), *torch.autograd.grad(a + c, params)]

    first = [x.clone() for x in both()]
    for x, y in zip(first, both()):
        assert torch.equal(x, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both()
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(first, other):
        assert torch.equal(x, y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(first, held):
            assert torch.equal(x, y)
        for x, y in zip(first, both()):
            assert torch.equal(x, y)


def test_autocast(cuda_device):
    """Under autocast f32 parameters are taken in the autocast dtype, and
    their gradients come back in f32."""
    h, w, b, labels = _inputs(cuda_device, 64, 48, 200, torch.float32, 12, bias=True)
    params = [x.requires_grad_(True) for x in (h, w, b)]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss, _ = linear_cross_entropy(h, w, labels, bias=b)
    grads = torch.autograd.grad(loss, params)
    low = [x.detach().bfloat16().requires_grad_(True) for x in params]
    want, _ = linear_cross_entropy(low[0], low[1], labels, bias=low[2])
    assert torch.equal(loss, want)
    for a, r in zip(grads, torch.autograd.grad(want, low)):
        assert a.dtype == torch.float32 and torch.equal(a, r.float())


def test_loss_may_change_in_place(cuda_device):
    """Dividing the loss in place (gradient accumulation) leaves what the
    backward needs alone."""
    h, w, _, labels = _inputs(cuda_device, 30, 16, 60, torch.float32, 12)
    h.requires_grad_(True)
    loss, _ = linear_cross_entropy(h, w, labels)
    want = torch.autograd.grad(loss, [h])[0]
    loss, _ = linear_cross_entropy(h, w, labels)
    loss /= 4
    assert float((torch.autograd.grad(loss, [h])[0] - want / 4).abs().max()) <= 1e-7


def test_skips_what_needs_no_gradient(cuda_device):
    h, w, b, labels = _inputs(cuda_device, 90, 48, 200, torch.bfloat16, 12, bias=True)
    every = [x.requires_grad_(True) for x in (h, w, b)]
    loss, _ = linear_cross_entropy(h, w, labels, bias=b)
    want = torch.autograd.grad(loss, every)
    for i in range(3):
        parts = [x.detach().requires_grad_(j == i) for j, x in enumerate(every)]
        loss, _ = linear_cross_entropy(parts[0], parts[1], labels, bias=parts[2])
        assert torch.equal(torch.autograd.grad(loss, [parts[i]])[0], want[i])


def test_refusals(cuda_device):
    h, w, b, labels = _inputs(cuda_device, 8, 16, 30, torch.float32, 1, bias=True)
    index = torch.zeros(8, 2, dtype=torch.int32, device=cuda_device)
    t = torch.zeros(8, 2, device=cuda_device)
    for call, err in [
        (lambda: linear_cross_entropy(h.cpu(), w, labels), RuntimeError),
        (lambda: linear_cross_entropy(h, w.cpu(), labels), RuntimeError),
        (lambda: linear_cross_entropy(h, w, labels.cpu()), RuntimeError),
        (lambda: linear_cross_entropy(h, w[:, :8], labels), ValueError),
        (lambda: linear_cross_entropy(h[0], w, labels), ValueError),
        (lambda: linear_cross_entropy(h, w.half(), labels), TypeError),
        (lambda: linear_cross_entropy(h.double(), w.double(), labels), TypeError),
        (lambda: linear_cross_entropy(h, w, labels, bias=b[:-1]), ValueError),
        (lambda: linear_cross_entropy(h, w, labels, bias=b.half()), TypeError),
        (lambda: linear_cross_entropy(h, w, labels.int()), ValueError),
        (lambda: linear_cross_entropy(h, w, labels[:, None]), ValueError),
        (lambda: linear_cross_entropy(h[:4], w, labels), ValueError),
        (lambda: linear_cross_entropy(h, w, labels, rows=labels[:3]), ValueError),
        (lambda: linear_cross_entropy(h, w, labels, rows=labels.int()), ValueError),
        (lambda: linear_cross_entropy(h, w, labels, reduction="sum"), ValueError),
        (lambda: linear_distill(h, w, index.float(), t), ValueError),
        (lambda: linear_distill(h, w, index, t[:, :1]), ValueError),
        (lambda: linear_distill(h, w, index, index), ValueError),
        (lambda: linear_distill(h, w, index[:, :0], t[:, :0]), ValueError),
        (lambda: linear_distill(h, w, index, t, temperature=0.0), ValueError),
        (lambda: linear_distill(h, w, index, t, temperature=math.nan), ValueError),
        (lambda: linear_distill(h, w, None, None), ValueError),
    ]:
        with pytest.raises(err):
            call()
