"""layers.linear_log_probs (csrc/head.hip) against the definitions in 64 bits.

Bounds, per element.  A logit is an fp32 sum of D products, each step off by
2^-23 of the sum of magnitudes (f32 operands, split in three, leave out less):
dz = (D + 8) 2^-23 sum |h||w| + 2^-22 |z|, the largest of a row.  x = (m - z)
/ T is then off by 2 dz / T, and as csrc/logp.hip's by 2^-22 x; sums of the
row's terms go through V / 1024 + 64 steps (a lane's and its strip's, the
strips'): c = (V / 1024 + 64) 2^-23.  With R = sum p x:
  log s    off by  ds = 2 dz / T + 2^-22 R + 2^-20 + c
  logp     off by  2 dz / T + 2^-22 x + ds + 2^-22 |logp|
  entropy  off by  ds + (2 dz / T + 2^-20 + c) R + 2^-22 sum p x^2
                   + R ds + 2^-22 H
(the strips' references are rounded products m log2(e) / T: what that takes is
put back to within 2^-22 of x or of the largest |z| / T, which dz holds).  A
gradient a [given] - p w, w = A + b (ln p + H), is formed in fp32, rounded to
the operands' type (u; f16 with 2^15 over the largest row's bound in front, so
2^-40 of that at least), summed in fp32 over V classes or n rows and rounded
once."""
import math

import pytest
import torch

from graph_rws_amd.core import _lib as L
from graph_rws_amd.core import ops
from graph_rws_amd.layers import LinearHead, linear_log_probs, log_probs

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
U = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 1e-30, torch.float16: 2.0 ** -24, torch.bfloat16: 1e-30}


def _inputs(dev, n, width, classes, dt, k, seed, nodes=None, bias=False, scale=1.0):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    h = (torch.randn(nodes or n, width, generator=g, device=dev) * scale).to(dt)
    w = (torch.randn(classes, width, generator=g, device=dev) * 2 / math.sqrt(width)).to(dt)
    b = torch.randn(classes, generator=g, device=dev).to(dt) if bias else None
    index = torch.randint(0, classes, (n, k), generator=g, device=dev)
    rows = torch.randperm(nodes, generator=g, device=dev)[:n] if nodes else None
    up = torch.randn(n, k, generator=g, device=dev), torch.randn(n, generator=g, device=dev)
    return h, w, b, rows, index, up


class _Ref:
    def __init__(self, h, w, b, rows, index, temperature=1.0, live=None):
        n = index.shape[0]
        self.dt, self.T, self.hid, self.bias = h.dtype, temperature, h.shape, b is not None
        self.rows = rows if rows is not None else torch.arange(n, device=h.device)
        self.live = live if live is not None else torch.ones(n, dtype=torch.bool, device=h.device)
        V, D = w.shape
        index = index.view(n, -1).long()
        x = h.double()[self.rows.clamp(0, h.shape[0] - 1)]
        x[~self.live] = 0
        wd = w.double()
        z = x @ wd.t()
        mag = x.abs() @ wd.abs().t()
        if b is not None:
            z = z + b.double()
            mag = mag + b.double().abs().nan_to_num(posinf=0.0)
        z[~self.live] = 0
        self.z = z
        zz = z.nan_to_num(neginf=0.0)
        dz = ((D + 8) * 2.0 ** -23 * mag + 2.0 ** -22 * zz.abs()).amax(1, keepdim=True)
        y = z / temperature
        self.lp = torch.log_softmax(y, 1)
        self.p = self.lp.exp()
        m = y.max(1, keepdim=True).values
        dist = torch.where(z > -math.inf, m - y, 0.0)
        self.H = torch.special.entr(self.p).sum(1)
        self.given = (index >= 0) & (index < V) & self.live[:, None]
        self.at = index.clamp(0, V - 1)
        self.logp = self.lp.gather(1, self.at).masked_fill(index < 0, 0.0).masked_fill(index >= V, math.nan)
        self.logp[~self.live], self.H[~self.live] = math.nan, math.nan
        e = 2 * dz[:, 0] / temperature
        c = (V / 1024 + 64) * 2.0 ** -23
        R = (self.p * dist).sum(1)
        ds = e + 2.0 ** -22 * R + 2.0 ** -20 + c
        self.tol = (e + ds)[:, None] + 2.0 ** -22 * dist + 2.0 ** -22 * torch.where(z > -math.inf, -self.lp, 0.0)
        self.tol_H = (ds + (e + 2.0 ** -20 + c) * R + 2.0 ** -22 * (self.p * dist ** 2).sum(1) + R * ds
                      + 2.0 ** -22 * torch.special.entr(self.p).sum(1))
        self.x, self.w = x, wd

    @staticmethod
    def _near(got, ref, tol, what):
        got = got.detach().double().view(ref.shape)
        ok = (got == ref) | (got.isnan() & ref.isnan()) | ((got - ref).abs() <= tol)
        assert bool(ok.all()), (what, got[~ok][:4], ref[~ok][:4], tol.expand_as(ref)[~ok][:4])

    def check(self, got, shape):
        assert got.logp.shape == shape and got.logp.dtype == got.entropy.dtype == torch.float32
        self._near(got.logp, self.logp, self.tol.gather(1, self.at), "logp")
        self._near(got.entropy, self.H, self.tol_H, "entropy")

    def check_top(self, got, top):
        """Values in order, each near what its class has; the classes are
        distinct, and none that was left out is clearly larger."""
        at = got.top_index.long()
        assert at.shape == (self.z.shape[0], top) and bool(((at >= 0) & (at < self.z.shape[1])).all())
        self._near(got.top_logp, self.lp.gather(1, at), self.tol.gather(1, at), "top_logp")
        assert all(len(set(r)) == top for r in at.tolist())
        best = torch.sort(self.lp, dim=1, descending=True).values[:, :top]
        self._near(got.top_logp, best, self.tol.amax(1, keepdim=True), "top_logp in order")
        assert bool((got.top_logp[:, 1:] <= got.top_logp[:, :-1]).all())

    def check_grads(self, grads, a, b, scale=1.0):
        n, k = self.at.shape
        zero = torch.zeros(n, dtype=torch.float64, device=self.p.device)
        a = torch.where(self.given, a.double().view(n, k), 0.0) if a is not None else zero[:, None].expand(n, k)
        b = torch.where(self.live, b.double(), 0.0) if b is not None else zero
        H = self.H.nan_to_num(0.0)
        lp = torch.where(self.p > 0, self.lp, 0.0)
        A, mag = a.sum(1), a.abs().sum(1)
        w = A[:, None] + b[:, None] * (lp + H[:, None])
        wmag = mag[:, None] + b.abs()[:, None] * (lp.abs() + H[:, None])
        g = (-self.p * w).scatter_add_(1, self.at, a) / self.T
        dw = b.abs()[:, None] * (self.tol + self.tol_H[:, None]) + (2.0 ** -20 + k * 2.0 ** -22) * wmag
        dg = self.p * ((self.tol + 2.0 ** -21) * w.abs() + dw + 2.0 ** -21 * wmag)
        dg = (dg + torch.zeros_like(g).scatter_add_(1, self.at, a.abs()) * (2.0 ** -21 + k * 2.0 ** -22)) / self.T
        dg = dg + U[self.dt] * (g.abs() + dg)
        if self.dt == torch.float16:
            dg = dg + float((mag + b.abs() * (H + 1)).max()) * 2.0 ** -40 / self.T
        dead = ~self.live
        g[dead], dg[dead] = 0, 0
        V = g.shape[1]
        u, tiny = U[self.dt], TINY[self.dt]

        def close(got, ref, tol, what):
            tol = tol + u * (ref.abs() + tol) + tiny
            d = (got.double() - ref).abs()
            assert bool((d <= tol).all()), f"{what}: {float((d / tol).max())} of the bound"

        dh, dwt, *db = grads
        ref = torch.zeros(self.hid, dtype=torch.float64, device=g.device)
        tol = torch.zeros_like(ref)
        ref[self.rows[self.live]] = (g @ self.w)[self.live]
        tol[self.rows[self.live]] = (dg @ self.w.abs() + (V + 8) * 2.0 ** -23 * (g.abs() @ self.w.abs()))[self.live]
        close(dh, ref, tol, "d_hidden")
        x = self.x.abs()
        close(dwt, g.t() @ self.x, dg.t() @ x + (n + 8) * 2.0 ** -23 * (g.abs().t() @ x), "d_weight")
        if self.bias:
            # (lists: whole units of 2^-40 of the largest row's bound)
            unit = n * k * 2.0 ** -41 * float((mag + b.abs() * (H + 1)).max()) / self.T if k > 1 else 0.0
            close(db[0], g.sum(0), dg.sum(0) + (n + 8) * 2.0 ** -23 * g.abs().sum(0) + unit, "d_bias")


def _run(h, w, b, rows, index, up, temperature=1.0, **kw):
    params = [h, w] + ([b] if b is not None else [])
    for p in params:
        p.requires_grad_()
    got = linear_log_probs(h, w, index, bias=b, rows=rows, temperature=temperature, **kw)
    grads = torch.autograd.grad([got.logp, got.entropy], params, [up[0].view(index.shape), up[1]])
    for p in params:
        p.requires_grad_(False)
    return got, grads


SHAPES = [(1, 16, 47), (1, 8, 1), (2, 1, 2), (5, 13, 257), (17, 64, 128), (64, 250, 129), (130, 96, 300),
          (129, 256, 172), (300, 1433, 7), (257, 40, 1003), (1024, 256, 172), (1, 512, 10007), (2051, 72, 4099)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("k", [1, 5])
def test_values_and_gradients(cuda_device, dt, shape, k):
    n, D, V = shape
    bias = k == 5
    h, w, b, rows, index, up = _inputs(cuda_device, n, D, V, dt, k, n + D + V, nodes=2 * n + 3 if bias else None,
                                       bias=bias)
    temperature = 1.4 if bias else 1.0
    if k > 1:
        index[torch.rand(n, k, device=cuda_device) < 0.3] = -1
        index[:, 4] = index[:, 0]  # a class given twice
        index = index.int()
    else:
        index = index[:, 0]
        index[::7] = -100
    ref = _Ref(h, w, b, rows, index, temperature)
    got, grads = _run(h, w, b, rows, index, up, temperature)
    ref.check(got, index.shape)
    ref.check_grads(grads, *up)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("shape,top", [((1, 16, 47), 5), ((1, 64, 1), 1), ((3, 40, 1000), 17), ((40, 64, 3001), 8),
                                       ((200, 96, 5003), 16), ((130, 32, 1030), 200), ((2, 72, 70001), 8),
                                       ((1024, 256, 172), 5), ((5, 8, 2000), 1000)])
def test_alternatives(cuda_device, dt, shape, top):
    n, D, V = shape
    h, w, b, rows, index, up = _inputs(cuda_device, n, D, V, dt, 2, n + V, bias=True)
    ref = _Ref(h, w, b, rows, index, 0.8)
    got = linear_log_probs(h, w, index, bias=b, temperature=0.8, top=top)
    ref.check(got, index.shape)
    ref.check_top(got, top)
    # one given class, and gradients beside alternatives
    got, grads = _run(h, w, b, rows, index[:, :1], (up[0][:, :1], up[1]), 0.8, top=top)
    one = _Ref(h, w, b, rows, index[:, :1], 0.8)
    one.check(got, (n, 1))
    one.check_grads(grads, up[0][:, :1], up[1])


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("shape", [(1, 40, 300), (7, 16, 3001), (40, 64, 3001), (300, 32, 5003)])
def test_whole_numbers_are_ordered_exactly(cuda_device, dt, shape):
    """Small whole numbers: logits are exact, equal ones are many, and the
    lowest class goes first."""
    n, D, V = shape
    g = torch.Generator(device=cuda_device)
    g.manual_seed(V)
    h = torch.randint(-3, 4, (n, D), generator=g, device=cuda_device).to(dt)
    w = torch.randint(-2, 3, (V, D), generator=g, device=cuda_device).to(dt)
    b = torch.randint(-1, 2, (V,), generator=g, device=cuda_device).to(dt)
    z = h.double() @ w.double().t() + b.double()
    order = torch.argsort(z, dim=1, descending=True, stable=True)
    index = torch.zeros(n, dtype=torch.int64, device=cuda_device)
    for top in (1, 16, 100, min(V, 500)):
        got = linear_log_probs(h, w, index, bias=b, top=top)
        assert torch.equal(got.top_index.long(), order[:, :top])
        kept = log_probs(z.float(), index, top=top)
        assert torch.equal(kept.top_index, got.top_index)


def test_bad_rows_and_classes(cuda_device):
    for n, V in ((6, 300), (200, 1500)):
        for dt in DTYPES:
            h, w, b, rows, index, up = _inputs(cuda_device, n, 48, V, dt, 3, 5, nodes=2 * n, bias=True)
            rows[1], rows[2], rows[3] = -1, 2 * n, 2 ** 40
            index[0] = torch.tensor([V, 1, -1])
            index[5] = torch.tensor([2 ** 30, -2 ** 40, 2])
            index[4] = torch.tensor([-2 ** 40, 0, 2 ** 40])  # in 32 bits: three times class 0
            h[0] = math.nan  # a row that is not asked for
            rows[rows == 0] = 2 * n - 1 if not bool((rows == 2 * n - 1).any()) else rows[4]
            live = torch.ones(n, dtype=torch.bool, device=cuda_device)
            live[1:4] = False
            if len(set(rows[live].tolist())) != int(live.sum()):
                rows[live] = torch.arange(1, 1 + int(live.sum()), device=cuda_device)
            up[0][1] = math.nan
            up[1][2] = math.inf
            hz = h.clone()
            hz[0] = 0
            for i, u in ((index, up), (index[:, :1], (up[0][:, :1], up[1]))):
                ref = _Ref(hz, w, b, rows, i, 1.0, live)
                got, grads = _run(h, w, b, rows, i, u)
                ref.check(got, i.shape)
                ref.check_grads(grads, *u)
                got = linear_log_probs(h, w, i, bias=b, rows=rows, top=4)
                ref.check(got, i.shape)
                assert bool(got.top_logp[~live].isnan().all()) and not bool(got.top_logp[live].isnan().any())


@pytest.mark.parametrize("dt", DTYPES)
def test_masked_classes(cuda_device, dt):
    """Biases of -inf and of the type's lowest value; all of them."""
    for n, V in ((5, 200), (150, 1300)):
        h, w, b, rows, index, up = _inputs(cuda_device, n, 32, V, dt, 2, 8, bias=True)
        b[: V // 2] = -math.inf
        ref = _Ref(h, w, b, rows, index)
        for top in (0, 3):
            got, grads = _run(h, w, b, rows, index, up, top=top)
            ref.check(got, index.shape)
            ref.check_grads(grads, *up)
        assert float(got.logp[index < V // 2].max()) == -math.inf
        # nothing is left: not a number, and no gradient
        b[:] = -math.inf
        got, grads = _run(h, w, b, rows, index, up)
        assert bool(got.logp.isnan().all()) and bool(got.entropy.isnan().all())
        assert all(bool((g == 0).all()) for g in grads)
        # all alike, of the lowest value: uniform
        zero = torch.zeros_like(h)
        b[:] = torch.finfo(dt).min
        for top in (0, 3):
            got, grads = _run(zero, w, b, rows, index, up, top=top)
            assert float((got.logp + math.log(V)).abs().max()) < 1e-5
            assert float((got.entropy - math.log(V)).abs().max()) < 1e-5
            assert all(bool(g.isfinite().all()) for g in grads)
        assert bool((got.top_index == torch.arange(3, device=cuda_device)).all())


def test_upstream_not_finite_stays_in_its_row(cuda_device):
    for n in (7, 200):
        h, w, b, rows, index, up = _inputs(cuda_device, n, 48, 900, torch.bfloat16, 1, 9)
        up[0][2], up[1][5] = math.nan, math.inf
        got, grads = _run(h, w, b, rows, index, up)
        bad = torch.zeros(n, dtype=torch.bool, device=cuda_device)
        bad[[2, 5]] = True
        assert bool(grads[0][~bad].isfinite().all()) and not bool(grads[0][bad].isfinite().all(1).any())
        clean = (up[0].clone(), up[1].clone())
        clean[0][2], clean[1][5] = 0, 0
        ref = _Ref(h, w, b, rows, index)
        _, fine = _run(h, w, b, rows, index, clean)
        assert torch.equal(fine[0][~bad], grads[0][~bad])
        ref.check_grads(fine, *clean)


@pytest.mark.parametrize("n", [64, 200])
def test_given_entries_take_the_product_s_probabilities(cuda_device, n):
    """The logits' gradient of a log probability sums to nothing over the
    classes, whatever the logits' own rounding, if the probability taken off at
    a given class is the one that the others have.  A column of ones in weight
    makes that sum a column of d_hidden.  Its terms have 5 roundings of 2^-23 of
    a row's sum |a| or fewer (exponential, factor, bracket, product, sum), of
    either sign: their mean square over the rows is below 5 of them."""
    g = torch.Generator(device=cuda_device)
    g.manual_seed(8)
    D, V = 16384, 58
    w = torch.randn(V, D, generator=g, device=cuda_device) / math.sqrt(D)
    best = torch.randint(0, V, (n,), generator=g, device=cuda_device)
    h = torch.randn(n, D, generator=g, device=cuda_device) + 12.0 * w[best]
    w[:, 0] = 1.0
    index = torch.stack([best, (best + 3) % V, (best + 3) % V], 1)
    a = torch.randn(n, 3, generator=g, device=cuda_device)
    h.requires_grad_()
    dh, = torch.autograd.grad(linear_log_probs(h, w, index).logp, h, a)
    off = dh[:, 0].double() / a.double().abs().sum(1)
    assert float(off.square().mean().sqrt()) < 5 * 2.0 ** -23


def test_one_upstream_alone_and_scales(cuda_device):
    for dt in DTYPES:
        h, w, b, rows, index, up = _inputs(cuda_device, 150, 64, 2000, dt, 2, 10, bias=True)
        ref = _Ref(h, w, b, rows, index)
        for p in (h, w, b):
            p.requires_grad_()
        got = linear_log_probs(h, w, index, bias=b)
        ref.check_grads(torch.autograd.grad(got.logp, [h, w, b], up[0], retain_graph=True), up[0], None)
        ref.check_grads(torch.autograd.grad(got.entropy, [h, w, b], up[1], retain_graph=True), None, up[1])
        zeros = torch.autograd.grad(got.entropy, [h, w, b], torch.zeros_like(up[1]), retain_graph=True)
        assert all(bool((g == 0).all()) for g in zeros)
        # hidden or weight alone
        only, = torch.autograd.grad([got.logp, got.entropy], [w], up, retain_graph=True)
        both = torch.autograd.grad([got.logp, got.entropy], [h, w, b], up, retain_graph=True)
        assert torch.equal(only, both[1])
        big = tuple(u * 2.0 ** 10 for u in up) if dt != torch.float16 else tuple(u * 2.0 ** -4 for u in up)
        ref.check_grads(torch.autograd.grad([got.logp, got.entropy], [h, w, b], big, retain_graph=True), *big)
        with pytest.raises(RuntimeError, match="second derivative"):
            g = torch.autograd.grad(got.logp.sum(), h, create_graph=True)[0]
            torch.autograd.grad(g.sum(), w)


def test_differences(cuda_device):
    """The gradient against central differences of the 64-bit definitions."""
    h, w, b, rows, index, up = _inputs(cuda_device, 3, 6, 20, torch.float32, 2, 12, bias=True)
    _, grads = _run(h, w, b, rows, index, up, 1.3)

    def value(x, y, z):
        lp = torch.log_softmax((x @ y.t() + z) / 1.3, 1)
        return float((lp.gather(1, index) * up[0].double()).sum() - ((lp * lp.exp()).sum(1) * up[1].double()).sum())

    args = [t.double() for t in (h, w, b)]
    e = 1e-5  # off by e^2 times a third derivative (below 100 here)
    for a, g in zip(args, grads):
        flat = a.view(-1)
        for j in range(flat.numel()):
            keep = float(flat[j])
            flat[j] = keep + e
            up_value = value(*args)
            flat[j] = keep - e
            down_value = value(*args)
            flat[j] = keep
            assert abs((up_value - down_value) / (2 * e) - float(g.reshape(-1)[j])) < 3e-5


@pytest.mark.parametrize("dt", DTYPES)
def test_strides_alignment_and_repeated_rows(cuda_device, dt):
    g = torch.Generator(device=cuda_device)
    g.manual_seed(3)
    for n, D, V in ((9, 50, 400), (140, 72, 700)):
        wide = torch.randn(n, D + 9, generator=g, device=cuda_device).to(dt)
        tall = (torch.randn(V, D + 5, generator=g, device=cuda_device) / math.sqrt(D)).to(dt)
        index = torch.randint(0, V, (n, 2), generator=g, device=cuda_device)
        up = torch.randn(n, 2, generator=g, device=cuda_device), torch.randn(n, generator=g, device=cuda_device)
        for h, w in ((wide[:, 1:1 + D], tall[:, 3:3 + D]), (wide[:, :D].t().contiguous().t(), tall[:, :D])):
            i = index.t().contiguous().t()
            ref = _Ref(h, w, None, None, i)
            got, grads = _run(h.detach(), w.detach(), None, None, i, up, top=2)
            ref.check(got, i.shape)
            ref.check_top(got, 2)
            ref.check_grads(grads, *up)
        # rows listed twice: the values are fine, their hidden row's gradient is seen to be missing
        h, w = wide[:, :D].contiguous(), tall[:, :D].contiguous()
        rows = torch.arange(n, device=cuda_device)
        rows[3] = rows[1]
        got, grads = _run(h, w, None, rows, index, up)
        _Ref(h, w, None, rows, index).check(got, index.shape)
        assert bool(grads[0][1].isnan().all()) and bool((grads[0][3] == 0).all())
        assert bool(grads[1].isfinite().all())


def test_no_rows(cuda_device):
    h = torch.zeros(0, 24, device=cuda_device, requires_grad=True)
    w = torch.ones(30, 24, device=cuda_device, requires_grad=True)
    got = linear_log_probs(h, w, torch.zeros(0, 2, dtype=torch.int64, device=cuda_device), top=4)
    assert got.logp.shape == (0, 2) and got.entropy.shape == (0,) and got.top_logp.shape == (0, 4)
    dh, dw = torch.autograd.grad(got.entropy.sum(), [h, w])
    assert dh.shape == (0, 24) and bool((dw == 0).all())


def test_blocks_and_pieces(cuda_device):
    """Rows in several blocks and classes in several pieces (by the plan)."""
    dev = cuda_device
    n, D, V = 140000, 8, 9001
    h, w, b, rows, index, up = _inputs(dev, n, D, V, torch.bfloat16, 1, 14)
    call = ops.given_call(h, w, index, b, rows, 1.0)
    import ctypes
    plan = (ctypes.c_int64 * 10)()
    view = call.view
    assert L.load().grws_head_plan(ctypes.byref(view), 1, plan) == L.GRWS_OK
    assert plan[0] > 1 and plan[2] > 1, list(plan)
    got, grads = _run(h, w, b, rows, index[:, 0], (up[0][:, 0], up[1]))
    dh = torch.zeros(n, D, dtype=torch.float64, device=dev)
    dw = torch.zeros(V, D, dtype=torch.float64, device=dev)
    # the same rows in calls of one block each
    parts = []
    for i in range(0, n, 20000):
        s = slice(i, i + 20000)
        p, g = _run(h[s].clone(), w, b, None, index[s, 0], (up[0][s, 0], up[1][s]))
        parts.append(p)
        dh[s] = g[0].double()
        dw += g[1].double()
    assert float((torch.cat([p.logp for p in parts]) - got.logp).abs().max()) < 1e-5
    assert float((torch.cat([p.entropy for p in parts]) - got.entropy).abs().max()) < 1e-5
    # both are rounded to bf16 (G to it once before): 3 roundings of 2^-8, of the sums' magnitudes
    assert float((dh - grads[0].double()).norm() / dh.norm()) < 3 * 2.0 ** -8
    assert float((dw - grads[1].double()).norm() / dw.norm()) < 3 * 2.0 ** -8
    few = linear_log_probs(h, w, index[:, 0], top=3)  # kept logits, a block of rows at a time
    assert torch.equal(few.top_index[:50], linear_log_probs(h[:50].clone(), w, index[:50, 0], top=3).top_index)
    assert float((few.logp - got.logp).abs().max()) < 1e-5


def test_linear_head_autocast_streams_and_graphs(cuda_device):
    dev = cuda_device
    torch.manual_seed(0)
    head = LinearHead(64, 3001).to(dev)
    h = torch.randn(333, 64, device=dev)
    index = torch.randint(0, 3001, (333,), device=dev)
    a = head.log_probs(h, index, temperature=1.2, top=2)
    ref = _Ref(h, head.weight.detach(), head.bias.detach(), None, index, 1.2)
    ref.check(a, (333,))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        c = head.log_probs(h, index)
    half = _Ref(h.bfloat16(), head.weight.detach().bfloat16(), head.bias.detach().bfloat16(), None, index)
    half.check(c, (333,))
    (c.logp.mean() + 0.1 * c.entropy.mean()).backward()
    assert head.weight.grad.dtype == torch.float32 and bool(head.weight.grad.isfinite().all())

    def step(x, w):
        got = linear_log_probs(x, w, index, top=4)
        lists = linear_log_probs(x, w, torch.stack([index, index.flip(0)], 1))
        return [got.logp, got.entropy, got.top_logp, got.top_index] + list(torch.autograd.grad(
            got.logp.sum() - got.entropy.sum() + lists.logp.sum(), [x, w]))

    x = h.bfloat16().requires_grad_()
    w = head.weight.detach().bfloat16().requires_grad_()
    first = [t.detach().clone() for t in step(x, w)]
    assert all(torch.equal(p, q) for p, q in zip(first, step(x, w)))
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        other = step(x, w)
    torch.cuda.current_stream(dev).wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(first, other))
    static = [h.bfloat16().requires_grad_() for _ in range(2)]
    graphs = []
    for s in static:
        leaf = w.detach().clone().requires_grad_()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(s, leaf)
        graphs.append((g, out))
    for turn in range(3):
        for (g, out), s in zip(graphs, static):
            new = torch.randn(333, 64, device=dev).bfloat16()
            with torch.no_grad():
                s.copy_(new)
            g.replay()
            eager = step(new.requires_grad_(), w)
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, eager))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("k", [1, 3])
@pytest.mark.parametrize("n,V", [(6, 300), (200, 1500), (1300, 1100)])
def test_rows_without_a_number(cuda_device, dt, k, n, V):
    """A hidden row that is not a number makes NaN of its own gradient, of the
    weight's and of the bias's, as F.linear and log_softmax do; the other rows'
    are as they are without it."""
    h, w, b, rows, index, up = _inputs(cuda_device, n, 72, V, dt, k, n, bias=True)
    _, clean = _run(h, w, b, rows, index, up)
    h[2] = math.nan
    h[4, 5] = math.nan
    rest = torch.ones(n, dtype=torch.bool, device=cuda_device)
    rest[[2, 4]] = False
    for top in (0, 3):
        got, grads = _run(h, w, b, rows, index, up, top=top)
        assert bool(got.logp[~rest].isnan().all()) and bool(got.entropy[~rest].isnan().all())
        assert not bool(got.logp[rest].isnan().any()) and not bool(got.entropy[rest].isnan().any())
        assert bool(grads[0][~rest].isnan().all())
        assert bool(grads[1].isnan().all()) and bool(grads[2].isnan().all())
        assert bool(grads[0][rest].isfinite().all())
        # (the factor in front is the largest row's, which may have been one of the two)
        far = (grads[0][rest].double() - clean[0][rest].double()).norm() / clean[0][rest].double().norm()
        assert float(far) < 2 * U[dt] + 2.0 ** -16
    # a row that has nothing but classes of -inf stays out of the gradients
    b[:] = -math.inf
    h.nan_to_num_()
    _, grads = _run(h, w, b, rows, index, up)
    assert all(bool((g == 0).all()) for g in grads)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [5, 300])
def test_upstream_near_the_largest_float(cuda_device, dt, n):
    """Finite upstream gradients whose row's bound, sum |a| + |b| (H + 1), goes
    past f32: gradients are those of 2^-20 times it, 2^20 times."""
    h, w, b, rows, index, up = _inputs(cuda_device, n, 32, 700, dt, 3, 31, bias=True)
    for t in (h, w, b):  # products with them stay below the largest float
        t.mul_(2.0 ** -8)
    a = torch.tensor([1.5 * 2.0 ** 127, -1.5 * 2.0 ** 127, 2.0 ** 100], device=cuda_device).expand(n, 3)
    e = up[1].sign() * 2.0 ** 126
    zero = torch.zeros_like
    for big in ((a, zero(e)), (zero(a), e)):
        # (another row's bound is in front: the sums are rounded elsewhere)
        _, x = _run(h, w, b, rows, index, big)
        _, y = _run(h, w, b, rows, index, tuple(t * 2.0 ** -20 for t in big))
        for p, q in zip(x[:2], y[:2]):
            q = q.double() * 2.0 ** 20
            assert float((p.double() - q).norm() / q.norm()) < 2 * U[dt] + 708 * 2.0 ** -23


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_lists_in_blocks_and_pieces(cuda_device, dt):
    """Lists of given classes (repeats, negative and far ones), a bias and rows
    of a node table, with rows in several blocks and classes in several pieces,
    against 64 bits.  Bounds, of the sums' magnitudes M (|terms| added up): a
    probability and its bracket are off by 2^-13 of the row's sum |a| + |b|
    (|ln p| + H) or less (a logit by 24 steps of 2^-23 of 60 or less, 2^-14; T,
    sums and exponentials below 2^-15), G's planes by 2^-16, a sum of N terms by
    N 2^-23, the bias's units of 2^-40 by less, and the result is rounded once."""
    import ctypes
    dev = cuda_device
    n, D, V, k, T = 140000, 8, 9001, 4, 1.25
    nodes = n + 1234
    h, w, b, rows, index, up = _inputs(dev, n, D, V, dt, k, 21, nodes=nodes, bias=True)
    g = torch.Generator(device=dev)
    g.manual_seed(22)
    index[:, 2] = index[:, 0]
    index[torch.rand(n, k, generator=g, device=dev) < 0.2] = -1
    index[::1000, 3] = V + 5
    plan = (ctypes.c_int64 * 10)()
    view = ops.given_call(h, w, index[:, :1], b, rows, 1.0).view
    assert L.load().grws_head_plan(ctypes.byref(view), 1, plan) == L.GRWS_OK
    assert plan[0] > 1 and plan[2] > 1, list(plan)
    got, grads = _run(h, w, b, rows, index, up, T)
    kept = linear_log_probs(h, w, index, bias=b, rows=rows, temperature=T, top=5)  # blocks of kept logits
    wd, bd = w.double(), b.double()
    dw, mw = torch.zeros(2, V, D, dtype=torch.float64, device=dev)
    db, mb = torch.zeros(2, V, dtype=torch.float64, device=dev)
    u, tiny = torch.finfo(dt).eps / 2, TINY[dt]

    def close(x, ref, mag, terms, what):
        tol = (2.0 ** -13 + 2.0 ** -16 + terms * 2.0 ** -23) * mag
        tol = tol + u * (ref.abs() + tol) + tiny
        worst = ((x.double() - ref).abs() / tol).max()
        assert float(worst) <= 1.0, f"{what}: {float(worst)} of the bound"

    seen = torch.zeros(nodes, dtype=torch.bool, device=dev)
    for i in range(0, n, 20000):
        s = slice(i, i + 20000)
        x = h.double()[rows[s]]
        z = x @ wd.t() + bd
        lp = torch.log_softmax(z / T, 1)
        p = lp.exp()
        H = torch.special.entr(p).sum(1)
        given = (index[s] >= 0) & (index[s] < V)
        at = index[s].clamp(0, V - 1)
        ref = lp.gather(1, at).masked_fill(index[s] < 0, 0.0).masked_fill(index[s] >= V, math.nan)
        for out in (got, kept):
            off = (out.logp[s].double() - ref).abs()
            assert bool((out.logp[s].isnan() == ref.isnan()).all()) and float(off.nan_to_num(0.0).max()) < 2.0 ** -13
            assert float((out.entropy[s].double() - H).abs().max()) < 2.0 ** -13 * (1 + float(H.max()))
        best = torch.topk(lp, 5, dim=1).values
        assert float((kept.top_logp[s].double() - best).abs().max()) < 2.0 ** -13
        assert float((lp.gather(1, kept.top_index[s].long()) - best).abs().max()) < 2.0 ** -13
        a = torch.where(given, up[0][s].double(), 0.0)
        e = up[1][s].double()
        grad = -p * (a.sum(1)[:, None] + e[:, None] * (lp + H[:, None]))
        grad = grad.scatter_add_(1, at, a) / T
        mag = p * (a.abs().sum(1)[:, None] + e.abs()[:, None] * (lp.abs() + H[:, None]))
        mag = mag.scatter_add_(1, at, a.abs()) / T
        close(grads[0][rows[s]], grad @ wd, mag @ wd.abs(), V + 8, "d_hidden")
        seen[rows[s]] = True
        dw += grad.t() @ x
        mw += mag.t() @ x.abs()
        db += grad.sum(0)
        mb += mag.sum(0)
    assert bool((grads[0][~seen] == 0).all())
    close(grads[1], dw, mw, n + 8, "d_weight")
    close(grads[2], db, mb, n + 8, "d_bias")
    # far tighter than a sum's worst case, of the whole: G's rounding and the result's
    for x, ref in ((grads[1], dw), (grads[2], db)):
        assert float((x.double() - ref).norm() / ref.norm()) < u + 2.0 ** -10


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("n,V", [(5, 300), (200, 1500), (1300, 1100)])
@pytest.mark.parametrize("k", [1, 3])
def test_far_from_zero(cuda_device, dt, n, V, k):
    """Whole numbers, whose logits are exact, at temperatures next to greedy
    ones, and under biases that lie far from zero: logits of 2^24 T and more."""
    g = torch.Generator(device=cuda_device)
    g.manual_seed(n + k)
    D = 72
    h = torch.randint(-2, 3, (n, D), generator=g, device=cuda_device).to(dt)
    w = torch.randint(-2, 3, (V, D), generator=g, device=cuda_device).to(dt)
    index = torch.randint(0, V, (n, k), generator=g, device=cuda_device)
    up = torch.randn(n, k, generator=g, device=cuda_device), torch.randn(n, generator=g, device=cuda_device)
    z = h.double() @ w.double().t()
    index[:, 0] = z.argmax(1)
    zero = torch.zeros(V, device=cuda_device, dtype=dt)
    far = (zero - 1e30 if dt != torch.float16 else zero - 65504) * 1.0
    half = zero.clone()
    half[::2] = far[0]
    for b, temperature in ((zero, 2.0 ** -20), (zero, 1e-8), (zero, 1e-12), (zero, 1e-30), (zero, 1e-37),
                           (far, 1.0), (far, 1e-8), (half, 1e-9)):
        T = float(torch.tensor(temperature))
        y = (h.float() @ w.float().t() + b.float()).double() / T  # (a logit is rounded to f32 once)
        lp = torch.log_softmax(y, 1)
        p = lp.exp()
        H = torch.special.entr(p).sum(1)
        want = lp.gather(1, index)
        a, e = up[0] * T, up[1] * T  # gradients of the size of weights
        for top in (0, 3):
            got, grads = _run(h, w, b, None, index, (a, e), temperature, top=top)
            off = (got.logp.detach().double() - want).abs()
            # 2^-22 of what lies between, and of a sum's logarithm the sum's steps
            c = (V / 1024 + 64) * 2.0 ** -23 + 2.0 ** -20
            same = got.logp.double() == want.clamp(min=-math.inf).where(want > -3.4e38, torch.tensor(-math.inf, dtype=torch.float64, device=cuda_device))
            assert bool((same | (off <= 2.0 ** -21 * want.abs() + c)).all())
            assert float((got.entropy.double() - H).abs().max()) <= c * (1 + float(H.max()))
            if top:
                best = torch.topk(lp, 3, dim=1).values
                assert bool(((got.top_logp.double() - best).abs() <= 2.0 ** -21 * best.abs() + c)
                            .logical_or(best < -3.4e38).all())
            given = a.double()
            ent = torch.where(p > 0, lp, 0.0) + H[:, None]
            gr = -p * (given.sum(1)[:, None] + e.double()[:, None] * ent)
            mag = p * (given.abs().sum(1)[:, None] + e.double().abs()[:, None] * (ent.abs() + H[:, None]))
            gr = gr.scatter_add_(1, index, given) / T
            mag = mag.scatter_add_(1, index, given.abs()) / T
            u = torch.finfo(dt).eps / 2
            for x, r, m, steps in ((grads[0], gr @ w.double(), mag @ w.double().abs(), V),
                                   (grads[1], gr.t() @ h.double(), mag.t() @ h.double().abs(), n)):
                tol = m * (u + 2.0 ** -13 + (steps + 8) * 2.0 ** -23)
                if dt == torch.float16:
                    tol = tol + float((a.abs().sum(1) + e.abs() * (H.float() + 1)).max()) / T * 2.0 ** -30
                tol = tol + u * (r.abs() + tol) + TINY[dt]
                worst = ((x.double() - r).abs() / tol).max()
                assert float(worst) <= 1.0, (temperature, float(worst))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [6, 300])
def test_a_gradient_past_f32_stays_in_its_row(cuda_device, dt, n):
    """A row whose upstream over T is more than f32 holds; the others' hidden
    gradients are as without it (rounded beside another factor)."""
    T = 2.0 ** -100
    h, w, b, rows, index, up = _inputs(cuda_device, n, 40, 500, dt, 1, 41)
    a, e = up[0].sign().clone(), torch.zeros_like(up[1])
    _, clean = _run(h, w, b, rows, index, (a, e), T)
    a[3] = 2.0 ** 40
    _, grads = _run(h, w, b, rows, index, (a, e), T)
    rest = torch.arange(n, device=cuda_device) != 3
    x, y = grads[0][rest].double(), clean[0][rest].double()
    assert bool(y.isfinite().all()) and float((x - y).norm() / y.norm()) < 2 * U[dt] + 508 * 2.0 ** -23
    assert not bool(grads[0][3].isfinite().all())
