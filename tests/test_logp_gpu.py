"""layers.log_probs (csrc/logp.hip) against the definitions in 64 bits.

Bounds, per element.  x = (m - z) / T is how far a logit lies below the
largest one.  It is formed by a difference, a factor log2(e) / T (itself
rounded) and a product, so it is off by 2^-22 x; 2^-x is then off by 2^-22 x
+ 2^-22 of itself.  A sum of a row's V terms goes through V / 256 + 48 steps
at most on its way (a thread's, its wave's, the work-group's or the
stretches'): c = (V / 256 + 48) 2^-23.  With R = sum p x:
  log s    off by  ds = 2^-22 R + 2^-21 + c
  logp     off by  2^-22 x + ds + 2^-22 |logp|
  entropy  off by  ds + 2^-22 sum p x^2 + (2^-21 + c) R + R ds + 2^-22 H
A gradient (a [given] - p w) / T, w = A + b (ln p + H), has p off by logp's
bound of itself, w by |b| times logp's and the entropy's and the roundings
of its terms, and is rounded to the logits' type once."""
import math

import pytest
import torch

from graph_rws_amd.layers import log_probs

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
LEAST = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}


class _Ref:
    def __init__(self, logits, index, temperature=1.0):
        z = logits.double()
        n, V = z.shape
        self.dt, self.T, self.V = logits.dtype, temperature, V
        index = index.view(n, -1).long()
        y = z / temperature
        self.logp_all = torch.log_softmax(y, 1)
        self.p = self.logp_all.exp()
        m = y.max(1, keepdim=True).values
        self.x = torch.where(z > -math.inf, m - y, 0.0)
        self.H = torch.special.entr(self.p).sum(1)
        self.given = (index >= 0) & (index < V)
        self.at = index.clamp(0, V - 1)
        self.logp = self.logp_all.gather(1, self.at).masked_fill(index < 0, 0.0).masked_fill(index >= V, math.nan)
        c = (V / 256 + 48) * 2.0 ** -23
        R = (self.p * self.x).sum(1)
        ds = 2.0 ** -22 * R + 2.0 ** -21 + c
        self.tol_all = 2.0 ** -22 * self.x + ds[:, None] + 2.0 ** -22 * torch.where(z > -math.inf, -self.logp_all, 0.0)
        self.tol_H = (ds + 2.0 ** -22 * (self.p * self.x ** 2).sum(1) + (2.0 ** -21 + c) * R + R * ds
                      + 2.0 ** -22 * self.H)

    def check(self, got, shape):
        assert got.logp.shape == shape and got.logp.dtype == got.entropy.dtype == torch.float32
        lp = got.logp.detach().double().view(self.logp.shape)
        # what f32 does not hold is -inf there
        low = self.logp < -float(torch.finfo(torch.float32).max)
        self.logp = torch.where(low, -math.inf, self.logp)
        tol = self.tol_all.gather(1, self.at)
        same = (lp == self.logp) | (lp.isnan() & self.logp.isnan())
        bad = ~same & ~((lp - self.logp).abs() <= tol)
        assert not bool(bad.any()), (lp[bad][:4], self.logp[bad][:4], tol[bad][:4])
        worst = ((got.entropy.detach().double() - self.H).abs() / self.tol_H).max()
        assert float(worst) <= 1.0, f"entropy: {float(worst)} of the bound"

    def check_top(self, got, logits, top):
        order = torch.argsort(logits.double(), dim=1, descending=True, stable=True)[:, :top]
        assert torch.equal(got.top_index.long(), order)
        ref, tol = self.logp_all.gather(1, order), self.tol_all.gather(1, order)
        lp = got.top_logp.double()
        assert bool(((lp == ref) | ((lp - ref).abs() <= tol)).all())

    def check_grad(self, grad, a, b):
        """a as the given classes, b [n] (None: zeros)."""
        n, k = self.at.shape
        zero = torch.zeros(n, dtype=torch.float64, device=grad.device)
        a = torch.where(self.given, a.double().view(n, k), 0.0) if a is not None else zero[:, None].expand(n, k)
        b = b.double() if b is not None else zero
        A, mag = a.sum(1), a.abs().sum(1)
        lp = torch.where(self.p > 0, self.logp_all, 0.0)
        w = A[:, None] + b[:, None] * (lp + self.H[:, None])
        g = -self.p * w
        g.scatter_add_(1, self.at, a)
        g /= self.T
        wmag = mag[:, None] + b.abs()[:, None] * (lp.abs() + self.H[:, None])
        dw = b.abs()[:, None] * (self.tol_all + self.tol_H[:, None]) + (2.0 ** -21 + k * 2.0 ** -23) * wmag
        tol = self.p * ((self.tol_all + 2.0 ** -22) * w.abs() + dw + 2.0 ** -22 * wmag)
        spread = torch.zeros_like(g).scatter_add_(1, self.at, a.abs())
        tol = (tol + (2.0 ** -22 + k * 2.0 ** -23) * spread + 2.0 ** -120 * wmag) / self.T
        u = torch.finfo(self.dt).eps / 2
        tol = tol * (1 + u) + u * g.abs() + LEAST[self.dt]
        assert grad.dtype == self.dt
        d = (grad.double() - g).abs()
        worst = float((d / tol).max())
        assert worst <= 1.0, f"gradient: {worst} of the bound"


def _inputs(dev, n, V, dt, k, seed, spread=3.0):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    z = (torch.randn(n, V, generator=g, device=dev) * spread).to(dt)
    index = torch.randint(0, V, (n, k), generator=g, device=dev)
    a = torch.randn(n, k, generator=g, device=dev)
    b = torch.randn(n, generator=g, device=dev)
    return z, index, a, b


SHAPES = [(1, 1), (1, 2), (3, 47), (5, 64), (4, 65), (2, 256), (7, 257), (1024, 172), (3, 1000), (9, 1024), (2, 1025),
          (5, 2047), (3, 4096), (1, 8191), (2, 8193), (17, 10007), (1100, 1111), (1030, 2051), (1, 131072), (3, 50021)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_values_and_gradients(cuda_device, dt, shape):
    n, V = shape
    for k, temperature in ((1, 1.0), (4, 0.7), (3, 2.5)):
        z, index, a, b = _inputs(cuda_device, n, V, dt, k, n + V + k)
        if k > 1:  # nothing asked, a class given twice
            index[torch.rand(n, k, device=cuda_device) < 0.3] = -1
            index[:, k - 1] = index[:, 0]
        if k == 1:
            index, a = index[:, 0], a[:, 0]
        if k == 3:
            index = index.int()
        ref = _Ref(z, index, temperature)
        z.requires_grad_()
        got = log_probs(z, index, temperature=temperature)
        assert got.top_logp is None and got.top_index is None
        ref.check(got, index.shape)
        grad, = torch.autograd.grad([got.logp, got.entropy], [z], [a, b])
        ref.check_grad(grad, a, b)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("shape,top", [((1, 1), 1), ((5, 7), 7), ((33, 172), 5), ((3, 1024), 16), ((4, 1024), 17),
                                       ((2, 1025), 8), ((1, 131072), 8), ((3, 50021), 64), ((1100, 3001), 16),
                                       ((2, 20000), 128), ((2, 20000), 129), ((3, 30011), 1000), ((1, 1024), 1024)])
def test_alternatives(cuda_device, dt, shape, top):
    n, V = shape
    z, index, _, _ = _inputs(cuda_device, n, V, dt, 2, n * V + top)
    if n > 2:
        z[1] = z[1].round()  # ties
        z[2] = 1.5
    if n > 3:
        z[3] = torch.linspace(-5, 5, V, device=cuda_device).to(dt)  # rising: the bound comes late
    ref = _Ref(z, index, 0.9)
    got = log_probs(z, index, temperature=0.9, top=top)
    ref.check(got, index.shape)
    ref.check_top(got, z, top)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("V", [50, 700, 5000, 70001])
def test_masks(cuda_device, dt, V):
    """-inf and the type's lowest value in some places, or in all."""
    lowest = torch.finfo(dt).min
    z, index, a, b = _inputs(cuda_device, 8, V, dt, 2, V)
    z[0, V // 3:] = -math.inf
    index[0] = torch.tensor([V - 1, 0])
    z[1, : V // 2] = lowest
    index[1] = torch.tensor([0, V - 1])
    z[2] = lowest  # all alike: uniform
    z[3] = -math.inf
    z[3, V - 1] = 2.0  # one class is left
    index[3] = torch.tensor([V - 1, 1])
    z[4] = lowest
    z[4, 7] = -lowest
    index[4] = torch.tensor([7, 8])
    z[5, 1:] = -math.inf
    z[5, 0] = lowest
    index[5] = torch.tensor([0, -1])
    z[6] = -math.inf
    z[7] = z[7] * 100
    live = [0, 1, 2, 3, 4, 5, 7]
    z.requires_grad_()
    got = log_probs(z, index, top=3)
    assert bool(got.logp[6].isnan().all()) and bool(got.entropy[6].isnan())
    # a row that has nothing is left out of the loss: zeros reach it
    a[6], b[6] = 0, 0
    grad, = torch.autograd.grad([got.logp, got.entropy], [z], [a, b])
    assert bool((grad[6] == 0).all())
    zz = z.detach()[live]
    ref = _Ref(zz, index[live])
    ref.check(type(got)(got.logp[live], got.entropy[live]), (len(live), 2))
    ref.check_grad(grad[live], a[live], b[live])
    assert float(got.logp[0, 0]) == -math.inf and float(got.entropy[3]) == 0.0 and float(got.logp[3, 0]) == 0.0
    order = torch.argsort(z.detach().double(), dim=1, descending=True, stable=True)[:, :3]
    assert torch.equal(got.top_index.long(), order)


def test_not_finite_stays_in_its_row(cuda_device):
    for V in (40, 3000):
        z, index, a, b = _inputs(cuda_device, 4, V, torch.float32, 1, V)
        z[1, 5], z[2, 6] = math.inf, math.nan
        z.requires_grad_()
        got = log_probs(z, index)
        assert bool(got.logp[1:3].isnan().all()) and bool(got.entropy[1:3].isnan().all())
        a[0] = math.inf
        grad, = torch.autograd.grad([got.logp, got.entropy], [z], [a, b])
        assert bool(grad[1:3].isnan().any(1).all()) and bool(grad[0].isfinite().logical_not().any())
        ref = _Ref(z.detach()[3:], index[3:])
        ref.check(type(got)(got.logp[3:], got.entropy[3:]), (1, 1))
        ref.check_grad(grad[3:], a[3:], b[3:])


def test_given_out_of_range_and_nothing_asked(cuda_device):
    for V in (100, 5000):
        z, index, a, b = _inputs(cuda_device, 3, V, torch.float32, 3, 9)
        index[0] = torch.tensor([V, 1, -1])
        index[1] = torch.tensor([2 ** 40, -100, -2 ** 40])
        a[1] = math.nan  # nothing of that row is given
        z.requires_grad_()
        got = log_probs(z, index)
        assert got.logp[0].isnan().tolist() == [True, False, False] and float(got.logp[0, 2]) == 0.0
        assert got.logp[1].isnan().tolist() == [True, False, False]
        ref = _Ref(z.detach(), index)
        ref.check(got, (3, 3))
        grad, = torch.autograd.grad([got.logp, got.entropy], [z], [a, b])
        ref.check_grad(grad, a.nan_to_num(), b)


def test_many_given(cuda_device):
    """1,024 given classes of 700: every one given again."""
    for dt in DTYPES:
        z, index, a, b = _inputs(cuda_device, 3, 700, dt, 1024, 3)
        ref = _Ref(z, index)
        z.requires_grad_()
        got = log_probs(z, index)
        ref.check(got, index.shape)
        grad, = torch.autograd.grad([got.logp, got.entropy], [z], [a, b])
        ref.check_grad(grad, a, b)


@pytest.mark.parametrize("V", [60, 3001])
def test_one_upstream_alone(cuda_device, V):
    z, index, a, b = _inputs(cuda_device, 6, V, torch.float32, 2, 11)
    ref = _Ref(z, index)
    z.requires_grad_()
    got = log_probs(z, index)
    ref.check_grad(torch.autograd.grad(got.logp, z, a, retain_graph=True)[0], a, None)
    ref.check_grad(torch.autograd.grad(got.entropy, z, b, retain_graph=True)[0], None, b)
    ref.check_grad(torch.autograd.grad(got.entropy.sum(), z, retain_graph=True)[0], None, torch.ones_like(b))
    with pytest.raises(RuntimeError, match="second derivative"):
        g, = torch.autograd.grad(got.logp.sum(), z, create_graph=True)
        torch.autograd.grad(g.sum(), z)


def test_differences(cuda_device):
    """The gradient against central differences of the 64-bit definitions."""
    z, index, a, b = _inputs(cuda_device, 2, 30, torch.float32, 2, 12)
    z.requires_grad_()
    got = log_probs(z, index, temperature=1.3)
    grad, = torch.autograd.grad([got.logp, got.entropy], [z], [a, b])

    def value(y):
        lp = torch.log_softmax(y / 1.3, 1)
        return float((lp.gather(1, index) * a.double()).sum() - ((lp * lp.exp()).sum(1) * b.double()).sum())

    h = 1e-5  # off by h^2 times a third derivative (below 10 here), and 2^-52 / h
    for r in range(2):
        for v in range(30):
            up, down = z.detach().double(), z.detach().double()
            up[r, v] += h
            down[r, v] -= h
            assert abs((value(up) - value(down)) / (2 * h) - float(grad[r, v])) < 1e-5


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("V", [333, 9001])
def test_strides_and_alignment(cuda_device, dt, V):
    wide, index, a, b = _inputs(cuda_device, 6, V + 40, dt, 2, V)
    index %= V
    for z in (wide[:, 3:3 + V], wide[:, 8:8 + V], wide[::2, 1:1 + V], wide.t().contiguous().t()[:, :V],
              wide[:1].expand(6, V + 40)[:, :V]):
        n = z.shape[0]
        i = index[:n].t().contiguous().t()  # rows of classes that do not lie together
        ref = _Ref(z, i)
        x = z.detach()
        x = x.requires_grad_() if x.is_leaf else x
        got = log_probs(x, i, top=2)
        ref.check(got, i.shape)
        ref.check_top(got, z, 2)
        grad, = torch.autograd.grad([got.logp, got.entropy], [x], [a[:n], b[:n]])
        ref.check_grad(grad, a[:n], b[:n])


def test_more_rows_than_a_launch_takes(cuda_device):
    """A wave a row: 2^25 rows a launch."""
    n, last = (1 << 25) + 5, 1000
    g = torch.Generator(device=cuda_device)
    g.manual_seed(1)
    z = torch.randn(n, 3, generator=g, device=cuda_device, dtype=torch.float16).requires_grad_()
    index = torch.randint(0, 3, (n,), generator=g, device=cuda_device, dtype=torch.int32)
    got = log_probs(z, index, top=1)
    a = torch.ones(n, device=cuda_device)
    grad, = torch.autograd.grad(got.logp, z, a)
    tail = z.detach()[-last:].clone().requires_grad_()
    ref = log_probs(tail, index[-last:], top=1)
    assert torch.equal(got.logp[-last:], ref.logp) and torch.equal(got.entropy[-last:], ref.entropy)
    assert torch.equal(got.top_index[-last:], ref.top_index) and torch.equal(got.top_logp[-last:], ref.top_logp)
    assert torch.equal(grad[-last:], torch.autograd.grad(ref.logp, tail, a[-last:])[0])


def test_not_finite_alternatives(cuda_device):
    """NaN first, as a sort has it; +inf before what is finite."""
    for V in (300, 20000):
        z, index, _, _ = _inputs(cuda_device, 3, V, torch.bfloat16, 1, V)
        z[0, [7, 200, 250]] = math.nan
        z[1, [9, 100]] = math.inf
        z[2, ::2] = math.nan
        order = torch.argsort(z.float(), dim=1, descending=True, stable=True)
        for top in (2, 8, 20, 200):
            got = log_probs(z, index, top=top)
            assert torch.equal(got.top_index[:2].long(), order[:2, :top])
            assert bool(got.top_index[2].remainder(2).eq(0).all()) or top > V // 2


def test_no_rows(cuda_device):
    z = torch.zeros(0, 30, device=cuda_device, requires_grad=True)
    got = log_probs(z, torch.zeros(0, dtype=torch.int64, device=cuda_device), top=4)
    assert got.logp.shape == (0,) and got.entropy.shape == (0,) and got.top_index.shape == (0, 4)
    grad, = torch.autograd.grad(got.entropy.sum(), z)
    assert grad.shape == (0, 30)


def test_same_bits_streams_and_graphs(cuda_device):
    dev = cuda_device
    z, index, a, b = _inputs(dev, 5, 70003, torch.bfloat16, 2, 13)

    def step(x):
        got = log_probs(x, index, top=8)
        return [got.logp, got.entropy, got.top_logp, got.top_index] + list(
            torch.autograd.grad([got.logp, got.entropy], [x], [a, b]))

    x = z.clone().requires_grad_()
    first = [t.detach().clone() for t in step(x)]
    assert all(torch.equal(s, t) for s, t in zip(first, step(x)))
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        other = step(x)
    torch.cuda.current_stream(dev).wait_stream(side)
    assert all(torch.equal(s, t) for s, t in zip(first, other))
    # two captures of one leaf, replayed in turn
    static = [z.clone().requires_grad_() for _ in range(2)]
    graphs = []
    for s in static:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(s)
        graphs.append((g, out))
    for turn in range(3):
        for (g, out), s in zip(graphs, static):
            new = _inputs(dev, 5, 70003, torch.bfloat16, 2, 20 + turn)[0]
            with torch.no_grad():
                s.copy_(new)
            g.replay()
            eager = step(new.requires_grad_())
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, eager))


def test_second_derivative_is_refused_whatever_the_strides(cuda_device):
    """Also beside a term of the loss that has one, and of logits that are
    copied for the kernels."""
    index = torch.tensor([0, 2, 4, 1], device=cuda_device)
    for shape, view in (((4, 5), lambda t: t), ((5, 4), lambda t: t.t()), ((4, 10), lambda t: t[:, ::2]),
                        ((1, 5), lambda t: t.expand(4, 5))):
        leaf = torch.randn(shape, device=cuda_device).requires_grad_()
        g, = torch.autograd.grad(log_probs(view(leaf), index).logp.sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="second derivative"):
            (leaf.square().sum() + g.square().sum()).backward()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("V", [40, 700, 5000, 140001])
def test_rows_without_a_number(cuda_device, dt, V):
    """Rows of NaN alone, or of NaN and -inf, have NaN for a gradient in every
    place, where one of nothing but -inf has zeros."""
    for n in (6, 1030) if V < 10000 else (6,):
        z, index, a, b = _inputs(cuda_device, n, V, dt, 2, V + n)
        z[1] = math.nan
        z[2], z[2, V // 2] = -math.inf, math.nan
        z[3] = -math.inf
        z[4, V - 1] = math.nan
        z.requires_grad_()
        got = log_probs(z, index, top=3)
        assert bool(got.logp[1:5].isnan().all()) and bool(got.entropy[1:5].isnan().all())
        for up in ((a, b), (a, None), (None, b)):
            given = [(o, u) for o, u in zip((got.logp, got.entropy), up) if u is not None]
            grad, = torch.autograd.grad([o for o, _ in given], [z], [u for _, u in given], retain_graph=True)
            assert bool(grad[[1, 2, 4]].isnan().all())
            assert bool((grad[3] == 0).all())
            rest = [0, *range(5, n)]
            ref = _Ref(z.detach()[rest], index[rest])
            ref.check_grad(grad[rest], *(u[rest] if u is not None else None for u in up))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("V", [700, 5000, 140001])
def test_far_from_zero(cuda_device, dt, V):
    """Logits whose size over T is past 2^24, where a product with log2(e) / T
    has no fraction left: rows of nothing but masks of -1e30 (or what the type
    holds), large offsets, temperatures next to greedy ones."""
    most = float(torch.finfo(dt).max)
    z, index, a, b = _inputs(cuda_device, 9, V, dt, 2, V + 5)
    z[0] = max(-1e30, -most)
    z[1] = max(-1e10, -most)
    z[2] = -1e9 if most > 1e9 else -6e4
    z[2, ::3] = z[2, 1] / 2  # a mask that is a mask of another
    z[3] = min(1e30, most)
    z[4] = (z[4].float() * 1e4).clamp(-most, most).to(dt)
    z[5] = (z[5].float() * 1e-3 * most).to(dt)
    z[6] = min(1e30, most / 2)
    z[6, V - 2] *= -1
    for temperature in (1.0, 2.0 ** -20, 1e-8, 1e-12, 1e-20, 1e-37):
        ref = _Ref(z, index, float(torch.tensor(temperature)))
        x = z.detach().clone().requires_grad_()
        got = log_probs(x, index, temperature=temperature, top=3)
        low = ref.logp < -float(torch.finfo(torch.float32).max)
        assert not bool(got.logp.isnan().any()) and not bool(got.entropy.isnan().any())
        ref.check(got, index.shape)
        assert bool((got.logp[low] == -math.inf).all())
        order = torch.argsort(z.double(), dim=1, descending=True, stable=True)[:, :3]
        assert torch.equal(got.top_index.long(), order)
        grad, = torch.autograd.grad(got.logp, [x], [a * temperature])
        ref.check_grad(grad, a * temperature, None)


def test_offsets_past_32_bits(cuda_device):
    """More than 2^32 logits: the last rows as in a call of their own."""
    n, V, k, last = 70001, 65537, 2, 300
    g = torch.Generator(device=cuda_device)
    g.manual_seed(2)
    z = torch.empty(n, V, device=cuda_device, dtype=torch.float16)
    z.normal_(generator=g)
    index = torch.randint(0, V, (n, k), generator=g, device=cuda_device)
    a = torch.randn(n, k, generator=g, device=cuda_device)
    z.requires_grad_()
    got = log_probs(z, index, top=3)
    grad, = torch.autograd.grad([got.logp, got.entropy], [z], [a, a[:, 0]])
    tail = z.detach()[-last:].clone().requires_grad_()
    ref = log_probs(tail, index[-last:], top=3)
    for p, q in zip(got[:2] + got[2:], ref[:2] + ref[2:]):
        assert torch.allclose(p[-last:].float(), q.float(), rtol=2.0 ** -20, atol=2.0 ** -20)
    assert torch.equal(got.top_index[-last:], ref.top_index)
    want, = torch.autograd.grad([ref.logp, ref.entropy], [tail], [a[-last:], a[-last:, 0]])
    assert float((grad[-last:].float() - want.float()).abs().max()) <= 2.0 ** -10 * float(want.abs().max())
