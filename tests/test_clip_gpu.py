"""core.grad_norm and core.clip_grads (csrc/clip.hip) against 64 bits.

Bounds.  Squares of the gradients' types are exact in 64 bits (f32: 48 bits)
and their sum of N numbers is off by N 2^-53 of itself at most, so a norm has
the rounding to f32 alone: 2^-24 and N 2^-53.  The factor is rounded to f32
(2^-24; with a scale, which is a power of two here, no further), its product
with the gradient to f32 (2^-24) and to the output's type (eps / 2, or half
of the smallest number)."""
import math

import pytest
import torch

from graph_rws_amd.core import clip_grads, grad_norm
from graph_rws_amd.helper import clip_grad_norm_

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
LEAST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def _make(dev, sizes, dtypes, seed, level=1.0):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return [(torch.randn(n, generator=g, device=dev) * level).to(dt) for n, dt in zip(sizes, dtypes)]


def _norm(grads, scale=1.0):
    return scale * math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads))


def _check_norm(got, ref, n):
    assert got.dtype == torch.float32 and got.dim() == 0
    assert abs(float(got) - ref) <= ref * (2.0 ** -24 + n * 2.0 ** -52) * 1.01, (float(got), ref)


def _check_clipped(got, grads, max_norm, scale=1.0):
    norm = _norm(grads, scale)
    f = min(1.0, max_norm / (norm + 1e-6)) * scale
    for o, g in zip(got, grads):
        ref = g.double() * f
        half = torch.finfo(o.dtype).eps / 2
        tol = ref.abs() * (2.0 ** -23 + half) * 1.01 + LEAST[o.dtype]
        assert bool(((o.double() - ref).abs() <= tol).all()), (o.dtype, g.shape)


SIZES = [[1], [7], [8, 1], [0, 5, 0], [4096], [4095, 4097, 1], [3, 100003, 17], [1 << 20, 12345], list(range(200)),
         [257] * 129, [5000001]]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
def test_norm_and_clip(cuda_device, dt, sizes):
    grads = _make(cuda_device, sizes, [dt] * len(sizes), 1)
    n, ref = sum(sizes), _norm(grads)
    keep = [g.clone() for g in grads]
    _check_norm(grad_norm(grads), ref, n)
    assert all(torch.equal(a, b) for a, b in zip(grads, keep))
    # into f32 outputs, a guard behind each
    room = [torch.full((m + 3,), 7.0, device=cuda_device) for m in sizes]
    out = [r[:m] for r, m in zip(room, sizes)]
    _check_norm(clip_grads(grads, 0.5, out=out), ref, n)
    _check_clipped(out, keep, 0.5)
    assert all(bool((r[m:] == 7.0).all()) for r, m in zip(room, sizes))
    assert all(torch.equal(a, b) for a, b in zip(grads, keep))
    # in place, and again: the second norm is the clipped gradients'
    _check_norm(clip_grads(grads, 0.5), ref, n)
    _check_clipped(grads, keep, 0.5)
    _check_norm(grad_norm(grads), _norm(grads), n)


def test_types_together_and_scale(cuda_device):
    sizes = [1000, 31, 4097, 70000]
    dts = [torch.bfloat16, torch.float32, torch.float16, torch.bfloat16]
    grads = _make(cuda_device, sizes, dts, 2, level=64.0)
    scale = torch.tensor(1.0 / 1024.0, device=cuda_device)
    ref = _norm(grads, 1.0 / 1024.0)
    _check_norm(grad_norm(grads, scale=scale), ref, sum(sizes))
    out = [torch.empty(n, device=cuda_device) for n in sizes]
    _check_norm(clip_grads(grads, 1.0, out=out, scale=scale), ref, sum(sizes))
    _check_clipped(out, grads, 1.0, 1.0 / 1024.0)
    same = [torch.empty_like(g) for g in grads]
    clip_grads(grads, 1.0, out=same, scale=scale)
    _check_clipped(same, grads, 1.0, 1.0 / 1024.0)
    # nothing to clip: the scale alone, exactly
    clip_grads(grads, 1e9, out=out, scale=scale)
    assert all(torch.equal(o, g.float() / 1024.0) for o, g in zip(out, grads))
    keep = [g.clone() for g in grads]
    clip_grads(grads, 1e9)
    assert all(torch.equal(o, g) for o, g in zip(grads, keep))
    clip_grads(grads, 0.0)
    assert all(bool((g == 0).all()) for g in grads)


@pytest.mark.parametrize("offset", [1, 2, 3, 5])
def test_unaligned(cuda_device, offset):
    for dt in DTYPES:
        base = _make(cuda_device, [9000], [dt], offset)[0]
        g = base[offset:offset + 8193]
        keep, whole = g.clone(), base.clone()
        _check_norm(grad_norm([g]), _norm([keep]), 8193)
        clip_grads([g], 0.25)
        _check_clipped([g], [keep], 0.25)
        assert torch.equal(base[:offset], whole[:offset]) and torch.equal(base[offset + 8193:], whole[offset + 8193:])


def test_strides(cuda_device):
    """Transposed gradients in place as they lie; views with gaps through a copy."""
    a = torch.randn(96, 50, device=cuda_device).t()
    b = torch.randn(64, 40, device=cuda_device)[:, ::2]
    c = torch.randn(3, 4, 5, 6, device=cuda_device).to(memory_format=torch.channels_last)
    d = torch.randn((), device=cuda_device)
    grads = [a, b, c, d]
    keep = [g.clone() for g in grads]
    _check_norm(grad_norm(grads), _norm(keep), 10000)
    out = [torch.empty_like(g) for g in grads]
    clip_grads(grads, 1.0, out=out)
    _check_clipped(out, keep, 1.0)
    out = [torch.empty(g.shape, device=cuda_device) for g in grads]
    clip_grads(grads, 1.0, out=out)
    _check_clipped(out, keep, 1.0)
    with pytest.raises(ValueError, match="strides"):
        clip_grads([torch.randn(50, 96, device=cuda_device)], 1.0, out=[torch.empty(96, 50, device=cuda_device).t()])
    clip_grads(grads, 1.0)
    _check_clipped(grads, keep, 1.0)


def test_far_ends_of_f32(cuda_device):
    """Squares that f32 does not hold."""
    for level in (1e-30, 1e25):
        g = [torch.full((4099,), level, device=cuda_device)]
        ref = level * math.sqrt(4099.0)
        # the level itself is rounded to f32
        assert abs(float(grad_norm(g)) - ref) <= ref * 2.0 ** -22
        clip_grads(g, 1.0)
        want = level * min(1.0, 1.0 / (ref + 1e-6))
        assert float((g[0].double() - want).abs().max()) <= want * 2.0 ** -21


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_not_finite(cuda_device, bad):
    """As torch's clip_grad_norm_: infinities make zeros and a NaN, a NaN makes NaN."""
    mine = _make(cuda_device, [100, 5000], [torch.float32] * 2, 3)
    mine[1][4321] = bad
    p = [torch.nn.Parameter(torch.zeros_like(g)) for g in mine]
    for q, g in zip(p, mine):
        q.grad = g.clone()
    ref = torch.nn.utils.clip_grad_norm_(p, 1.0)
    got = clip_grads(mine, 1.0)
    assert torch.equal(got, ref) or (bool(got.isnan()) and bool(ref.isnan()))
    for q, g in zip(p, mine):
        assert torch.equal(g.nan_to_num(nan=5.0), q.grad.nan_to_num(nan=5.0))


def test_same_bits_and_versions(cuda_device):
    grads = _make(cuda_device, [1234567, 89], [torch.bfloat16] * 2, 4)
    norms = {float(grad_norm(grads)) for _ in range(5)}
    assert len(norms) == 1
    before = [g._version for g in grads]
    clip_grads(grads, 1.0)
    assert all(g._version > v for g, v in zip(grads, before))
    with pytest.raises(Exception, match="overlap"):
        clip_grads([grads[0], grads[0]], 1.0)
    with pytest.raises(TypeError):
        clip_grads([torch.zeros(3, device=cuda_device)], 1.0,
                   out=[torch.zeros(3, device=cuda_device, dtype=torch.bfloat16)])
    with pytest.raises(TypeError):
        grad_norm([torch.zeros(3, device=cuda_device, dtype=torch.float64)])


def test_inference_mode(cuda_device):
    with torch.inference_mode():
        grads = _make(cuda_device, [1000, 7], [torch.float32, torch.bfloat16], 9)
        keep = [g.clone() for g in grads]
        out = [torch.empty(g.shape, device=cuda_device) for g in grads]
        _check_norm(clip_grads(grads, 1.0, out=out), _norm(keep), 1007)
        _check_clipped(out, keep, 1.0)
        clip_grads(grads, 1.0)
        _check_clipped(grads, keep, 1.0)


def test_other_stream_and_graph(cuda_device):
    """A call on a stream of its own, and two captured ones replayed in turn
    with eager calls between."""
    grads = _make(cuda_device, [60001, 33], [torch.float32, torch.bfloat16], 5)
    out = [torch.empty(g.shape, device=cuda_device) for g in grads]
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        norm = clip_grads(grads, 1.0, out=out)
    torch.cuda.current_stream(cuda_device).wait_stream(side)
    _check_norm(norm, _norm(grads), 60034)
    _check_clipped(out, grads, 1.0)
    other = [torch.empty_like(o) for o in out]
    graphs, norms = [], []
    for target in (out, other):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            norms.append(clip_grads(grads, 1.0, out=target))
        graphs.append(g)
    for turn in range(4):
        for t, new in zip(grads, _make(cuda_device, [60001, 33], [torch.float32, torch.bfloat16], 10 + turn)):
            t.copy_(new)
        for g, n, target in zip(graphs, norms, (out, other)):
            for o in target:
                o.zero_()
            g.replay()
            eager = [torch.empty_like(o) for o in target]
            ref = clip_grads(grads, 1.0, out=eager)
            assert torch.equal(n, ref)
            assert all(torch.equal(a, b) for a, b in zip(target, eager))


def test_parameters(cuda_device):
    """helper.clip_grad_norm_ against torch's, whose f32 norm is off by its
    sums' roundings (up to 2^-20 of these)."""
    def params(dt):
        g = torch.Generator(device=cuda_device)
        g.manual_seed(6)
        p = [torch.nn.Parameter(torch.zeros(s, device=cuda_device, dtype=dt)) for s in [(40, 30), (30,), (7, 1, 3)]]
        for q in p[:2]:
            q.grad = torch.randn(q.shape, generator=g, device=cuda_device).to(dt)
        return p

    a, b = params(torch.float32), params(torch.float32)
    na, nb = clip_grad_norm_(a, 1.0), torch.nn.utils.clip_grad_norm_(b, 1.0)
    assert abs(float(na) - float(nb)) <= 2.0 ** -20 * float(nb)
    for x, y in zip(a[:2], b[:2]):
        assert float((x.grad - y.grad).abs().max()) <= 2.0 ** -19 * float(y.grad.abs().max())
    assert a[2].grad is None
    # one that is listed twice, and types that the kernels do not take, are torch's
    c = params(torch.float64)
    clip_grad_norm_(c, 1.0)
    assert abs(math.sqrt(sum(float((q.grad ** 2).sum()) for q in c[:2])) - 1.0) < 1e-6
    a, b = params(torch.float32), params(torch.float32)
    clip_grad_norm_([a[0], a[0]], 1.0)
    torch.nn.utils.clip_grad_norm_([b[0], b[0]], 1.0)
    assert torch.equal(a[0].grad, b[0].grad)


def test_norm_beyond_f32(cuda_device):
    """A norm that f32 does not hold is infinite, and clips to zeros, as
    torch's does."""
    for dt, level in ((torch.float32, 1e38), (torch.bfloat16, 2.0 ** 126)):
        g = [torch.full((4099,), level, device=cuda_device, dtype=dt), torch.ones(5, device=cuda_device, dtype=dt)]
        assert float(grad_norm(g)) == math.inf
        out = [torch.full(t.shape, 7.0, device=cuda_device) for t in g]
        assert float(clip_grads(g, 1.0, out=out)) == math.inf
        assert all(bool((o == 0).all()) for o in out)
        p = [torch.nn.Parameter(torch.zeros_like(t)) for t in g]
        for q, t in zip(p, g):
            q.grad = t.clone()
        torch.nn.utils.clip_grad_norm_(p, 1.0)
        assert float(clip_grads(g, 1.0)) == math.inf
        assert all(torch.equal(t, q.grad) for t, q in zip(g, p))
        # a scale that brings the norm back
        g = [torch.full((4099,), level, device=cuda_device, dtype=dt)]
        scale = torch.tensor(2.0 ** -30, device=cuda_device)
        ref = _norm(g, 2.0 ** -30)
        _check_norm(clip_grads(g, 1.0, out=out[:1], scale=scale), ref, 4099)
        _check_clipped(out[:1], g, 1.0, 2.0 ** -30)


@pytest.mark.parametrize("max_norm", [2.0 ** -7, 2.0 ** -17, 2.0 ** -66, 2.0 ** -113])
def test_factors_below_the_smallest_float(cuda_device, max_norm):
    """max_norm / norm is a number that f32 holds with few bits or not at all,
    the clipped gradients are not.  (The bounds of the file's head.)"""
    for dt in (torch.float32, torch.bfloat16):
        g = _make(cuda_device, [4099, 12], [dt] * 2, 3, level=1e36)
        keep = [t.clone() for t in g]
        out = [torch.empty(t.shape, device=cuda_device) for t in g]
        _check_norm(clip_grads(g, max_norm, out=out), _norm(keep), 4111)
        _check_clipped(out, keep, max_norm)
        clip_grads(g, max_norm)
        _check_clipped(g, keep, max_norm)
        assert not bool((g[0] == 0).all())


def test_parameters_whose_gradients_share_memory(cuda_device):
    """Views of one buffer that overlap go to torch, as a gradient that is
    listed twice does; ones that lie apart do not.  (Torch scales what is
    shared more than once and in no order, so nothing is clipped here.)"""
    from graph_rws_amd.helper import engine
    buf = torch.randn(64, 48, device=cuda_device)

    def params(*grads):
        p = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
        for q, g in zip(p, grads):
            q.grad = g
        return p

    for views in ((buf, buf.view(-1)), (buf[:40], buf[30:]), (buf[:, :30], buf[:, 20:]), (buf.view(-1)[5:9], buf.t())):
        p = params(*views)
        keep = buf.clone()
        norm = clip_grad_norm_(p, 1e6)
        ref = math.sqrt(sum(float((v.double() ** 2).sum()) for v in views))
        assert abs(float(norm) - ref) <= 2.0 ** -18 * ref
        assert torch.equal(buf, keep)
    clipped = []
    real = engine.torch.nn.utils.clip_grad_norm_
    try:
        engine.torch.nn.utils.clip_grad_norm_ = lambda *a, **k: clipped.append(1)
        clip_grad_norm_(params(buf[:32], buf[32:]), 1.0)
        clip_grad_norm_(params(buf[::2], buf[:0], torch.ones(3, device=cuda_device)), 1.0)
    finally:
        engine.torch.nn.utils.clip_grad_norm_ = real
    assert not clipped


def test_offsets_past_32_bits(cuda_device):
    """A tensor of 2^32 gradients and more, with another behind it."""
    n = (1 << 32) + 4099
    big = torch.full((n,), 0.5, device=cuda_device, dtype=torch.bfloat16)
    small = torch.full((77,), 3.0, device=cuda_device)
    big[-1] = 64.0
    ref = math.sqrt((n - 1) * 0.25 + 64.0 ** 2 + 77 * 9.0)
    norm = clip_grads([big, small], 1024.0)
    assert abs(float(norm) - ref) <= ref * 2.0 ** -23
    f = 1024.0 / (ref + 1e-6)
    for got, g in ((big[:3], 0.5), (big[1 << 31:(1 << 31) + 3], 0.5), (big[-3:-1], 0.5), (big[-1:], 64.0), (small, 3.0)):
        want = g * f
        assert float((got.double() - want).abs().max()) <= want * (2.0 ** -8 + 2.0 ** -22)
