"""core.top_logits (csrc/top.hip) against a stable sort: values and classes
are equal, so there is no tolerance."""
import math

import pytest
import torch

from graph_rws_amd.core import top_logits

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _check(x, k):
    values, index = top_logits(x, k)
    v, i = torch.sort(x, dim=1, descending=True, stable=True)
    assert values.dtype == x.dtype and index.dtype == torch.int32
    assert torch.equal(index.long(), i[:, :k])
    assert torch.equal(values.nan_to_num(nan=12345.0), v[:, :k].nan_to_num(nan=12345.0))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,classes,k", [(1, 1, 1), (1, 5, 5), (3, 64, 64), (7, 47, 5), (1024, 172, 5),
                                            (33, 2049, 1), (5, 4097, 100), (2, 1024, 1024), (1, 131072, 8),
                                            (1, 50021, 1000), (300, 50021, 64), (9, 12289, 257), (2000, 9001, 33)])
def test_matches_sort(cuda_device, dt, rows, classes, k):
    print(f"case top {dt} {rows}x{classes} k={k}", flush=True)
    g = torch.Generator(device=cuda_device)
    g.manual_seed(rows + classes)
    _check((torch.randn(rows, classes, generator=g, device=cuda_device) * 3).to(dt), k)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows", [1, 700])
def test_ties_and_special_values(cuda_device, dt, rows):
    classes, k = 9000, 70
    x = torch.zeros(rows, classes, device=cuda_device, dtype=dt)
    _check(x, k)  # all equal
    x[:, 1::2] = -0.0
    _check(x, k)  # -0 equals +0
    x = torch.randint(-2, 3, (rows, classes), device=cuda_device).to(dt)
    _check(x, k)
    x[:, ::3] = -math.inf
    _check(x, k)
    x[:, 5::17] = math.inf
    x[:, 100] = torch.finfo(dt).max
    x[:, 101] = torch.finfo(dt).min
    _check(x, k)
    x[:] = -math.inf
    x[:, 8000] = 1.0
    _check(x, k)
    x[:, 4000:4003] = math.nan
    _check(x, k)
    x[:] = math.nan
    _check(x, k)


@pytest.mark.parametrize("dt", DTYPES)
def test_rising_and_falling_rows(cuda_device, dt):
    """Rising rows raise the bound with every step."""
    r = torch.linspace(-4, 4, 30011, device=cuda_device).to(dt)
    x = torch.stack([r, r.flip(0), r.roll(7777)])
    for k in (1, 64, 1024):
        _check(x, k)


@pytest.mark.parametrize("dt", DTYPES)
def test_strides(cuda_device, dt):
    x = torch.randn(60, 5007, device=cuda_device).to(dt)
    for v in (x[:, 1:], x[::2, 3:4000], x.t(), x[:1].expand(20, 5007), x[:0], x[:, 2:9]):
        _check(v, 6)


def test_streams_and_capture(cuda_device):
    x = torch.randn(3, 70000, device=cuda_device)
    want = top_logits(x, 40)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = top_logits(x, 40)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = top_logits(x, 40)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, held))
        assert all(torch.equal(a, b) for a, b in zip(want, top_logits(x, 40)))


def test_refusals(cuda_device):
    x = torch.randn(4, 30, device=cuda_device)
    for call, err in [(lambda: top_logits(x.cpu(), 2), RuntimeError), (lambda: top_logits(x[0], 2), ValueError),
                      (lambda: top_logits(x, 0), ValueError), (lambda: top_logits(x, 31), ValueError),
                      (lambda: top_logits(torch.randn(2, 2000, device=cuda_device), 1025), ValueError),
                      (lambda: top_logits(x.double(), 2), TypeError), (lambda: top_logits(x.long(), 2), TypeError),
                      (lambda: top_logits(x[:, :0], 1), ValueError)]:
        with pytest.raises(err):
            call()
