"""Host side of gradient norms and clipping: refusals before any launch (CPU
tier: nothing here touches a GPU)."""
import ctypes

import pytest
import torch

from graph_rws_amd.core import _lib as L
from graph_rws_amd.core import clip_grads, grad_norm
from graph_rws_amd.helper import clip_grad_norm_


def _call(grads, dtypes=None, sizes=None, outs=None, out_dtypes=None, max_norm=1.0, norm=1 << 20, ws=1 << 20,
          ws_bytes=1 << 30, count=None):
    """grws_clip_grads with made-up addresses, which a refused call never reads."""
    m = len(grads)
    dtypes = dtypes or [L.GRWS_F32] * m
    sizes = sizes or [16] * m
    ints = ctypes.c_int32 * m
    return L.load().grws_clip_grads(
        (ctypes.c_void_p * m)(*grads), ints(*dtypes), (ctypes.c_int64 * m)(*sizes),
        (ctypes.c_void_p * m)(*outs) if outs is not None else None,
        ints(*out_dtypes) if out_dtypes is not None else None, m if count is None else count, max_norm, None, norm, ws,
        ws_bytes, None)


A, B, C = 1 << 20, 2 << 20, 3 << 20


@pytest.mark.parametrize("kw,status,word", [
    (dict(grads=[A], count=-1), L.GRWS_E_INVALID, b"lists"),
    (dict(grads=[A], norm=None), L.GRWS_E_INVALID, b"nothing"),
    (dict(grads=[A], outs=[A], max_norm=-1.0), L.GRWS_E_INVALID, b"negative"),
    (dict(grads=[A], outs=[A], max_norm=float("nan")), L.GRWS_E_INVALID, b"negative"),
    (dict(grads=[A], dtypes=[5]), L.GRWS_E_DTYPE, b"dtype 5"),
    (dict(grads=[A], dtypes=[L.GRWS_F32], outs=[B], out_dtypes=[L.GRWS_BF16]), L.GRWS_E_DTYPE, b"output"),
    (dict(grads=[A], dtypes=[L.GRWS_BF16], outs=[A], out_dtypes=[L.GRWS_F32]), L.GRWS_E_INVALID, b"in place"),
    (dict(grads=[A], sizes=[-1]), L.GRWS_E_INVALID, b"negative size"),
    (dict(grads=[None]), L.GRWS_E_INVALID, b"null"), (dict(grads=[A], outs=[None]), L.GRWS_E_INVALID, b"null"),
    # memory that is shared: twice in place, an output twice, an output that
    # is another's gradient, one that begins inside its own gradient
    (dict(grads=[A, A], outs=[A, A]), L.GRWS_E_INVALID, b"overlap"),
    (dict(grads=[A, B], outs=[C, C]), L.GRWS_E_INVALID, b"overlap"),
    (dict(grads=[A, B], outs=[B, A]), L.GRWS_E_INVALID, b"overlap"),
    (dict(grads=[A], outs=[A + 32]), L.GRWS_E_INVALID, b"overlap"),
    (dict(grads=[A], outs=[A - 32]), L.GRWS_E_INVALID, b"overlap"),
    (dict(grads=[A, A + 32], sizes=[16, 4], outs=[A, A + 32]), L.GRWS_E_INVALID, b"overlap"),
    (dict(grads=[A, A + 32], sizes=[16, 4], outs=[B, A + 32]), L.GRWS_E_INVALID, b"overlap"),
    (dict(grads=[A], ws_bytes=8), L.GRWS_E_CAPACITY, b"workspace"),
    (dict(grads=[A], ws=None), L.GRWS_E_CAPACITY, b"workspace"),
])
def test_refuses(kw, status, word):
    assert _call(**kw) == status
    assert word in L.load().grws_last_error()


def test_workspace_grows_with_the_launches():
    f = L.load().grws_clip_workspace_bytes
    assert 0 < f(0) <= f(1) <= f(64) <= f(65) <= f(1000)
    assert f(1000) >= 16 * 1024 * 8  # 16 launches of up to 1,024 sums


def test_python_refusals():
    with pytest.raises(ValueError, match="no gradients"):
        grad_norm([])
    with pytest.raises(RuntimeError, match="CUDA"):
        clip_grads([torch.zeros(3)], 1.0)
    with pytest.raises(ValueError, match="negative"):
        clip_grads([torch.zeros(3)], -1.0)
    with pytest.raises(ValueError, match="negative"):
        clip_grads([torch.zeros(3)], float("nan"))
    with pytest.raises(ValueError, match="shapes"):
        clip_grads([torch.zeros(3)], 1.0, out=[torch.zeros(4)])
    with pytest.raises(TypeError, match="dense"):
        grad_norm([torch.zeros(3, 3).to_sparse()])


def test_parameters_off_the_gpu_go_to_torch():
    """Gradients that the kernels do not take, and parameters without any."""
    p = [torch.nn.Parameter(torch.ones(3, 2)), torch.nn.Parameter(torch.ones(4)), torch.nn.Parameter(torch.ones(2))]
    assert float(clip_grad_norm_(p, 1.0)) == 0.0
    p[0].grad = torch.full((3, 2), 2.0)
    p[2].grad = torch.full((2,), 1.0)
    norm = clip_grad_norm_(iter(p), 1.0)
    assert abs(float(norm) - 26.0 ** 0.5) < 1e-5
    assert abs(float(p[0].grad[0, 0]) - 2.0 / 26.0 ** 0.5) < 1e-5
    assert abs(float(clip_grad_norm_(p[0], 10.0)) - (24.0 / 26.0) ** 0.5) < 1e-5


def test_gradients_that_share_memory():
    """What helper.clip_grad_norm_ leaves to torch: views that overlap, one
    that overlaps itself, and what only might."""
    from graph_rws_amd.helper.engine import _share_memory
    buf = torch.zeros(64, 48)
    other = torch.zeros(5)
    for grads in ([buf, buf], [buf, buf.view(-1)], [buf[:40], other, buf[30:]], [buf[:, :30], buf[:, 20:]],
                  [buf.view(-1)[5:9], buf.t()], [other.expand(3, 5)], [other[:1].expand(7)],
                  [buf.as_strided((4, 8), (4, 1))], [buf, other, buf[63, 47:]]):
        assert _share_memory(grads)
        assert _share_memory(grads[::-1])
    for grads in ([], [buf], [buf.t()], [buf[:32], buf[32:]], [buf[32:], other, buf[:32]], [buf[::2], other],
                  [buf[:, ::3]], [other, torch.zeros(0), torch.zeros(())], [torch.zeros(2, 3, 4, 5).permute(3, 0, 2, 1)],
                  [buf.view(-1)[:7].bfloat16(), buf]):
        assert not _share_memory(grads)
        assert not _share_memory(grads[::-1])
