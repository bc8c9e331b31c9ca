"""Host side of log_probs: refusals before any launch, and workspace sizes
(CPU tier: nothing here touches a GPU)."""
import ctypes

import pytest
import torch

from graph_rws_amd.core import _lib as L
from graph_rws_amd.layers import linear_log_probs, log_probs

P = 1 << 20  # never read


def _fwd(dtype=0, ld=100, rows=4, classes=100, k=1, top=0, temperature=1.0, logits=P, index=P, logp=P, entropy=P,
         top_logp=P, top_index=P, ws=None, ws_bytes=0):
    return L.load().grws_log_probs_fwd(logits, dtype, ld, rows, classes, index, 1, k, top, temperature, logp, entropy,
                                       None, top_logp, top_index, ws, ws_bytes, None)


def _bwd(dtype=0, ld=100, rows=4, classes=100, k=1, temperature=1.0, saved=P, entropy=P, grad=P, ldg=100):
    return L.load().grws_log_probs_bwd(P, dtype, ld, rows, classes, P, 1, k, temperature, saved, entropy, P, P, grad,
                                       ldg, None)


@pytest.mark.parametrize("call,kw,status,word", [
    (_fwd, dict(dtype=3), L.GRWS_E_DTYPE, b"dtype"), (_fwd, dict(ld=99), L.GRWS_E_INVALID, b"sizes"),
    (_fwd, dict(rows=-1), L.GRWS_E_INVALID, b"sizes"), (_fwd, dict(classes=0), L.GRWS_E_INVALID, b"sizes"),
    (_fwd, dict(classes=2 ** 31, ld=2 ** 31), L.GRWS_E_INVALID, b"sizes"),
    (_fwd, dict(k=0), L.GRWS_E_INVALID, b"given"), (_fwd, dict(k=1025), L.GRWS_E_INVALID, b"given"),
    (_fwd, dict(top=-1), L.GRWS_E_INVALID, b"top"), (_fwd, dict(top=101), L.GRWS_E_INVALID, b"top"),
    (_fwd, dict(top=1025, classes=2000, ld=2000), L.GRWS_E_INVALID, b"top"),
    (_fwd, dict(temperature=0.0), L.GRWS_E_INVALID, b"temperature"),
    (_fwd, dict(temperature=float("nan")), L.GRWS_E_INVALID, b"temperature"),
    (_fwd, dict(temperature=1e-45), L.GRWS_E_INVALID, b"temperature"),
    (_fwd, dict(logits=None), L.GRWS_E_INVALID, b"null"), (_fwd, dict(index=None), L.GRWS_E_INVALID, b"null"),
    (_fwd, dict(logp=None), L.GRWS_E_INVALID, b"null"), (_fwd, dict(entropy=None), L.GRWS_E_INVALID, b"null"),
    (_fwd, dict(top=2, top_index=None), L.GRWS_E_INVALID, b"null"),
    (_fwd, dict(rows=1, classes=100000, ld=100000), L.GRWS_E_CAPACITY, b"workspace"),
    (_bwd, dict(dtype=-1), L.GRWS_E_DTYPE, b"dtype"), (_bwd, dict(ldg=99), L.GRWS_E_INVALID, b"sizes"),
    (_bwd, dict(saved=None), L.GRWS_E_INVALID, b"null"), (_bwd, dict(grad=None), L.GRWS_E_INVALID, b"null"),
    (_bwd, dict(temperature=-1.0), L.GRWS_E_INVALID, b"temperature"),
])
def test_refuses(call, kw, status, word):
    assert call(**kw) == status
    assert word in L.load().grws_last_error()


def test_no_rows_is_nothing():
    assert _fwd(rows=0, logits=None, index=None, logp=None, entropy=None) == L.GRWS_OK
    assert _bwd(rows=0, saved=None, entropy=None, grad=None) == L.GRWS_OK


def test_workspace():
    f = L.load().grws_log_probs_workspace_bytes
    assert f(0, 1000, 0) == f(-1, 10, 0) == f(5, 0, 0) == f(5, 10, -1) == 0
    assert f(1024, 100000, 64) == 0  # a work-group a row
    assert f(1, 1000, 16) == 0  # a wave a row
    assert 0 < f(1, 131072, 0) < f(1, 131072, 8) < 1 << 16
    assert f(1, 2 ** 30, 1024) < 64 << 20


def test_python_refusals():
    z, i = torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        log_probs(z, i)


# ---------------------------------------------------------------------------
# of a classifier whose logits are not kept
# ---------------------------------------------------------------------------
def _head(**kw):
    v = dict(hidden=P, weight=P, bias=None, rows=None, labels=P, teacher_index=None, teacher_logits=None,
             ld_hidden=64, ld_weight=64, hidden_rows=100, n=100, width=64, classes=1000, dtype=L.GRWS_BF16, k=0,
             index_is_i64=0, temperature=1.5)
    v.update(kw)
    return L.HeadView(*(v[name] for name, _ in L.HeadView._fields_))


def _head_fwd(head, top=0, logp=P, saved=P, top_index=P, ws_bytes=1 << 40):
    return L.load().grws_head_log_probs_fwd(ctypes.byref(head), top, logp, P, saved, P, top_index, P, ws_bytes, None)


def _head_bwd(head, saved=P, logp=P, ld=64, ws_bytes=1 << 40):
    return L.load().grws_head_log_probs_bwd(ctypes.byref(head), saved, logp, P, P, P, P, ld, P, 64, P, P, ws_bytes,
                                            None)


LISTS = dict(labels=None, teacher_index=P, k=4)


@pytest.mark.parametrize("kw,call,status,word", [
    (dict(dtype=7), {}, L.GRWS_E_DTYPE, b"dtype"), (dict(n=-1), {}, L.GRWS_E_INVALID, b"row count"),
    (dict(labels=None), {}, L.GRWS_E_INVALID, b"classes"), (dict(k=4), {}, L.GRWS_E_INVALID, b"classes"),
    (dict(LISTS, labels=P), {}, L.GRWS_E_INVALID, b"classes"),
    (dict(temperature=0.0), {}, L.GRWS_E_INVALID, b"temperature"),
    (dict(temperature=1e-42), {}, L.GRWS_E_INVALID, b"temperature"),
    (dict(weight=None), {}, L.GRWS_E_INVALID, b"null"),
    (dict(k=1025, labels=None, teacher_index=P), {}, L.GRWS_E_INVALID, b"1024"),
    ({}, dict(top=-1), L.GRWS_E_INVALID, b"top"), ({}, dict(top=1001), L.GRWS_E_INVALID, b"top"),
    (dict(classes=5000), dict(top=1025), L.GRWS_E_INVALID, b"top"),
    ({}, dict(logp=None), L.GRWS_E_INVALID, b"null"), ({}, dict(saved=None), L.GRWS_E_INVALID, b"null"),
    ({}, dict(top=2, top_index=None), L.GRWS_E_INVALID, b"null"),
])
def test_head_refuses(kw, call, status, word):
    assert _head_fwd(_head(**kw), **call) == status
    assert word in L.load().grws_last_error()


def test_head_workspaces():
    lib = L.load()
    for kw in ({}, LISTS):
        h = _head(**kw)
        for top in (0, 8):
            need = lib.grws_head_log_probs_fwd_workspace_bytes(ctypes.byref(h), top)
            assert need > 0 and _head_fwd(h, top=top, ws_bytes=need - 1) == L.GRWS_E_CAPACITY
        need = lib.grws_head_log_probs_bwd_workspace_bytes(ctypes.byref(h))
        assert need > 0 and _head_bwd(h, ws_bytes=need - 1) == L.GRWS_E_CAPACITY
        assert _head_bwd(h, ld=63) == L.GRWS_E_INVALID and _head_bwd(h, saved=None) == L.GRWS_E_INVALID
        assert _head_bwd(h, logp=None) == L.GRWS_E_INVALID
    assert lib.grws_head_log_probs_fwd_workspace_bytes(ctypes.byref(_head(dtype=9)), 0) == 0
    # kept logits: a block of the rows
    for n, classes in ((8192, 131072), (30000, 1000000), (1, 2000000)):
        h = _head(n=n, hidden_rows=n, classes=classes)
        assert lib.grws_head_log_probs_fwd_workspace_bytes(ctypes.byref(h), 8) < 3 << 29
        assert lib.grws_head_log_probs_fwd_workspace_bytes(ctypes.byref(h), 0) < 1 << 30
    assert _head_fwd(_head(n=0)) == L.GRWS_OK


def test_linear_python_refusals():
    h, w, i = torch.zeros(3, 5), torch.zeros(7, 5), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        linear_log_probs(h, w, i)


def test_second_derivative_is_refused_whatever_the_strides(monkeypatch):
    """Logits whose columns are not next to each other, or whose rows are one,
    are copied for the kernels: a second derivative through them is an error as
    it is through others, beside a term of the loss that has a gradient."""
    from graph_rws_amd.core import ops
    from graph_rws_amd.layers import logp as module

    def fwd(x, index, temperature, top, save):
        assert x.stride(1) == 1 and index.is_contiguous()
        lp = torch.log_softmax(x / temperature, 1)
        return lp.gather(1, index[:, None])[:, 0], -(lp.exp() * lp).sum(1), lp[:, :2].contiguous(), None, None

    def bwd(x, index, temperature, saved, entropy, dlogp, dentropy):
        assert x.stride(1) == 1
        g = -torch.softmax(x / temperature, 1) * dlogp[:, None]
        return g.scatter_add(1, index[:, None], dlogp[:, None]) / temperature

    monkeypatch.setattr(ops, "check_log_probs", lambda *a: None)
    monkeypatch.setattr(ops, "log_probs_fwd", fwd)
    monkeypatch.setattr(ops, "log_probs_bwd", bwd)
    index = torch.tensor([0, 2, 4, 1])
    for shape, view in (((4, 5), lambda t: t), ((5, 4), lambda t: t.t()), ((4, 10), lambda t: t[:, ::2]),
                        ((1, 5), lambda t: t.expand(4, 5)), ((8,), lambda t: t.as_strided((4, 5), (1, 1)))):
        leaf = torch.randn(shape, requires_grad=True)
        first, = torch.autograd.grad(module.log_probs(view(leaf), index).logp.sum(), leaf)
        twin = leaf.detach().clone().requires_grad_()
        want, = torch.autograd.grad(torch.log_softmax(view(twin), 1).gather(1, index[:, None]).sum(), twin)
        assert torch.allclose(first, want, atol=1e-6)
        g, = torch.autograd.grad(module.log_probs(view(leaf), index).logp.sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="second derivative"):
            (leaf.square().sum() + g.square().sum()).backward()
