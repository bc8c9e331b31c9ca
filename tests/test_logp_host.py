"""Host side of log_probs: refusals before any launch, and workspace sizes
(CPU tier: nothing here touches a GPU)."""
import pytest
import torch

from graph_rws_amd.core import _lib as L
from graph_rws_amd.layers import log_probs

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
