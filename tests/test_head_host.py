"""Host side of the fused classifier and of top_logits: refusals before any
launch, and workspace sizes (CPU tier: nothing here touches a GPU)."""
import ctypes

import pytest
import torch

from graph_rws_amd.core import _lib as L
from graph_rws_amd.core import top_logits
from graph_rws_amd.layers import linear_cross_entropy, linear_distill


def _head(**kw):
    at = 1 << 20  # never read
    v = dict(hidden=at, weight=at, bias=None, rows=None, labels=at, teacher_index=None, teacher_logits=None,
             ld_hidden=64, ld_weight=64, hidden_rows=100, n=100, width=64, classes=1000, dtype=L.GRWS_BF16, k=0,
             index_is_i64=0, temperature=1.0)
    v.update(kw)
    return L.HeadView(*(v[name] for name, _ in L.HeadView._fields_))


def _fwd(head):
    p = ctypes.c_void_p(1 << 20)
    return L.load().grws_head_fwd(ctypes.byref(head), p, p, p, p, p, p, p, 1 << 40, None)


@pytest.mark.parametrize("kw,status,word", [
    (dict(dtype=7), L.GRWS_E_DTYPE, b"dtype"), (dict(n=-1), L.GRWS_E_INVALID, b"row count"),
    (dict(hidden_rows=-1), L.GRWS_E_INVALID, b"row count"), (dict(width=0), L.GRWS_E_INVALID, b"width"),
    (dict(width=65537, ld_hidden=65537, ld_weight=65537), L.GRWS_E_INVALID, b"width"),
    (dict(classes=0), L.GRWS_E_INVALID, b"class"), (dict(classes=2 ** 31), L.GRWS_E_INVALID, b"class"),
    (dict(ld_hidden=63), L.GRWS_E_INVALID, b"leading"), (dict(ld_weight=2 ** 21 + 1), L.GRWS_E_INVALID, b"leading"),
    (dict(hidden=None), L.GRWS_E_INVALID, b"null"), (dict(weight=None), L.GRWS_E_INVALID, b"null"),
    (dict(labels=None), L.GRWS_E_INVALID, b"labels"), (dict(temperature=2.0), L.GRWS_E_INVALID, b"temperature"),
    (dict(temperature=0.0), L.GRWS_E_INVALID, b"temperature"),
    (dict(temperature=float("nan")), L.GRWS_E_INVALID, b"temperature"),
    (dict(k=1025), L.GRWS_E_INVALID, b"1024"), (dict(k=4), L.GRWS_E_INVALID, b"teacher"),
    (dict(k=4, labels=None, teacher_index=8), L.GRWS_E_INVALID, b"teacher"),
])
def test_head_refuses_bad_descriptions(kw, status, word):
    assert _fwd(_head(**kw)) == status
    assert word in L.load().grws_last_error()


def test_head_null_and_small_workspace():
    lib = L.load()
    p = ctypes.c_void_p(1 << 20)
    assert lib.grws_head_fwd(None, p, p, p, p, p, p, p, 0, None) == L.GRWS_E_INVALID
    h = _head()
    assert lib.grws_head_fwd(ctypes.byref(h), p, p, p, None, None, p, p, 1 << 40, None) == L.GRWS_E_INVALID
    need = lib.grws_head_fwd_workspace_bytes(ctypes.byref(h))
    assert need > 0
    assert lib.grws_head_fwd(ctypes.byref(h), p, p, p, p, p, p, p, need - 1, None) == L.GRWS_E_CAPACITY
    need = lib.grws_head_bwd_workspace_bytes(ctypes.byref(h))
    assert lib.grws_head_bwd(ctypes.byref(h), p, p, p, p, p, 0, p, 64, p, 64, p, p, need - 1, None) == \
        L.GRWS_E_CAPACITY
    assert lib.grws_head_bwd(ctypes.byref(h), p, p, p, p, p, 0, p, 63, p, 64, p, p, need, None) == L.GRWS_E_INVALID


@pytest.mark.parametrize("dtype", [L.GRWS_F32, L.GRWS_F16, L.GRWS_BF16])
def test_head_workspaces_are_bounded(dtype):
    """The scratch does not grow with rows x classes: pieces of the classes."""
    lib = L.load()
    most = 0
    for n, width, classes in [(1, 16, 7), (100, 64, 1000), (8192, 4096, 131072), (30000, 1024, 1000000),
                              (1, 4096, 2000000)]:
        h = _head(n=n, hidden_rows=n, width=width, ld_hidden=width, ld_weight=width, classes=classes, dtype=dtype)
        fwd = lib.grws_head_fwd_workspace_bytes(ctypes.byref(h))
        bwd = lib.grws_head_bwd_workspace_bytes(ctypes.byref(h))
        assert 0 < fwd and 0 < bwd
        most = max(most, bwd)
    assert most < 2 << 30  # 30,000 x 1,000,000 logits alone are 60 GB in 16 bits


def test_top_logits_refuses_bad_arguments():
    lib = L.load()
    p = ctypes.c_void_p(1 << 20)
    for dtype, ld, rows, classes, k, status in [(9, 10, 1, 10, 1, L.GRWS_E_DTYPE), (0, 9, 1, 10, 1, L.GRWS_E_INVALID),
                                                (0, 10, -1, 10, 1, L.GRWS_E_INVALID), (0, 10, 1, 0, 1, L.GRWS_E_INVALID),
                                                (0, 10, 1, 10, 0, L.GRWS_E_INVALID), (0, 10, 1, 10, 11, L.GRWS_E_INVALID),
                                                (0, 4096, 1, 4096, 1025, L.GRWS_E_INVALID)]:
        assert lib.grws_top_logits(p, dtype, ld, rows, classes, k, p, p, p, 1 << 30, None) == status
    assert lib.grws_top_logits(None, 0, 10, 1, 10, 1, p, p, p, 1 << 30, None) == L.GRWS_E_INVALID
    need = lib.grws_top_logits_workspace_bytes(1, 131072, 8)
    assert need > 0
    assert lib.grws_top_logits(p, 0, 131072, 1, 131072, 8, p, p, p, need - 1, None) == L.GRWS_E_CAPACITY
    assert lib.grws_top_logits(p, 0, 10, 0, 10, 1, p, p, None, 0, None) == L.GRWS_OK  # no rows, no launch


def test_host_tensors_are_refused():
    h, w, y = torch.zeros(4, 8), torch.zeros(9, 8), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: linear_cross_entropy(h, w, y),
                 lambda: linear_distill(h, w, torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2)),
                 lambda: top_logits(h, 2)):
        with pytest.raises(RuntimeError):
            call()


def test_products_use_no_scratch(tmp_path):
    """The products stage their operands by direct loads into LDS and fill the
    registers: none of them may spill."""
    from test_kernel_resources import _kernel_metadata
    kernels = {k: v for k, v in _kernel_metadata(tmp_path).items()
               if any(x in k for x in ("head_stats", "head_grad", "head_dweight", "head_dhidden"))}
    assert len(kernels) >= 16
    for k, v in kernels.items():
        assert v.get("private_segment_fixed_size", 0) == 0 and v.get("vgpr_spill_count", 0) == 0, f"{k}: {v}"
        assert v["vgpr_count"] <= 256, f"{k} leaves fewer than two waves per SIMD: {v}"


@pytest.mark.parametrize("dtype", [L.GRWS_F32, L.GRWS_F16, L.GRWS_BF16])
@pytest.mark.parametrize("k", [0, 32])
def test_both_workspaces_are_bounded_in_rows_and_classes(dtype, k):
    """What grows with rows x classes is taken in blocks of rows and pieces of
    classes: 1 GiB of G, 1 of packed rows, half of statistics, 0.25 of packed
    weight, 0.27 of runs at most; beyond it the scratch grows with the hidden
    rows (their f32 sums) and with nothing else."""
    lib = L.load()
    for n, width, classes in [(100, 64, 1000), (8192, 4096, 131072), (30000, 1024, 1000000), (1, 4096, 2000000),
                              (2449029, 100, 47), (2449029, 256, 100003), (1600000, 256, 131072), (111059956, 128, 172),
                              (50000, 65536, 50000), (300, 65536, 2000000000), (20000000, 8, 1000)]:
        h = _head(n=n, hidden_rows=n, width=width, ld_hidden=width, ld_weight=width, classes=classes, dtype=dtype)
        if k:
            h = _head(n=n, hidden_rows=n, width=width, ld_hidden=width, ld_weight=width, classes=classes, dtype=dtype,
                      k=k, labels=None, teacher_index=8, teacher_logits=8)
        padded = (width + 63) // 64 * 64
        # 256 rows are the least, and a row has a loss of its own in the join
        fwd = 7 << 28 if 8 * classes // 64 * 256 < 1 << 29 else (5 << 28) + 8 * classes // 64 * 256 + (1 << 20)
        assert lib.grws_head_fwd_workspace_bytes(ctypes.byref(h)) <= fwd + 8 * n
        assert lib.grws_head_bwd_workspace_bytes(ctypes.byref(h)) <= (4 << 30) + n * (4 + 4 * padded)


def _plan(backward, **kw):
    out = (ctypes.c_int64 * 10)()
    assert L.load().grws_head_plan(ctypes.byref(_head(**kw)), backward, out) == L.GRWS_OK
    return list(out)


def test_blocks_of_rows_cover_the_rows():
    for n in (1, 128, 129, 300, 100000, 5000001, 2 ** 31 - 1):
        for classes in (1, 47, 5000, 10 ** 6):
            for backward in (0, 1):
                blocks, rows, pieces, some = _plan(backward, n=n, hidden_rows=n, classes=classes)[:4]
                assert (blocks - 1) * rows < n <= blocks * rows and (blocks == 1 or rows % 256 == 0)
                assert (pieces - 1) * some < classes <= pieces * some and some % 128 == 0
                assert rows <= 1 << 20
    lib = L.load()
    out = (ctypes.c_int64 * 10)()
    assert lib.grws_head_plan(ctypes.byref(_head(n=0)), 0, out) == L.GRWS_E_INVALID
    assert lib.grws_head_plan(ctypes.byref(_head()), 0, None) == L.GRWS_E_INVALID
