"""core.top_logits over more rows than one launch takes (2^32 threads at 256 a
row), against a stable sort: equal."""
import pytest
import torch

from graph_rws_amd.core import top_logits

pytestmark = pytest.mark.gpu


# a wave a row (k up to 16), and a work-group a row
@pytest.mark.parametrize("rows,classes,k", [((1 << 23) + 5, 5, 3), ((1 << 24) + 3, 18, 17)])
def test_many_rows(cuda_device, rows, classes, k):
    print(f"case top {rows}x{classes} k={k}", flush=True)
    x = torch.randn(rows, classes, device=cuda_device).bfloat16()
    values, index = top_logits(x, k)
    for r in range(0, rows, 1 << 22):
        v, i = torch.sort(x[r:r + (1 << 22)], dim=1, descending=True, stable=True)
        assert torch.equal(index[r:r + (1 << 22)].long(), i[:, :k])
        assert torch.equal(values[r:r + (1 << 22)], v[:, :k])
