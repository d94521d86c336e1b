"""Calls of the serving operators beside those of test_serving_gpu.py, whose references and tolerances they use."""
import math

import pytest
import torch

from test_serving_gpu import HALF, Paged, check_attn, check_verify, drafts, gen, verify_ref, within  # noqa: F401

pytestmark = pytest.mark.gpu

bf16, f32, f64, i32 = torch.bfloat16, torch.float32, torch.float64, torch.int32


# ----------------------------------------------------------------------------- tables
@pytest.mark.parametrize("max_len", [1, 100000])
def test_attn_shared_table_row(dev, max_len):
    """Requests that share one page list: an expanded row, and rows that overlap, against the same rows laid out."""
    from grove_amd import ops
    c = Paged(dev, [200], 2, 64, 16, seed=11)
    q = torch.randn(7, 4, 64, generator=gen(12)).to(bf16).to(dev)
    cu, kv_len = torch.tensor([0, 2, 3, 7], dtype=i32, device=dev), torch.tensor([200, 64, 131], dtype=i32, device=dev)
    wide = torch.cat([c.table[0], c.table[0, :4]])
    for table in (c.table.expand(3, -1), wide.as_strided((3, c.table.shape[1]), (2, 1))):
        a, b = (ops.kv4_attn(q, c.cache, t, kv_len, cu, 4, 0.125, max_len=max_len) for t in (table, table.contiguous()))
        assert torch.equal(a, b) and a.isfinite().all() and not (a == 0).all(1).any()
