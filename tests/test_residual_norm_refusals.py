"""Calls of the norms around a branch that have no right answer: refused before anything is launched."""
import pytest
import torch

from .test_residual_norm import EPS, host_ops, inputs


def test_weights_gradients_that_share_memory():
    """Both halves of the sum would write the same place."""
    ops, v = host_ops(), inputs(5, 64)
    h, z, stats = ops.residual_norm(v["x"], v["y"], v["w_post"], v["w_pre"], EPS)
    n, both = len(ops.calls), torch.empty(128, dtype=torch.bfloat16)
    for a, b in ((both[:64], both[:64]), (both[:64], both[32:96]), (both[64:], both[8:72])):
        with pytest.raises(ValueError, match="memory of their own"):
            ops.residual_norm_bwd(v["dh"], v["dz"], v["y"], h, stats, v["w_post"], v["w_pre"], a, b)
    assert len(ops.calls) == n
    ops.residual_norm_bwd(v["dh"], v["dz"], v["y"], h, stats, v["w_post"], v["w_pre"], both[:64], both[64:])   # one behind the other is fine
    ops.residual_norm_bwd(v["dh"], v["dz"], v["y"], h, stats, v["w_post"], v["w_pre"], both[64:], both[:64])
    assert len(ops.calls) == n + 2


def test_more_rows_than_the_kernels_count():
    """2^31 rows of 8 are 34 GB: their number arrived as none, and nothing was written."""
    ops = host_ops()
    y, w = torch.empty(1 << 31, 8, dtype=torch.bfloat16, device="meta"), torch.empty(8, dtype=torch.bfloat16, device="meta")
    with pytest.raises(ValueError, match="more than the kernels count"):
        ops.residual_norm(y, y, w, w, EPS)
    s = torch.empty(1 << 31, device="meta")
    with pytest.raises(ValueError, match="more than the kernels count"):
        ops.residual_norm_bwd(y, y, y, y, (s, s), w, w, torch.empty_like(w), torch.empty_like(w))
    assert not ops.calls
