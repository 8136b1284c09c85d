"""Paths of the epilogue kernels that the shapes of test_gpu_linear.py reach only in part (same tolerances)."""
import pytest
import torch

from helpers import weight
from test_gpu_linear import ACTS, BF16, F32, close, expect, plan_of, rn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("tiles", [1, 3, 9, 17])
def test_half_warps_of_rows_in_the_element_wise_epilogue(tiles, act):
    """An odd number of 16-row tiles leaves a warp of the tensor-core kernels 16 rows: half its lanes run the epilogue (and
    its activation's own branches), then all of them read the next group of the accumulator together."""
    import mbp
    n, k, m = 16 * tiles, 256, 70
    w = weight(2 * n, k, seed=tiles).view(2, n, k) * 8
    x, bias, res = rn(m, k, seed=1), rn(n, seed=2, dtype=F32) * 4, rn(m, n, seed=3, dtype=F32)
    ref, bound = expect(x, w[0], act, bias, None, res, k)
    out = torch.full((m, n + 5), 7.0, device="cuda")
    mbp.linear(mbp.pack_c12(w[0].contiguous()), x, bias=bias, activation=act, residual=res, out=out[:, 3:n + 3])
    close(out[:, 3:n + 3], ref, bound)
    assert bool((out[:, :3] == 7.0).all()) and bool((out[:, n + 3:] == 7.0).all())
    eb = torch.stack([bias, bias.flip(0)])
    got = mbp.expert_linear(mbp.pack_experts(w), x, plan_of([41, 29], m), bias=eb, activation=act, residual=res,
                            out_dtype=F32, tensor_cores=True)
    close(got[:41], ref[:41], bound[:41])
    close(got[41:], *expect(x[41:], w[1], act, eb[1], None, res[41:], k))
    assert mbp.device_status() == 0
