"""Paths of the epilogue kernels that the shapes of test_gpu_linear.py reach only in part (same tolerances)."""
import pytest
import torch

from helpers import weight
from test_gpu_linear import ACTS, BF16, F32, act64, close, expect, plan_of, rn

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


@pytest.mark.parametrize("act", ["silu", "sigmoid", "gelu_tanh"])
def test_activations_where_the_exponential_leaves_the_range(act):
    """Arguments whose e^|u| passes 2^126 and then 2^128, whose results are still above the smallest FP32 numbers.

    Bound: 16 steps of the value as everywhere (for gelu_tanh the argument's own rounding too), and where e^-|u| or the result is
    subnormal two steps of 2^-149 for the exponential and two for the quotient, which silu and gelu_tanh scale by |z|."""
    import mbp
    n, k = 512, 64
    z = torch.linspace(-11.0, -9.0, n) if act == "gelu_tanh" else torch.linspace(-104.0, -80.0, n)
    bias = z.cuda()
    ref = act64(bias.double(), act)
    zz = bias.double().abs()
    u = 1.6 * (zz + 0.045 * zz ** 3) if act == "gelu_tanh" else zz
    rel = 16 * 2.0 ** -23 + (2.0 ** -22 * u if act == "gelu_tanh" else 0)
    bound = rel * ref.abs() + 2.0 ** -149 * 4 * (1 if act == "sigmoid" else zz + 1)
    w = weight(2 * n, k, seed=1).view(2, n, k)
    x = torch.zeros(70, k, dtype=BF16, device="cuda")
    p, pe = mbp.pack_c12(w[0].contiguous()), mbp.pack_experts(w)
    eb = torch.stack([bias, bias])
    got = [mbp.linear(p, x[:m], bias=bias, activation=act, out_dtype=F32) for m in (5, 70)]
    got += [mbp.expert_linear(pe, x, plan_of([30, 40], 70), bias=eb, activation=act, out_dtype=F32, tensor_cores=tc)
            for tc in (False, True)]
    for y in got:
        err = (y.double() - ref).abs()
        assert bool((err <= bound).all()), float((err / bound).max())
