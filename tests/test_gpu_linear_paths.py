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


def test_out_over_an_operand_is_refused():
    """Memory that other blocks of the call still read: bias, router weights, plan, packed weights."""
    import mbp
    n, k, m = 64, 128, 6
    w = weight(4 * n, k, seed=1)
    p, pe, x = mbp.pack_c12(w[:n].contiguous()), mbp.pack_experts(w.view(4, n, k)), rn(m, k, seed=2)
    mem = torch.zeros(m * 4 * n, dtype=F32, device="cuda")
    out, low = mem[:m * n].view(m, n), mem.view(BF16)[:m * n].view(m, n)
    plan = plan_of([1, 2, 0, 3], m)
    held = mbp.ExpertPlan(mem.view(torch.int32)[:m].view(m, 1).copy_(plan.pos), plan.src,
                          mem.view(torch.int32)[m:m + 5].copy_(plan.offsets))
    wts = torch.ones(m, 1, device="cuda")
    calls = [lambda: mbp.linear(p, x, bias=mem[n:2 * n], out=out), lambda: mbp.linear(p, x, bias=mem.view(BF16)[:n], out=low),
             lambda: mbp.linear(p, x, bias=mem[m * n - 1:(m + 1) * n - 1], out=out),
             lambda: mbp.linear(p, x, out=p.units.view(-1)[:m * n * 2].view(BF16).view(m, n)),
             lambda: mbp.expert_linear(pe, x, plan, bias=mem[:4 * n].view(4, n), out=out),
             lambda: mbp.expert_linear(pe, x, held, out=out),
             lambda: mbp.expert_gather(x.float(), held, out=mem[:m * k].view(m, k)),
             lambda: mbp.expert_combine(rn(m, n, seed=3, dtype=F32), mem[:m].view(m, 1), plan, out=out),
             lambda: mbp.expert_combine(rn(m, n, seed=3, dtype=F32), wts, held, out=out),
             lambda: mbp.expert_gather_grad(rn(m, n, seed=3, dtype=F32), held, out=out),
             lambda: mbp.expert_combine_grad(rn(m, n, seed=3, dtype=F32), rn(m, n, seed=4, dtype=F32), mem[:m].view(m, 1), plan, out=out),
             lambda: mbp.expert_combine_grad(rn(m, n, seed=3, dtype=F32), rn(m, n, seed=4, dtype=F32), wts, held, out=out)]
    kept = mem.clone(), p.units.clone()
    for i, f in enumerate(calls):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was not refused")
    assert torch.equal(mem.view(torch.int32), kept[0].view(torch.int32)) and torch.equal(p.units, kept[1])
    # the neighbours of an operand are free to be written
    bias = mem[m * n:m * n + n]
    ref, bound = expect(x, w[:n], "none", bias, None, None, k)
    close(mbp.linear(p, x, bias=bias, out=out), ref, bound)
