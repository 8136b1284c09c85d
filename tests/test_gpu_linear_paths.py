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


@pytest.mark.parametrize("tensor_cores", [False, True])
@pytest.mark.parametrize("borders,owners", [([0, 5, 1000, 1000, 2000], {0: (0, 5), 1: (5, 20)}),
                                            ([-50, 5, 10, 8, 20], {0: (0, 5), 1: (5, 8), 3: (10, 20)}),
                                            ([20, 20, 20, 20, 20], {}), ([7, 7, 3, 9, 2 ** 31 - 1], {2: (3, 9), 3: (9, 20)})])
def test_borders_out_of_range_leave_the_neighbours_alone(tensor_cores, borders, owners):
    """Clamped to the rows: rows of a single owner hold its product, rows outside the tensors are neither read nor written.
    (Descending borders give a row two owners; such rows hold one of their products.)"""
    import mbp
    w = weight(4 * 32, 64, seed=1).view(4, 32, 64)
    p = mbp.pack_experts(w)
    around = torch.full((60, 64), float("nan"), dtype=BF16, device="cuda")
    x = around[20:40]
    x.copy_(rn(20, 64, seed=2))
    src = torch.arange(20, dtype=torch.int32, device="cuda")
    plan = mbp.ExpertPlan(src.view(20, 1), src, torch.tensor(borders, dtype=torch.int32, device="cuda"))
    buf = torch.full((60, 40), 7.0, device="cuda")
    mbp.expert_linear(p, x, plan, out=buf[20:40, 4:36], tensor_cores=tensor_cores)
    for e, (a, b) in owners.items():
        close(buf[20 + a:20 + b, 4:36], *expect(x[a:b], w[e], "none", None, None, None, 64))
    assert not bool(torch.isnan(buf).any())
    if not owners:
        assert bool((buf == 7.0).all())
    buf[20:40, 4:36] = 7.0
    assert bool((buf == 7.0).all())
    assert mbp.device_status() == 0


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [5, 70])
def test_each_activation_within_its_own_bound(act, m):
    """Arguments from -60 to 60, FP32.  none and relu are exact, relu2 is one rounding.  gelu: the argument of erfc carries
    two roundings, each of which moves erfc(a) by 2 a^2 = z^2 times as much, and 16 steps for erfc itself and the products;
    silu and sigmoid 16 steps; gelu_tanh those and the roundings of its argument u = 1.6 (z + 0.045 z^3), four at most.
    Where the exponential or erfc is subnormal, 4 steps of 2^-149, scaled by |z|."""
    import mbp
    z = torch.linspace(-60, 60, 512, device="cuda")
    p = mbp.pack_c12(weight(512, 64, seed=7))
    got = mbp.linear(p, torch.zeros(m, 64, dtype=BF16, device="cuda"), bias=z, activation=act, out_dtype=F32)
    zd = z.double()
    ref, step = act64(zd, act), 2.0 ** -23
    u = 1.6 * (zd.abs() + 0.045 * zd.abs() ** 3)
    rel = {"none": 0.0, "relu": 0.0, "relu2": step / 2, "gelu": (zd ** 2 + 16) * step, "gelu_tanh": (2 * u + 16) * step}.get(act, 16 * step)
    bound = rel * ref.abs() + (0 if act in ("none", "relu") else 2.0 ** -149 * 4 * (zd.abs() + 1))
    err = (got.double() - ref).abs()
    assert bool((err <= bound).all()), float((err - bound).max())


@pytest.mark.parametrize("m", [1, 16, 300])
def test_as_many_experts_as_the_router_has(m):
    """256 experts of 1536 x 6144, 8 for each token: the router's own widths, on both kernels."""
    import mbp
    e, n, k = 256, 1536, 6144
    base = weight(n, k, seed=5)
    scale = 2.0 ** (torch.arange(e, device="cuda") % 5 - 2)  # exact in BF16, so that the experts differ
    w = base.unsqueeze(0) * scale.view(e, 1, 1).to(BF16)
    p = mbp.pack_experts(w)
    g = torch.Generator(device="cuda").manual_seed(m)
    ids = torch.randn(m, e, generator=g, device="cuda").topk(8, dim=1).indices.to(torch.int32)
    plan = mbp.expert_sort(ids, e)
    x = rn(m, k, seed=m)
    xs = mbp.expert_gather(x, plan)
    owner = ids.reshape(-1)[plan.src.long()].long()
    ref, bound = expect(xs, base, "none", None, None, None, k)
    ref, bound = ref * scale[owner].view(-1, 1), bound * scale[owner].view(-1, 1)
    for kw in ({}, {"tensor_cores": False}, {"tensor_cores": True}):
        close(mbp.expert_linear(p, xs, plan, **kw), ref, bound)
    assert mbp.device_status() == 0
