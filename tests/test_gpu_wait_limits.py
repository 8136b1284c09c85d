"""Waits inside the expert kernels that run out: no failure is made, the limit is set far below what a call's
own work takes.  The kernel gives up, records why, lets its copies and matrix products finish, gives TMEM back and returns;
the next call with the default limit is exact."""
import time

import pytest
import torch

from helpers import weight
from test_gpu_linear import BF16, close, expect, plan_of, rn

pytestmark = pytest.mark.gpu


def gives_up_and_recovers(call, reference, must_run_out):
    import mbp
    call()  # attributes and tensor maps
    torch.cuda.synchronize()
    assert mbp.device_status() == 0
    mbp.set_wait_limit(1)
    try:
        for _ in range(3):
            t0 = time.perf_counter()
            call()
            torch.cuda.synchronize()
            assert time.perf_counter() - t0 < 1.0
            code = mbp.device_status()
            assert 0 <= code <= 3
            assert code or not must_run_out
    finally:
        mbp.set_wait_limit(0)
    close(call(), *reference)
    assert mbp.device_status() == 0


@pytest.mark.parametrize("tensor_cores", [False, True])
@pytest.mark.parametrize("counts", [[2, 0, 1], [130, 3, 300]])
def test_experts(tensor_cores, counts):
    """128 stages a tile: the epilogue's first wait takes longer than a sleep of 20 us."""
    import mbp
    n, k, rows = 272, 16384, sum(counts)
    w = weight(3 * n, k, seed=1).view(3, n, k)
    p, x, plan = mbp.pack_experts(w), rn(rows, k, seed=2), plan_of(counts, rows)
    parts = [expect(x[a:a + c], w[e], "silu", None, None, None, k)
             for e, (a, c) in enumerate(zip([0, counts[0], counts[0] + counts[1]], counts)) if c]
    ref = tuple(torch.cat(t) for t in zip(*parts))
    gives_up_and_recovers(lambda: mbp.expert_linear(p, x, plan, activation="silu", tensor_cores=tensor_cores, out_dtype=BF16),
                          ref, tensor_cores)
