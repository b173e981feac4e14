"""GPU tests of nsq_linear and the experts' layer at the limits of what their
documentation allows: kept workspaces, odd edges, routers of every size,
alignments, and the launch-planning switches."""
import numpy as np
import pytest
import torch

from planejaja_b200 import _lib
from planejaja_b200 import quantize as Q
from planejaja_b200.formats import Q4_0, Q4_K, Q5_K, Q6_K, Q8_0

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    from planejaja_b200.engine import CudaEngine
    e = CudaEngine(0)
    yield e
    assert e.device_status() == 0


@pytest.mark.parametrize("t", [Q4_K, Q8_0])
def test_linear_kept_workspace_serves_smaller_calls(eng, t):
    """A workspace made for m tokens and k, used by every smaller call: with divided tasks (512 rows) and without."""
    for n, k in ((512, 1024), (4096, 512)):
        w = eng.upload(Q.synthetic_weights(n, k, t, seed=n))
        x = torch.randn(16, k, device="cuda")
        want = [eng.linear(x[:m].contiguous(), w, t, n, k) for m in range(1, 17)]
        for made_for in (9, 12, 15, 16, 40):
            ws = eng.linear_workspace(made_for, n, k)
            for m in range(1, min(made_for, 16) + 1):
                y = eng.linear(x[:m].contiguous(), w, t, n, k, workspace=ws)
                assert torch.equal(y, want[m - 1]), (made_for, m)


# ---------------------------------------------------------------- mixture of experts
def experts(eng, e, d, f, t_in, t_down, seed=0):
    from planejaja_b200.engine import MoeExperts
    w = [eng.upload(Q.synthetic_weights(e * n, k, t, seed=seed + i))
         for i, (n, k, t) in enumerate(((f, d, t_in), (f, d, t_in), (d, f, t_down)))]
    return MoeExperts(*w, e, d, f, t_in, t_down)


def test_moe_kept_workspace_serves_smaller_calls(eng):
    """One made for 17 tokens of 2 picks: groups of 16 there, of up to 8 for fewer tokens."""
    e, d, f = 8, 512, 768
    moe = experts(eng, e, d, f, Q4_K, Q4_K)
    x, wr = torch.randn(17, d, device="cuda"), torch.randn(e, d, device="cuda")
    ws = eng.moe_workspace(moe, 17, 2)
    for m, k in ((17, 2), (16, 2), (9, 1), (17, 1), (8, 2), (1, 1), (16, 1)):
        want = eng.moe_layer(moe, wr, x[:m].contiguous(), k)
        got = eng.moe_layer(moe, wr, x[:m].contiguous(), k, workspace=ws)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), (m, k)
