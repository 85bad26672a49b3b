"""Large batches of grouped products and the router on an MI355X."""
import numpy as np
import pytest

import expert_model as M
from cllm_inference_amd import synth as S

pytestmark = pytest.mark.gpu


def _cu(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def test_more_entries_than_their_own_rows_would_allow(gpu, orc):
    """140000 rows of 32 experts each: 4.5 million entries, whose operand would pass 4 GiB if each had a row."""
    import torch
    rows, k, n, experts = 140000, 64, 3, 32
    qt = S.Q8_0
    w = S.make_weight(qt, experts * n, k, 1)
    x = S.make_activation(rows, k, 2)
    ids = torch.arange(experts, dtype=torch.int32, device="cuda").repeat(rows)
    g = gpu.group_rows_dev(ids, experts)
    y = gpu.moe_matmul_dev(_cu(x), _cu(w), qt, n, g, per_row=experts).view(rows, experts, n)
    at = np.concatenate([np.arange(5), np.random.default_rng(3).integers(0, rows, 200), np.arange(rows - 5, rows)])
    values, mags = M.expert_values(w, qt, experts, n, k)
    xr = M.q8_values(orc, x[at])
    got = y[torch.from_numpy(at).cuda()].cpu().numpy()
    for e in range(experts):
        assert (np.abs(got[:, e] - xr @ values[e].T) <= M.product_bound(mags[e], xr, k)).all()
