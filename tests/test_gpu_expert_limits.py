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


@pytest.mark.parametrize("adapters,mats,rank,k", [(4, 3, 16, 4096), (5, 1, 32, 4096), (3, 2, 12, 1000)])
def test_one_adapter_workspace_for_batches_of_all_sizes(gpu, adapters, mats, rank, k):
    """The workspace of the largest batch takes the smaller ones, and no batch writes behind its own size."""
    import ctypes

    import torch
    lib = gpu.load_library()
    rng = np.random.default_rng(adapters)
    most, out = 5500, 24
    x = _cu(rng.standard_normal((most, k)).astype(np.float32))
    a = [_cu((rng.standard_normal((adapters, rank, k)) / np.sqrt(k)).astype(np.float16)) for _ in range(mats)]
    b = [_cu(rng.standard_normal((adapters, out, rank)).astype(np.float16)) for _ in range(mats)]
    ids = _cu(rng.integers(0, adapters, most).astype(np.int32))
    size = lambda n: lib.cllm_hip_lora_ws_bytes(k, mats, adapters, rank, n)  # noqa: E731
    whole = torch.empty(size(most) + 4096, dtype=torch.uint8, device="cuda")
    ptrs = ctypes.c_void_p * mats
    for n in (1, 15, 333, 720, 1040, 2048, 2272, 3199, 3200, 4097, 5000, 5407, 5408, 5500):
        g = gpu.group_rows_dev(ids[:n], adapters)
        want = gpu.lora_dev(x[:n], a, b, g)
        ys = [torch.empty((n, out), device="cuda") for _ in range(mats)]
        whole.fill_(0x5A)
        # (once with the room of the largest batch, once with no more than its own)
        for room in (size(most), size(n)):
            rc = lib.cllm_hip_lora_dev(1, k, mats, ptrs(*[t.data_ptr() for t in a]), ptrs(*[t.data_ptr() for t in b]),
                                       (ctypes.c_int * mats)(*[out] * mats), adapters, rank, None, None, x.data_ptr(), n,
                                       g.offsets.data_ptr(), g.order.data_ptr(), None,
                                       ptrs(*[t.data_ptr() for t in ys]), whole.data_ptr(), room,
                                       torch.cuda.current_stream().cuda_stream)
            assert rc == 0, (n, lib.cllm_hip_last_error())
            assert all(torch.equal(y, w) for y, w in zip(ys, want)), n
        assert (whole[size(n):] == 0x5A).all(), n


def test_more_rows_than_a_grid_has_threads_for(gpu):
    """2^26 + 5 rows of two experts: a wave each would be 2^32 threads and more."""
    import torch
    rows = (1 << 26) + 5
    z = torch.zeros((rows, 2), device="cuda")
    z[1::2, 1] = 1.0
    z[-1] = torch.tensor([3.0, -3.0])
    print("route", rows, flush=True)
    r = gpu.moe_route_dev(z, 1, normalise=True)
    ids = r.ids.view(-1)
    want = (z[:, 1] > z[:, 0]).to(torch.int32)
    assert torch.equal(ids, want) and bool((r.weights == 1).all())
    assert r.offsets.tolist() == [0, int((want == 0).sum()), rows]
    order = torch.cat([torch.nonzero(want == 0).view(-1), torch.nonzero(want == 1).view(-1)]).to(torch.int32)
    assert torch.equal(r.order, order)


@pytest.mark.parametrize("experts,top_k", [(8, 1), (8, 2), (32, 4), (64, 8), (256, 8), (256, 32), (512, 8), (1024, 8)])
@pytest.mark.parametrize("bias", [False, True])
def test_a_row_is_routed_alike_in_batches_of_any_size(gpu, experts, top_k, bias):
    """One launch or two, with a wave's rows in turn or apart: a row's choice is the same, and so is the order."""
    import torch
    gen = torch.Generator("cuda").manual_seed(experts + top_k)
    z = torch.randn((65, experts), device="cuda", generator=gen)
    b = torch.randn(experts, device="cuda", generator=gen) * 0.1 if bias else None
    whole = gpu.moe_route_dev(z, top_k, bias=b, sigmoid=bias)
    for m in (1, 2, 3, 4, 5, 7, 8, 9, 10, 15, 16, 17, 31, 32, 33, 64):
        r = gpu.moe_route_dev(z[:m], top_k, bias=b, sigmoid=bias)
        assert torch.equal(r.ids, whole.ids[:m]) and torch.equal(r.weights, whole.weights[:m]), m
        offsets, order = M.grouped(r.ids.cpu().numpy().reshape(-1), experts)
        assert np.array_equal(r.offsets.cpu().numpy(), offsets) and np.array_equal(r.order.cpu().numpy(), order), m


# many tiles of narrow columns, several column blocks to a workgroup; the same of long ranks, which take wide ones; columns
# that end inside a block, rows that end inside a tile
@pytest.mark.parametrize("rows,adapters,rank,outs", [(70, 32, 64, [14336, 130]), (1500, 3, 20, [4100]), (1003, 5, 8, [2050, 515]),
                                                     (300, 9, 132, [8200]), (1200, 2, 256, [1028])])
@pytest.mark.parametrize("dt", [np.float16, np.float32])
def test_wide_outputs_of_many_rows(gpu, rows, adapters, rank, outs, dt):
    import test_gpu_lora as L
    c = L._case(rows, adapters, rank, 96, outs, dt, rows)
    print("lora", rows, adapters, rank, outs, dt.__name__, flush=True)
    for i, y in enumerate(L._run(gpu, c)):
        want, tol = L._want(c, i)
        assert (np.abs(y.cpu().numpy() - want) <= tol).all()
        out = (c["ids"] < 0) | (c["ids"] >= adapters)
        assert np.array_equal(y.cpu().numpy()[out], c["base"][i][out])
