"""Where the experts' weights lie, on an MI355X: matrices past 4 GiB, and the 3-d tensors of a GGUF file."""
import ctypes

import numpy as np
import pytest

import expert_model as M
import gguf_writer as G
from cllm_inference_amd import synth as S

pytestmark = pytest.mark.gpu


def _cu(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _groups(gpu, ids, experts):
    offsets, order = M.grouped(ids.reshape(-1), experts)
    return gpu.MoeRoute(_cu(ids), None, _cu(offsets), _cu(order))


def _far_expert(qt, experts, n, k, seed):
    """[experts] matrices of zeros but for the last, and that one."""
    import torch
    one = S.make_weight(qt, n, k, seed).reshape(n, -1)
    w = torch.zeros((experts, one.size), dtype=torch.uint8, device="cuda")
    w[experts - 1] = _cu(one.reshape(-1))
    assert w.numel() - one.size > 1 << 32
    return w, one


def _some(one, qt, k, cols):
    """Values and magnitudes of some rows of a matrix."""
    v, m = M.expert_values(np.ascontiguousarray(one[cols]).reshape(-1), qt, 1, len(cols), k)
    return v[0], m[0]


# blocks with a scale each, and a type whose headers reach LDS on a way of their own
@pytest.mark.parametrize("qt,experts", [(S.Q8_0, 80), (S.Q4_K, 140), (S.Q6_K, 100)], ids=["Q8_0", "Q4_K", "Q6_K"])
@pytest.mark.parametrize("each,kernel", [(1, "k_expert_few"), (20, "k_expert_wide<32>"), (44, "k_expert_wide<64>")])
def test_an_expert_past_4_gib(gpu, orc, qt, experts, each, kernel):
    n, k = 14336, 4096
    rows = experts * each
    assert kernel in gpu.moe_plan(qt, 1, k, n, experts, rows)
    w, one = _far_expert(qt, experts, n, k, 61)
    x = S.make_activation(64, k, 62)[np.arange(rows) % 64]
    ids = np.full((rows, 1), experts - 1, np.int32)
    ids[:3] = 0
    print("past 4 GiB", S.TYPE_NAMES[qt], rows, gpu.moe_plan(qt, 1, k, n, experts, rows), flush=True)
    y = gpu.moe_matmul_dev(_cu(x), w, qt, n, _groups(gpu, ids, experts))
    assert not bool(y[:3].any())  # an expert of zeros
    at, cols = [3, 40, rows - 1], np.r_[0:40, 7000:7040, n - 40:n]
    values, mags = _some(one, qt, k, cols)
    xr = M.q8_values(orc, x[at])
    got = y[at].cpu().numpy()[:, cols]
    assert (np.abs(got - xr @ values.T) <= M.product_bound(mags, xr, k)).all()
    # every one of equal rows alike, every column
    same = y[3:].view(rows - 3, n)
    assert bool((same[64:] == same[:-64]).all())


@pytest.mark.parametrize("each,kernel", [(20, "k_expert_wide<32>"), (44, "k_expert_wide<64>")])
def test_gate_and_up_past_4_gib(gpu, orc, each, kernel):
    qt, experts, n, k = S.Q4_K, 140, 14336, 4096
    rows = experts * each
    assert kernel in gpu.moe_plan(qt, 2, k, n, experts, rows)
    wg, one_g = _far_expert(qt, experts, n, k, 63)
    wu, one_u = _far_expert(qt, experts, n, k, 64)
    x = S.make_activation(64, k, 65)[np.arange(rows) % 64]
    ids = np.full((rows, 1), experts - 1, np.int32)
    h = gpu.moe_swiglu_dev(_cu(x), wg, wu, qt, n, _groups(gpu, ids, experts)).view(rows, n)
    at, cols = [0, 40, rows - 1], np.r_[0:40, n - 40:n]
    xr = M.q8_values(orc, x[at])
    (vg, mg), (vu, mu) = _some(one_g, qt, k, cols), _some(one_u, qt, k, cols)
    g, u = xr @ vg.T, xr @ vu.T
    eg, eu = M.product_bound(mg, xr, k), M.product_bound(mu, xr, k)
    want = M.silu(g) * u
    # |silu'| <= 1.1; expf within 2 steps (2^-22 of exp, which 1 + exp only dampens), the sum, quotient and product
    bound = 1.1 * eg * (np.abs(u) + eu) + np.abs(M.silu(g)) * eu + np.abs(want) * 2.0 ** -21 + 2.0 ** -126
    assert (np.abs(h[at].cpu().numpy()[:, cols] - want) <= bound).all()


@pytest.mark.parametrize("rows", [1, 30])
def test_the_3d_tensors_of_a_file(gpu, tmp_path, rows):
    """[expert][row][blocks] tensors of a GGUF file, at the addresses that its upload gives: the results of copies."""
    import torch
    experts, top_k, k, n_ff, qt, qd = 5, 2, 512, 768, S.Q4_K, S.Q6_K
    mats = [("blk.0.ffn_gate_exps.weight", qt, (experts, n_ff, k)), ("blk.0.ffn_up_exps.weight", qt, (experts, n_ff, k)),
            ("blk.0.ffn_down_exps.weight", qd, (experts, k, n_ff))]
    raw = [S.make_weight(t, s[0] * s[1], s[2], 90 + i) for i, (_, t, s) in enumerate(mats)]
    path = tmp_path / "experts.gguf"
    G.write_gguf(path, [("general.architecture", G.STR, "llama")],
                 [(name, s, t, w.tobytes()) for (name, t, s), w in zip(mats, raw)])
    x = _cu(S.make_activation(rows, k, 95))
    r = gpu.moe_route_dev(torch.randn((rows, experts), device="cuda", generator=torch.Generator("cuda").manual_seed(3)), top_k)
    h = gpu.moe_swiglu_dev(x, _cu(raw[0].reshape(-1)), _cu(raw[1].reshape(-1)), qt, n_ff, r)
    y = gpu.moe_down_dev(h, _cu(raw[2].reshape(-1)), qd, k, r, base=x)
    lib = gpu.load_library()
    with gpu.GgufFile(path, upload=True) as g:
        t = [g.tensor(g.find(name)) for name, _, _ in mats]
        for info, (_, typ, shape) in zip(t, mats):
            assert info.shape == shape and info.type == typ and info.dev % 16 == 0
        s = torch.cuda.current_stream().cuda_stream
        p = lambda a: ctypes.c_void_p(a.data_ptr())  # noqa: E731
        h2, y2 = torch.empty_like(h), torch.empty_like(y)
        nb = lib.cllm_hip_moe_matmul_ws_bytes(qt, k, rows)
        ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
        assert lib.cllm_hip_moe_swiglu_dev(qt, k, n_ff, experts, t[0].dev, t[1].dev, None, None, p(x), rows, top_k,
                                           p(r.offsets), p(r.order), p(h2), p(ws), nb, s) == 0
        nb = lib.cllm_hip_moe_down_ws_bytes(qd, n_ff, k, rows, top_k)
        ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
        assert lib.cllm_hip_moe_down_dev(qd, n_ff, k, experts, t[2].dev, None, p(h2), rows, top_k, p(r.ids), p(r.weights),
                                         p(r.offsets), p(r.order), p(x), p(y2), p(ws), nb, s) == 0
        torch.cuda.synchronize()
    assert torch.equal(h, h2) and torch.equal(y, y2)
