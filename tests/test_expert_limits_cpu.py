"""Sizes of grouped products, router and adapters that one call takes, without a GPU: calls that pass every check of
sizes end at a workspace that is too small, before any device is asked for."""
import ctypes

import pytest

import cllm_inference_amd as C

BUF = ctypes.create_string_buffer(4096 + 16)
PTR = (ctypes.addressof(BUF) + 15) // 16 * 16  # a 16-byte aligned address that no call may reach
ARG = 3
Q8_0, Q4_K = 8, 12


def _call(which, t, k, n, experts, rows, per):
    lib = C.load_library()
    if which == "matmul":
        return lib.cllm_hip_moe_matmul_dev(t, k, n, experts, PTR, None, PTR, rows, per, PTR, PTR, PTR, PTR, 16, None)
    if which == "swiglu":
        return lib.cllm_hip_moe_swiglu_dev(t, k, n, experts, PTR, PTR, None, None, PTR, rows, per, PTR, PTR, PTR, PTR,
                                           16, None)
    return lib.cllm_hip_moe_down_dev(t, k, n, experts, PTR, None, PTR, rows, per, PTR, PTR, PTR, PTR, None, PTR, PTR, 16,
                                     None)


def _err():
    return C.load_library().cllm_hip_last_error().decode()


@pytest.mark.parametrize("which", ["matmul", "swiglu"])
@pytest.mark.parametrize("t,k,per", [(Q4_K, 7168, 8), (Q4_K, 4096, 8), (Q8_0, 96, 32), (Q4_K, 14336, 1)])
def test_the_quantized_rows_are_the_rows_of_x(which, t, k, per):
    """An operand of less than 4 GiB is taken, however many entries its rows have."""
    most = ((1 << 32) - 1) // ((k + 255) // 256 * 1024)
    assert most * per <= 1 << 28
    assert _call(which, t, k, 64, 256, most, per) == ARG and "workspace" in _err()
    assert _call(which, t, k, 64, 256, most + 1, per) == ARG and "too large" in _err()


def test_the_way_down_quantizes_every_entry():
    most = ((1 << 32) - 1) // (28 * 1024) // 8
    assert most < 65535
    assert _call("down", Q4_K, 7168, 64, 256, most, 8) == ARG and "workspace" in _err()
    assert _call("down", Q4_K, 7168, 64, 256, most + 1, 8) == ARG and "too large" in _err()


def test_plans_of_many_entries():
    assert "k_expert_wide" in C.moe_plan(Q4_K, 2, 7168, 2048, 256, 160000)
    assert "k_expert_wide" in C.moe_plan(Q4_K, 1, 7168, 2048, 256, 1 << 22)
    assert C.moe_plan(Q4_K, 2, 7168, 2048, 256, (1 << 28) + 1) == "none"


@pytest.mark.parametrize("k,mats,adapters,rank", [(4096, 3, 4, 16), (4096, 1, 5, 32), (4096, 2, 32, 64), (896, 4, 1023, 8),
                                                  (14336, 4, 1, 256), (512, 1, 1, 4), (1000, 2, 7, 12)])
def test_an_adapter_workspace_serves_every_smaller_batch(k, mats, adapters, rank):
    size = C.load_library().cllm_hip_lora_ws_bytes
    sizes = [size(k, mats, adapters, rank, n) for n in range(1, 17001)]
    assert all(a <= b for a, b in zip(sizes, sizes[1:]))
    assert sizes[0] >= mats * rank * 4
    # a row's sums, once for each projection at least
    assert all(s >= mats * rank * 4 * n for n, s in enumerate(sizes, 1))
    assert size(k, mats, adapters, rank, 1 << 24) >= sizes[-1]


def test_expert_workspaces_serve_every_smaller_batch():
    lib = C.load_library()
    for t, k in ((Q8_0, 96), (Q4_K, 768)):
        m = [lib.cllm_hip_moe_matmul_ws_bytes(t, k, n) for n in range(1, 300)]
        assert m == sorted(m)
        for per in (1, 5):
            d = [lib.cllm_hip_moe_down_ws_bytes(t, k, 33, n, per) for n in range(1, 300)]
            assert d == sorted(d)
