"""The GPU tests of the experts' products reach every kernel for every type, by the plans of their shapes."""
import pytest

import cllm_inference_amd as C
import test_gpu_expert_spread as P
import test_gpu_experts as T
from cllm_inference_amd import synth as S

KERNELS = {"k_expert_few<4,4>", "k_expert_few<8,4>", "k_expert_few<4,8>", "k_expert_few<1,16>", "k_expert_wide<32>",
           "k_expert_wide<64>"}


def _cases(test, *names):
    """The values of a test's parametrization of these names."""
    for m in test.pytestmark:
        if m.name == "parametrize" and tuple(m.args[0].split(",")) == names:
            return m.args[1]
    raise AssertionError(names)


def _kernel(t, mats, k, n, experts, entries):
    return C.moe_plan(t, mats, k, n, experts, entries).split()[0]


@pytest.mark.parametrize("qt", T.TYPES, ids=lambda t: S.TYPE_NAMES[t])
def test_products_reach_every_kernel(qt):
    got = set()
    for rows, experts, per, k, n in T.SHAPES:
        if qt in (S.Q4_0, S.Q5_0, S.Q8_0):
            k += 32 * (rows % 5) + (96 if rows == 1 else 0)
        got.add(_kernel(qt, 1, k, n, experts, rows * per))
    assert got == KERNELS


@pytest.mark.parametrize("qt", T.TYPES, ids=lambda t: S.TYPE_NAMES[t])
def test_gate_and_up_reach_every_kernel(qt):
    got = {_kernel(qt, 2, k, n, experts, rows * top_k)
           for rows, experts, top_k, k, n in _cases(T.test_moe_swiglu, "rows", "experts", "top_k", "k", "n")}
    for rows, _ in _cases(T.test_swiglu_of_long_rows_with_an_expert_chosen_twice, "rows", "tile"):
        got.add(_kernel(qt, 2, 8448, 37, 2, rows * 2))
    assert got == KERNELS


@pytest.mark.parametrize("qt", T.TYPES, ids=lambda t: S.TYPE_NAMES[t])
@pytest.mark.parametrize("mats", [1, 2])
def test_rows_of_any_spread_reach_every_kernel(qt, mats):
    got = set()
    for rows, experts, per, k, n, _ in P.SHAPES:
        if qt in (S.Q4_0, S.Q5_0, S.Q8_0):
            k += 96
        got.add(_kernel(qt, mats, k, n, experts, rows * per))
    assert got == KERNELS
