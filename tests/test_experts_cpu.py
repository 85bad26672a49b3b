"""Grouped products, router and adapters without a GPU: sizes, refusals, and the models the GPU tests
compare with."""
import ctypes

import numpy as np
import pytest

import cllm_inference_amd as C
import expert_model as M

BUF = ctypes.create_string_buffer(4096 + 16)
PTR = (ctypes.addressof(BUF) + 15) // 16 * 16  # a 16-byte aligned address that no call may reach
SHAPE, TYPE, ARG = 1, 2, 3
Q4_0, Q8_0, Q4_K, F16 = 2, 8, 12, 1
BIG = 1 << 40


def _err():
    return C.load_library().cllm_hip_last_error().decode()


def _matmul(**o):
    a = dict(t=Q4_K, k=512, n=64, experts=4, w=PTR, bias=None, x=PTR, rows=3, per=2, off=PTR, order=PTR, y=PTR,
             ws=PTR, nb=BIG)
    a.update(o)
    return C.load_library().cllm_hip_moe_matmul_dev(a["t"], a["k"], a["n"], a["experts"], a["w"], a["bias"], a["x"],
                                                    a["rows"], a["per"], a["off"], a["order"], a["y"], a["ws"],
                                                    a["nb"], None)


def _swiglu(**o):
    a = dict(t=Q4_K, k=512, n=64, experts=4, w=PTR, w2=PTR, bias=None, bias2=None, x=PTR, rows=3, per=2, off=PTR,
             order=PTR, y=PTR, ws=PTR, nb=BIG)
    a.update(o)
    return C.load_library().cllm_hip_moe_swiglu_dev(a["t"], a["k"], a["n"], a["experts"], a["w"], a["w2"], a["bias"],
                                                    a["bias2"], a["x"], a["rows"], a["per"], a["off"], a["order"],
                                                    a["y"], a["ws"], a["nb"], None)


def _down(**o):
    a = dict(t=Q4_K, k=512, n=64, experts=4, w=PTR, bias=None, x=PTR, rows=3, per=2, ids=PTR, weights=PTR, off=PTR,
             order=PTR, base=None, y=PTR, ws=PTR, nb=BIG)
    a.update(o)
    return C.load_library().cllm_hip_moe_down_dev(a["t"], a["k"], a["n"], a["experts"], a["w"], a["bias"], a["x"],
                                                  a["rows"], a["per"], a["ids"], a["weights"], a["off"], a["order"],
                                                  a["base"], a["y"], a["ws"], a["nb"], None)


@pytest.mark.parametrize("call", [_matmul, _swiglu, _down])
@pytest.mark.parametrize("over,rc,text", [
    (dict(t=F16), TYPE, "type"), (dict(t=3), TYPE, "type"), (dict(t=99), TYPE, "type"),
    (dict(k=500), SHAPE, "block size"), (dict(k=0), SHAPE, "block size"), (dict(k=-256), SHAPE, "block size"),
    (dict(n=-1), ARG, "negative"), (dict(rows=-1), ARG, "negative"), (dict(experts=0), ARG, "experts"),
    (dict(experts=1025), ARG, "experts"), (dict(per=0), ARG, "of a row"), (dict(per=33), ARG, "of a row"),
    (dict(rows=1 << 24), ARG, "too large"), (dict(k=1 << 20, rows=1 << 12), ARG, "too large"),
    (dict(w=None), ARG, "null"), (dict(x=None), ARG, "null"), (dict(y=None), ARG, "null"), (dict(off=None), ARG, "null"),
    (dict(order=None), ARG, "null"), (dict(w=PTR + 8), ARG, "misaligned"), (dict(x=PTR + 4), ARG, "misaligned"),
    (dict(y=PTR + 2), ARG, "misaligned"), (dict(bias=PTR + 1), ARG, "misaligned"), (dict(off=PTR + 2), ARG, "misaligned"),
    (dict(order=PTR + 1), ARG, "misaligned"), (dict(ws=None), ARG, "workspace"), (dict(nb=100), ARG, "workspace"),
    (dict(ws=PTR + 8), ARG, "misaligned"),
])
def test_bad_expert_products_are_refused(call, over, rc, text):
    assert call(**over) == rc
    assert text in _err()


def test_more_refusals_of_expert_products():
    for call, over in ((_swiglu, dict(w2=None)), (_down, dict(ids=None)), (_down, dict(weights=None))):
        assert call(**over) == ARG and "null" in _err()
    for call, over in ((_swiglu, dict(w2=PTR + 8)), (_swiglu, dict(bias2=PTR + 2)), (_down, dict(ids=PTR + 2)),
                       (_down, dict(base=PTR + 4)), (_down, dict(y=PTR + 4)), (_down, dict(weights=PTR + 3))):
        assert call(**over) == ARG and "misaligned" in _err()
    assert _down(rows=65536, per=1) == ARG and "too large" in _err()
    # nothing to do: no device needed
    for call in (_matmul, _swiglu, _down):
        assert call(rows=0) == 0 and call(n=0) == 0


def test_sizes_and_plans():
    lib = C.load_library()
    assert lib.cllm_hip_moe_matmul_ws_bytes(Q8_0, 96, 3) >= 3 * (1024 + 4)
    assert lib.cllm_hip_moe_matmul_ws_bytes(Q4_K, 512, 3) >= 3 * (2 * 1088 + 4)
    assert lib.cllm_hip_moe_down_ws_bytes(Q8_0, 96, 7, 3, 2) >= 6 * (1028 + 28)
    for bad in ((F16, 512, 3), (Q4_K, 0, 3), (Q4_K, 512, 0), (Q4_K, 512, -4)):
        assert lib.cllm_hip_moe_matmul_ws_bytes(*bad) == 0
    assert lib.cllm_hip_moe_down_ws_bytes(Q4_K, 512, 0, 3, 2) == 0
    assert C.moe_plan(Q4_K, 2, 4096, 14336, 8, 2) != "none"
    for bad in ((F16, 1, 512, 64, 4, 8), (Q4_K, 3, 512, 64, 4, 8), (Q4_K, 1, 500, 64, 4, 8), (Q4_K, 1, 512, 64, 0, 8),
                (Q4_K, 1, 512, 64, 4, 0)):
        assert C.moe_plan(*bad) == "none"


def _route(**o):
    a = dict(z=PTR, stride=16, bias=None, rows=2, experts=16, k=4, sig=0, norm=1, scale=1.0, groups=1, top=1, ids=PTR,
             w=PTR, off=PTR, order=PTR)
    a.update(o)
    return C.load_library().cllm_hip_moe_route_dev(a["z"], a["stride"], a["bias"], a["rows"], a["experts"], a["k"],
                                                   a["sig"], a["norm"], a["scale"], a["groups"], a["top"], a["ids"],
                                                   a["w"], a["off"], a["order"], None)


@pytest.mark.parametrize("over,text", [
    (dict(experts=0), "experts"), (dict(experts=1025, stride=2000), "experts"), (dict(stride=15), "experts"),
    (dict(rows=-1), "experts"), (dict(k=0), "top_k"), (dict(k=17), "top_k"), (dict(experts=64, stride=64, k=33), "top_k"),
    (dict(groups=0), "groups"), (dict(groups=3), "groups"), (dict(groups=65, experts=65, stride=65), "groups"),
    (dict(groups=4, top=0), "groups"), (dict(groups=4, top=5), "groups"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(rows=1 << 30), "too large"), (dict(z=None), "null"),
    (dict(ids=None), "null"), (dict(w=None), "null"), (dict(off=None), "null"), (dict(order=None), "null"),
    (dict(z=PTR + 2), "misaligned"), (dict(bias=PTR + 1), "misaligned"), (dict(off=PTR + 2), "misaligned"),
])
def test_a_bad_route_is_refused(over, text):
    assert _route(**over) == ARG
    assert text in _err()


@pytest.mark.parametrize("args,text", [
    ((PTR, -1, 4, PTR, PTR), "groups"), ((PTR, 5, 0, PTR, PTR), "groups"), ((PTR, 5, 1025, PTR, PTR), "groups"),
    ((PTR, (1 << 28) + 1, 4, PTR, PTR), "too large"), ((None, 5, 4, PTR, PTR), "null"), ((PTR, 5, 4, None, PTR), "null"),
    ((PTR, 5, 4, PTR, None), "null"), ((PTR, 0, 4, None, PTR), "null"), ((PTR + 2, 5, 4, PTR, PTR), "misaligned"),
    ((PTR, 5, 4, PTR + 1, PTR), "misaligned"), ((PTR, 5, 4, PTR, PTR + 2), "misaligned"),
])
def test_a_bad_grouping_is_refused(args, text):
    assert C.load_library().cllm_hip_group_rows_dev(*args, None) == ARG
    assert text in _err()


def _lora(**o):
    a = dict(t=F16, k=64, a=[PTR, PTR], b=[PTR, PTR], outs=[32, 8], slots=3, rank=8, ranks=None, scales=None, x=PTR,
             rows=5, off=PTR, order=PTR, base=None, y=[PTR, PTR], ws=PTR, nb=BIG)
    a.update(o)
    n = o.get("mats", len(a["outs"]))
    arr = lambda v: None if v is None else (ctypes.c_void_p * len(v))(*v)  # noqa: E731
    return C.load_library().cllm_hip_lora_dev(a["t"], a["k"], n, arr(a["a"]), arr(a["b"]), (ctypes.c_int * len(a["outs"]))(*a["outs"]),
                                              a["slots"], a["rank"], a["ranks"], a["scales"], a["x"], a["rows"], a["off"],
                                              a["order"], arr(a["base"]), arr(a["y"]), a["ws"], a["nb"], None)


@pytest.mark.parametrize("over,rc,text", [
    (dict(t=Q8_0), TYPE, "F16 or F32"), (dict(mats=0), ARG, "projections"), (dict(outs=[1] * 5, mats=5), ARG, "projections"),
    (dict(k=0), SHAPE, "in_dim"), (dict(k=66), SHAPE, "in_dim"), (dict(rank=0), SHAPE, "max_rank"),
    (dict(rank=6), SHAPE, "max_rank"), (dict(rank=260), SHAPE, "max_rank"), (dict(slots=0), ARG, "adapters"),
    (dict(slots=1024), ARG, "adapters"), (dict(rows=-1), ARG, "too large"), (dict(rows=(1 << 24) + 1), ARG, "too large"),
    (dict(outs=[32, -1]), ARG, "negative"), (dict(outs=[1 << 21, 1]), ARG, "too wide"), (dict(x=None), ARG, "null"),
    (dict(a=None), ARG, "null"), (dict(b=None), ARG, "null"), (dict(y=None), ARG, "null"), (dict(a=[PTR, None]), ARG, "null"),
    (dict(y=[None, PTR]), ARG, "null"), (dict(off=None), ARG, "null"), (dict(b=[PTR, PTR + 8]), ARG, "misaligned"),
    (dict(base=[PTR + 4, None]), ARG, "misaligned"), (dict(x=PTR + 8), ARG, "misaligned"), (dict(ranks=PTR + 2), ARG, "misaligned"),
    (dict(ws=None), ARG, "workspace"), (dict(nb=8), ARG, "workspace"),
])
def test_bad_adapters_are_refused(over, rc, text):
    assert _lora(**over) == rc
    assert text in _err()


def test_adapters_of_no_rows():
    assert _lora(rows=0) == 0
    lib = C.load_library()
    assert lib.cllm_hip_lora_ws_bytes(64, 2, 3, 8, 5) >= 2 * 5 * 8 * 4
    for bad in ((0, 2, 3, 8, 5), (64, 5, 3, 8, 5), (64, 2, 0, 8, 5), (64, 2, 3, 260, 5), (64, 2, 3, 8, 0)):
        assert lib.cllm_hip_lora_ws_bytes(*bad) == 0


def test_the_models():
    offsets, order = M.grouped(np.array([2, -1, 0, 2, 7, 0], np.int32), 3)
    assert offsets.tolist() == [0, 2, 2, 4] and order.tolist() == [2, 5, 0, 3, 1, 4]
    z = np.array([[1, 1, -np.inf, 0], [np.nan, np.inf, 2, np.inf]], np.float32)
    ids, w = M.route(z, 3)
    assert ids.tolist() == [[0, 1, 3], [1, 3, 2]]
    e = np.exp(-1.0)
    assert np.allclose(w, [[1 / (2 + e), 1 / (2 + e), e / (2 + e)], [0.5, 0.5, 0]])
    ids, w = M.route(z[:1], 4, sigmoid=True, normalise=False, scale=2.0)
    assert ids.tolist() == [[0, 1, 3, -1]] and np.allclose(w, [[2 / (1 + e), 2 / (1 + e), 1, 0]])
    # the second pair has the larger sum of two, the first the largest key
    z = np.array([[3, 0, 2, 2]], np.float32)
    assert M.route(z, 1, parts=2, top_parts=1)[0].tolist() == [[0]]
    assert M.route(z, 1, bias=np.zeros(4, np.float32), sigmoid=True, parts=2, top_parts=1)[0].tolist() == [[2]]
