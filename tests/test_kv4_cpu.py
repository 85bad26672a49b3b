"""The 4-bit cache and the log probabilities without a GPU: sizes, refusals, and the model the GPU
tests compare with."""
import ctypes

import numpy as np
import pytest

import cllm_inference_amd as C
import kv4_model as M

BUF = ctypes.create_string_buffer(4096 + 16)
PTR = (ctypes.addressof(BUF) + 15) // 16 * 16  # a 16-byte aligned address that no call may reach


def _cache(**over):
    f = dict(pages=PTR, table=PTR, lens=PTR, refs=PTR, work=PTR, n_layers=2, n_pages=8, page_size=64,
             n_head_kv=2, head_dim=128, max_seqs=4, max_pages=4)
    f.update(over)
    return C._Kv4CacheStruct(*[f[n] for n, _ in C._Kv4CacheStruct._fields_])


def _err():
    return C.load_library().cllm_hip_last_error().decode()


def test_sizes():
    for page in (32, 64, 1024):
        for hd in (64, 128, 256):
            assert C.kv4_page_bytes(page, 3, hd) == 3 * page * hd * 9 // 8
    for bad in ((16, 1, 64), (48, 1, 64), (2048, 1, 64), (0, 1, 64), (-32, 1, 64), (64, 0, 64), (64, -1, 64),
                (64, 1, 96), (64, 1, 512), (64, 1, 0), (64, 2000, 64)):
        assert C.kv4_page_bytes(*bad) == 0
    lib = C.load_library()
    assert lib.cllm_hip_kv4_work_ints(100, 4, 4) >= 301
    assert lib.cllm_hip_kv4_work_ints(10, 500, 1000) >= 500 * 1001
    assert lib.cllm_hip_kv4_work_ints(0, 4, 4) == 0
    assert lib.cllm_hip_logprobs_ws_bytes(3, 8192, 5) == 3 * (32 + 40)
    assert lib.cllm_hip_logprobs_ws_bytes(3, 8193, 5) == 6 * (32 + 40)
    assert lib.cllm_hip_logprobs_ws_bytes(3, 8193, 65) == 0


@pytest.mark.parametrize("over,text", [
    (dict(page_size=48), "page_size"), (dict(page_size=2048), "page_size"), (dict(head_dim=96), "head_dim"),
    (dict(n_head_kv=0), "n_head_kv"), (dict(n_layers=0), "shape"), (dict(n_pages=0), "shape"),
    (dict(max_seqs=0), "shape"), (dict(max_pages=-1), "shape"), (dict(max_pages=1 << 26), "shape"),
    (dict(max_seqs=1 << 20, max_pages=1 << 12), "shape"),
    (dict(pages=0), "null"), (dict(table=0), "null"), (dict(lens=0), "null"), (dict(refs=0), "null"),
    (dict(work=0), "null"), (dict(pages=PTR + 8), "misaligned"), (dict(table=PTR + 2), "misaligned"),
    (dict(refs=PTR + 1), "misaligned"),
])
def test_a_bad_cache_is_refused(over, text):
    lib = C.load_library()
    c = _cache(**over)
    assert lib.cllm_hip_kv4_extend_dev(ctypes.byref(c), None, PTR, 1, PTR, None) == 3
    assert text in _err()
    if "work" not in over:
        assert lib.cllm_hip_kv4_load_dev(ctypes.byref(c), 0, None, PTR, 1, 1, PTR, PTR, None) == 3
        assert text in _err()
        assert lib.cllm_hip_kv4_attention_ws_bytes(ctypes.byref(c), 1, 1, 1, 100, 2) == 0
        assert lib.cllm_hip_kv4_attention_plan(ctypes.byref(c), 1, 1, 1, 100, 2) == b"none"


def test_bad_arguments_are_refused():
    lib = C.load_library()
    c = _cache()
    r = ctypes.byref(c)
    ext, fork, trunc = lib.cllm_hip_kv4_extend_dev, lib.cllm_hip_kv4_fork_dev, lib.cllm_hip_kv4_truncate_dev
    store, load, att = lib.cllm_hip_kv4_store_dev, lib.cllm_hip_kv4_load_dev, lib.cllm_hip_kv4_attention_dev
    bad = [
        lambda: ext(None, None, PTR, 1, PTR, None), lambda: ext(r, None, None, 1, PTR, None),
        lambda: ext(r, None, PTR, 1025, PTR, None), lambda: ext(r, None, PTR, -1, PTR, None),
        lambda: ext(r, PTR + 1, PTR, 1, PTR, None), lambda: ext(r, None, PTR, 1, None, None),
        lambda: fork(r, PTR, None, 1, None), lambda: fork(r, None, PTR, 1, None),
        lambda: fork(r, PTR, PTR, 5, None),  # more entries than slots
        lambda: trunc(r, None, None, 1, None), lambda: trunc(r, PTR, PTR + 2, 1, None),
        lambda: lib.cllm_hip_kv4_compact_dev(r, None, None),
        lambda: lib.cllm_hip_kv4_copy_pages_dev(r, PTR, None, 1, None),
        lambda: store(r, 2, PTR, PTR, None, 0, 0.0, None, PTR, 1, 1, None),
        lambda: store(r, -1, PTR, PTR, None, 0, 0.0, None, PTR, 1, 1, None),
        lambda: store(r, 0, None, PTR, None, 0, 0.0, None, PTR, 1, 1, None),
        lambda: store(r, 0, PTR, PTR + 4, None, 0, 0.0, None, PTR, 1, 1, None),
        lambda: store(r, 0, PTR, PTR, None, 0, 0.0, None, None, 1, 1, None),
        lambda: store(r, 0, PTR, PTR, None, 0, 0.0, None, PTR, -1, 1, None),
        lambda: store(r, 0, PTR, PTR, None, 0, 0.0, None, PTR, 70000, 1, None),
        lambda: store(r, 0, PTR, PTR, None, 0, -1.0, None, PTR, 1, 1, None),
        lambda: store(r, 0, PTR, PTR, None, 0, float("nan"), None, PTR, 1, 1, None),
        lambda: store(r, 0, PTR, PTR, PTR, 4, 0.0, None, PTR, 1, 1, None),
        lambda: store(r, 0, PTR, PTR, PTR, 0, 1e4, None, PTR, 1, 1, None),
        lambda: load(r, 0, None, PTR, 1, 1, None, PTR, None),
        lambda: load(r, 0, None, PTR, 1, 1, PTR, PTR + 8, None),
        lambda: att(r, 0, PTR, None, PTR, 1, 1, 1, 100, 3, PTR, None, 0, None),  # 3 heads over 2
        lambda: att(r, 0, PTR, None, PTR, 1, 1, 1, 100, 0, PTR, None, 0, None),
        lambda: att(r, 5, PTR, None, PTR, 1, 1, 1, 100, 4, PTR, None, 0, None),
        lambda: att(r, 0, None, None, PTR, 1, 1, 1, 100, 4, PTR, None, 0, None),
        lambda: att(r, 0, PTR, None, PTR, 1, 1, 1, 100, 4, PTR + 4, None, 0, None),
        lambda: att(r, 0, PTR, None, PTR, 1, 1, -1, 100, 4, PTR, None, 0, None),
        lambda: att(r, 0, PTR, None, PTR, 1, 1, 1, -1, 4, PTR, None, 0, None),
    ]
    for i, call in enumerate(bad):
        assert call() == 3, i
        assert _err().startswith("kv4_"), i
    # a workspace that is too small
    big = _cache(max_pages=4096, n_pages=100)
    args = (1, 1, 1, 200000, 4)
    need = lib.cllm_hip_kv4_attention_ws_bytes(ctypes.byref(big), *args)
    assert need > 0
    for ws, n in ((PTR, need - 1), (None, need), (PTR + 4, need)):
        assert att(ctypes.byref(big), 0, PTR, None, PTR, *args, PTR, ws, n, None) == 3
    # nothing to do is no error, and needs no GPU
    assert store(r, 0, None, None, None, 0, 0.0, None, None, 0, 0, None) == 0
    assert load(r, 0, None, None, 0, 0, None, None, None) == 0
    assert att(r, 0, None, None, None, 0, 0, 0, 0, 4, None, None, 0, None) == 0
    assert fork(r, None, None, 0, None) == 0


def test_launches_past_32_bits_are_refused():
    """The threads of a launch are counted in 32 bits."""
    lib = C.load_library()
    c = _cache(max_pages=4096, max_seqs=65536)
    r = ctypes.byref(c)
    for args in ((65536, 1 << 26, 1 << 26, 100, 65536), (65536, 1 << 26, 1024, 100, 64), (65536, 1 << 26, 8, 100000, 65536)):
        assert lib.cllm_hip_kv4_attention_dev(r, 0, PTR, None, PTR, *args, PTR, PTR, 1 << 60, None) == 3, args
        assert "too large" in _err()
        assert lib.cllm_hip_kv4_attention_ws_bytes(r, *args) == 0
        assert lib.cllm_hip_kv4_attention_plan(r, *args) == b"none"
    assert lib.cllm_hip_kv4_attention_plan(r, 65536, 65536, 1, 100000, 16) != b"none"
    f = lib.cllm_hip_logprobs_dev
    assert f(PTR, 100, 1 << 24, 100, PTR, 0, PTR, PTR, PTR, PTR, None, None, PTR, 1 << 60, None) == 3
    assert "too large" in _err()


def test_logprobs_refusals():
    f = C.load_library().cllm_hip_logprobs_dev
    ok = dict(logits=PTR, stride=100, rows=2, vocab=100, tokens=PTR, k=5, lp=PTR, rk=PTR, en=PTR, ls=PTR, ti=PTR,
              tl=PTR, ws=PTR, n=1 << 20, s=None)
    for over in (dict(logits=None), dict(logits=PTR + 2), dict(stride=99), dict(rows=-1), dict(vocab=0),
                 dict(vocab=-5), dict(k=-1), dict(k=65), dict(k=101, vocab=100), dict(tokens=None), dict(ws=None),
                 dict(n=10), dict(ws=PTR + 4), dict(lp=PTR + 1), dict(ti=PTR + 2), dict(vocab=4, stride=4, k=5)):
        assert f(*{**ok, **over}.values()) == 3, over
        assert _err().startswith("logprobs"), over
    assert f(*{**ok, "rows": 0, "logits": None, "ws": None}.values()) == 0


def test_places_cover_a_tile_once():
    """Every nibble of the code bytes and every scale is some element's."""
    for hd in (64, 128, 256):
        seen, scales = set(), set()
        for value in (False, True):
            b, s, sc = M.places(hd, value)
            seen |= set(zip(b.reshape(-1).tolist(), s.reshape(-1).tolist()))
            scales |= set(sc.reshape(-1).tolist())
        assert seen == {(b, s) for b in range(32 * hd) for s in (0, 4)}
        assert scales == set(range(32 * hd, 36 * hd, 2))


def test_quantize_model():
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((200, 64)) * np.exp(3 * rng.standard_normal((200, 1)))).astype(np.float32)
    x[0] = 0
    x[1] = 1e-9
    x[2] *= 1e7
    c, d = M.quantize(x)
    assert c.min() >= 0 and c.max() <= 15
    assert np.array_equal(d, d.astype(np.float16).astype(np.float64)) and np.abs(d).max() <= 8160
    y = ((c - 8).reshape(200, 2, 32) * d[..., None])
    assert np.array_equal(y, y.astype(np.float16).astype(np.float64))  # exact in fp16
    ok = np.arange(200) > 2
    err = np.abs(y.reshape(200, 64) - x)[ok].reshape(-1, 2, 32).max(-1)
    # half a step; the side opposite the extreme ends at 7 steps, one short, less the scale's rounding
    assert (err <= np.abs(d[ok]) * 1.04).all()
