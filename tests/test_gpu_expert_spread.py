"""The experts' products of rows whose blocks lie far apart, on an MI355X against 64 bits: what a quiet block adds
is as exact as fp32 sums have it, however loud another block of the row is."""
import numpy as np
import pytest

import expert_model as M
from cllm_inference_amd import synth as S

pytestmark = pytest.mark.gpu

TYPES = [S.Q4_0, S.Q5_0, S.Q8_0, S.Q4_K, S.Q5_K, S.Q6_K]
# every tile: 4 entries (K in 4 and in 8 parts), 8, 16, 32 and 64
SHAPES = [(2, 4, 1, 512, 50, "<4,4>"), (2, 4, 1, 8448, 33, "<8,4>"), (7, 2, 2, 8448, 37, "<4,8>"),
          (33, 8, 2, 256, 130, "<1,16>"), (24, 2, 2, 512, 290, "<32>"), (90, 2, 2, 768, 140, "<64>")]


def _cu(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _route(gpu, ids, experts, weights=None):
    offsets, order = M.grouped(ids.reshape(-1), experts)
    return gpu.MoeRoute(_cu(ids), None if weights is None else _cu(weights), _cu(offsets), _cu(order))


def _silence(w, t, rows, k, block):
    """The weights (GGUF rows) with the values of one block of 32 set to zero; of K-quants one of a super-block's
    first four, by its 6-bit scale and minimum (Q6_K: its two scales), the others of its super-block stay."""
    w = w.reshape(rows, -1).copy()
    if t in (S.Q4_0, S.Q5_0, S.Q8_0):
        size = w.shape[1] // (k // 32)
        w[:, size * block:size * block + 2] = 0
        return w
    assert block % 8 < 4
    size = w.shape[1] // (k // 256)
    at, j = size * (block // 8), block % 8
    if t == S.Q6_K:
        w[:, at + 192 + 2 * j:at + 194 + 2 * j] = 0
    else:
        w[:, at + 4 + j] &= 0xC0
        w[:, at + 8 + j] &= 0xC0
    return w


def _loud(x, block, bits, every=1):
    """x with one block 2^bits above the rest, in every `every`-th row."""
    x = x.copy()
    x[::every, 32 * block:32 * block + 32] *= np.float32(2.0 ** bits)
    return x


def _bound(mag, x, k):
    """Sums of k products in fp32, [m][n] of mag [n][k] and x [m][k].
      rows within the operand's range: a value as hi + lo to 2^-23, one product of Q6_K left out (2^-22), and a
      matrix instruction's and the joins' additions (product_bound: up to 26 a super-block, one after each, 10) of 2^-23;
      rows of codes: a block's sum is exact; its scale's product with dx is off by 2^-24; two additions a block
      (products, minimum) and the joins' of 2^-24 each."""
    chunks, blocks = (k + 255) // 256, k // 32
    near = 2.0 ** -22 + 2.0 ** -23 + (26 + chunks + 10) * 2.0 ** -23
    far = 2.0 ** -24 + (2 * blocks + 10) * 2.0 ** -24
    return np.abs(x) @ mag.T * max(near, far)


def _case(t, rows, experts, per, k, n, seed):
    if t in (S.Q4_0, S.Q5_0, S.Q8_0):
        k += 96  # ends inside a super-block's length
    block = 3 if rows % 2 else 8 * (k // 256 - 1) + 1
    w = _silence(S.make_weight(t, experts * n, k, seed), t, experts * n, k, block)
    x = S.make_activation(rows, k, seed + 1)
    ids = np.argsort(np.random.default_rng(seed).random((rows, experts)), 1)[:, :per].astype(np.int32)
    return k, block, w, x, ids


def _products(orc, w, t, x, ids, per, experts, n, k):
    values, mags = M.expert_values(w.reshape(-1), t, experts, n, k)
    xr = M.q8_values(orc, x)
    flat = ids.reshape(-1)
    y, b = np.zeros((flat.size, n)), np.zeros((flat.size, n))
    for e in range(experts):
        at = np.nonzero(flat == e)[0]
        y[at] = xr[at // per] @ values[e].T
        b[at] = _bound(mags[e], xr[at // per], k)
    return y, b


@pytest.mark.parametrize("qt", TYPES, ids=lambda t: S.TYPE_NAMES[t])
@pytest.mark.parametrize("rows,experts,per,k,n,tile", SHAPES)
@pytest.mark.parametrize("bits", [3, 16, 30, 100])
def test_quiet_blocks_beside_a_loud_one(gpu, orc, qt, rows, experts, per, k, n, tile, bits):
    """Weights that are zero in the loud block: the quiet ones are all there is."""
    k, block, w, x, ids = _case(qt, rows, experts, per, k, n, 7 * rows + qt)
    plan = gpu.moe_plan(qt, 1, k, n, experts, rows * per)
    print("spread", S.TYPE_NAMES[qt], rows, experts, per, k, n, bits, plan, flush=True)
    assert tile in plan
    x = _loud(x, block, bits)
    y = gpu.moe_matmul_dev(_cu(x), _cu(w), qt, n, _route(gpu, ids, experts), per_row=per).cpu().numpy()
    want, bound = _products(orc, w, qt, x, ids, per, experts, n, k)
    err = np.abs(y - want)
    assert (err <= bound).all(), float((err / bound).max())
    # roundings of either sign: far inside the bound together
    assert np.linalg.norm(err) <= 2.0 ** -20 * np.linalg.norm(want)


@pytest.mark.parametrize("qt", TYPES, ids=lambda t: S.TYPE_NAMES[t])
@pytest.mark.parametrize("rows,experts,per,k,n,tile", SHAPES)
def test_rows_beside_rows_of_another_spread(gpu, orc, qt, rows, experts, per, k, n, tile):
    """Every other row with blocks of all loudnesses between 2^-40 and 2^40, zeros among them: within the bound, and
    the rows between have the bits that they have without them."""
    k, _, w, x, ids = _case(qt, rows, experts, per, k, n, 11 * rows + qt)
    rng = np.random.default_rng(rows)
    far = x.copy()
    scale = 2.0 ** rng.integers(-40, 41, (len(far[::2]), k // 32))
    scale[:, 5] = 0
    far[::2] = (far[::2].reshape(-1, k // 32, 32) * scale[..., None]).reshape(-1, k).astype(np.float32)
    bias = rng.standard_normal((experts, n)).astype(np.float32)
    g = _route(gpu, ids, experts)
    near = gpu.moe_matmul_dev(_cu(x), _cu(w), qt, n, g, bias=_cu(bias), per_row=per).cpu().numpy()
    y = gpu.moe_matmul_dev(_cu(far), _cu(w), qt, n, g, bias=_cu(bias), per_row=per).cpu().numpy()
    want, bound = _products(orc, w, qt, far, ids, per, experts, n, k)
    want = want + bias[ids.reshape(-1)]
    err = np.abs(y - want)
    assert (err <= bound + np.abs(want) * 2.0 ** -24).all()
    odd = np.arange(rows * per) // per % 2 == 1
    assert np.array_equal(y[odd], near[odd])


@pytest.mark.parametrize("qt", TYPES, ids=lambda t: S.TYPE_NAMES[t])
@pytest.mark.parametrize("rows,experts,per,k,n,tile", SHAPES)
def test_gate_and_up_of_a_loud_block(gpu, orc, qt, rows, experts, per, k, n, tile):
    k, block, wg, x, ids = _case(qt, rows, experts, per, k, n, 13 * rows + qt)
    wu = _silence(S.make_weight(qt, experts * n, k, 3), qt, experts * n, k, block)
    x = _loud(x, block, 40, every=2 if rows > 2 else 1)
    rng = np.random.default_rng(rows)
    bg, bu = (rng.standard_normal((experts, n)).astype(np.float32) for _ in range(2))
    print("gate and up", S.TYPE_NAMES[qt], rows, k, n, gpu.moe_plan(qt, 2, k, n, experts, rows * per), flush=True)
    h = gpu.moe_swiglu_dev(_cu(x), _cu(wg), _cu(wu), qt, n, _route(gpu, ids, experts), bias_gate=_cu(bg),
                           bias_up=_cu(bu)).cpu().numpy().reshape(-1, n)
    flat = ids.reshape(-1)
    g, eg = _products(orc, wg, qt, x, ids, per, experts, n, k)
    u, eu = _products(orc, wu, qt, x, ids, per, experts, n, k)
    g, u = g + bg[flat], u + bu[flat]
    eg, eu = eg + np.abs(g) * 2.0 ** -24, eu + np.abs(u) * 2.0 ** -24
    want = M.silu(g) * u
    # |silu'| <= 1.1; expf within 2 steps (2^-22 of exp, which 1 + exp only dampens), the sum, quotient and product
    bound = 1.1 * eg * (np.abs(u) + eu) + np.abs(M.silu(g)) * eu + np.abs(want) * 2.0 ** -21 + 2.0 ** -126
    assert (np.abs(h - want) <= bound).all(), float((np.abs(h - want) / bound).max())


@pytest.mark.parametrize("qt", [S.Q5_0, S.Q4_K, S.Q6_K], ids=lambda t: S.TYPE_NAMES[t])
def test_down_of_a_loud_block(gpu, orc, qt):
    rows, experts, top_k, k, n = 40, 4, 2, 512, 96
    block = 2
    w = _silence(S.make_weight(qt, experts * n, k, 1), qt, experts * n, k, block)
    h = _loud(S.make_activation(rows * top_k, k, 2), block, 36, every=3)
    rng = np.random.default_rng(4)
    ids = np.argsort(rng.random((rows, experts)), 1)[:, :top_k].astype(np.int32)
    p = rng.random((rows, top_k)).astype(np.float32)
    y = gpu.moe_down_dev(_cu(h), _cu(w), qt, n, _route(gpu, ids, experts, p)).cpu().numpy()
    v, b = _products(orc, w, qt, h, ids, 1, experts, n, k)
    terms = v.reshape(rows, top_k, n) * p[..., None]
    tol = (b.reshape(rows, top_k, n) * p[..., None]).sum(1) + np.abs(terms).sum(1) * (top_k + 2) * 2.0 ** -24
    assert (np.abs(y - terms.sum(1)) <= tol).all()


@pytest.mark.parametrize("qt", TYPES, ids=lambda t: S.TYPE_NAMES[t])
def test_scaled_rows_of_a_wide_spread_keep_their_bits(gpu, qt):
    """Powers of two, infinities and NaN: a row of codes scales exactly, and one that is not finite gives NaN."""
    rows, experts, k, n = 40, 2, 512, 70
    w = _cu(S.make_weight(qt, experts * n, k, 5))
    x = _loud(S.make_activation(rows, k, 6), 9, 33)
    g = _route(gpu, np.zeros((rows, 1), np.int32), experts)
    clean = gpu.moe_matmul_dev(_cu(x), w, qt, n, g).cpu().numpy()
    x2 = x * np.float32(2.0 ** -30)
    x2[1, 3], x2[2, 300] = np.inf, np.nan
    y = gpu.moe_matmul_dev(_cu(x2), w, qt, n, g).cpu().numpy()
    assert np.isnan(y[1:3]).all()
    keep = np.delete(np.arange(rows), [1, 2])
    assert np.array_equal(y[keep], clean[keep] * np.float32(2.0 ** -30))


@pytest.mark.parametrize("qt", [S.Q8_0, S.Q4_K, S.Q6_K], ids=lambda t: S.TYPE_NAMES[t])
@pytest.mark.parametrize("rows", [1, 40])
def test_long_rows_with_loud_blocks_at_both_ends(gpu, orc, qt, rows):
    """Rows of 264 super-blocks' length: more blocks than a wave looks up in one step."""
    k, n, experts = 264 * 256, 20, 1
    w = S.make_weight(qt, n, k, 71)
    for block in (1, 264 * 8 - 6):
        w = _silence(w, qt, n, k, block)
    x = S.make_activation(rows, k, 72)
    for block in (1, 264 * 8 - 6):
        x = _loud(x, block, 25)
    x[-1, 32 * 8 * 260:32 * 8 * 260 + 32] *= np.float32(2.0 ** 20)  # not silent: its products are most of the sum
    ids = np.zeros((rows, 1), np.int32)
    y = gpu.moe_matmul_dev(_cu(x), _cu(w), qt, n, _route(gpu, ids, experts)).cpu().numpy()
    want, bound = _products(orc, w, qt, x, ids, 1, experts, n, k)
    assert (np.abs(y - want) <= bound).all(), float((np.abs(y - want) / bound).max())


def test_a_captured_call_takes_rows_of_any_spread(gpu, orc):
    """A graph captured on ordinary rows, replayed on rows with blocks apart and on ordinary ones again."""
    import torch
    qt, rows, experts, k, n = S.Q4_K, 24, 4, 512, 96
    w = _cu(S.make_weight(qt, experts * n, k, 81))
    near = S.make_activation(rows, k, 82)
    x = _cu(near)
    g = _route(gpu, (np.arange(rows, dtype=np.int32) % experts).reshape(rows, 1), experts)
    run = lambda: gpu.moe_matmul_dev(x, w, qt, n, g)  # noqa: E731
    run()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            y = run()
    torch.cuda.current_stream().wait_stream(s)
    for i in range(6):
        x.copy_(_cu(_loud(near, i, 30, every=i + 1) if i % 2 else near))
        graph.replay()
        eager = run()
        torch.cuda.synchronize()
        assert torch.equal(y, eager)


@pytest.mark.parametrize("rows", [2, 70])
def test_rows_of_subnormals(gpu, orc, rows):
    """Rows whose blocks' largest elements are subnormals (scales round up to twice their value there, codes to -128),
    alone and beside a loud block; weights that bring the products back to normal numbers."""
    k, n, experts = 512, 40, 1
    w = S.make_weight(S.Q8_0, n, k, 9).reshape(n, -1, 34).copy()
    w[:, :, :2] = np.full(2, 30000, np.float16).view(np.uint8)[:2]
    rng = np.random.default_rng(rows)
    tops = rng.choice([1, 63, 64, 65, 100, 127, 128, 190, 191, 255, 4000, 70000, 1 << 22, 1 << 25], (rows, k // 32, 1))
    x = (rng.integers(-tops, tops + 1, (rows, k // 32, 32)) * 2.0 ** -149).astype(np.float32)
    x[:, :, 3:4] = (tops * 2.0 ** -149).astype(np.float32)
    x[1::2, 4] *= np.float32(2.0 ** 90)
    x[0] = np.where(np.arange(k // 32)[:, None] == 2, x[0], 0)
    x = x.reshape(rows, k)
    y = gpu.moe_matmul_dev(_cu(x), _cu(w.reshape(-1)), S.Q8_0, n, _route(gpu, np.zeros((rows, 1), np.int32), experts))
    want, bound = _products(orc, w, S.Q8_0, x, np.zeros((rows, 1), np.int32), 1, experts, n, k)
    # (a result among the subnormals is rounded to a step of 2^-149)
    assert (np.abs(y.cpu().numpy() - want) <= bound + 2.0 ** -149).all()
