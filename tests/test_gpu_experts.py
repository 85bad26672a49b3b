"""Entries grouped by index, the router and the experts' products on an MI355X against 64 bits."""
import ctypes

import numpy as np
import pytest

import expert_model as M
from cllm_inference_amd import synth as S

pytestmark = pytest.mark.gpu

TYPES = [S.Q4_0, S.Q5_0, S.Q8_0, S.Q4_K, S.Q5_K, S.Q6_K]


def _cu(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


# ---- entries grouped by index ---------------------------------------------------------------------

@pytest.mark.parametrize("n", [0, 1, 2, 63, 64, 65, 1023, 1025, 70001])
@pytest.mark.parametrize("groups", [1, 2, 7, 64, 65, 1000, 1024])
def test_group_rows(gpu, n, groups):
    rng = np.random.default_rng(n * 7 + groups)
    ids = rng.integers(-2, groups + 2, n).astype(np.int32)
    if n > 4:
        ids[:2] = [np.iinfo(np.int32).min, np.iinfo(np.int32).max]
    print("group_rows", n, groups, flush=True)
    g = gpu.group_rows_dev(_cu(ids), groups)
    offsets, order = M.grouped(ids, groups)
    assert np.array_equal(g.offsets.cpu().numpy(), offsets)
    assert np.array_equal(g.order.cpu().numpy(), order)


def test_group_rows_of_one_group(gpu):
    """Every entry of the same group, and none of any."""
    for v in (3, -1):
        ids = np.full(5000, v, np.int32)
        g = gpu.group_rows_dev(_cu(ids), 5)
        offsets, order = M.grouped(ids, 5)
        assert np.array_equal(g.offsets.cpu().numpy(), offsets) and np.array_equal(g.order.cpu().numpy(), order)


# ---- the router -------------------------------------------------------------------------------------

def _check_route(gpu, z, top_k, logits=None, **kw):
    parts = dict(parts=kw.pop("n_groups", 1), top_parts=kw.pop("top_groups", 1))
    bias = kw.pop("bias", None)
    r = gpu.moe_route_dev(_cu(z) if logits is None else logits, top_k, bias=None if bias is None else _cu(bias),
                          n_groups=parts["parts"], top_groups=parts["top_parts"], **kw)
    ids, w = M.route(z, top_k, bias, **parts, **kw)
    assert np.array_equal(r.ids.cpu().numpy(), ids)
    # formed in 64 bits and rounded once (2^-24 of the value); the smallest of fp32 round by 2^-150
    got = r.weights.cpu().numpy()
    assert (np.abs(got - w) <= np.abs(w) * 2.0 ** -23 + 2.0 ** -149).all(), np.abs(got - w).max()
    offsets, order = M.grouped(ids.reshape(-1), z.shape[1])
    assert np.array_equal(r.offsets.cpu().numpy(), offsets)
    assert np.array_equal(r.order.cpu().numpy(), order)
    return r


@pytest.mark.parametrize("rows,experts,top_k", [(1, 1, 1), (1, 8, 2), (3, 60, 4), (64, 64, 8), (65, 65, 5),
                                                (7, 128, 32), (33, 160, 6), (300, 256, 8), (17, 512, 10),
                                                (5, 1000, 3), (200, 1024, 32)])
@pytest.mark.parametrize("kind", ["softmax", "sigmoid", "raw", "bias"])
def test_route(gpu, rows, experts, top_k, kind):
    rng = np.random.default_rng(rows * 13 + experts)
    z = (rng.standard_normal((rows, experts)) * 2).astype(np.float32)
    print("route", rows, experts, top_k, kind, flush=True)
    kw = {"softmax": {}, "sigmoid": dict(sigmoid=True, scale=2.5), "raw": dict(normalise=False),
          "bias": dict(sigmoid=True, bias=(rng.standard_normal(experts) * 0.2).astype(np.float32))}[kind]
    _check_route(gpu, z, top_k, **kw)


@pytest.mark.parametrize("rows,experts,n_groups,top_groups,top_k", [
    (9, 8, 2, 1, 2), (70, 256, 8, 4, 8), (5, 64, 64, 5, 5), (3, 60, 4, 4, 6), (40, 1024, 64, 3, 9),
    (66, 160, 5, 2, 8), (4, 6, 3, 1, 2)])
@pytest.mark.parametrize("biased", [False, True])
def test_route_from_the_best_groups(gpu, rows, experts, n_groups, top_groups, top_k, biased):
    rng = np.random.default_rng(experts + n_groups)
    z = rng.standard_normal((rows, experts)).astype(np.float32)
    bias = (rng.standard_normal(experts) * 0.3).astype(np.float32) if biased else None
    for sigmoid in (False, True):
        _check_route(gpu, z, top_k, bias=bias, sigmoid=sigmoid, n_groups=n_groups, top_groups=top_groups,
                     normalise=not sigmoid)


def test_route_ties_go_to_the_lower_expert(gpu):
    rng = np.random.default_rng(5)
    z = np.round(rng.standard_normal((40, 96)) * 2).astype(np.float32) / 2
    z[3] = 0.0
    z[4, ::2] = -0.0
    _check_route(gpu, z, 8)
    _check_route(gpu, z, 8, n_groups=8, top_groups=3)
    # 192 experts are four to a lane
    _check_route(gpu, np.concatenate([z, z], 1), 9, sigmoid=True)


def test_route_masks_and_values_that_are_not_finite(gpu):
    """Masked experts are never chosen; a row that masks leave fewer than top_k has -1 behind them, an empty
    one nothing; logits of the type's lowest value are numbers; infinite ones share."""
    rng = np.random.default_rng(6)
    z = rng.standard_normal((12, 16)).astype(np.float32)
    z[0] = -np.inf
    z[1] = np.nan
    z[2, 3:] = -np.inf
    z[3, 1:] = np.nan
    z[4, 2:] = np.finfo(np.float32).min
    z[5] = np.finfo(np.float32).min
    z[6, [4, 9]] = np.inf
    z[7, 5] = np.nan
    z[8] = 3e38
    z[9] = -3e38
    z[9, 2] = 3e38
    z[10, 8:] = -np.inf
    for kw in ({}, dict(normalise=False), dict(sigmoid=True, normalise=False), dict(sigmoid=True),
               dict(n_groups=4, top_groups=2)):
        _check_route(gpu, z, 5, **kw)
    bias = rng.standard_normal(16).astype(np.float32)
    bias[1] = -np.inf
    bias[2] = np.nan
    for kw in ({}, dict(sigmoid=True, normalise=False), dict(n_groups=2, top_groups=1)):
        _check_route(gpu, z, 5, bias=bias, **kw)


def test_route_rows_apart(gpu):
    """Rows of a wider tensor; top_k of all experts; no rows."""
    import torch
    rng = np.random.default_rng(7)
    wide = _cu(rng.standard_normal((70, 40)).astype(np.float32))
    part = wide[:, 3:27]
    _check_route(gpu, part.cpu().numpy(), 24, logits=part)
    r = gpu.moe_route_dev(torch.empty((0, 24), device="cuda"), 4)
    assert r.ids.shape == (0, 4) and not r.offsets.any()


# ---- the experts' products --------------------------------------------------------------------------

def _ids(rng, rows, experts, top_k, kind="spread"):
    if kind == "one":  # all of one expert
        return np.tile(np.arange(top_k, dtype=np.int32), (rows, 1))
    ids = np.argsort(rng.random((rows, experts)) + 0.3 * rng.random(experts), 1)[:, :top_k].astype(np.int32)
    if kind == "dropped":
        ids[rng.random(ids.shape) < 0.4] = -1
        ids[0, 0] = experts + 3
    return ids


def _groups(gpu, ids, experts):
    offsets, order = M.grouped(ids.reshape(-1), experts)
    return gpu.MoeRoute(_cu(ids), None, _cu(offsets), _cu(order))


def _norm(a):
    return np.sqrt((a.astype(np.float64) ** 2).sum())


def _entry_products(orc, x, per_row, ids, values, mags, k):
    """[entries][n] products and bounds of the entries with an expert (others NaN)."""
    flat = ids.reshape(-1)
    xr = M.q8_values(orc, x)
    n = values.shape[1]
    y = np.full((flat.size, n), np.nan)
    b = np.zeros((flat.size, n))
    for e in range(values.shape[0]):
        at = np.nonzero(flat == e)[0]
        if at.size:
            rows = xr[at // per_row]
            y[at] = rows @ values[e].T
            b[at] = M.product_bound(mags[e], rows, k)
    return y, b


# rows x per_row entries over the experts: single tokens, a few rows to an expert, tens (32-entry tiles),
# hundreds (64-entry tiles, more than one to an expert); weight rows no multiple of any tile; odd lengths
SHAPES = [(1, 4, 1, 256, 16), (1, 8, 2, 512, 100), (2, 2, 2, 2048, 33), (5, 16, 3, 768, 257), (33, 8, 2, 256, 130),
          (24, 2, 2, 512, 290), (150, 3, 1, 768, 300), (90, 2, 2, 256, 70), (13, 2, 1, 8192, 40), (3, 4, 1, 8448, 65)]


@pytest.mark.parametrize("qt", TYPES, ids=lambda t: S.TYPE_NAMES[t])
@pytest.mark.parametrize("rows,experts,per_row,k,n", SHAPES)
@pytest.mark.parametrize("kind", ["spread", "dropped", "one"])
def test_moe_matmul(gpu, orc, qt, rows, experts, per_row, k, n, kind):
    import torch
    rng = np.random.default_rng(qt * 100 + rows)
    if qt in (S.Q4_0, S.Q5_0, S.Q8_0):
        k += 32 * (rows % 5) + (96 if rows == 1 else 0)  # rows that end inside a super-block's length
    w = S.make_weight(qt, experts * n, k, 11 + rows)
    x = S.make_activation(rows, k, 5 + rows, outliers=True)
    ids = _ids(rng, rows, experts, per_row, kind)
    g = _groups(gpu, ids, experts)
    print("moe_matmul", S.TYPE_NAMES[qt], rows, experts, per_row, k, n, kind,
          gpu.moe_plan(qt, 1, k, n, experts, rows * per_row), flush=True)
    y = torch.full((rows * per_row, n), 7.5, device="cuda")
    bias = rng.standard_normal((experts, n)).astype(np.float32)
    gpu.moe_matmul_dev(_cu(x), _cu(w), qt, n, g, bias=_cu(bias), per_row=per_row, y=y)
    values, mags = M.expert_values(w, qt, experts, n, k)
    want, bound = _entry_products(orc, x, per_row, ids, values, mags, k)
    flat = ids.reshape(-1)
    live = (flat >= 0) & (flat < experts)
    got = y.cpu().numpy()
    assert (got[~live] == 7.5).all()  # entries of no expert: left as they were
    if not live.any():
        return
    full = want[live] + bias[flat[live]]
    err = np.abs(got[live] - full)
    # (the bias adds one rounding)
    assert (err <= bound[live] + np.abs(full) * 2.0 ** -24).all(), float((err / bound[live]).max())
    # roundings of either sign in some 40 places: far inside the bound together
    assert _norm(err) <= 2.0 ** -20 * _norm(full), _norm(err) / _norm(full)


@pytest.mark.parametrize("qt", TYPES, ids=lambda t: S.TYPE_NAMES[t])
@pytest.mark.parametrize("rows,experts,top_k,k,n", [(1, 8, 2, 512, 48), (7, 16, 4, 256, 113), (60, 4, 2, 512, 130),
                                                    (200, 3, 2, 256, 257)])
def test_moe_swiglu(gpu, orc, qt, rows, experts, top_k, k, n):
    rng = np.random.default_rng(qt + rows)
    wg, wu = S.make_weight(qt, experts * n, k, 3), S.make_weight(qt, experts * n, k, 4)
    x = S.make_activation(rows, k, 9)
    ids = _ids(rng, rows, experts, top_k)
    print("moe_swiglu", S.TYPE_NAMES[qt], rows, experts, top_k, k, n, gpu.moe_plan(qt, 2, k, n, experts, rows * top_k),
          flush=True)
    bg, bu = (rng.standard_normal((experts, n)).astype(np.float32) for _ in range(2))
    h = gpu.moe_swiglu_dev(_cu(x), _cu(wg), _cu(wu), qt, n, _groups(gpu, ids, experts), bias_gate=_cu(bg),
                           bias_up=_cu(bu)).cpu().numpy().reshape(-1, n)
    flat = ids.reshape(-1)
    g, eg = _entry_products(orc, x, top_k, ids, *M.expert_values(wg, qt, experts, n, k), k)
    u, eu = _entry_products(orc, x, top_k, ids, *M.expert_values(wu, qt, experts, n, k), k)
    g, u = g + bg[flat], u + bu[flat]
    eg, eu = eg + np.abs(g) * 2.0 ** -24, eu + np.abs(u) * 2.0 ** -24
    want = M.silu(g) * u
    # |silu'| <= 1.1; expf within 2 steps (2^-22 of exp, which 1 + exp only dampens), the sum, quotient and product
    bound = 1.1 * eg * (np.abs(u) + eu) + np.abs(M.silu(g)) * eu + np.abs(want) * 2.0 ** -21 + 2.0 ** -126
    err = np.abs(h - want)
    assert (err <= bound).all(), float((err / bound).max())
    assert _norm(err) <= 2.0 ** -19 * _norm(want), _norm(err) / _norm(want)


@pytest.mark.parametrize("qt", TYPES, ids=lambda t: S.TYPE_NAMES[t])
@pytest.mark.parametrize("rows,tile", [(1, "<8,4>"), (7, "<4,8>")])
def test_swiglu_of_long_rows_with_an_expert_chosen_twice(gpu, orc, qt, rows, tile):
    rng = np.random.default_rng(qt + rows)
    experts, k, n = 2, 8448, 37
    assert tile in gpu.moe_plan(qt, 2, k, n, experts, rows * 2)
    wg, wu = S.make_weight(qt, experts * n, k, 31), S.make_weight(qt, experts * n, k, 32)
    x = S.make_activation(rows, k, 33)
    ids = rng.integers(0, experts, (rows, 2)).astype(np.int32)
    ids[0] = 1  # the same expert in both places
    h = gpu.moe_swiglu_dev(_cu(x), _cu(wg), _cu(wu), qt, n, _groups(gpu, ids, experts)).cpu().numpy().reshape(-1, n)
    assert np.array_equal(h[0], h[1])
    g, eg = _entry_products(orc, x, 2, ids, *M.expert_values(wg, qt, experts, n, k), k)
    u, eu = _entry_products(orc, x, 2, ids, *M.expert_values(wu, qt, experts, n, k), k)
    want = M.silu(g) * u
    # as above
    bound = 1.1 * eg * (np.abs(u) + eu) + np.abs(M.silu(g)) * eu + np.abs(want) * 2.0 ** -21 + 2.0 ** -126
    assert (np.abs(h - want) <= bound).all(), float((np.abs(h - want) / bound).max())


@pytest.mark.parametrize("qt", TYPES, ids=lambda t: S.TYPE_NAMES[t])
@pytest.mark.parametrize("rows,experts,top_k,k,n", [(1, 8, 2, 512, 64), (9, 16, 4, 256, 99), (70, 4, 2, 768, 130)])
@pytest.mark.parametrize("kind", ["spread", "dropped"])
def test_moe_down(gpu, orc, qt, rows, experts, top_k, k, n, kind):
    rng = np.random.default_rng(qt + rows)
    w = S.make_weight(qt, experts * n, k, 21)
    h = S.make_activation(rows * top_k, k, 22)
    ids = _ids(rng, rows, experts, top_k, kind)
    if kind == "dropped":
        ids[rows // 2] = -1
    p = rng.random((rows, top_k)).astype(np.float32)
    base = rng.standard_normal((rows, n)).astype(np.float32)
    bias = rng.standard_normal((experts, n)).astype(np.float32)
    r = _groups(gpu, ids, experts)
    r.weights = _cu(p)
    print("moe_down", S.TYPE_NAMES[qt], rows, experts, top_k, k, n, kind, flush=True)
    flat = ids.reshape(-1)
    live = ((flat >= 0) & (flat < experts)).reshape(rows, top_k, 1)
    v, bound = _entry_products(orc, h, 1, ids, *M.expert_values(w, qt, experts, n, k), k)
    v = v + np.where(live.reshape(-1, 1), bias[np.where(live.reshape(-1), flat, 0)], 0)
    v = np.where(live, np.nan_to_num(v).reshape(rows, top_k, n), 0)
    terms = v * p[..., None]
    want = terms.sum(1)
    # a rounding of each term's product, bias and sum beside the products' own
    tol = (bound.reshape(rows, top_k, n) * p[..., None]).sum(1) + (np.abs(terms).sum(1) * (top_k + 2) + np.abs(base)) * 2.0 ** -24
    args = (_cu(h), _cu(w), qt, n, r)
    y = gpu.moe_down_dev(*args, bias=_cu(bias)).cpu().numpy()
    assert (np.abs(y - want) <= tol).all()
    if kind == "dropped":
        assert (y[rows // 2] == 0).all()
    b = _cu(base)
    out = gpu.moe_down_dev(*args, bias=_cu(bias), base=b)
    assert (np.abs(out.cpu().numpy() - (want + base)) <= tol + np.abs(want + base) * 2.0 ** -24).all()
    same = gpu.moe_down_dev(*args, bias=_cu(bias), base=b, y=b)  # the residual in place
    assert same is b and np.array_equal(b.cpu().numpy(), out.cpu().numpy())


@pytest.mark.parametrize("qt", TYPES, ids=lambda t: S.TYPE_NAMES[t])
@pytest.mark.parametrize("rows", [3, 100])
def test_rows_that_are_not_finite_tiny_or_huge(gpu, orc, qt, rows):
    """A row with an infinity or a NaN gives NaN and touches no other; rows at the ends of fp32's range
    keep their relative precision; a row of zeros gives zeros."""
    k, n, experts = 512, 70, 2
    w = S.make_weight(qt, experts * n, k, 31)
    x = S.make_activation(rows, k, 32)
    clean = gpu.moe_matmul_dev(_cu(x), _cu(w), qt, n, _groups(gpu, np.zeros((rows, 1), np.int32), experts)).cpu().numpy()
    x[0] = 0
    x[1, 5] = np.inf
    x[2, 100] = np.nan
    bad = [1, 2]
    scale = {}
    if rows > 3:
        scale = {10: 2.0 ** -100, 11: 2.0 ** 90, 12: 2.0 ** -20}
        for r, s in scale.items():
            x[r] *= np.float32(s)
    y = gpu.moe_matmul_dev(_cu(x), _cu(w), qt, n, _groups(gpu, np.zeros((rows, 1), np.int32), experts)).cpu().numpy()
    assert (y[0] == 0).all() and np.isnan(y[bad]).all()
    for r in range(3, rows):
        assert np.array_equal(y[r], clean[r] * np.float32(scale.get(r, 1.0))), r


@pytest.mark.parametrize("qt", [S.Q8_0, S.Q4_K, S.Q6_K], ids=lambda t: S.TYPE_NAMES[t])
@pytest.mark.parametrize("rows", [2, 40, 150])
def test_a_weight_row_that_is_not_finite_spoils_its_own_outputs(gpu, qt, rows):
    k, n, experts = 512, 70, 2
    size = S.row_bytes(qt, k)
    w = S.make_weight(qt, experts * n, k, 41).reshape(experts * n, size)
    x = S.make_activation(rows, k, 42)
    g = _groups(gpu, np.ones((rows, 1), np.int32), experts)
    clean = gpu.moe_matmul_dev(_cu(x), _cu(w.reshape(-1)), qt, n, g).cpu().numpy()
    w2 = w.copy()
    at = 208 if qt == S.Q6_K else 0
    w2[n + 7, at:at + 2] = np.array([np.nan], np.float16).view(np.uint8)
    y = gpu.moe_matmul_dev(_cu(x), _cu(w2.reshape(-1)), qt, n, g).cpu().numpy()
    assert np.isnan(y[:, 7]).all()
    assert np.array_equal(np.delete(y, 7, 1), np.delete(clean, 7, 1))


def test_experts_past_4_gib(gpu, orc):
    """The last of 80 experts of 14336 x 4096 Q8_0 (5 GB): offsets past 32 bits, both kernels."""
    import torch
    qt, n, k, experts = S.Q8_0, 14336, 4096, 80
    one = S.make_weight(qt, n, k, 51)
    w = torch.zeros((experts, one.size), dtype=torch.uint8, device="cuda")
    w[experts - 1] = _cu(one.reshape(-1))
    for rows in (1, 100):
        x = S.make_activation(rows, k, 52)
        ids = np.full((rows, 1), experts - 1, np.int32)
        ids[0] = 40 if rows > 1 else experts - 1
        y = gpu.moe_matmul_dev(_cu(x), w, qt, n, _groups(gpu, ids, experts)).cpu().numpy()
        if rows > 1:
            assert (y[0] == 0).all()  # an expert of zeros
        values, mags = M.expert_values(one, qt, 1, n, k)
        xr = M.q8_values(orc, x[-1:])
        assert (np.abs(y[-1:] - xr @ values[0].T) <= M.product_bound(mags[0], xr, k)).all()


def test_bad_offsets_and_order_stay_in_bounds(gpu):
    """Entries out of range are no entries, whatever offsets and order hold; outputs beside them are as ever."""
    import torch
    qt, n, k, experts, rows = S.Q4_0, 40, 64, 4, 50
    w, x = _cu(S.make_weight(qt, experts * n, k, 1)), _cu(S.make_activation(rows, k, 2))
    order = np.arange(rows, dtype=np.int32)
    order[3], order[9] = -5, 1 << 30
    offsets = np.array([0, 10, 20, 30, 50], np.int32)
    good = gpu.moe_matmul_dev(x, w, qt, n, gpu.RowGroups(_cu(offsets), _cu(np.arange(rows, dtype=np.int32))))
    for off in (offsets, np.array([0, 10, 20, 30, 1 << 30], np.int32), np.array([-7, 10, 20, 30, 60], np.int32),
                np.array([0, 0, 0, 0, 0], np.int32)):
        y = torch.full((rows, n), 3.0, device="cuda")
        gpu.moe_matmul_dev(x, w, qt, n, gpu.RowGroups(_cu(off), _cu(order)), y=y)
        y = y.cpu().numpy()
        assert (y[3] == 3.0).all() and (y[9] == 3.0).all()
        if off is offsets:
            keep = np.delete(np.arange(rows), [3, 9])
            assert np.array_equal(y[keep], good.cpu().numpy()[keep])


# ---- together, captured, on other streams ---------------------------------------------------------------

class _Layer:
    """A feed-forward of experts as a model has it: router, gate and up, down, residual."""

    def __init__(self, gpu, rows, experts=8, top_k=2, k=256, n_ff=512, qt=S.Q4_K, qd=S.Q6_K, seed=0):
        rng = np.random.default_rng(seed)
        self.gpu, self.k, self.n_ff, self.qt, self.qd, self.top_k = gpu, k, n_ff, qt, qd, top_k
        self.router = rng.standard_normal((experts, k)).astype(np.float32) / 16
        self.wg, self.wu = (S.make_weight(qt, experts * n_ff, k, seed + i) for i in (1, 2))
        self.wd = S.make_weight(qd, experts * k, n_ff, seed + 3)
        self.x = _cu(S.make_activation(rows, k, seed + 4))
        self.dev = [_cu(a.reshape(-1)) for a in (self.router.view(np.uint8), self.wg, self.wu, self.wd)]
        self.experts = experts

    def run(self, x):
        g = self.gpu
        logits = g.matmul_quant_dev(x, self.dev[0], S.F32 if hasattr(S, "F32") else 0, None, self.k, self.experts)
        r = g.moe_route_dev(logits, self.top_k)
        h = g.moe_swiglu_dev(x, self.dev[1], self.dev[2], self.qt, self.n_ff, r)
        return logits, r, h, g.moe_down_dev(h, self.dev[3], self.qd, self.k, r, base=x)


@pytest.mark.parametrize("rows", [1, 6, 100])
def test_a_layer(gpu, orc, rows):
    lay = _Layer(gpu, rows)
    logits, r, h, y = lay.run(lay.x)
    x = lay.x.cpu().numpy()
    z = logits.cpu().numpy()
    assert np.abs(z - x.astype(np.float64) @ lay.router.T).max() < 1e-4
    ids, p = M.route(z, lay.top_k)
    assert np.array_equal(r.ids.cpu().numpy(), ids)
    hv = h.cpu().numpy().reshape(-1, lay.n_ff)
    g, eg = _entry_products(orc, x, lay.top_k, ids, *M.expert_values(lay.wg, lay.qt, lay.experts, lay.n_ff, lay.k), lay.k)
    u, eu = _entry_products(orc, x, lay.top_k, ids, *M.expert_values(lay.wu, lay.qt, lay.experts, lay.n_ff, lay.k), lay.k)
    want = M.silu(g) * u
    assert (np.abs(hv - want) <= 1.1 * eg * (np.abs(u) + eu) + np.abs(M.silu(g)) * eu + np.abs(want) * 2.0 ** -21 + 2.0 ** -126).all()
    # the down projection on the h that it was given
    v, ev = _entry_products(orc, hv, 1, ids, *M.expert_values(lay.wd, lay.qd, lay.experts, lay.k, lay.n_ff), lay.n_ff)
    terms = v.reshape(rows, lay.top_k, -1) * p[..., None]
    out = terms.sum(1) + x
    tol = (ev.reshape(rows, lay.top_k, -1) * p[..., None]).sum(1) + (np.abs(terms).sum(1) * 4 + 2 * np.abs(x) + np.abs(out)) * 2.0 ** -23
    assert (np.abs(y.cpu().numpy() - out) <= tol).all()


@pytest.mark.parametrize("rows", [1, 40])
def test_a_captured_layer_replays(gpu, rows):
    """A graph of the layer, replayed on new inputs with eager work between, gives the eager results."""
    import torch
    lay = _Layer(gpu, rows, seed=50)
    x = lay.x.clone()
    lay.run(x)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        lay.run(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs = lay.run(x)
    torch.cuda.current_stream().wait_stream(s)
    for i in range(4):
        x.copy_(_cu(S.make_activation(rows, lay.k, 60 + i)))
        graph.replay()
        eager = lay.run(x)
        torch.cuda.synchronize()
        assert torch.equal(outs[3], eager[3]) and torch.equal(outs[1].ids, eager[1].ids)
        assert torch.equal(outs[1].order, eager[1].order)
        torch.empty(1 << 20, device="cuda").fill_(float("nan"))


def test_two_streams_at_once(gpu):
    import torch
    lays = [_Layer(gpu, 30, seed=70), _Layer(gpu, 30, seed=80)]
    want = [lay.run(lay.x)[3].clone() for lay in lays]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(lays[i].run(lays[i].x)[3])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


def test_the_same_call_gives_the_same_bits(gpu):
    import torch
    lay = _Layer(gpu, 130, experts=4, seed=90)
    a = lay.run(lay.x)
    for _ in range(3):
        b = lay.run(lay.x)
        assert torch.equal(a[2], b[2]) and torch.equal(a[3], b[3])


def test_refusals_of_the_bindings(gpu):
    import torch
    qt, n, k, experts, rows = S.Q4_0, 32, 64, 4, 3
    w, x = _cu(S.make_weight(qt, experts * n, k, 1).reshape(-1)), _cu(S.make_activation(rows, k, 2))
    g = _groups(gpu, np.zeros((rows, 1), np.int32), experts)
    g.weights = torch.ones((rows, 1), device="cuda")
    bad = [
        lambda: gpu.moe_matmul_dev(x.half(), w, qt, n, g), lambda: gpu.moe_matmul_dev(x, w[:-1], qt, n, g),
        lambda: gpu.moe_matmul_dev(x, w, qt, n + 1, g), lambda: gpu.moe_matmul_dev(x.cpu(), w, qt, n, g),
        lambda: gpu.moe_matmul_dev(x, w, 3, n, g), lambda: gpu.moe_matmul_dev(x.t(), w, qt, n, g),
        lambda: gpu.moe_matmul_dev(x, w, qt, n, gpu.RowGroups(g.offsets, g.order[:2])),
        lambda: gpu.moe_matmul_dev(x, w, qt, n, gpu.RowGroups(g.offsets.long(), g.order)),
        lambda: gpu.moe_matmul_dev(x, w, qt, n, g, per_row=33), lambda: gpu.moe_matmul_dev(x, w, qt, n, g, per_row=0),
        lambda: gpu.moe_swiglu_dev(x[:2], w, w, qt, n, g), lambda: gpu.moe_swiglu_dev(x, w, w[1:], qt, n, g),
        lambda: gpu.moe_down_dev(x[:2], w, qt, n, g), lambda: gpu.moe_down_dev(x, w, qt, n, g, base=x),
        lambda: gpu.moe_route_dev(x, 0), lambda: gpu.moe_route_dev(x, 33), lambda: gpu.moe_route_dev(x, 65),
        lambda: gpu.moe_route_dev(x.t(), 2), lambda: gpu.moe_route_dev(x, 2, bias=x[0, :5]),
        lambda: gpu.moe_route_dev(x, 2, n_groups=7), lambda: gpu.moe_route_dev(x, 2, scale=float("nan")),
        lambda: gpu.group_rows_dev(x, 4), lambda: gpu.group_rows_dev(g.order, 0),
        lambda: gpu.group_rows_dev(g.order, 1025),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            print("not refused:", i)
    lib = gpu.load_library()
    y = torch.empty((rows, n), device="cuda")
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    need = lib.cllm_hip_moe_matmul_ws_bytes(qt, k, rows)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    call = lambda ws_p, nb: lib.cllm_hip_moe_matmul_dev(  # noqa: E731
        qt, k, n, experts, p(w), None, p(x), rows, 1, p(g.offsets), p(g.order), p(y), ws_p, nb, None)
    assert call(None, need) == 3 and call(p(ws), need - 1) == 3 and call(ctypes.c_void_p(ws.data_ptr() + 8), need) == 3
    assert call(p(ws), need) == 0
    torch.cuda.synchronize()
