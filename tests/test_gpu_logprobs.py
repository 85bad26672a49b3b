"""Log probabilities on an MI355X against 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _exact(x, tok, top_k):
    """In 64 bits, rows of finite values and -inf with at least one finite."""
    x = x.astype(np.float64)
    m = x.max(1, keepdims=True)
    with np.errstate(invalid="ignore"):
        # log S as log1p of the sum without one largest term: a confident row's is below 2^-53
        e = np.exp(x - m)
        e[np.arange(len(x)), x.argmax(1)] = 0
        log_s = np.log1p(e.sum(1))
        lse = m[:, 0] + log_s
        lp = (x - m) - log_s[:, None]
        p = np.exp(lp)
        # sum p (lse - x), the terms without probability left out
        ent = np.where(p > 0, p * np.where(p > 0, -lp, 0), 0).sum(1)
    order = np.argsort(-x, axis=1, kind="stable")
    place = np.empty_like(order)
    np.put_along_axis(place, order, np.arange(x.shape[1])[None], 1)
    i = np.arange(len(x))
    return lse, lp[i, tok], place[i, tok], ent, order[:, :top_k], np.take_along_axis(lp, order[:, :top_k], 1)


def _check(gpu, x, tok, top_k, logits=None):
    """Tolerances: log S is off by the mean of its terms' relative errors, |x - m| 2^-23 (the product
    with log2 e and its rounding) + 2^-22 (the exponential) + 40 * 2^-24 (the sums): the mean of |x - m|
    under the weights is at most entropy + log S, here below 2 * 13. The results round once more. The
    entropy's terms have the same relative errors twice over."""
    import torch
    t = torch.from_numpy(np.asarray(tok, np.int32)).cuda()
    r = gpu.logprobs_dev(torch.from_numpy(x).cuda() if logits is None else logits, t, top_k=top_k)
    lse, lp, rank, ent, ids, tops = _exact(x, tok, top_k)
    d_log = 26 * 2.0 ** -23 + 2.0 ** -22 + 40 * 2.0 ** -24
    got = {n: getattr(r, n).cpu().numpy() for n in ("logprobs", "ranks", "entropy", "lse", "top_ids", "top_logprobs")}
    assert np.array_equal(got["ranks"], rank)
    assert np.array_equal(got["top_ids"], ids)
    for name, want in (("lse", lse), ("logprobs", lp), ("top_logprobs", tops)):
        inf = np.isinf(want)
        assert np.array_equal(np.isneginf(got[name]), inf), name
        err = np.abs(np.where(inf, 0, got[name]) - np.where(inf, 0, want))
        assert (err <= d_log + np.where(inf, 0, np.abs(want)) * 2.0 ** -23).all(), (name, float(err.max()))
    # a confident row: log S = log1p(S') keeps relative precision
    assert (np.abs(got["entropy"] - ent) <= ent * (2 * d_log + 2.0 ** -21)).all()
    best = np.abs(got["top_logprobs"][:, 0] - tops[:, 0]) if top_k else np.zeros(1)
    assert top_k == 0 or (best <= np.abs(tops[:, 0]) * (d_log + 2.0 ** -22)).all()
    return got


@pytest.mark.parametrize("rows,vocab,top_k", [(1, 1, 1), (3, 2, 2), (5, 7, 0), (2, 64, 64), (4, 1000, 20),
                                              (3, 8191, 5), (2, 8192, 64), (3, 8193, 64), (2, 32003, 20),
                                              (1, 128256, 5), (3, 151936, 64), (65, 50257, 1)])
@pytest.mark.parametrize("kind", ["plain", "ties", "masked", "sharp"])
def test_logprobs(gpu, rows, vocab, top_k, kind):
    rng = np.random.default_rng(rows * 1000 + vocab)
    x = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    if kind == "ties":
        x = np.round(x * 4) / 4
    if kind == "sharp":
        x[np.arange(rows), rng.integers(0, vocab, rows)] += 40 * rng.random(rows).astype(np.float32)
    if kind == "masked":  # a grammar leaves a few tokens
        keep = rng.random((rows, vocab)) < 12 / vocab
        keep[:, rng.integers(0, vocab)] = True
        x = np.where(keep, x, np.float32(-np.inf))
    print("logprobs", rows, vocab, top_k, kind, flush=True)
    tok = np.where(rng.random(rows) < 0.5, x.argmax(1), rng.integers(0, vocab, rows))
    _check(gpu, x, tok, top_k)


def test_many_large_logits_in_every_part(gpu):
    """Sixty-three of the 64 wanted could come from any stretch of the vocabulary but the last, whose
    logits are low: no bound of the stretches' lists leaves few."""
    rng = np.random.default_rng(8)
    vocab, stretch = 151936, 8192
    x = rng.standard_normal((3, vocab)).astype(np.float32)
    for row in x:
        for z in range(vocab // stretch):
            row[z * stretch + rng.permutation(stretch)[:63]] = rng.uniform(50, 60, 63)
    _check(gpu, x, x.argmax(1), 64)
    _check(gpu, x, rng.integers(0, vocab, 3), 20)


def test_equal_logits_stand_in_the_order_of_their_ids(gpu):
    """Rows of one value, and of two, over several parts; the lists keep the lowest ids."""
    x = np.zeros((4, 20000), np.float32)
    x[1, 7::3] = -0.0
    x[2, 100:] = -1
    x[2, :50] = -5
    x[3, ::2] = np.float32(1e-30)
    _check(gpu, x, np.array([19999, 8, 12345, 1]), 64)
    # descending and ascending rows: one wave's logits are the largest
    y = np.stack([np.linspace(0, -9, 9000), np.linspace(-9, 0, 9000)]).astype(np.float32)
    _check(gpu, y, np.array([4500, 4500]), 64)


def test_strided_rows_and_tokens_outside(gpu):
    import torch
    rng = np.random.default_rng(4)
    x = rng.standard_normal((6, 333)).astype(np.float32)
    wide = torch.full((6, 401), float("nan"), device="cuda")
    wide[:, 3:336] = torch.from_numpy(x).cuda()
    _check(gpu, x, np.array([0, 5, 332, 1, 2, 3]), 9, logits=wide[:, 3:336])
    r = gpu.logprobs_dev(torch.from_numpy(x).cuda(), torch.tensor([-1, 333, 1 << 30, -7, 0, 332], dtype=torch.int32,
                                                                  device="cuda"))
    lp, rank = r.logprobs.cpu().numpy(), r.ranks.cpu().numpy()
    assert np.isneginf(lp[:4]).all() and (rank[:4] == -1).all() and np.isfinite(lp[4:]).all() and (rank[4:] >= 0).all()
    assert r.top_ids.shape == (6, 0)
    assert gpu.logprobs_dev(torch.from_numpy(x).cuda()).logprobs is None
    assert gpu.logprobs_dev(torch.zeros(0, 5, device="cuda"), top_k=2).top_ids.shape == (0, 2)


def test_rows_without_a_finite_maximum(gpu):
    """All -inf: nothing is possible. NaN or +inf: NaN, the order with NaN last."""
    import torch
    n = 9000
    x = np.random.default_rng(6).standard_normal((5, n)).astype(np.float32)
    x[0] = -np.inf
    x[1, 8500] = np.nan
    x[2, 17] = np.inf
    x[3] = np.nan
    x[3, 5], x[3, 8999], x[3, 7] = 1.0, 2.0, -np.inf
    r = gpu.logprobs_dev(torch.from_numpy(x).cuda(), torch.zeros(5, dtype=torch.int32, device="cuda"), top_k=6)
    lp, tops, ids = r.logprobs.cpu().numpy(), r.top_logprobs.cpu().numpy(), r.top_ids.cpu().numpy()
    ent, lse = r.entropy.cpu().numpy(), r.lse.cpu().numpy()
    assert np.isneginf(lp[0]) and np.isneginf(lse[0]) and ent[0] == 0 and np.isneginf(tops[0]).all()
    assert ids[0].tolist() == [0, 1, 2, 3, 4, 5]
    for i in (1, 2, 3):
        assert np.isnan(lp[i]) and np.isnan(lse[i]) and np.isnan(ent[i]) and np.isnan(tops[i]).all(), i
    assert ids[1].tolist() == np.argsort(-np.nan_to_num(x[1], nan=-np.inf), kind="stable")[:6].tolist()
    assert ids[2, 0] == 17
    assert ids[3].tolist() == [8999, 5, 7, 0, 1, 2]
    assert np.isfinite(lp[4])


def test_captured(gpu):
    """A captured call replayed with new logits gives the eager bits, whatever ran between."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(3, 20011, device="cuda", generator=gen)
    t = torch.tensor([1, 2, 20010], dtype=torch.int32, device="cuda")
    gpu.logprobs_dev(x, t, top_k=5)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = gpu.logprobs_dev(x, t, top_k=5)
    for i in range(4):
        x.copy_(torch.randn(3, 20011, device="cuda", generator=gen))
        g.replay()
        e = gpu.logprobs_dev(x, t, top_k=5)
        torch.cuda.synchronize()
        for name in ("logprobs", "ranks", "entropy", "lse", "top_ids", "top_logprobs"):
            assert torch.equal(getattr(r, name), getattr(e, name)), (i, name)
        torch.randn(1 << 20, device="cuda")


def test_masks_of_finite_values(gpu):
    """Rows whose masked tokens hold the type's lowest value, or another far below the rest, over whole parts
    of the vocabulary; and one token far above all others: finite, with the probabilities of -inf masks."""
    rng = np.random.default_rng(12)
    for vocab in (8193, 20000, 50257):
        x = (rng.standard_normal((8, vocab)) * 3).astype(np.float32)
        low = np.finfo(np.float32).min
        x[0, 8192:] = low                       # the last part
        x[1, :8192] = low                       # the first part
        x[2, 100:] = -1e38
        x[3] = low
        x[3, [7, 8192]] = [1.0, 2.5]            # two tokens left
        x[4, 8190:] = -np.inf                   # both kinds of masks
        x[4, 8192:] = low
        x[5, 8192] = 3e38                       # (differences past fp32's range from here)
        x[6, 5:] = -1e30
        x[7, :] = low                           # nothing but the mask: equal probabilities
        tok = np.array([8192, 5, 3, 8192, 8192, 8192, 4, vocab - 1])
        for top_k in (0, 5, 64):
            got = _check(gpu, x, tok, top_k)
            assert all(np.isfinite(got[n]).all() for n in ("entropy", "lse")), vocab
            assert np.isfinite(got["logprobs"]).all()
