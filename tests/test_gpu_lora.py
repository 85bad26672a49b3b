"""Low-rank adapters on an MI355X against 64 bits."""
import numpy as np
import pytest

import expert_model as M

pytestmark = pytest.mark.gpu


def _cu(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _case(rows, adapters, rank, k, outs, dt, seed, none=0.2, garbage=True):
    rng = np.random.default_rng(seed)
    c = {"x": rng.standard_normal((rows, k)).astype(np.float32)}
    c["ids"] = np.where(rng.random(rows) < none, rng.choice([-1, adapters, adapters + 9], rows),
                        rng.integers(0, adapters, rows)).astype(np.int32)
    c["ranks"] = rng.integers(0, rank + 1, adapters).astype(np.int32)
    c["ranks"][0] = rank
    c["scales"] = rng.uniform(0.5, 2, adapters).astype(np.float32)
    c["a"] = [(rng.standard_normal((adapters, rank, k)) / np.sqrt(k)).astype(dt) for _ in outs]
    c["b"] = [(rng.standard_normal((adapters, n, rank)) / np.sqrt(rank)).astype(dt) for n in outs]
    if garbage:  # what stands past an adapter's rank is not used
        for s, r in enumerate(c["ranks"]):
            for a, b in zip(c["a"], c["b"]):
                a[s, r:] = np.nan
                b[s, :, r:] = np.inf
    c["base"] = [rng.standard_normal((rows, n)).astype(np.float32) for n in outs]
    return c


def _want(c, i, base=True):
    """y, and the bound: sums of k and of the rank's products in fp32, in any order (each term through at most
    as many additions as there are terms), the scale's rounding and the addition of base."""
    rows, k = c["x"].shape
    n = c["b"][i].shape[1]
    y = c["base"][i].astype(np.float64) if base else np.zeros((rows, n))
    tol = np.abs(y) * 2.0 ** -24
    for s in range(len(c["ranks"])):
        at = np.nonzero(c["ids"] == s)[0]
        r = c["ranks"][s]
        if not at.size or r == 0:
            continue
        a, b, x = c["a"][i][s, :r].astype(np.float64), c["b"][i][s, :, :r].astype(np.float64), c["x"][at].astype(np.float64)
        sc = float(c["scales"][s])
        y[at] += sc * (x @ a.T) @ b.T
        mag = sc * (np.abs(x) @ np.abs(a).T) @ np.abs(b).T
        tol[at] += mag * (k + r + 4) * 2.0 ** -24
    return y, tol + np.abs(y) * 2.0 ** -24


def _run(gpu, c, **kw):
    g = gpu.group_rows_dev(_cu(c["ids"]), len(c["ranks"]))
    args = dict(ranks=_cu(c["ranks"]), scales=_cu(c["scales"]), base=[_cu(b) for b in c["base"]])
    args.update(kw)
    return gpu.lora_dev(_cu(c["x"]), [_cu(a) for a in c["a"]], [_cu(b) for b in c["b"]], g, **args)


SHAPES = [(1, 1, 4, 4, [1]), (1, 4, 16, 512, [256, 64, 64]), (3, 2, 8, 100, [37, 40]), (17, 40, 12, 260, [129]),
          (64, 32, 64, 1024, [300, 300]), (65, 3, 36, 896, [896, 128, 128, 5]), (200, 2, 256, 68, [72]),
          (500, 5, 32, 2052, [516])]


@pytest.mark.parametrize("rows,adapters,rank,k,outs", SHAPES)
@pytest.mark.parametrize("dt", [np.float16, np.float32])
def test_lora(gpu, rows, adapters, rank, k, outs, dt):
    c = _case(rows, adapters, rank, k, outs, dt, rows + rank)
    print("lora", rows, adapters, rank, k, outs, dt.__name__, flush=True)
    for i, y in enumerate(_run(gpu, c)):
        want, tol = _want(c, i)
        err = np.abs(y.cpu().numpy() - want)
        assert (err <= tol).all(), float((err - tol).max())
        d = want - c["base"][i]
        if np.abs(d).max() > 0:  # roundings of either sign: far inside the bound together
            assert np.linalg.norm(err) <= 2.0 ** -20 * np.linalg.norm(want)
        out = (c["ids"] < 0) | (c["ids"] >= adapters)
        assert np.array_equal(y.cpu().numpy()[out], c["base"][i][out])  # rows of no adapter: the projection's


def test_without_base_in_place_and_defaults(gpu):
    import torch
    c = _case(70, 6, 16, 256, [100, 64], np.float16, 3, garbage=False)
    for i, y in enumerate(_run(gpu, c, base=None)):
        want, tol = _want(c, i, base=False)
        assert (np.abs(y.cpu().numpy() - want) <= tol).all()
    apart = _run(gpu, c)
    base = [_cu(b) for b in c["base"]]
    same = _run(gpu, c, base=base, ys=base)
    assert all(torch.equal(s, a) and s is b for s, a, b in zip(same, apart, base))
    mixed = _run(gpu, c, base=[None, _cu(c["base"][1])])
    assert torch.equal(mixed[1], apart[1])
    c["ranks"][:] = 16
    c["scales"][:] = 1
    full = _run(gpu, c, ranks=None, scales=None)
    for i, y in enumerate(full):
        want, tol = _want(c, i)
        assert (np.abs(y.cpu().numpy() - want) <= tol).all()


def test_a_row_alone_equals_itself_in_a_batch(gpu):
    """A row's adapter result does not hang on the rows beside it (as long as K is split alike)."""
    c = _case(48, 3, 16, 384, [200], np.float16, 5, none=0.0)
    whole = _run(gpu, c)[0].cpu().numpy()
    for r in (0, 20, 47):
        one = {**c, "x": c["x"][r:r + 1], "ids": c["ids"][r:r + 1], "base": [b[r:r + 1] for b in c["base"]]}
        assert np.array_equal(_run(gpu, one)[0].cpu().numpy()[0], whole[r])


def test_infinities_stay_in_their_rows(gpu):
    c = _case(40, 2, 8, 128, [96], np.float32, 6, none=0.1, garbage=False)
    clean = _run(gpu, c)[0].cpu().numpy()
    c["ids"][4] = 1
    c["ranks"][:] = 8
    clean = _run(gpu, c)[0].cpu().numpy()
    c["x"][4, 7] = np.inf
    got = _run(gpu, c)[0].cpu().numpy()
    assert not np.isfinite(got[4]).any()
    assert np.array_equal(np.delete(got, 4, 0), np.delete(clean, 4, 0))


def test_beside_a_shared_projection_in_a_graph(gpu):
    """matmul_quant of a batch, then its adapters in place, captured and replayed with eager work between."""
    import torch
    from cllm_inference_amd import synth as S
    rows, k, n, adapters = 24, 512, 768, 5
    c = _case(rows, adapters, 16, k, [n], np.float16, 9)
    w = _cu(S.make_weight(S.Q4_K, n, k, 1).reshape(-1))
    x, ids = _cu(c["x"]), _cu(c["ids"])
    a, b, ranks, scales = [_cu(c["a"][0])], [_cu(c["b"][0])], _cu(c["ranks"]), _cu(c["scales"])

    def step():
        y = gpu.matmul_quant_dev(x, w, S.Q4_K, None, k, n)
        g = gpu.group_rows_dev(ids, adapters)
        p = y.clone()
        return p, gpu.lora_dev(x, a, b, g, ranks=ranks, scales=scales, base=[y], ys=[y])[0]

    step()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = step()
    torch.cuda.current_stream().wait_stream(s)
    rng = np.random.default_rng(1)
    for _ in range(4):
        c["x"] = rng.standard_normal((rows, k)).astype(np.float32)
        c["ids"] = rng.integers(-1, adapters, rows).astype(np.int32)
        x.copy_(_cu(c["x"]))
        ids.copy_(_cu(c["ids"]))
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        torch.cuda.synchronize()
        assert torch.equal(out[1], eager[1])
        c["base"] = [out[0].cpu().numpy()]
        want, tol = _want(c, 0)
        assert (np.abs(out[1].cpu().numpy() - want) <= tol).all()


def test_refusals(gpu):
    import torch
    c = _case(5, 3, 8, 64, [32], np.float16, 2, garbage=False)
    x, a, b = _cu(c["x"]), _cu(c["a"][0]), _cu(c["b"][0])
    g = gpu.group_rows_dev(_cu(c["ids"]), 3)
    bad = [lambda: gpu.lora_dev(x, [a], [b.float()], g), lambda: gpu.lora_dev(x, [a], [], g),
           lambda: gpu.lora_dev(x[:, :60], [a], [b], g), lambda: gpu.lora_dev(x[:4], [a], [b], g),
           lambda: gpu.lora_dev(x, [a.bfloat16()], [b.bfloat16()], g), lambda: gpu.lora_dev(x, [a] * 5, [b] * 5, g),
           lambda: gpu.lora_dev(x, [a], [b], gpu.RowGroups(g.offsets[:3], g.order)),
           lambda: gpu.lora_dev(x, [a], [b], g, ranks=_cu(c["ranks"]).long()),
           lambda: gpu.lora_dev(x, [a], [b], g, base=[x]), lambda: gpu.lora_dev(x.cpu(), [a], [b], g),
           lambda: gpu.lora_dev(x, [a[:, :6].contiguous()], [b[..., :6].contiguous()], g)]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
    torch.cuda.synchronize()
