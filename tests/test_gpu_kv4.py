"""The paged KV cache in 4 bits on an MI355X: rows stored and read back (exactly the model's values),
page calls (exactly the model's tables, lengths, counts and pages), attention against 64 bits
(tolerances in kv4_model.attention_bound), and all of them together, eager and captured."""
import ctypes

import numpy as np
import pytest

import kv4_model as M

pytestmark = pytest.mark.gpu


def _i32(x):
    import torch
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def _dev(x):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).cuda()


class Pair:
    """A cache of the library and its model, kept alike. Unwritten pages hold NaN scales."""

    def __init__(self, gpu, n_layers, n_pages, max_seqs, max_pages, page, n_kv, hd):
        self.gpu = gpu
        self.c = gpu.Kv4Cache(n_layers, n_pages, max_seqs, max_pages, page_size=page, n_head_kv=n_kv, head_dim=hd)
        self.c.pages.fill_(0xFF)
        self.m = M.Cache(n_layers, n_pages, max_seqs, max_pages, page, n_kv, hd)
        self.m.kv[:] = np.nan  # what they read back as
        self.n_kv, self.hd, self.layers = n_kv, hd, n_layers

    def extend(self, slots, counts):
        got = self.gpu.kv4_extend_dev(self.c, _i32(slots), _i32(counts))
        want = self.m.extend(slots, counts)
        assert int(got) == want, (slots, counts, int(got), want)
        self.same()
        return want

    def fork(self, src, dst):
        self.gpu.kv4_fork_dev(self.c, _i32(src), _i32(dst))
        self.m.fork(src, dst)
        self.same()

    def truncate(self, slots, new=None):
        self.gpu.kv4_truncate_dev(self.c, _i32(slots), None if new is None else _i32(new))
        self.m.truncate(slots, new)
        self.same()

    def compact(self):
        got = int(self.gpu.kv4_compact_dev(self.c))
        assert got == self.m.compact()
        self.same()

    def same(self):
        for name in ("table", "lens", "refs"):
            assert np.array_equal(getattr(self.c, name).cpu().numpy(), getattr(self.m, name)), name

    def store(self, rng, layer, slots, rows, scale=1.0):
        starts = np.concatenate([[0], np.cumsum(rows)])
        k = (rng.standard_normal((starts[-1], self.n_kv, self.hd)) * scale).astype(np.float32)
        v = (rng.standard_normal(k.shape) * scale).astype(np.float32)
        self.gpu.kv4_store_dev(self.c, layer, _dev(k), _dev(v), _i32(starts), slots=_i32(slots))
        for s, a, b in zip(slots, starts, starts[1:]):
            self.m.store(layer, s, k[a:b], v[a:b])

    def check_rows(self, layer, slots):
        """Every position of the slots reads back as the model's."""
        lens = [int(self.m.lens[s]) for s in slots]
        starts = np.concatenate([[0], np.cumsum(lens)])
        k, v = self.gpu.kv4_load_dev(self.c, layer, _i32(starts), int(starts[-1]), slots=_i32(slots))
        k, v = (x.cpu().numpy().reshape(-1, self.n_kv, self.hd) for x in (k, v))
        for s, a, b in zip(slots, starts, starts[1:]):
            mk, mv, _ = self.m.rows(layer, s, b - a)
            assert np.array_equal(k[a:b], mk, equal_nan=True), s
            assert np.array_equal(v[a:b], mv, equal_nan=True), s

    def attend(self, rng, layer, slots, rows, n_head, scale=1.0, max_rows=None, max_len=None, rms=False):
        starts = np.concatenate([[0], np.cumsum(rows)])
        q = (rng.standard_normal((starts[-1], n_head, self.hd)) * scale).astype(np.float32)
        max_len = max(1, int(self.m.lens[slots].max())) if max_len is None else max_len
        plan = self.gpu.kv4_attention_plan(self.c, len(slots), int(starts[-1]), max(rows), max_len, n_head)
        print("attention", self.hd, n_head, self.n_kv, "slots", slots, "rows", rows,
              "lens", [int(self.m.lens[s]) for s in slots], plan, flush=True)
        out = self.gpu.kv4_attention_dev(self.c, layer, _dev(q), _i32(starts), slots=_i32(slots), n_head=n_head,
                                         max_rows=max_rows or max(rows), max_len=max_len)
        out = out.cpu().numpy().reshape(q.shape)
        for s, a, b in zip(slots, starts, starts[1:]):
            n = int(self.m.lens[s])
            k, v, ok = self.m.rows(layer, s, n)
            want, *sizes = M.attention(q[a:b], k, v, ok, n - (b - a))
            bound = M.attention_bound(self.hd, n, *sizes)
            err = np.abs(out[a:b] - want)
            assert (err <= bound).all(), (s, float((err - bound).max()), float(err.max()))
            if rms:
                e = float(np.sqrt((err ** 2).mean() / (want ** 2).mean()))
                print("rms", e, flush=True)
                assert e <= M.attention_rms_bound()
        return out


# ---- store and load ---------------------------------------------------------------------------

@pytest.mark.parametrize("hd,n_kv,page", [(64, 2, 32), (64, 1, 256), (128, 8, 64), (128, 1, 32), (256, 2, 128)])
def test_store_and_load(gpu, hd, n_kv, page):
    """Rows appended over several calls (one token, odd counts, whole tiles, across tiles and pages)
    read back as the quantization's definition in 64 bits; rows stored before keep their values."""
    rng = np.random.default_rng(hd + n_kv)
    p = Pair(gpu, 2, 40, 4, 2 + 400 // page, page, n_kv, hd)
    for step in ([1, 5, 33], [1, 1, 1], [40, 27, 0], [64, 3, 1], [30, 0, 70]):
        slots = [2, 0, 3]
        assert p.extend(slots, step) == 0
        p.store(rng, 1, slots, step, scale=float(10.0 ** rng.integers(-3, 3)))
        p.check_rows(1, slots)


def test_the_bytes_of_a_page(gpu):
    """The tiles of the pages lie as kv4_model.places says."""
    for hd in (64, 128, 256):
        rng = np.random.default_rng(hd)
        p = Pair(gpu, 1, 3, 1, 3, 64, 2, hd)
        assert p.extend([0], [77]) == 0
        p.store(rng, 0, [0], [77])
        pages = p.c.pages.cpu().numpy().reshape(3, 2, 2, 36 * hd)
        k, v, _ = p.m.rows(0, 0, 77)
        for value, want in ((False, k), (True, v)):
            b, s, sc = M.places(hd, value)
            for pos in (0, 1, 17, 31, 32, 50, 63, 64, 76):
                page, tile, i = int(p.m.table[0, pos // 64]), pos % 64 // 32, pos % 32
                for h in range(2):
                    t = pages[page, h, tile]
                    c = (t[b[i]] >> s[i]).astype(np.int64) & 15
                    d = (t[sc[i]].astype(np.uint16) | (t[sc[i] + 1].astype(np.uint16) << 8)).view(np.float16)
                    assert np.array_equal((c - 8) * d.astype(np.float64), want[pos, h]), (hd, value, pos, h)


def test_store_of_odd_values(gpu):
    """Zeros, subnormals, ties, one-sided blocks, values past fp16, and rows that are not finite."""
    import torch
    rng = np.random.default_rng(3)
    hd, r = 128, 96
    k = rng.standard_normal((r, 1, hd)).astype(np.float32)
    v = rng.standard_normal((r, 1, hd)).astype(np.float32)
    k[0] = 0
    v[0] = -0.0
    k[1] *= 1e-7
    k[2] *= 1e-38
    v[3] *= 3e38 / 8
    k[4] = 65504 * np.sign(k[4])
    k[5] = np.abs(k[5])
    v[5] = -np.abs(v[5])
    for i in range(6, 40):  # multiples of half a step of a scale of few bits: ties
        k[i] = rng.integers(-16, 17, (1, hd)) * np.float32(0.5 * 2.0 ** (i - 20))
    k[40:50, 0, ::32] = 8.03  # scales whose rounding moves the quotients
    k[60, 0, 5] = np.nan
    v[61, 0, 100] = np.inf
    k[62, 0, 127] = -np.inf
    c = gpu.Kv4Cache(1, 2, 1, 2, page_size=64, n_head_kv=1, head_dim=hd)
    assert int(gpu.kv4_extend_dev(c, None, _i32([r]))) == 0
    gpu.kv4_store_dev(c, 0, _dev(k), _dev(v), _i32([0, r]))
    gk, gv = gpu.kv4_load_dev(c, 0, _i32([0, r]), r)
    mk, mv = M.stored(k, v)
    assert np.array_equal(gk.cpu().numpy().reshape(mk.shape), mk, equal_nan=True)
    assert np.array_equal(gv.cpu().numpy().reshape(mv.shape), mv, equal_nan=True)
    # a row that is not finite reaches the queries that see it, and no others
    q = rng.standard_normal((r, 2, hd)).astype(np.float32)
    k[1:5] = v[1:5] = 1  # (values of ordinary size)
    gpu.kv4_store_dev(c, 0, _dev(k), _dev(v), _i32([0, r]))
    for rows in (r, 1):
        out = gpu.kv4_attention_dev(c, 0, _dev(q[-rows:]), _i32([0, rows]), n_head=2, max_rows=rows, max_len=r)
        nan = torch.isnan(out).all(1).cpu().numpy()
        assert not torch.isnan(out[~torch.from_numpy(nan)]).any()
        assert np.array_equal(nan, np.arange(r - rows, r) >= 60)


def test_store_leaves_the_rest(gpu):
    """Rows of no sequence, sequences without rows or slots, and positions without a page: nothing is
    written, and load gives 0 or leaves its output."""
    import torch
    rng = np.random.default_rng(5)
    p = Pair(gpu, 1, 6, 3, 4, 32, 2, 64)
    p.extend([0, 1], [70, 10])
    p.store(rng, 0, [0, 1], [70, 10])
    before = p.c.pages.clone()
    k = torch.randn(20, 128, device="cuda")
    # a slot out of range, an empty sequence, rows before the first position of slot 2 (length 0)
    gpu.kv4_store_dev(p.c, 0, k, k, _i32([0, 5, 5, 9]), slots=_i32([7, 0, 2]))
    gpu.kv4_store_dev(p.c, 0, k, k, _i32([0, 5]), slots=_i32([-1]))
    gpu.kv4_store_dev(p.c, 0, k, k, _i32([3, 3, 30, 25]), slots=_i32([0, 2, 2]))  # malformed starts
    assert torch.equal(p.c.pages, before)
    # a page taken out of the table: its rows are dropped, the others stored
    p.c.table[0, 1] = -1
    p.m.table[0, 1] = -1
    p.store(rng, 0, [0], [70])
    p.check_rows(0, [0, 1])
    p.c.table[0, 1] = 99
    p.m.table[0, 1] = 99
    p.store(rng, 0, [0], [50])
    p.check_rows(0, [0, 1])
    # load: zeros before the first position, rows of no sequence left
    ko, vo = torch.full((20, 128), 7.0, device="cuda"), torch.full((20, 128), 7.0, device="cuda")
    gpu.kv4_load_dev(p.c, 0, _i32([2, 15]), 20, slots=_i32([1]), k=ko, v=vo)
    mk, mv, _ = p.m.rows(0, 1, 10)
    for got, want in ((ko, mk), (vo, mv)):
        got = got.cpu().numpy()
        assert (got[:2] == 7).all() and (got[15:] == 7).all() and (got[2:5] == 0).all()
        assert np.array_equal(got[5:15].reshape(want.shape), want)


def test_store_turns_keys_and_queries(gpu):
    """theta_base: the bits of rope_neox2_dev at each sequence's positions, then the store."""
    import torch
    for hd in (64, 128, 256):
        n_kv, n_head = 2, 6
        mk = lambda: gpu.Kv4Cache(1, 24, 3, 8, page_size=32, n_head_kv=n_kv, head_dim=hd)  # noqa: E731
        a, b = mk(), mk()
        lens, rows = [200, 40, 97], [37, 1, 64]
        for c in (a, b):
            assert int(gpu.kv4_extend_dev(c, None, _i32(lens))) == 0
        starts = np.concatenate([[0], np.cumsum(rows)])
        gen = torch.Generator(device="cuda").manual_seed(hd)
        k, v = (torch.randn(102, n_kv * hd, device="cuda", generator=gen) for _ in range(2))
        q = torch.randn(102, n_head * hd, device="cuda", generator=gen)
        k2, q2 = k.clone(), q.clone()
        gpu.kv4_store_dev(a, 0, k, v, _i32(starts), q=q, n_head=n_head, theta_base=500000.0)
        assert torch.equal(k, k2)  # the key rows stay
        for n, r, s in zip(lens, rows, starts):
            gpu.rope_neox2_dev(q2[s:s + r], n_head, k2[s:s + r], n_kv, hd, n - r, 500000.0)
        gpu.kv4_store_dev(b, 0, k2, v, _i32(starts))
        assert torch.equal(q, q2)
        for x, y in zip(gpu.kv4_load_dev(a, 0, _i32(starts), 102), gpu.kv4_load_dev(b, 0, _i32(starts), 102)):
            assert torch.equal(x, y)


# ---- attention ----------------------------------------------------------------------------------

@pytest.mark.parametrize("hd,n_kv,group,page,lens,rows", [
    (128, 2, 4, 64, [129], [1]),
    (128, 1, 1, 32, [1], [1]),
    (128, 1, 8, 64, [31, 32, 33, 64, 65], [1, 1, 1, 1, 1]),
    (64, 2, 7, 32, [1, 700, 64, 255], [1, 1, 1, 1]),
    (256, 1, 4, 128, [300, 17], [5, 5]),
    (128, 2, 16, 64, [200], [3]),
    (64, 1, 17, 64, [90], [2]),   # more query heads than a column tile
    (128, 2, 3, 64, [150, 40], [7, 40]),
    (256, 2, 2, 32, [129], [129]),
    (64, 1, 4, 64, [400, 33], [130, 33]),
    (128, 1, 5, 64, [500], [77]),
])
def test_attention(gpu, hd, n_kv, group, page, lens, rows):
    """Decode, drafts and prompts; ragged lengths; tiles and pages that end inside."""
    rng = np.random.default_rng(sum(lens) + hd)
    p = Pair(gpu, 2, sum(-(-n // page) for n in lens) + 3, len(lens), 2 + max(lens) // page, page, n_kv, hd)
    slots = list(rng.permutation(len(lens)))
    assert p.extend(slots, lens) == 0
    p.store(rng, 1, slots, lens)
    p.attend(rng, 1, slots, rows, n_kv * group, scale=1.5, rms=True)


@pytest.mark.parametrize("hd,n,rows,max_len", [(128, 5000, 1, None), (64, 3000, 4, None), (128, 1111, 1, 8192),
                                               (128, 2500, 1, 64), (128, 2000, 70, None)])
def test_attention_over_splits(gpu, hd, n, rows, max_len):
    """Sequences long enough to be split, with a max_len above and (results unchanged) below them."""
    rng = np.random.default_rng(n)
    p = Pair(gpu, 1, 100, 2, 80 if max_len != 8192 else 128, 64, 2, hd)
    assert p.extend([0, 1], [n, 30]) == 0
    p.store(rng, 0, [0, 1], [n, 30])
    p.attend(rng, 0, [0, 1], [rows, 1], 8, scale=1.0, max_len=max_len, rms=True)
    p.attend(rng, 0, [0, 1], [rows, 1], 8, scale=2.0, max_len=max_len)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("form,n_kv,group,seqs,rows,hint", [
    ("k_kv4_attention splits=0", 8, 2, 20, 1, 8192),       # shares of equal work across units
    ("k_kv4_attention splits=0", 4, 4, 9, 16, 8192),       # the same, four column tiles
    ("k_kv4_attention splits=1", 8, 4, 70, 1, 200),        # a workgroup per unit
    ("k_kv4_attention splits=2", 1, 8, 1, 100, 400),       # many column tiles of one sequence
    ("k_kv4_many_rows", 2, 4, 3, 60, 8192),                # split
    ("k_kv4_many_rows splits=1", 8, 4, 5, 44, 256),        # not split
])
def test_attention_in_every_form(gpu, hd, form, n_kv, group, seqs, rows, hint):
    """Each kernel and split of the work, over ragged lengths with an empty sequence and rows that see
    nothing (max_len is a hint: results do not depend on it)."""
    rng = np.random.default_rng([hd, n_kv, group, seqs, rows])
    p = Pair(gpu, 1, 5 * seqs + 8, seqs, 8192 // 64, 64, n_kv, hd)
    slots = [int(x) for x in rng.permutation(seqs)]
    lens = [int(x) for x in rng.integers(1, 1 + min(hint, 260), seqs)]
    lens[0] = max(lens[0], rows)
    if seqs > 1:
        lens[1] = 0
    assert p.extend(slots, lens) == 0
    p.store(rng, 0, slots, lens)
    r = [rows] + [int(x) for x in rng.integers(1, rows + 1, seqs - 1)]  # (more rows than positions, some)
    plan = p.gpu.kv4_attention_plan(p.c, seqs, sum(r), rows, hint, n_kv * group)
    assert all(word in plan.replace("<", " <") for word in form.split()), plan
    p.attend(rng, 0, slots, r, n_kv * group, max_len=hint, rms=False)


def test_attention_of_sharp_and_large_scores(gpu):
    """Queries whose scores spread over hundreds (one position has all the weight), tiny queries
    (nearly equal weights), and rows that differ by 2^60 in size beside one another."""
    rng = np.random.default_rng(11)
    p = Pair(gpu, 1, 20, 1, 16, 64, 1, 128)
    assert p.extend([0], [600]) == 0
    p.store(rng, 0, [0], [600])
    for scale in (100.0, 1e-6, 1e-30):
        p.attend(rng, 0, [0], [9], 4, scale=scale)
    q = rng.standard_normal((2, 1, 128)).astype(np.float32)
    q[1] *= 2.0 ** -60
    out = gpu.kv4_attention_dev(p.c, 0, _dev(q), _i32([0, 2]), n_head=1, max_rows=2, max_len=600)
    k, v, ok = p.m.rows(0, 0, 600)
    want, *sizes = M.attention(q, k, v, ok, 598)
    assert (np.abs(out.cpu().numpy().reshape(want.shape) - want) <= M.attention_bound(128, 600, *sizes)).all()


def test_attention_sees_nothing(gpu):
    """Rows before the first position, empty sequences, slots out of range and sequences without
    pages give 0; pages taken out of the middle are not seen; rows of no sequence stay."""
    import torch
    rng = np.random.default_rng(13)
    p = Pair(gpu, 1, 12, 4, 8, 32, 2, 64)
    assert p.extend([0, 1, 3], [10, 200, 40]) == 0
    p.store(rng, 0, [0, 1, 3], [10, 200, 40])
    p.attend(rng, 0, [0, 1], [16, 3], 4)  # slot 0: rows at -6 .. 9
    for hole in (0, 3, 6):
        p.c.table[1, hole] = p.m.table[1, hole] = -1
    p.c.table[3, 0] = p.m.table[3, 0] = 12  # past the pool
    p.attend(rng, 0, [1, 3], [70, 40], 4)
    p.attend(rng, 0, [1, 1], [1, 1], 4)  # one slot twice
    p.c.table[3] = -1
    p.m.table[3] = -1
    p.attend(rng, 0, [3, 2], [1, 2], 4)
    q = torch.randn(30, 256, device="cuda")
    out = torch.full_like(q, 5.0)
    gpu.kv4_attention_dev(p.c, 0, q, _i32([2, 6, 6, 9]), slots=_i32([0, 1, 99]), n_head=4, max_rows=4,
                          max_len=200, out=out)
    o = out.cpu().numpy()
    assert (o[:2] == 5).all() and (o[6:] == 5).all() and (o[2:6] != 5).all() and np.isfinite(o).all()
    # malformed starts stay within the rows
    out.fill_(5.0)
    gpu.kv4_attention_dev(p.c, 0, q, _i32([-3, 4, 2, 99]), slots=_i32([0, 0, 0]), n_head=4, max_rows=30,
                          max_len=200, out=out)
    assert torch.isfinite(out).all()


def test_attention_on_another_stream_and_layout(gpu):
    """Non-default streams, and offsets of a batch inside larger buffers."""
    import torch
    rng = np.random.default_rng(17)
    p = Pair(gpu, 3, 40, 2, 32, 64, 2, 128)
    assert p.extend([0, 1], [1500, 3]) == 0
    p.store(rng, 2, [0, 1], [1500, 3])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a = p.attend(np.random.default_rng(1), 2, [0, 1], [2, 1], 8)
    b = p.attend(np.random.default_rng(1), 2, [0, 1], [2, 1], 8)
    assert np.array_equal(a, b)


# ---- page calls ---------------------------------------------------------------------------------

def test_page_calls_at_random(gpu):
    """Two hundred calls at random on one cache: tables, lengths, counts, statuses and what the
    sequences hold are the model's after each, refusals and shared partly filled pages among them."""
    rng = np.random.default_rng(23)
    p = Pair(gpu, 2, 30, 8, 6, 32, 1, 64)
    refused = copied = 0
    for step in range(200):
        op = rng.integers(0, 10)
        n = int(rng.integers(1, 8))
        slots = rng.permutation(8)[:n].tolist()
        if op < 4:
            counts = rng.choice([0, 1, 1, 2, 31, 33, 64, 100], n).tolist()
            if rng.random() < 0.1:
                slots[0] = int(rng.choice([-1, 8, slots[-1]]))
            if rng.random() < 0.05:
                counts[0] = -1
            before = p.m.refs.copy()
            if p.extend(slots, counts) == 0:
                copied += int((p.m.refs < before).any())
                p.store(rng, step % 2, slots, counts)
            else:
                refused += 1
        elif op < 7:
            src = rng.integers(0, 8, n).tolist()
            if rng.random() < 0.1:
                src[0] = 9
            p.fork(src, rng.integers(0, 8, n).tolist() if rng.random() < 0.2 else slots)
        elif op < 9:
            p.truncate(slots, None if rng.random() < 0.2 else rng.integers(-1, 150, n).tolist())
        else:
            p.compact()
        p.check_rows(step % 2, list(range(8)))
        used = np.bincount(p.m.table[p.m.table >= 0], minlength=30)
        assert np.array_equal(used, p.m.refs)
    assert refused > 3 and copied > 3


def test_extend_is_all_or_nothing(gpu):
    p = Pair(gpu, 1, 5, 4, 4, 32, 1, 64)
    assert p.extend([0, 1], [100, 20]) == 0   # 4 + 1 pages
    assert p.extend([2], [1]) == 1
    assert p.extend([1, 2, 3], [10, 40, 64]) == 4
    assert p.extend([1, 0], [12, 200]) == -1  # more than max_pages
    assert p.extend([1, 1], [1, 1]) == -1
    assert p.extend([1], [12]) == 0
    assert p.extend([0, 1, 2, 3], [0, 0, 0, 0]) == 0
    p.truncate([0, 0, 9, 1], [33, 0, 0, 0])   # the first entry of a slot stands
    assert int(p.m.lens[0]) == 33
    assert p.extend([3], [96]) == 0
    # the largest call: every slot of a large cache, many pages
    big = Pair(gpu, 1, 9000, 1024, 8, 32, 1, 64)
    rng = np.random.default_rng(2)
    assert big.extend(list(range(1024)), rng.integers(0, 250, 1024).tolist()) == 0
    big.fork(rng.integers(0, 1024, 1024).tolist(), list(range(1024)))
    assert big.extend(list(rng.permutation(1024)), [1] * 1024) == 0
    big.truncate(list(range(0, 1024, 3)))
    big.compact()
    assert big.extend(list(range(1024)), [1] * 1024) == 0


def test_copy_pages(gpu):
    import torch
    c = gpu.Kv4Cache(3, 9, 1, 1, page_size=64, n_head_kv=3, head_dim=128)
    c.pages.copy_(torch.randint(0, 256, c.pages.shape, dtype=torch.uint8, device="cuda"))
    want = c.pages.clone()
    src, dst = [0, 4, 4, 8, -1, 3, 2, 9], [1, 5, 6, 8, 7, 9, -5, 7]
    gpu.kv4_copy_pages_dev(c, _i32(src), _i32(dst))
    for s, d in zip(src, dst):
        if 0 <= s < 9 and 0 <= d < 9:
            want[:, d] = want[:, s]
    assert torch.equal(c.pages, want)


# ---- together -------------------------------------------------------------------------------------

def test_a_beam_search_step_after_step(gpu):
    """A prompt, forked into beams; then, eager and as a replayed graph: fork by parents, extend,
    store with rotation, attention. The graph gives the eager steps' bits, replay after replay."""
    import torch
    hd, n_kv, n_head, beams, page = 128, 2, 8, 4, 32
    rng = np.random.default_rng(31)
    caches = [Pair(gpu, 1, 40, beams, 8, page, n_kv, hd) for _ in range(2)]
    prompt = rng.standard_normal((2, 45, n_kv, hd)).astype(np.float32)
    steps = 9
    par = rng.integers(0, beams, (steps, beams))
    kv = rng.standard_normal((steps, 3, beams, max(n_kv, n_head) * hd)).astype(np.float32)
    bufs = []
    for p in caches:
        assert p.extend([0], [45]) == 0
        gpu.kv4_store_dev(p.c, 0, _dev(prompt[0]), _dev(prompt[1]), _i32([0, 45]), slots=_i32([0]))
        p.fork([0] * 3, [1, 2, 3])
        bufs.append(dict(par=_i32(par[0]), one=_i32([1] * beams), beams=_i32(range(beams)),
                         starts=_i32(range(beams + 1)),
                         k=torch.empty(beams, n_kv * hd, device="cuda"), v=torch.empty(beams, n_kv * hd, device="cuda"),
                         q=torch.empty(beams, n_head * hd, device="cuda"),
                         out=torch.empty(beams, n_head * hd, device="cuda"),
                         status=torch.empty(1, dtype=torch.int32, device="cuda")))

    def step(p, b):
        gpu.kv4_fork_dev(p.c, b["par"], b["beams"])
        gpu.kv4_extend_dev(p.c, b["beams"], b["one"], status=b["status"])
        gpu.kv4_store_dev(p.c, 0, b["k"], b["v"], b["starts"], q=b["q"], n_head=n_head, theta_base=1e4)
        gpu.kv4_attention_dev(p.c, 0, b["q"], b["starts"], n_head=n_head, max_rows=1, max_len=8 * page, out=b["out"])

    def fill(b, i):
        b["par"].copy_(_i32(par[i]))
        b["k"].copy_(_dev(kv[i, 0, :, :n_kv * hd]))
        b["v"].copy_(_dev(kv[i, 1, :, :n_kv * hd]))
        b["q"].copy_(_dev(kv[i, 2, :, :n_head * hd]))

    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    fill(bufs[1], 0)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        step(caches[1], bufs[1])
    torch.cuda.synchronize()
    caches[1].same()  # nothing ran while it was recorded
    for i in range(steps):
        fill(bufs[0], i)
        fill(bufs[1], i)
        step(caches[0], bufs[0])
        graph.replay()
        torch.cuda.synchronize()
        assert int(bufs[0]["status"]) == int(bufs[1]["status"]) == 0
        assert torch.equal(bufs[0]["out"], bufs[1]["out"]), i
        for name in ("table", "lens", "refs"):
            assert torch.equal(getattr(caches[0].c, name), getattr(caches[1].c, name)), (i, name)
        # and the model: the beams' pages hold what each beam stored
        m = caches[0].m
        m.fork(par[i].tolist(), list(range(beams)))
        assert m.extend(list(range(beams)), [1] * beams) == 0
        caches[0].same()
        junk = torch.randn(1 << 20, device="cuda").sum()  # the program's own work between replays
        assert torch.isfinite(junk)
    starts = _i32(np.arange(beams + 1) * int(m.lens[0]))
    a, b = (gpu.kv4_load_dev(p.c, 0, starts, beams * int(m.lens[0])) for p in caches)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # against the fp32 attention over the read-back rows
    for s in range(beams):
        n = int(m.lens[0])
        k, v = a[0][s * n:(s + 1) * n].contiguous(), a[1][s * n:(s + 1) * n].contiguous()
        q = bufs[0]["q"][s:s + 1].contiguous()
        ref = gpu.attention_dev(q, k, v, n - 1, n_head, n_kv, hd)
        kk, vv = (x.cpu().numpy().reshape(n, n_kv, hd).astype(np.float64) for x in (k, v))
        want, *sizes = M.attention(q.cpu().numpy().reshape(1, n_head, hd), kk, vv, np.ones(n, bool), n - 1)
        bound = M.attention_bound(hd, n, *sizes)
        for got in (ref, bufs[0]["out"][s:s + 1]):
            assert (np.abs(got.cpu().numpy().reshape(want.shape) - want) <= bound).all()


def test_bindings_refuse(gpu):
    import torch
    c = gpu.Kv4Cache(1, 4, 2, 2, page_size=32, n_head_kv=2, head_dim=64)
    k = torch.randn(3, 128, device="cuda")
    bad = [
        lambda: gpu.kv4_store_dev(c, 0, k.double(), k, _i32([0, 3])),
        lambda: gpu.kv4_store_dev(c, 0, k, k[:2], _i32([0, 3])),
        lambda: gpu.kv4_store_dev(c, 0, k.t(), k, _i32([0, 3])),
        lambda: gpu.kv4_store_dev(c, 0, k.cpu(), k, _i32([0, 3])),
        lambda: gpu.kv4_store_dev(c, 0, k, k, torch.tensor([0, 3], device="cuda")),
        lambda: gpu.kv4_store_dev(c, 0, k, k, _i32([0, 1, 2, 3])),  # three sequences, two slots
        lambda: gpu.kv4_store_dev(c, 1, k, k, _i32([0, 3])),
        lambda: gpu.kv4_extend_dev(c, _i32([0]), _i32([1, 1])),
        lambda: gpu.kv4_fork_dev(c, _i32([0]), _i32([1, 1])),
        lambda: gpu.kv4_fork_dev(c, _i32([0] * 3), _i32([1] * 3)),
        lambda: gpu.kv4_attention_dev(c, 0, k, _i32([0, 3]), n_head=3, max_rows=3, max_len=3),
        lambda: gpu.kv4_attention_dev(c, 0, k, _i32([0, 3]), n_head=2, max_rows=3, max_len=3, out=k[:2]),
        lambda: gpu.Kv4Cache(1, 4, 2, 2, page_size=48, n_head_kv=2, head_dim=64),
        lambda: gpu.Kv4Cache.from_tensors(c.pages, c.table, c.lens[:1], c.refs, page_size=32, n_head_kv=2, head_dim=64),
        lambda: gpu.Kv4Cache.from_tensors(c.pages, c.table, c.lens, c.refs, page_size=64, n_head_kv=2, head_dim=64),
        lambda: gpu.logprobs_dev(k.double()),
        lambda: gpu.logprobs_dev(k.t()),
        lambda: gpu.logprobs_dev(k, _i32([1, 2])),
        lambda: gpu.logprobs_dev(k, top_k=65),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            print("not refused:", i)


# ---- the largest, and several at once ---------------------------------------------------------------

def test_many_sequences(gpu):
    """More sequences than a wave has lanes, empty ones among them: shares that cross sequences, segments
    found past the first 64, and many rows of many sequences."""
    rng = np.random.default_rng(41)
    n, page = 150, 32
    lens = rng.integers(0, 90, n)
    lens[[3, 70, 149]] = [400, 0, 333]
    p = Pair(gpu, 1, int(sum(-(-x // page) for x in lens)) + 2, n, 16, page, 2, 64)
    slots = rng.permutation(n).tolist()
    assert p.extend(slots, lens.tolist()) == 0
    p.store(rng, 0, slots, lens.tolist())
    p.check_rows(0, list(range(n)))
    held = [int(p.m.lens[s]) for s in slots]
    p.attend(rng, 0, slots, [min(1, x) for x in held], 4)           # decode, units of one column tile
    p.attend(rng, 0, slots, [min(5, x) for x in held], 4)           # drafts
    p.attend(rng, 0, slots, held, 4)                                # every row of every sequence
    plan = gpu.kv4_attention_plan(p.c, n, n, 1, 400, 4)
    assert "splits=1" in plan, plan


def test_many_sequences_in_shares(gpu):
    """The same in shares of equal work (which contexts that may be long get), and rows past max_rows there
    and in the kernel for many rows."""
    import torch
    rng = np.random.default_rng(42)
    n, page = 150, 32
    lens = rng.integers(0, 90, n)
    lens[[3, 70, 149]] = [400, 0, 333]
    p = Pair(gpu, 1, int(sum(-(-x // page) for x in lens)) + 2, n, 256, page, 2, 64)
    slots = rng.permutation(n).tolist()
    assert p.extend(slots, lens.tolist()) == 0
    p.store(rng, 0, slots, lens.tolist())
    held = [int(p.m.lens[s]) for s in slots]
    assert "splits=0" in gpu.kv4_attention_plan(p.c, n, n, 1, 8192, 4)
    p.attend(rng, 0, slots, [min(1, x) for x in held], 4, max_len=8192)
    p.attend(rng, 0, slots, [min(5, x) for x in held], 4, max_len=8192)
    q = torch.randn(400, 256, device="cuda")
    full = gpu.kv4_attention_dev(p.c, 0, q, _i32([0, 400]), n_head=4, slots=_i32([slots[3]]), max_rows=400, max_len=8192)
    for max_rows in (3, 150):
        assert ("many" in gpu.kv4_attention_plan(p.c, 1, 400, max_rows, 8192, 4)) == (max_rows == 150)
        out = torch.full_like(q, 5.0)
        gpu.kv4_attention_dev(p.c, 0, q, _i32([0, 400]), n_head=4, slots=_i32([slots[3]]), max_rows=max_rows,
                              max_len=8192, out=out)
        assert (out[max_rows:] == 5).all()
        assert torch.allclose(out[:max_rows], full[:max_rows], rtol=1e-4, atol=1e-5)


def test_extending_a_thousand(gpu):
    """1024 entries at once: pages that many of them hold, slots named twice far apart, too few pages."""
    rng = np.random.default_rng(47)
    n, page = 1024, 32
    p = Pair(gpu, 1, 4 * n, n, 4, page, 1, 64)
    roots = [int(x) for x in rng.permutation(n)[:40]]
    assert p.extend(roots, [int(x) for x in rng.integers(1, 100, 40)]) == 0
    p.fork([roots[int(x)] for x in rng.integers(0, 30, n)], list(range(n)))  # ten of the roots live no more
    slots = [int(x) for x in rng.permutation(n)]
    for first, second in ((0, n - 1), (511, 512), (1022, 1023)):
        twice = list(slots)
        twice[second] = twice[first]
        assert p.extend(twice, [1] * n) == -1
    assert p.extend(slots, [int(x) for x in rng.integers(0, 2, n)]) == 0     # some stay on shared pages
    assert p.extend(slots[:700], [1] * 700) == 0
    assert p.extend(slots, [1] * n) == 0                                     # none shared within
    assert p.extend(slots, [4 * page] * n) == -1
    assert p.extend(slots, [28 if x <= 100 else 0 for x in p.m.lens[slots]]) in (0, 1)
    while p.extend(slots, [page if x <= 96 else 0 for x in p.m.lens[slots]]) == 0 and p.m.lens.min() <= 96:
        pass
    p.truncate(slots)
    assert int(p.c.refs.abs().sum()) == 0


def test_rows_past_max_rows_stay(gpu):
    import torch
    rng = np.random.default_rng(43)
    p = Pair(gpu, 1, 30, 1, 20, 32, 2, 64)
    assert p.extend([0], [300]) == 0
    p.store(rng, 0, [0], [300])
    q = torch.randn(200, 256, device="cuda")
    full = gpu.kv4_attention_dev(p.c, 0, q, _i32([0, 200]), n_head=4, max_rows=200, max_len=300)
    for max_rows in (3, 150):
        out = torch.full_like(q, 5.0)
        gpu.kv4_attention_dev(p.c, 0, q, _i32([0, 200]), n_head=4, max_rows=max_rows, max_len=300, out=out)
        assert (out[max_rows:] == 5).all()
        assert torch.allclose(out[:max_rows], full[:max_rows], rtol=1e-4, atol=1e-5)


def test_a_pool_past_4_gib(gpu):
    """Page and layer offsets past 32 bits, in every call that moves or reads pages."""
    import torch
    rng = np.random.default_rng(47)
    page, n_kv, hd, layers, n_pages = 1024, 8, 256, 2, 1200  # 2.36 MB a page: 5.7 GB
    c = gpu.Kv4Cache(layers, n_pages, 2, 4, page_size=page, n_head_kv=n_kv, head_dim=hd)
    assert c.pages.numel() > (1 << 32) + (1 << 30)
    assert int(gpu.kv4_extend_dev(c, None, _i32([70, 1030]))) == 0
    c.table[0, 0], c.table[1, 0], c.table[1, 1] = 1199, 1100, 1198
    c.refs.zero_()
    c.refs[[1199, 1100, 1198]] = 1
    k = rng.standard_normal((100, n_kv, hd)).astype(np.float32)
    v = rng.standard_normal((100, n_kv, hd)).astype(np.float32)
    starts = _i32([0, 70, 100])
    gpu.kv4_store_dev(c, 1, _dev(k), _dev(v), starts)
    mk, mv = M.stored(k, v)
    q = rng.standard_normal((70, 8, hd)).astype(np.float32)
    want, *sizes = M.attention(q, mk[:70], mv[:70], np.ones(70, bool), 0)

    def check():
        gk, gv = gpu.kv4_load_dev(c, 1, starts, 100)
        assert np.array_equal(gk.cpu().numpy().reshape(mk.shape), mk)
        assert np.array_equal(gv.cpu().numpy().reshape(mv.shape), mv)
        for rows in (70, 1):
            out = gpu.kv4_attention_dev(c, 1, _dev(q[70 - rows:]), _i32([0, rows]), n_head=8, max_rows=rows, max_len=70)
            err = np.abs(out.cpu().numpy().reshape(rows, 8, hd) - want[70 - rows:])
            assert (err <= M.attention_bound(hd, 70, *sizes)[70 - rows:]).all()

    check()
    gpu.kv4_copy_pages_dev(c, _i32([1199]), _i32([1197]))
    c.table[0, 0] = 1197
    check()
    c.refs[1197], c.refs[1199] = 1, 0
    assert int(gpu.kv4_compact_dev(c)) == 3
    assert sorted(c.table[c.table >= 0].tolist()) == [0, 1, 2]
    check()
    gpu.kv4_fork_dev(c, _i32([0]), _i32([1]))
    assert int(gpu.kv4_extend_dev(c, _i32([1]), _i32([1]))) == 0  # a copy on write
    torch.cuda.synchronize()


def test_two_streams_and_two_graphs(gpu):
    """Attention calls that run at once, eager and as graphs, have scratch of their own."""
    import torch
    rng = np.random.default_rng(53)
    p = Pair(gpu, 1, 200, 3, 80, 64, 2, 128)
    assert p.extend([0, 1, 2], [5000, 4000, 900]) == 0
    p.store(rng, 0, [0, 1, 2], [5000, 4000, 900])
    starts = _i32([0, 1, 2, 3])
    qs = [torch.randn(3, 1024, device="cuda") for _ in range(2)]
    run = lambda q, out=None: gpu.kv4_attention_dev(p.c, 0, q, starts, n_head=8, max_rows=1, max_len=5000, out=out)  # noqa: E731
    want = [run(q) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs, outs = [], []
    for q, s in zip(qs, streams):
        g, out = torch.cuda.CUDAGraph(), torch.empty_like(q)
        with torch.cuda.graph(g, stream=s):
            run(q, out)
        graphs.append(g)
        outs.append(out)
    for turn in range(5):
        got = [[], []]
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                for _ in range(4):
                    if turn % 2:
                        graphs[i].replay()
                    else:
                        got[i].append(run(qs[i]))
        torch.cuda.synchronize()
        for i in range(2):
            for o in got[i] or [outs[i]]:
                assert torch.equal(o, want[i]), (turn, i)
        torch.randn(1 << 18, device="cuda")


def test_host_tensors_are_refused(gpu):
    import torch
    z = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(RuntimeError, match="needs CUDA tensors"):
        gpu.Kv4Cache.from_tensors(torch.zeros((1, 2, gpu.kv4_page_bytes(32, 1, 64)), dtype=torch.uint8), z(1, 1), z(1),
                                  z(2), page_size=32, n_head_kv=1, head_dim=64)
    with pytest.raises(RuntimeError, match="needs CUDA tensors"):
        gpu.logprobs_dev(torch.zeros(2, 5))


@pytest.mark.parametrize("hd,group,rows,n", [(64, 4, 1, 300), (128, 4, 1, 3000), (128, 4, 5, 700), (256, 2, 8, 400),
                                             (128, 4, 130, 130), (64, 4, 150, 700)])
@pytest.mark.parametrize("scale", [1e4, 1e8, 1e10, 1e12, 1e30])
def test_attention_of_huge_scores(gpu, hd, group, rows, n, scale):
    """Queries so large that one position has all the weight, scores of either sign: each output is that
    position's value row, to the 2^-20 of a weight in two fp16 parts and three roundings."""
    rng = np.random.default_rng([hd, group, rows, n])
    p = Pair(gpu, 1, n // 64 + 2, 1, n // 64 + 2, 64, 1, hd)
    assert p.extend([0], [n]) == 0
    p.store(rng, 0, [0], [n])
    k, v, _ = p.m.rows(0, 0, n)
    # along a key the row sees (its score is the largest), or against one
    along = rng.integers(0, n - rows + 1, (rows, group))
    sign = np.where(rng.random((rows, group)) < 0.5, 1, -1)
    sign[0] = -1
    q = (k[along, 0] * (sign * scale)[..., None]).astype(np.float32)
    print("huge", hd, group, rows, n, scale, gpu.kv4_attention_plan(p.c, 1, rows, rows, n, group), flush=True)
    out = gpu.kv4_attention_dev(p.c, 0, _dev(q), _i32([0, rows]), n_head=group, max_rows=rows, max_len=n)
    out = out.cpu().numpy().reshape(q.shape).astype(np.float64)
    checked = 0
    for t in range(rows):
        x = q[t].astype(np.float64) @ k[:n - rows + t + 1, 0].T / np.sqrt(hd)
        size = (np.abs(q[t].astype(np.float64)) @ np.abs(k[:n - rows + t + 1, 0].T)).max() / np.sqrt(hd)
        for h in range(group):
            best, *rest = np.argsort(-x[h])[:2]
            # (scores are off by 2^-17 of their terms at most; closer ones may share the weight)
            if rest and x[h, best] - x[h, rest[0]] < max(200.0, 2.0 ** -15 * size):
                continue
            want = v[best, 0]
            assert (np.abs(out[t, h] - want) <= np.abs(want) * (2.0 ** -20 + 3 * 2.0 ** -24)).all(), (t, h)
            checked += 1
    assert checked >= rows * group // 2


@pytest.mark.parametrize("hd,group,rows", [(64, 4, 1), (128, 4, 1), (128, 4, 5), (256, 2, 8), (128, 4, 100)])
@pytest.mark.parametrize("k_scale,v_scale", [(1e-4, 1e-4), (1e-5, 1.0), (1.0, 1e-5), (1e-6, 1.0), (1.0, 1e-6), (1.0, 3e-7)])
def test_attention_over_small_values(gpu, hd, group, rows, k_scale, v_scale):
    """Caches whose elements are fp16 subnormals (below 2^-14), with queries that give scores of ordinary
    spread. The MFMA does not normalise such an operand: of its products it keeps the 24 bits below the
    smallest normal exponent, so with z leading zeros of an element's significand 2^(z - 24) of the
    product, once for the keys (a score of unit spread) or the values, beside the other roundings."""
    n = 500
    rng = np.random.default_rng([hd, group, rows])
    k = (rng.standard_normal((n, 1, hd)) * k_scale).astype(np.float32)
    v = (rng.standard_normal((n, 1, hd)) * v_scale).astype(np.float32)
    q = (rng.standard_normal((rows, group, hd)) / k_scale).astype(np.float32)
    c = gpu.Kv4Cache(1, 9, 1, 9, page_size=64, n_head_kv=1, head_dim=hd)
    assert int(gpu.kv4_extend_dev(c, None, _i32([n]))) == 0
    gpu.kv4_store_dev(c, 0, _dev(k), _dev(v), _i32([0, n]))
    out = gpu.kv4_attention_dev(c, 0, _dev(q), _i32([0, rows]), n_head=group, max_rows=rows, max_len=n)
    want, *sizes = M.attention(q, *M.stored(k, v), np.ones(n, bool), n - rows)
    err = np.abs(out.cpu().numpy().reshape(q.shape) - want)
    zeros = [max(0, -14 - int(np.floor(np.log2(s)))) for s in (k_scale, v_scale)]
    lost = sum(2.0 ** (z - 24) for z in zeros if z)
    rms = float(np.sqrt((err ** 2).mean() / (want ** 2).mean()))
    print("small", hd, group, rows, k_scale, v_scale, rms, flush=True)
    assert rms <= M.attention_rms_bound() + lost
    size, mass, total = sizes
    assert (err <= M.attention_bound(hd, n, size, mass, total) + 2 * lost * (size + 1) * mass).all()
