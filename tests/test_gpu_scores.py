"""adjust_scores / top_scores against a plain implementation: the same elementary float32 operations in numpy (bit for bit: every operation is
rounded once, in the documented order) and the formula in float64, with a tolerance counted in roundings."""
import numpy as np
import pytest
import torch

from rankfm_amd import ScoreRules, adjust_scores, pack_allowed, top_scores

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
NAN, INF = float("nan"), float("inf")


def dev(a, dtype=None):
    return None if a is None else torch.as_tensor(a, dtype=dtype).cuda()


class Problem:
    """host-side rules of a call and the two plain forms"""

    def __init__(self, rows, items, seed=0, history=None, row_bias=None, masks=None, item_bias=False, dtype=F32, per_row=True, empty_mask=True):
        rng = np.random.default_rng(seed)
        self.rows, self.items, self.dtype = rows, items, dtype
        self.s = torch.from_numpy((rng.standard_normal((rows, items)) * 2).astype(np.float32)).to(dtype)
        self.hist = self.bias = self.mask = self.which = self.item_bias = self.hist_rows = None
        self.rho, self.phi, self.pi = np.ones(rows, np.float32), np.zeros(rows, np.float32), np.zeros(rows, np.float32)
        if history is not None:
            people = rows + 2
            self.hist = [rng.integers(-2, items + 2, rng.integers(0, history + 1)) for _ in range(people)]     # out-of-catalogue entries among them
            self.hist[0] = np.zeros(0, np.int64)
            self.hist[-1] = np.full(history, items // 2)                                                        # one item many times
            self.hist_rows = rng.integers(-1, people, rows).astype(np.int32)
            self.hist_rows[-1] = people - 1
            if per_row:
                self.rho = (0.5 + 2 * rng.random(rows)).astype(np.float32)
                self.phi = rng.standard_normal(rows).astype(np.float32)
                self.pi = rng.standard_normal(rows).astype(np.float32)
            else:
                self.rho[:], self.phi[:], self.pi[:] = 1.3, 0.25, 0.5
        self.per_row = per_row
        if item_bias:
            self.item_bias = rng.standard_normal(items).astype(np.float32)
        if row_bias is not None:
            self.bias = []
            for r in range(rows):
                k = int(rng.integers(0, row_bias + 1))
                ids = rng.integers(-1, items + 1, k)
                if k > 2:
                    ids[-1] = ids[0]                                                                            # the same index twice: the last entry holds
                self.bias.append((ids, rng.standard_normal(k).astype(np.float32)))
        if masks is not None:
            self.mask = rng.random((masks, items)) < 0.6
            if empty_mask:
                self.mask[0] = False
            self.which = rng.integers(-1, masks, rows).astype(np.int32) if masks not in (1, rows) else None

    def rules(self):
        def csr(lists):
            off = np.zeros(len(lists) + 1, np.int64)
            np.cumsum([len(x) for x in lists], out=off[1:])
            return dev(off), dev(np.concatenate(lists + [np.zeros(0, np.int64)]).astype(np.int32))
        kw = {}
        if self.hist is not None:
            kw.update(history=csr(self.hist), history_rows=dev(self.hist_rows))
            for k, v in (("repetition", self.rho), ("frequency", self.phi), ("presence", self.pi)):
                kw[k] = dev(v) if self.per_row else float(v[0])
        if self.bias is not None:
            off, ids = csr([b[0] for b in self.bias])
            kw["row_bias"] = (off, ids, dev(np.concatenate([b[1] for b in self.bias] + [np.zeros(0, np.float32)])))
        if self.mask is not None:
            kw.update(allowed=pack_allowed(dev(self.mask)), allowed_rows=dev(self.which))
        return ScoreRules(item_bias=dev(self.item_bias), **kw)

    def plain(self, kind):
        """the formula in numpy type `kind`, and the magnitude its roundings are relative to"""
        out = self.s.float().numpy().astype(kind)
        size = np.abs(out)
        for r in range(self.rows):
            s = out[r]
            if self.hist is not None and self.hist_rows[r] >= 0:
                ids = self.hist[self.hist_rows[r]]
                c = np.bincount(ids[(ids >= 0) & (ids < self.items)], minlength=self.items).astype(kind)
                rho, phi, pi = kind(self.rho[r]), kind(self.phi[r]), kind(self.pi[r])
                with np.errstate(all="ignore"):
                    x = np.where(s > 0, s / rho, s * rho) - phi * c
                s = np.where(c > 0, x - pi, s)
                size[r] = np.where(c > 0, np.maximum(size[r] * rho, size[r] / rho) + np.abs(phi) * c + np.abs(pi), size[r])
            if self.item_bias is not None:
                s = s + self.item_bias.astype(kind)
                size[r] += np.abs(self.item_bias)
            if self.bias is not None:
                extra = {int(i): v for i, v in zip(*self.bias[r]) if 0 <= i < self.items}
                for i, v in extra.items():
                    s[i] = s[i] + kind(v)
                    size[r, i] += abs(v)
            if self.mask is not None:
                m = r if self.which is None and len(self.mask) == self.rows else 0 if self.which is None else self.which[r]
                if m >= 0:
                    s = np.where(self.mask[m], s, kind(-INF))
            out[r] = s
        return out, size


def same(a, b):
    return torch.equal(a.view(torch.int32) if a.dtype == F32 else a.view(torch.int16), b.view(torch.int32) if b.dtype == F32 else b.view(torch.int16))


SHAPES = [dict(rows=1, items=1, history=3, row_bias=3), dict(rows=1, items=3706, history=165, row_bias=4, item_bias=True),
          dict(rows=5, items=31, history=9, masks=3), dict(rows=4, items=33, masks=4, item_bias=True), dict(rows=3, items=2047, history=40, row_bias=7),
          dict(rows=3, items=2048, history=5, masks=1), dict(rows=7, items=2049, history=700, row_bias=300, masks=5, item_bias=True),
          dict(rows=33, items=10_007, history=60, row_bias=9, masks=4, item_bias=True), dict(rows=2, items=70_001, history=3000, masks=2),
          dict(rows=6, items=4096, row_bias=5), dict(rows=6, items=4097, item_bias=True), dict(rows=3, items=50, history=0, row_bias=0)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%d" % (s["rows"], s["items"]))
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("per_row", [True, False], ids=["rows", "all"])
def test_adjusted_scores(shape, dtype, per_row):
    p = Problem(dtype=dtype, per_row=per_row, seed=shape["items"], **shape)
    scores = p.s.cuda()
    got = adjust_scores(scores, p.rules())
    want = torch.from_numpy(p.plain(np.float32)[0]).to(dtype)
    assert same(got.cpu(), want)
    assert same(scores.cpu(), p.s)                                               # the input is left alone
    # the formula in 64 bits: at most six roundings of intermediates no larger than `size`, one rounding to the type (2^-25 below fp16's normals)
    exact, size = p.plain(np.float64)
    half = torch.finfo(dtype).eps / 2
    tol = 6 * 2.0 ** -24 * size + half * np.abs(np.where(np.isinf(exact), 0, exact)) * (1 + 2.0 ** -10) + 2.0 ** -25
    g = got.float().cpu().numpy().astype(np.float64)
    assert np.array_equal(np.isinf(g), np.isinf(exact))
    with np.errstate(invalid="ignore"):
        assert (np.abs(g - exact)[~np.isinf(exact)] <= tol[~np.isinf(exact)]).all()
    assert adjust_scores(scores, p.rules(), out=scores) is scores and same(scores.cpu(), want)      # in place


def test_rows_may_be_strided_and_start_anywhere():
    p = Problem(rows=9, items=1001, history=30, row_bias=5, masks=9, item_bias=True, seed=5)
    want = torch.from_numpy(p.plain(np.float32)[0])
    for dtype in (F32, BF16):
        wide = torch.full((9, 1100), 7.0, dtype=dtype, device="cuda")
        for start in (0, 1, 3, 98):
            view = wide[:, start:start + 1001]
            view.copy_(p.s)
            ref = torch.from_numpy(p.plain(np.float32)[0]).to(dtype) if dtype == F32 else None
            out = torch.full((9, 1050), 3.0, dtype=dtype, device="cuda")
            got = adjust_scores(view, p.rules(), out=out[:, 2:1003])
            assert (out[:, :2] == 3).all() and (out[:, 1003:] == 3).all()        # nothing around the rows is touched
            if ref is not None:
                assert same(got.cpu().contiguous(), ref)
            top = top_scores(view, 7, p.rules())
            assert same(top.scores.cpu(), torch.sort(adjust_scores(view.float().contiguous(), p.rules()).cpu(), dim=1, descending=True, stable=True)[0][:, :7].contiguous())
            wide.fill_(7.0)
    assert want.shape == (9, 1001)


def test_masked_places_hold_anything():
    s = torch.tensor([[NAN, INF, -INF, 1.0, torch.finfo(F32).min, -0.0, 0.0, 5.0]]).cuda().repeat(3, 1)
    mask = torch.tensor([[0, 0, 0, 1, 1, 1, 1, 0], [1, 1, 1, 1, 1, 1, 1, 1], [0] * 8], dtype=torch.bool).cuda()
    rules = ScoreRules(allowed=pack_allowed(mask))
    got = adjust_scores(s, rules).cpu()
    assert torch.equal(got[0], torch.tensor([-INF, -INF, -INF, 1.0, torch.finfo(F32).min, 0.0, 0.0, -INF]))
    assert torch.isnan(got[1, 0]) and torch.equal(got[1, 1:], s[1, 1:].cpu()) and (got[2] == -INF).all()
    items, scores = (x.cpu() for x in top_scores(s, 8, rules))
    assert items.tolist() == [[3, 5, 6, 4, -1, -1, -1, -1], [1, 7, 3, 5, 6, 4, -1, -1], [-1] * 8]
    assert (scores[2] == -INF).all() and scores[1, 0] == INF and (scores[0, 4:] == -INF).all()


def test_rows_that_name_nothing_and_rows_that_name_too_much():
    s = torch.arange(12.0).reshape(4, 3).cuda()
    off, ids = dev(np.array([0, 2, 3]), torch.int64), dev([0, 0, 2], torch.int32)
    rows = dev([0, -1, 2, 1], torch.int32)                                       # list 2 does not exist
    got = adjust_scores(s, ScoreRules(history=(off, ids), history_rows=rows, frequency=1.0)).cpu()
    assert torch.equal(got[[0, 1, 3]], torch.tensor([[-2.0, 1, 2], [3, 4, 5], [9, 10, 10]])) and torch.isnan(got[2]).all()
    top = top_scores(s, 2, ScoreRules(history=(off, ids), history_rows=rows, frequency=1.0))
    assert top.items.tolist() == [[2, 1], [2, 1], [-1, -1], [1, 2]]
    bad_mask = ScoreRules(allowed=torch.full((1, 1), -1, dtype=torch.int32).cuda(), allowed_rows=dev([0, 1, -1, -5], torch.int32))
    got = adjust_scores(s, bad_mask).cpu()
    assert torch.isnan(got[1]).all() and torch.equal(got[[0, 2, 3]], s.cpu()[[0, 2, 3]])
    # offsets that run past the list or backwards are cut to the list
    wild = dev([5, 99, -7, 2, 1], torch.int64)
    assert torch.equal(adjust_scores(s, ScoreRules(history=(wild, ids), presence=1.0)).cpu(), torch.tensor([[0.0, 1, 2], [3, 4, 5], [5, 7, 8], [9, 10, 11]]))


def test_no_rows_and_no_rules():
    empty = torch.zeros(0, 5).cuda()
    assert adjust_scores(empty, ScoreRules()).shape == (0, 5)
    assert top_scores(empty, 2).items.shape == (0, 2)
    s = torch.randn(3, 5).cuda()
    assert same(adjust_scores(s, ScoreRules()).cpu(), s.cpu())
    none = ScoreRules(history=(torch.zeros(4, dtype=torch.int64).cuda(), torch.zeros(0, dtype=torch.int32).cuda()), presence=2.0,
                      row_bias=(torch.zeros(4, dtype=torch.int64).cuda(), torch.zeros(0, dtype=torch.int32).cuda(), torch.zeros(0).cuda()))
    assert same(adjust_scores(s, none).cpu(), s.cpu())


def plain_top(s, n):
    """descending, the lower index first among equals, NaN and -inf nowhere"""
    s = s.astype(np.float32)
    items, values = np.full((s.shape[0], n), -1, np.int32), np.full((s.shape[0], n), -INF, np.float32)
    for r in range(s.shape[0]):
        ok = np.flatnonzero(s[r] > -INF)
        order = ok[np.argsort(-s[r, ok].astype(np.float64), kind="stable")][:n]
        items[r, :len(order)], values[r, :len(order)] = order, s[r, order]
    return items, values


@pytest.mark.parametrize("rows, items, n", [(1, 1, 1), (3, 2, 2), (2, 33, 5), (5, 2047, 10), (4, 2048, 2048), (3, 2049, 64), (2, 8192, 256), (2, 8193, 257),
                                            (3, 9000, 129), (2, 20_001, 1024), (2, 20_001, 1025), (1, 5000, 5000), (1, 200_000, 100), (7, 50_001, 10),
                                            (600, 3001, 33), (40, 30_000, 500), (2, 48_034, 390), (1, 120_000, 1024), (3, 700, 700)])
@pytest.mark.parametrize("kind", ["normal", "ties", "ascending", "constant", "gaps"])
def test_top_scores(rows, items, n, kind):
    rng = np.random.default_rng(items + n)
    if kind == "normal":
        s = rng.standard_normal((rows, items)).astype(np.float32)
    elif kind == "ties":
        s = rng.integers(-3, 4, (rows, items)).astype(np.float32) * rng.choice([1.0, -1.0], (rows, items)).astype(np.float32)       # -0 and 0 are equal
    elif kind == "ascending":                                                    # every score beats all before it
        s = np.broadcast_to(np.arange(items, dtype=np.float32), (rows, items)).copy()
    elif kind == "constant":
        s = np.full((rows, items), -2.5, np.float32)
    else:                                                                        # most of the row does not rank
        s = rng.standard_normal((rows, items)).astype(np.float32)
        s[rng.random((rows, items)) < 0.95] = -INF
        s[rng.random((rows, items)) < 0.01] = NAN
        s[rng.random((rows, items)) < 0.001] = INF
    got = top_scores(torch.from_numpy(s).cuda(), n)
    want_items, want_values = plain_top(s, n)
    assert np.array_equal(got.items.cpu().numpy(), want_items)
    assert np.array_equal(got.scores.cpu().numpy(), want_values)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_top_scores_of_half_width_rows(dtype):
    s = torch.randn(6, 30_003).to(dtype)                                         # (many ties)
    got = top_scores(s.cuda(), 40)
    want_items, want_values = plain_top(s.float().numpy(), 40)
    assert np.array_equal(got.items.cpu().numpy(), want_items) and np.array_equal(got.scores.cpu().numpy(), want_values)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows, items, n", [(700, 3, 1), (700, 5, 4), (700, 130, 128), (700, 655, 2), (700, 655, 600), (600, 900, 100), (6, 3204, 365), (6, 3204, 3), (3, 17_421, 3),
                                            (3, 17_421, 500), (2, 1030, 1029)])
def test_short_rows_and_short_ends(rows, items, n, dtype):
    """rows, or last segments of rows, whose vectors do not reach every wavefront"""
    s = torch.from_numpy(np.random.default_rng(items + n).standard_normal((rows, items)).astype(np.float32)).to(dtype)
    got = top_scores(s.cuda(), n)
    want_items, want_values = plain_top(s.float().numpy(), n)
    assert np.array_equal(got.items.cpu().numpy(), want_items) and np.array_equal(got.scores.cpu().numpy(), want_values)


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%d" % (s["rows"], s["items"]))
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_top_scores_under_rules_are_those_of_the_adjusted_rows(shape, dtype):
    p = Problem(dtype=dtype, seed=shape["items"] + 1, **shape)
    adjusted = p.plain(np.float32)[0]
    for n in {1, min(10, p.items), min(300, p.items), min(700, p.items)}:
        got = top_scores(p.s.cuda(), n, p.rules())
        want_items, want_values = plain_top(adjusted, n)
        assert np.array_equal(got.items.cpu().numpy(), want_items) and np.array_equal(got.scores.cpu().numpy(), want_values)


def test_rows_behind_two_thousand_million_elements():
    stride = 2 ** 31 + 24                                                        # the third row starts behind 2^32 elements
    store = torch.empty(2 * stride + 5000, dtype=F16, device="cuda")
    rows = torch.as_strided(store, (3, 4999), (stride, 1))
    p = Problem(rows=3, items=4999, history=50, row_bias=5, masks=3, dtype=F16, seed=9, empty_mask=False)
    rows.copy_(p.s)
    want = p.plain(np.float32)[0]
    got = top_scores(rows, 12, p.rules())
    assert np.array_equal(got.items.cpu().numpy(), plain_top(want, 12)[0])
    adjust_scores(rows, p.rules(), out=rows)
    assert same(rows.cpu().contiguous(), torch.from_numpy(want).to(F16))


def test_calls_on_another_stream_and_in_a_graph():
    p = Problem(rows=40, items=20_011, history=60, row_bias=9, masks=4, item_bias=True, seed=2)
    q = Problem(rows=40, items=20_011, history=60, row_bias=9, masks=4, item_bias=True, seed=3)
    rules, scores = p.rules(), p.s.cuda()
    one = p.s[:1].cuda()                                                         # few rows: the segments' workspace
    eager = adjust_scores(scores, rules).clone(), top_scores(scores, 20, rules), top_scores(one, 50)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = adjust_scores(scores, rules), top_scores(scores, 20, rules), top_scores(one, 50)
    torch.cuda.current_stream().wait_stream(side)
    assert same(other[0], eager[0]) and torch.equal(other[1].items, eager[1].items) and torch.equal(other[2].items, eager[2].items)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = adjust_scores(scores, rules), top_scores(scores, 20, rules), top_scores(one, 50)
    for source in (q, p, q):
        scores.copy_(source.s)
        one.copy_(source.s[:1])
        torch.cuda.synchronize()
        want = adjust_scores(scores, rules), top_scores(scores, 20, rules), top_scores(one, 50)      # (eager work between the replays)
        graph.replay()
        torch.cuda.synchronize()
        assert same(held[0], want[0])
        for h, w in zip(held[1:], want[1:]):
            assert torch.equal(h.items, w.items) and same(h.scores, w.scores)


def test_refusals_on_the_device():
    s = torch.zeros(2, 6).cuda()
    for bad in (0, 7):
        with pytest.raises(ValueError):
            top_scores(s, bad)
    with pytest.raises(ValueError):
        adjust_scores(s, ScoreRules(item_bias=torch.zeros(6)))                   # the bias is in host memory
    with pytest.raises(ValueError):
        adjust_scores(torch.zeros(2, 6), ScoreRules())                           # the scores are
    wide = torch.zeros(3, 6).cuda()
    with pytest.raises(ValueError):
        adjust_scores(wide[:2], ScoreRules(), out=wide[1:])                      # overlaps
    for out in (torch.zeros(2, 5).cuda(), torch.zeros(2, 6, dtype=F16).cuda(), torch.zeros(2, 6), torch.zeros(6, 2).cuda().t()):
        with pytest.raises(ValueError):
            adjust_scores(s, ScoreRules(), out=out)


def test_calls_on_two_streams_at_once():
    """rows cut into segments, whose keys go through a workspace: one per call"""
    s = [torch.randn(3, 120_001).cuda(), torch.randn(40, 30_011).cuda()]
    want = [top_scores(x, 50) for x in s]
    adjusted = [adjust_scores(x, ScoreRules(item_bias=torch.arange(x.shape[1], dtype=torch.float32).cuda() / 1000)) for x in s]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(8):
        for st, x, out in zip(streams, s, got):
            with torch.cuda.stream(st):
                bias = torch.arange(x.shape[1], dtype=torch.float32, device="cuda") / 1000
                out.append((top_scores(x, 50), adjust_scores(x, ScoreRules(item_bias=bias))))
    torch.cuda.synchronize()
    for w, a, results in zip(want, adjusted, got):
        for top, rows in results:
            assert torch.equal(top.items, w.items) and torch.equal(top.scores, w.scores) and torch.equal(rows, a)


@pytest.mark.parametrize("listed, kinds", [(700, 1), (760, 760), (769, 769), (1024, 1024), (2000, 767), (2000, 770), (5000, 40), (5000, 5000)])
@pytest.mark.parametrize("rows, items", [(2, 9000), (3, 60_007)], ids=["one segment or two", "many segments"])
def test_top_scores_under_long_lists(rows, items, listed, kinds):
    """lists of `listed` entries that name `kinds` different items: few enough for the table of items, just too many, far too many"""
    rng = np.random.default_rng(listed + kinds)
    p = Problem(rows, items, seed=listed, history=4, row_bias=3, item_bias=True, masks=rows)
    p.hist = [rng.choice(items, kinds, replace=False)[rng.permutation(np.arange(listed) % kinds)] for _ in range(rows)]
    p.hist_rows = np.arange(rows, dtype=np.int32)[::-1].copy()
    p.mask[0] = True
    adjusted = p.plain(np.float32)[0]
    for n in (5, 300, 384, 385, 800):
        got = top_scores(p.s.cuda(), n, p.rules())
        want_items, want_values = plain_top(adjusted, n)
        assert np.array_equal(got.items.cpu().numpy(), want_items) and np.array_equal(got.scores.cpu().numpy(), want_values)
    assert same(adjust_scores(p.s.cuda(), p.rules()).cpu(), torch.from_numpy(adjusted))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("kind", ["normal", "few values", "ascending", "late"])
def test_long_lists_of_long_rows(dtype, kind):
    """more candidates than a wavefront holds, again and again: thresholds from what it has, shared among the four"""
    rng = np.random.default_rng(8)
    if kind == "normal":
        s = rng.standard_normal((600, 40_003))
    elif kind == "few values":
        s = rng.integers(0, 5, (600, 40_003)) - 2.0
    elif kind == "ascending":
        s = np.sort(rng.standard_normal((600, 40_003)))
    else:                                                                        # all that counts stands in what one wavefront reads
        s = rng.standard_normal((600, 40_003)) * 0.01
        s[:, 20_000:20_256] += 3.0
    s = torch.from_numpy(s.astype(np.float32)).to(dtype)
    for n in (200, 500, 768, 769, 1540):
        got = top_scores(s.cuda(), n)
        want_items, want_values = plain_top(s[:5].float().numpy(), n)
        assert np.array_equal(got.items[:5].cpu().numpy(), want_items) and np.array_equal(got.scores[:5].cpu().numpy(), want_values)
        value, _ = torch.sort(s.cuda().float(), dim=1, descending=True)
        assert torch.equal(got.scores, value[:, :n])


@pytest.mark.parametrize("rows", [255, 256, 511, 512])
@pytest.mark.parametrize("ruled", [False, True], ids=["plain", "ruled"])
def test_rows_around_the_counts_that_are_cut(rows, ruled):
    s = torch.from_numpy(np.random.default_rng(rows).standard_normal((rows, 110_003)).astype(np.float32)).to(F16).cuda()
    bias = torch.linspace(-0.1, 0.1, 110_003).cuda()
    got = top_scores(s, 70, ScoreRules(item_bias=bias) if ruled else None)
    full = s.float() + bias if ruled else s.float()
    value, _ = torch.sort(full, dim=1, descending=True)
    assert torch.equal(got.scores, value[:, :70]) and torch.equal(full.gather(1, got.items.long()), got.scores)
