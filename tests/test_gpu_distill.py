"""distill_loss / distill_gradients against the formula in float64 and against differences of it.

Tolerances, with E = 2^-24 (half a step of float32) and S = max over (row, item) of sum_k |u_k v_k| + |bias|:
  a score is a sum of K products and a bias: off by at most (K + 4) E S, so z / tau by ez = (K + 6) E S / tau;
  exp, log and the division are good to 2 steps (4 E); the sum over I items adds at most (I / 32 + 64) E (partial sums over lanes, wavefronts
  and slices are shorter than I / 32 + 64 additions for the sizes below): q is off by eq = 2 ez + (I / 32 + 80) E of itself, and so is p by
  ep = (n + 80 + 8 T) E, T the largest |teacher score| / tau;
  loss: tau^2 (2 ez + (eq + ep) + (n + 80) E L), L the largest |log p| + |z| / tau + |lse|;
  a gradient sums terms |dz| |factor| over I items (or R rows): relative to the sum of the terms' sizes, (I + 64) E (or R) for the additions and
  eq + ep for the terms."""
import numpy as np
import pytest
import torch

from rankfm_amd import distill_gradients, distill_loss, pack_allowed

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
NAN, INF = float("nan"), float("inf")


class Problem:
    def __init__(self, rows, items, factors, n, tau=1.0, mask=None, weight=True, bias=True, seed=0, spread=1.2):
        rng = np.random.default_rng(seed)
        scale = (spread / np.sqrt(factors)) ** 0.5
        self.tau = tau
        self.u, self.v = (rng.standard_normal((rows, factors)) * scale).astype(np.float32), (rng.standard_normal((items, factors)) * scale).astype(np.float32)
        self.b = (rng.standard_normal(items) * 0.5).astype(np.float32) if bias else None
        self.t = (rng.standard_normal((rows, n)) * 2).astype(np.float32)
        self.ti = rng.integers(-1, items + 1, (rows, n)).astype(np.int32)         # padding, entries behind the catalogue, some items twice
        if n > 3 and rows > 1:
            self.ti[1, 2] = self.ti[1, 0] = 0
            self.ti[0] = -1                                                       # nothing to learn from
            self.t[-1, 0] = -INF
        self.g = (rng.random(rows) + 0.5).astype(np.float32) if weight else None
        self.mask = self.which = None
        if mask == "rows":
            self.mask = rng.random((rows, items)) < 0.7
            self.mask[rows // 2] = False                                          # a row that nothing is left of
        elif mask == "one":
            self.mask = rng.random((1, items)) < 0.5
        elif mask == "few":
            self.mask = rng.random((3, items)) < 0.7
            self.which = rng.integers(-1, 3, rows).astype(np.int32)

    def given(self):
        dev = lambda a: None if a is None else torch.from_numpy(a).cuda()        # noqa: E731
        return ((dev(self.u), dev(self.v), dev(self.b), dev(self.ti), dev(self.t)),
                dict(temperature=self.tau, allowed=None if self.mask is None else pack_allowed(dev(self.mask)), allowed_rows=dev(self.which)))

    def exact(self, u=None, v=None, b=None):
        """loss, gradients (of sum g loss) in float64, and the sizes their errors are relative to"""
        rows, items, tau = self.u.shape[0], self.v.shape[0], self.tau
        u = (self.u if u is None else u).astype(np.float64)
        v = (self.v if v is None else v).astype(np.float64)
        b = np.zeros(items) if self.b is None else (self.b if b is None else b).astype(np.float64)
        g = np.ones(rows) if self.g is None else self.g.astype(np.float64)
        z = (u @ v.T + b) / tau
        ok = np.ones((rows, items), bool)
        if self.mask is not None:
            for r in range(rows):
                m = self.which[r] if self.which is not None else (r if len(self.mask) == rows else 0)
                ok[r] = self.mask[m] if m >= 0 else True
        loss, dz, big = np.zeros(rows), np.zeros((rows, items)), 1.0
        pq = np.zeros((rows, items))
        for r in range(rows):
            use = [j for j in range(self.ti.shape[1]) if 0 <= self.ti[r, j] < items and ok[r, self.ti[r, j]] and self.t[r, j] > -INF]
            if not use:
                continue
            t = self.t[r, use].astype(np.float64) / tau
            log_p = t - t.max() - np.log(np.exp(t - t.max()).sum())
            zr = np.where(ok[r], z[r], -INF)
            lse = zr.max() + np.log(np.exp(zr - zr.max()).sum())
            ids = self.ti[r, use]
            loss[r] = tau * tau * (np.exp(log_p) * (log_p - z[r, ids] + lse)).sum()
            big = max(big, np.abs(log_p).max() + np.abs(z[r, ids]).max() + abs(lse))
            q = np.exp(zr - lse)
            dz[r], pq[r] = q, q
            np.subtract.at(dz[r], ids, np.exp(log_p))
            np.add.at(pq[r], ids, np.exp(log_p))
        coef = (tau * g)[:, None]
        dz, pq = dz * coef, np.abs(pq * coef)
        s = (np.abs(u) @ np.abs(v).T + np.abs(b)).max()
        n, k = self.ti.shape[1], u.shape[1]
        ez = (k + 6) * E * s / tau
        eq, ep = 2 * ez + (items / 32 + 80) * E, (n + 80 + 8 * np.abs(np.where(np.isinf(self.t), 0, self.t)).max() / tau) * E
        tol = (tau * tau * (2 * ez + eq + ep + (n + 80) * E * big), (eq + ep + (items + 64) * E) * (pq @ np.abs(v)) + 1e-30,
               (eq + ep + (rows + 64) * E) * (pq.T @ np.abs(u)) + 1e-30, (eq + ep + (rows + 64) * E) * pq.sum(0) + 1e-30)
        return (loss, dz @ v, dz.T @ u, dz.sum(0)), tol


CASES = [dict(rows=1, items=1, factors=1, n=1), dict(rows=1, items=33, factors=3, n=3), dict(rows=2, items=2, factors=7, n=5),
         dict(rows=3, items=64, factors=16, n=4, tau=0.5), dict(rows=5, items=1000, factors=20, n=10, mask="rows"), dict(rows=31, items=127, factors=32, n=6, mask="few"),
         dict(rows=64, items=257, factors=50, n=7, tau=3.0), dict(rows=129, items=2049, factors=64, n=32, mask="one"), dict(rows=130, items=1023, factors=64, n=33, mask="rows"),
         dict(rows=33, items=777, factors=128, n=64), dict(rows=257, items=300, factors=96, n=11, mask="rows"), dict(rows=70, items=500, factors=130, n=5, mask="few"),
         dict(rows=9, items=300, factors=257, n=3), dict(rows=300, items=5003, factors=31, n=12, weight=False, bias=False), dict(rows=1000, items=90, factors=12, n=100, tau=2.0),
         dict(rows=4, items=20_011, factors=65, n=1000, mask="few"), dict(rows=2, items=3, factors=1024, n=2)]


def ids(c):
    return "%dx%dx%d n%d %s" % (c["rows"], c["items"], c["factors"], c["n"], c.get("mask", ""))


@pytest.mark.parametrize("case", CASES, ids=ids)
def test_loss_and_gradients(case):
    p = Problem(seed=case["items"], **case)
    (args, kw) = p.given()
    want, tol = p.exact()
    loss = distill_loss(*args, **kw)
    got = distill_gradients(*args, row_weight=None if p.g is None else torch.from_numpy(p.g).cuda(), **kw)
    for name, g, w, t in (("loss", loss, want[0], tol[0]), ("loss", got.loss, want[0], tol[0]), ("users", got.users, want[1], tol[1]), ("items", got.items, want[2], tol[2]),
                          ("bias", got.bias, want[3], tol[3])):
        if name == "bias" and p.b is None:
            assert g is None
            continue
        off = np.abs(g.cpu().numpy().astype(np.float64) - w) / t
        assert (off <= 1).all(), (name, float(off.max()), int(off.argmax()))
    if case["n"] > 3 and case["rows"] > 1:
        assert got.loss[0] == 0 and (got.users[0] == 0).all()
    again = distill_gradients(*args, row_weight=None if p.g is None else torch.from_numpy(p.g).cuda(), **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, again) if a is not None)    # the same bits


def test_gradients_are_those_of_differences():
    """central differences of the float64 loss along random directions: error h^2 of the third derivative; h = 1e-4 and a relative bound of 1e-5 hold by a
    wide margin for losses of this size"""
    p = Problem(rows=40, items=300, factors=24, n=8, tau=1.5, mask="few", seed=4)
    args, kw = p.given()
    got = distill_gradients(*args, row_weight=torch.from_numpy(p.g).cuda(), **kw)
    rng, h = np.random.default_rng(1), 1e-4
    total = lambda **w: float((p.g * p.exact(**w)[0][0]).sum())                   # noqa: E731
    for name, x, grad in (("u", p.u, got.users), ("v", p.v, got.items), ("b", p.b, got.bias)):
        d = rng.standard_normal(x.shape)
        slope = (total(**{name: x + h * d}) - total(**{name: x - h * d})) / (2 * h)
        size = float((np.abs(grad.cpu().numpy()) * np.abs(d)).sum())
        assert abs(slope - float((grad.cpu().numpy().astype(np.float64) * d).sum())) <= 1e-5 * size, name


def test_rows_may_be_strided():
    p = Problem(rows=37, items=210, factors=20, n=6, seed=7)
    args, kw = p.given()
    wide_u, wide_v = torch.full((37, 32), NAN).cuda(), torch.full((210, 27), NAN).cuda()
    wide_u[:, 5:25], wide_v[:, 1:21] = args[0], args[1]
    a = distill_gradients(*args, **kw)
    b = distill_gradients(wide_u[:, 5:25], wide_v[:, 1:21], *args[2:], **kw)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_large_scores_do_not_overflow():
    p = Problem(rows=20, items=400, factors=40, n=5, seed=8, spread=400.0)
    want, tol = p.exact()
    args, kw = p.given()
    got = distill_gradients(*args, row_weight=torch.from_numpy(p.g).cuda(), **kw)
    for g, w, t in zip(got, want, tol):
        assert (np.abs(g.cpu().numpy() - w) <= t).all()


def test_infinities_and_nan():
    p = Problem(rows=6, items=70, factors=8, n=4, seed=9)
    p.ti = np.abs(p.ti) % 60
    args, kw = p.given()
    clean = distill_gradients(*args, **kw)
    bias = args[2].clone()
    bias[65] = -INF                                                               # an item that cannot come out: its share of q is 0
    off = distill_gradients(args[0], args[1], bias, *args[3:], **kw)
    assert torch.isfinite(off.loss).all() and torch.isfinite(off.users).all() and (off.items[65] == 0).all() and off.bias[65] == 0
    bad = args[0].clone()
    bad[2, 3] = NAN                                                               # a bad user row spoils its own loss and what is summed over rows
    got = distill_gradients(bad, *args[1:], **kw)
    keep = [0, 1, 3, 4, 5]
    assert torch.isnan(got.loss[2]) and torch.isnan(got.users[2]).all() and torch.isnan(got.items).any()
    assert torch.equal(got.loss[keep], clean.loss[keep]) and torch.equal(got.users[keep], clean.users[keep])
    scores = args[4].clone()
    scores[1] = -INF                                                              # every entry off: an empty row
    got = distill_gradients(*args[:4], scores, **kw)
    assert got.loss[1] == 0 and (got.users[1] == 0).all() and torch.equal(got.loss[keep[2:]], clean.loss[keep[2:]])
    allowed = torch.full((1, 3), -1, dtype=torch.int32).cuda()
    which = torch.tensor([0, 0, 1, -1, 0, 0], dtype=torch.int32).cuda()           # mask 1 does not exist
    got = distill_gradients(*args, temperature=1.0, allowed=allowed, allowed_rows=which)
    assert torch.isnan(got.loss[2]) and torch.isfinite(got.items).all() and (got.users[2] == 0).all()
    assert torch.equal(got.loss[keep], clean.loss[keep])


def test_no_rows():
    v, b = torch.randn(30, 8).cuda(), torch.randn(30).cuda()
    u, ti, t = torch.zeros(0, 8).cuda(), torch.zeros(0, 3, dtype=torch.int32).cuda(), torch.zeros(0, 3).cuda()
    assert distill_loss(u, v, b, ti, t).shape == (0,)
    got = distill_gradients(u, v, b, ti, t)
    assert got.users.shape == (0, 8) and (got.items == 0).all() and (got.bias == 0).all()


def test_streams_and_graphs():
    p, q = (Problem(rows=150, items=3001, factors=40, n=9, mask="few", seed=s) for s in (1, 2))
    args, kw = p.given()
    eager = distill_gradients(*args, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = distill_gradients(*args, **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = distill_gradients(*args, **kw)
        held_loss = distill_loss(*args, **kw)
    for source in (q, p, q):
        for a, s in zip(args, source.given()[0]):
            a.copy_(s)
        torch.cuda.synchronize()
        want = distill_gradients(*args, **kw)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)) and torch.equal(held_loss, distill_loss(*args, **kw))


def test_refusals():
    args, kw = Problem(rows=4, items=9, factors=3, n=2).given()
    u, v, b, ti, t = args
    for bad in ((u.cpu(), v, b, ti, t), (u, v[:, :2], b, ti, t), (u, v, b[:8], ti, t), (u, v, b, ti.long(), t), (u, v, b, ti, t[:, :1]), (u, v, b, ti[:3], t[:3]),
                (u.double(), v, b, ti, t), (u, v.cpu(), b, ti, t), (u, v, b, ti[:, :0], t[:, :0]), (u, v[:0], b[:0], ti, t)):
        with pytest.raises(ValueError):
            distill_loss(*bad)
    for bad in (dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=NAN), dict(temperature=INF), dict(allowed=torch.zeros(4, 2, dtype=torch.int32).cuda()),
                dict(allowed=torch.zeros(3, 1, dtype=torch.int32).cuda()), dict(allowed_rows=torch.zeros(4, dtype=torch.int32).cuda()), dict(row_weight=torch.ones(3).cuda())):
        with pytest.raises(ValueError):
            distill_gradients(*args, **bad)
    many = torch.zeros(4, 1025, dtype=torch.int32).cuda()
    with pytest.raises(ValueError):
        distill_loss(u, v, b, many, many.float())


def test_padding_rows_do_not_reach_the_gradients_whatever_they_hold():
    for factors in (20, 200):                                                     # both paths
        p = Problem(rows=70, items=400, factors=factors, n=6, seed=11)
        p.ti = np.abs(p.ti) % 400
        args, kw = p.given()
        weight = torch.from_numpy(p.g).cuda()
        pad = [3, 31, 32, 69]
        keep = [r for r in range(70) if r not in pad]
        ti = args[3].clone()
        ti[pad] = -1
        clean = distill_gradients(*args[:3], ti, args[4], row_weight=weight, **kw)
        u, t, g = args[0].clone(), args[4].clone(), weight.clone()
        u[pad[0]], u[pad[1]], u[pad[2]], u[pad[3]] = NAN, INF, -INF, 3e38
        t[pad] = NAN
        g[pad] = NAN
        got = distill_gradients(u, args[1], args[2], ti, t, row_weight=g, **kw)
        assert (got.loss[pad] == 0).all() and (got.users[pad] == 0).all()
        for a, b in zip(got, clean):
            assert torch.equal(a[keep], b[keep]) if a.shape[0] == 70 else torch.equal(a, b)


def test_many_entries_in_one_tile_and_items_twice():
    """every row's list in the same 32 items, some of them several times: the teacher's patch is full"""
    p = Problem(rows=100, items=5000, factors=40, n=60, seed=12)
    p.ti = 640 + np.random.default_rng(0).integers(0, 32, (100, 60)).astype(np.int32)
    want, tol = p.exact()
    args, kw = p.given()
    got = distill_gradients(*args, row_weight=torch.from_numpy(p.g).cuda(), **kw)
    for g, w, t in zip(got, want, tol):
        assert (np.abs(g.cpu().numpy() - w) <= t).all()


@pytest.mark.parametrize("factors", [20, 50, 100, 200])
def test_masked_items_may_hold_anything(factors):
    """an item that a row's mask takes out reaches neither the row's loss nor its gradient, and the row does not reach the item's.  (Not the bits of a clean
    call: the power of two that a tile of 32 items is scaled by is that of its largest finite factor, masked or not, and what is below the 22 bits of a
    weight's two parts is cut elsewhere.  The bounds are those above.)"""
    p = Problem(rows=70, items=400, factors=factors, n=6, mask="one", seed=13)
    p.ti = np.abs(p.ti) % 400
    p.mask[0, [0, 17, 64, 399]] = False
    args, kw = p.given()
    want, tol = p.exact()
    weight = torch.from_numpy(p.g).cuda()
    v = args[1].clone()
    v[0], v[17], v[64, 3], v[399] = NAN, INF, -INF, NAN
    got = distill_gradients(args[0], v, *args[2:], row_weight=weight, **kw)
    for x, w, t in zip((*got, distill_loss(args[0], v, *args[2:], **kw)), (*want, want[0]), (*tol, tol[0])):
        assert (np.abs(x.cpu().numpy() - w) <= t).all()
    u = args[0].clone()
    u[5, 1], u[40] = NAN, INF
    got = distill_gradients(u, *args[1:], **kw)
    off = torch.from_numpy(~p.mask[0]).cuda()
    assert torch.isnan(got.loss[[5, 40]]).all() and torch.isnan(got.users[[5, 40]]).all()
    assert (got.items[off] == 0).all() and (got.bias[off] == 0).all() and torch.isnan(got.items[~off]).all() and torch.isnan(got.bias[~off]).all()


@pytest.mark.parametrize("rows,items,factors,n,given", [(4129, 32_801, 20, 9, True), (1030, 129_037, 64, 40, True), (4500, 30_001, 33, 6, False)], ids=["long", "wide", "plain"])
def test_large_problems(rows, items, factors, n, given):
    """more than 2^17 pairs of tiles of 32 rows and 32 items: wavefronts with two column tiles each.  The reference is the formula in float64 on the device"""
    tau = 1.5
    p = Problem(rows, items, factors, n, tau=tau, weight=given, bias=given, seed=factors)
    args, kw = p.given()
    dev = lambda a: torch.from_numpy(a).cuda().double()                           # noqa: E731
    u, v = dev(p.u), dev(p.v)
    b, g = dev(p.b) if given else torch.zeros(items, dtype=torch.float64, device="cuda"), dev(p.g) if given else torch.ones(rows, dtype=torch.float64, device="cuda")
    z = (u @ v.T + b) / tau
    lse = torch.logsumexp(z, 1)
    ti, t = args[3].long(), args[4].double() / tau
    ok = (ti >= 0) & (ti < items) & (t > -INF)
    live = ok.any(1)
    log_p = torch.where(ok, t, -INF)
    log_p = torch.where(ok, log_p - torch.logsumexp(torch.where(live[:, None], log_p, 0.0), 1, keepdim=True), 0.0)
    share = torch.where(ok, log_p.exp(), 0.0)
    at = torch.where(ok, z.gather(1, ti.clamp(0, items - 1)), 0.0)
    loss = torch.where(live, tau * tau * (share * (log_p - at + lse[:, None])).sum(1), 0.0)
    big = float((log_p.abs().amax(1) + at.abs().amax(1) + lse.abs()).max().clamp(min=1.0))
    s = float((u.abs() @ v.abs().T + b.abs()).max())
    coef = (tau * g * live)[:, None]
    q = (z - lse[:, None]).exp_()
    q *= coef
    teacher = torch.zeros_like(q).scatter_add_(1, ti.clamp(0, items - 1), share * coef)
    dz, pq = q - teacher, q + teacher
    ez = (factors + 6) * E * s / tau
    eq, ep = 2 * ez + (items / 32 + 80) * E, (n + 80 + 8 * float(np.abs(np.where(np.isinf(p.t), 0, p.t)).max()) / tau) * E
    rel_i, rel_r = eq + ep + (items + 64) * E, eq + ep + (rows + 64) * E
    got = distill_gradients(*args, row_weight=torch.from_numpy(p.g).cuda() if given else None, **kw)
    alone = distill_loss(*args, **kw)
    tol = tau * tau * (2 * ez + eq + ep + (n + 80) * E * big)
    for name, x, want, t in (("loss", alone, loss, tol), ("loss", got.loss, loss, tol), ("users", got.users, dz @ v, rel_i * (pq @ v.abs()) + 1e-30),
                             ("items", got.items, dz.T @ u, rel_r * (pq.T @ u.abs()) + 1e-30), ("bias", got.bias, dz.sum(0), rel_r * pq.sum(0) + 1e-30)):
        if x is None:
            assert name == "bias" and not given
            continue
        off = float(((x.double() - want).abs() / t).max())
        assert off <= 1, (name, off)
    again = distill_gradients(*args, row_weight=torch.from_numpy(p.g).cuda() if given else None, **kw)
    assert all(torch.equal(x, y) for x, y in zip(got, again) if x is not None)


@pytest.mark.parametrize("factors", [24, 64, 128])
def test_rows_of_very_different_size_share_a_tile(factors):
    """users from 1e-2 to 1e2 of the others' size, every size in every tile of 32.  A row's bound counts its own scores, and what a factor may be off by next to
    the largest of its tile: 2^-40 of that, against the item's factors (and the other way round), summed over the factors"""
    p = Problem(rows=100, items=700, factors=factors, n=8, tau=1.0, seed=14)
    p.u *= (10.0 ** (np.arange(100) % 5 - 2.0))[:, None].astype(np.float32)
    want, _ = p.exact()
    args, kw = p.given()
    u, v = np.abs(p.u).astype(np.float64), np.abs(p.v).astype(np.float64)
    s = (u @ v.T + np.abs(p.b)).max(1)
    ez = (factors + 6) * E * s + 2.0 ** -40 * factors * (u.max() * v.max() + u.max(1) * v.max())
    t = np.abs(np.where(np.isinf(p.t), 0, p.t)).max(1)
    eq, ep = 2 * ez + (700 / 32 + 80) * E, (8 + 80 + 8 * t) * E
    big = 2 * t + np.log(8) + 2 * s + np.log(700)                                 # |log p| <= 2 max |t| + log n;  |z|, |lse| <= s, s + log I
    tol = 2 * ez + eq + ep + 88 * E * big
    for got in (distill_loss(*args, **kw), distill_gradients(*args, **kw).loss):
        assert (np.abs(got.cpu().numpy() - want[0]) <= tol).all()


def test_calls_on_two_streams_at_once():
    """every call has a workspace of its own: many in flight on two streams, with different inputs and sizes, give what they give alone"""
    problems = [Problem(rows=600, items=9001, factors=48, n=12, mask="few", seed=21), Problem(rows=333, items=20_005, factors=100, n=30, seed=22)]
    given = [p.given() for p in problems]
    alone = [distill_gradients(*args, **kw) for args, kw in given]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(6):
        for s, (args, kw), out in zip(streams, given, got):
            with torch.cuda.stream(s):
                out.append(distill_gradients(*args, **kw))
    torch.cuda.synchronize()
    for want, results in zip(alone, got):
        assert all(torch.equal(a, b) for r in results for a, b in zip(r, want))


def test_two_graphs_in_turn_and_at_once():
    given = [Problem(rows=90, items=1500, factors=24, n=6, seed=s).given() for s in (31, 32)]
    want = [distill_gradients(*args, **kw) for args, kw in given]
    torch.cuda.synchronize()
    graphs, held = [], []
    for args, kw in given:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(distill_gradients(*args, **kw))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for h, w in zip(held, want) for a, b in zip(h, w))
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for h, w in zip(held, want) for a, b in zip(h, w))


@pytest.mark.parametrize("factors", [20, 64, 128, 200])
@pytest.mark.parametrize("what", ["zero users", "zero items", "zero both", "one tile of zeros", "small"])
def test_factors_of_nothing(factors, what):
    """zeros: a fresh model's.  small: everything 1e-7 of the usual size, the scores all but equal and the gradients as small as the factors"""
    p = Problem(rows=70, items=333, factors=factors, n=6, seed=15)
    if what in ("zero users", "zero both"):
        p.u[:] = 0
    if what in ("zero items", "zero both"):
        p.v[:] = 0
    if what == "one tile of zeros":
        p.u[32:64], p.v[64:96] = 0, 0
    if what == "small":
        p.u, p.v = p.u * np.float32(1e-7), p.v * np.float32(1e-7)
    want, tol = p.exact()
    args, kw = p.given()
    got = distill_gradients(*args, row_weight=torch.from_numpy(p.g).cuda(), **kw)
    for x, w, t in zip((*got, distill_loss(*args, **kw)), (*want, want[0]), (*tol, tol[0])):
        assert (np.abs(x.cpu().numpy() - w) <= t).all()


@pytest.mark.parametrize("case", [dict(rows=r, items=i, factors=k, n=n, mask=m, tau=1.5) for r, i, k, n, m in (
    (1, 1, 1, 1, None), (2, 31, 7, 3, "rows"), (31, 4097, 20, 9, "rows"), (32, 9001, 32, 5, None), (33, 5003, 33, 7, "few"), (64, 20_011, 64, 40, "one"), (63, 8192, 79, 12, "rows"),
    (65, 7777, 96, 6, None), (96, 12_345, 101, 33, "few"), (97, 3001, 128, 10, "rows"), (128, 30_007, 50, 20, None), (128, 6007, 127, 20, "rows"), (129, 6007, 127, 20, "rows"),
    (20, 70_001, 60, 200, "few"), (29, 20_500, 128, 9, "rows"), (64, 20_511, 97, 9, None), (33, 5122, 32, 9, "rows"), (64, 10_250, 64, 9, "one"))], ids=ids)
def test_few_rows(case):
    """one or two tiles of rows, and more; catalogues on both sides of the sizes from which their tables are taken as they are, reaching every workgroup once,
    several times or not at all"""
    p = Problem(seed=case["items"], **case)
    want, tol = p.exact()
    args, kw = p.given()
    weight = torch.from_numpy(p.g).cuda()
    got = distill_gradients(*args, row_weight=weight, **kw)
    for x, w, t in zip((*got, distill_loss(*args, **kw)), (*want, want[0]), (*tol, tol[0])):
        assert (np.abs(x.cpu().numpy() - w) <= t).all()
    again = distill_gradients(*args, row_weight=weight, **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    wide_u, wide_v = torch.full((case["rows"], 131), NAN).cuda(), torch.full((case["items"], 133), NAN).cuda()
    k = case["factors"]
    wide_u[:, 1:k + 1], wide_v[:, 3:k + 3] = args[0], args[1]
    strided = distill_gradients(wide_u[:, 1:k + 1], wide_v[:, 3:k + 3], *args[2:], row_weight=weight, **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, strided))


@pytest.mark.parametrize("factors", [20, 64, 128])
def test_few_rows_and_masked_items_that_hold_anything(factors):
    p = Problem(rows=40, items=3000, factors=factors, n=6, mask="one", seed=23)
    p.ti = np.abs(p.ti) % 3000
    p.mask[0, [0, 17, 64, 2999]] = False
    args, kw = p.given()
    want, tol = p.exact()
    v = args[1].clone()
    v[0], v[17], v[64, 3], v[2999] = NAN, INF, -INF, NAN
    got = distill_gradients(args[0], v, *args[2:], row_weight=torch.from_numpy(p.g).cuda(), **kw)
    for x, w, t in zip((*got, distill_loss(args[0], v, *args[2:], **kw)), (*want, want[0]), (*tol, tol[0])):
        assert (np.abs(x.cpu().numpy() - w) <= t).all()
    v[5, 2] = NAN                                                                 # and an item that may be had
    if p.mask[0, 5]:
        got = distill_gradients(args[0], v, *args[2:], **kw)
        assert torch.isnan(got.loss[2:]).all() and torch.isnan(got.users[2:]).all()
