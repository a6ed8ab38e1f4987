"""distill_loss / distill_gradients where the scores themselves carry no rounding: factors of 0 and +-1, whole biases, a temperature of log2(e), so that
softmax weights are powers of two and their sums exact.  What is left are a handful of roundings, whatever the catalogue's length, and every tile of 32 rows
or items has a factor of its own class: a tile left out or taken twice is off by percents of a gradient, against tolerances of 1e-5.

Tolerances, with E = 2^-24 and D the largest |log2 q| + |lse| + |z| (log2 units; ln 2 < 0.7 turns them into relative ones):
  eq   a weight q: the temperature's own rounding, the lse's, the exponent's and its parts', each at most E of D, one step of the logarithm and two
       of exp2, 2^-23 for a weight's two half-precision parts:  E (0.7 * 5 D + 12).  Beyond 128 factors expf of natural units: the same count
  ep   a teacher's p (equal scores):  E (n + 8)
  a gradient is a sum of terms |dz| |factor| (exact factors): eq + ep of each, and the additions -- 100 in a tile of 32 rows, one per tile and split
  a weight's parts are cut at 2^-40 of the largest weight that its column has in the tile:  2^-40 of that for each of the 32 terms
  loss: tau^2 (p's part: (n + 8) E of its size; lse and z: 4 E D)"""
import numpy as np
import pytest
import torch

from rankfm_amd import distill_gradients, distill_loss, pack_allowed

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
TAU = float(np.float32(1.4426950408889634))
NAN, INF = float("nan"), float("inf")


def check(users, items, bias, ti, weight=None, mask=None, which=None, additions=None):
    """both calls against float64; teacher scores are all equal.  mask: bool [masks, items] on the device"""
    rows, catalogue, n = users.shape[0], items.shape[0], ti.shape[1]
    t = torch.zeros(ti.shape, device="cuda")
    kw = dict(temperature=TAU, allowed=None if mask is None else pack_allowed(mask), allowed_rows=which)
    got = distill_gradients(users, items, bias, ti, t, row_weight=weight, **kw)
    alone = distill_loss(users, items, bias, ti, t, **kw)
    u, v = users.double(), items.double()
    z2 = u @ v.T + bias.double()                                                  # log2 units but for the temperature's rounding
    z = z2 / TAU
    usable = (ti >= 0) & (ti < catalogue)
    at = ti.long().clamp(0, catalogue - 1)
    if mask is not None:
        ok = mask.expand(rows, -1) if which is None else torch.where(which[:, None] >= 0, mask[which.long().clamp(min=0)], True)
        z = torch.where(ok, z, -INF)
        usable = usable & ok.gather(1, at)
    live = usable.any(1)
    lse = torch.where(live, torch.logsumexp(z, 1), 0.0)
    count = usable.sum(1, keepdim=True).clamp(min=1)
    p = usable.double() / count
    log_q = torch.where(usable, z.gather(1, at) - lse[:, None], 0.0)
    loss = torch.where(live, TAU * TAU * (p * (-torch.log(count.double()) - log_q)).sum(1), 0.0)
    q = torch.where(live[:, None], torch.exp(z - lse[:, None]), 0.0)
    teacher = torch.zeros_like(q).scatter_add_(1, at, p)
    coef = (TAU * live * (weight.double() if weight is not None else 1.0))[:, None]
    coef = torch.where(live[:, None], coef, 0.0)                                  # (a dead row's weight may be anything)
    dz, size = (q - teacher) * coef, (q + teacher) * coef.abs()
    finite = torch.where(z > -INF, z, 0.0)
    D = float((finite - lse[:, None]).abs().max() + lse.abs().max() + finite.abs().max()) * 1.4427
    eq, ep = E * (0.7 * 5 * D + 12), E * (n + 8)
    # 2^-40 of a tile's largest weight per row, for each of its items; and per item, for each of a tile's rows
    pad = (-catalogue) % 32
    by_tile = torch.nn.functional.pad(q, (0, pad)).view(rows, -1, 32).amax(2).sum(1) * 32 * 2.0 ** -40
    cut_u = (coef.abs()[:, 0] * by_tile)[:, None] * v.abs().amax(0)
    pad = (-rows) % 32
    by_tile = torch.nn.functional.pad(size, (0, 0, 0, pad)).view(-1, 32, catalogue).amax(1).sum(0) * 32 * 2.0 ** -40
    cut_i = by_tile[:, None] * u.abs().amax(0)
    deep_i = E * (rows / 32 + 160)
    if u.shape[1] > 128:                                                         # a slice of the items is one chain of additions there, then the slices
        slices = max(1, min(16, catalogue // 2048))
        additions = catalogue / slices + slices + 32
    deep_u = E * (additions or 100)
    tol = TAU * TAU * ((n + 8) * E * float(np.log(n) + 1) + 4 * E * D) * torch.ones_like(loss)
    for name, x, want, bound in (("loss", alone, loss, tol), ("loss", got.loss, loss, tol), ("users", got.users, dz @ v, (eq + ep + deep_u) * (size @ v.abs()) + cut_u),
                                 ("items", got.items, dz.T @ u, (eq + ep + deep_i) * (size.T @ u.abs()) + cut_i), ("bias", got.bias, dz.sum(0), (eq + ep + deep_i) * size.sum(0) + by_tile)):
        off = (x.double() - want).abs() / (bound + 1e-38)
        assert float(off.max()) <= 1, (name, float(off.max()), int(off.argmax()))
    return got


SIZES = [(4129, 32_801, 20), (1030, 129_037, 64), (1000, 20_011, 96), (300, 60_007, 128), (29, 150_001, 60), (64, 200_003, 33), (5, 21_001, 128), (33, 9001, 20), (130, 3001, 50),
         (1, 5, 3), (257, 20_011, 130), (70, 5003, 300)]


@pytest.mark.parametrize("rows,items,factors", SIZES, ids=lambda x: str(x))
@pytest.mark.parametrize("masks", [None, "one", "rows"])
def test_every_tile_counts_once(rows, items, factors, masks):
    """one column tile per wavefront and two, few rows, long splits, the path without registers; with masks that leave whole tiles out"""
    if masks == "rows" and rows * items > 60_000_000:
        pytest.skip("masks of that size take too long to make")
    gen = torch.Generator(device="cuda").manual_seed(items)
    classes = factors - 1
    sign = lambda n: torch.randint(0, 2, (n,), generator=gen, device="cuda").float() * 2 - 1      # noqa: E731
    users, table = torch.zeros(rows, factors, device="cuda"), torch.zeros(items, factors, device="cuda")
    for t in (users, table):
        n = t.shape[0]
        if classes:
            t[torch.arange(n, device="cuda"), torch.arange(n, device="cuda") // 32 % classes] = 1.0
        t[:, factors - 1] = sign(n)
    bias = torch.randint(0, 2, (items,), generator=gen, device="cuda").float()
    ti = torch.randint(-1, items + 1, (rows, 8), generator=gen, device="cuda", dtype=torch.int32)
    if rows > 40:
        ti[37] = -1
    mask = which = None
    if masks == "one":
        mask = torch.rand(1, items, generator=gen, device="cuda") < 0.7
        mask[:, items // 3:items // 3 + 200] = False
    elif masks == "rows":
        mask = torch.rand(rows, items, generator=gen, device="cuda") < 0.7
        mask[rows // 2, items // 2:] = False
    check(users, table, bias, ti, torch.rand(rows, generator=gen, device="cuda") + 0.5, mask, which)


@pytest.mark.parametrize("factors,items", [(20, 6001), (64, 11_003), (128, 21_003), (200, 3001)])
@pytest.mark.parametrize("rows", [40, 300])
@pytest.mark.parametrize("nats", [12, 16, 20, 26])
@pytest.mark.parametrize("masked", [False, True], ids=["", "masked"])
def test_a_long_tail_behind_a_peak(factors, items, rows, nats, masked):
    """one item holds nearly all of a row's mass, is what the teacher says, and has no factors: the users' gradient is the tail's, thousands of items that are
    `nats` down each.  (A weight cut at 2^-32 of the peak's: 1.4e-3 at 16 nats, a tenth at 20)"""
    torch.manual_seed(factors)
    users, table = torch.zeros(rows, factors, device="cuda"), torch.zeros(items, factors, device="cuda")
    table[:, 0] = 1.0
    users[:, factors - 1] = 1.0
    bias = torch.full((items,), 0.4541, device="cuda")
    peak = 1234
    table[peak], bias[peak] = 0.0, 0.4541 + nats * 1.4427
    ti = torch.full((rows, 2), -1, dtype=torch.int32, device="cuda")
    ti[:, 1] = peak
    mask = torch.rand(1, items, device="cuda") < 0.8 if masked else None
    if masked:
        mask[0, peak] = True
    got = check(users, table, bias, ti, None, mask, additions=items / 32 + 160)
    # (the head's own share of that gradient is 0: nothing but the tail's is in it)
    assert (got.users[:, 0] > 0).all()


@pytest.mark.parametrize("factors", [20, 64, 128, 200])
@pytest.mark.parametrize("rows", [60, 1500])
@pytest.mark.parametrize("down", [8.3, 16.3])
@pytest.mark.parametrize("masked", [False, True], ids=["", "masked"])
def test_an_item_that_one_user_holds(factors, rows, down, masked):
    """an item's column: one user gives it all, the others 2^-19 and 2^-27 of that; in a factor that the one lacks the items' gradient is theirs"""
    torch.manual_seed(factors)
    items, special = 3001, 777
    if rows == 60:
        items = {20: 6001, 64: 11_003, 128: 21_003, 200: 3001}[factors]
    users, table = torch.zeros(rows, factors, device="cuda"), torch.zeros(items, factors, device="cuda")
    users[:, 0], users[:, 1] = -down, 1.0
    users[5, 0], users[5, 1] = 30.0, 0.0
    table[special, 0] = 1.0
    ti = torch.full((rows, 2), 50, dtype=torch.int32, device="cuda")
    ti[5] = special                                                              # (what the one user's teacher says: its dz is next to nothing)
    mask = torch.rand(1, items, device="cuda") < 0.8 if masked else None
    if masked:
        mask[0, [special, 50]] = True
    got = check(users, table, torch.zeros(items, device="cuda"), ti, None, mask, additions=items / 32 + 160)
    assert got.items[special, 1] > 0


@pytest.mark.parametrize("factors", [20, 64, 128, 200])
@pytest.mark.parametrize("rows,items", [(40, 21_003), (300, 901)])
def test_rows_with_nothing_to_learn_reach_nothing(factors, rows, items):
    """a batch of empty lists: all gradients are 0, whatever the table and the biases hold"""
    torch.manual_seed(factors)
    users, table, bias = torch.randn(rows, factors, device="cuda"), torch.randn(items, factors, device="cuda"), torch.randn(items, device="cuda")
    table[3, 1], table[40], bias[7], bias[8], bias[9] = NAN, INF, INF, NAN, -INF
    ti = torch.full((rows, 3), -1, dtype=torch.int32, device="cuda")
    got = distill_gradients(users, table, bias, ti, torch.zeros(rows, 3, device="cuda"), temperature=2.0)
    for x in got:
        assert (x == 0).all()
    # and one tile of such rows among others: theirs alone
    ti[:32, 0] = 11
    table[3, 1], table[40], bias[7], bias[8], bias[9] = 0.5, 0.25, 1.0, 2.0, 3.0
    both = distill_gradients(users, table, bias, ti, torch.zeros(rows, 3, device="cuda"), temperature=2.0)
    alone = distill_gradients(users[:32], table, bias, ti[:32].contiguous(), torch.zeros(32, 3, device="cuda"), temperature=2.0)
    assert (both.loss[32:] == 0).all() and (both.users[32:] == 0).all()
    for a, b in ((both.items, alone.items), (both.bias, alone.bias)):            # (32 terms of products within 1e-5: other splits, another order of sums)
        assert torch.allclose(a, b, rtol=0, atol=1e-4)


@pytest.mark.parametrize("factors", [20, 64, 128, 200])
@pytest.mark.parametrize("rows,items", [(40, 21_003), (300, 901)])
def test_the_largest_factors(factors, rows, items):
    """2^120 in a table whose scores are finite, and 2^80 in both where no score has them"""
    users, table = torch.zeros(rows, factors, device="cuda"), torch.zeros(items, factors, device="cuda")
    users[:, 0] = 2.0 ** 120
    table[::2, 0] = 1.0
    ti = torch.zeros(rows, 2, dtype=torch.int32, device="cuda")
    ti[:, 1] = 1                                                                 # half the teacher's mass on items that are 2^120 down
    t, bias = torch.zeros(rows, 2, device="cuda"), torch.zeros(items, device="cuda")
    want = TAU * TAU * 0.5 * 2.0 ** 120 / TAU
    for loss in (distill_loss(users, table, bias, ti, t, temperature=TAU), distill_gradients(users, table, bias, ti, t, temperature=TAU).loss):
        assert ((loss.double() - want).abs() <= 16 * E * want).all()
    users, table = torch.zeros_like(users), torch.zeros_like(table)
    users[:, 0], table[:, 1] = 2.0 ** 80, 2.0 ** 80
    got = distill_gradients(users, table, bias, ti, t, temperature=TAU)
    want = TAU * TAU * (np.log(items) - np.log(2))
    assert ((got.loss.double() - want).abs() <= 40 * E * (np.log(items) * TAU * TAU)).all()
    assert torch.isfinite(got.users).all() and torch.isfinite(got.items).all()


@pytest.mark.parametrize("factors", [8, 64, 128, 256])
@pytest.mark.parametrize("rows,items", [(40, 21_003), (300, 901)])
def test_factors_whose_second_parts_are_largest(factors, rows, items):
    """(1 + 2^-11) 2^j: what a product of two such factors loses (the product of their second parts, 2^-22 of it) has one sign in all of them.  Off by at most
    2^-21 of the sum of the products' sizes, which enters the loss once (the teacher's scores are float32 products), and the float32 roundings of
    the scores themselves"""
    gen = torch.Generator(device="cuda").manual_seed(factors)
    draw = lambda n: (1 + 2.0 ** -11) * 2.0 ** torch.randint(-1, 2, (n, factors), generator=gen, device="cuda").float() / factors ** 0.5      # noqa: E731
    users, table = draw(rows), draw(items)
    ti = torch.randint(0, items, (rows, 4), generator=gen, device="cuda", dtype=torch.int32)
    t, bias = torch.zeros(rows, 4, device="cuda"), torch.zeros(items, device="cuda")
    z = users.double() @ table.double().T / TAU
    lse = torch.logsumexp(z, 1)
    want = TAU * TAU * (-np.log(4) - z.gather(1, ti.long()).mean(1) + lse)
    s = float(z.max()) * TAU
    tol = TAU * TAU * (s * (2.0 ** -21 + 12 * E) + 24 * E * (float(lse.max()) + s) + 2 * factors ** 0.5 * E * s)
    for loss in (distill_loss(users, table, bias, ti, t, temperature=TAU), distill_gradients(users, table, bias, ti, t, temperature=TAU).loss):
        assert float((loss.double() - want).abs().max()) <= tol


@pytest.mark.parametrize("factors", [20, 64, 128, 200])
@pytest.mark.parametrize("rows,items", [(40, 21_003), (300, 901)])
def test_rows_of_very_different_weight_share_a_tile(factors, rows, items):
    """weights from 2^-12 to 2^12, both signs and 0, in every tile of 32 rows.  In the items' gradient a row's factors times its weight are cut at 2^-40 of the
    tile's largest such product: 2^-40 of that, times the row's share of the item, comes to a term's bound; the users' gradient and the loss are a
    row's own"""
    gen = torch.Generator(device="cuda").manual_seed(rows)
    users, table = torch.zeros(rows, factors, device="cuda"), torch.zeros(items, factors, device="cuda")
    users[torch.arange(rows), torch.arange(rows) % factors] = 1.0
    table[torch.arange(items), torch.arange(items) // 7 % factors] = 1.0
    weight = 2.0 ** (torch.arange(rows, device="cuda") % 25 - 12).float() * (1 + torch.rand(rows, generator=gen, device="cuda") / 2)
    weight[3::5] *= -1
    weight[4::9] = 0
    ti = torch.randint(0, items, (rows, 6), generator=gen, device="cuda", dtype=torch.int32)
    bias = torch.randint(0, 3, (items,), generator=gen, device="cuda").float()
    t = torch.zeros(rows, 6, device="cuda")
    z = (users.double() @ table.double().T + bias.double()) / TAU
    lse = torch.logsumexp(z, 1)
    q = torch.exp(z - lse[:, None])
    teacher = torch.zeros_like(q).scatter_add_(1, ti.long(), torch.full(ti.shape, 1 / 6, dtype=torch.float64, device="cuda"))
    coef = (TAU * weight.double())[:, None]
    dz, size = (q - teacher) * coef, (q + teacher) * coef.abs()
    D = float(2 * z.abs().max() + 2 * lse.max()) * 1.4427
    rel = E * (0.7 * 5 * D + 12 + 14)
    pad = (-rows) % 32
    largest = torch.nn.functional.pad(coef.abs()[:, 0], (0, pad)).view(-1, 32).amax(1).repeat_interleave(32)[:rows, None]       # (factors are 1 at most)
    cut = 2.0 ** -40 * ((q + teacher) * largest).sum(0)[:, None]
    by_tile = torch.nn.functional.pad(size, (0, 0, 0, pad)).view(-1, 32, items).amax(1).sum(0) * 32 * 2.0 ** -40
    got = distill_gradients(users, table, bias, ti, t, temperature=TAU, row_weight=weight)
    per_user = items / max(1, min(16, items // 2048)) + 48 if factors > 128 else items / 32 + 160
    per_item = rows / 32 + 160 if factors <= 128 else rows + 32
    for name, x, want, tol in (("users", got.users, dz @ table.double(), (rel + E * per_user) * (size @ table.double())),
                               ("items", got.items, dz.T @ users.double(), (rel + E * per_item) * (size.T @ users.double()) + cut + by_tile[:, None]),
                               ("bias", got.bias, dz.sum(0), (rel + E * per_item) * size.sum(0) + by_tile)):
        off = (x.double() - want).abs() / (tol + 1e-38)
        assert float(off.max()) <= 1, (name, float(off.max()))


@pytest.mark.parametrize("factors", [20, 64, 128, 200])
@pytest.mark.parametrize("rows,items", [(40, 21_003), (300, 901)])
def test_a_factor_that_counts_spoils_its_rows_alone(factors, rows, items):
    """even rows may have the first half of the catalogue, odd ones the second: a NaN in an item of the first half is in the even rows' losses and gradients, in
    all of the first half's items, and nowhere else"""
    torch.manual_seed(factors)
    half = items // 2
    users, table, bias = torch.randn(rows, factors, device="cuda") / 4, torch.randn(items, factors, device="cuda") / 4, torch.randn(items, device="cuda")
    mask = (torch.arange(items, device="cuda") < half)[None] ^ (torch.arange(rows, device="cuda") % 2 == 1)[:, None]
    ti = torch.randint(0, half, (rows, 4), device="cuda", dtype=torch.int32) + half * (torch.arange(rows, device="cuda") % 2)[:, None].int()
    t, kw = torch.randn(rows, 4, device="cuda"), dict(allowed=pack_allowed(mask), temperature=1.5)
    clean = distill_gradients(users, table, bias, ti, t, **kw)
    table[5, 2] = NAN
    got, alone = distill_gradients(users, table, bias, ti, t, **kw), distill_loss(users, table, bias, ti, t, **kw)
    assert torch.isnan(got.loss[::2]).all() and torch.isnan(alone[::2]).all() and torch.isnan(got.users[::2]).all()
    assert torch.isnan(got.items[:half]).all() and torch.isnan(got.bias[:half]).all()
    for a, b in ((got.loss[1::2], clean.loss[1::2]), (alone[1::2], clean.loss[1::2]), (got.users[1::2], clean.users[1::2]), (got.items[half:], clean.items[half:]), (got.bias[half:], clean.bias[half:])):
        assert torch.isfinite(a).all() and torch.allclose(a, b, rtol=1e-4, atol=1e-5)        # (a tile's scale is that of what is finite in it)


@pytest.mark.parametrize("factors", [20, 64, 128, 200])
@pytest.mark.parametrize("rows,items", [(40, 21_003), (300, 901), (4100, 33_000)])
@pytest.mark.parametrize("masked", [False, True], ids=["", "masked"])
def test_next_to_no_temperature(factors, rows, items, masked):
    """temperatures at which a step of float32 in a score is more than all of the softmax: q is 1 for the best item, which leads by at least 0.001 here (100 times
    the largest temperature, and a score is off by 2^-21 of the sum of its products' sizes, 10 at most), and the gradients are plain differences of rows"""
    if rows * items > 30_000_000 and (factors not in (20, 64) or masked):
        pytest.skip("two column tiles per wavefront: up to 64 factors, without masks")
    torch.manual_seed(rows + factors)
    users, table = torch.zeros(rows, factors, device="cuda"), torch.rand(items, factors, device="cuda") / 2
    best = torch.randint(0, items, (rows,), device="cuda")
    users[torch.arange(rows), torch.arange(rows) % factors] = torch.rand(rows, device="cuda") * 7 + 1
    table[best, torch.arange(rows, device="cuda") % factors] = 1.0                # (several of these lead where rows share a factor: the bias decides)
    bias = torch.rand(items, device="cuda") * 0.3
    ti = torch.randint(0, items, (rows, 3), device="cuda", dtype=torch.int32)
    mask = torch.rand(1, items, device="cuda") < 0.7 if masked else None
    z = users.double() @ table.double().T + bias.double()
    usable = torch.ones_like(ti, dtype=torch.bool)
    if masked:
        z = torch.where(mask, z, -INF)
        usable = mask.expand(rows, -1).gather(1, ti.long())
    top2 = z.topk(2, dim=1).values
    clear = (top2[:, 0] - top2[:, 1] > 1e-3) & usable.any(1)
    ti[~clear] = -1                                                              # (rows without a clear best have nothing to learn)
    usable &= clear[:, None]
    t = torch.zeros(rows, 3, device="cuda")
    p = usable.double() / usable.sum(1, keepdim=True).clamp(min=1)
    dz = torch.zeros_like(z).scatter_(1, z.argmax(1, keepdim=True), clear[:, None].double()).scatter_add_(1, ti.long().clamp(min=0), -p)
    size = dz.abs()
    for tau in (1e-5, 3e-6, 1e-6, 3e-7, 1e-7, 3e-8, 1e-9, 1e-12, 1e-20):
        kw = dict(temperature=tau, allowed=None if mask is None else pack_allowed(mask))
        got, alone = distill_gradients(users, table, bias, ti, t, **kw), distill_loss(users, table, bias, ti, t, **kw)
        for name, x, want, tol in (("users", got.users, dz @ table.double(), size @ table.double()), ("items", got.items, dz.T @ users.double(), size.T @ users.double()),
                                   ("bias", got.bias, dz.sum(0), size.sum(0))):
            off = (x.double() / tau - want).abs() / (1e-4 * tol + 1e-30)
            assert float(off.max()) <= 1, (name, tau, float(off.max()))
        want = tau * (top2[:, 0] - (torch.where(usable, z.gather(1, ti.long().clamp(min=0)), 0.0) * p).sum(1)) * clear
        for loss in (got.loss, alone):
            assert ((loss.double() - want).abs() <= 1e-4 * tau * 10).all(), tau
