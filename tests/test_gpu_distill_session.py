"""The operators as they are used together, on resident sessions: a teacher's score rows, its answers under rules, and a student that learns from them.
Scores are checked against `predict` (the existing per-pair kernel; summation order differs: 2^-24 per addition of the terms' sizes), everything
behind them against float64."""
import numpy as np
import pytest
import torch

from rankfm_amd import ScoreRules, pack_allowed, synthetic
from rankfm_amd.engine import WEIGHT_NAMES, DeviceSession

pytestmark = pytest.mark.gpu
E = 2.0 ** -24


def session(U=60, I=130, F=12, P=0, Q=0, seed=0, **kw):
    rng = np.random.default_rng(seed)
    pairs, csr = synthetic.make_interactions(U, I, 900, seed=5)
    x_uf = (rng.random((U, P)) < 0.4).astype(np.float32) if P else np.zeros((U, 1), np.float32)
    x_if = (rng.random((I, Q)) < 0.4).astype(np.float32) if Q else np.zeros((I, 1), np.float32)
    w = dict(w_i=rng.standard_normal(I) * 0.3, w_if=rng.standard_normal(max(Q, 1)) * (Q > 0), v_u=rng.standard_normal((U, F)) * 0.4, v_i=rng.standard_normal((I, F)) * 0.4,
             v_uf=rng.standard_normal((max(P, 1), F)) * 0.2 * (P > 0), v_if=rng.standard_normal((max(Q, 1), F)) * 0.2 * (Q > 0))
    w = {k: np.ascontiguousarray(v, dtype=np.float32) for k, v in w.items()}
    return DeviceSession(pairs, np.ones(len(pairs), np.float32), csr.offsets, csr.items, x_uf, x_if, w, **kw), csr


def effective(s):
    """the scores' two tables and bias in float64"""
    w = {k: v.astype(np.float64) for k, v in s.weights_to_host().items()}
    x_uf, x_if = s.x_uf.cpu().numpy().astype(np.float64), s.x_if.cpu().numpy().astype(np.float64)
    u, v, b = w["v_u"], w["v_i"], w["w_i"]
    if s.has_uf:
        u = u + x_uf @ w["v_uf"]
    if s.has_if:
        u, v, b = np.hstack([u, w["v_u"]]), np.hstack([v, x_if @ w["v_if"]]), b + x_if @ w["w_if"]
    return u, v, b, x_uf, x_if


@pytest.mark.parametrize("P, Q", [(0, 0), (3, 0), (0, 4), (3, 4)])
def test_score_rows_are_predictions(P, Q):
    s, _ = session(P=P, Q=Q, seed=P + Q)
    users = np.array([3, 0, np.nan, 59, 3, 60, -1], dtype=np.float32)              # 60 and -1 are nobody
    rows = s.scores(users).cpu().numpy()
    assert np.isnan(rows[[2, 5, 6]]).all()
    for r in (0, 1, 3, 4):
        pairs = np.stack([np.full(130, users[r]), np.arange(130)], 1).astype(np.float32)
        u, v, b, *_ = effective(s)
        size = np.abs(u[int(users[r])]) @ np.abs(v).T + np.abs(b)
        assert (np.abs(rows[r] - s.predict(pairs)) <= 80 * E * size).all()
    assert s.scores(np.zeros(0, np.float32)).shape == (0, 130)


def test_answers_under_rules_and_what_they_were_scored():
    s, csr = session(seed=2)
    users = np.array([5, np.nan, 0, 41, 17], dtype=np.float32)
    rows = s.scores(users).cpu().numpy()
    masks = np.random.default_rng(0).random((2, 130)) < 0.6
    bias = np.linspace(-1, 1, 130).astype(np.float32)
    rules = ScoreRules(repetition=1.5, frequency=0.25, item_bias=torch.from_numpy(bias).cuda(), allowed=pack_allowed(torch.from_numpy(masks).cuda()),
                       allowed_rows=torch.tensor([0, 0, -1, 1, 1], dtype=torch.int32).cuda())
    want = rows.copy()
    for r, u in enumerate(users):
        if np.isnan(u):
            continue
        c = np.bincount(csr[int(u)], minlength=130).astype(np.float32)
        x = np.where(rows[r] > 0, rows[r] / np.float32(1.5), rows[r] * np.float32(1.5)) - np.float32(0.25) * c
        want[r] = np.where(c > 0, x, rows[r]) + bias
        m = [0, 0, -1, 1, 1][r]
        if m >= 0:
            want[r] = np.where(masks[m], want[r], -np.inf)
    for previous in (False, True):
        best = s.top_scores(users, 12, rules, filter_previous=previous)
        w = want.copy()
        if previous:
            for r, u in enumerate(users):
                if not np.isnan(u):
                    w[r, csr[int(u)]] = -np.inf
        for r in range(5):
            order = np.argsort(-w[r].astype(np.float64), kind="stable")[:12] if r != 1 else np.full(12, -1)
            assert best.items[r].tolist() == order.tolist(), (r, previous)
            if r != 1:
                assert np.array_equal(best.scores[r].cpu().numpy(), w[r, order])
        rec = s.recommend(users, 12, filter_previous=previous, rules=rules)
        assert rec.dtype == np.float32 and np.isnan(rec[1]).all() and np.array_equal(rec[0].astype(np.int64), best.items[0].cpu().numpy())
    s.SCORE_BYTES = 4 * 130 * 2                                                   # two rows at a time: the same answers
    again = s.top_scores(users, 12, rules, filter_previous=True)
    assert torch.equal(again.items, best.items) and torch.equal(again.scores, best.scores)
    plain = s.recommend(users, 12, filter_previous=True)                          # what ran before: equal where no two scores are
    assert np.array_equal(plain, s.recommend(users, 12, filter_previous=True, rules=ScoreRules()), equal_nan=True)
    with pytest.raises(ValueError):
        s.top_scores(users, 0)
    with pytest.raises(ValueError):
        s.top_scores(users, 131, rules)


@pytest.mark.parametrize("P, Q", [(0, 0), (3, 0), (0, 4), (3, 4)])
def test_a_student_learns_from_a_teacher(P, Q):
    """gradients by weight against float64 (and, through the chain rule, against differences of the float64 loss), and the step that they make"""
    teacher, _ = session(F=24, seed=11)
    student, _ = session(F=10, P=P, Q=Q, seed=12, keep_layout=True)
    student.run(1)                                                                # the engine's layout is in the workspace when the step comes
    users = np.array([7, 2, 33, 0, 58, 19])
    answers = teacher.top_scores(users.astype(np.float32), 9, ScoreRules(presence=0.5), filter_previous=True)
    weight = torch.rand(6).cuda() + 0.5
    before = student.weights_to_host()
    ti, t, g, tau = answers.items.cpu().numpy(), answers.scores.cpu().numpy().astype(np.float64), weight.cpu().numpy().astype(np.float64), 1.7

    def total(w):
        x_uf, x_if = student.x_uf.cpu().numpy().astype(np.float64)[users], student.x_if.cpu().numpy().astype(np.float64)
        z = w["w_i"] + x_if @ w["w_if"] + (w["v_u"][users] + x_uf @ w["v_uf"]) @ w["v_i"].T + w["v_u"][users] @ (x_if @ w["v_if"]).T
        loss = []
        for r in range(6):
            use = ti[r] >= 0
            lp = t[r, use] / tau
            lp = lp - lp.max() - np.log(np.exp(lp - lp.max()).sum())
            lq = z[r] / tau
            lq = lq - lq.max() - np.log(np.exp(lq - lq.max()).sum())
            loss.append(tau * tau * (np.exp(lp) * (lp - lq[ti[r, use]])).sum())
        return np.array(loss)

    w64 = {k: v.astype(np.float64) for k, v in before.items()}
    loss, grad = student.distill(users, answers.items, answers.scores, temperature=tau, row_weight=weight, learning_rate=0.1)
    assert set(grad) == {"w_i", "v_u", "v_i"} | ({"w_if", "v_if"} if Q else set()) | ({"v_uf"} if P else set())
    assert (np.abs(loss.cpu().numpy() - total(w64)) <= 1e-5 * (1 + np.abs(total(w64)))).all()      # some 100 roundings of values below 10
    rng, h = np.random.default_rng(0), 1e-4
    for name, got in grad.items():
        got = got.cpu().numpy().astype(np.float64)
        d = rng.standard_normal(got.shape)
        full = np.zeros_like(w64[name])
        if name == "v_u":
            full[users] = d
        else:
            full = d
        slope = float((g * (total(dict(w64, **{name: w64[name] + h * full})) - total(dict(w64, **{name: w64[name] - h * full})))).sum()) / (2 * h)
        assert abs(slope - (got * d).sum()) <= 2e-5 * np.abs(got * d).sum(), name
    after = student.weights_to_host()
    for name in WEIGHT_NAMES:
        want = w64[name].copy()
        if name in grad:
            step = 0.1 * grad[name].cpu().numpy().astype(np.float64)
            if name == "v_u":
                want[users] -= step
            else:
                want -= step
        assert (np.abs(after[name] - want) <= 2 * E * (np.abs(want) + np.abs(w64[name])) + 1e-12).all(), name
    student.run(1)                                                                # and training goes on from there
    for bad in (dict(users=[1, 1, 2, 3, 4, 5]), dict(users=[1, 2, 3, 4, 5, 60]), dict(users=[0.5, 1, 2, 3, 4, 5]), dict(users=[np.nan, 1, 2, 3, 4, 5]), dict(learning_rate=0.0)):
        kw = dict(dict(users=users, learning_rate=None), **bad)
        with pytest.raises(ValueError):
            student.distill(np.array(kw["users"]), answers.items, answers.scores, learning_rate=kw["learning_rate"])


def test_rules_of_other_rows_than_the_users_are_refused():
    s, _ = session(seed=4)
    users = np.arange(5, dtype=np.float32)
    masks = pack_allowed(torch.ones((6, 130), dtype=torch.bool).cuda())
    for rules in (ScoreRules(allowed=masks), ScoreRules(allowed=masks, allowed_rows=torch.zeros(6, dtype=torch.int32).cuda()), ScoreRules(presence=torch.ones(6).cuda()),
                  ScoreRules(row_bias=(torch.zeros(7, dtype=torch.int64).cuda(), torch.zeros(0, dtype=torch.int32).cuda(), torch.zeros(0).cuda())),
                  ScoreRules(item_bias=torch.zeros(131).cuda()), "none"):
        with pytest.raises(ValueError):
            s.top_scores(users, 3, rules)
        with pytest.raises(ValueError):
            s.recommend(users, 3, rules=rules)
