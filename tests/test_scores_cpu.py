"""Refusals and host logic of the catalogue-score operators (rules, top scores, distillation): no GPU."""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from conftest import ROOT

import rankfm_amd
from rankfm_amd import ScoreRules, _build, _hip, pack_allowed
from rankfm_amd.scores import _check_scores, _rules_struct
from rankfm_amd.distill import _factor_rows

CPU = torch.device("cpu")


@pytest.fixture(scope="module")
def lib():
    _build.build()
    return _hip.lib()


def test_struct_layouts_match_the_header(tmp_path):
    structs = {"rfm_score_rules": _hip.ScoreRulesStruct, "rfm_distill_args": _hip.DistillArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "rankfm_hip.h"', 'int main(void){']
    for cname, ct in structs.items():
        lines.append('printf("%s %%zu\\n", sizeof(%s));' % (cname, cname))
        for f, _ in ct._fields_:
            lines.append('printf("%s.%s %%zu\\n", offsetof(%s, %s));' % (cname, f, cname, f))
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    got = dict(l.split() for l in subprocess.check_output([str(exe)], text=True).splitlines())
    for cname, ct in structs.items():
        assert int(got[cname]) == C.sizeof(ct), cname
        for f, _ in ct._fields_:
            assert int(got["%s.%s" % (cname, f)]) == getattr(ct, f).offset, (cname, f)


def test_the_package_still_imports_without_pytorch():
    code = "import sys; sys.modules['torch'] = None; import rankfm_amd; assert rankfm_amd.RankFM"
    subprocess.check_call([sys.executable, "-c", code], cwd=ROOT)
    with pytest.raises(AttributeError):
        rankfm_amd.no_such_name


def test_pack_allowed_is_one_bit_per_item():
    rng = np.random.default_rng(3)
    for items in (1, 31, 32, 33, 64, 100):
        mask = torch.from_numpy(rng.random((5, items)) < 0.5)
        words = pack_allowed(mask).numpy().astype(np.int64) & 0xffffffff
        assert words.shape == (5, (items + 31) // 32)
        back = (words[:, np.arange(items) // 32] >> (np.arange(items) % 32)) & 1
        assert np.array_equal(back.astype(bool), mask.numpy())
    for bad in (torch.zeros(4, dtype=torch.bool), torch.zeros(2, 4), np.zeros((2, 4), bool)):
        with pytest.raises(ValueError):
            pack_allowed(bad)


def _lists(n, k=3):
    return torch.arange(n + 1, dtype=torch.int64) * k, torch.zeros(n * k, dtype=torch.int32)


def test_good_rules_fill_the_struct():
    offsets, ids = _lists(4)
    u = _rules_struct(ScoreRules(history=(offsets, ids), repetition=torch.ones(4), frequency=0.5, item_bias=torch.zeros(40),
                                 row_bias=(offsets, ids, torch.zeros(12)), allowed=torch.zeros(1, 2, dtype=torch.int32)), 4, 40, CPU)
    assert u.n_history == 4 and u.n_history_items == 12 and u.frequency_all == 0.5 and u.presence_all == 0.0 and u.repetition
    assert not u.frequency and u.n_allowed == 1 and u.n_bias_items == 12
    assert not ScoreRules().penalises() and ScoreRules(presence=0.1).penalises() and ScoreRules(repetition=torch.ones(3)).penalises()


@pytest.mark.parametrize("rules", [
    dict(presence=1.0),                                                                     # penalties without a history
    dict(history_rows=torch.zeros(4, dtype=torch.int32)),
    dict(history=_lists(3)),                                                                # neither a list per row nor rows
    dict(history=(torch.zeros(5), torch.zeros(2, dtype=torch.int32))),                      # float offsets
    dict(history=(torch.zeros(0, dtype=torch.int64), torch.zeros(2, dtype=torch.int32)), history_rows=torch.zeros(4, dtype=torch.int32)),
    dict(history=_lists(4), history_rows=torch.zeros(3, dtype=torch.int32)),
    dict(history=_lists(4), history_rows=torch.zeros(4, dtype=torch.int64)),
    dict(history=_lists(4), repetition=0.0), dict(history=_lists(4), repetition=-1.0), dict(history=_lists(4), repetition=float("nan")),
    dict(history=_lists(4), frequency=float("inf")), dict(history=_lists(4), presence=torch.zeros(3)),
    dict(history=_lists(4), frequency=torch.zeros(4, dtype=torch.float64)),
    dict(item_bias=torch.zeros(39)), dict(item_bias=torch.zeros(40, dtype=torch.float16)), dict(item_bias=np.zeros(40, np.float32)),
    dict(item_bias=torch.zeros(80)[::2]),                                                   # not contiguous
    dict(row_bias=(torch.zeros(4, dtype=torch.int64), torch.zeros(2, dtype=torch.int32), torch.zeros(2))),
    dict(row_bias=(torch.zeros(5, dtype=torch.int64), torch.zeros(2, dtype=torch.int32), torch.zeros(3))),
    dict(allowed=torch.zeros(4, 1, dtype=torch.int32)), dict(allowed=torch.zeros(3, 2, dtype=torch.int32)),
    dict(allowed=torch.zeros(0, 2, dtype=torch.int32), allowed_rows=torch.zeros(4, dtype=torch.int32)),
    dict(allowed=torch.zeros(4, 2, dtype=torch.int64)), dict(allowed_rows=torch.zeros(4, dtype=torch.int32)),
    dict(allowed=torch.zeros(3, 2, dtype=torch.int32), allowed_rows=torch.zeros(4)),
])
def test_bad_rules_are_refused(rules):
    with pytest.raises(ValueError):
        _rules_struct(ScoreRules(**rules), 4, 40, CPU)


def test_bad_rows_are_refused():
    for bad in (torch.zeros(4), torch.zeros(2, 3, dtype=torch.float64), torch.zeros(2, 0), torch.zeros(4, 6).t(), torch.zeros(2, 6)[:, ::2],
                torch.zeros(1, 5).expand(3, 5), np.zeros((2, 3), np.float32)):
        with pytest.raises(ValueError):
            _check_scores(bad)
    with pytest.raises(ValueError):
        _rules_struct({"presence": 1.0}, 4, 40, CPU)
    for bad in (torch.zeros(4), torch.zeros(4, 3, dtype=torch.float16), torch.zeros(3, 4).t(), torch.zeros(2, 1025), torch.zeros(2, 0),
                torch.zeros(1, 5).expand(3, 5)):
        with pytest.raises(ValueError):
            _factor_rows(bad, "users")


def test_without_a_gpu_the_calls_say_so():
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    with pytest.raises(_hip.EngineUnavailable):
        rankfm_amd.adjust_scores(torch.zeros(2, 3), ScoreRules())
    with pytest.raises(_hip.EngineUnavailable):
        rankfm_amd.top_scores(torch.zeros(2, 3), 1)
    with pytest.raises(_hip.EngineUnavailable):
        rankfm_amd.distill_loss(torch.zeros(2, 3), torch.zeros(4, 3), None, torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, 1))


def test_the_c_entries_refuse_bad_arguments(lib):
    u = _hip.ScoreRulesStruct(repetition_all=1.0)
    one = C.c_void_p(64)                                            # (a pointer that nothing follows: the calls below are refused first)
    adjust = lambda r=u, t=_hip.F32, rows=2, items=8, i=one, si=8, o=one, so=8: lib.rfm_adjust_scores_device(C.byref(r) if r else None, t, rows, items, i, si, o, so, None)   # noqa: E731
    assert adjust(rows=0) == _hip.OK
    for kw in (dict(r=None), dict(t=3), dict(t=-1), dict(rows=-1), dict(items=0), dict(si=7), dict(so=7), dict(i=None), dict(o=None)):
        assert adjust(**kw) == _hip.ERR_BAD_ARG, kw
    for bad in (dict(history_offsets=64, n_history=1, history_items=64, n_history_items=2), dict(history_offsets=64, n_history=-1),
                dict(history_offsets=64, n_history=2, n_history_items=3), dict(history_offsets=64, n_history=2, repetition_all=0.0),
                dict(bias_offsets=64, n_bias_items=2), dict(allowed=64), dict(allowed=64, n_allowed=0), dict(history_offsets=64, n_history=2, frequency_all=float("nan"))):
        r = _hip.ScoreRulesStruct(**dict(dict(repetition_all=1.0), **bad))
        assert adjust(r=r) == _hip.ERR_BAD_ARG, bad
    top = lambda rows=2, items=8, n=3, s=one, ws=one, b=1 << 20, o=one: lib.rfm_top_scores_device(None, _hip.F32, rows, items, s, 8, n, o, one, ws, b, None)   # noqa: E731
    for kw in (dict(n=0), dict(n=9), dict(items=0), dict(rows=-1), dict(s=None), dict(o=None)):
        assert top(**kw) == _hip.ERR_BAD_ARG, kw
    assert top(ws=None) == _hip.ERR_WORKSPACE and top(b=0) == _hip.ERR_WORKSPACE and top(rows=0) == _hip.OK
    assert lib.rfm_top_scores_workspace_bytes(1, 8, 9) == 0 and lib.rfm_top_scores_workspace_bytes(1, 200_000, 100) > 0

    def args(**kw):
        base = dict(n_rows=2, n_items=8, n_factors=4, n_teacher=2, temperature=1.0, users=64, items=64, user_stride=4, item_stride=4, teacher_items=64,
                    teacher_scores=64, loss=64)
        return _hip.DistillArgs(**dict(base, **kw))
    assert lib.rfm_distill_workspace_bytes(C.byref(args())) > 0
    for kw, rc in ((dict(n_rows=-1), -1), (dict(n_items=0), -1), (dict(n_factors=0), -1), (dict(n_teacher=0), -1), (dict(temperature=0.0), -1),
                   (dict(temperature=float("nan")), -1), (dict(temperature=float("inf")), -1), (dict(user_stride=3), -1), (dict(item_stride=3), -1), (dict(d_users=64), -1),
                   (dict(d_items=64), -1), (dict(d_bias=64), -1), (dict(allowed=64, n_allowed=0), -1), (dict(users=None), -1), (dict(loss=None), -1),
                   (dict(n_factors=1025, user_stride=1025, item_stride=1025), -5), (dict(n_teacher=1025), -5)):
        a = args(**kw)
        assert lib.rfm_distill_device(C.byref(a), one, 1 << 40, None) == rc, kw
    assert lib.rfm_distill_device(C.byref(args()), None, 1 << 40, None) == _hip.ERR_WORKSPACE
    assert lib.rfm_distill_device(C.byref(args()), one, 8, None) == _hip.ERR_WORKSPACE
    assert lib.rfm_distill_device(None, one, 8, None) == _hip.ERR_BAD_ARG and lib.rfm_distill_workspace_bytes(None) == 0
    mv = _hip.ModelView()
    assert lib.rfm_scores_workspace_bytes(C.byref(mv), 3) == 0 and lib.rfm_effective_factors(C.byref(mv)) == 0
    assert lib.rfm_scores_device(C.byref(mv), 1, one, one, one, 1 << 30, None) == _hip.ERR_BAD_ARG
    assert lib.rfm_effective_factors_device(C.byref(mv), 1, one, one, one, one, None) == _hip.ERR_BAD_ARG


def test_sizes_that_distillation_does_not_take(lib):
    base = dict(n_rows=2, n_items=8, n_factors=4, n_teacher=2, temperature=1.0, users=64, items=64, user_stride=4, item_stride=4, teacher_items=64, teacher_scores=64,
                loss=64, d_users=64, d_items=64)
    for kw in (dict(n_items=(1 << 25) + 1), dict(n_rows=(1 << 24) + 1), dict(n_factors=1025, user_stride=1025, item_stride=1025), dict(n_teacher=1025)):
        a = _hip.DistillArgs(**dict(base, **kw))
        assert lib.rfm_distill_workspace_bytes(C.byref(a)) == 0
        assert lib.rfm_distill_device(C.byref(a), C.c_void_p(64), 1 << 60, None) == -5, kw
    for kw in (dict(n_items=1 << 25), dict(n_rows=1 << 24), dict(n_factors=1024, user_stride=1024, item_stride=1024), dict(n_teacher=1024)):
        assert lib.rfm_distill_workspace_bytes(C.byref(_hip.DistillArgs(**dict(base, **kw)))) > 0, kw
