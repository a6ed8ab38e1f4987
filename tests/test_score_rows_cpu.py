"""Where score rows lie, and what a call says of tensors that it cannot take: no GPU."""
import ctypes as C
import itertools
import warnings

import pytest
import torch

import rankfm_amd
from rankfm_amd import ScoreRules, _build, _hip
from rankfm_amd.scores import _overlap


def test_overlap_is_that_of_the_elements():
    """every pair of row layouts in a small store, against the sets of their elements"""
    store = torch.zeros(40)
    layouts = [(first, stride) for first in range(0, 14) for stride in (3, 5, 7, 8)]
    for rows, items in itertools.product((1, 2, 3), (1, 2, 3)):
        views = [torch.as_strided(store, (rows, items), (stride, 1), first) for first, stride in layouts if first + (rows - 1) * stride + items <= 40]
        cells = [set((v.storage_offset() + v.stride(0) * r + k) for r in range(rows) for k in range(items)) for v in views]
        for (x, a), (y, b) in itertools.product(zip(views, cells), repeat=2):
            if a & b:
                assert _overlap(x, y)
            elif x.stride(0) == y.stride(0) or max(a) < min(b) or max(b) < min(a):
                assert not _overlap(x, y)


def test_halves_of_wider_rows_do_not_overlap():
    wide = torch.zeros(4, 10, dtype=torch.bfloat16)
    assert not _overlap(wide[:, :5], wide[:, 5:]) and not _overlap(wide[:, 6:], wide[:, :4])
    assert _overlap(wide[:, :6], wide[:, 4:]) and _overlap(wide[:3], wide[1:])


def test_calls_that_cut_the_graph_say_so():
    """before anything else is looked at: here the calls end for want of a GPU, with the warning given"""
    scores, ti = torch.zeros(2, 3, requires_grad=True), torch.zeros(2, 1, dtype=torch.int32)
    calls = [lambda s: rankfm_amd.adjust_scores(s, ScoreRules()), lambda s: rankfm_amd.top_scores(s, 1), lambda s: rankfm_amd.distill_loss(s, torch.zeros(4, 3), None, ti, torch.zeros(2, 1)),
             lambda s: rankfm_amd.distill_loss(torch.zeros(2, 3), torch.zeros(4, 3), None, ti, s[:, :1].contiguous())]
    for call in calls:
        with pytest.warns(UserWarning, match="not recorded by autograd"), pytest.raises((_hip.EngineUnavailable, ValueError)):
            call(scores)
        for quiet in (scores.detach(), scores):
            with warnings.catch_warnings(), torch.set_grad_enabled(quiet is not scores), pytest.raises((_hip.EngineUnavailable, ValueError)):
                warnings.simplefilter("error")
                call(quiet)


def test_temperatures_without_an_inverse_are_refused():
    _build.build()
    lib = _hip.lib()

    def args(t):
        return _hip.DistillArgs(n_rows=2, n_items=8, n_factors=4, n_teacher=2, temperature=t, users=64, items=64, user_stride=4, item_stride=4, teacher_items=64, teacher_scores=64, loss=64)
    for t in (0.0, 1e-39, 2.0 ** -127, -1.0, float("nan"), float("inf")):
        assert lib.rfm_distill_workspace_bytes(C.byref(args(t))) == 0
        assert lib.rfm_distill_device(C.byref(args(t)), C.c_void_p(64), 1 << 40, None) == _hip.ERR_BAD_ARG, t
    for t in (2.0 ** -126, 1e-20, 1.0, 3e38):
        assert lib.rfm_distill_workspace_bytes(C.byref(args(t))) > 0
