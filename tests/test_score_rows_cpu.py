"""Where score rows lie, and what a call says of tensors that it cannot take: no GPU."""
import itertools

import pytest
import torch

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
