"""Score rows that lie in wider ones, and what autograd is told, on the device."""
import numpy as np
import pytest
import torch

from rankfm_amd import ScoreRules, adjust_scores, distill_gradients, top_scores

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def rules(rows, items, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    offsets = torch.arange(rows + 1, device="cuda") * 5
    listed = torch.randint(-1, items + 1, (rows * 5,), generator=gen, device="cuda", dtype=torch.int32)
    return ScoreRules(history=(offsets, listed), frequency=0.25, presence=0.5, item_bias=torch.randn(items, generator=gen, device="cuda"))


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_halves_of_wider_rows(dtype):
    for rows, items in ((1, 7), (9, 1001), (3, 4096), (5, 6001)):
        r = rules(rows, items)
        wide = torch.randn(rows, 2 * items, device="cuda").to(dtype)
        kept = wide[:, :items].clone()
        want = adjust_scores(kept, r)
        got = adjust_scores(wide[:, :items], r, out=wide[:, items:])
        assert got.data_ptr() == wide[:, items:].data_ptr() and torch.equal(got, want) and torch.equal(wide[:, :items], kept)
        with pytest.raises(ValueError):
            adjust_scores(wide[:, :items], r, out=wide[:, 1:items + 1])
    row = torch.randn(1, 4096, device="cuda").to(dtype)                          # one row, the stride of which means nothing
    want = adjust_scores(row.clone(), rules(1, 4096))
    assert torch.equal(adjust_scores(row, rules(1, 4096), out=torch.as_strided(row, (1, 4096), (9999, 1))), want) and torch.equal(row, want)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_strided_rows_are_adjusted_as_contiguous_ones(dtype):
    """bit for bit, at every alignment; contiguous rows are held to the definition elsewhere"""
    for rows, items in ((9, 1001), (4, 2049)):
        r, s = rules(rows, items), torch.randn(rows, items, device="cuda").to(dtype)
        want, top = adjust_scores(s, r), top_scores(s, 12, r)
        for start in (0, 1, 2, 3, 7, 98):
            wide = torch.full((rows, items + 99), 7.0, dtype=dtype, device="cuda")
            wide[:, start:start + items] = s
            out = torch.full((rows, items + 50), 3.0, dtype=dtype, device="cuda")
            got = adjust_scores(wide[:, start:start + items], r, out=out[:, 2:items + 2])
            assert torch.equal(got, want) and (out[:, :2] == 3).all() and (out[:, items + 2:] == 3).all()
            again = top_scores(wide[:, start:start + items], 12, r)
            assert torch.equal(again.items, top.items) and torch.equal(again.scores, top.scores)
        assert torch.equal(adjust_scores(s.float(), r).to(dtype), want)          # (one rounding, at the end)


def test_autograd_hears_of_a_row_that_changed():
    x = torch.randn(3, 50, device="cuda", requires_grad=True)
    y = x.exp()                                                                  # (keeps its result for the backward pass)
    with torch.no_grad():
        adjust_scores(y, ScoreRules(item_bias=torch.ones(50, device="cuda")), out=y)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.inference_mode():
        z = torch.randn(3, 50, device="cuda")
        adjust_scores(z, ScoreRules(item_bias=torch.ones(50, device="cuda")), out=z)


def test_calls_that_cut_the_graph_say_so():
    x = torch.randn(3, 50, device="cuda", requires_grad=True)
    with pytest.warns(UserWarning, match="not recorded by autograd"):
        assert not adjust_scores(x, ScoreRules()).requires_grad
    u, ti = torch.randn(4, 8, device="cuda", requires_grad=True), torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    got = distill_gradients(u, torch.randn(20, 8, device="cuda"), None, ti, torch.zeros(4, 2, device="cuda"))     # (what it is for: no warning)
    assert not got.users.requires_grad and np.isfinite(got.users.cpu().numpy()).all()


@pytest.mark.parametrize("entries", [20, 3000], ids=["few", "many"])
def test_ids_of_any_32_bits(entries):
    """the smallest and largest ids among those of the catalogue: skipped, on every path that looks at lists"""
    gen = torch.Generator(device="cuda").manual_seed(entries)
    for items in (700, 9001):
        good = torch.randint(0, items, (entries,), generator=gen, device="cuda", dtype=torch.int32)
        edges = torch.tensor([-2 ** 31, 2 ** 31 - 1, -2 ** 31 + items - 1, -2 ** 31 + 4095, -1, items], dtype=torch.int64).int().cuda()
        wild = torch.cat([edges, good, edges])
        scores, value = torch.randn(1, items, device="cuda"), torch.randn(entries + 12, generator=gen, device="cuda")
        lists = lambda x: (torch.tensor([0, x.numel()], device="cuda"), x)       # noqa: E731
        a = ScoreRules(history=lists(good), presence=0.5, row_bias=(*lists(good), value[6:-6].contiguous()))
        b = ScoreRules(history=lists(wild), presence=0.5, row_bias=(*lists(wild), value))
        assert torch.equal(adjust_scores(scores, a), adjust_scores(scores, b))
        for x, y in zip(top_scores(scores, 30, a), top_scores(scores, 30, b)):
            assert torch.equal(x, y)
