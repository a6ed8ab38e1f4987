"""Rows of catalogue scores on the device: rules applied to them (`adjust_scores`) and their best entries (`top_scores`).

The reference hands out ranked items only and knows one rule, `filter_previous` (rankfm/_rankfm.pyx:450-451).  Here the caller says what
else holds: penalties for what a user has already had, biases, and masks of what may be shown at all.  Tensors are torch tensors on one
MI355X; work is enqueued on that device's current stream and nothing synchronises, so the calls may be captured into a graph.  Nothing is
recorded by autograd: a call whose result looks differentiable and is not warns (UserWarning).
"""
import ctypes as C
import warnings
from dataclasses import dataclass
from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _hip

_DTYPES = {torch.float32: _hip.F32, torch.float16: _hip.F16, torch.bfloat16: _hip.BF16}


@dataclass
class ScoreRules:
    """what holds for the rows of a call; every field is optional, tensors live on the scores' device

    In this order, c being how often item i stands in the row's history and each operation rounded once in float32:

        c > 0:                   s = s / repetition if s > 0 else s * repetition;  s -= frequency * c;  s -= presence
        item_bias:               s += item_bias[i]
        row_bias names i:        s += the value of the last entry that does
        i is not allowed:        s = -inf, whatever it was

    history        (offsets int64 [H + 1], items int32): lists in any order, with repeats
    history_rows   int32 [rows], the list of each row (negative: none); without it row r has list r
    repetition, frequency, presence    a number for all rows or float32 [rows]; they need `history`
    item_bias      float32 [items]
    row_bias       (offsets int64 [rows + 1], items int32, values float32): the rows' own biases
    allowed        int32 [masks, ceil(items / 32)]: bit b of word w allows item 32 w + b (`pack_allowed` makes it)
    allowed_rows   int32 [rows], the mask of each row (negative: none); without it row r has mask r, or every row the only one

    Items outside the catalogue in a list are skipped.  A row that names a history or a mask behind the last one comes out NaN.
    """
    history: Optional[Tuple[torch.Tensor, torch.Tensor]] = None
    history_rows: Optional[torch.Tensor] = None
    repetition: Union[float, torch.Tensor] = 1.0
    frequency: Union[float, torch.Tensor] = 0.0
    presence: Union[float, torch.Tensor] = 0.0
    item_bias: Optional[torch.Tensor] = None
    row_bias: Optional[Tuple[torch.Tensor, torch.Tensor, torch.Tensor]] = None
    allowed: Optional[torch.Tensor] = None
    allowed_rows: Optional[torch.Tensor] = None

    def rows(self, begin, end):
        """the rules of rows begin .. end - 1 of a call"""
        def cut(v):
            return v[begin:end] if isinstance(v, torch.Tensor) else v
        per_row = self.allowed is not None and self.allowed_rows is None and self.allowed.shape[0] > 1
        history = self.history
        if history is not None and self.history_rows is None:
            history = (history[0][begin:end + 1], history[1])
        return ScoreRules(history, cut(self.history_rows), cut(self.repetition), cut(self.frequency), cut(self.presence), self.item_bias,
                          None if self.row_bias is None else (self.row_bias[0][begin:end + 1],) + tuple(self.row_bias[1:]),
                          cut(self.allowed) if per_row else self.allowed, cut(self.allowed_rows))

    def penalises(self):
        """whether the rules look at a history at all"""
        rho, phi, pi = self.repetition, self.frequency, self.presence
        return isinstance(rho, torch.Tensor) or isinstance(phi, torch.Tensor) or isinstance(pi, torch.Tensor) or not rho == 1.0 or not phi == 0.0 == pi


class TopScores(NamedTuple):
    """int32 / float32 [rows, n]: items by descending score and the scores; -1 and -inf behind the last ranking item"""
    items: torch.Tensor
    scores: torch.Tensor


def pack_allowed(mask):
    """bool [masks, items] -> int32 [masks, ceil(items / 32)], bit b of word w for item 32 w + b"""
    if not isinstance(mask, torch.Tensor) or mask.dtype != torch.bool or mask.dim() != 2:
        raise ValueError("[mask] must be a bool tensor [masks, items]")
    words = (mask.shape[1] + 31) // 32
    full = torch.zeros((mask.shape[0], words * 32), dtype=torch.bool, device=mask.device)
    full[:, :mask.shape[1]] = mask
    value = (full.view(mask.shape[0], words, 32).long() << torch.arange(32, device=mask.device)).sum(-1)
    return torch.where(value >= 2 ** 31, value - 2 ** 32, value).int()


def check_tensor(t, name, dtype, shape, device):
    """a contiguous tensor of this type and shape (None: any size) on this device, or ValueError"""
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.device == device and t.is_contiguous() and (
            t.shape == shape or None in shape and t.dim() == len(shape) and all(w is None or g == w for g, w in zip(t.shape, shape))):
        return t.data_ptr()
    if not isinstance(t, torch.Tensor):
        raise ValueError("[%s] must be a torch tensor" % name)
    if t.dtype != dtype:
        raise ValueError("[%s] must be %s, got %s" % (name, str(dtype).replace("torch.", ""), str(t.dtype).replace("torch.", "")))
    if t.device != device:
        raise ValueError("[%s] is on %s, the call on %s" % (name, t.device, device))
    if not t.is_contiguous():
        raise ValueError("[%s] must be contiguous" % name)
    raise ValueError("[%s] must have shape %s, got %s" % (name, list(shape), list(t.shape)))


def launch(device, entry, *args):
    """entry(*args, the device's current stream) with `device` the current one; the exception of its status if it refuses.  (A small call's time is the
    host's: no stream object is made, and no device switched that is the current one)"""
    stream = torch._C._cuda_getCurrentRawStream(device.index)
    if torch.cuda.current_device() == device.index:
        rc = entry(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = entry(*args, stream)
    if rc != _hip.OK:
        _hip.raise_for_status(rc)


def check_device(t, name):
    if t.device.type != "cuda":
        if not torch.cuda.is_available():
            raise _hip.EngineUnavailable("no MI355X visible to PyTorch-ROCm: rankfm_amd has no CPU fallback")
        raise ValueError("[%s] must be on the GPU" % name)
    return t.device


def warn_if_cut(call, *tensors):
    """UserWarning where autograd would have followed these tensors into a call's result"""
    if not torch.is_grad_enabled():
        return
    for t in tensors:
        if getattr(t, "requires_grad", False):
            warnings.warn("%s is not recorded by autograd: its result does not depend on tensors that require a gradient (detach them, or call it under "
                          "torch.no_grad())" % call, UserWarning, stacklevel=3)
            return


def _check_scores(scores):
    if not isinstance(scores, torch.Tensor) or scores.dtype not in _DTYPES or scores.dim() != 2:
        raise ValueError("[scores] must be a float32, float16 or bfloat16 tensor [rows, items]")
    rows, items = scores.shape
    if items < 1:
        raise ValueError("[scores] must have at least one item")
    if not scores.is_contiguous() and (items > 1 and scores.stride(1) != 1 or rows > 1 and scores.stride(0) < items):
        raise ValueError("[scores] must have rows of consecutive items that do not overlap")
    return check_device(scores, "scores")


def _row_stride(t):
    rows, items = t.shape
    return t.stride(0) if rows > 1 else items              # (the stride of a single row means nothing)


def _number_or_rows(u, name, value, rows, device):
    if isinstance(value, torch.Tensor):
        setattr(u, name, check_tensor(value, name, torch.float32, (rows,), device))
    else:
        value = float(value)
        if not (value > 0.0 if name == "repetition" else value == value) or value in (float("inf"), float("-inf")):
            raise ValueError("[%s] must be a finite number%s" % (name, " above 0" if name == "repetition" else ""))
        setattr(u, name + "_all", value)


def allowed_fields(u, allowed, allowed_rows, rows, items, device):
    """the mask fields of rfm_score_rules / rfm_distill_args"""
    if allowed is None:
        if allowed_rows is not None:
            raise ValueError("[allowed_rows] needs [allowed]")
        return
    u.allowed = check_tensor(allowed, "allowed", torch.int32, (None, (items + 31) // 32), device)
    u.n_allowed = allowed.shape[0]
    if u.n_allowed < 1:
        raise ValueError("[allowed] must hold at least one mask")
    if allowed_rows is not None:
        u.allowed_rows = check_tensor(allowed_rows, "allowed_rows", torch.int32, (rows,), device)
    elif u.n_allowed not in (1, rows):
        raise ValueError("[allowed] must hold one mask, or one per row, or be given [allowed_rows]")


def _rules_struct(rules, rows, items, device):
    """rfm_score_rules of a call of `rows` rows, or ValueError"""
    if not isinstance(rules, ScoreRules):
        raise ValueError("[rules] must be a rankfm_amd.ScoreRules")
    u = _hip.ScoreRulesStruct(repetition_all=1.0)
    if rules.history is not None:
        offsets, listed = rules.history
        u.history_offsets = check_tensor(offsets, "history offsets", torch.int64, (None,), device)
        u.history_items = check_tensor(listed, "history items", torch.int32, (None,), device)
        u.n_history, u.n_history_items = offsets.shape[0] - 1, listed.shape[0]
        if u.n_history < 0:
            raise ValueError("[history offsets] must have at least one entry")
        if rules.history_rows is not None:
            u.history_rows = check_tensor(rules.history_rows, "history_rows", torch.int32, (rows,), device)
        elif u.n_history != rows:
            raise ValueError("[history] must hold one list per row, or be given [history_rows]")
        for name in ("repetition", "frequency", "presence"):
            _number_or_rows(u, name, getattr(rules, name), rows, device)
    elif rules.history_rows is not None or rules.penalises():
        raise ValueError("[repetition], [frequency], [presence] and [history_rows] need [history]")
    if rules.item_bias is not None:
        u.item_bias = check_tensor(rules.item_bias, "item_bias", torch.float32, (items,), device)
    if rules.row_bias is not None:
        offsets, listed, values = rules.row_bias
        u.bias_offsets = check_tensor(offsets, "row_bias offsets", torch.int64, (rows + 1,), device)
        u.bias_items = check_tensor(listed, "row_bias items", torch.int32, (None,), device)
        u.bias_values = check_tensor(values, "row_bias values", torch.float32, tuple(listed.shape), device)
        u.n_bias_items = listed.shape[0]
    allowed_fields(u, rules.allowed, rules.allowed_rows, rows, items, device)
    return u


def check_rules(rules, rows, items, device):
    """ValueError unless the rules are those of a call of `rows` rows"""
    _rules_struct(rules, rows, items, device)


def _byte_range(t):
    return t.data_ptr(), t.data_ptr() + ((t.shape[0] - 1) * t.stride(0) + (t.shape[1] - 1) * t.stride(1) + 1) * t.element_size()


def _overlap(x, y):
    """whether rows of one shape share an element.  Exact for rows equally far apart, which may lie between each other (halves of wider rows); others
    overlap if their ranges do"""
    (a, b), (c, d) = _byte_range(x), _byte_range(y)
    if b <= c or d <= a:
        return False
    rows, items = x.shape
    stride, size = _row_stride(x), x.element_size()
    if rows == 1 or _row_stride(y) != stride:
        return True
    apart = (c - a) % (stride * size)                            # from a row of x to the next row of y
    return apart < items * size or apart > (stride - items) * size


def adjust_scores(scores, rules, out=None):
    """the score rows under the rules, rounded once to the scores' type

    scores   float32, float16 or bfloat16 [rows, items], rows of consecutive items (the rows themselves may be strided)
    out      None (a new tensor), `scores` itself (in place), or a tensor of the same type and shape that does not overlap it
    """
    warn_if_cut("adjust_scores", scores)
    device = _check_scores(scores)
    rows, items = scores.shape
    given = out
    if out is None:
        out = torch.empty_like(scores) if scores.is_contiguous() else scores.new_empty((rows, items))
    elif out is not scores:
        if not isinstance(out, torch.Tensor) or out.dtype != scores.dtype or out.shape != scores.shape or out.device != device:
            raise ValueError("[out] must be a tensor of the scores' type, shape and device")
        if items > 1 and out.stride(1) != 1 or rows > 1 and out.stride(0) < items:
            raise ValueError("[out] must have rows of consecutive items that do not overlap")
        if rows and (out.data_ptr(), _row_stride(out)) != (scores.data_ptr(), _row_stride(scores)) and _overlap(scores, out):
            raise ValueError("[out] must be [scores] itself or not overlap it")
    u = _rules_struct(rules, rows, items, device)
    if rows == 0:
        return out
    launch(device, _hip.lib().rfm_adjust_scores_device, C.byref(u), _DTYPES[scores.dtype], rows, items, scores.data_ptr(), _row_stride(scores), out.data_ptr(),
           _row_stride(out))
    if given is not None and not given.is_inference():
        torch.autograd.graph.increment_version(given)            # (a backward pass that has kept it says so instead of using what it is now)
    return out


def top_scores(scores, n, rules=None):
    """the `n` best items of every row and their scores under the rules: `TopScores(items, scores)`

    By descending score, the lower index first among equals; NaN and -inf never rank.  The adjusted rows are not written anywhere.

    One pass over the rows up to 768 wanted (384 under rules); a longer list is taken in rounds of that many, each a pass of its own, and from 1025 on
    by one workgroup per row: 0.3 ms for 1024 of one row of 200 k, 1.0 ms for 5000, 4.7 ms for 20,000 and 74 ms for all of it (116 under rules).  For a
    ranking of everything a sort is the better tool.
    """
    warn_if_cut("top_scores", scores)
    device = _check_scores(scores)
    rows, items = scores.shape
    n = int(n)
    if n < 1 or n > items:
        raise ValueError("[n] must be between 1 and the number of items")
    u = None if rules is None else _rules_struct(rules, rows, items, device)
    best = torch.empty((rows, n), dtype=torch.int32, device=device)
    value = torch.empty((rows, n), dtype=torch.float32, device=device)
    if rows == 0:
        return TopScores(best, value)
    lib = _hip.lib()
    ws = scores.new_empty(lib.rfm_top_scores_workspace_bytes(rows, items, n), dtype=torch.uint8)
    launch(device, lib.rfm_top_scores_device, C.byref(u) if u is not None else None, _DTYPES[scores.dtype], rows, items, scores.data_ptr(), _row_stride(scores), n,
           best.data_ptr(), value.data_ptr(), ws.data_ptr(), ws.numel())
    return TopScores(best, value)
