"""Learning from another model's answers: a student's catalogue distribution against a teacher's top scores.

Student: z[r, i] = <users[r], items[i]> + bias[i], q = softmax(z / temperature) over the allowed items.  Teacher: a list of items and scores
per row (`top_scores` makes one), p = softmax(scores / temperature) over the usable entries: item in the catalogue (-1 is padding) and
allowed, score not -inf; an item that stands there twice counts twice.

    loss[r] = temperature^2 * sum_j p_j (log p_j - log q[item_j])                   a row without a usable entry: 0
    gradients of sum_r row_weight[r] * loss[r]:  dz = temperature * row_weight * (q - p),  dz . items,  dz^T . users,  column sums

All float32, like the model's weights; sums are float32.  Up to 128 factors the products are made of two half-precision parts per factor: a product of two
factors is off by up to 2^-21 of its size and by 2^-24.2 in the mean (a float32 product: 2^-24, 2^-25.5).  The parts are scaled by a power of two
per tile of 32 consecutive rows of [users] or [items].  That holds for factors down to 2^-16 of the largest finite one of their tile; below, a factor is off by
up to 2^-40 of the largest (or by 2^-65, in a tile that holds nothing above 2^-26).  In the items' gradient it is a row's factor times
its row_weight that counts so.  The weights q and p of the gradients are cut likewise: at 2^-40 of the largest that a row has among a tile's 32
items, or an item among a tile's 32 rows.  A factor that is not finite spoils the rows it counts in, and nothing where a mask takes it out.  At most
2^24 rows, 2^25 items, 1024 factors and 1024 entries per list.

The device's current stream; no host synchronisation.  The gradients are returned, not recorded by
autograd.  Sums have a fixed order: the same call gives the same bits.
"""
import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import _hip
from .scores import allowed_fields, check_device, check_tensor, launch, warn_if_cut


class DistillGradients(NamedTuple):
    loss: torch.Tensor                   # [rows], unweighted
    users: torch.Tensor                  # [rows, factors]
    items: torch.Tensor                  # [items, factors]
    bias: Optional[torch.Tensor]         # [items]; None without a bias


def _factor_rows(t, name, device=None):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.dim() != 2:
        raise ValueError("[%s] must be a float32 tensor [rows, factors]" % name)
    if t.shape[1] < 1 or t.shape[1] > 1024:
        raise ValueError("[%s] must have between 1 and 1024 factors" % name)
    if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError("[%s] must have rows of consecutive factors that do not overlap" % name)
    if device is not None and t.device != device:
        raise ValueError("[%s] is on %s, the call on %s" % (name, t.device, device))
    return t.data_ptr(), t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _call(users, items, bias, teacher_items, teacher_scores, temperature, allowed, allowed_rows, row_weight, gradients):
    a = _hip.DistillArgs()
    a.users, a.user_stride = _factor_rows(users, "users")
    device = check_device(users, "users")
    a.items, a.item_stride = _factor_rows(items, "items", device)
    rows, factors = users.shape
    if items.shape[0] < 1 or items.shape[1] != factors:
        raise ValueError("[items] must have at least one row and as many factors as [users]")
    a.n_rows, a.n_items, a.n_factors = rows, items.shape[0], factors
    a.bias = None if bias is None else check_tensor(bias, "bias", torch.float32, (a.n_items,), device)
    a.teacher_items = check_tensor(teacher_items, "teacher_items", torch.int32, (rows, None), device)
    a.teacher_scores = check_tensor(teacher_scores, "teacher_scores", torch.float32, tuple(teacher_items.shape), device)
    a.n_teacher = teacher_items.shape[1]
    if a.n_teacher < 1 or a.n_teacher > 1024:
        raise ValueError("[teacher_items] must have between 1 and 1024 entries per row")
    a.temperature = float(temperature)
    if not 2.0 ** -126 <= a.temperature < float("inf"):          # (below, its inverse is infinite in float32)
        raise ValueError("[temperature] must be a finite number above 0, 2^-126 at least")
    allowed_fields(a, allowed, allowed_rows, rows, a.n_items, device)
    if row_weight is not None:
        a.row_weight = check_tensor(row_weight, "row_weight", torch.float32, (rows,), device)
    loss = users.new_empty(rows)
    a.loss = loss.data_ptr()
    d_users = d_items = d_bias = None
    if gradients:
        d_users = users.new_empty((rows, factors))
        d_items = users.new_empty((a.n_items, factors))
        if rows == 0:
            return DistillGradients(loss, d_users, d_items.zero_(), None if bias is None else torch.zeros_like(bias))
        a.d_users, a.d_items = d_users.data_ptr(), d_items.data_ptr()
        if bias is not None:
            d_bias = users.new_empty(a.n_items)
            a.d_bias = d_bias.data_ptr()
    elif rows == 0:
        return loss
    lib = _hip.lib()
    ws = users.new_empty(lib.rfm_distill_workspace_bytes(C.byref(a)), dtype=torch.uint8)
    launch(device, lib.rfm_distill_device, C.byref(a), ws.data_ptr(), ws.numel())
    return DistillGradients(loss, d_users, d_items, d_bias) if gradients else loss


def distill_loss(users, items, bias, teacher_items, teacher_scores, *, temperature=1.0, allowed=None, allowed_rows=None):
    """loss [rows] of the student's rows against the teacher's lists

    users            float32 [rows, factors], items float32 [items, factors] (rows may be strided), bias float32 [items] or None
    teacher_items    int32 [rows, n], -1 for padding; teacher_scores float32 [rows, n]
    allowed, allowed_rows    masks of the items the student's distribution ranges over, as in `ScoreRules`

    The loss cannot be differentiated (its gradients are `distill_gradients`'): with tensors that require a gradient the call warns.
    """
    warn_if_cut("distill_loss", users, items, bias, teacher_scores)
    return _call(users, items, bias, teacher_items, teacher_scores, temperature, allowed, allowed_rows, None, False)


def distill_gradients(users, items, bias, teacher_items, teacher_scores, *, temperature=1.0, allowed=None, allowed_rows=None, row_weight=None):
    """`DistillGradients`: the loss of `distill_loss` and the gradients of sum(row_weight * loss) with respect to users, items and bias"""
    return _call(users, items, bias, teacher_items, teacher_scores, temperature, allowed, allowed_rows, row_weight, True)
