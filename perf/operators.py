"""Cases of the catalogue-score operators: answering under rules (`adjust_scores`, `top_scores`) and learning from another model's
answers (`distill_loss`, `distill_gradients`), with their plain forms in elementary torch operations."""
import math

import torch

own = False

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
WORD = 32                      # items per word of an allowed-items mask


def listed():
    return [
        # one user's answer over a MovieLens-1M-sized catalogue: the call a web request waits for
        dict(name="adjust_one_user", op="adjust", rows=1, items=3706, type="float32", history=165, masks=0, row_bias=4, item_bias=True),
        # a serving batch over a grocery catalogue (an odd item count: no row but the first is 16-byte aligned), every rule at once
        dict(name="adjust_batch", op="adjust", rows=1000, items=34977, type="float32", history=55, masks=16, row_bias=8, item_bias=True),
        # half-width rows of a large catalogue, regional masks and repeat penalties
        dict(name="adjust_bf16_200k", op="adjust", rows=512, items=200_000, type="bfloat16", history=50, masks=8, row_bias=0, item_bias=False),
        # one row of a large catalogue, a long list: nothing but the row itself to spread over the chip
        dict(name="top_one_row", op="top", rows=1, items=200_000, type="float32", n=100, ruled=False, history=0, masks=0, row_bias=0, item_bias=False),
        # a serving batch: the ten best under every rule, the adjusted rows themselves are not wanted
        dict(name="top_under_rules", op="top", rows=1024, items=50_000, type="float32", n=10, ruled=True, history=50, masks=16, row_bias=8, item_bias=True),
        # a teacher's lists for a training batch
        dict(name="top_teacher_lists", op="top", rows=4096, items=50_000, type="float32", n=64, ruled=False, history=0, masks=0, row_bias=0, item_bias=False),
        # held-out loss of a small student on a handful of users
        dict(name="loss_small", op="loss", rows=64, items=3706, factors=20, n=10, masked=False, temperature=1.0),
        # held-out loss of a k = 64 student over the 50 k catalogue
        dict(name="loss_large", op="loss", rows=8192, items=50_000, factors=64, n=32, masked=False, temperature=2.0),
        # a small student's training step
        dict(name="grad_small", op="grad", rows=100, items=3706, factors=20, n=10, masked=False, temperature=1.0),
        # every size odd, and each user's observed items left out of the student's distribution
        dict(name="grad_masked", op="grad", rows=1503, items=34977, factors=50, n=10, masked=True, temperature=1.5),
        # a k = 64 student's training step over the 50 k catalogue
        dict(name="grad_large", op="grad", rows=8192, items=50_000, factors=64, n=32, masked=False, temperature=2.0),
        # a k = 128 student over a 200 k catalogue, long teacher lists
        dict(name="grad_wide", op="grad", rows=2048, items=200_000, factors=128, n=64, masked=False, temperature=2.0),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["adjust", "top", "loss", "grad"])
    items = log_int(500, 200_000)
    if op in ("adjust", "top"):
        rows = log_int(1, min(4096, 100_000_000 // items))
        case = dict(op=op, rows=rows, items=items, type=rng.choice(list(TYPES)), history=rng.choice([0, log_int(1, 400)]),
                    masks=rng.choice([0, 1, rng.randint(2, 32)]), row_bias=rng.choice([0, rng.randint(1, 32)]), item_bias=rng.random() < 0.5)
        if op == "top":
            case.update(n=min(log_int(1, 500), items), ruled=rng.random() < 0.5)
            if not case["ruled"]:
                case.update(history=0, masks=0, row_bias=0, item_bias=False)
        elif not (case["history"] or case["masks"] or case["row_bias"]):
            case["item_bias"] = True
        return case
    factors = log_int(8, 128)
    rows = log_int(16, max(17, min(8192, 26_000_000_000 // (items * factors))))
    return dict(op=op, rows=rows, items=items, factors=factors, n=log_int(1, 128), masked=rng.random() < 0.4,
                temperature=rng.choice([0.5, 1.0, 1.5, 2.0, 4.0]))


# ---- inputs -------------------------------------------------------------------------------------------------------------------------------

def _lists(rows, mean, items, gen):
    """back-to-back item lists with repeats (popular items more often, in no order), some of them empty: offsets [rows + 1], items"""
    length = (torch.rand(rows, generator=gen, device="cuda") * (2 * mean + 1)).long()
    if rows > 1:
        length[0] = 0
    length[-1].clamp_(min=mean)
    offsets = torch.zeros(rows + 1, dtype=torch.int64, device="cuda")
    offsets[1:] = length.cumsum(0)
    total = int(offsets[-1])
    entry = (torch.rand(total, generator=gen, device="cuda", dtype=torch.float64) ** 3 * items).long().clamp_(max=items - 1)
    return offsets, ((entry * 7919) % items).int()


def _masks(count, items, share, gen):
    """`count` masks of allowed items, one bit per item (the bits behind the last item are set and mean nothing)"""
    words = (items + WORD - 1) // WORD
    bits = torch.rand(count, words, WORD, generator=gen, device="cuda") < share
    value = (bits.long() << torch.arange(WORD, device="cuda")).sum(-1)
    return torch.where(value >= 2 ** 31, value - 2 ** 32, value).int()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, items = case["rows"], case["items"]
    state = {k: v for k, v in case.items() if k not in ("history", "row_bias", "item_bias", "masks")}

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    if case["op"] in ("adjust", "top"):
        state["scores"] = (normal(rows, items) * 1.5).to(TYPES[case["type"]])
        if case["history"]:
            people = rows + 3                       # the lists of all users; a row names its own
            state["history"] = _lists(people, case["history"], items, gen)
            state["history_rows"] = torch.randperm(people, generator=gen, device="cuda")[:rows].int()
            if rows > 2:
                state["history_rows"][rows // 2] = -1   # somebody unknown: no history
            state["repetition"] = 1.0 + uniform(rows)
            state["frequency"] = 0.5 * uniform(rows)
            state["presence"] = 0.25
        if case["masks"]:
            state["allowed"] = _masks(case["masks"], items, 0.7, gen)
            if case["masks"] > 4:
                state["allowed"][0] = 0             # a region that nothing is sold in
            which = (uniform(rows) * (case["masks"] + 1)).int().clamp_(max=case["masks"]) - 1
            state["allowed_rows"] = which           # -1: everything is allowed
        if case["item_bias"]:
            state["item_bias"] = normal(items) * 0.2
        if case["row_bias"]:
            offsets, ids = _lists(rows, case["row_bias"], items, gen)
            state["row_bias"] = (offsets, ids, normal(ids.numel()))
        return state

    factors, n = case["factors"], case["n"]
    scale = (1.5 / math.sqrt(factors)) ** 0.5
    state["users"], state["item_rows"] = normal(rows, factors) * scale, normal(items, factors) * scale
    state["bias"] = normal(items) * 0.5
    # a teacher's lists: popular items more often, no item twice in a row, scores descending; some rows are shorter (-1 behind their end)
    popular = torch.log(torch.arange(1, items + 1, device="cuda") ** -0.8)[torch.randperm(items, generator=gen, device="cuda")]
    value, entry = torch.topk(popular - torch.log(-torch.log(uniform(rows, items).clamp_(1e-7, 1 - 1e-7))), min(n, items), dim=1)
    state["teacher_items"], state["teacher_scores"] = entry.int(), (2.0 * value).contiguous()
    short = uniform(rows) < 0.05
    state["teacher_items"][short, n // 2:] = -1
    state["row_weight"] = (0.5 + uniform(rows)) / rows
    if case["masked"]:
        state["allowed"] = _masks(rows, items, 0.98, gen)     # a user's unobserved items
        state["allowed"][rows // 3] = 0                       # somebody who has seen everything
    return state


# ---- the operators in plain form ------------------------------------------------------------------------------------------------------------

def _allowed(state, items):
    """bool [rows, items]: the row's mask, everything where it has none"""
    bits = (state["allowed"].unsqueeze(-1) >> torch.arange(WORD, device="cuda", dtype=torch.int32)) & 1
    bits = bits.flatten(1)[:, :items].bool()
    which = state.get("allowed_rows")
    if which is None:
        return bits
    return bits[which.long().clamp(min=0)] | (which < 0).unsqueeze(1)


def _entries(offsets, listed_rows):
    """(row of the call, position in the lists) of every entry of the listed rows"""
    known = listed_rows >= 0
    at = listed_rows.long().clamp(min=0)
    begin = offsets[at]
    length = torch.where(known, offsets[at + 1] - begin, 0)
    row = torch.repeat_interleave(torch.arange(length.numel(), device="cuda"), length)
    first = length.cumsum(0) - length
    return row, begin[row] + torch.arange(row.numel(), device="cuda") - first[row]


def _per_row(value):
    return value.unsqueeze(1) if isinstance(value, torch.Tensor) else value


def _adjusted(state):
    rows, items = state["rows"], state["items"]
    s = state["scores"].float()
    if state.get("history") is not None:
        offsets, ids = state["history"]
        row, at = _entries(offsets, state["history_rows"])
        count = torch.zeros(rows * items, device="cuda")
        count = count.index_add_(0, row * items + ids[at].long(), torch.ones(row.numel(), device="cuda")).view(rows, items)
        rho = _per_row(state["repetition"])
        penal = torch.where(s > 0, s / rho, s * rho)
        penal = penal - _per_row(state["frequency"]) * count
        penal = penal - _per_row(state["presence"])
        s = torch.where(count > 0, penal, s)
    if state.get("item_bias") is not None:
        s = s + state["item_bias"]
    if state.get("row_bias") is not None:
        offsets, ids, values = state["row_bias"]
        row, at = _entries(offsets, torch.arange(rows, device="cuda"))
        last = torch.full((rows * items,), -1, dtype=torch.int64, device="cuda")
        last = last.scatter_reduce_(0, row * items + ids[at].long(), at, "amax").view(rows, items)
        s = torch.where(last >= 0, s + values[last.clamp(min=0)], s)
    if state.get("allowed") is not None:
        s = torch.where(_allowed(state, items), s, -math.inf)
    return s


def _top(s, n):
    s = torch.where(torch.isnan(s), -math.inf, s)
    value, item = torch.sort(s, dim=1, descending=True, stable=True)
    value, item = value[:, :n].contiguous(), item[:, :n]
    return torch.where(value > -math.inf, item, -1).int(), value


def _distilled(state, gradients):
    tau = state["temperature"]
    z = (state["users"] @ state["item_rows"].T + state["bias"]) / tau
    ids, t = state["teacher_items"].long(), state["teacher_scores"] / tau
    usable = ids >= 0
    ids = ids.clamp(min=0)
    if state.get("allowed") is not None:
        allowed = _allowed(state, state["items"])
        z = torch.where(allowed, z, -math.inf)
        usable = usable & allowed.gather(1, ids)
    some = usable.any(1, keepdim=True)
    top = torch.where(usable, t, -math.inf).amax(1, keepdim=True)
    e = torch.where(usable, torch.exp(t - torch.where(some, top, 0.0)), 0.0)
    mass = e.sum(1, keepdim=True)
    p = torch.where(some, e / torch.where(some, mass, 1.0), 0.0)
    log_p = torch.where(usable, t - top - torch.log(mass), 0.0)
    best = z.amax(1, keepdim=True)
    best = torch.where(best > -math.inf, best, 0.0)
    ez = torch.exp(z - best)
    total = ez.sum(1, keepdim=True)
    log_q = torch.where(usable, z.gather(1, ids), 0.0) - best - torch.log(torch.where(total > 0, total, 1.0))
    loss = tau * tau * (p * (log_p - log_q)).sum(1)
    if not gradients:
        return loss
    dz = torch.where(some, ez / torch.where(total > 0, total, 1.0), 0.0)
    dz = dz.scatter_add_(1, ids, -p) * (tau * state["row_weight"].unsqueeze(1))
    return loss, dz @ state["item_rows"], dz.T @ state["users"], dz.sum(0)


def _rules(state):
    from rankfm_amd import ScoreRules
    return ScoreRules(history=state.get("history"), history_rows=state.get("history_rows"), repetition=state.get("repetition", 1.0),
                      frequency=state.get("frequency", 0.0), presence=state.get("presence", 0.0), item_bias=state.get("item_bias"),
                      row_bias=state.get("row_bias"), allowed=state.get("allowed"), allowed_rows=state.get("allowed_rows"))


def run(state):
    op = state["op"]
    if own:
        import rankfm_amd
        if op == "adjust":
            return rankfm_amd.adjust_scores(state["scores"], _rules(state))
        if op == "top":
            return tuple(rankfm_amd.top_scores(state["scores"], state["n"], _rules(state) if state["ruled"] else None))
        given = (state["users"], state["item_rows"], state["bias"], state["teacher_items"], state["teacher_scores"])
        if op == "loss":
            return rankfm_amd.distill_loss(*given, temperature=state["temperature"], allowed=state.get("allowed"))
        return tuple(rankfm_amd.distill_gradients(*given, temperature=state["temperature"], allowed=state.get("allowed"), row_weight=state["row_weight"]))
    if op == "adjust":
        return _adjusted(state).to(state["scores"].dtype)
    if op == "top":
        return _top(_adjusted(state) if state["ruled"] else state["scores"].float(), state["n"])
    return _distilled(state, op == "grad")


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------------------------

def work(case):
    rows, items = case["rows"], case["items"]
    if case["op"] in ("adjust", "top"):
        size = 4 if case["type"] == "float32" else 2
        lists = rows * (4 * case["history"] + 8 * case["row_bias"]) + 4 * items * bool(case["item_bias"]) + case["masks"] * items // 8
        out = rows * items * size if case["op"] == "adjust" else rows * case["n"] * 8
        return {"bytes": rows * items * size + lists + out, "flops": rows * items * 2}
    factors, n = case["factors"], case["n"]
    product = 2 * rows * items * factors
    tables = 4 * (rows * factors + items * factors + items) + 8 * rows * n + (rows * items // 8 if case["masked"] else 0)
    if case["op"] == "loss":
        return {"bytes": tables + 4 * rows, "flops": product}
    return {"bytes": tables + 4 * (rows * factors + items * factors + items + 2 * rows), "flops": 3 * product}


# ---- the definitions, in 64 bits and row by row or block by block of rows ----------------------------------------------------------------------

def _exact_rows(state, r):
    """row r under its rules"""
    items = state["items"]
    s = state["scores"][r].double()
    if state.get("history") is not None:
        who = int(state["history_rows"][r])
        if who >= 0:
            a, b = state["history"][0][who:who + 2].tolist()
            count = torch.bincount(state["history"][1][a:b].long(), minlength=items).double()
            rho, phi = state["repetition"][r].double(), state["frequency"][r].double()
            hit = count > 0
            s[hit] = torch.where(s[hit] > 0, s[hit] / rho, s[hit] * rho) - phi * count[hit] - state["presence"]
    if state.get("item_bias") is not None:
        s = s + state["item_bias"].double()
    if state.get("row_bias") is not None:
        a, b = state["row_bias"][0][r:r + 2].tolist()
        extra = dict(zip(state["row_bias"][1][a:b].tolist(), state["row_bias"][2][a:b].tolist()))     # the last entry of an item stays
        if extra:
            s[torch.tensor(list(extra), device="cuda")] += torch.tensor(list(extra.values()), dtype=torch.float64, device="cuda")
    if state.get("allowed") is not None:
        which = int(state["allowed_rows"][r])
        if which >= 0:
            item = torch.arange(items, device="cuda")
            off = (state["allowed"][which][item // WORD] >> (item % WORD)) & 1 == 0
            s[off] = -math.inf
    return s


def exact(case, seed):
    state = prepare(case, seed)
    op, rows, items = case["op"], case["rows"], case["items"]
    if op == "adjust":
        return torch.stack([_exact_rows(state, r) for r in range(rows)])
    if op == "top":
        value, item = [], []
        for r in range(rows):
            s = _exact_rows(state, r) if case["ruled"] else state["scores"][r].double()
            v, i = s.sort(descending=True, stable=True)
            value.append(v[:case["n"]])
            item.append(torch.where(v[:case["n"]] > -math.inf, i[:case["n"]], -1).int())
        # (under rules the order is that of the adjusted scores in 32 bits: 64 bits may rank two of them the other way round)
        return (None if case["ruled"] else torch.stack(item)), torch.stack(value)
    tau, v = case["temperature"], state["item_rows"].double()
    losses, d_users = [], []
    d_items, d_bias = torch.zeros_like(v), torch.zeros(items, dtype=torch.float64, device="cuda")
    step = max(1, 60_000_000 // items)
    for a in range(0, rows, step):
        u = state["users"][a:a + step].double()
        z = (u @ v.T + state["bias"].double()) / tau
        ids = state["teacher_items"][a:a + step].long()
        t = state["teacher_scores"][a:a + step].double() / tau
        t = t.masked_fill(ids < 0, -math.inf)
        if state.get("allowed") is not None:
            item = torch.arange(items, device="cuda")
            off = (state["allowed"][a:a + step][:, item // WORD] >> (item % WORD).int()) & 1 == 0
            z = z.masked_fill(off, -math.inf)
            t = t.masked_fill(off.gather(1, ids.clamp(min=0)), -math.inf)
        empty = (t == -math.inf).all(1)
        log_q = torch.log_softmax(z, 1)
        log_p = torch.log_softmax(t, 1)
        p = log_p.exp().masked_fill(t == -math.inf, 0.0)
        cross = log_p - log_q.gather(1, ids.clamp(min=0))
        losses.append((tau * tau * (p * cross).masked_fill(t == -math.inf, 0.0).sum(1)).masked_fill(empty, 0.0))
        if op == "grad":
            dz = log_q.exp().scatter_add(1, ids.clamp(min=0), -p).masked_fill(empty.unsqueeze(1), 0.0)
            dz = dz * (tau * state["row_weight"][a:a + step].double()).unsqueeze(1)
            d_users.append(dz @ v)
            d_items += dz.T @ u
            d_bias += dz.sum(0)
    loss = torch.cat(losses)
    return loss if op == "loss" else (loss, torch.cat(d_users), d_items, d_bias)
