"""Reports on choices and distillation, case by case, in a plain form and through the package's entry points.

A case is a dict of plain values. `op` names what a user calls:

  report   choice_report: of each set the chosen row's log-probability, the entropy, and the `top` rows of largest
           probability with theirs
  bonus    choice_report without lists and choice_report_backward: a training step whose loss has the chosen rows'
           log-probabilities and the sets' entropies
  distill  distillation_loss: the divergence from a teacher of which each set's `top` best rows are known, its
           value and the scores' gradient; `tail`: the rest of the teacher's probability counts as one more row

`spread` says how the rows fall into sets: "even" (all of one size), "ragged" (exponential sizes, empty sets among
them) or "heavy" (lognormal: a few sets hold most rows). `bias` is the number of position buckets (0: no position
bias) and `reach` the distance from which the last bucket is used. `mask` is the share of candidates left out; what
they hold is not meant to be read (NaN, infinities and the type's lowest value among it), and one set in a hundred is
left without any candidate. `teacher` is the type of the teacher's values; a few of its entries are absent, masked for the
student, or beyond their set.

`prepare` makes what a user's program holds before the call, `run` makes one pass, `exact` computes the same in 64 bits
on the host.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SETS = dict(dtype="f32", spread="ragged", mask=0.0, bias=0, reach=128, temperature=1.0)
REPORT = dict(SETS, op="report")
BONUS = dict(SETS, op="bonus")
DISTILL = dict(SETS, op="distill", tail=False, teacher="f32", weighted=False)


def listed():
    return [
        # one request: how sure the model is about a short list of candidates and its best ones, where latency counts
        dict(REPORT, name="report_request", rows=37, sets=1, spread="even", top=5),
        # one decision over a large fixed inventory, with the 20 best alternatives beside what was taken
        dict(REPORT, name="report_single", rows=32_000, sets=1, spread="even", dtype="bf16", top=20),
        # a served batch of lists with unavailable items, shown in an order the model has a bias for
        dict(REPORT, name="report_lists", rows=200_003, sets=16_000, mask=0.1, bias=32, top=8, temperature=0.7),
        # a few requests over a whole catalogue, to keep a teacher's 64 best of each
        dict(REPORT, name="report_catalogue", rows=5_000_000, sets=24, spread="heavy", top=64),
        # the log of a rollout over a large fixed inventory: a set per step, scores kept in bf16
        dict(REPORT, name="report_inventory", rows=4096 * 32_000, sets=4096, spread="even", dtype="bf16", top=8),
        # an entropy bonus on a handful of decisions, where latency counts
        dict(BONUS, name="bonus_small", rows=1_500, sets=200),
        # clicks on lists of the panel's size with an entropy term, the position bias learned beside the scores
        dict(BONUS, name="bonus_clicks", rows=2_400_000, sets=100_003, mask=0.02, bias=64, reach=200),
        # a large rollout of uneven decisions, from one candidate to many thousands, scores kept in bf16
        dict(BONUS, name="bonus_rollout", rows=40_000_003, sets=100_000, spread="heavy", dtype="bf16", temperature=1.5),
        # a student on a handful of lists, where latency counts
        dict(DISTILL, name="distill_small", rows=1_500, sets=200, top=4, temperature=2.0),
        # a student of a larger model's best eight on lists of the panel's size
        dict(DISTILL, name="distill_lists", rows=2_400_000, sets=100_003, mask=0.05, bias=64, reach=200, top=8, tail=True,
             weighted=True),
        # a student over catalogues of uneven size, the teacher's 64 best of each kept
        dict(DISTILL, name="distill_catalogue", rows=10_000_000, sets=300, spread="heavy", top=64, tail=True),
        # a student over a large fixed inventory, scores and the teacher's best 16 kept in bf16
        dict(DISTILL, name="distill_inventory", rows=4096 * 32_000, sets=4096, spread="even", dtype="bf16", top=16,
             teacher="bf16", temperature=2.0),
    ]


# ------------------------------------------------------------------------------------ drawn cases
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["report", "report", "bonus", "distill", "distill"])
    kind = rng.choice(["short", "short", "long", "even"])
    c = dict(SETS, op=op, dtype=rng.choice(["f32", "f32", "bf16", "f16"]), mask=rng.choice([0.0, 0.0, 0.1, 0.5]),
             bias=rng.choice([0, 0, 16, 32, 64]), reach=rng.choice([64, 128, 500]),
             temperature=rng.choice([1.0, 1.0, 0.5, 0.8, 2.0, 4.0]))
    if kind == "short":
        c.update(rows=_log(rng, 100, 20_000_000))
        c.update(sets=max(1, c["rows"] // _log(rng, 2, 60)), spread=rng.choice(["ragged", "heavy"]))
    elif kind == "long":
        c.update(rows=_log(rng, 5_000, 20_000_000))
        c.update(sets=max(1, c["rows"] // _log(rng, 500, 200_000)), spread=rng.choice(["ragged", "heavy"]))
    else:
        size = _log(rng, 2, 60_000)
        c.update(sets=_log(rng, 1, max(1, 20_000_000 // size)), spread="even")
        c.update(rows=size * c["sets"])
    if op != "bonus":  # lists of at most about 64M entries
        c.update(top=_log(rng, 1, max(1, min(64, 64_000_000 // c["sets"]))))
    if op == "distill":
        c = dict(DISTILL, **c)
        c.update(tail=rng.random() < 0.5, teacher=rng.choice(["f32", "f32", "bf16", "f16"]), weighted=rng.random() < 0.5)
    return c


# ------------------------------------------------------------------------------------ inputs
def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _uniform(n, g):
    return torch.rand(n, device=DEV, generator=g, dtype=torch.float64)


def _offsets(n, parts, spread, g):
    """int64 [parts + 1]: n rows in `parts` runs."""
    if spread == "even":
        return torch.arange(parts + 1, device=DEV, dtype=torch.int64) * (n // parts)
    w = -torch.log(_uniform(parts, g).clamp_min(1e-12))
    if spread == "heavy":
        w = torch.exp(1.5 * torch.randn(parts, device=DEV, generator=g, dtype=torch.float64))
    off = torch.zeros(parts + 1, device=DEV, dtype=torch.int64)
    off[1:] = torch.floor(torch.cumsum(w, 0) / w.sum() * n).to(torch.int64).clamp_(max=n)
    off[-1] = n
    return off


def _spread_over(v, off, n):
    """v[set of row i] for every row."""
    return torch.repeat_interleave(v, off[1:] - off[:-1], output_size=n)


def _best(z, off, k, even):
    """int64 [sets, k]: each set's rows of largest z, within the set; equal ones by index; -1 behind the last.
    Rows of z = -inf are not listed."""
    n, sets = z.numel(), off.numel() - 1
    if n == 0:
        return torch.full((sets, k), -1, device=DEV, dtype=torch.int64)
    if even:  # the largest of keys that no two rows share
        size = n // sets
        bits = (z + 0.0).view(torch.int32).long()
        key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) << 32
        key |= 0xFFFFFFFF - torch.arange(size, device=DEV).repeat(sets)
        best = key.view(sets, size).topk(min(k, size), dim=1).indices
        best = torch.where(z.view(sets, size).gather(1, best) == -math.inf, -1, best)
        return torch.cat([best, torch.full((sets, k - best.shape[1]), -1, device=DEV)], 1)
    seg = _spread_over(torch.arange(sets, device=DEV), off, n)
    order = torch.sort(z, descending=True, stable=True).indices
    order = order[torch.sort(seg[order], stable=True).indices]  # by set, within it by z, within that by index
    at = off[:-1].unsqueeze(1) + torch.arange(k, device=DEV)
    there = at < off[1:].unsqueeze(1)
    row = order[at.clamp(max=n - 1)]
    return torch.where(there & (z[row] != -math.inf), row - off[:-1].unsqueeze(1), -1)


def _double_set_lse(x, off, even):
    """log of the sum of exponentials over each set, in 64 bits; 0 where that is nothing."""
    n, sets = x.numel(), off.numel() - 1
    if even:
        lse = torch.logsumexp(x.view(sets, -1), 1)
    else:
        seg = _spread_over(torch.arange(sets, device=DEV), off, n)
        top = torch.full((sets,), -math.inf, device=DEV, dtype=torch.float64).scatter_reduce_(0, seg, x, "amax")
        top = torch.where(torch.isinf(top), 0.0, top)
        lse = top + torch.log(torch.zeros(sets, device=DEV, dtype=torch.float64).index_add_(0, seg, torch.exp(x - top[seg])))
    return torch.where(torch.isinf(lse), 0.0, lse)


def _inputs(case, seed):
    """What the program holds, on the GPU, from the seed alone."""
    g = _generator(seed)
    d = {}
    n, sets, even = case["rows"], case["sets"], case["spread"] == "even"
    off = d["offsets"] = _offsets(n, sets, case["spread"], g)
    size = off[1:] - off[:-1]
    chosen = torch.floor(_uniform(sets, g) * size).to(torch.int32)
    chosen[_uniform(sets, g) < 0.05] = -1
    base = 2.0 * torch.randn(n, device=DEV, generator=g)
    if case["mask"] > 0:
        keep = torch.rand(n, device=DEV, generator=g) >= case["mask"]
        keep[(off[:-1] + chosen.clamp_min(0)).clamp(max=n - 1)] = True  # what was taken was on offer
        keep &= ~_spread_over(_uniform(sets, g) < 0.01, off, n)
        d["mask"] = keep
        junk = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(TYPES[case["dtype"]]).min], device=DEV)
        idle = torch.nonzero(~keep).reshape(-1)
        base[idle] = junk[idle % 4]
    d["scores"] = base.to(TYPES[case["dtype"]])
    if case["bias"]:
        local = torch.arange(n, device=DEV) - _spread_over(off[:-1], off, n)
        origin = torch.floor(_uniform(sets, g) * size).to(torch.int64)
        d["positions"] = (local - _spread_over(origin, off, n)).to(torch.int32)
        d["table"] = 0.5 * torch.randn(case["bias"], device=DEV, generator=g)
    if case["op"] != "distill":
        d["chosen"] = chosen
    if case["op"] == "bonus":
        d["grad_log_probs"] = -torch.rand(sets, device=DEV, generator=g)
        d["grad_entropy"] = -0.05 * torch.rand(sets, device=DEV, generator=g)
    if case["op"] == "distill":
        t = d["scores"].float() + torch.randn(n, device=DEV, generator=g)  # the teacher: what the student half knows
        if case["mask"] > 0:
            t = torch.where(d["mask"], t, -math.inf)
        best = _best(t, off, case["top"], even)
        value = t.double()[(off[:-1].unsqueeze(1) + best.clamp_min(0)).clamp(max=n - 1)] / case["temperature"]
        if case["tail"]:
            value = value - _double_set_lse(t.double() / case["temperature"], off, even).unsqueeze(1)
        else:
            value = value * case["temperature"]
        d["teacher_logits"] = torch.where(best < 0, 0.0, value).to(TYPES[case["teacher"]])
        lost = torch.rand(best.shape, device=DEV, generator=g)
        best = torch.where(lost < 0.02, -1, best)
        best = torch.where((lost > 0.99) & (best >= 0), size.unsqueeze(1) + best, best)  # of an older, longer list
        d["teacher_index"] = best.to(torch.int32)
        if case["mask"] > 0:  # and a few that are not on offer any more
            gone = torch.rand(best.shape, device=DEV, generator=g) < 0.02
            at = (off[:-1].unsqueeze(1) + best.clamp_min(0))[gone & (best >= 0)].clamp(max=n - 1)
            d["mask"][at] = False
        if case["weighted"]:
            d["weights"] = torch.rand(sets, device=DEV, generator=g)
    return d


def _bucket_table(num, reach):
    """Bucket of every distance 0 .. reach, for one side of num buckets: exact below num // 2, then
    equal steps of the distance's logarithm, by whole numbers."""
    first, table = num // 2, []
    steps = num - first
    for dist in range(reach + 1):
        if dist < first:
            table.append(dist)
            continue
        k = 0  # the most k with (dist / first)^steps >= (reach / first)^k
        while k + 1 < steps and dist ** steps * first ** (k + 1) >= reach ** (k + 1) * first ** steps:
            k += 1
        table.append(first + k)
    return table


_TABLES: dict = {}


def _bucket_ids(positions, num, reach):
    """Buckets of relative positions: the first half up to and at the reference, the second after it."""
    key = (num, reach)
    if key not in _TABLES:  # a constant of (num, reach)
        _TABLES[key] = torch.tensor(_bucket_table(num // 2, reach), device=DEV)
    p = positions.long()
    return _TABLES[key][p.abs().clamp(max=reach)] + (p > 0) * (num // 2)


def prepare(case, seed):
    d = _inputs(case, seed)
    state = {"case": case, "in": d}
    if own:
        from packboost_amd import ChoiceSets, PositionBias, PositionBuckets

        state["sets"] = ChoiceSets(d["offsets"])
        if "table" in d:
            state["bias"] = PositionBias(d["table"], d["positions"],
                                         PositionBuckets(case["bias"], case["reach"], bidirectional=True))
    else:
        if case["spread"] != "even":
            state["seg"] = _spread_over(torch.arange(case["sets"], device=DEV), d["offsets"], case["rows"])
        if "table" in d:
            _bucket_ids(d["positions"][:1], case["bias"], case["reach"])
    return state


# ------------------------------------------------------------------------------------ plain form
def _set_sum(state, v):
    """Sums over the sets, in 64 bits: they can be long, and a divergence is what their logarithms leave."""
    if "seg" not in state:
        return v.view(state["case"]["sets"], -1).sum(1, dtype=torch.float64)
    return torch.segment_reduce(v.double(), "sum", offsets=state["in"]["offsets"], initial=0.0, unsafe=True)


def _set_max(state, v):
    if "seg" not in state:
        return v.view(state["case"]["sets"], -1).amax(1)
    return torch.segment_reduce(v, "max", offsets=state["in"]["offsets"], initial=-math.inf, unsafe=True)


def _to_rows(state, v):
    if "seg" not in state:
        return v.view(-1, 1).expand(-1, state["case"]["rows"] // state["case"]["sets"]).reshape(-1)
    return v[state["seg"]]


def _plain_logits(state):
    case, d = state["case"], state["in"]
    z = d["scores"].float()
    if "table" in d:
        z = z + d["table"][_bucket_ids(d["positions"], case["bias"], case["reach"])]
    if "mask" in d:
        z = torch.where(d["mask"], z, -math.inf)
    return z


def _plain_softmax(state, z):
    """Largest logit (0 for none), each row's distance to it over the temperature, its exponential, and their sum."""
    top = _set_max(state, z)
    top = torch.where(top == -math.inf, 0.0, top)
    x = (z - _to_rows(state, top)) / state["case"]["temperature"]
    e = torch.exp(x)
    return top, x, e, _set_sum(state, e)


def _plain_report(state, z, top, x, e, total):
    """The chosen rows, whether they count, their log-probabilities, the entropies, the sets' lse, and the
    logarithms of the sums."""
    case, d = state["case"], state["in"]
    off, c = d["offsets"], d["chosen"].long()
    mean = _set_sum(state, torch.where(e == 0, 0.0, e * x)) / torch.where(total == 0, 1.0, total)
    log_total = torch.log(total)
    entropy = torch.where(total == 0, 0.0, log_total - mean).float()
    lse = (top.double() / case["temperature"] + log_total).float()
    log_total = log_total.float()
    counts = (c >= 0) & (c < off[1:] - off[:-1]) & (total != 0)
    at = (off[:-1] + c).clamp(0, z.numel() - 1)
    if "mask" in d:
        counts &= d["mask"][at]
    return at, counts, torch.where(counts, x[at] - log_total, 0.0), entropy, lse, log_total


def _plain_grads(state, g):
    case, d = state["case"], state["in"]
    if "mask" in d:
        g = torch.where(d["mask"], g, 0.0)
    out = (g.to(d["scores"].dtype),)
    if "table" in d:
        ids = _bucket_ids(d["positions"], case["bias"], case["reach"])
        out += (torch.stack([torch.where(ids == b, g, 0.0).sum() for b in range(case["bias"])]),)
    return out


def _plain_distill(state, z):
    case, d = state["case"], state["in"]
    off, k, temp = d["offsets"], case["top"], case["temperature"]
    index = d["teacher_index"].long()
    at = (off[:-1].unsqueeze(1) + index).clamp(0, z.numel() - 1)
    counts = (index >= 0) & (index < (off[1:] - off[:-1]).unsqueeze(1))
    if "mask" in d:
        counts &= d["mask"][at]
    for j in range(1, k):  # of entries that name one row the first counts
        counts[:, j] &= ~((index[:, :j] == index[:, j:j + 1]) & counts[:, :j]).any(1)
    # the student: the listed rows and the rest apart
    listed = torch.zeros(z.numel(), dtype=torch.bool, device=DEV)
    listed[at[counts]] = True
    rest_top, _, rest_e, rest_sum = _plain_softmax(state, torch.where(listed, -math.inf, z))
    has_rest = rest_sum != 0
    zj = torch.where(counts, z[at], -math.inf)
    top = torch.maximum(zj.amax(1), torch.where(has_rest, rest_top, -math.inf))
    top = torch.where(top == -math.inf, 0.0, top)
    xj = (zj - top.unsqueeze(1)) / temp
    rest_x = (rest_top - top) / temp
    rest_part = torch.where(has_rest, torch.exp(rest_x.double()) * rest_sum, 0.0)
    total = torch.exp(xj.double()).sum(1) + rest_part
    # the teacher, in 64 bits: what its list leaves over is small
    t = torch.where(counts, d["teacher_logits"].double(), -math.inf)
    if case["tail"]:
        t_top = torch.zeros(case["sets"], 1, dtype=torch.float64, device=DEV)
    else:
        t = t / temp
        t_top = t.amax(1, keepdim=True)
        t_top = torch.where(t_top == -math.inf, 0.0, t_top)
    mass = torch.exp(t - t_top).sum(1)
    on = (mass != 0) & (total != 0)
    open_ = has_rest & (mass < 1) if case["tail"] else torch.zeros_like(on)
    log_mass = torch.where(open_ | ~on, 0.0, torch.log(mass))
    log_q = t - t_top - log_mass.unsqueeze(1)
    q = torch.exp(log_q)
    rho = torch.where(open_, 1 - mass, 0.0)
    log_total = torch.log(total)
    terms = torch.where(q == 0, 0.0, q * (log_q - (xj.double() - log_total.unsqueeze(1)))).sum(1)
    log_rest = rest_x.double() + torch.log(rest_sum) - log_total
    kl = torch.where(on, terms + torch.where(rho == 0, 0.0, rho * (torch.log(rho) - log_rest)), 0.0)
    w = d["weights"] if "weights" in d else torch.ones(case["sets"], device=DEV)
    loss = temp * temp * (w.double() * kl).sum()
    w = torch.where(on, w * temp, 0.0)
    # p of the rows not listed, less their share of the teacher's rest
    part = torch.where(has_rest & on, w * ((rest_part / total - rho) / rest_sum).float(), 0.0)
    g = rest_e * _to_rows(state, part)
    over = torch.where(on.unsqueeze(1), torch.exp(xj.double()) / total.unsqueeze(1) - q, 0.0)
    g[at[counts]] = (w.unsqueeze(1) * over.float())[counts]
    return (loss.float(), kl.float()) + _plain_grads(state, g)


def _run_plain(state):
    case, d = state["case"], state["in"]
    z = _plain_logits(state)
    if case["op"] == "distill":
        return _plain_distill(state, z)
    top, x, e, total = _plain_softmax(state, z)
    at, counts, lp, entropy, lse, log_total = _plain_report(state, z, top, x, e, total)
    if case["op"] == "report":
        best = _best(z, d["offsets"], case["top"], case["spread"] == "even")
        row = (d["offsets"][:-1].unsqueeze(1) + best).clamp(0, z.numel() - 1)
        best_lp = torch.where(best < 0, -math.inf, x[row] - log_total.unsqueeze(1))
        return lp, entropy, lse, best.to(torch.int32), best_lp
    coef = torch.where(counts, d["grad_log_probs"], 0.0)
    safe = torch.where(total == 0, 1.0, total).float()
    log_p = x - _to_rows(state, log_total)
    slope = -_to_rows(state, coef) - _to_rows(state, d["grad_entropy"]) * (log_p + _to_rows(state, entropy))
    g = torch.where(e == 0, 0.0, e / _to_rows(state, safe) * slope)
    g = g.index_add_(0, at, coef) / case["temperature"]
    return (lp, entropy, lse) + _plain_grads(state, g)


# ------------------------------------------------------------------------------------ the package's
def _run_own(state):
    import packboost_amd as pb

    case, d = state["case"], state["in"]
    how = dict(mask=d.get("mask"), bias=state.get("bias"), temperature=case["temperature"])
    if case["op"] == "distill":
        r = pb.distillation_loss(d["scores"], state["sets"], d["teacher_index"], d["teacher_logits"], tail=case["tail"],
                                 weights=d.get("weights"), **how)
        out = (r.loss, r.kl, r.grad_scores)
        return out if r.grad_table is None else out + (r.grad_table,)
    r = pb.choice_report(d["scores"], state["sets"], chosen=d["chosen"], top=case.get("top", 0), **how)
    out = (r.log_probs, r.entropy, r.lse)
    if case["op"] == "report":
        return out + (r.top_index, r.top_log_probs)
    gs, gt = pb.choice_report_backward(d["grad_log_probs"], d["grad_entropy"], d["scores"], state["sets"],
                                       chosen=d["chosen"], **how)
    return out + ((gs,) if gt is None else (gs, gt))


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------ floors
def work(case):
    n, sets, b, k = case["rows"], case["sets"], TYPES[case["dtype"]].itemsize, case.get("top", 0)
    size = n * (b + (case["mask"] > 0) + 4 * (case["bias"] > 0)) + 8 * sets
    if case["op"] == "report":
        return {"bytes": size + sets * (16 + 8 * k), "flops": 10 * n + 20 * sets}
    size += n * b + 8 * case["bias"]
    if case["op"] == "bonus":
        return {"bytes": size + sets * 24, "flops": 14 * n + 20 * sets}
    entry = 4 + TYPES[case["teacher"]].itemsize
    return {"bytes": size + sets * (4 + 4 * case["weighted"] + k * entry), "flops": 12 * n + sets * (20 + 40 * k)}


# ------------------------------------------------------------------------------------ 64 bits
class _Sets:
    """Sums and maxima over the runs of a table, in NumPy."""

    def __init__(self, off):
        self.off, self.size = off, np.diff(off)
        self.full = np.flatnonzero(self.size)

    def over(self, f, v, empty):
        out = np.full(self.size.size, empty, dtype=np.float64)
        if self.full.size:
            out[self.full] = f.reduceat(v, self.off[:-1][self.full])
        return out

    def rows(self, v):
        return np.repeat(v, self.size)

    def log_sum(self, x):
        """log of the sum of exp(x) over each set, -inf where that is 0."""
        top = self.over(np.maximum, x, -np.inf)
        top[np.isneginf(top)] = 0.0
        with np.errstate(divide="ignore"):
            return top + np.log(self.over(np.add, np.exp(x - self.rows(top)), 0.0))


def _exact_best(sets, z, k):
    """Each set's rows of largest float32 logit, equal ones by index; -1 behind the last."""
    out = np.full((sets.size.size, k), -1, dtype=np.int64)
    live = np.flatnonzero(z != -np.inf)
    seg = sets.rows(np.arange(sets.size.size))[live]
    order = np.lexsort((live, -z[live], seg))
    live, seg = live[order], seg[order]
    place = np.arange(live.size) - np.searchsorted(seg, seg)
    near = place < k
    out[seg[near], place[near]] = live[near] - sets.off[seg[near]]
    return out


def exact(case, seed):
    if case["rows"] > 50_000_000:
        return None
    raw = _inputs(case, seed)
    d = {k: (v.double() if v.is_floating_point() else v).cpu().numpy() for k, v in raw.items()}
    n, temp, sets = case["rows"], case["temperature"], _Sets(d["offsets"])
    on = d.get("mask", np.ones(n, dtype=bool))
    z, ids = d["scores"], None
    with np.errstate(invalid="ignore"):
        if "table" in d:
            half, pos = case["bias"] // 2, d["positions"].astype(np.int64)
            ids = np.array(_bucket_table(half, case["reach"]))[np.minimum(np.abs(pos), case["reach"])] + half * (pos > 0)
            z = z + d["table"][ids]
        z = np.where(on, z, -np.inf)
    x = z / temp
    lse = sets.log_sum(x)
    alive = ~np.isneginf(lse)
    log_p = x - sets.rows(np.where(alive, lse, 0.0))
    p = np.exp(log_p)
    some = p > 0

    def grads(g):
        g = np.where(on, g, 0.0)
        return (g,) if ids is None else (g, np.bincount(ids, g, minlength=case["bias"]))

    if case["op"] != "distill":
        c = d["chosen"].astype(np.int64)
        at = np.clip(sets.off[:-1] + c, 0, n - 1)
        counts = (c >= 0) & (c < sets.size) & alive & on[at]
        lp = np.where(counts, log_p[at], 0.0)
        entropy = -sets.over(np.add, p * np.where(some, log_p, 0.0), 0.0)
        if case["op"] == "report":
            z32 = np.where(on, z, -np.inf).astype(np.float32)  # a bias makes its sum in float32, which orders the rows
            best = _exact_best(sets, z32, case["top"])
            row = np.clip(sets.off[:-1, None] + best, 0, n - 1)
            return lp, entropy, lse, best.astype(np.int32), np.where(best < 0, -np.inf, log_p[row])
        coef = np.where(counts, d["grad_log_probs"], 0.0)
        g = -p * (sets.rows(coef) + sets.rows(d["grad_entropy"]) * (np.where(some, log_p, 0.0) + sets.rows(entropy)))
        g[at[counts]] += coef[counts]
        return (lp, entropy, lse) + grads(g / temp)

    # distillation, entry by entry in a flat list of those that count
    index = d["teacher_index"].astype(np.int64)
    g_of, j_of = np.nonzero((index >= 0) & (index < sets.size[:, None]))
    row = sets.off[g_of] + index[g_of, j_of]
    first = np.zeros(row.size, dtype=bool)
    first[np.unique(row, return_index=True)[1]] = True  # by set, then by place: the first that names a row
    first &= on[row]
    g_of, row, t = g_of[first], row[first], d["teacher_logits"][g_of[first], j_of[first]]
    many = sets.size.size
    if not case["tail"]:
        t = t / temp
    t_top = np.full(many, -np.inf)
    np.maximum.at(t_top, g_of, t)
    t_top = np.where(np.isneginf(t_top) | case["tail"], 0.0, t_top)
    mass = np.bincount(g_of, np.exp(t - t_top[g_of]), minlength=many)
    listed = np.zeros(n, dtype=bool)
    listed[row] = True
    rest = sets.log_sum(np.where(listed, -np.inf, x)) - np.where(alive, lse, 0.0)  # log of the student's rest
    use = (mass > 0) & alive
    left = use & ~np.isneginf(rest) & (mass < 1) & case["tail"]
    with np.errstate(divide="ignore", invalid="ignore"):
        rho = np.where(left, 1 - mass, 0.0)
        log_q = t - t_top[g_of] - np.where(left | ~use, 0.0, np.log(mass))[g_of]
        q = np.where(use[g_of], np.exp(log_q), 0.0)
        kl = np.bincount(g_of, np.where(q > 0, q * (log_q - log_p[row]), 0.0), minlength=many)
        kl += np.where(left, rho * (np.log(rho) - rest), 0.0)
    kl = np.where(use, kl, 0.0)
    w = d.get("weights", np.ones(many))
    share = np.exp(log_p - sets.rows(np.where(np.isneginf(rest), 0.0, rest)))  # of the student's rest
    g = np.where(listed, p, share * sets.rows(np.exp(rest) - rho))
    g[row] -= q
    g = g * sets.rows(np.where(use, w * temp, 0.0))
    return (temp * temp * np.sum(w * kl), kl) + grads(g)
