"""The operators for learning from choices and preferences, case by case, in a plain form and through
the package's entry points.

A case is a dict of plain values. `op` names what a user calls:

  rows        choice_log_probs(scores, sets): every candidate's log-probability within its set
  listwise    the same, and choice_log_probs_backward for soft targets over each list
  steps       choice_log_probs(..., chosen=...) of the taken candidates, and its backward
  preference  preference_loss of pairs of values (a score per row, a reference score per row)
  sequences   preference_loss of pairs of sequences of choices: the steps' log-probabilities, the loss,
              the gradient back to the scores
  policy      policy_loss: the clipped loss with its KL term and the scores' gradient

`spread` says how the rows fall into sets: "even" (all of one size), "ragged" (exponential sizes, empty
sets among them) or "heavy" (lognormal: a few sets hold most rows). `bias` is the number of position
buckets (0: no position bias) and `reach` the distance from which the last bucket is used. `mask` is
the share of candidates left out; what they hold is not meant to be read (NaN, infinities and the
type's lowest value among it), and one set in a hundred is left without any candidate.

`prepare` makes what a user's program holds before the call, `run` makes one pass, `exact` computes the
same in 64 bits on the host.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SETS = dict(dtype="f32", spread="ragged", mask=0.0, bias=0, reach=128)
POLICY = dict(SETS, op="policy", clip_low=0.2, clip_high=0.2, kl=0.05, weighted=False)
PAIRS = dict(beta=0.5, smoothing=0.0, weighted=False)


def listed():
    return [
        # one request: the probabilities of a short list of candidates, where latency counts
        dict(SETS, name="rows_request", op="rows", rows=37, sets=1, spread="even"),
        # a served batch of lists with unavailable items, shown in an order the model has a bias for
        dict(SETS, name="rows_lists", op="rows", rows=200_003, sets=16_000, mask=0.1, bias=32),
        # a few requests over a whole catalogue: long sets, fewer than the chip has compute units
        dict(SETS, name="rows_catalogue", op="rows", rows=5_000_000, sets=24, spread="heavy"),
        # listwise training on graded lists
        dict(SETS, name="listwise", op="listwise", rows=1_000_000, sets=40_000, mask=0.05, bias=32),
        # clicks on lists of the panel's size, with the position bias learned beside the scores
        dict(SETS, name="steps_clicks", op="steps", rows=2_400_000, sets=100_003, mask=0.02, bias=64, reach=200),
        # one choice out of a large fixed inventory per step, scores kept in bf16
        dict(SETS, name="steps_inventory", op="steps", rows=4096 * 32_000, sets=4096, spread="even", dtype="bf16"),
        # preferred rows in a table of the usual size: a first reward model
        dict(PAIRS, name="preference_small", op="preference", values=10_000, pairs=5_000),
        # many comparisons of the same rows, some rows in very many of them, noisy labels
        dict(PAIRS, name="preference_hubs", op="preference", values=1_000_000, pairs=5_000_003, smoothing=0.1,
             weighted=True),
        # sequences of choices, pairs of which were compared
        dict({**SETS, **PAIRS}, name="sequences", op="sequences", rows=6_000_000, sets=300_000, seqs=4_001, pairs=6_000,
             beta=0.1, mask=0.05),
        # a policy step on a handful of decisions, where latency counts
        dict(POLICY, name="policy_small", rows=1_500, sets=200),
        # a policy over the panel's rows, a few candidates a decision
        dict(POLICY, name="policy_panel", rows=2_400_000, sets=480_000, mask=0.1, bias=32, clip_high=0.28),
        # a large rollout of uneven decisions, from one candidate to many thousands, scores kept in bf16
        dict(POLICY, name="policy_rollout", rows=40_000_003, sets=100_000, spread="heavy", dtype="bf16", weighted=True),
    ]


# ------------------------------------------------------------------------------------ drawn cases
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rows", "listwise", "steps", "steps", "preference", "preference", "sequences", "policy", "policy"])
    if op == "preference":
        n = _log(rng, 50, 2_000_000)
        return dict(PAIRS, op=op, values=n, pairs=_log(rng, 20, 4_000_000), beta=rng.choice([0.1, 0.5, 1.0]),
                    smoothing=rng.choice([0.0, 0.1]), weighted=rng.random() < 0.5)
    kind = rng.choice(["short", "short", "long", "even"])
    c = dict(SETS, op=op, dtype=rng.choice(["f32", "f32", "bf16", "f16"]), mask=rng.choice([0.0, 0.0, 0.1, 0.5]),
             bias=rng.choice([0, 0, 16, 32, 64]), reach=rng.choice([64, 128, 500]))
    if kind == "short":
        c.update(rows=_log(rng, 100, 20_000_000))
        c.update(sets=max(1, c["rows"] // _log(rng, 2, 60)), spread=rng.choice(["ragged", "heavy"]))
    elif kind == "long":
        c.update(rows=_log(rng, 5_000, 20_000_000))
        c.update(sets=max(1, c["rows"] // _log(rng, 500, 200_000)), spread=rng.choice(["ragged", "heavy"]))
    else:
        size = _log(rng, 1, 60_000)
        c.update(sets=_log(rng, 1, max(1, 20_000_000 // size)), spread="even")
        c.update(rows=size * c["sets"])
    if op == "sequences":
        c = dict(c, **PAIRS)
        c.update(seqs=_log(rng, 2, max(2, c["sets"])), beta=rng.choice([0.05, 0.1, 0.5]), weighted=rng.random() < 0.5)
        c.update(pairs=_log(rng, 1, 4 * c["seqs"]), smoothing=rng.choice([0.0, 0.1]))
    if op == "policy":
        c = dict(POLICY, **c)
        c.update(kl=rng.choice([0.0, 0.05]), clip_high=rng.choice([0.2, 0.28]), weighted=rng.random() < 0.5)
    return c


# ------------------------------------------------------------------------------------ inputs
def _generator(case, seed):
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


def _draw_pairs(n, pairs, g):
    """Winners and losers among n values, low indices far more often than high ones."""
    w = torch.floor(_uniform(pairs, g) ** 3 * n).to(torch.int64).clamp_(max=n - 1)
    step = 1 + torch.floor(_uniform(pairs, g) * (n - 1)).to(torch.int64).clamp_(max=max(0, n - 2))
    return w, (w + step) % n


def _spread_over(v, off, n):
    """v[set of row i] for every row."""
    return torch.repeat_interleave(v, off[1:] - off[:-1], output_size=n)


def _double_log_prob(x, off, at):
    """Log-probabilities, in 64 bits, of rows `at` (one a set); rows of no use are finite."""
    n, sets = x.numel(), off.numel() - 1
    x = x.double()
    size = off[1:] - off[:-1]
    if n and n == sets * int(size[0]) and bool((size == size[0]).all()):
        lse = torch.logsumexp(x.view(sets, -1), 1)
    else:
        seg = _spread_over(torch.arange(sets, device=DEV), off, n)
        top = torch.full((sets,), -math.inf, device=DEV, dtype=torch.float64).scatter_reduce_(0, seg, x, "amax")
        top = torch.where(torch.isinf(top), 0.0, top)
        lse = top + torch.log(torch.zeros(sets, device=DEV, dtype=torch.float64).index_add_(
            0, seg, torch.exp(x - top[seg])))
    return torch.nan_to_num(x[at.clamp(0, n - 1)] - lse, nan=-1.0, posinf=-1.0, neginf=-1.0)


def _inputs(case, seed):
    """What the program holds, on the GPU, from the seed alone."""
    g = _generator(case, seed)
    d = {}
    if case["op"] == "preference":
        n = case["values"]
        d["winners"], d["losers"] = _draw_pairs(n, case["pairs"], g)
        d["values"] = 2.0 * torch.randn(n, device=DEV, generator=g)
        d["ref"] = d["values"] + torch.randn(n, device=DEV, generator=g)
    else:
        n, sets = case["rows"], case["sets"]
        off = d["offsets"] = _offsets(n, sets, case["spread"], g)
        size = off[1:] - off[:-1]
        d["chosen"] = torch.floor(_uniform(sets, g) * size).to(torch.int32)
        d["chosen"][_uniform(sets, g) < 0.05] = -1
        base = 2.0 * torch.randn(n, device=DEV, generator=g)
        at = off[:-1] + d["chosen"].clamp_min(0)
        if case["mask"] > 0:
            keep = torch.rand(n, device=DEV, generator=g) >= case["mask"]
            keep[at.clamp(max=n - 1)] = True  # what was taken was on offer
            none = _uniform(sets, g) < 0.01
            keep &= ~_spread_over(none, off, n)
            d["mask"] = keep
            junk = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(TYPES[case["dtype"]]).min], device=DEV)
            idle = torch.nonzero(~keep).reshape(-1)
            base[idle] = junk[idle % 4]
        d["scores"] = base.to(TYPES[case["dtype"]])
        total = d["scores"].float()
        if case["bias"]:
            local = torch.arange(n, device=DEV) - _spread_over(off[:-1], off, n)
            origin = torch.floor(_uniform(sets, g) * size).to(torch.int64)
            d["positions"] = (local - _spread_over(origin, off, n)).to(torch.int32)
            d["table"] = 0.5 * torch.randn(case["bias"], device=DEV, generator=g)
            total = total + d["table"][_bucket_ids(d["positions"], case["bias"], case["reach"])]
        if case["mask"] > 0:
            total = torch.where(d["mask"], total, -math.inf)
        if case["op"] == "listwise":  # graded lists: the target is a distribution over each list
            t = torch.rand(n, device=DEV, generator=g)
            if case["mask"] > 0:
                t = torch.where(d["mask"], t, 0.0)
            t = t / _spread_over((size + 1).float(), off, n)
            d["grad"] = -t
        elif case["op"] == "steps":
            d["grad"] = -torch.rand(sets, device=DEV, generator=g)
        elif case["op"] == "sequences":
            d["seq_offsets"] = _offsets(sets, case["seqs"], "ragged", g)
            d["winners"], d["losers"] = _draw_pairs(case["seqs"], case["pairs"], g)
            lp = _double_log_prob(total, off, at)
            ref = lp + 0.3 * torch.randn(sets, device=DEV, generator=g)
            taken = (d["chosen"] >= 0) & (size > 0)  # the reference model leaves out the same steps
            if case["mask"] > 0:
                taken &= d["mask"][at.clamp(max=n - 1)]
            d["ref"] = torch.where(taken, ref, 0.0).float()
        elif case["op"] == "policy":
            lp = _double_log_prob(total, off, at)
            old = lp + 0.25 * torch.randn(sets, device=DEV, generator=g)
            # the loss has a kink where the ratio meets its bounds; ratios stay a rounding away from it
            for edge in (math.log1p(case["clip_high"]), math.log1p(-case["clip_low"])):
                old = torch.where((lp - old - edge).abs() < 1e-4, old - 4e-4, old)
            d["old"] = old.float()
            d["ref"] = (old + 0.1 * torch.randn(sets, device=DEV, generator=g)).float()
            d["advantages"] = torch.randn(sets, device=DEV, generator=g)
            if case["weighted"]:
                d["weights"] = torch.rand(sets, device=DEV, generator=g)
    if "winners" in d and case["weighted"]:
        d["weights"] = torch.rand(case["pairs"], device=DEV, generator=g)
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
        from packboost_amd import ChoiceSets, PositionBias, PositionBuckets, PreferencePairs

        if "offsets" in d:
            state["sets"] = ChoiceSets(d["offsets"])
        if "winners" in d:
            state["pairs"] = PreferencePairs(d["winners"], d["losers"], num_values=case.get("values"),
                                             offsets=d.get("seq_offsets"))
        if "table" in d:
            state["bias"] = PositionBias(d["table"], d["positions"],
                                         PositionBuckets(case["bias"], case["reach"], bidirectional=True))
    else:
        if "offsets" in d and case["spread"] != "even":
            state["seg"] = _spread_over(torch.arange(case["sets"], device=DEV), d["offsets"], case["rows"])
        if "seq_offsets" in d:
            state["seq"] = _spread_over(torch.arange(case["seqs"], device=DEV), d["seq_offsets"], case["sets"])
        if "table" in d:
            _bucket_ids(d["positions"][:1], case["bias"], case["reach"])
    return state


# ------------------------------------------------------------------------------------ plain form
def _set_sum(state, v):
    if "seg" not in state:
        return v.view(state["case"]["sets"], -1).sum(1)
    return torch.segment_reduce(v, "sum", offsets=state["in"]["offsets"], initial=0.0, unsafe=True)


def _set_max(state, v):
    if "seg" not in state:
        return v.view(state["case"]["sets"], -1).amax(1)
    return torch.segment_reduce(v, "max", offsets=state["in"]["offsets"], initial=-math.inf, unsafe=True)


def _to_rows(state, v):
    if "seg" not in state:
        return v.view(-1, 1).expand(-1, state["case"]["rows"] // state["case"]["sets"]).reshape(-1)
    return v[state["seg"]]


def _plain_softmax(state):
    """x, the sets' log of the sum of exponentials, and that sum relative to its largest term."""
    case, d = state["case"], state["in"]
    x = d["scores"].float()
    if "table" in d:
        x = x + d["table"][_bucket_ids(d["positions"], case["bias"], case["reach"])]
    if "mask" in d:
        x = torch.where(d["mask"], x, -math.inf)
    top = _set_max(state, x)
    top = torch.where(top == -math.inf, 0.0, top)
    total = _set_sum(state, torch.exp(x - _to_rows(state, top)))
    return x, top + torch.log(total), total


def _plain_steps(state, x, lse, total):
    """Rows taken, whether the step counts, and its log-probability."""
    d = state["in"]
    off, c = d["offsets"], d["chosen"].long()
    counts = (c >= 0) & (c < off[1:] - off[:-1]) & (total != 0)
    at = (off[:-1] + c).clamp(0, x.numel() - 1)
    if "mask" in d:
        counts &= d["mask"][at]
    return at, counts, torch.where(counts, x[at] - lse, 0.0)


def _plain_back(state, x, lse, total, at, counts, dstep):
    """Gradients of the scores and the table from those of the steps' log-probabilities."""
    d = state["in"]
    coef = torch.where(counts, dstep, 0.0)
    p = torch.exp(x - _to_rows(state, torch.where(total == 0, 0.0, lse)))
    g = -p * _to_rows(state, coef)
    g = g.index_add_(0, at, coef)
    return _plain_grads(state, g)


def _plain_grads(state, g):
    case, d = state["case"], state["in"]
    if "mask" in d:
        g = torch.where(d["mask"], g, 0.0)
    out = (g.to(d["scores"].dtype),)
    if "table" in d:
        ids = _bucket_ids(d["positions"], case["bias"], case["reach"])
        out += (torch.stack([torch.where(ids == b, g, 0.0).sum() for b in range(case["bias"])]),)
    return out


def _plain_preference(state, a):
    """Loss, gradient of the paired values and margins."""
    case, d = state["case"], state["in"]
    z = case["beta"] * (a[d["winners"]] - a[d["losers"]])
    w = d["weights"] if "weights" in d else torch.ones_like(z)
    soft = torch.log1p(torch.exp(-z.abs()))
    e = case["smoothing"]
    loss = (w * ((1 - e) * (soft + torch.clamp(-z, min=0)) + e * (soft + torch.clamp(z, min=0)))).sum()
    dz = case["beta"] * w * (1 / (1 + torch.exp(-z)) - (1 - e))
    grad = torch.zeros_like(a).index_add_(0, d["winners"], dz).index_add_(0, d["losers"], -dz)
    return loss, grad, z


def _run_plain(state):
    case, d = state["case"], state["in"]
    op = case["op"]
    if op == "preference":
        return _plain_preference(state, d["values"] - d["ref"])
    x, lse, total = _plain_softmax(state)
    if op in ("rows", "listwise"):
        lp = torch.where(x == -math.inf, -math.inf, x - _to_rows(state, lse))
        if op == "rows":
            return lp, lse
        p = torch.exp(x - _to_rows(state, torch.where(total == 0, 0.0, lse)))
        g = d["grad"] if "mask" not in d else torch.where(d["mask"], d["grad"], 0.0)
        return (lp, lse) + _plain_grads(state, g - p * _to_rows(state, _set_sum(state, g)))
    at, counts, lp = _plain_steps(state, x, lse, total)
    if op == "steps":
        return (lp, lse) + _plain_back(state, x, lse, total, at, counts, d["grad"])
    if op == "sequences":
        a = torch.zeros(case["seqs"], device=DEV).index_add_(0, state["seq"], lp - d["ref"])
        loss, grad, z = _plain_preference(state, a)
        return (loss, z, lp) + _plain_back(state, x, lse, total, at, counts, grad[state["seq"]])
    adv, old, ref = d["advantages"], d["old"], d["ref"]
    w = d["weights"] if "weights" in d else torch.ones_like(adv)
    w = torch.where(counts, w, 0.0)
    ratio = torch.exp(lp - old)
    free = ratio * adv
    held = torch.clamp(ratio, 1 - case["clip_low"], 1 + case["clip_high"]) * adv
    gap = torch.exp(ref - lp)
    kl = gap - (ref - lp) - 1
    loss = (w * (case["kl"] * kl - torch.minimum(free, held))).sum()
    dlp = w * (torch.where(free <= held, -free, 0.0) + case["kl"] * (1 - gap))
    return (loss, lp, (w * kl).sum(), (w * (free > held)).sum()) + _plain_back(state, x, lse, total, at, counts, dlp)


# ------------------------------------------------------------------------------------ the package's
def _run_own(state):
    import packboost_amd as pb

    case, d = state["case"], state["in"]
    op = case["op"]
    if op == "preference":
        r = pb.preference_loss(d["values"], state["pairs"], ref_values=d["ref"], weights=d.get("weights"),
                               beta=case["beta"], label_smoothing=case["smoothing"])
        return r.loss, r.grad, r.margins
    how = dict(mask=d.get("mask"), bias=state.get("bias"))
    if op == "policy":
        r = pb.policy_loss(d["scores"], state["sets"], d["chosen"], d["advantages"], d["old"], ref_log_probs=d["ref"],
                           weights=d.get("weights"), clip=(case["clip_low"], case["clip_high"]), kl_weight=case["kl"],
                           **how)
        out = (r.loss, r.log_probs, r.kl, r.clipped, r.grad_scores)
        return out if r.grad_table is None else out + (r.grad_table,)
    if op != "rows" and op != "listwise":
        how["chosen"] = d["chosen"]
    lp, lse = pb.choice_log_probs(d["scores"], state["sets"], **how)
    if op == "rows":
        return lp, lse
    out, grad = (lp, lse), d.get("grad")
    if op == "sequences":
        r = pb.preference_loss(lp, state["pairs"], ref_values=d["ref"], weights=d.get("weights"), beta=case["beta"],
                               label_smoothing=case["smoothing"])
        out, grad = (r.loss, r.margins, lp), r.grad
    ds, dt = pb.choice_log_probs_backward(grad, d["scores"], lse, state["sets"], **how)
    return out + ((ds,) if dt is None else (ds, dt))


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------ floors
def work(case):
    if case["op"] == "preference":
        n, p = case["values"], case["pairs"]
        return {"bytes": 12 * n + p * (12 + 4 * case["weighted"]), "flops": 3 * n + 20 * p}
    n, sets, b = case["rows"], case["sets"], TYPES[case["dtype"]].itemsize
    scores = n * (b + (case["mask"] > 0) + 4 * (case["bias"] > 0))
    back = n * b + 4 * case["bias"]
    ops = {"rows": 8, "listwise": 14, "steps": 12, "sequences": 12, "policy": 12}[case["op"]]
    if case["op"] == "rows":
        size = scores + 4 * n + 12 * sets
    elif case["op"] == "listwise":
        size = scores + 8 * n + 12 * sets + back
    elif case["op"] == "steps":
        size = scores + 24 * sets + back
    elif case["op"] == "sequences":
        size = scores + 20 * sets + 8 * case["seqs"] + case["pairs"] * (12 + 4 * case["weighted"]) + back
    else:
        size = scores + sets * (28 + 4 * case["weighted"]) + back
    return {"bytes": size, "flops": ops * n + 20 * sets}


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


def _exact_preference(case, d, a):
    w, l = d["winners"], d["losers"]
    z = case["beta"] * (a[w] - a[l])
    e, weight = case["smoothing"], d.get("weights", np.ones(z.size))
    loss = np.sum(weight * ((1 - e) * np.logaddexp(0.0, -z) + e * np.logaddexp(0.0, z)))
    dz = case["beta"] * weight * (np.exp(-np.logaddexp(0.0, -z)) - 1 + e)
    grad = np.bincount(w, dz, minlength=a.size) - np.bincount(l, dz, minlength=a.size)
    return loss, grad, z


def exact(case, seed):
    if case.get("rows", 0) > 50_000_000:
        return None
    d = {k: (v.double() if v.is_floating_point() else v).cpu().numpy() for k, v in _inputs(case, seed).items()}
    op = case["op"]
    if op == "preference":
        return _exact_preference(case, d, d["values"] - d["ref"])
    sets, chosen = _Sets(d["offsets"]), d["chosen"].astype(np.int64)
    on = d.get("mask", np.ones(case["rows"], dtype=bool))
    x = np.where(on, d["scores"], -np.inf)
    ids = None
    if "table" in d:
        half, q = case["bias"] // 2, d["positions"].astype(np.int64)
        ids = np.array(_bucket_table(half, case["reach"]))[np.minimum(np.abs(q), case["reach"])] + half * (q > 0)
        x = np.where(on, x + d["table"][ids], -np.inf)
    top = sets.over(np.maximum, x, -np.inf)
    top[np.isneginf(top)] = 0.0
    e = np.exp(x - sets.rows(top))
    total = sets.over(np.add, e, 0.0)
    p = e / sets.rows(np.where(total == 0, 1.0, total))
    with np.errstate(divide="ignore"):
        lse = top + np.log(total)
        row_lp = np.where(np.isneginf(x), -np.inf, x - sets.rows(np.where(total == 0, 0.0, lse)))

    def grads(g):
        g = np.where(on, g, 0.0)
        return (g,) if ids is None else (g, np.bincount(ids, g, minlength=case["bias"]))

    if op == "rows":
        return row_lp, lse
    if op == "listwise":
        g = np.where(on, d["grad"], 0.0)
        return (row_lp, lse) + grads(g - p * sets.rows(sets.over(np.add, g, 0.0)))
    at = np.clip(sets.off[:-1] + chosen, 0, case["rows"] - 1)
    counts = (chosen >= 0) & (chosen < sets.size) & (total > 0) & on[at]
    lp = np.where(counts, row_lp[at], 0.0)

    def back(dstep):
        coef = np.where(counts, dstep, 0.0)
        g = -p * sets.rows(coef)
        g[at[counts]] += coef[counts]
        return grads(g)

    if op == "steps":
        return (lp, lse) + back(d["grad"])
    if op == "sequences":
        seqs = _Sets(d["seq_offsets"])
        a = seqs.over(np.add, lp - d["ref"], 0.0)
        loss, grad, z = _exact_preference(case, d, a)
        return (loss, z, lp) + back(seqs.rows(grad))
    adv, w = d["advantages"], np.where(counts, d.get("weights", 1.0), 0.0)
    ratio, gap = np.exp(lp - d["old"]), np.exp(d["ref"] - lp)
    free, held = ratio * adv, np.clip(ratio, 1 - case["clip_low"], 1 + case["clip_high"]) * adv
    kl = gap - (d["ref"] - lp) - 1
    dlp = w * (np.where(free <= held, -free, 0.0) + case["kl"] * (1 - gap))
    return (np.sum(w * (case["kl"] * kl - np.minimum(free, held))), lp, np.sum(w * kl),
            np.sum(w * (free > held))) + back(dlp)
