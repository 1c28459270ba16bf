"""Choices and preferences on the GPU against the formulas in 64 bits.

Tolerances. A set's sum of exponentials is a sum of positive float32 terms in which any term passes
through at most 32 additions of a lane, 6 of a wave, 4 of a workgroup and, per 2048 rows of a longer
set, as many again; expf and logf are good to 2 units. The logit's own roundings (the bias, the
difference to the maximum) are at most half a unit of the largest logit each. So a log-probability is
within LP = 2^-24 * (4 max|x| + 100) of the formula's, and a probability within LP of itself. A gradient
c ([i = chosen] - p) is then within |c| (LP + 2^-22), plus the rounding to the scores' type; the table's
within the sum of its rows' bounds plus 2^-31 of the largest gradient a row, plus its own rounding."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": (torch.float32, 2.0 ** -24, 0.0), "bf16": (torch.bfloat16, 2.0 ** -8, 0.0),
         "f16": (torch.float16, 2.0 ** -11, 2.0 ** -25)}
DEV = "cuda"

rs = np.random.RandomState(7)
LAYOUTS = {
    "one_row": [1],
    "one_set": [37],
    "no_rows": [0, 0, 0],
    "singles": [1] * 700,
    "empties": [0, 3, 0, 0, 5, 1, 0, 64, 0],
    "many_empty": [0] * 2500 + [2] + [0] * 1030,
    "small": list(rs.randint(0, 9, 1001)),
    "wave": [63, 64, 65, 127, 128, 129, 255, 256, 257],
    "tile_edges": [511, 512, 513, 1, 2047, 2048, 2049, 4096, 4097],
    "mixed": [1, 2, 512, 1, 1, 3, 512, 0, 900, 2, 7, 1500, 4, 0, 2500, 1],
    "long": [100_001],
    "long_pair": [5_000, 0, 70_000, 3],
}


def offsets_of(sizes):
    return np.concatenate([[0], np.cumsum(np.asarray(sizes, dtype=np.int64))]).astype(np.int64)


def make(sizes, dtype="f32", masked=False, biased=False, seed=0, buckets=32, reach=64):
    """Device inputs and their float64 copies."""
    from packboost_amd import ChoiceSets, PositionBias, PositionBuckets

    r = np.random.default_rng(seed)
    off = offsets_of(sizes)
    n, g = int(off[-1]), len(sizes)
    size = np.diff(off)
    scores = torch.from_numpy((2.5 * r.standard_normal(n)).astype(np.float32)).to(TYPES[dtype][0])
    chosen = np.floor(r.random(g) * size).astype(np.int32)
    chosen[r.random(g) < 0.1] = -1
    if g > 4:
        chosen[1], chosen[3] = size[1], 2 ** 31 - 1  # outside their sets
    keep = None
    if masked:
        keep = r.random(n) > 0.25
        keep &= ~np.repeat(r.random(g) < 0.1, size)  # sets without any candidate
        junk = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(scores.dtype).min])
        idle = np.flatnonzero(~keep)
        scores[torch.from_numpy(idle)] = junk[torch.from_numpy(idle % 4)].to(scores.dtype)
    d = {"off": off, "size": size, "sets": ChoiceSets(off), "scores": scores.to(DEV),
         "chosen": torch.from_numpy(chosen).to(DEV), "c": chosen.astype(np.int64), "r": r,
         "keep": np.ones(n, bool) if keep is None else keep,
         "mask": None if keep is None else torch.from_numpy(keep).to(DEV), "bias": None, "dtype": dtype}
    x = scores.double().numpy()
    if biased:
        origin = np.floor(r.random(g) * size).astype(np.int64)
        pos = (np.arange(n) - np.repeat(off[:-1] + origin, size)).astype(np.int32)
        table = r.standard_normal(buckets).astype(np.float32)
        pb = PositionBuckets(buckets, reach)
        d["ids"] = pb(pos).astype(np.int64)
        d["bias"] = PositionBias(torch.from_numpy(table).to(DEV), torch.from_numpy(pos).to(DEV), pb)
        x = x + table.astype(np.float64)[d["ids"]]
    d["x"] = np.where(d["keep"], x, -np.inf)
    return d


def per_set(d, f, v, empty):
    out = np.full(len(d["size"]), empty, dtype=np.float64)
    full = np.flatnonzero(d["size"])
    if full.size:
        out[full] = f.reduceat(v, d["off"][:-1][full])
    return out


def reference(d):
    """p, row log-probabilities, lse, steps that count, their log-probabilities and rows."""
    x, size = d["x"], d["size"]
    top = per_set(d, np.maximum, x, -np.inf)
    top = np.where(np.isneginf(top), 0.0, top)
    e = np.exp(x - np.repeat(top, size))
    s = per_set(d, np.add, e, 0.0)
    p = e / np.repeat(np.where(s == 0, 1.0, s), size)
    with np.errstate(divide="ignore"):
        lse = top + np.log(s)
    lp = np.where(np.isneginf(x), -np.inf, x - np.repeat(np.where(s == 0, 0.0, lse), size))
    ok = (d["c"] >= 0) & (d["c"] < size) & (s > 0)
    at = np.where(ok, d["off"][:-1] + d["c"], 0)
    if len(x):
        ok &= d["keep"][at]
        step = np.where(ok, lp[at], 0.0)
    else:
        step = np.zeros(len(size))
    return p, lp, lse, ok, step, at


def bound_lp(d):
    live = d["x"][np.isfinite(d["x"])]
    return U * (4 * (np.abs(live).max() if live.size else 0.0) + 100)


def back(d, p, ok, at, dstep):
    coef = np.where(ok, dstep, 0.0)
    g = -p * np.repeat(coef, d["size"])
    g[at[ok]] += coef[ok]
    size = np.abs(np.repeat(coef, d["size"])) * np.where(d["keep"], p, 0.0)
    size[at[ok]] += np.abs(coef[ok])
    return np.where(d["keep"], g, 0.0), size


def check_grads(d, got, table, g, size, lp_tol):
    """size: sum of the absolute terms of each row's gradient."""
    _, unit, tiny = TYPES[d["dtype"]]
    got = got.double().cpu().numpy()
    room = size * (lp_tol + 4 * U)
    assert np.all(np.abs(got - g) <= room + unit * np.abs(g) * 1.01 + unit * room + tiny)
    assert np.all(got[~d["keep"]] == 0)
    if d["bias"] is None:
        assert table is None
        return
    nb = d["bias"].buckets.num_buckets
    want = np.bincount(d["ids"], g, minlength=nb)
    count = np.bincount(d["ids"], minlength=nb)
    big = np.abs(g).max() if g.size else 0.0
    room = np.bincount(d["ids"], room, minlength=nb) + count * big * 2.0 ** -30 + 2 * U * np.abs(want)
    assert np.all(np.abs(table.double().cpu().numpy() - want) <= room)


def same_or_close(got, want, tol):
    got = got.double().cpu().numpy()
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf])
    assert np.all(np.abs(got[~inf] - want[~inf]) <= tol)


VARIANTS = [("f32", False, False), ("f32", True, True), ("bf16", True, False), ("f16", False, True)]


@pytest.mark.parametrize("dtype,masked,biased", VARIANTS)
@pytest.mark.parametrize("layout", list(LAYOUTS))
def test_rows(hip, layout, dtype, masked, biased):
    from packboost_amd import choice_log_probs, choice_log_probs_backward

    d = make(LAYOUTS[layout], dtype, masked, biased)
    kw = dict(mask=d["mask"], bias=d["bias"])
    p, lp, lse, *_ = reference(d)
    tol = bound_lp(d)
    got, got_lse = choice_log_probs(d["scores"], d["sets"], **kw)
    same_or_close(got, lp, tol)
    same_or_close(got_lse, lse, tol)
    up = d["r"].standard_normal(len(lp)).astype(np.float32)
    up_dev = torch.from_numpy(np.where(d["keep"], up, np.nan).astype(np.float32)).to(DEV)
    gs, gt = choice_log_probs_backward(up_dev, d["scores"], got_lse, d["sets"], **kw)
    u = np.where(d["keep"], up.astype(np.float64), 0.0)
    total = np.repeat(per_set(d, np.add, u, 0.0), d["size"])
    absolute = np.repeat(per_set(d, np.add, np.abs(u), 0.0), d["size"])
    # the set's sum of gradients is a float32 sum of at most 100 levels of roundings
    check_grads(d, gs, gt, np.where(d["keep"], u - p * total, 0.0), np.abs(u) + p * absolute * (1 + 100 * U / (tol + 4 * U)), tol)


@pytest.mark.parametrize("dtype,masked,biased", VARIANTS)
@pytest.mark.parametrize("layout", list(LAYOUTS))
def test_steps(hip, layout, dtype, masked, biased):
    from packboost_amd import choice_log_probs, choice_log_probs_backward

    d = make(LAYOUTS[layout], dtype, masked, biased, seed=1)
    kw = dict(chosen=d["chosen"], mask=d["mask"], bias=d["bias"])
    p, _, lse, ok, step, at = reference(d)
    tol = bound_lp(d)
    got, got_lse = choice_log_probs(d["scores"], d["sets"], **kw)
    same_or_close(got, step, tol)
    same_or_close(got_lse, lse, tol)
    up = d["r"].standard_normal(len(step)).astype(np.float32)
    gs, gt = choice_log_probs_backward(torch.from_numpy(up).to(DEV), d["scores"], got_lse, d["sets"], **kw)
    g, size = back(d, p, ok, at, up.astype(np.float64))
    check_grads(d, gs, gt, g, size, tol)


def policy_inputs(d, step, weighted=True, ref=True):
    r, g = d["r"], len(step)
    low, high, kw = 0.2, 0.28, 0.07
    old = step + 0.3 * r.standard_normal(g)
    for edge in (math.log1p(high), math.log1p(-low)):  # ratios a rounding away from their bounds
        old = np.where(np.abs(step - old - edge) < 1e-3, old - 4e-3, old)
    v = {"advantages": r.standard_normal(g), "old_log_probs": old}
    if ref:
        v["ref_log_probs"] = old + 0.2 * r.standard_normal(g)
    if weighted:
        v["weights"] = r.random(g)
    v = {k: a.astype(np.float32) for k, a in v.items()}
    return v, low, high, kw


def policy_reference(v, ok, step, low, high, kw, scale):
    a, old = v["advantages"].astype(np.float64), v["old_log_probs"].astype(np.float64)
    w = np.where(ok, v.get("weights", np.ones(1)).astype(np.float64), 0.0) * scale
    ratio = np.exp(step - old)
    free, held = ratio * a, np.clip(ratio, 1 - low, 1 + high) * a
    kl, slope = np.zeros_like(a), np.where(free <= held, -free, 0.0)
    if "ref_log_probs" in v:
        gap = v["ref_log_probs"].astype(np.float64) - step
        kl = np.exp(gap) - gap - 1
        slope = slope + kw * (1 - np.exp(gap))
    loss = w * (kw * kl - np.minimum(free, held))
    return loss, w * kl, w * (free > held), w * slope, w


@pytest.mark.parametrize("dtype,masked,biased", VARIANTS)
@pytest.mark.parametrize("layout", list(LAYOUTS))
def test_policy(hip, layout, dtype, masked, biased):
    from packboost_amd import policy_loss

    d = make(LAYOUTS[layout], dtype, masked, biased, seed=2)
    p, _, _, ok, step, at = reference(d)
    tol = bound_lp(d)
    v, low, high, kw = policy_inputs(d, step, weighted=dtype != "bf16", ref=dtype != "f16")
    dev = {k: torch.from_numpy(a).to(DEV) for k, a in v.items()}
    scale = 0.5
    r = policy_loss(d["scores"], d["sets"], d["chosen"], **dev, mask=d["mask"], bias=d["bias"], clip=(low, high),
                    kl_weight=kw, scale=scale)
    loss, kl, clipped, slope, w = policy_reference(v, ok, step, low, high, kw, scale)
    same_or_close(r.log_probs, step, tol)
    # a step's terms move by at most (ratio |A| + kw |1 - e^d|) w per unit of log p; their own few float32
    # roundings are 16 units of their size
    ratio = np.exp(step - v["old_log_probs"])
    gap = np.exp(v["ref_log_probs"] - step) if "ref_log_probs" in v else np.zeros_like(step)
    term = w * (ratio * np.abs(v["advantages"]) + (kw * (gap + 1 + np.abs(np.log(np.where(gap > 0, gap, 1)))) if kw else 0))
    room = (tol + 16 * U) * term
    assert abs(float(r.loss) - loss.sum()) <= room.sum() + U * abs(loss.sum())
    kl_room = (tol + 16 * U) * w * (gap + 1 + np.abs(np.log(np.where(gap > 0, gap, 1))))
    assert abs(float(r.kl) - kl.sum()) <= kl_room.sum() + U * abs(kl.sum())
    assert abs(float(r.clipped) - clipped.sum()) <= 4 * U * (1 + clipped.sum())
    g, size = back(d, p, ok, at, slope)
    _, extra = back(d, p, ok, at, room)
    check_grads(d, r.grad_scores, r.grad_table, g, size + extra / (tol + 4 * U), tol)


def test_policy_without_old_names(hip):
    """weights, reference and position bias are optional, and their absence is weight 1 and no KL term."""
    from packboost_amd import policy_loss

    d = make(LAYOUTS["mixed"], seed=3)
    _, _, _, ok, step, _ = reference(d)
    v, low, high, _ = policy_inputs(d, step, weighted=False, ref=False)
    dev = {k: torch.from_numpy(a).to(DEV) for k, a in v.items()}
    plain = policy_loss(d["scores"], d["sets"], d["chosen"], **dev, clip=(low, high))
    ones = policy_loss(d["scores"], d["sets"], d["chosen"], **dev, clip=(low, high), kl_weight=0.0,
                       weights=torch.ones(len(step), device=DEV), ref_log_probs=dev["old_log_probs"])
    assert float(plain.kl) == 0.0 and float(ones.kl) >= 0.0
    assert float(plain.loss) == float(ones.loss)
    assert torch.equal(plain.grad_scores, ones.grad_scores)


def pref_reference(a, w, l, weight, beta, e, scale):
    z = beta * (a[w] - a[l])
    loss = scale * np.sum(weight * ((1 - e) * np.logaddexp(0, -z) + e * np.logaddexp(0, z)))
    dz = scale * beta * weight * (np.exp(-np.logaddexp(0, -z)) - 1 + e)
    grad = np.bincount(w, dz, minlength=a.size) - np.bincount(l, dz, minlength=a.size)
    absolute = np.bincount(w, scale * beta * weight, minlength=a.size) + np.bincount(l, scale * beta * weight, minlength=a.size)
    return z, loss, grad, absolute


@pytest.mark.parametrize("values,pairs,hub", [(1, 0, 0), (2, 1, 0), (50, 300, 0), (1000, 1, 0), (5000, 20_000, 1),
                                              (3, 9_000, 0), (100_000, 60_001, 0)])
@pytest.mark.parametrize("smoothing,weighted,ref", [(0.0, False, True), (0.2, True, False)])
def test_preference_values(hip, values, pairs, hub, smoothing, weighted, ref):
    from packboost_amd import PreferencePairs, preference_loss

    r = np.random.default_rng(values + pairs)
    w = r.integers(0, values, pairs)
    if hub:
        w[r.random(pairs) < 0.4] = 7  # one value in thousands of pairs
    l = (w + 1 + r.integers(0, max(1, values - 1), pairs)) % values
    v = (3 * r.standard_normal(values)).astype(np.float32)
    rv = (v + r.standard_normal(values)).astype(np.float32) if ref else np.zeros(values, np.float32)
    weight = r.random(pairs).astype(np.float32) if weighted else np.ones(pairs, np.float32)
    beta, scale = 0.7, 2.0
    out = preference_loss(torch.from_numpy(v).to(DEV), PreferencePairs(w, l, num_values=values),
                          ref_values=torch.from_numpy(rv).to(DEV) if ref else None,
                          weights=torch.from_numpy(weight).to(DEV) if weighted else None, beta=beta,
                          label_smoothing=smoothing, scale=scale)
    z, loss, grad, absolute = pref_reference(v.astype(np.float64) - rv, w, l, weight.astype(np.float64), beta, smoothing, scale)
    # z is one rounding of a difference taken in double (and beta's own); every pair's term a few float32
    # roundings of at most w (|z| + 1), every slope of at most beta w
    assert np.all(np.abs(out.margins.double().cpu().numpy() - z) <= 2.1 * U * np.abs(z))
    assert abs(float(out.loss) - loss) <= 12 * U * scale * np.sum(weight * (np.abs(z) + 1)) + U * loss
    zmax = np.abs(z).max() if pairs else 0.0
    assert np.all(np.abs(out.grad.double().cpu().numpy() - grad) <= (12 + 3 * zmax) * U * absolute + U * np.abs(grad))


@pytest.mark.parametrize("lengths,pairs", [([1, 1], 1), ([0, 4, 0, 7], 5), (list(rs.randint(0, 40, 500)), 900),
                                           ([3000, 1, 9000, 600, 0, 2], 12)])
def test_preference_sequences(hip, lengths, pairs):
    from packboost_amd import PreferencePairs, preference_loss

    r = np.random.default_rng(len(lengths))
    off = offsets_of(lengths)
    n, s = int(off[-1]), len(lengths)
    w = r.integers(0, s, pairs)
    l = (w + 1 + r.integers(0, s - 1, pairs)) % s
    v = (-2 * r.random(n)).astype(np.float32)
    rv = (v + 0.3 * r.standard_normal(n)).astype(np.float32)
    out = preference_loss(torch.from_numpy(v).to(DEV), PreferencePairs(w, l, offsets=off),
                          ref_values=torch.from_numpy(rv).to(DEV), beta=0.1)
    a = np.array([np.sum(v[b:e].astype(np.float64) - rv[b:e]) for b, e in zip(off[:-1], off[1:])])
    z, loss, grad, absolute = pref_reference(a, w, l, np.ones(pairs), 0.1, 0.0, 1.0)
    # the sequences' sums are taken in double and rounded once
    room = 0.1 * U * (np.abs(a[w]) + np.abs(a[l])) + 2.1 * U * np.abs(z)
    assert np.all(np.abs(out.margins.double().cpu().numpy() - z) <= room)
    assert abs(float(out.loss) - loss) <= np.sum(room) + 12 * U * np.sum(np.abs(z) + 1) + U * loss
    per_step = np.repeat(grad, lengths)
    rel = (12 + 3 * np.abs(z).max()) * U + room.max()
    assert np.all(np.abs(out.grad.double().cpu().numpy() - per_step) <= np.repeat(absolute, lengths) * rel + U * np.abs(per_step))


def test_extreme_margins(hip):
    """Margins far outside float32's exponentials give the loss's limits, not NaN."""
    from packboost_amd import PreferencePairs, preference_loss

    v = torch.tensor([1e6, -1e6, 0.0], device=DEV)
    out = preference_loss(v, PreferencePairs([0, 1, 0], [1, 0, 2], num_values=3), beta=1.0)
    assert out.margins.tolist() == [2e6, -2e6, 1e6]
    assert float(out.loss) == 2e6
    assert out.grad.tolist() == [1.0, -1.0, 0.0]
    bad = preference_loss(torch.tensor([math.nan, 0.0, 1.0, 2.0], device=DEV),
                          PreferencePairs([0, 2], [1, 3], num_values=4), beta=1.0)
    assert math.isnan(float(bad.loss)) and math.isnan(float(bad.margins[0])) and not math.isnan(float(bad.margins[1]))
    g = bad.grad.tolist()
    assert math.isnan(g[0]) and math.isnan(g[1]) and g[2] == pytest.approx(-g[3])


def test_special_scores(hip):
    """Infinities, the lowest value and NaN on offer: only the sets that hold them see them."""
    from packboost_amd import choice_log_probs, choice_log_probs_backward

    low = torch.finfo(torch.float32).min
    inf, nan = math.inf, math.nan
    sizes = [3, 2, 2, 2, 3, 2, 600]
    s = [0.0, -inf, 0.0] + [low, low] + [-inf, -inf] + [nan, 1.0] + [1.0, low, 1.0] + [inf, 0.0] + [0.0] * 600
    from packboost_amd import ChoiceSets

    sets = ChoiceSets(offsets_of(sizes))
    scores = torch.tensor(s, device=DEV)
    lp, lse = choice_log_probs(scores, sets)
    lp, lse = lp.cpu().numpy(), lse.cpu().numpy()
    half = np.float32(-math.log(2))
    assert lp[0] == half and lp[1] == -inf and lp[2] == half
    assert lp[3] == half and lp[4] == half            # all at the lowest value: a uniform choice
    assert lse[2] == -inf and lp[5] == -inf and lp[6] == -inf
    assert np.isnan(lse[3]) and np.isnan(lp[7:9]).all()
    assert lp[9] == half and lp[11] == half and lp[10] == low
    assert np.isnan(lse[5]) and np.isnan(lp[12:14]).any()
    assert np.allclose(lp[14:], -math.log(600), atol=1e-6)
    chosen = torch.tensor([0, 1, 0, 1, 0, 1, 5], dtype=torch.int32, device=DEV)
    slp, slse = choice_log_probs(scores, sets, chosen=chosen)
    assert float(slp[2]) == 0.0 and math.isnan(float(slp[3]))
    gs, _ = choice_log_probs_backward(torch.ones(7, device=DEV), scores, slse, sets, chosen=chosen)
    gs = gs.cpu().numpy()
    assert gs[:3].tolist() == [0.5, 0.0, -0.5] and gs[5:7].tolist() == [0.0, 0.0] and np.isnan(gs[7:9]).all()
    assert np.isfinite(gs[9:12]).all() and np.isfinite(gs[14:]).all()


def test_step_left_out_hides_what_its_set_holds(hip):
    """A step without a choice gives no gradient, whatever its scores are."""
    from packboost_amd import ChoiceSets, policy_loss

    sets = ChoiceSets([0, 3, 5])
    scores = torch.tensor([math.nan, math.inf, 1.0, 0.5, 0.25], device=DEV)
    chosen = torch.tensor([-1, 1], dtype=torch.int32, device=DEV)
    one = torch.ones(2, device=DEV)
    r = policy_loss(scores, sets, chosen, one, -one, ref_log_probs=-one, kl_weight=0.1)
    assert r.grad_scores[:3].tolist() == [0.0, 0.0, 0.0]
    assert math.isfinite(float(r.loss)) and float(r.log_probs[0]) == 0.0


def test_table_gradient_that_is_not_finite(hip):
    from packboost_amd import ChoiceSets, PositionBias, PositionBuckets, choice_log_probs, choice_log_probs_backward

    sets = ChoiceSets([0, 2, 4])
    scores = torch.tensor([math.nan, 1.0, 0.5, 0.25], device=DEV)
    pos = torch.tensor([0, 1, -1, -2], dtype=torch.int32, device=DEV)
    bias = PositionBias(torch.zeros(16, device=DEV), pos, PositionBuckets(16, 32))
    chosen = torch.zeros(2, dtype=torch.int32, device=DEV)
    _, lse = choice_log_probs(scores, sets, chosen=chosen, bias=bias)
    _, gt = choice_log_probs_backward(torch.ones(2, device=DEV), scores, lse, sets, chosen=chosen, bias=bias)
    ids = bias.buckets([0, 1, -1, -2])
    got = gt.cpu().numpy()
    assert np.isnan(got[ids[0]]) and np.isnan(got[ids[1]])
    assert got[ids[2]] == pytest.approx(-got[ids[3]]) and np.isfinite(np.delete(got, ids[:2])).all()


@pytest.mark.parametrize("buckets,reach,both", [(4, 2, True), (256, 1000, True), (31, 64, False), (64, 40, True)])
def test_position_bias_shapes(hip, buckets, reach, both):
    """Few and many buckets, one side only, positions at the ends of int32."""
    from packboost_amd import ChoiceSets, PositionBias, PositionBuckets, choice_log_probs, choice_log_probs_backward

    r = np.random.default_rng(buckets)
    sizes = [700, 3, 0, 2500]
    off = offsets_of(sizes)
    n = int(off[-1])
    pos = r.integers(-2 * reach, 2 * reach, n).astype(np.int32)
    pos[[0, 1, 2, 700, 2000]] = [-2 ** 31, 2 ** 31 - 1, 0, reach, -reach]
    pb = PositionBuckets(buckets, reach, bidirectional=both)
    table = r.standard_normal(buckets).astype(np.float32)
    s = r.standard_normal(n).astype(np.float32)
    d = {"off": off, "size": np.diff(off), "keep": np.ones(n, bool), "dtype": "f32", "ids": pb(pos).astype(np.int64),
         "c": np.zeros(4, np.int64), "bias": PositionBias(torch.from_numpy(table).to(DEV), torch.from_numpy(pos).to(DEV), pb)}
    d["x"] = s.astype(np.float64) + table[d["ids"]]
    sets = ChoiceSets(off)
    chosen = torch.zeros(4, dtype=torch.int32, device=DEV)
    p, _, lse, ok, step, at = reference(d)
    got, got_lse = choice_log_probs(torch.from_numpy(s).to(DEV), sets, chosen=chosen, bias=d["bias"])
    same_or_close(got, step, bound_lp(d))
    up = np.array([1.0, -2.0, 3.0, 1e-3], np.float32)
    gs, gt = choice_log_probs_backward(torch.from_numpy(up).to(DEV), torch.from_numpy(s).to(DEV), got_lse, sets,
                                       chosen=chosen, bias=d["bias"])
    g, size = back(d, p, ok, at, up.astype(np.float64))
    check_grads(d, gs, gt, g, size, bound_lp(d))


def test_gradients_against_differences(hip):
    """Central differences of the losses themselves: with h = 1/64 the loss (below 16) is rounded to
    2^-20, its difference quotient to 2^-15, and the third derivative's term is below h^2 = 2^-12."""
    from packboost_amd import ChoiceSets, PositionBias, PositionBuckets, PreferencePairs, policy_loss, preference_loss

    r = np.random.default_rng(5)
    off = offsets_of([3, 1, 4, 2])
    sets = ChoiceSets(off)
    n, h, tol = int(off[-1]), 1.0 / 64, 2.0 ** -11
    s = torch.from_numpy(r.standard_normal(n).astype(np.float32)).to(DEV)
    chosen = torch.tensor([1, 0, 3, 0], dtype=torch.int32, device=DEV)
    adv = torch.tensor([1.0, -0.5, 0.7, -1.0], device=DEV)
    pos = torch.arange(n, dtype=torch.int32, device=DEV) - 4
    table = torch.from_numpy(0.3 * r.standard_normal(8).astype(np.float32)).to(DEV)
    pb = PositionBuckets(8, 4)
    from packboost_amd import choice_log_probs

    start, _ = choice_log_probs(s, sets, chosen=chosen, bias=PositionBias(table, pos, pb))
    old = start - torch.tensor([0.05, 0.0, -0.05, 0.02], device=DEV)  # inside the bounds, away from the kinks

    def loss(sv, tv):
        return policy_loss(sv, sets, chosen, adv, old, ref_log_probs=old + 0.1, bias=PositionBias(tv, pos, pb),
                           clip=(0.3, 0.3), kl_weight=0.2)

    out = loss(s, table)
    for i in range(n):
        e = torch.zeros_like(s)
        e[i] = h
        assert abs((float(loss(s + e, table).loss) - float(loss(s - e, table).loss)) / (2 * h) - float(out.grad_scores[i])) < tol
    for b in range(8):
        e = torch.zeros_like(table)
        e[b] = h
        assert abs((float(loss(s, table + e).loss) - float(loss(s, table - e).loss)) / (2 * h) - float(out.grad_table[b])) < tol
    pairs = PreferencePairs([0, 2, 4, 0], [1, 3, 0, 4], num_values=5)
    v = s[:5].clone()

    def pl(x):
        return preference_loss(x, pairs, beta=0.8, label_smoothing=0.1)

    got = pl(v)
    for i in range(5):
        e = torch.zeros_like(v)
        e[i] = h
        assert abs((float(pl(v + e).loss) - float(pl(v - e).loss)) / (2 * h) - float(got.grad[i])) < tol


def test_strides_and_streams(hip):
    """Scores with a stride, other columns that are views, calls on a stream of the caller's."""
    from packboost_amd import policy_loss

    d = make(LAYOUTS["mixed"], masked=True, biased=True, seed=8)
    _, _, _, _, step, _ = reference(d)
    v, low, high, kw = policy_inputs(d, step)
    dev = {k: torch.from_numpy(a).to(DEV) for k, a in v.items()}
    args = dict(clip=(low, high), kl_weight=kw)
    want = policy_loss(d["scores"], d["sets"], d["chosen"], **dev, mask=d["mask"], bias=d["bias"], **args)
    wide = torch.zeros((d["scores"].numel(), 3), device=DEV)
    wide[:, 1] = d["scores"]
    views = {k: torch.stack([a, a], 1).reshape(-1)[::2] for k, a in dev.items()}
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = policy_loss(wide[:, 1], d["sets"], d["chosen"], **views, mask=d["mask"], bias=d["bias"], **args)
    stream.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    shifted = torch.zeros(d["scores"].numel() + 1, device=DEV)  # a start that is not 16-byte aligned
    shifted[1:] = d["scores"]
    for a, b in zip(policy_loss(shifted[1:], d["sets"], d["chosen"], **dev, mask=d["mask"], bias=d["bias"], **args), want):
        assert torch.equal(a, b)


def test_same_results_every_time(hip):
    from packboost_amd import PreferencePairs, choice_log_probs, choice_log_probs_backward, preference_loss

    d = make(list(rs.randint(0, 60, 9000)) + [30_000], masked=True, biased=True, seed=9)
    up = torch.from_numpy(d["r"].standard_normal(len(d["size"])).astype(np.float32)).to(DEV)
    w = d["r"].integers(0, 50, 40_000)
    pairs = PreferencePairs(w, (w + 1) % 50, num_values=50)
    runs = []
    for _ in range(3):
        lp, lse = choice_log_probs(d["scores"], d["sets"], chosen=d["chosen"], mask=d["mask"], bias=d["bias"])
        gs, gt = choice_log_probs_backward(up, d["scores"], lse, d["sets"], chosen=d["chosen"], mask=d["mask"], bias=d["bias"])
        runs.append((lp, lse, gs, gt) + tuple(preference_loss(up[:50], pairs)))
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_graph_replays(hip):
    """Captured calls: every replay on new inputs equals the eager calls, eager work between them."""
    from packboost_amd import PreferencePairs, choice_log_probs, choice_log_probs_backward, policy_loss, preference_loss

    d = make(LAYOUTS["mixed"] + [3] * 3000, masked=True, biased=True, seed=10)
    g = len(d["size"])
    pairs = PreferencePairs(np.arange(0, g - 1), np.arange(1, g), num_values=g)
    s, old = d["scores"].clone(), torch.full((g,), -1.0, device=DEV)
    adv = torch.from_numpy(d["r"].standard_normal(g).astype(np.float32)).to(DEV)
    kw = dict(mask=d["mask"], bias=d["bias"])

    def calls():
        lp, lse = choice_log_probs(s, d["sets"], chosen=d["chosen"], **kw)
        pref = preference_loss(lp, pairs)
        return (lp, lse, *pref, *choice_log_probs_backward(pref.grad, s, lse, d["sets"], chosen=d["chosen"], **kw),
                *policy_loss(s, d["sets"], d["chosen"], adv, old, **kw))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = calls()
    for k in range(4):
        s.copy_(torch.where(d["mask"], d["scores"] * (1 + k), d["scores"]))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = calls()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k


def test_rows_past_32_bits(hip):
    """A table of more than 2^31 rows: the last sets' values are those of the same rows alone."""
    from packboost_amd import ChoiceSets, choice_log_probs, choice_log_probs_backward

    free, _ = torch.cuda.mem_get_info()
    if free < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    n = 2 ** 31 + 70_001
    off = np.concatenate([np.arange(0, n - 70_000, 2 ** 21), [n - 60_000, n - 59_990, n - 1, n]]).astype(np.int64)
    off[0] = 0
    scores = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    tail = torch.randn(70_001, device=DEV).to(torch.bfloat16)
    scores[-70_001:] = tail
    sets = ChoiceSets(off)
    g = sets.num_sets
    chosen = torch.zeros(g, dtype=torch.int32, device=DEV)
    lp, lse = choice_log_probs(scores, sets, chosen=chosen)
    up = torch.ones(g, device=DEV)
    gs, _ = choice_log_probs_backward(up, scores, lse, sets, chosen=chosen)
    # from the multiple of 8 before them on: sums of rows that start elsewhere in their lanes differ in their
    # last bits
    start = int(off[-4]) & ~7
    small = ChoiceSets(np.concatenate([[0], off[-4:] - start]))
    part = scores[start:].contiguous()
    lp2, lse2 = (t[1:] for t in choice_log_probs(part, small, chosen=chosen[:4]))
    gs2, _ = choice_log_probs_backward(up[:4], part, choice_log_probs(part, small, chosen=chosen[:4])[1], small,
                                       chosen=chosen[:4])
    gs2 = gs2[int(off[-4]) - start:]
    assert torch.equal(lp[-3:], lp2) and torch.equal(lse[-3:], lse2)
    assert torch.equal(gs[int(off[-4]):], gs2)
    assert float(lse[1]) == pytest.approx(math.log(2 ** 21), rel=1e-6)


def test_refusals(hip):
    from packboost_amd import (ChoiceSets, PositionBias, PositionBuckets, PreferencePairs, choice_log_probs,
                               choice_log_probs_backward, policy_loss, preference_loss)

    sets = ChoiceSets([0, 2, 5])
    s = torch.zeros(5, device=DEV)
    c = torch.zeros(2, dtype=torch.int32, device=DEV)
    f = torch.zeros(2, device=DEV)
    pb = PositionBuckets(8, 16)
    pos = torch.zeros(5, dtype=torch.int32, device=DEV)
    bad_calls = [
        lambda: choice_log_probs(s[:4], sets),
        lambda: choice_log_probs(s.double(), sets),
        lambda: choice_log_probs(s.cpu(), sets),
        lambda: choice_log_probs(s.view(5, 1), sets),
        lambda: choice_log_probs(s, [0, 2, 5]),
        lambda: choice_log_probs(s, sets, chosen=c.long()),
        lambda: choice_log_probs(s, sets, chosen=c[:1]),
        lambda: choice_log_probs(s, sets, mask=s),
        lambda: choice_log_probs(s, sets, bias=PositionBias(torch.zeros(7, device=DEV), pos, pb)),
        lambda: choice_log_probs(s, sets, bias=PositionBias(torch.zeros(8, device=DEV), pos.long(), pb)),
        lambda: choice_log_probs_backward(f, s, f, sets),
        lambda: choice_log_probs_backward(f, s, f[:1], sets, chosen=c),
        lambda: policy_loss(s, sets, c, f, f[:1]),
        lambda: policy_loss(s, sets, c, None, f),
        lambda: policy_loss(s, sets, c, f, f, clip=(-0.1, 0.2)),
        lambda: policy_loss(s, sets, c, f, f, kl_weight=math.nan),
        lambda: preference_loss(f, PreferencePairs([0], [1], num_values=3)),
        lambda: preference_loss(f, PreferencePairs([0], [1], num_values=2), label_smoothing=1.5),
        lambda: preference_loss(f, PreferencePairs([0], [1], num_values=2), beta=math.inf),
        lambda: preference_loss(f, sets),
    ]
    for i, call in enumerate(bad_calls):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    for w, l, kw in (([0], [2], dict(num_values=2)), ([-1], [0], dict(num_values=2)), ([0, 1], [1], dict(num_values=2)),
                     ([0], [1], {}), ([0], [1], dict(num_values=2, offsets=[0, 1, 2])),
                     ([0], [1], dict(offsets=[0, 2, 1]))):
        with pytest.raises(ValueError):
            PreferencePairs(w, l, **kw)
    for off in ([], [1, 2], [0, 3, 2], [[0, 1]], [0.0, 1.0]):
        with pytest.raises(ValueError):
            ChoiceSets(off)
    sets.close()
    with pytest.raises(ValueError):
        choice_log_probs(s, sets)


def test_no_sets(hip):
    from packboost_amd import (ChoiceSets, PositionBias, PositionBuckets, choice_log_probs, choice_log_probs_backward,
                               policy_loss)

    sets = ChoiceSets([0])
    none = torch.zeros(0, device=DEV)
    c = torch.zeros(0, dtype=torch.int32, device=DEV)
    bias = PositionBias(torch.zeros(8, device=DEV), torch.zeros(0, dtype=torch.int32, device=DEV), PositionBuckets(8, 16))
    lp, lse = choice_log_probs(none, sets)
    assert lp.numel() == 0 and lse.numel() == 0
    gs, gt = choice_log_probs_backward(none, none, none, sets, chosen=c, bias=bias)
    assert gs.numel() == 0 and gt.tolist() == [0.0] * 8
    r = policy_loss(none, sets, c, none, none, bias=bias)
    assert float(r.loss) == 0.0 and float(r.kl) == 0.0 and r.grad_table.tolist() == [0.0] * 8
