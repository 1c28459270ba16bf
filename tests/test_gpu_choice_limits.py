"""The choice and preference operators at the limits of their numbers: terms that count for nothing beside
ones that overflow, gradients and scores far apart in size, long sums that nearly cancel. Each bound is one
of the formula in 64 bits and of the sizes that the value itself is made of."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from test_gpu_choices import (DEV, LAYOUTS, U, back, bound_lp, check_grads, make, offsets_of, per_set, policy_reference,
                              reference, same_or_close)

pytestmark = pytest.mark.gpu

SIZES = [2, 700, 3000, 9000, 3]  # a tile's sets, a wave's, a workgroup's, one in parts


def policy_case(scores, sizes, chosen, adv, old, ref=None, weights=None, kl=0.0):
    """policy_loss and the formula's log-probabilities, terms and gradients, in the bounds of test_gpu_choices."""
    from packboost_amd import ChoiceSets, policy_loss

    off = offsets_of(sizes)
    v = {"advantages": adv, "old_log_probs": old}
    if ref is not None:
        v["ref_log_probs"] = ref
    if weights is not None:
        v["weights"] = weights
    v = {k: np.asarray(a, dtype=np.float32) for k, a in v.items()}
    c = np.asarray(chosen, dtype=np.int32)
    s = np.asarray(scores, dtype=np.float32)
    d = {"off": off, "size": np.diff(off), "x": s.astype(np.float64), "keep": np.ones(len(s), bool), "c": c.astype(np.int64)}
    r = policy_loss(torch.from_numpy(s).to(DEV), ChoiceSets(off), torch.from_numpy(c).to(DEV),
                    **{k: torch.from_numpy(a).to(DEV) for k, a in v.items()}, kl_weight=kl)
    p, _, _, ok, step, at = reference(d)
    loss, _, clipped, slope, w = policy_reference(v, ok, step, 0.2, 0.2, kl, 1.0)
    g, size = back(d, p, ok, at, slope)
    tol = U * (4 * np.abs(s).max() + 100)
    # a slope of rA moves by itself per unit of log p, one of the KL term by e^d, each only where it counts
    gap = np.exp(v["ref_log_probs"].astype(np.float64) - step) if kl else np.zeros(len(c))
    term = w * (np.where(slope != 0, np.exp(step - v["old_log_probs"]) * np.abs(v["advantages"]), 0.0) + kl * (gap + 1 + np.abs(np.log(gap + (gap == 0)))))
    _, extra = back(d, p, ok, at, term * (tol + 16 * U))
    assert abs(float(r.loss) - loss.sum()) <= (np.abs(loss) * (tol + 16 * U) + term * (tol + 16 * U)).sum() + U * abs(loss.sum())
    assert float(r.clipped) == clipped.sum()
    got = r.grad_scores.double().cpu().numpy()
    assert np.all(np.abs(got - g) <= size * (tol + 4 * U) + extra + U * np.abs(g))
    return r


def far_choices(sizes):
    """Scores of 0 but for the chosen row's -100, and the steps' log-probabilities."""
    off = offsets_of(sizes)
    chosen = np.asarray(sizes) - 1
    s = np.zeros(int(off[-1]))
    s[off[:-1] + chosen] = -100.0
    return s, chosen, -100.0 - np.log(np.asarray(sizes) - 1.0)


def test_no_weight_on_the_kl_term(hip):
    """e^(ref - log p) overflows, and kl_weight, the default, is 0: neither loss nor gradients see it."""
    sizes = SIZES * 3
    s, chosen, lp = far_choices(sizes)
    adv = np.where(np.arange(len(sizes)) % 2, 0.5, -0.75)
    r = policy_case(s, sizes, chosen, adv, lp, ref=np.full(len(sizes), -1.0))
    assert torch.isfinite(r.grad_scores).all() and math.isfinite(float(r.loss))
    assert float(r.kl) == math.inf  # what it is told as, it is


@pytest.mark.parametrize("kl", [0.0, 0.05])
def test_steps_of_no_weight(hip, kl):
    """Steps of weight 0 whose ratio and KL term overflow, beside steps that count."""
    sizes = SIZES * 2
    s, chosen, lp = far_choices(sizes)
    n = len(sizes)
    far = np.arange(n) < len(SIZES)
    old = np.where(far, -250.0, lp - 0.1)
    ref = np.where(far, -1.0, lp + 0.1)
    adv = np.where(np.arange(n) % 2, 0.5, -0.75)
    r = policy_case(s, sizes, chosen, adv, old, ref=ref, weights=np.where(far, 0.0, 0.5), kl=kl)
    first = int(sum(SIZES))
    assert torch.equal(r.grad_scores[:first], torch.zeros(first, device=DEV))
    assert math.isfinite(float(r.kl))


def test_steps_without_advantage(hip):
    """A ratio that overflows times an advantage of 0 is 0."""
    s, chosen, lp = far_choices(SIZES)
    r = policy_case(s, SIZES, chosen, np.zeros(len(SIZES)), lp - 100.0)
    assert float(r.loss) == 0.0 and float(r.clipped) == 0.0
    assert torch.equal(r.grad_scores, torch.zeros_like(r.grad_scores))


@pytest.mark.parametrize("ref", [False, True])
def test_preference_terms_of_no_weight(hip, ref):
    """Margins that are infinite on the side of a factor of 0, and pairs of weight 0, count for nothing."""
    from packboost_amd import PreferencePairs, preference_loss

    inf, nan = math.inf, math.nan
    v = torch.tensor([0.5, 0.25, -inf, 1.0, nan], device=DEV)
    kw = dict(ref_values=torch.zeros(5, device=DEV)) if ref else {}
    alone = preference_loss(v[:2].contiguous(), PreferencePairs([0], [1], num_values=2), beta=1.0)
    # the loser cannot be had at all: the loss's limit is 0, and so is the slope's
    r = preference_loss(v, PreferencePairs([0, 3], [1, 2], num_values=5), beta=1.0, **kw)
    assert float(r.loss) == float(alone.loss) and float(r.margins[1]) == inf
    assert r.grad.tolist() == alone.grad.tolist() + [0.0, 0.0, 0.0]
    # the same with labels the other way round
    one = preference_loss(v[:2].contiguous(), PreferencePairs([0], [1], num_values=2), beta=1.0, label_smoothing=1.0)
    r = preference_loss(v, PreferencePairs([0, 2], [1, 3], num_values=5), beta=1.0, label_smoothing=1.0, **kw)
    assert float(r.loss) == float(one.loss) and r.grad.tolist() == one.grad.tolist() + [0.0, 0.0, 0.0]
    # weight 0: margins of -inf, inf and NaN
    w = torch.tensor([1.0, 0.0, 0.0, 0.0], device=DEV)
    for e in (0.0, 0.25, 1.0):
        want = preference_loss(v[:2].contiguous(), PreferencePairs([0], [1], num_values=2), beta=1.0, label_smoothing=e)
        r = preference_loss(v, PreferencePairs([0, 2, 3, 4], [1, 3, 2, 0], num_values=5), beta=1.0, label_smoothing=e,
                            weights=w, **kw)
        assert float(r.loss) == float(want.loss) and r.grad.tolist() == want.grad.tolist() + [0.0, 0.0, 0.0]
    # what does count stays visible
    assert float(preference_loss(v, PreferencePairs([2], [3], num_values=5), beta=1.0, **kw).loss) == inf
    assert math.isnan(float(preference_loss(v, PreferencePairs([4], [3], num_values=5), beta=1.0, **kw).loss))


def test_preference_of_steps_that_cannot_be(hip):
    """A choice whose score is -inf has log-probability -inf; the sequence that holds it loses for nothing."""
    from packboost_amd import ChoiceSets, PreferencePairs, choice_log_probs, preference_loss

    s = torch.tensor([0.0, 1.0, -math.inf, 0.5, 0.0, 0.0], device=DEV)
    lp, _ = choice_log_probs(s, ChoiceSets([0, 2, 4, 6]), chosen=torch.zeros(3, dtype=torch.int32, device=DEV))
    assert float(lp[1]) == -math.inf
    r = preference_loss(lp, PreferencePairs([0, 0], [1, 2], offsets=[0, 1, 2, 3]), beta=0.5)
    z = 0.5 * (float(lp[0]) - float(lp[2]))
    assert float(r.loss) == pytest.approx(math.log1p(math.exp(-z)), rel=8 * U)
    assert torch.isfinite(r.grad).all() and float(r.grad[1]) == 0.0


def bucket_case(sizes, far_sets, seed=0, num=16, reach=32):
    """Sets whose positions name buckets up to the reference, but for those of `far_sets`, which name the ones
    after it."""
    from packboost_amd import ChoiceSets, PositionBias, PositionBuckets

    r = np.random.default_rng(seed)
    off = offsets_of(sizes)
    n = int(off[-1])
    pos = -(np.arange(n) % 23).astype(np.int32)
    far = np.repeat(np.isin(np.arange(len(sizes)), list(far_sets)), sizes)
    pos[far] = 1 - pos[far]
    pb = PositionBuckets(num, reach)
    table = (0.3 * r.standard_normal(num)).astype(np.float32)
    s = r.standard_normal(n).astype(np.float32)
    d = {"off": off, "size": np.diff(off), "keep": np.ones(n, bool), "ids": pb(pos).astype(np.int64), "r": r,
         "c": np.floor(r.random(len(sizes)) * np.diff(off)).astype(np.int64), "sets": ChoiceSets(off), "scores": torch.from_numpy(s).to(DEV),
         "bias": PositionBias(torch.from_numpy(table).to(DEV), torch.from_numpy(pos).to(DEV), pb)}
    d["x"] = s.astype(np.float64) + table.astype(np.float64)[d["ids"]]
    d["chosen"] = torch.from_numpy(d["c"].astype(np.int32)).to(DEV)
    return d


def check_buckets(d, got, g, size, room=0.0):
    """A bucket's sum is off by what its own rows' gradients are off by (`size`, the sum of a row's absolute terms,
    and `room`), by 2^-30 of its own largest one a row, and by its rounding. No other bucket's size comes in."""
    nb = d["bias"].buckets.num_buckets
    tol = U * (4 * np.abs(d["x"]).max() + 100)
    want = np.bincount(d["ids"], g, minlength=nb)
    big = np.zeros(nb)
    np.maximum.at(big, d["ids"], np.abs(g))
    lim = np.bincount(d["ids"], size * (tol + 4 * U) + room, minlength=nb) + np.bincount(d["ids"], minlength=nb) * big * 2.0 ** -30
    assert np.all(np.abs(got.double().cpu().numpy() - want) <= lim + 2 * U * np.abs(want))
    near = np.unique(d["ids"][d["ids"] < nb // 2])
    assert np.all(lim[near] < 1e-3 * np.bincount(d["ids"], np.abs(g), minlength=nb)[near])  # the bound says something


OUTLIERS = {
    "tile": ([3] * 300, [0]),
    "tile_last": ([5] * 400, [399]),
    "tiles": ([4] * 1_200_000, [0, 40_000, 1_199_999]),  # more than one to a wave
    "wave": ([600, 900, 600, 700], [0]),
    "group": ([3000, 5000, 2500], [1]),
    "parts": ([30_000, 20_000], [0]),
    "mixture": ([3, 700, 3, 4000, 2, 20_000, 3] * 3, [0, 3]),
}


@pytest.mark.parametrize("case", list(OUTLIERS))
@pytest.mark.parametrize("size", [1e8, 1e30])
def test_a_buckets_gradient_is_its_own(hip, case, size):
    """A few steps' gradients 1e8 (1e30) times the others', whose rows lie in buckets of their own: the other
    buckets' gradients keep their bits."""
    from packboost_amd import choice_log_probs, choice_log_probs_backward

    sizes, far = OUTLIERS[case]
    d = bucket_case(sizes, far, seed=len(sizes))
    p, _, _, ok, _, at = reference(d)
    _, lse = choice_log_probs(d["scores"], d["sets"], chosen=d["chosen"], bias=d["bias"])
    up = d["r"].uniform(0.5, 1.0, len(sizes)).astype(np.float32)
    up[far] *= size
    _, gt = choice_log_probs_backward(torch.from_numpy(up).to(DEV), d["scores"], lse, d["sets"], chosen=d["chosen"], bias=d["bias"])
    check_buckets(d, gt, *back(d, p, ok, at, up.astype(np.float64)))
    rows = d["r"].standard_normal(len(d["x"])).astype(np.float32)
    rows[np.repeat(np.isin(np.arange(len(sizes)), far), sizes)] *= size
    _, gt = choice_log_probs_backward(torch.from_numpy(rows).to(DEV), d["scores"], lse, d["sets"], bias=d["bias"])
    u = rows.astype(np.float64)
    total, absolute = (np.repeat(per_set(d, np.add, v, 0.0), d["size"]) for v in (u, np.abs(u)))
    # the sum of a set's gradients passes at most 100 roundings
    check_buckets(d, gt, u - p * total, np.abs(u) + p * absolute, 100 * U * p * absolute)


def test_policy_with_a_stale_step(hip):
    """The ratio is not held where the advantage is below 0: a log-probability 20 nats off takes e^20."""
    from packboost_amd import policy_loss

    d = bucket_case([4] * 2000, [7], seed=3)
    p, _, _, ok, step, at = reference(d)
    old = (step - 0.01).astype(np.float32)
    old[7] -= 20
    adv = np.where(np.arange(2000) == 7, -1.0, d["r"].uniform(0.5, 1, 2000)).astype(np.float32)
    r = policy_loss(d["scores"], d["sets"], d["chosen"], torch.from_numpy(adv).to(DEV), torch.from_numpy(old).to(DEV), bias=d["bias"])
    _, _, _, slope, w = policy_reference({"advantages": adv, "old_log_probs": old}, ok, step, 0.2, 0.2, 0.0, 1.0)
    tol = U * (4 * np.abs(d["x"]).max() + 100)
    g, size = back(d, p, ok, at, slope)
    check_buckets(d, r.grad_table, g, size, size * (tol + 16 * U))


def test_bucket_gradients_that_grow(hip):
    """A bucket's gradients rise by many powers of two along the rows, each bucket's in its own way."""
    from packboost_amd import choice_log_probs, choice_log_probs_backward

    sets = 700_000  # more than a tile a wave
    d = bucket_case([8] * sets, range(1, sets, 2), seed=5)
    p, _, _, ok, _, at = reference(d)
    i = np.arange(sets)
    up = np.where(i % 2, 2.0 ** (i // 2 % 120 - 60), 2.0 ** (40 - i // 2 % 90)).astype(np.float32) * d["r"].uniform(0.5, 1, sets).astype(np.float32)
    _, lse = choice_log_probs(d["scores"], d["sets"], chosen=d["chosen"], bias=d["bias"])
    _, gt = choice_log_probs_backward(torch.from_numpy(up).to(DEV), d["scores"], lse, d["sets"], chosen=d["chosen"], bias=d["bias"])
    check_buckets(d, gt, *back(d, p, ok, at, up.astype(np.float64)))


@pytest.mark.parametrize("offset", [16.0, -100.0, 8192.0, -8192.0])
@pytest.mark.parametrize("sizes", [[2] * 300, [60, 1, 0, 200, 30], [700, 3000, 5], [9000, 2], [30_000, 9000, 700, 3, 17_000]])
def test_an_offset_of_the_scores_changes_nothing(hip, sizes, offset):
    """Scores in units of 2^-10 below 8 and an offset below 2^13 add without rounding: the gradients are the
    softmax's of the scores alone, in a bound without the offset."""
    from packboost_amd import ChoiceSets, choice_log_probs, choice_log_probs_backward

    r = np.random.default_rng(len(sizes))
    off = offsets_of(sizes)
    n, g = int(off[-1]), len(sizes)
    x = r.integers(-8 << 10, 8 << 10, n) / 1024.0
    d = {"off": off, "size": np.diff(off), "x": x, "keep": np.ones(n, bool),
         "c": np.floor(r.random(g) * np.diff(off)).astype(np.int64)}
    p, _, _, ok, _, at = reference(d)
    sets, tol = ChoiceSets(off), U * (4 * 8 + 100)
    chosen = torch.from_numpy(d["c"].astype(np.int32)).to(DEV)
    scores = torch.from_numpy((x + offset).astype(np.float32)).to(DEV)
    assert np.array_equal(scores.double().cpu().numpy(), x + offset)
    up = r.standard_normal(g).astype(np.float32)
    _, lse = choice_log_probs(scores, sets, chosen=chosen)
    gs, _ = choice_log_probs_backward(torch.from_numpy(up).to(DEV), scores, lse, sets, chosen=chosen)
    want, size = back(d, p, ok, at, up.astype(np.float64))
    assert np.all(np.abs(gs.double().cpu().numpy() - want) <= size * (tol + 4 * U) + U * np.abs(want))
    rows = r.standard_normal(n).astype(np.float32)
    _, lse = choice_log_probs(scores, sets)
    gs, _ = choice_log_probs_backward(torch.from_numpy(rows).to(DEV), scores, lse, sets)
    u = rows.astype(np.float64)
    total, absolute = (np.repeat(per_set(d, np.add, v, 0.0), sizes) for v in (u, np.abs(u)))
    want = u - p * total
    room = np.abs(u) * 4 * U + p * absolute * (tol + 104 * U) + U * np.abs(want)
    assert np.all(np.abs(gs.double().cpu().numpy() - want) <= room)


@pytest.mark.parametrize("score", [3.0e9, -3.0e9, 1e30])
@pytest.mark.parametrize("size", [3, 700, 2500, 20_000])
def test_equal_scores_of_any_size(hip, size, score):
    """A uniform choice, whose lse has no room for the log of the number of rows."""
    from packboost_amd import ChoiceSets, choice_log_probs, choice_log_probs_backward

    sets = ChoiceSets([0, size])
    s = torch.full((size,), score, device=DEV)
    chosen = torch.zeros(1, dtype=torch.int32, device=DEV)
    _, lse = choice_log_probs(s, sets, chosen=chosen)
    gs, _ = choice_log_probs_backward(torch.ones(1, device=DEV), s, lse, sets, chosen=chosen)
    want = np.full(size, -1.0 / size)
    want[0] += 1.0
    assert np.all(np.abs(gs.double().cpu().numpy() - want) <= 8 * U / size + U * np.abs(want))


def test_a_neighbour_far_off_changes_nothing(hip):
    """Sets of one tile, one of them offset: the others' gradients are to the bit what they are without it."""
    from packboost_amd import ChoiceSets, choice_log_probs, choice_log_probs_backward

    s = torch.randn(90, device=DEV)
    moved = s.clone()
    moved[30:60] += 4096.0
    sets, chosen = ChoiceSets([0, 30, 60, 90]), torch.zeros(3, dtype=torch.int32, device=DEV)
    out = []
    for t in (s, moved):
        lp, lse = choice_log_probs(t, sets, chosen=chosen)
        rows, _ = choice_log_probs_backward(t.abs() * 1e-3, t, lse, sets)
        out.append((lp, lse, choice_log_probs_backward(torch.ones(3, device=DEV), t, lse, sets, chosen=chosen)[0], rows))
    for a, b in zip(*out):
        k = len(a) // 3
        assert torch.equal(a[:k], b[:k]) and torch.equal(a[2 * k:], b[2 * k:])


@pytest.mark.parametrize("length", [400, 1900, 7000, 10_000, 30_000])
def test_long_sequences_that_nearly_cancel(hip, length):
    """Sequences' sums are large and their differences small: a margin is the difference of two sums in double,
    rounded once (and beta's own rounding)."""
    from packboost_amd import PreferencePairs, preference_loss

    r = np.random.default_rng(length)
    seqs = 8
    off = offsets_of([length] * seqs)
    v = (-4 * r.random(length * seqs)).astype(np.float32)
    a = np.array([v[b:e].astype(np.float64).sum() for b, e in zip(off[:-1], off[1:])])
    for k in range(1, seqs):  # a last step that brings the sum next to the first sequence's
        v[off[k + 1] - 1] += np.float32(a[0] - a[k] + r.uniform(-1, 1))
    a = np.array([v[b:e].astype(np.float64).sum() for b, e in zip(off[:-1], off[1:])])
    w, l = np.repeat(np.arange(seqs), seqs), np.tile(np.arange(seqs), seqs)
    out = preference_loss(torch.from_numpy(v).to(DEV), PreferencePairs(w, l, offsets=off), beta=0.5)
    z = 0.5 * (a[w] - a[l])
    # a term (2 on average) passes at most 2^8 additions in double, here and there
    assert np.all(np.abs(out.margins.double().cpu().numpy() - z) <= 2.1 * U * np.abs(z) + 2.0 ** -44 * length)


def test_kl_term_near_its_zero(hip):
    """A set of one row has log p = 0, so ref_log_probs is d itself: e^d - d - 1, and its slope e^d - 1 on one
    of two equal rows. Both are formed without cancellation that the formula does not have: within 5 units in
    the last place (a unit is at most 2^-23 of the value)."""
    from packboost_amd import ChoiceSets, policy_loss

    d = np.concatenate([np.linspace(-2.2, 2.2, 2001), [1e-4, -1e-4, 0.3465, 0.3467, -0.3465, -0.3467, 0.351, 1e-15, 0.0, 80.0, -80.0]])
    d = d.astype(np.float32)
    one = torch.ones(1, device=DEV)
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    sets, row = ChoiceSets([0, 1]), torch.zeros(1, device=DEV)
    refs = torch.from_numpy(d).to(DEV)
    got = torch.stack([policy_loss(row, sets, zero, one, row, ref_log_probs=refs[i: i + 1], kl_weight=1.0).kl for i in range(len(d))])
    x = d.astype(np.float64)
    want = np.expm1(x) - x
    small = np.abs(x) < 0.1  # where that cancels too: the series
    want[small] = sum(x[small] ** k / math.factorial(k) for k in range(2, 14))
    assert np.all(np.abs(got.double().cpu().numpy() - want) <= 5 * 2 * U * np.abs(want))
    # slopes: two equal rows, log p = -log 2 in more bits than float32's
    n = len(d)
    ref = (d - math.log(2)).astype(np.float32)
    r = policy_loss(torch.zeros(2 * n, device=DEV), ChoiceSets(np.arange(n + 1) * 2), torch.zeros(n, dtype=torch.int32, device=DEV),
                    torch.zeros(n, device=DEV), torch.zeros(n, device=DEV), ref_log_probs=torch.from_numpy(ref).to(DEV), kl_weight=1.0)
    gap = ref.astype(np.float64) + math.log(2)
    want = -0.5 * np.expm1(gap)
    # log 2 itself is known to 2^-30
    assert np.all(np.abs(r.grad_scores[::2].double().cpu().numpy() - want) <= 5 * 2 * U * np.abs(want) + 2.0 ** -30 * np.exp(gap))


def test_small_probabilities_keep_their_bits(hip):
    """Two rows, {0, -t}: the second's probability, down to e^-87, is good to 10 units of itself (the exponential
    2, sum and quotient 2 each, products) and what the difference to a rounded lse takes."""
    from packboost_amd import ChoiceSets, choice_log_probs, choice_log_probs_backward, policy_loss

    t = np.arange(1, 2000) * 0.0434
    t = np.round(t * 65536) / 65536  # differences without rounding
    g = len(t)
    x = np.stack([np.zeros(g), -t], 1).reshape(-1)
    s = torch.from_numpy(x.astype(np.float32)).to(DEV)
    assert np.array_equal(s.double().cpu().numpy(), x)
    sets, c, one = ChoiceSets(np.arange(g + 1) * 2), torch.zeros(g, dtype=torch.int32, device=DEV), torch.ones(g, device=DEV)
    p = np.exp(-t) / (1 + np.exp(-t))
    lp, lse = choice_log_probs(s, sets, chosen=c)
    shift = lse.double().cpu().numpy()
    room = (10 * U + np.where(shift != 0, U * (np.abs(t + shift) + np.abs(shift)), 0.0)) * p
    gs, _ = choice_log_probs_backward(one, s, lse, sets, chosen=c)
    assert np.all(np.abs(gs.double().cpu().numpy()[1::2] + p) <= room)
    rows = torch.tensor([1.0, 0.0], device=DEV).repeat(g)
    gs, _ = choice_log_probs_backward(rows, s, lse, sets)
    assert np.all(np.abs(gs.double().cpu().numpy()[1::2] + p) <= room)
    gs = policy_loss(s, sets, c, one, lp).grad_scores.double().cpu().numpy()[1::2]
    ratio = np.exp(-np.log1p(np.exp(-t)) - lp.double().cpu().numpy())  # a rounding of lp away from 1
    assert np.all(np.abs(gs - ratio * p) <= 12 * U * p)


@pytest.mark.parametrize("size", [700, 2500, 9000])
def test_small_probabilities_of_longer_sets(hip, size):
    """The same by a wave, a workgroup and in parts, whose sums of positive terms pass at most 43 roundings more."""
    from packboost_amd import ChoiceSets, policy_loss

    r = np.random.default_rng(size)
    x = -np.round(r.uniform(0, 86.9, size) * 1024) / 1024
    x[0], x[-1] = 0.0, -86.5
    d = {"off": offsets_of([size]), "size": np.array([size]), "x": x, "keep": np.ones(size, bool), "c": np.array([0])}
    p, lp, *_ = reference(d)
    s = torch.from_numpy(x.astype(np.float32)).to(DEV)
    one, old = torch.ones(1, device=DEV), torch.from_numpy(lp[:1].astype(np.float32)).to(DEV)
    gs = policy_loss(s, ChoiceSets([0, size]), torch.zeros(1, dtype=torch.int32, device=DEV), one, old).grad_scores
    want = math.exp(lp[0] - float(old[0])) * p
    other = np.arange(size) != 0
    # what lies below 2^-126 may be 0
    assert np.all(np.abs(gs.double().cpu().numpy() - want)[other] <= 55 * U * want[other] + 2.0 ** -126)


def test_layouts_and_buckets_around_a_capture(hip):
    """A layout that goes while a graph is captured leaves the capture whole and is freed after it; what needs the
    host is refused inside one, by name."""
    from packboost_amd import ChoiceSets, PositionBias, PositionBuckets, PreferencePairs, choice_log_probs, choices

    s = torch.randn(5, device=DEV)
    pos = torch.arange(5, dtype=torch.int32, device=DEV)
    bias = PositionBias(torch.randn(8, device=DEV), pos, PositionBuckets(8, 16))
    fresh = PositionBias(bias.table, pos, PositionBuckets(8, 16))
    bias.buckets.on(s.device)
    sets, other, pairs = ChoiceSets([0, 2, 5]), ChoiceSets([0, 5]), PreferencePairs([0], [1], num_values=2)
    want = choice_log_probs(s, sets, bias=bias)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for build in (lambda: ChoiceSets([0, 2]), lambda: PreferencePairs([0], [1], num_values=2),
                      lambda: choice_log_probs(s, sets, bias=fresh)):
            with pytest.raises(RuntimeError, match="captur"):
                build()
        other.close()
        del pairs
        assert len(choices._dropped) == 2
        got = choice_log_probs(s, sets, bias=bias)
    with pytest.raises(ValueError, match="closed"):
        choice_log_probs(s, other)
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        ChoiceSets([0, 2]).close()
        assert not choices._dropped
    assert torch.equal(choice_log_probs(s, sets, bias=fresh)[0], want[0])


@pytest.mark.parametrize("dtype,masked,biased", [("f32", False, False), ("f32", True, True), ("f32", False, True),
                                                 ("bf16", True, False), ("bf16", True, True), ("f16", False, True),
                                                 ("f16", True, False), ("f32", True, False)])
@pytest.mark.parametrize("layout", ["small", "empties", "wave", "tile_edges", "mixed", "long_pair"])
def test_offset_scores_of_every_kind(hip, layout, dtype, masked, biased):
    """Scores near 64, whose sets are summed anew in the backward passes: masks, biases, 16-bit scores and every
    kind of set, in the bounds of test_gpu_choices."""
    from packboost_amd import choice_log_probs, choice_log_probs_backward

    d = make(LAYOUTS[layout], dtype, masked, biased, seed=33)
    kw = dict(mask=d["mask"], bias=d["bias"])
    moved = (d["scores"].float() + 64).to(d["scores"].dtype)
    by = (moved.double() - d["scores"].double()).cpu().numpy()
    d["x"] = np.where(d["keep"], d["x"] + np.where(d["keep"], by, 0.0), -np.inf)
    p, _, lse, ok, step, at = reference(d)
    tol = bound_lp(d)
    got, got_lse = choice_log_probs(moved, d["sets"], chosen=d["chosen"], **kw)
    same_or_close(got, step, tol)
    same_or_close(got_lse, lse, tol)
    up = d["r"].standard_normal(len(step)).astype(np.float32)
    gs, gt = choice_log_probs_backward(torch.from_numpy(up).to(DEV), moved, got_lse, d["sets"], chosen=d["chosen"], **kw)
    g, size = back(d, p, ok, at, up.astype(np.float64))
    check_grads(d, gs, gt, g, size, tol)
    rows = d["r"].standard_normal(len(d["x"])).astype(np.float32)
    gs, gt = choice_log_probs_backward(torch.from_numpy(rows).to(DEV), moved, got_lse, d["sets"], **kw)
    u = np.where(d["keep"], rows.astype(np.float64), 0.0)
    total, absolute = (np.repeat(per_set(d, np.add, v, 0.0), d["size"]) for v in (u, np.abs(u)))
    check_grads(d, gs, gt, np.where(d["keep"], u - p * total, 0.0),
                np.abs(u) + p * absolute * (1 + 100 * U / (tol + 4 * U)), tol)


@pytest.mark.parametrize("size", [3, 700, 3000, 9000])
def test_a_choice_that_cannot_be(hip, size):
    """A chosen row whose score is -inf: its log-probability is -inf, its ratio 0 and its KL term inf, which without
    weight changes nothing."""
    from packboost_amd import ChoiceSets, policy_loss

    s = torch.zeros(size, device=DEV)
    s[1] = -math.inf
    one = torch.ones(1, device=DEV)
    r = policy_loss(s, ChoiceSets([0, size]), torch.ones(1, dtype=torch.int32, device=DEV), one, -one, ref_log_probs=-one)
    assert float(r.log_probs[0]) == -math.inf and float(r.kl) == math.inf
    assert float(r.loss) == 0.0 and torch.equal(r.grad_scores, torch.zeros_like(s))
