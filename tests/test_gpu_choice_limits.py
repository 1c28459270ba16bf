"""The choice and preference operators at the limits of their numbers: terms that count for nothing beside
ones that overflow, gradients and scores far apart in size, long sums that nearly cancel. Each bound is one
of the formula in 64 bits and of the sizes that the value itself is made of."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from test_gpu_choices import DEV, U, back, offsets_of, per_set, policy_reference, reference

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
