"""Distillation with a teacher's log-probabilities (tail) far from 0, against the formulas in 64 bits.

Tolerances. An exponential over a list's largest value is within 2^-22 of itself and the rounding of its distance, 2^-24 |d|
with |d| <= 8 here (logits: 4): within 2^-21 at most. A probability is such a term over the sum of such terms, and its
factor and product are rounded once each: p and q are within 2^-19 of themselves. A divergence
sum q (log q - log p) has the same terms in its sums and in q, so that a term's error d_j moves it by q_j d_j (log q_j -
log p_j - kl); the logarithm of the student's sum adds 2^-21 and the result's rounding 2^-24 of it. 16-bit gradients add
half a step."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from test_gpu_choice_layouts import EDGES
from test_gpu_choices import DEV, LAYOUTS, TYPES, U, make, offsets_of
from test_gpu_reports import check_distill, teacher_of

pytestmark = pytest.mark.gpu

Z = np.array([0.5, -0.25, 0.0, 1.0, -1.5])
ORDER = [3, 0, 4, 1, 2]
STEPS = np.array([-1.0, -2.0, -0.875, -3.5, -2.5])  # over `level`, by entry
PADS = [0, 700, 5000, 9000, 70_000]
LEVELS = [-60.0, -89.0, -95.0, -110.0, -300.0, -700.0, 60.0, 100.0, 1000.0]


def softmax(x):
    e = np.exp(x - x.max())
    return e / e.sum()


def closed(z, t):
    """(kl, gradient, bound of the kl) of a list that holds every row with probability."""
    p, q = softmax(z), softmax(t)
    with np.errstate(divide="ignore", invalid="ignore"):
        terms = np.where(q > 0, np.log(q) - np.log(p), 0.0)
    kl = np.sum(q * terms)
    return kl, p - q, 2.0**-21 + 2.0**-21 * np.sum(q * np.abs(terms - kl)) + 2 * U * abs(kl), 2.0**-19 * (p + q)


def close(got, want, room, dtype="f32"):
    unit = TYPES[dtype][1]
    assert np.all(np.abs(got - want) <= room + unit * (np.abs(want) + room) + TYPES[dtype][2]), (got, want)


def sets_of(pad, alone):
    """Sizes, and which of the sets are far from the teacher."""
    return ([5 + pad], [0]) if alone else ([5 + pad, 7, 5 + pad, 0, 3], [0, 2])


@pytest.mark.parametrize("alone", [True, False])
@pytest.mark.parametrize("pad", PADS)
@pytest.mark.parametrize("level", LEVELS)
def test_whole_list_far_from_zero(hip, level, pad, alone):
    """Every row with probability is listed: q is divided by its sum, whatever that is."""
    from packboost_amd import ChoiceSets, distillation_loss

    sizes, far = sets_of(pad, alone)
    off = offsets_of(sizes)
    z = np.zeros(int(off[-1]), np.float32)
    index, value = np.full((len(sizes), 5), -1), np.full((len(sizes), 5), -1.0)
    for g in far:
        z[off[g]: off[g + 1]] = np.concatenate([Z, np.full(pad, -np.inf)])
        index[g], value[g] = ORDER, level + STEPS
    for dtype, teacher in (("f32", "f32"), ("f32", "bf16"), ("bf16", "f16")):
        t = torch.from_numpy(value).to(TYPES[teacher][0])
        r = distillation_loss(torch.from_numpy(z).to(DEV).to(TYPES[dtype][0]), ChoiceSets(off), torch.from_numpy(index).int().to(DEV),
                              t.to(DEV), tail=True)
        grad = r.grad_scores.double().cpu().numpy()
        total = room = 0.0
        for g in far:
            kl, want, kl_room, grad_room = closed(Z[ORDER], t[g].double().numpy())
            close(grad[off[g]: off[g] + 5][ORDER], want, grad_room, dtype)
            assert not grad[off[g] + 5: off[g + 1]].any()
            assert abs(float(r.kl[g]) - kl) <= kl_room
            total, room = total + kl, room + kl_room
        assert abs(float(r.loss) - total) <= room + U * abs(total)
        for g in set(range(len(sizes))) - set(far):
            assert float(r.kl[g]) == 0 and not grad[off[g]: off[g + 1]].any()


@pytest.mark.parametrize("pad", PADS)
@pytest.mark.parametrize("level", [-60.0, -95.0, -110.0, -700.0])
def test_best_row_is_not_on_offer(hip, level, pad):
    """The mask takes the teacher's best row and all that are not listed, what they hold is not read; with a position bias."""
    from packboost_amd import ChoiceSets, PositionBias, PositionBuckets, distillation_loss

    sizes, far = sets_of(pad, False)
    off = offsets_of(sizes)
    n = int(off[-1])
    z, keep = np.zeros(n, np.float32), np.ones(n, bool)
    index, value = np.full((len(sizes), 6), -1), np.zeros((len(sizes), 6))
    for g in far:
        z[off[g]: off[g + 1]] = np.concatenate([Z, np.full(pad, np.nan)])
        keep[off[g] + 5: off[g + 1]] = False
        keep[off[g] + 3] = False
        index[g], value[g, 1:] = [3] + ORDER, level + STEPS
    buckets = PositionBuckets(8, 16)
    pos = (np.arange(n) - np.repeat(off[:-1] + 2, sizes)).astype(np.int32)
    ids = buckets(pos).astype(np.int64)
    table = (np.arange(8) / 8.0).astype(np.float32)
    r = distillation_loss(torch.from_numpy(z).to(DEV), ChoiceSets(off), torch.from_numpy(index).int().to(DEV),
                          torch.from_numpy(value).float().to(DEV), tail=True, mask=torch.from_numpy(keep).to(DEV),
                          bias=PositionBias(torch.from_numpy(table).to(DEV), torch.from_numpy(pos).to(DEV), buckets))
    grad = r.grad_scores.double().cpu().numpy()
    by_bucket, room = np.zeros(8), np.zeros(8)
    for g in far:
        rows = off[g] + np.array(ORDER[1:])
        kl, want, kl_room, grad_room = closed(Z[ORDER[1:]] + table[ids[rows]], level + STEPS[1:])
        close(grad[rows], want, grad_room)
        assert abs(float(r.kl[g]) - kl) <= kl_room
        grad[rows] = 0.0
        np.add.at(by_bucket, ids[rows], want)
        np.add.at(room, ids[rows], grad_room + 4 * U)
    assert not grad.any()
    assert np.all(np.abs(r.grad_table.double().cpu().numpy() - by_bucket) <= room)


@pytest.mark.parametrize("pad", PADS)
@pytest.mark.parametrize("level", [-20.0, -60.0, -95.0, -110.0, -300.0, -700.0])
def test_small_list_beside_a_rest(hip, level, pad):
    """The list's sum is next to nothing and the rest has probability: nearly all of the teacher's is the rest's, and the
    listed rows keep the student's own gradient. Sets of weight 0 stay out of it."""
    from packboost_amd import ChoiceSets, distillation_loss

    sizes = [5 + pad, 9, 5 + pad, 5 + pad]
    off = offsets_of(sizes)
    z = np.zeros(int(off[-1]), np.float32)
    index, value = np.full((4, 3), -1), np.full((4, 3), -1.0)
    for g in (0, 2, 3):
        z[off[g]: off[g + 1]] = np.concatenate([Z, np.full(pad, -np.inf)])
        index[g], value[g] = [3, 0, 4], level + STEPS[:3]
    weights = np.array([1.0, 1.0, 0.0, 0.5])
    r = distillation_loss(torch.from_numpy(z).to(DEV), ChoiceSets(off), torch.from_numpy(index).int().to(DEV),
                          torch.from_numpy(value).float().to(DEV), tail=True, weights=torch.from_numpy(weights).float().to(DEV))
    grad = r.grad_scores.double().cpu().numpy()
    p, q = softmax(Z), np.exp(level + STEPS[:3])
    rho, pi = 1.0 - q.sum(), p[1] + p[2]
    kl = np.sum(q * (level + STEPS[:3] - np.log(p[[3, 0, 4]]))) + rho * (np.log(rho) - np.log(pi))
    want = p.copy()
    want[[3, 0, 4]] -= q
    want[1:3] -= rho * p[1:3] / pi
    for g in (0, 2, 3):
        assert abs(float(r.kl[g]) - kl) <= 2.0**-19 * (1 + abs(kl))
        close(grad[off[g]: off[g] + 5], weights[g] * want, weights[g] * 2.0**-18 * np.maximum(p, p / pi))
        assert not grad[off[g] + 5: off[g + 1]].any()


@pytest.mark.parametrize("pad", PADS)
def test_list_of_no_probability_in_64_bits(hip, pad):
    """Values whose exponentials are 0 in 64 bits: the teacher's entries have no probability, the set is left out."""
    from packboost_amd import ChoiceSets, distillation_loss

    for rows in ([3, 0, 4], ORDER):
        z = np.concatenate([Z, np.full(pad, -np.inf)]).astype(np.float32)
        value = torch.linspace(-800.0, -3e38, len(rows), device=DEV).view(1, -1)
        r = distillation_loss(torch.from_numpy(z).to(DEV), ChoiceSets([0, z.size]), torch.tensor([rows], dtype=torch.int32, device=DEV),
                              value, tail=True)
        assert float(r.loss) == 0 and float(r.kl[0]) == 0 and not r.grad_scores.any()


@pytest.mark.parametrize("pad", PADS)
def test_values_of_any_size(hip, pad):
    """Sums far above 1, NaN and infinities among the values: one entry takes all, or the set alone has no numbers."""
    from packboost_amd import ChoiceSets, distillation_loss

    def run(value):
        z = np.concatenate([Z, np.full(pad, -np.inf), Z]).astype(np.float32)
        r = distillation_loss(torch.from_numpy(z).to(DEV), ChoiceSets([0, 5 + pad, 10 + pad]),
                              torch.tensor([[3, 0], [3, 0]], dtype=torch.int32, device=DEV),
                              torch.tensor([value, [-1.0, -2.0]], device=DEV), tail=True)
        g = r.grad_scores.double().cpu().numpy()
        return float(r.kl[0]), g[:5], float(r.kl[1]), g[5 + pad:]

    p = softmax(Z)
    _, _, kl, grad = run([-1.0, -2.0])
    for value in ([3e38, -1.0], [3e38, -3e38], [1e30, 1e29], [800.0, 0.0]):
        a, g, b, h = run(value)
        assert abs(a + np.log(p[3])) <= 2.0**-20 and np.all(np.abs(g - (p - np.eye(5)[3])) <= 2.0**-19)
        assert b == kl and np.array_equal(h, grad)
    for value in ([math.nan, -1.0], [math.inf, -1.0]):
        a, g, b, h = run(value)
        assert math.isnan(a) and math.isnan(g[3]) and b == kl and np.array_equal(h, grad)


@pytest.mark.parametrize("pad", [0, 700, 9000])
def test_sharp_teacher_and_a_mask(hip, pad):
    """A teacher's own full lists at a low temperature, its best row masked for the student: values near -100."""
    from packboost_amd import ChoiceSets, choice_report, distillation_loss

    temperature = 0.0625
    teacher = np.array([8.0, 0.75, 1.125, 0.5, -0.625, 1.5])
    student = np.array([0.0, 0.25, -0.125, 0.375, 0.0, 0.125])
    tail = np.full(pad, -np.inf)
    off = offsets_of([6 + pad, 6 + pad])
    sets = ChoiceSets(off)
    row = lambda v: torch.from_numpy(np.concatenate([v, tail, v, tail]).astype(np.float32)).to(DEV)
    best = choice_report(row(teacher), sets, top=6, temperature=temperature)
    assert float(best.top_log_probs[0, 1:].max()) < -100
    keep = torch.ones(int(off[-1]), dtype=torch.bool, device=DEV)
    keep[[0, 6 + pad]] = False
    r = distillation_loss(row(student), sets, best.top_index, best.top_log_probs, tail=True, temperature=temperature, mask=keep)
    grad, kls = r.grad_scores.double().cpu().numpy(), r.kl.double().cpu().numpy()
    for g in range(2):
        listed = best.top_index[g, 1:].cpu().numpy()
        t = best.top_log_probs[g, 1:].double().cpu().numpy()
        p, q = softmax(student[listed] / temperature), softmax(t)
        kl = np.sum(q * (np.log(q) - np.log(p)))
        # logits over the temperature and values lie up to 40 apart: 2^-24 of that in an exponential
        room = 2.0**-22 + 40 * 2.0**-24
        assert abs(kls[g] - kl) <= 4 * room * (1 + abs(kl))
        assert np.all(np.abs(grad[off[g] + listed] - temperature * (p - q)) <= 4 * room * temperature * (p + q))
    assert np.isfinite(grad).all() and np.all(grad[[0, 6 + pad]] == 0)


def test_objective_with_a_sharp_teacher(hip):
    """A fit on such lists: its rounds' gradients are finite."""
    from packboost_amd import ChoiceSets, DistillationObjective, PackBoost, PackBoostConfig, choice_report

    r = np.random.default_rng(31)
    sizes = np.full(300, 5)
    off = offsets_of(sizes)
    X = r.standard_normal((1500, 4)).astype(np.float32)
    scores = torch.from_numpy((4 * X[:, 0]).astype(np.float32)).to(DEV)
    best = choice_report(scores, ChoiceSets(off), top=5, temperature=2.0**-5)
    mask = np.ones(1500, bool)
    mask[off[:-1] + best.top_index[:, 0].cpu().numpy()] = False
    assert float(best.top_log_probs[:, 1].min()) < -100
    obj = DistillationObjective(off, best.top_index, best.top_log_probs, tail=True, mask=mask, temperature=2.0**-5)
    cfg = PackBoostConfig(pack_size=2, max_depth=3, learning_rate=0.5, max_bins=16, min_samples_leaf=5, random_state=3)
    model = PackBoost(cfg).fit(X, None, np.repeat(np.arange(300) % 3, 5), num_rounds=4, objective=obj)
    assert np.isfinite(model.predict(X)).all()


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("pad", PADS)
@pytest.mark.parametrize("below", [-80.0, -95.0, -600.0])
def test_faint_entry_of_a_row_far_below(hip, below, pad, tail):
    """An entry whose probability is next to nothing counts where the student's is as far off: a row of the type's lowest
    value, and one of no probability, which makes the divergence infinite."""
    from packboost_amd import ChoiceSets, distillation_loss

    for low in (float(torch.finfo(torch.float32).min), -math.inf):
        z = np.concatenate([[0.0, low, 0.5, -1.0], np.full(pad, -np.inf)]).astype(np.float32)
        value = np.array([-0.5, below - 0.5])
        r = distillation_loss(torch.from_numpy(z).to(DEV), ChoiceSets([0, z.size]), torch.tensor([[0, 1]], dtype=torch.int32, device=DEV),
                              torch.from_numpy(value).float().view(1, 2).to(DEV), tail=tail)
        s = 1.0 + math.exp(0.5) + math.exp(-1.0)
        q = np.exp(value)
        rest = 0.0
        if tail:
            pi = (s - 1.0) / s
            rest = (1.0 - q.sum()) * (math.log(1.0 - q.sum()) - math.log(pi))
        else:
            q /= q.sum()
        near, far = q[0] * (math.log(q[0]) + math.log(s)) + rest, q[1] * (math.log(q[1]) + math.log(s) - low)
        assert float(r.kl[0]) == math.inf if low == -math.inf else abs(float(r.kl[0]) - near - far) <= 2.0**-20 * (4 + far)
        grad = r.grad_scores.double().cpu().numpy()
        p = np.array([1.0, 0.0, math.exp(0.5), math.exp(-1.0)]) / s
        want = p - [q[0], q[1], 0.0, 0.0]
        if tail:
            want[2:] -= (1.0 - q.sum()) * p[2:] / pi
        assert np.all(np.abs(grad[:4] - want) <= 2.0**-18) and not grad[4:].any()


@pytest.mark.parametrize("dtype,masked,biased", [("f32", True, True), ("bf16", False, False), ("f16", True, False), ("f32", False, False)])
@pytest.mark.parametrize("layout", list(LAYOUTS) + list(EDGES))
def test_lists_at_any_level(hip, layout, dtype, masked, biased):
    """Every layout, each set's values moved to a level of its own: next to nothing, their own, or far more than 1."""
    d = make({**EDGES, **LAYOUTS}[layout], dtype, masked, biased, seed=50)
    for k in (3, 64 if masked else 20):
        index, value = teacher_of(d, k, True, 1.5, 51)
        level = np.random.default_rng(52).choice([0.0, 0.0, -5.0, -60.0, -90.0, -200.0, -600.0, 5.0, 100.0], (len(d["size"]), 1))
        value = (value.double() + torch.from_numpy(level)).float()
        check_distill(d, k, True, 1.5, 53, lists=(index, value))
