"""Reports on choices, their backward and distillation on the GPU against the formulas in 64 bits.

Tolerances. LP bounds a log-probability as in test_gpu_choices, with the logits over the temperature: 2^-24 * (4 max|z| / T +
100), and a probability within LP of itself. The entropy is log s - u / (T s), |u / (T s)| <= log n: the sums' terms are
within LP of themselves, so it is within LP (2 + log n). Its gradient h p (log p + H) is then within |h| p LP
(|log p + H| + 3 + log n). A divergence sum q (log q - log p) + rho (log rho - log pi) has q and rho from the given
values in double, so it is within LP (its weights sum to 1) and 16 units of its terms; rho is a difference, good to
2^-40. A listed row's gradient w (p - q) is within w (p + q) LP, another's w r (pi - rho) within w r (pi + rho) LP, each
plus 4 units; 16-bit types add half a step."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from test_gpu_choice_layouts import EDGES
from test_gpu_choices import DEV, LAYOUTS, U, VARIANTS, bound_lp, check_grads, make, offsets_of, per_set, reference, same_or_close

pytestmark = pytest.mark.gpu


def heated(d, temperature):
    """The same inputs as their formulas see them: logits over the temperature."""
    return dict(d, x=d["x"] / temperature)


def logits32(d):
    """The logits as float32: what orders the rows."""
    z = d["scores"].float().cpu().numpy().copy()
    if d["bias"] is not None:
        z = z + d["bias"].table.cpu().numpy()[d["ids"]]
    assert z.dtype == np.float32
    return np.where(d["keep"], z, -np.inf).astype(np.float32)


def best_rows(d, k):
    """int64 [sets, k] by sorting each set: larger first, NaN above all, equal ones by index."""
    z, off = logits32(d), d["off"]
    out = np.full((len(d["size"]), k), -1, dtype=np.int64)
    for g in range(len(d["size"])):
        x = z[off[g]: off[g + 1]]
        key = np.where(np.isnan(x), np.inf, x.astype(np.float64))
        order = np.lexsort((np.arange(x.size), -key, ~np.isnan(x)))
        order = order[x[order] != -np.inf][:k]
        out[g, : order.size] = order
    return out


def entropy_of(d, p, lp):
    t = np.where(p > 0, -p * np.where(p > 0, lp, 0.0), 0.0)
    return per_set(d, np.add, t, 0.0)


def log_size(d):
    return np.log(np.maximum(d["size"], 1))


def check_report(d, k, temperature, seed=0):
    from packboost_amd import choice_report

    kw = dict(mask=d["mask"], bias=d["bias"], temperature=temperature)
    h = heated(d, temperature)
    p, lp, lse, ok, step, at = reference(h)
    tol = bound_lp(h)
    r = choice_report(d["scores"], d["sets"], chosen=d["chosen"], top=k, **kw)
    same_or_close(r.log_probs, step, tol)
    same_or_close(r.lse, lse, tol)
    want = entropy_of(d, p, lp)
    assert np.all(np.abs(r.entropy.double().cpu().numpy() - want) <= tol * (2 + log_size(d)))
    best = best_rows(d, k)
    assert np.array_equal(r.top_index.cpu().numpy(), best)
    n = len(lp)
    row = np.clip(d["off"][:-1, None] + best, 0, max(n - 1, 0))
    same_or_close(r.top_log_probs, np.where(best < 0, -np.inf, lp[row] if n else 0.0), tol)
    bare = choice_report(d["scores"], d["sets"], **kw)
    assert bare.log_probs is None and bare.top_index is None and bare.top_log_probs is None
    assert torch.equal(bare.entropy, r.entropy) and torch.equal(bare.lse, r.lse)
    return r


@pytest.mark.parametrize("dtype,masked,biased", VARIANTS)
@pytest.mark.parametrize("layout", list(LAYOUTS))
def test_report(hip, layout, dtype, masked, biased):
    k, temperature = {"f32": (8, 1.0), "bf16": (64, 0.7), "f16": (1, 2.5)}[dtype]
    check_report(make(LAYOUTS[layout], dtype, masked, biased, seed=2), k, temperature)


@pytest.mark.parametrize("k", [1, 2, 3, 5, 17, 32, 33, 63, 64])
@pytest.mark.parametrize("edges", ["tile_rows", "tile_sets", "wave_rows", "group_rows", "mixture"])
def test_report_lists(hip, edges, k):
    check_report(make(EDGES[edges], "bf16" if k & 1 else "f32", k % 3 == 0, k % 4 == 0, seed=k), k, 1.0)


@pytest.mark.parametrize("lead", [0, 1, 5])
def test_empty_sets_behind_full_tiles(hip, lead):
    """A tile that is full to its last row, a longer set, and empty sets that still belong to the tile: they lie past its
    rows. A few of each, and more tiles than workgroups share."""
    for times in (3, 1100):
        d = make(([500, 12] if lead == 0 else [lead, 500, 11 - lead] if lead == 1 else [lead, 490, 16]) + ([603, 0, 0, 512, 0, 13, 498, 700, 0] * times)
                 + [2], "f32", True, False, seed=lead)
        check_report(d, 3, 1.0)
        check_backward(d, 1.0)
        check_distill(d, 3, True, 1.0, lead)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("sizes", [[300, 7, 0, 3000, 1], [9000, 40], [70_001], [20, 20, 500, 2047]])
def test_report_ties(hip, sizes, dtype):
    """Rows of few values, all of one value, both zeros, and lists longer than their sets."""
    from packboost_amd import ChoiceSets, choice_report

    off = offsets_of(sizes)
    n = int(off[-1])
    r = np.random.default_rng(n)
    for kind in range(4):
        x = [r.integers(0, 3, n) - 1.0, np.zeros(n), np.where(r.random(n) < 0.5, 0.0, -0.0), r.integers(0, n // 3 + 2, n) / 64.0][kind]
        z = torch.from_numpy(x.astype(np.float32)).to({"f32": torch.float32, "bf16": torch.bfloat16}[dtype])
        got = choice_report(z.to(DEV), ChoiceSets(off), top=50).top_index.cpu().numpy()
        v = z.float().numpy()
        for g in range(len(sizes)):
            order = np.argsort(-v[off[g]: off[g + 1]], kind="stable")[:50]
            assert np.array_equal(got[g, : order.size], order) and np.all(got[g, order.size:] == -1), (kind, g)


@pytest.mark.parametrize("sizes", [[6, 3, 4, 5], [700, 6, 300, 9000], [40_000, 30_000, 600, 70_000]])
def test_report_of_what_is_not_finite(hip, sizes):
    """NaN stands above all, -inf is not listed, infinities make NaN of their set alone."""
    from packboost_amd import ChoiceSets, choice_report

    off = offsets_of(sizes)
    z = np.linspace(-1, 1, int(off[-1])).astype(np.float32)
    z[off[0] + 4], z[off[0] + 2] = np.nan, -np.nan
    z[off[1]: off[2]] = -np.inf
    z[off[2]: off[3] - 2] = -np.inf
    z[off[3] + 1] = np.inf
    r = choice_report(torch.from_numpy(z).to(DEV), ChoiceSets(off), top=3, chosen=torch.zeros(4, dtype=torch.int32, device=DEV))
    top, lp = r.top_index.cpu().numpy(), r.top_log_probs.cpu().numpy()
    assert list(top[0]) == [2, 4, sizes[0] - 1] and np.all(np.isnan(lp[0]))
    assert list(top[1]) == [-1, -1, -1] and np.all(lp[1] == -np.inf)
    assert list(top[2]) == [sizes[2] - 1, sizes[2] - 2, -1] and np.all(np.isfinite(lp[2, :2])) and lp[2, 2] == -np.inf
    assert top[3, 0] == 1 and np.all(np.isnan(lp[3]))
    h, lse, step = (v.cpu().numpy() for v in (r.entropy, r.lse, r.log_probs))
    assert np.isnan(h[0]) and h[1] == 0 and np.isfinite(h[2]) and np.isnan(h[3])
    assert np.isnan(lse[0]) and lse[1] == -np.inf and np.isfinite(lse[2])
    assert np.isnan(step[0]) and step[1] == 0 and step[2] == -np.inf and np.isnan(step[3])


@pytest.mark.parametrize("dtype,masked,biased", [("f32", True, True), ("bf16", False, False), ("f16", True, False)])
@pytest.mark.parametrize("few", [1, 256, 4096, 4097])
def test_few_short_sets_beside_longer_ones(hip, few, dtype, masked, biased):
    """Up to 4096 short sets are taken by the waves of the longer ones, more by tiles; empty ones, single rows and the
    largest that are short are among them."""
    r = np.random.default_rng(few)
    short = ([0, 1, 504, 505 - 1, 2, 0] + r.integers(0, 120, 4100).tolist())[:few] if few > 1 else [5]
    sizes = short[: few // 2] + [700, 20_000] + short[few // 2:] + [9000, 2500]
    d = make(sizes, dtype, masked, biased, seed=few)
    check_report(d, 6, 1.0)
    check_backward(d, 1.3)
    check_distill(d, 6, few % 2 == 0, 1.0, few)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size,temperature", [(24.0, 2.0**-20), (24.0, 2.0**-15), (-1.5 * 2**30, 1.0), (1.5 * 2**100, 2.0**20),
                                              (-1.5 * 2**100, 2.0**-20), (2.0**31, 1.0)])
def test_large_logits_over_the_temperature(hip, size, temperature, dtype):
    """Sets' rows are z or lie below it by |z| 2^-6 and more, which over the temperature is 10^4 and more: a set is the
    uniform distribution over its best rows. The exponents' common rounding, up to S = 2^-24 |z / T| in lanes' sums of 64
    rows and more each, leaves an entropy within 130 * 2^-24 S as long as S < 2^7, and nothing beyond."""
    from packboost_amd import ChoiceSets, choice_report, choice_report_backward, distillation_loss

    sizes = [3, 300, 1, 1500, 7000, 31_000, 60_000, 140_000]
    sets = ChoiceSets(offsets_of(sizes), device=DEV)
    r = np.random.default_rng(5)
    step = r.integers(0, 4, sum(sizes)) / 64.0
    off = np.concatenate([[0], np.cumsum(sizes)])
    step[off[:-1]] = 0.0
    z = size * (1.0 + step * (1 if size < 0 else -1))
    x = torch.from_numpy(z).to(DEV).to({"f32": torch.float32, "bf16": torch.bfloat16}[dtype])
    assert np.array_equal(x.double().cpu().numpy(), z)
    best = np.add.reduceat((step == 0).astype(np.float64), off[:-1])
    chosen = torch.zeros(len(sizes), dtype=torch.int32, device=DEV)
    rep = choice_report(x, sets, chosen=chosen, temperature=temperature)
    shift = abs(size) / temperature * 2.0**-24
    tol = 2.0**-20 + (130 * 2.0**-24 * shift if shift < 2**8 else 0.0)
    assert np.all(np.abs(rep.entropy.double().cpu().numpy() - np.log(best)) <= tol)
    assert np.all(np.abs(rep.log_probs.double().cpu().numpy() + np.log(best)) <= tol)
    lse = rep.lse.double().cpu().numpy()
    assert np.all(np.abs(lse - size / temperature - np.log(best)) <= 2.0**-22 * abs(size / temperature))
    ones = torch.ones(len(sizes), device=DEV)
    p = np.where(step == 0, 1.0 / np.repeat(best, sizes), 0.0)
    at = np.zeros(len(z))
    at[off[:-1]] = 1.0
    half = 2.0**-8 if dtype == "bf16" else 0.0
    gs, _ = choice_report_backward(ones, None, x, sets, chosen=chosen, temperature=temperature)
    want = (at - p) / temperature
    assert np.all(np.abs(gs.double().cpu().numpy() - want) <= (tol + half) * (at + p) / temperature)
    # the entropy's gradient is p (log p + H) / T, and log p + H is 0 but for the roundings of both
    gs, _ = choice_report_backward(None, ones, x, sets, temperature=temperature)
    assert np.all(np.abs(gs.double().cpu().numpy()) <= 2 * tol * p / temperature)
    # a teacher that names the first row, and one other
    index = torch.zeros((len(sizes), 2), dtype=torch.int32, device=DEV)
    index[:, 1] = -1
    value = torch.zeros((len(sizes), 2), device=DEV)
    for tail in (False, True):
        loss, gs, _, _ = distillation_loss(x, sets, index, value if not tail else value - 1.0 / 1024, tail=tail,
                                           temperature=temperature)
        if not tail:
            assert abs(float(loss) / temperature**2 - np.log(best).sum()) <= len(sizes) * tol
            assert np.all(np.abs(gs.double().cpu().numpy() / temperature**2 + want) <= (tol + half) * (at + p) / temperature)
        assert torch.isfinite(gs).all()


def check_backward(d, temperature, which="both"):
    from packboost_amd import choice_report_backward

    h = heated(d, temperature)
    p, lp, lse, ok, step, at = reference(h)
    tol = bound_lp(h)
    g = len(step)
    a, b = (d["r"].standard_normal(g).astype(np.float32) for _ in range(2))
    ga = torch.from_numpy(a).to(DEV) if which != "entropy" else None
    gb = torch.from_numpy(b).to(DEV) if which != "steps" else None
    gs, gt = choice_report_backward(ga, gb, d["scores"], d["sets"], chosen=d["chosen"] if ga is not None else None,
                                    mask=d["mask"], bias=d["bias"], temperature=temperature)
    coef = np.where(ok, a.astype(np.float64), 0.0) * (ga is not None)
    slope = np.repeat(b.astype(np.float64) * (gb is not None), d["size"])
    H = np.repeat(entropy_of(d, p, lp), d["size"])
    around = np.where(p > 0, np.where(p > 0, lp, 0.0) + H, 0.0)
    want = -p * np.repeat(coef, d["size"]) - slope * p * around
    size = np.abs(np.repeat(coef, d["size"])) * p + np.abs(slope) * p * (np.abs(around) + 3 + np.repeat(log_size(d), d["size"]))
    want[at[ok]] += coef[ok]
    size[at[ok]] += np.abs(coef[ok])
    want, size = np.where(d["keep"], want, 0.0) / temperature, np.where(d["keep"], size, 0.0) / temperature
    check_grads(d, gs, gt, want, size, tol)
    return gs, gt


@pytest.mark.parametrize("dtype,masked,biased", VARIANTS)
@pytest.mark.parametrize("layout", list(LAYOUTS))
def test_backward(hip, layout, dtype, masked, biased):
    temperature, which = {"f32": (1.0, "both"), "bf16": (0.6, "entropy"), "f16": (3.0, "both")}[dtype]
    check_backward(make(LAYOUTS[layout], dtype, masked, biased, seed=3), temperature, which)


@pytest.mark.parametrize("dtype,masked,biased", [("f32", True, True), ("bf16", False, False), ("f16", True, False)])
@pytest.mark.parametrize("edges", list(EDGES))
def test_backward_layouts(hip, edges, dtype, masked, biased):
    d = make(EDGES[edges], dtype, masked, biased, seed=4)
    check_backward(d, 1.7)
    check_backward(d, 1.0, "steps")


def teacher_of(d, k, tail, temperature, seed, dtype="f32", lost=0.1):
    """Lists of a teacher near the student, with entries absent, beyond their set, masked and named twice."""
    r = np.random.default_rng(seed)
    size, off, n = d["size"], d["off"], int(d["off"][-1])
    x = np.where(np.isfinite(d["x"]), d["x"], 0.0) + r.standard_normal(n)
    lse = per_set(d, np.logaddexp, x / temperature, -np.inf)
    index = np.full((len(size), k), -1, dtype=np.int64)
    value = np.full((len(size), k), -3.0)
    for g in range(len(size)):
        order = np.argsort(-x[off[g]: off[g + 1]], kind="stable")[:k]
        index[g, : order.size] = order
        t = x[off[g] + order]
        value[g, : order.size] = t / temperature - lse[g] - 1e-3 if tail else t + 100 * r.standard_normal()
    if k > 1:
        twice = r.random(index.shape) < 0.1
        index = np.where(twice, np.roll(index, 1, axis=1), index)
    index = np.where(r.random(index.shape) < lost, -1 - (r.random(index.shape) < 0.5) * 7, index)
    index = np.where(r.random(index.shape) < lost, size[:, None] + np.abs(index), index)
    t = torch.from_numpy(value.astype(np.float32)).to({"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype])
    return index.astype(np.int32), t


def divergence(d, index, value, tail, temperature, weights, scale):
    """(kl, loss, gradient, size of its terms, bound of the kl) in 64 bits, set by set."""
    h = heated(d, temperature)
    x, off, keep = h["x"], d["off"], d["keep"]
    n, sets = int(off[-1]), len(d["size"])
    kl, grad, size, terms = np.zeros(sets), np.zeros(n), np.zeros(n), np.zeros(sets)
    p, lp, *_ = reference(h)
    for g in range(sets):
        rows, t = [], []
        for j, i in enumerate(index[g]):
            if 0 <= i < d["size"][g] and keep[off[g] + i] and off[g] + i not in rows:
                rows.append(off[g] + i)
                t.append(value[g, j] if tail else value[g, j] / temperature)
        all_rows = np.arange(off[g], off[g + 1])
        rest = np.setdiff1d(all_rows[x[all_rows] > -np.inf], rows)
        if not rows or not np.any(x[all_rows] > -np.inf):
            continue
        t = np.array(t)
        if not tail:
            t = t - t.max()
        mass = np.exp(t).sum()
        rho = 1 - mass if tail and rest.size and mass < 1 else 0.0
        if rho == 0:
            t = t - np.log(mass)
        q, pi = np.exp(t), p[rest].sum()
        kl[g] = np.sum(q * (t - lp[rows]))
        terms[g] = np.sum(q * np.abs(t - lp[rows]))
        if rho > 0:
            kl[g] += rho * (np.log(rho) - np.log(pi))
            terms[g] += rho * abs(np.log(rho) - np.log(pi)) + 2.0 ** -16 * abs(np.log(rho) - np.log(pi) + 1)  # rho to 2^-40
        w = weights[g] * scale * temperature
        grad[rows], size[rows] = w * (p[rows] - q), abs(w) * (p[rows] + q)
        if rest.size:
            share = p[rest] / pi
            grad[rest], size[rest] = w * share * (pi - rho), abs(w) * share * (pi + rho)
    tol = bound_lp(h)
    factor = scale * temperature ** 2
    return kl, factor * np.sum(weights * kl), grad, size, tol + 16 * U * terms, tol


def check_distill(d, k, tail, temperature, seed=0, teacher="f32", weighted=True, scale=1.0, lists=None):
    from packboost_amd import distillation_loss

    index, value = teacher_of(d, k, tail, temperature, seed, teacher) if lists is None else lists
    r = np.random.default_rng(seed + 1)
    g = len(d["size"])
    w = r.random(g).astype(np.float32) if weighted else np.ones(g, np.float32)
    w[r.random(g) < 0.1 * weighted] = 0.0
    out = distillation_loss(d["scores"], d["sets"], torch.from_numpy(index).to(DEV), value.to(DEV), tail=tail,
                            weights=torch.from_numpy(w).to(DEV) if weighted else None, mask=d["mask"], bias=d["bias"],
                            temperature=temperature, scale=scale)
    kl, loss, grad, size, room, tol = divergence(d, index, value.double().numpy(), tail, temperature, w.astype(np.float64), scale)
    got = out.kl.double().cpu().numpy()
    assert np.all(np.abs(got - kl) <= room + U * np.abs(kl))
    total = scale * temperature ** 2 * np.sum(w * (room + U * np.abs(kl)))
    assert abs(float(out.loss) - loss) <= total + 2 * U * abs(loss)
    check_grads(d, out.grad_scores, out.grad_table, np.where(d["keep"], grad, 0.0), size, tol)
    return out


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype,masked,biased", VARIANTS)
@pytest.mark.parametrize("layout", list(LAYOUTS))
def test_distill(hip, layout, dtype, masked, biased, tail):
    k, temperature, teacher = {"f32": (8, 1.0, "f32"), "bf16": (64, 2.0, "bf16"), "f16": (1, 0.8, "f16")}[dtype]
    check_distill(make(LAYOUTS[layout], dtype, masked, biased, seed=5), k, tail, temperature, 6, teacher, scale=0.5)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("k", [2, 3, 16, 33])
@pytest.mark.parametrize("edges", ["tile_rows", "tile_sets", "wave_rows", "group_rows", "parts", "mixture"])
def test_distill_layouts(hip, edges, k, tail):
    d = make(EDGES[edges], "bf16" if k == 16 else "f32", k == 3, k == 33, seed=k)
    check_distill(d, k, tail, 1.5 if k == 2 else 1.0, k, weighted=k != 3)


LONG = [40_000, 3, 32_768, 70_001, 65_500, 0, 32_769, 900, 66_000, 9000]


@pytest.mark.parametrize("dtype,masked,biased,many", [("f32", False, False, 1030), ("bf16", True, False, 1020), ("f16", False, True, 12),
                                                      ("f32", True, False, 12), ("bf16", False, False, 0)])
def test_many_long_sets(hip, dtype, masked, biased, many):
    """So many long sets that each has a workgroup, longer ones in parts beside them; fewer, in parts; a handful."""
    d = make(list(np.random.RandomState(40).randint(8193, 8300, many)) + LONG, dtype, masked, biased, seed=41)
    check_backward(d, 1.0 if masked else 1.3)
    check_distill(d, 24, not masked, 1.0, 42)
    check_report(d, 24, 1.0)


@pytest.mark.parametrize("sizes", [[100_000, 700, 2_100_000], [1_200_000, 9000]])
def test_lists_of_parts_that_are_ordered(hip, sizes):
    """Rising, falling and equal scores: all of a set's best rows lie in one part, or each part has as good ones."""
    from packboost_amd import ChoiceSets, choice_report

    off = offsets_of(sizes)
    n = int(off[-1])
    for z in (np.arange(n), -np.arange(n), np.zeros(n), np.arange(n) % 4096):
        z = (z / 1e6).astype(np.float32)
        got = choice_report(torch.from_numpy(z).to(DEV), ChoiceSets(off), top=64).top_index.cpu().numpy()
        for g in range(len(sizes)):
            assert np.array_equal(got[g], np.argsort(-z[off[g]: off[g + 1]], kind="stable")[:64])


def test_distill_many_sets(hip):
    """Thousands of lists, a few of their sets empty or without candidates."""
    d = make(EDGES["many"], "f32", True, True, seed=9)
    check_distill(d, 5, True, 1.0, 10)
    check_distill(d, 4, False, 2.0, 11)


@pytest.mark.parametrize("pad", [0, 700, 9000, 70_000])
def test_distill_edges(hip, pad):
    """Lists that hold the whole set, masses of 1 and more, entries of no mass, none that count, and rows of -inf."""
    from packboost_amd import ChoiceSets, distillation_loss

    def run(z, index, value, tail, keep=None):
        z = np.concatenate([z, np.full(pad, -np.inf)]).astype(np.float32)  # rows without probability change nothing
        m = None if keep is None else torch.from_numpy(np.concatenate([keep, np.ones(pad, bool)])).to(DEV)
        r = distillation_loss(torch.from_numpy(z).to(DEV), ChoiceSets([0, z.size]), torch.tensor([index], dtype=torch.int32, device=DEV),
                              torch.tensor([value], device=DEV), tail=tail, mask=m)
        return float(r.loss), r.grad_scores.cpu().numpy()[: z.size - pad], r

    z = np.array([0.5, -0.25, 0.0], np.float32)
    p = np.exp(z.astype(np.float64)) / np.exp(z.astype(np.float64)).sum()
    ten = 10 * U
    # the list holds every row: no rest, whatever the sum leaves
    for value in ([-1.0, -2.0, -0.9], [-3.0, -4.0, -5.0], [0.5, 0.25, 0.125]):
        q = np.exp(value) / np.exp(value).sum()
        loss, grad, _ = run(z, [0, 1, 2], value, True)
        assert abs(loss - np.sum(q * np.log(q / p))) <= ten and np.all(np.abs(grad - (p - q)) <= ten)
    # a mass of 1 and more: divided by it, nothing left
    for value in ([0.0, -1.0], [0.3, 0.2]):
        q = np.exp(value) / np.exp(value).sum()
        loss, grad, _ = run(z, [2, 0], value, True)
        assert abs(loss - np.sum(q * np.log(q / p[[2, 0]]))) <= ten
        assert np.all(np.abs(grad - (p - np.array([q[1], 0, q[0]]))) <= ten)
    # an entry of no mass: its row is listed, with q = 0
    loss, grad, _ = run(z, [1, 0], [-math.inf, -0.5], True)
    q0 = math.exp(-0.5)
    assert abs(loss - (q0 * math.log(q0 / p[0]) + (1 - q0) * math.log((1 - q0) / p[2]))) <= ten
    assert np.all(np.abs(grad - [p[0] - q0, p[1], p[2] - (1 - q0)]) <= ten)
    # none that count, no mass at all, or a student without probability
    for index, value in (([-1, 3 + pad], [0.0, 0.0]), ([0, 1], [-math.inf, -math.inf])):
        for tail in (False, True):
            loss, grad, r = run(z, index, value, tail)
            assert loss == 0 and float(r.kl[0]) == 0 and not grad.any()
    loss, grad, _ = run(np.full(3, -np.inf), [0, 1], [-1.0, -1.0], True)
    assert loss == 0 and not grad.any()
    # a listed row of no probability makes the divergence infinite, the gradients stay
    loss, grad, _ = run(np.array([0.0, -np.inf, 0.0], np.float32), [1, 0], [math.log(0.25), math.log(0.5)], True)
    assert loss == math.inf and np.all(np.abs(grad - [0.0, -0.25, 0.25]) <= ten)
    # the mask takes entries out; the first of two that name a row counts
    loss, grad, _ = run(z, [2, 0], [-0.7, -1.1], False, np.array([True, True, False]))
    p2 = np.exp(z[:2].astype(np.float64)) / np.exp(z[:2].astype(np.float64)).sum()
    assert abs(loss + math.log(p2[0])) <= ten and np.all(np.abs(grad - [p2[0] - 1, p2[1], 0]) <= ten)
    a, b = run(z, [0, 0, 1, 0], [1.0, 9.0, 0.5, 3.0], False)[1], run(z, [0, 1], [1.0, 0.5], False)[1]
    assert np.all(np.abs(a - b) <= ten)


def test_distill_weight_zero_counts_for_nothing(hip):
    from packboost_amd import ChoiceSets, distillation_loss

    z = torch.tensor([0.0, -math.inf, 1.0, 2.0], device=DEV)
    r = distillation_loss(z, ChoiceSets([0, 2, 4]), torch.tensor([[1], [0]], dtype=torch.int32, device=DEV),
                          torch.zeros(2, 1, device=DEV), weights=torch.tensor([0.0, 1.0], device=DEV))
    assert float(r.kl[0]) == math.inf and not r.grad_scores[:2].any()
    assert abs(float(r.loss) - math.log(1 + math.e)) <= 8 * U


def test_gradients_against_differences(hip):
    """Both gradients along random directions against central differences of the formulas. The second derivatives of a
    step are below the set sizes, so the differences at 1e-4 are within 1e-6 of the derivative relative to the terms."""
    from packboost_amd import choice_report_backward

    d = make([5, 40, 700, 0, 3000], "f32", True, True, seed=12)
    r = np.random.default_rng(13)
    n, g = int(d["off"][-1]), len(d["size"])
    a, b = r.standard_normal(g), r.standard_normal(g)
    index, value = teacher_of(d, 6, True, 1.3, 14)
    w = np.ones(g)
    out = check_distill(d, 6, True, 1.3, weighted=False, lists=(index, value))
    gs, _ = choice_report_backward(torch.from_numpy(a.astype(np.float32)).to(DEV), torch.from_numpy(b.astype(np.float32)).to(DEV),
                                   d["scores"], d["sets"], chosen=d["chosen"], mask=d["mask"], bias=d["bias"], temperature=1.3)

    def bonus(x):
        p, lp, lse, ok, step, at = reference(dict(d, x=x / 1.3))
        return np.sum(a.astype(np.float32) * step + b.astype(np.float32) * entropy_of(d, p, lp))

    def loss(x):
        return divergence(dict(d, x=x), index, value.double().numpy(), True, 1.3, w, 1.0)[1]

    for f, grad in ((bonus, gs), (loss, out.grad_scores)):
        grad = grad.double().cpu().numpy()
        for _ in range(4):
            v = r.standard_normal(n)
            step = 1e-4
            diff = (f(d["x"] + step * v) - f(d["x"] - step * v)) / (2 * step)
            along = np.where(d["keep"], grad * v, 0.0)
            assert abs(diff - along.sum()) <= 2e-6 * (np.abs(along).sum() + 1)


@pytest.mark.parametrize("shift", [1, 3, 4])
def test_tables_that_start_anywhere(hip, shift):
    """Rows off their alignment, scores with a stride, columns of a wider table: the values of aligned ones."""
    from packboost_amd import PositionBias, choice_report, choice_report_backward, distillation_loss

    d = make([3, 700, 0, 41, 2600, 5, 9000], "f32" if shift == 3 else "bf16", True, True, seed=shift)
    n = d["scores"].numel()
    index, value = teacher_of(d, 7, True, 1.0, 15)

    def moved(t):
        out = torch.zeros(n + 8, dtype=t.dtype, device=DEV)
        out[shift: shift + n] = t
        return out[shift: shift + n]

    def strided(t):
        out = torch.zeros(n, 3, dtype=t.dtype, device=DEV)
        out[:, 1] = t
        return out[:, 1]

    def wide(t):
        out = torch.zeros(t.shape[0], 12, dtype=t.dtype, device=DEV)
        out[:, 2: 2 + t.shape[1]] = t
        return out[:, 2: 2 + t.shape[1]]

    def run(f, lists):
        bias = PositionBias(d["bias"].table, f(d["bias"].positions), d["bias"].buckets)
        kw = dict(mask=f(d["mask"]), bias=bias)
        z = f(d["scores"])
        rep = choice_report(z, d["sets"], chosen=d["chosen"], top=9, **kw)
        g = torch.linspace(-1, 1, len(d["size"]), device=DEV)
        gs, gt = choice_report_backward(g, g, z, d["sets"], chosen=d["chosen"], **kw)
        r = distillation_loss(z, d["sets"], *lists, tail=True, **kw)
        return [*rep, gs, gt, *r]

    lists = [torch.from_numpy(index).to(DEV), value.to(DEV)]
    base = run(lambda t: t, lists)
    for got in (run(moved, lists), run(strided, [wide(t) for t in lists])):
        for x, y in zip(got, base):
            assert torch.equal(x, y)


def test_no_sets_and_no_rows(hip):
    from packboost_amd import ChoiceSets, PositionBias, PositionBuckets, choice_report, choice_report_backward, distillation_loss

    for off in ([0], [0, 0, 0]):
        g, sets, none = len(off) - 1, ChoiceSets(off), torch.empty(0, device=DEV)
        bias = PositionBias(torch.ones(8, device=DEV), torch.empty(0, dtype=torch.int32, device=DEV), PositionBuckets(8, 16))
        r = choice_report(none, sets, top=3, bias=bias)
        assert r.top_index.shape == (g, 3) and torch.all(r.top_index == -1) and torch.all(r.entropy == 0)
        assert torch.all(r.lse == -math.inf)
        gs, gt = choice_report_backward(None, torch.ones(g, device=DEV), none, sets, bias=bias)
        assert gs.numel() == 0 and torch.equal(gt, torch.zeros(8, device=DEV))
        d = distillation_loss(none, sets, torch.zeros(g, 2, dtype=torch.int32, device=DEV), torch.zeros(g, 2, device=DEV), bias=bias)
        assert float(d.loss) == 0 and torch.equal(d.grad_table, torch.zeros(8, device=DEV)) and not d.kl.any()


def test_refusals(hip):
    from packboost_amd import ChoiceSets, choice_report, choice_report_backward, distillation_loss

    sets = ChoiceSets([0, 3, 5])
    z = torch.zeros(5, device=DEV)
    c, f = torch.zeros(2, dtype=torch.int32, device=DEV), torch.zeros(2, device=DEV)
    index, value = torch.zeros(2, 4, dtype=torch.int32, device=DEV), torch.zeros(2, 4, device=DEV)
    bad = [
        lambda: choice_report(z[:4], sets), lambda: choice_report(z.double(), sets), lambda: choice_report(z.cpu(), sets),
        lambda: choice_report(z, sets, top=65), lambda: choice_report(z, sets, top=-1),
        lambda: choice_report(z, sets, temperature=0.0), lambda: choice_report(z, sets, temperature=math.nan),
        lambda: choice_report(z, sets, temperature=math.inf), lambda: choice_report(z, sets, chosen=c.long()),
        lambda: choice_report(z, sets, chosen=c[:1]), lambda: choice_report(z, [0, 5]),
        lambda: choice_report_backward(f, None, z, sets), lambda: choice_report_backward(f[:1], None, z, sets, chosen=c),
        lambda: choice_report_backward(None, f.double(), z, sets), lambda: choice_report_backward(None, f, z, sets, temperature=-1.0),
        lambda: distillation_loss(z, sets, index, value[:1]), lambda: distillation_loss(z, sets, index.long(), value),
        lambda: distillation_loss(z, sets, index[:, :3], value), lambda: distillation_loss(z, sets, index[:, :0], value[:, :0]),
        lambda: distillation_loss(z, sets, index, value.double()), lambda: distillation_loss(z, sets, index.cpu(), value),
        lambda: distillation_loss(z, sets, index.repeat(1, 17), value.repeat(1, 17)),
        lambda: distillation_loss(z, sets, index, value, weights=f[:1]), lambda: distillation_loss(z, sets, index, value, scale=math.inf),
        lambda: distillation_loss(z, sets, index, value, temperature=2.0 ** 21), lambda: distillation_loss(z, sets, index[0], value[0]),
        lambda: distillation_loss(z, sets, index, value, mask=torch.ones(4, dtype=torch.bool, device=DEV)),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {k} was taken")
    sets.close()
    with pytest.raises(ValueError):
        choice_report(z, sets)


def test_lists_of_sets_too_long_are_refused(hip):
    """A set whose rows an int32 does not number: no list, before anything is read."""
    from packboost_amd import ChoiceSets, choice_report

    n = 2 ** 31
    sets = ChoiceSets([0, n])
    with pytest.raises(RuntimeError, match="2\\^31"):
        choice_report(torch.zeros(1, device=DEV).expand(n), sets, top=1)
    sets.close()


def test_replayed_and_beside_each_other(hip):
    """Captured calls replayed on new inputs, eager ones between; two streams at once, each with its own workspace."""
    from packboost_amd import choice_report, choice_report_backward, distillation_loss

    d = make([5, 300, 0, 2100, 9000, 40, 70_000], "f32", True, True, seed=20)
    index, value = (t.to(DEV) for t in (lambda p: (torch.from_numpy(p[0]), p[1]))(teacher_of(d, 9, True, 1.0, 21)))
    g = torch.linspace(-1, 1, len(d["size"]), device=DEV)
    kw = dict(mask=d["mask"], bias=d["bias"])

    def calls(z):
        rep = choice_report(z, d["sets"], chosen=d["chosen"], top=9, **kw)
        gs, gt = choice_report_backward(g, g, z, d["sets"], chosen=d["chosen"], **kw)
        return [*rep, gs, gt, *distillation_loss(z, d["sets"], index, value, tail=True, **kw)]

    z = d["scores"].clone()
    calls(z)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = calls(z)
    for k in range(4):
        z.copy_(d["scores"] + 0.25 * k)
        graph.replay()
        want = calls(z)
        torch.cuda.synchronize()
        for x, y in zip(held, want):
            assert torch.equal(x, y)
    streams = [torch.cuda.Stream() for _ in range(2)]
    inputs = [d["scores"], d["scores"] * 0.5]
    want = [calls(v) for v in inputs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(calls(inputs[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for out in got[k]:
            for x, y in zip(out, want[k]):
                assert torch.equal(x, y)


@pytest.mark.parametrize("dtype,masked", [("f32", True), ("bf16", False)])
@pytest.mark.parametrize("sizes", [[9000], [33_000], [65_530, 9001], [9000, 33_000] * 130, [0] * 4100 + [12_000, 40_000, 3]])
def test_long_sets_alone(hip, sizes, dtype, masked):
    """Sets of more than 8192 and at most 65536 rows with nothing else for the kernels of parts: one workgroup each, in
    one launch and in two, and beside tiles."""
    d = make(sizes, dtype, masked, False, seed=len(sizes))
    check_report(d, 9, 0.8)
    check_backward(d, 1.0)
    check_distill(d, 9, masked, 1.0, 3)


def test_long_sets_replayed_on_two_streams(hip):
    """Captured and eager calls at once, on layouts of one workgroup to a set and of few short sets beside longer ones."""
    from packboost_amd import choice_report, choice_report_backward, distillation_loss

    for sizes in ([30_000, 64_000, 9000], [7, 0, 30_000, 700, 5, 9000]):
        d = make(sizes, "bf16", False, False, seed=30)
        index, value = (t.to(DEV) for t in (lambda p: (torch.from_numpy(p[0]), p[1]))(teacher_of(d, 5, False, 1.0, 31)))
        g = torch.linspace(-1, 1, len(sizes), device=DEV)

        def calls(z):
            rep = choice_report(z, d["sets"], chosen=d["chosen"], top=5)
            gs, _ = choice_report_backward(g, g, z, d["sets"], chosen=d["chosen"])
            return [*rep, gs, *(v for v in distillation_loss(z, d["sets"], index, value) if v is not None)]

        z, other = d["scores"].clone(), d["scores"] * 0.5
        want_other = calls(other)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = calls(z)
        side = torch.cuda.Stream()
        for k in range(4):
            z.copy_(d["scores"] * (1.0 + 0.5 * k))
            want = calls(z)
            torch.cuda.synchronize()
            graph.replay()
            with torch.cuda.stream(side):
                got_other = calls(other)
            torch.cuda.synchronize()
            for x, y in [*zip(held, want), *zip(got_other, want_other)]:
                assert torch.equal(x, y)


def test_teacher_to_student(hip):
    """The run together: a report of the teacher's scores is what the student is distilled from; a student with the
    teacher's own scores has no divergence and no gradient."""
    from packboost_amd import choice_report, distillation_loss

    d = make([5, 300, 0, 2100, 9000, 40], "f32", True, True, seed=22)
    kw = dict(mask=d["mask"], bias=d["bias"], temperature=1.5)
    best = choice_report(d["scores"], d["sets"], top=12, **kw)
    tol = bound_lp(heated(d, 1.5))
    r = distillation_loss(d["scores"], d["sets"], best.top_index, best.top_log_probs, tail=True, **kw)
    # log-probabilities within tol on both sides: what is left of the rest differs by as much
    assert float(r.kl.abs().max()) <= 4 * tol and float(r.grad_scores.abs().max()) <= 8 * tol
    other = torch.zeros_like(d["scores"])
    r = distillation_loss(other, d["sets"], best.top_index, best.top_log_probs, tail=True, **kw)
    down = distillation_loss(other - 0.1 * r.grad_scores, d["sets"], best.top_index, best.top_log_probs, tail=True, **kw)
    assert float(down.loss) < float(r.loss)


def test_distillation_objective(hip):
    """Fits take the objective's gradients: those of distillation_loss at zero predictions, in the order of the eras."""
    from packboost_amd import DistillationObjective, PackBoost, PackBoostConfig, PositionBuckets, choice_report, distillation_loss

    r = np.random.default_rng(30)
    sizes = r.integers(1, 30, 400)
    off = offsets_of(sizes)
    n = int(off[-1])
    X = r.standard_normal((n, 6)).astype(np.float32)
    era = np.repeat(np.arange(400) % 5, sizes)  # a set's rows are of one era; eras interleave
    from packboost_amd import ChoiceSets

    scores = torch.from_numpy((2 * X[:, 0] - X[:, 2]).astype(np.float32)).to(DEV)
    best = choice_report(scores, ChoiceSets(off), top=6)
    pos = (np.arange(n) - np.repeat(off[:-1], sizes)).astype(np.int32)
    cfg = PackBoostConfig(pack_size=2, max_depth=3, learning_rate=0.5, max_bins=16, min_samples_leaf=5, random_state=3)
    for extra in ({}, dict(positions=pos, buckets=PositionBuckets(8, 32), mask=r.random(n) < 0.9, weights=r.random(400))):
        obj = DistillationObjective(off, best.top_index, best.top_log_probs, tail=True, **extra)
        model = PackBoost(cfg).fit(X, None, era, num_rounds=6, objective=obj)
        pred = model.predict(X)
        assert np.all(np.isfinite(pred)) and pred.std() > 0
        assert (obj.table is not None) == bool(extra)
    obj = DistillationObjective(off, best.top_index, best.top_log_probs, tail=True)
    perm = np.argsort(era, kind="stable")
    obj.bind(perm, n, torch.device("cuda", 0))
    loss, grad = obj.gradient(torch.zeros(n, device=DEV))
    want = distillation_loss(torch.zeros(n, device=DEV), ChoiceSets(off), best.top_index, best.top_log_probs, tail=True)
    assert abs(float(loss) - float(want.loss)) <= 16 * U * abs(float(want.loss))
    # sets at other places of the table are summed over other lanes
    assert np.all(np.abs(grad.cpu().numpy() - want.grad_scores.cpu().numpy()[perm]) <= 100 * U)
    obj.release()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("size", [3, 300, 700, 5000, 9000, 70_000])
def test_entropy_is_not_negative(hip, size, dtype):
    """Sets of one row with probability, by its score's or by the mask's word, and of one row far above the others: the
    entropy is 0 within its roundings, and never below."""
    from packboost_amd import ChoiceSets, choice_report

    r = np.random.default_rng(size)
    many = 64
    z = np.full((many, size), -np.inf)
    at = r.integers(0, size, many)
    z[np.arange(many), at] = 3 * r.standard_normal(many)
    sets = ChoiceSets(np.arange(many + 1) * size)
    for kind in ("lone", "masked", "far"):
        if kind == "far":
            z = np.where(np.isneginf(z), z[np.arange(many), at][:, None] - 30.0, z)
        x = torch.from_numpy(z if kind != "masked" else np.where(np.isneginf(z), 1.0, z)).to(DEV)
        mask = torch.from_numpy(~np.isneginf(z).reshape(-1)).to(DEV) if kind == "masked" else None
        x = x.to({"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype]).reshape(-1)
        for temperature in (1.0, 0.3):
            h = choice_report(x, sets, mask=mask, temperature=temperature).entropy
            # log(1) and u / s of one term are within 4 units of 0; e^-30 of 70 thousand others is 1e-8 times 30 at most
            assert float(h.min()) >= 0 and float(h.max()) <= 2.0**-21 + (3e-7 if kind == "far" else 0.0)
