"""Fits on choices and preferences: the rounds take the objective's gradients, whatever the order of the
eras, in either fit mode; the position bias is learned beside the trees; bad inputs are refused."""

from __future__ import annotations

import math
import warnings

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

KEYS = ("feature", "threshold", "left", "right", "value", "is_leaf")


def config(**kw):
    from packboost_amd import PackBoostConfig

    base = dict(pack_size=2, max_depth=4, learning_rate=0.1, min_samples_leaf=5, max_bins=16, random_state=3)
    return PackBoostConfig(**{**base, **kw})


def decisions(sets=400, features=8, eras=5, seed=0):
    """Lists of 2 to 7 candidates whose choice follows two features and the place in the list."""
    r = np.random.default_rng(seed)
    size = r.integers(2, 8, sets)
    off = np.concatenate([[0], np.cumsum(size)])
    n = int(off[-1])
    X = r.standard_normal((n, features)).astype(np.float32)
    place = (np.arange(n) - np.repeat(off[:-1], size)).astype(np.int32)
    utility = 1.5 * X[:, 0] - X[:, 3] - 0.6 * place
    noisy = utility + r.gumbel(size=n)
    chosen = np.array([int(np.argmax(noisy[a:b])) for a, b in zip(off[:-1], off[1:])], dtype=np.int32)
    era = np.repeat(np.sort(r.integers(0, eras, sets)), size)
    return X, off, chosen, place, era, utility


def same_trees(a, b):
    assert len(a._rounds) == len(b._rounds)
    for x, y in zip(a._rounds, b._rounds):
        for k in KEYS:
            assert np.array_equal(np.asarray(x[k]), np.asarray(y[k])), k


def policy(off, chosen, seed=1, **kw):
    from packboost_amd import PolicyObjective

    r = np.random.default_rng(seed)
    size = np.diff(off)
    adv = np.where(r.random(size.size) < 0.8, 1.0, -0.3)
    old = -np.log(np.maximum(size, 1))
    return PolicyObjective(off, chosen, adv, old, ref_log_probs=old, kl_weight=0.02, clip=(0.5, 4.0), **kw)


def test_first_round_is_the_squared_loss_of_the_gradients(hip):
    """From zero predictions, a round on given gradients g and a squared-loss round on y = -g are the same
    arithmetic: grad = 0 - (-g)."""
    from packboost_amd import PackBoost

    X, off, chosen, place, era, _ = decisions()
    for objective in (policy(off, chosen), policy(off, chosen, positions=place, mask=place < 6)):
        model = PackBoost(config()).fit(X, None, era, num_rounds=1, objective=objective)
        objective.bind(None, len(X), torch.device("cuda", 0))
        loss, g = objective.gradient(torch.zeros(len(X), device="cuda"))
        objective.release()
        assert model.round_metrics[0]["train_loss"] == float(loss)
        plain = PackBoost(config()).fit(X, -g.cpu().numpy(), era, num_rounds=1)
        same_trees(model, plain)


def test_policy_learns(hip):
    from packboost_amd import ChoiceSets, PackBoost, choice_log_probs

    X, off, chosen, place, era, utility = decisions(sets=1500)
    objective = policy(off, chosen, positions=place, bias_rate=0.3)
    model = PackBoost(config()).fit(X, None, era, num_rounds=40, objective=objective)
    losses = [m["train_loss"] for m in model.round_metrics]
    assert losses[-1] < losses[0] and all(math.isfinite(v) for v in losses)
    # the learned bias falls with the place, as the choices were made
    ids = objective._buckets(np.arange(6))
    assert np.all(np.diff(objective.table[ids]) < 0)
    pred = model.predict(X)
    assert np.corrcoef(pred, 1.5 * X[:, 0] - X[:, 3])[0, 1] > 0.8
    # served: probabilities within each set
    lp, lse = choice_log_probs(torch.from_numpy(pred).to("cuda"), ChoiceSets(off))
    total = np.add.reduceat(np.exp(lp.double().cpu().numpy()), off[:-1])
    assert np.allclose(total, 1.0, atol=1e-5)


def test_preference_learns(hip):
    from packboost_amd import PackBoost, PreferenceObjective

    r = np.random.default_rng(4)
    X = r.standard_normal((3000, 6)).astype(np.float32)
    a, b = r.integers(0, 3000, 8000), r.integers(0, 3000, 8000)
    u = X[:, 1] - 2 * X[:, 4]
    first = u[a] - u[b] + r.logistic(size=8000) > 0
    w, l = np.where(first, a, b), np.where(first, b, a)
    era = r.integers(0, 4, 3000)  # unsorted eras
    model = PackBoost(config()).fit(X, u, era, num_rounds=40, objective=PreferenceObjective(w, l))
    assert model.round_metrics[0]["train_loss"] == pytest.approx(8000 * math.log(2), rel=1e-6)
    assert model.round_metrics[-1]["train_loss"] < 0.7 * 8000 * math.log(2)
    assert model.round_metrics[-1]["train_corr"] > 0.8
    assert np.corrcoef(model.predict(X), u)[0, 1] > 0.8


def shuffled_eras(off, era, seed=5):
    """A row order in which whole sets come in a random order."""
    r = np.random.default_rng(seed)
    sets = r.permutation(len(off) - 1)
    rows = np.concatenate([np.arange(off[g], off[g + 1]) for g in sets])
    # what a stable sort by era makes of it
    return sets, rows, rows[np.argsort(era[rows], kind="stable")]


def test_row_order_does_not_matter(hip):
    """Sets given in any order of their eras: the fit is that of the rows sorted by era beforehand."""
    from packboost_amd import ChoicePreferenceObjective, PackBoost, PreferenceObjective

    X, off, chosen, place, era, utility = decisions(sets=300)
    off = np.concatenate([off, off[-1:]])  # an empty set at the end
    chosen = np.concatenate([chosen, [0]]).astype(np.int32)
    size = np.diff(off)
    sets, rows, by_era = shuffled_eras(off, era)
    sorted_sets = [g for g in sets if size[g] == 0] + [g for g in
                   sorted((g for g in sets if size[g]), key=lambda g: (era[off[g]], list(sets).index(g)))]
    assert np.array_equal(by_era, np.concatenate([np.arange(off[g], off[g + 1]) for g in sorted_sets]))
    r = np.random.default_rng(6)
    adv, old = r.standard_normal(len(size)), -np.log(np.maximum(size, 1)) + 0.1 * r.standard_normal(len(size))
    mask = r.random(len(X)) > 0.1
    from packboost_amd import PolicyObjective

    def build(order, row_order, seqs=None):
        o = np.concatenate([[0], np.cumsum(size[order])])
        return PolicyObjective(o, chosen[order], adv[order], old[order], weights=np.abs(adv[order]), mask=mask[row_order],
                               positions=place[row_order])

    a = PackBoost(config()).fit(X[rows], None, era[rows], num_rounds=6, objective=build(sets, rows))
    b = PackBoost(config()).fit(X[by_era], None, era[by_era], num_rounds=6, objective=build(sorted_sets, by_era))
    same_trees(a, b)
    # pairs of rows
    w, l = r.integers(0, len(X), 500), r.integers(0, len(X), 500)
    where = lambda order: np.argsort(order)
    a = PackBoost(config()).fit(X[rows], None, era[rows], num_rounds=4,
                                objective=PreferenceObjective(where(rows)[w], where(rows)[l], ref_scores=utility[rows]))
    b = PackBoost(config()).fit(X[by_era], None, era[by_era], num_rounds=4, objective=PreferenceObjective(
        where(by_era)[w], where(by_era)[l], ref_scores=utility[by_era]))
    same_trees(a, b)
    # sequences of three sets, whose steps the era order takes apart: the loss at zero predictions is the
    # sequences' own
    o = np.concatenate([[0], np.cumsum(size[sets])])
    seq = np.arange(0, len(size) + 1, 3) if len(size) % 3 == 0 else np.append(np.arange(0, len(size), 3), len(size))
    s = len(seq) - 1
    cw, cl = r.integers(0, s, 50), r.integers(0, s, 50)
    ref = old.astype(np.float32)
    obj = ChoicePreferenceObjective(o, chosen[sets], seq, cw, cl, ref_log_probs=ref[sets])
    m = PackBoost(config()).fit(X[rows], None, era[rows], num_rounds=2, objective=obj)
    lp = np.where(size[sets] > 0, -np.log(np.maximum(size[sets], 1)), 0.0) - ref[sets].astype(np.float64)
    val = np.array([lp[b0:b1].sum() for b0, b1 in zip(seq[:-1], seq[1:])])
    want = np.logaddexp(0, -0.1 * (val[cw] - val[cl])).sum()
    assert m.round_metrics[0]["train_loss"] == pytest.approx(want, rel=1e-5)
    assert m.round_metrics[1]["train_loss"] < m.round_metrics[0]["train_loss"]


def test_choice_preference_first_gradient(hip):
    """The gradient of sequences out of era order against differences of the formula in 64 bits."""
    from packboost_amd import ChoicePreferenceObjective

    X, off, chosen, place, era, _ = decisions(sets=12, eras=3, seed=9)
    size = np.diff(off)
    sets, rows, by_era = shuffled_eras(off, era, seed=2)
    o = np.concatenate([[0], np.cumsum(size[sets])])
    seq = np.array([0, 2, 5, 6, 12])
    w, l = np.array([0, 1, 2, 3]), np.array([1, 2, 3, 0])
    c = chosen[sets]
    obj = ChoicePreferenceObjective(o, c, seq, w, l, beta=0.7, label_smoothing=0.1)
    perm = np.argsort(era[rows], kind="stable")
    obj.bind(perm, len(X), torch.device("cuda", 0))
    p = np.random.default_rng(1).standard_normal(len(X)).astype(np.float32)  # by the caller's rows
    loss, g = obj.gradient(torch.from_numpy(p[perm]).to("cuda"))
    got = np.empty(len(X))
    got[perm] = g.cpu().numpy()
    obj.release()

    def f(x):
        lp = np.array([x[a + k] - np.log(np.exp(x[a:b]).sum()) for a, b, k in zip(o[:-1], o[1:], c)])
        v = np.array([lp[a:b].sum() for a, b in zip(seq[:-1], seq[1:])])
        z = 0.7 * (v[w] - v[l])
        return np.sum(0.9 * np.logaddexp(0, -z) + 0.1 * np.logaddexp(0, z))

    x = p.astype(np.float64)
    assert float(loss) == pytest.approx(f(x), rel=1e-5)
    h = 1e-5  # central differences in 64 bits: good to about 1e-9; the float32 gradient to about 1e-5
    for i in range(len(X)):
        e = np.zeros_like(x)
        e[i] = h
        assert abs((f(x + e) - f(x - e)) / (2 * h) - got[i]) < 2e-5


def test_fit_modes_agree(hip, monkeypatch):
    from packboost_amd import PackBoost

    X, off, chosen, place, era, _ = decisions(sets=500)
    models = []
    for mode in ("planes", "segments"):
        monkeypatch.setenv("PB_FIT_MODE", mode)
        monkeypatch.setenv("PB_SEG_FROM_DEPTH", "1")
        models.append(PackBoost(config(max_bins=32)).fit(X, None, era, num_rounds=5,
                                                         objective=policy(off, chosen, positions=place)))
        assert models[-1]._fit_mode == mode
    same_trees(*models)


def test_root_that_cannot_split(hip):
    from packboost_amd import PackBoost, PreferenceObjective

    X = np.random.default_rng(0).standard_normal((8, 3)).astype(np.float32)
    m = PackBoost(config(min_samples_leaf=20)).fit(X, None, None, num_rounds=2, objective=PreferenceObjective([0, 1], [2, 3]))
    assert len(m._rounds) == 2 and m.round_metrics[0]["train_loss"] == pytest.approx(2 * math.log(2), rel=1e-6)
    assert np.all(m.predict(X) == 0.0)  # the pairs' gradients cancel in the one leaf


def test_gradients_that_are_not_finite(hip):
    """A loss that overflows ends the fit as non-finite squared-loss gradients do; a truncated fit keeps
    the position bias of its finite rounds."""
    from packboost_amd import PackBoost, PolicyObjective

    X, off, chosen, place, era, _ = decisions(sets=100)
    old = np.full(len(off) - 1, -1.0, np.float32)
    adv = np.ones(len(off) - 1, np.float32)
    adv[5] = np.inf

    def fit(policy_name):
        obj = PolicyObjective(off, chosen, adv, old, positions=place)
        model = PackBoost(config(), nonfinite=policy_name)
        return obj, model.fit(X, None, era, num_rounds=4, objective=obj)

    with pytest.raises(FloatingPointError):
        fit("raise")
    with warnings.catch_warnings(record=True) as caught:
        warnings.simplefilter("always")
        obj, model = fit("truncate")
    assert any("truncate" in str(w.message) for w in caught)
    assert len(model._rounds) == 0 and np.all(obj.table == 0.0)


def test_rewind(hip):
    X, off, chosen, place, era, _ = decisions(sets=50)
    obj = policy(off, chosen, positions=place)
    obj.bind(None, len(X), torch.device("cuda", 0))
    preds = torch.zeros(len(X), device="cuda")
    tables = []
    for _ in range(4):
        tables.append(obj._bias.table.clone())
        obj.gradient(preds)
    obj.rewind(2)
    assert torch.equal(obj._bias.table, tables[2]) and not torch.equal(tables[2], tables[3])
    obj.release()
    assert np.array_equal(obj.table, tables[2].cpu().numpy())


def test_refusals(hip):
    from packboost_amd import ChoicePreferenceObjective, PackBoost, PolicyObjective, PreferenceObjective

    X, off, chosen, place, era, _ = decisions(sets=30)
    g = len(off) - 1
    one = np.ones(g)
    fit = lambda obj, e=era: PackBoost(config()).fit(X, None, e, num_rounds=1, objective=obj)
    with pytest.raises(TypeError):
        fit(lambda p: p)
    with pytest.raises(ValueError, match="one era"):
        fit(PolicyObjective(off, chosen, one, one), np.arange(len(X)) % 2)
    with pytest.raises(ValueError, match="rows"):
        fit(PolicyObjective(off[:-1], chosen[:-1], one[:-1], one[:-1]))
    with pytest.raises(ValueError, match="name rows"):
        fit(PreferenceObjective([0], [len(X)]))
    for bad in (lambda: PolicyObjective(off, chosen[:-1], one, one), lambda: PolicyObjective(off, chosen, one[1:], one),
                lambda: PolicyObjective(off[1:], chosen[1:], one[1:], one[1:]),
                lambda: ChoicePreferenceObjective(off, chosen, [0, 2], [0], [0]),
                lambda: PreferenceObjective([0], [1], weights=[1.0, 2.0])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(ValueError):
        fit(ChoicePreferenceObjective(off, chosen, [0, 10, g], [0], [2]))
    with pytest.raises(ValueError):
        fit(PreferenceObjective([0], [1], label_smoothing=2.0))
    fit(PolicyObjective(off, chosen, one, one))  # and the model still fits


def test_rows_as_a_list(hip):
    """Without targets, features in any form that a fit takes with them."""
    from packboost_amd import PackBoost, PreferenceObjective

    X = np.random.default_rng(2).standard_normal((200, 4)).astype(np.float32)
    obj = lambda: PreferenceObjective(np.arange(100), np.arange(100, 200))
    a, b = (PackBoost(config()).fit(t, None, None, num_rounds=2, objective=obj()) for t in (X, X.tolist()))
    same_trees(a, b)
