"""The choice operators where their layout changes: sets at the sizes from which a tile, a wave, a
workgroup or several of them take a set, tables with many longer sets, runs that start anywhere in the
rows, and position lookups too long for on-chip memory. Bounds as in test_gpu_choices."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gpu_choices import (DEV, U, back, bound_lp, check_grads, make, offsets_of, per_set, policy_inputs,
                              policy_reference, reference, same_or_close)

pytestmark = pytest.mark.gpu

rs = np.random.RandomState(11)
EDGES = {
    "tile_rows": [255, 256, 257, 503, 504, 505, 3, 506, 511, 512, 1],
    "tile_sets": [1] * 127 + [0] * 3 + [2] * 129 + [0] * 300 + [1],
    "wave_rows": [2039, 2040, 5, 2041, 2047, 2048, 1, 2049, 2050, 7, 2056],
    "group_rows": [8183, 3, 8184, 8185, 8191, 8192, 1, 8193, 8200],
    "parts": [16_367, 1, 16_368, 16_369, 24_553],
    "many": list(np.where(rs.rand(9000) < 0.5, rs.randint(257, 504, 9000), rs.randint(0, 6, 9000))),
    "mixture": list(np.exp(1.8 * rs.randn(3000) + 4).astype(int)),
}


@pytest.mark.parametrize("dtype,masked,biased", [("f32", True, True), ("bf16", False, False), ("f16", True, False)])
@pytest.mark.parametrize("edges", list(EDGES))
def test_every_operator(hip, edges, dtype, masked, biased):
    from packboost_amd import choice_log_probs, choice_log_probs_backward, policy_loss

    d = make(EDGES[edges], dtype, masked, biased, seed=21)
    kw = dict(mask=d["mask"], bias=d["bias"])
    p, lp, lse, ok, step, at = reference(d)
    tol = bound_lp(d)
    rows, got_lse = choice_log_probs(d["scores"], d["sets"], **kw)
    same_or_close(rows, lp, tol)
    same_or_close(got_lse, lse, tol)
    steps, step_lse = choice_log_probs(d["scores"], d["sets"], chosen=d["chosen"], **kw)
    same_or_close(steps, step, tol)
    same_or_close(step_lse, lse, tol)
    up = d["r"].standard_normal(len(step)).astype(np.float32)
    gs, gt = choice_log_probs_backward(torch.from_numpy(up).to(DEV), d["scores"], step_lse, d["sets"], chosen=d["chosen"], **kw)
    g, size = back(d, p, ok, at, up.astype(np.float64))
    check_grads(d, gs, gt, g, size, tol)
    rows_up = d["r"].standard_normal(len(lp)).astype(np.float32)
    gs, gt = choice_log_probs_backward(torch.from_numpy(rows_up).to(DEV), d["scores"], step_lse, d["sets"], **kw)
    u = np.where(d["keep"], rows_up.astype(np.float64), 0.0)
    total = np.repeat(per_set(d, np.add, u, 0.0), d["size"])
    absolute = np.repeat(per_set(d, np.add, np.abs(u), 0.0), d["size"])
    check_grads(d, gs, gt, np.where(d["keep"], u - p * total, 0.0),
                np.abs(u) + p * absolute * (1 + 100 * U / (tol + 4 * U)), tol)
    v, low, high, kl = policy_inputs(d, step)
    dev = {k: torch.from_numpy(a).to(DEV) for k, a in v.items()}
    r = policy_loss(d["scores"], d["sets"], d["chosen"], **dev, clip=(low, high), kl_weight=kl, **kw)
    loss, _, clipped, slope, w = policy_reference(v, ok, step, low, high, kl, 1.0)
    same_or_close(r.log_probs, step, tol)
    gap = np.exp(v["ref_log_probs"] - step)
    term = w * (np.exp(step - v["old_log_probs"]) * np.abs(v["advantages"]) + kl * (gap + 1 + np.abs(np.log(gap))))
    room = (tol + 16 * U) * term
    assert abs(float(r.loss) - loss.sum()) <= room.sum() + U * abs(loss.sum())
    assert abs(float(r.clipped) - clipped.sum()) <= 4 * U * (1 + clipped.sum())
    g, size = back(d, p, ok, at, slope)
    _, extra = back(d, p, ok, at, room)
    check_grads(d, r.grad_scores, r.grad_table, g, size + extra / (tol + 4 * U), tol)


@pytest.mark.parametrize("shift", range(1, 8))
def test_tables_that_start_anywhere(hip, shift):
    """Scores, masks and positions at every offset from an aligned address: the values of aligned ones."""
    from packboost_amd import PositionBias, choice_log_probs, choice_log_probs_backward

    d = make([3, 700, 0, 41, 2600, 5], "f32" if shift % 2 else "bf16", True, True, seed=shift)
    n = d["scores"].numel()

    def moved(t):
        out = torch.zeros(n + 8, dtype=t.dtype, device=DEV)
        out[shift: shift + n] = t
        return out[shift: shift + n]

    bias = PositionBias(d["bias"].table, moved(d["bias"].positions), d["bias"].buckets)
    want = choice_log_probs(d["scores"], d["sets"], mask=d["mask"], bias=d["bias"])
    for scores, mask, b in ((moved(d["scores"]), d["mask"], d["bias"]), (d["scores"], moved(d["mask"]), d["bias"]),
                            (d["scores"], d["mask"], bias), (moved(d["scores"]), moved(d["mask"]), bias)):
        got = choice_log_probs(scores, d["sets"], mask=mask, bias=b)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    up = torch.from_numpy(d["r"].standard_normal(n).astype(np.float32)).to(DEV)
    first = choice_log_probs_backward(up, d["scores"], want[1], d["sets"], mask=d["mask"], bias=d["bias"])
    again = choice_log_probs_backward(moved(up), moved(d["scores"]), want[1], d["sets"], mask=moved(d["mask"]), bias=bias)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_a_set_does_not_see_its_neighbours(hip):
    """NaN and infinities in the sets on either side, in every kind of item, leave a set as it is alone."""
    from packboost_amd import ChoiceSets, choice_log_probs

    for size in (1, 7, 64, 300, 505, 2040, 3001, 9000):
        s = torch.randn(size, device=DEV)
        alone, alone_lse = choice_log_probs(s, ChoiceSets([0, size]))
        for before, after in ((3, 5), (600, 1), (13, 2100)):
            wide = torch.cat([torch.full((before,), float("nan"), device=DEV), s,
                              torch.full((after,), float("inf"), device=DEV)])
            lp, lse = choice_log_probs(wide, ChoiceSets(offsets_of([before, size, after])))
            # the sums' order may differ with the set's place in a tile: each is within the bound of the formula's
            room = 2 * U * (4 * float(s.abs().max()) + 100)
            assert float((lp[before: before + size] - alone).abs().max()) <= room
            assert torch.isnan(lse[0]) and torch.isnan(lse[2]) and abs(float(lse[1] - alone_lse[0])) <= room


@pytest.mark.parametrize("reach", [1023, 1024, 5000])
def test_long_lookups(hip, reach):
    from packboost_amd import ChoiceSets, PositionBias, PositionBuckets, choice_log_probs

    r = np.random.default_rng(reach)
    sizes = [6000, 40, 3, 700]
    off = offsets_of(sizes)
    n = int(off[-1])
    pos = r.integers(-6000, 6000, n).astype(np.int32)
    pb = PositionBuckets(64, reach)
    table = r.standard_normal(64).astype(np.float32)
    s = r.standard_normal(n).astype(np.float32)
    x = s.astype(np.float64) + table[pb(pos)]
    lp, lse = choice_log_probs(torch.from_numpy(s).to(DEV), ChoiceSets(off),
                               bias=PositionBias(torch.from_numpy(table).to(DEV), torch.from_numpy(pos).to(DEV), pb))
    want = np.array([np.log(np.exp(x[a:b]).sum()) for a, b in zip(off[:-1], off[1:])])
    same_or_close(lse, want, U * (4 * np.abs(x).max() + 100))
    same_or_close(lp, x - np.repeat(want, sizes), U * (4 * np.abs(x).max() + 100))


def test_gradients_that_grow(hip):
    """Gradients of the table whose size rises by many powers of two along the rows, and falls again."""
    from packboost_amd import ChoiceSets, PositionBias, PositionBuckets, choice_log_probs, choice_log_probs_backward

    g = 40_000
    off = np.arange(g + 1, dtype=np.int64) * 3
    sets = ChoiceSets(off)
    s = torch.zeros(3 * g, device=DEV)
    pos = (np.arange(3 * g) % 3 - 1).astype(np.int32)
    pb = PositionBuckets(8, 4)
    bias = PositionBias(torch.zeros(8, device=DEV), torch.from_numpy(pos).to(DEV), pb)
    chosen = torch.zeros(g, dtype=torch.int32, device=DEV)
    _, lse = choice_log_probs(s, sets, chosen=chosen, bias=bias)
    i = np.arange(g)
    up = (2.0 ** ((i % 64) - 32)).astype(np.float32) * np.where(i % 2, -1, 1).astype(np.float32)
    _, gt = choice_log_probs_backward(torch.from_numpy(up).to(DEV), s, lse, sets, chosen=chosen, bias=bias)
    per = up.astype(np.float64)[:, None] * np.array([2 / 3, -1 / 3, -1 / 3])
    ids = pb(pos)
    want = np.bincount(ids, per.reshape(-1), minlength=8)
    # a row's gradient: 8 units of itself; a rounding of the sums: 2^-30 of the largest gradient a row
    room = np.bincount(ids, 8 * U * np.abs(per).reshape(-1), minlength=8) + np.bincount(ids, minlength=8) * np.abs(per).max() * 2.0 ** -30
    assert np.all(np.abs(gt.double().cpu().numpy() - want) <= room + U * np.abs(want))


def test_sets_may_go_before_the_call_ends(hip):
    from packboost_amd import ChoiceSets, choice_log_probs

    n = 20_000_000
    s = torch.zeros(n, device=DEV)
    lp, lse = choice_log_probs(s, ChoiceSets(np.arange(0, n + 1, 1000)))
    assert torch.allclose(lse, torch.full_like(lse, float(np.log(1000))), atol=1e-5)
    assert float(lp[-1]) == pytest.approx(-np.log(1000), abs=1e-5)
