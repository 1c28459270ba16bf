"""Pairs laid out on the device: every value's entries are found, in one order, from either side."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24


def draw(values, pairs, hubs, seed):
    r = np.random.default_rng(seed)
    w = np.minimum((r.random(pairs) ** (6 if hubs else 1) * values).astype(np.int64), values - 1)
    l = r.integers(0, values, pairs)  # some compare a value with itself
    return r, w, l


# around the entries of a wave and a workgroup, and around the digits that a value has
@pytest.mark.parametrize("values,pairs", [(1, 1), (1, 5000), (2, 31), (3, 32), (255, 33), (256, 511), (257, 512),
                                          (300, 513), (7, 2047), (65_535, 2048), (65_536, 2049), (65_537, 20_000),
                                          (100_003, 300_001), (70_001, 530_003), ((1 << 24) + 3, 4097)])
@pytest.mark.parametrize("hubs", [False, True])
def test_gradients(hip, values, pairs, hubs):
    """The slopes of a value's pairs, summed in double: each is below 1 and off by at most 40 U (margins of up to
    4 with one rounding, an exponential and a reciprocal of a few U), the sum is rounded once."""
    from packboost_amd import PreferencePairs, preference_loss

    r, w, l = draw(values, pairs, hubs, values + pairs)
    v = (2 * r.random(values) - 1).astype(np.float32)
    scores = torch.from_numpy(v).to(DEV)
    here = preference_loss(scores, PreferencePairs(torch.from_numpy(w).to(DEV), torch.from_numpy(l).to(DEV),
                                                   num_values=values), beta=1.0)
    there = preference_loss(scores, PreferencePairs(w, l, num_values=values), beta=1.0)
    for a, b in zip(here, there):
        assert torch.equal(a, b)
    z = v[w].astype(np.float64) - v[l]
    slope = -1.0 / (1.0 + np.exp(z))
    want, size = np.zeros(values), np.zeros(values)
    np.add.at(want, w, slope)
    np.add.at(want, l, -slope)
    np.add.at(size, w, 1.0)
    np.add.at(size, l, 1.0)
    got = here.grad.cpu().numpy()
    assert np.all(np.abs(got - want) <= 40 * U * size + U * np.abs(want))
    assert np.all(got[size == 0] == 0)
    assert np.all(np.abs(here.margins.cpu().numpy() - z) <= 4 * U)


def test_types_strides_and_streams(hip):
    from packboost_amd import PreferencePairs, preference_loss

    r, w, l = draw(500, 3000, True, 3)
    scores = torch.from_numpy(r.standard_normal(500).astype(np.float32)).to(DEV)
    want = preference_loss(scores, PreferencePairs(w, l, num_values=500))
    for dtype in (torch.int16, torch.int32, torch.int64):
        both = torch.from_numpy(np.stack([w, l], 1)).to(DEV, dtype)
        for pairs in (PreferencePairs(both[:, 0], both[:, 1], num_values=500),
                      PreferencePairs(both[:, 0], torch.from_numpy(l), num_values=500)):
            for a, b in zip(preference_loss(scores, pairs), want):
                assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pairs = PreferencePairs(torch.from_numpy(w).to(DEV) + 0, torch.from_numpy(l).to(DEV) + 0, num_values=500)
        got = preference_loss(scores, pairs)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("lengths", [[3, 0, 5, 1], [700, 2, 9000, 40]])
def test_sequences(hip, lengths):
    from packboost_amd import PreferencePairs, preference_loss

    off = np.concatenate([[0], np.cumsum(lengths)])
    w, l = np.array([0, 1, 2, 3, 0]), np.array([1, 2, 3, 0, 2])
    steps = torch.from_numpy(np.random.default_rng(1).standard_normal(off[-1]).astype(np.float32)).to(DEV)
    want = preference_loss(steps, PreferencePairs(w, l, offsets=off))
    got = preference_loss(steps, PreferencePairs(torch.from_numpy(w).to(DEV), torch.from_numpy(l).to(DEV), offsets=off))
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_none_and_refusals(hip):
    from packboost_amd import PreferencePairs, preference_loss

    none = torch.empty(0, dtype=torch.int64, device=DEV)
    out = preference_loss(torch.ones(4, device=DEV), PreferencePairs(none, none, num_values=4))
    assert float(out.loss) == 0 and torch.equal(out.grad, torch.zeros(4, device=DEV)) and out.margins.numel() == 0
    at = lambda *v: torch.tensor(v, device=DEV)
    for w, l, n in ((at(0, 3), at(1, 1), 3), (at(0, 1), at(1, -1), 3), (at(0, 1 << 40), at(1, 1), 3), (at(0), at(0), 0),
                    (at(0, 1), at(1), 3), (at(0.0), at(1), 3), (at(True), at(1), 3), (at(0).reshape(1, 1), at(1), 3)):
        with pytest.raises(ValueError):
            PreferencePairs(w, l, num_values=n)
