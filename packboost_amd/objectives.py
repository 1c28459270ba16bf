"""Objectives of PackBoost.fit beside the squared loss: choices and preferences.

An objective gives each round the gradient of its loss with respect to the training rows' predictions;
trees are grown on it as they are on preds - y (hessian 1 a row, so a leaf's value is the mean negative
gradient of its rows). Losses are sums over pairs or decisions, not means: a row's gradient does not
shrink with the table.

    PreferenceObjective          rows compared in pairs (a reward model, a ranker)
    ChoicePreferenceObjective    sequences of choices compared in pairs, against a reference model
    PolicyObjective              choices with advantages: the clipped policy loss with a KL term

The two objectives on choices can learn a position bias beside the trees: a bucket of positions is
fitted like a leaf, table -= bias_rate * (sum of its rows' gradients) / (number of its rows), each
round, and taken into account in the scores' gradients; the model's own predictions are free of it.
`table` holds it after the fit; a saved model holds the trees alone, so who serves with the bias keeps
`table` beside it.

Rows are the fit's, in the order they are passed in; a set's rows must be of one era (the fit sorts rows
by era, which keeps them together).
"""

from __future__ import annotations

import numpy as np
import torch

from .choices import (ChoiceSets, PositionBias, PositionBuckets, PreferencePairs, _host_int64, choice_log_probs,
                      choice_log_probs_backward, policy_loss, preference_loss)


def _array(name: str, v, n: int, dtype) -> np.ndarray:
    a = np.asarray(v.detach().cpu().numpy() if isinstance(v, torch.Tensor) else v)
    if a.shape != (n,):
        raise ValueError(f"{name} must hold {n} entries, got shape {a.shape}")
    return np.ascontiguousarray(a, dtype=dtype)


def _indices(name: str, v, n: int) -> np.ndarray:
    """int32 [n] of whole numbers that it holds."""
    a = np.asarray(v.detach().cpu().numpy() if isinstance(v, torch.Tensor) else v)
    if a.size and not np.issubdtype(a.dtype, np.integer):
        raise ValueError(f"{name} must be integers, got {a.dtype}")
    if a.size and (a.min() < -2 ** 31 or a.max() > 2 ** 31 - 1):
        raise ValueError(f"{name} must lie in int32's range")
    return _array(name, a, n, np.int32)


def _to(device: torch.device, a: np.ndarray | None) -> torch.Tensor | None:
    return None if a is None else torch.from_numpy(a).to(device)


class Objective:
    """What PackBoost.fit asks of an objective."""

    def bind(self, perm: np.ndarray | None, num_rows: int, device: torch.device) -> None:
        """Prepares for a fit whose row r is the caller's row perm[r] (None: r)."""
        raise NotImplementedError

    def gradient(self, preds: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """(loss, float32 gradient per row) at preds (float32 [rows]), on the current stream."""
        raise NotImplementedError

    def rewind(self, calls: int) -> None:
        """Forgets what `gradient` learned from its calls-th call on (at most two calls back)."""

    def release(self) -> None:
        """Frees what bind took."""


class PreferenceObjective(Objective):
    """Pairs of rows: the winner's prediction should lie above the loser's.

    winners, losers: row indices [pairs]; weights per pair; ref_scores: a reference model's scores per
    row, so that the margin is beta * ((s_w - ref_w) - (s_l - ref_l)) (see preference_loss)."""

    def __init__(self, winners, losers, *, weights=None, ref_scores=None, beta: float = 1.0,
                 label_smoothing: float = 0.0) -> None:
        self._w, self._l = _host_int64("winners", winners), _host_int64("losers", losers)
        self._weights = None if weights is None else _array("weights", weights, self._w.size, np.float32)
        self._ref_scores = ref_scores
        self._args = dict(beta=beta, label_smoothing=label_smoothing)
        self._pairs: PreferencePairs | None = None

    def bind(self, perm, num_rows, device):
        w, l, ref = self._w, self._l, self._ref_scores
        for name, a in (("winners", w), ("losers", l)):
            if a.size and (a.min() < 0 or a.max() >= num_rows):
                raise ValueError(f"{name} must name rows in [0, {num_rows})")
        ref = None if ref is None else _array("ref_scores", ref, num_rows, np.float32)
        if perm is not None:
            place = np.empty(num_rows, dtype=np.int64)
            place[perm] = np.arange(num_rows)
            w, l, ref = place[w], place[l], None if ref is None else ref[perm]
        self._pairs = PreferencePairs(w, l, num_values=num_rows, device=device)
        self._ref, self._wt = _to(device, ref), _to(device, self._weights)

    def gradient(self, preds):
        r = preference_loss(preds, self._pairs, ref_values=self._ref, weights=self._wt, **self._args)
        return r.loss, r.grad

    def release(self):
        if self._pairs is not None:
            self._pairs.close()
            self._pairs = self._ref = self._wt = None


class _Choices(Objective):
    """Sets of rows with one choice each, a mask and a learned position bias."""

    def __init__(self, offsets, chosen, *, mask=None, positions=None, buckets: PositionBuckets | None = None,
                 bias_rate: float = 0.1) -> None:
        self._off = _host_int64("offsets", offsets)
        if self._off.size == 0 or self._off[0] != 0 or np.any(self._off[1:] < self._off[:-1]):
            raise ValueError("offsets must start at 0 and not decrease")
        self._g, self._n = self._off.size - 1, int(self._off[-1])
        self._chosen = _indices("chosen", chosen, self._g)
        self._mask = None if mask is None else _array("mask", mask, self._n, bool)
        self._positions = None if positions is None else _indices("positions", positions, self._n)
        if buckets is not None and positions is None:
            raise ValueError("buckets need positions")
        self._buckets = buckets if buckets is not None or positions is None else PositionBuckets()
        self._bias_rate = float(bias_rate)
        self.table: np.ndarray | None = None
        self._sets: ChoiceSets | None = None
        self._bias: PositionBias | None = None

    def _bind_sets(self, perm, num_rows, device) -> np.ndarray | None:
        """Lays out the sets over the fit's rows; returns the order of the sets there (None: the caller's)."""
        if num_rows != self._n:
            raise ValueError(f"the sets hold {self._n} rows, the fit {num_rows}")
        off, order, mask, positions = self._off, None, self._mask, self._positions
        if perm is not None:
            place = np.empty(num_rows, dtype=np.int64)
            place[perm] = np.arange(num_rows)
            size = np.diff(off)
            full = size > 0
            start = np.full(self._g, -1, dtype=np.int64)  # empty sets come first
            start[full] = place[off[:-1][full]]
            if not np.array_equal(place, np.repeat(start, size) + np.arange(num_rows) - np.repeat(off[:-1], size)):
                raise ValueError("a set's rows must be of one era")
            order = np.argsort(start, kind="stable")
            off = np.concatenate([[0], np.cumsum(size[order])])
            mask = None if mask is None else mask[perm]
            positions = None if positions is None else positions[perm]
        self._sets = ChoiceSets(off, device=device)
        self._mask_dev = _to(device, mask)
        self._chosen_dev = self._steps(self._chosen, order, device)
        self._bias = None
        if positions is not None:
            nb = self._buckets.num_buckets
            count = np.bincount(self._buckets(positions), minlength=nb).astype(np.float32)
            self._step = _to(device, (self._bias_rate / np.maximum(count, 1.0)).astype(np.float32))
            self._bias = PositionBias(torch.zeros(nb, device=device), _to(device, positions), self._buckets)
            self._calls, self._past = 0, torch.zeros((2, nb), device=device)  # the table before the last two calls
        return order

    @staticmethod
    def _steps(a, order, device):
        return None if a is None else _to(device, a if order is None else np.ascontiguousarray(a[order]))

    def _learn(self, grad_table) -> None:
        if self._bias is not None:
            self._past[self._calls & 1].copy_(self._bias.table)
            self._calls += 1
            self._bias.table.addcmul_(self._step, grad_table, value=-1.0)

    def rewind(self, calls):
        if self._bias is not None and calls < self._calls:
            self._bias.table.copy_(self._past[calls & 1])
            self._calls = calls

    def release(self):
        if self._sets is not None:
            if self._bias is not None:
                self.table = self._bias.table.cpu().numpy()
            self._sets.close()
            self._sets = self._mask_dev = self._chosen_dev = self._bias = None


class PolicyObjective(_Choices):
    """One choice per set with an advantage: policy_loss on the softmax of the predictions.

    offsets, chosen, mask, positions: as ChoiceSets and choice_log_probs take them; advantages,
    old_log_probs, ref_log_probs, weights: per set."""

    def __init__(self, offsets, chosen, advantages, old_log_probs, *, ref_log_probs=None, weights=None, mask=None,
                 positions=None, buckets=None, bias_rate: float = 0.1, clip: tuple[float, float] = (0.2, 0.2),
                 kl_weight: float = 0.0) -> None:
        super().__init__(offsets, chosen, mask=mask, positions=positions, buckets=buckets, bias_rate=bias_rate)
        self._per_set = {k: _array(k, v, self._g, np.float32) for k, v in
                         (("advantages", advantages), ("old_log_probs", old_log_probs),
                          ("ref_log_probs", ref_log_probs), ("weights", weights)) if v is not None}
        self._args = dict(clip=clip, kl_weight=kl_weight)

    def bind(self, perm, num_rows, device):
        order = self._bind_sets(perm, num_rows, device)
        self._dev = {k: self._steps(v, order, device) for k, v in self._per_set.items()}

    def gradient(self, preds):
        r = policy_loss(preds, self._sets, self._chosen_dev, **self._dev, mask=self._mask_dev, bias=self._bias, **self._args)
        self._learn(r.grad_table)
        return r.loss, r.grad_scores

    def release(self):
        super().release()
        self._dev = None


class ChoicePreferenceObjective(_Choices):
    """Sequences of choices compared in pairs: preference_loss on their log-probabilities.

    Sequence k makes the choices of sets seq_offsets[k] .. seq_offsets[k + 1] - 1; winners and losers name
    sequences; ref_log_probs are a reference model's per set (0 where a step is left out), weights per
    pair."""

    def __init__(self, offsets, chosen, seq_offsets, winners, losers, *, ref_log_probs=None, weights=None, mask=None,
                 positions=None, buckets=None, bias_rate: float = 0.1, beta: float = 0.1,
                 label_smoothing: float = 0.0) -> None:
        super().__init__(offsets, chosen, mask=mask, positions=positions, buckets=buckets, bias_rate=bias_rate)
        self._seq = _host_int64("seq_offsets", seq_offsets)
        if self._seq.size == 0 or int(self._seq[-1]) != self._g:
            raise ValueError(f"seq_offsets must end at the {self._g} sets")
        self._w, self._l = _host_int64("winners", winners), _host_int64("losers", losers)
        self._ref_lp = None if ref_log_probs is None else _array("ref_log_probs", ref_log_probs, self._g, np.float32)
        self._weights = None if weights is None else _array("weights", weights, self._w.size, np.float32)
        self._args = dict(beta=beta, label_smoothing=label_smoothing)
        self._pairs: PreferencePairs | None = None

    def bind(self, perm, num_rows, device):
        order = self._bind_sets(perm, num_rows, device)
        self._pairs = PreferencePairs(self._w, self._l, offsets=self._seq, device=device)
        self._ref, self._wt = _to(device, self._ref_lp), _to(device, self._weights)
        # the fit's order of the sets, and back to the sequences' order
        self._order = self._back = None
        if order is not None:
            self._order = _to(device, order)
            self._back = torch.empty_like(self._order)
            self._back[self._order] = torch.arange(order.size, device=device)

    def gradient(self, preds):
        how = dict(chosen=self._chosen_dev, mask=self._mask_dev, bias=self._bias)
        lp, lse = choice_log_probs(preds, self._sets, **how)
        r = preference_loss(lp if self._back is None else lp[self._back], self._pairs, ref_values=self._ref,
                            weights=self._wt, **self._args)
        grad = r.grad if self._order is None else r.grad[self._order]
        gs, gt = choice_log_probs_backward(grad, preds, lse, self._sets, **how)
        self._learn(gt)
        return r.loss, gs

    def release(self):
        super().release()
        if self._pairs is not None:
            self._pairs.close()
            self._pairs = self._ref = self._wt = self._order = self._back = None
