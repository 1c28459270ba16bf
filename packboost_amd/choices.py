"""Learning from choices and preferences on ragged sets of candidate rows.

A table's rows fall into sets (`ChoiceSets`): the candidates of a decision, the items of a list. A
model's scores give each row a probability within its set:

    x_i = score_i (+ table[bucket(position_i)], PositionBias), left out where mask_i is false
    log p_i = x_i - log sum_j exp(x_j) over the set

`choice_log_probs` computes them for every row, or for the row chosen in each set (a step), and
`choice_log_probs_backward` takes gradients back to the scores and the bias table. `policy_loss` is the
clipped policy loss with a KL term, its value and gradients in one pass; `preference_loss` is the loss of
paired log ratios on values or on sequences of steps. `choice_report` tells how sure a model is of each set, the
entropy and the rows it finds most probable, at a temperature; `choice_report_backward` trains with that, and
`distillation_loss` on what such a report of a larger model lists.

All of them run on the device as HIP kernels on torch's current stream, allocate their outputs from
torch's allocator and wait for nothing, so a caller may capture them in a graph. The sets, pairs, buckets
and tensors of a captured call have to outlive the graph; sets and pairs are laid out before the capture,
and PositionBuckets that the device has not seen are sent there before it by `on`. Row and step
quantities are 1-D device tensors; scores are float32, bfloat16 or float16 (their gradient has the same
type), everything else is float32. Tables whose rows start off a 16-byte boundary and scores with a stride
are read row by row, which takes 1.1 to 5 times as long (see whole_run in csrc/choice_rows.h); columns with a
stride other than the scores are copied. The gradients are returned, not recorded: tensors that require
gradients are read like any others, and nothing here is part of autograd's graph.
"""

from __future__ import annotations

import ctypes
from contextlib import nullcontext
from typing import NamedTuple

import numpy as np
import torch

from .backends import _hip

MAX_BUCKETS = 256
MAX_TOP = 64
_SCORE_TYPES = {torch.float32: _hip.PB_F32, torch.bfloat16: _hip.PB_BF16, torch.float16: _hip.PB_F16}


def _device(device) -> torch.device:
    dev = torch.device("cuda" if device is None else device)
    if dev.type != "cuda":
        raise ValueError(f"choices and preferences run on the GPU only, got device {dev}")
    if not torch.cuda.is_available():
        raise RuntimeError("HIP error: no GPU device is visible to torch")
    return torch.device("cuda", torch.cuda.current_device() if dev.index is None else dev.index)


def _host_int64(name: str, v) -> np.ndarray:
    a = v.detach().cpu().numpy() if isinstance(v, torch.Tensor) else np.asarray(v)
    if a.ndim != 1 or not (a.size == 0 or np.issubdtype(a.dtype, np.integer)):
        raise ValueError(f"{name} must be a 1-D table of integers")
    return np.ascontiguousarray(a, dtype=np.int64)


def _device_int64(name: str, t: torch.Tensor) -> torch.Tensor:
    if t.dim() != 1 or t.dtype not in (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8):
        raise ValueError(f"{name} must be a 1-D table of integers")
    return t.detach().to(torch.int64).contiguous()


def _home(device, *tables) -> torch.device:
    """The device asked for, else that of the first table on one."""
    if device is None:
        device = next((t.device for t in tables if isinstance(t, torch.Tensor) and t.is_cuda), None)
    return _device(device)


def _column(name: str, t, n: int, device: torch.device, *dtypes: torch.dtype) -> torch.Tensor:
    """t as the kernels read it: n adjacent entries of a 1-D tensor on the device."""
    if not isinstance(t, torch.Tensor) or t.device != device:
        raise ValueError(f"{name} must be a tensor on {device}")
    if t.dim() != 1 or t.numel() != n:
        raise ValueError(f"{name} must hold {n} entries, got shape {tuple(t.shape)}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be {' or '.join(str(d)[6:] for d in dtypes)}, got {str(t.dtype)[6:]}")
    return t if t.stride(0) == 1 or n <= 1 else t.contiguous()


_dropped: list = []  # (destroy, handle, device): closed, not freed yet


def _free_dropped() -> None:
    """Frees the layouts that were closed. A capture allows neither the wait nor the free: they stay until the
    next layout is made or closed outside of one."""
    while _dropped and not torch.cuda.is_current_stream_capturing():
        destroy, h, device = _dropped.pop()
        torch.cuda.synchronize(device)
        getattr(_hip.load(), destroy)(h)


class _Handle:
    """A layout the library keeps on the device."""

    _destroy = ""

    def _before(self) -> None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"{type(self).__name__} cannot be laid out while a graph is captured")
        _free_dropped()

    def close(self) -> None:
        """Frees the device memory, once the calls that use it have ended (and a capture, if one is going on)."""
        h, self._handle = getattr(self, "_handle", None), None
        if h is not None and h.value:
            _dropped.append((self._destroy, h, self.device))
            _free_dropped()

    def __del__(self) -> None:  # pragma: no cover - best effort
        try:
            self.close()
        except Exception:
            pass

    def _open(self) -> ctypes.c_void_p:
        if self._handle is None:
            raise ValueError(f"{type(self).__name__} is closed")
        return self._handle


class ChoiceSets(_Handle):
    """The sets of a table's rows: set g holds rows offsets[g] .. offsets[g + 1] - 1.

    offsets: integers [sets + 1] that start at 0 and do not decrease (an array, a list or a tensor; a
    device tensor is read back). Sets may be empty and of any size. The layout is made once and serves
    any number of calls."""

    _destroy = "pb_sets_destroy"

    def __init__(self, offsets, *, device=None) -> None:
        self._handle = None
        off = _host_int64("offsets", offsets)
        if off.size == 0 or off[0] != 0 or np.any(off[1:] < off[:-1]):
            raise ValueError("offsets must start at 0 and not decrease")
        self.device = _home(device, offsets)
        self._before()
        self.num_sets, self.num_rows = int(off.size - 1), int(off[-1])
        h = ctypes.c_void_p()
        with torch.cuda.device(self.device):
            _hip.check(_hip.load().pb_sets_create(off.ctypes.data, self.num_sets, ctypes.byref(h)), "pb_sets_create")
        self._handle = h
        self._work: dict[tuple[int, int], int] = {}

    def _workspace(self, op: int, num_buckets: int) -> tuple[torch.Tensor | None, int]:
        n = self._work.get((op, num_buckets))
        if n is None:
            n = self._work[op, num_buckets] = int(_hip.load().pb_choice_work_bytes(self._open(), op, num_buckets))
        return (_empty(n, self.device, torch.uint8), n) if n else (None, 0)

    def _report_workspace(self, top: int, num_buckets: int) -> tuple[torch.Tensor | None, int]:
        key = -1, top, num_buckets
        n = self._work.get(key)
        if n is None:
            n = self._work[key] = int(_hip.load().pb_choice_report_work_bytes(self._open(), top, num_buckets))
        return (_empty(n, self.device, torch.uint8), n) if n else (None, 0)


class PositionBuckets:
    """Buckets of relative positions: distances are exact near the reference and share buckets on a
    logarithmic scale further out.

    num_buckets are split into two halves, one for positions up to the reference and one for those after
    it, or (bidirectional=False) all serve positions up to the reference and later ones count as
    distance 0. Of a side's n buckets, the first n // 2 hold one distance each; distance d beyond that falls
    into bucket e + k, e = n // 2, for the largest k < n - e with (d / e)^(n - e) >= (reach / e)^k; from
    `reach` on every distance falls into the last one."""

    def __init__(self, num_buckets: int = 32, reach: int = 128, *, bidirectional: bool = True) -> None:
        side = num_buckets // 2 if bidirectional else num_buckets
        if not 0 < num_buckets <= MAX_BUCKETS or side < 2 or (bidirectional and num_buckets % 2):
            raise ValueError(f"num_buckets must lie in [2, {MAX_BUCKETS}] (an even number of at least 4 where "
                             f"bidirectional), got {num_buckets}")
        if not side // 2 < reach <= 1 << 20:
            raise ValueError(f"reach must lie above the {side // 2} exact distances and be at most 2^20, got {reach}")
        self.num_buckets, self.reach, self.bidirectional = int(num_buckets), int(reach), bool(bidirectional)
        first = side // 2
        steps = side - first
        near = np.empty(self.reach + 1, dtype=np.uint8)
        near[:first] = np.arange(first)
        # where bucket first + k starts: the least d with d^steps first^k >= reach^k first^steps, in whole numbers
        start = first
        for k in range(steps):
            low, high = start, self.reach
            while low < high:
                mid = (low + high) // 2
                if mid ** steps * first ** k >= self.reach ** k * first ** steps:
                    high = mid
                else:
                    low = mid + 1
            start = low
            near[start:] = first + k
        far = near + side if bidirectional else np.zeros_like(near)
        self.lookup = np.concatenate([near, far])
        self._on: dict[torch.device, torch.Tensor] = {}

    def __call__(self, positions) -> np.ndarray:
        """Bucket of each position (host integers)."""
        q = np.asarray(positions, dtype=np.int64)
        return self.lookup[np.minimum(np.abs(q), self.reach) + (q > 0) * (self.reach + 1)]

    def on(self, device: torch.device) -> torch.Tensor:
        """The lookup on a device, sent there at the first call."""
        t = self._on.get(device)
        if t is None:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"PositionBuckets have not been on {device} yet: call on(device) before the capture")
            t = self._on[_device(device)] = torch.from_numpy(self.lookup).to(device)
        return t


class PositionBias(NamedTuple):
    """A learned bias by position: row i's logit is score_i + table[bucket of positions_i].

    table: float32 [num_buckets]; positions: int32 per row, relative to the reference (negative before
    it); buckets: their PositionBuckets."""

    table: torch.Tensor
    positions: torch.Tensor
    buckets: PositionBuckets


class PreferencePairs(_Handle):
    """Pairs (winner, loser) of values by index, laid out once for any number of calls.

    winners, losers: integers [pairs]. Of num_values values, or with offsets (integers [sequences + 1]
    that start at 0 and do not decrease) of sequences: sequence k's value is the sum over steps
    offsets[k] .. offsets[k + 1] - 1. A value may be in any number of pairs. Pairs that lie on the device
    are laid out there (5M pairs of 1M values in 4.4 ms; from host tables in 18 ms)."""

    _destroy = "pb_pairs_destroy"

    def __init__(self, winners, losers, *, num_values: int | None = None, offsets=None, device=None) -> None:
        self._handle = None
        self.device = _home(device, winners, losers, offsets)
        self._before()
        here = all(isinstance(t, torch.Tensor) and t.device == self.device for t in (winners, losers))
        table = _device_int64 if here else _host_int64
        w, l = table("winners", winners), table("losers", losers)
        if len(w) != len(l):
            raise ValueError(f"winners and losers differ in length ({len(w)} and {len(l)})")
        if (num_values is None) == (offsets is None):
            raise ValueError("give num_values or offsets")
        off = None
        if offsets is not None:
            off = _host_int64("offsets", offsets)
            if off.size == 0 or off[0] != 0 or np.any(off[1:] < off[:-1]):
                raise ValueError("offsets must start at 0 and not decrease")
        self.num_pairs = len(w)
        self.num_values = int(num_values) if off is None else int(off.size - 1)
        if self.num_values < 0:
            raise ValueError(f"num_values must not be negative, got {self.num_values}")
        self.num_steps = self.num_values if off is None else int(off[-1])
        h = ctypes.c_void_p()
        with torch.cuda.device(self.device):
            seq = None if off is None else off.ctypes.data
            if here:
                rc = _hip.load().pb_pairs_create_from_device(w.data_ptr(), l.data_ptr(), self.num_pairs, self.num_values,
                                                             seq, _hip.stream_ptr(), ctypes.byref(h))
            else:
                rc = _hip.load().pb_pairs_create(w.ctypes.data, l.ctypes.data, self.num_pairs, self.num_values, seq,
                                                 ctypes.byref(h))
            if rc == _hip.PB_ERR_RANGE:
                raise ValueError(f"pairs must name values in [0, {self.num_values})")
            _hip.check(rc, "pb_pairs_create")
        self._handle = h
        self._work_bytes = int(_hip.load().pb_preference_work_bytes(h))


class PolicyLoss(NamedTuple):
    loss: torch.Tensor               # float32 scalar
    grad_scores: torch.Tensor        # the scores' type, per row
    grad_table: torch.Tensor | None  # float32 per bucket
    log_probs: torch.Tensor          # float32 per step, 0 where left out
    kl: torch.Tensor                 # float32 scalar: scale * sum of w * kl
    clipped: torch.Tensor            # float32 scalar: scale * sum of w over the steps held by a bound


class PreferenceLoss(NamedTuple):
    loss: torch.Tensor     # float32 scalar
    grad: torch.Tensor     # float32 per value, or per step of the sequences
    margins: torch.Tensor  # float32 per pair: beta * (log ratio of the winner - the loser's)


class ChoiceReport(NamedTuple):
    log_probs: torch.Tensor | None      # float32 per set: the chosen row's, 0 where left out; None without `chosen`
    entropy: torch.Tensor               # float32 per set, 0 for a set without probability
    lse: torch.Tensor                   # float32 per set, -inf for a set without probability
    top_index: torch.Tensor | None      # int32 [sets, top] within the set, -1 behind the last; None where top is 0
    top_log_probs: torch.Tensor | None  # float32 [sets, top], -inf behind the last


class DistillationLoss(NamedTuple):
    loss: torch.Tensor               # float32 scalar
    grad_scores: torch.Tensor        # the scores' type, per row
    grad_table: torch.Tensor | None  # float32 per bucket
    kl: torch.Tensor                 # float32 per set: the divergence, 0 where left out


def _scores(scores, sets: ChoiceSets, mask, bias) -> tuple[_hip.PbChoiceScores, list]:
    """The struct of the scores' description and the tensors it points into."""
    if not isinstance(sets, ChoiceSets):
        raise ValueError("sets must be ChoiceSets")
    n, dev = sets.num_rows, sets.device
    if not isinstance(scores, torch.Tensor) or scores.device != dev:
        raise ValueError(f"scores must be a tensor on {dev}")
    if scores.dim() != 1 or scores.numel() != n:
        raise ValueError(f"scores must hold {n} entries, got shape {tuple(scores.shape)}")
    kind = _SCORE_TYPES.get(scores.dtype)
    if kind is None:
        raise ValueError(f"scores must be float32, bfloat16 or float16, got {str(scores.dtype)[6:]}")
    c, keep = _hip.PbChoiceScores(), []
    c.scores_dev, c.score_stride, c.score_type = scores.data_ptr(), scores.stride(0) if n > 1 else 1, kind
    if mask is not None:
        m = _column("mask", mask, n, dev, torch.bool, torch.uint8)
        keep.append(m)
        c.mask_dev = m.data_ptr()
    if bias is not None:
        table, positions, buckets = bias
        if not isinstance(buckets, PositionBuckets):
            raise ValueError("bias.buckets must be PositionBuckets")
        t = _column("bias.table", table, buckets.num_buckets, dev, torch.float32)
        q = _column("bias.positions", positions, n, dev, torch.int32)
        b = buckets.on(dev)
        keep += [t, q, b]
        c.table_dev, c.positions_dev, c.buckets_dev = t.data_ptr(), q.data_ptr(), b.data_ptr()
        c.num_buckets, c.reach = buckets.num_buckets, buckets.reach
    return c, keep


_HERE = nullcontext()


def _on(device: torch.device):
    """torch.cuda.device(device), for nothing where that is the current one."""
    return _HERE if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _empty(n: int, like: torch.device, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    return torch.empty(n, dtype=dtype, device=like)


def choice_log_probs(scores: torch.Tensor, sets: ChoiceSets, *, chosen: torch.Tensor | None = None,
                     mask: torch.Tensor | None = None, bias: PositionBias | None = None
                     ) -> tuple[torch.Tensor, torch.Tensor]:
    """(log-probabilities, lse): of every row within its set (-inf where masked), or with `chosen` (int32
    per set: an index within the set) of each step's chosen row. lse is each set's log of the sum of
    exponentials, -inf where the set has no probability. A step whose choice lies outside its set or is
    masked, or whose set has no probability, is left out: its log-probability is 0."""
    c, keep = _scores(scores, sets, mask, bias)
    dev = sets.device
    if chosen is not None:
        chosen = _column("chosen", chosen, sets.num_sets, dev, torch.int32)
    with _on(dev):
        out = _empty(sets.num_rows if chosen is None else sets.num_sets, dev)
        lse = _empty(sets.num_sets, dev)
        work, size = sets._workspace(_hip.PB_LOG_PROBS, c.num_buckets)
        _hip.check(_hip.load().pb_choice_log_probs(
            sets._open(), c, _hip.ptr(chosen), out.data_ptr(), lse.data_ptr(), _hip.ptr(work), size,
            _hip.stream_ptr()), "pb_choice_log_probs")
    return out, lse


def choice_log_probs_backward(grad: torch.Tensor, scores: torch.Tensor, lse: torch.Tensor, sets: ChoiceSets, *,
                              chosen: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                              bias: PositionBias | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """(gradient of the scores, gradient of the bias table or None) from `grad`, that of the
    log-probabilities `choice_log_probs` gave for the same arguments (per row, or per step with
    `chosen`). lse is that call's; where it is 16 or more in size, its rounding, which an offset of the
    scores brings, is made up for by another sum over the set. Masked rows and steps left out take and give
    no gradient. A bucket's gradient is its rows' sum, each rounded to 2^-34 or less of the bucket's largest,
    in an order that is always the same."""
    c, keep = _scores(scores, sets, mask, bias)
    dev = sets.device
    grad = _column("grad", grad, sets.num_rows if chosen is None else sets.num_sets, dev, torch.float32)
    lse = _column("lse", lse, sets.num_sets, dev, torch.float32)
    if chosen is not None:
        chosen = _column("chosen", chosen, sets.num_sets, dev, torch.int32)
    with _on(dev):
        gs = _empty(sets.num_rows, dev, scores.dtype)
        gt = _empty(c.num_buckets, dev) if bias is not None else None
        work, size = sets._workspace(_hip.PB_BACKWARD, c.num_buckets)
        _hip.check(_hip.load().pb_choice_log_probs_backward(
            sets._open(), c, _hip.ptr(chosen), grad.data_ptr(), lse.data_ptr(), gs.data_ptr(), _hip.ptr(gt),
            _hip.ptr(work), size, _hip.stream_ptr()), "pb_choice_log_probs_backward")
    return gs, gt


def _finite(name: str, v: float, low: float = -float("inf")) -> float:
    v = float(v)
    if not (low <= v < float("inf")):
        raise ValueError(f"{name} must be finite" + (f" and at least {low}" if low > -float("inf") else "") + f", got {v}")
    return v


def policy_loss(scores: torch.Tensor, sets: ChoiceSets, chosen: torch.Tensor, advantages: torch.Tensor,
                old_log_probs: torch.Tensor, *, ref_log_probs: torch.Tensor | None = None,
                weights: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                bias: PositionBias | None = None, clip: tuple[float, float] = (0.2, 0.2), kl_weight: float = 0.0,
                scale: float = 1.0) -> PolicyLoss:
    """The clipped policy loss of one choice per set, and its gradients.

    With log p the chosen row's log-probability, r = exp(log p - old_log_probs), A the advantage and
    d = ref_log_probs - log p,

        loss = scale * sum of w * (kl_weight * (e^d - d - 1) - min(r A, clip(r, 1 - clip[0], 1 + clip[1]) A))

    over the steps (sets) that are not left out (see choice_log_probs). advantages, old_log_probs,
    ref_log_probs and weights (w, default 1) are float32 per set; without ref_log_probs there is no KL
    term. What has weight, kl_weight or advantage 0 counts for nothing, also where it overflows (`kl` tells the
    KL term whatever its weight). scale is the caller's mean: 1 / the number of steps, or 1 for the sum that a boosting round
    takes."""
    c, keep = _scores(scores, sets, mask, bias)
    dev, g = sets.device, sets.num_sets
    chosen = _column("chosen", chosen, g, dev, torch.int32)
    t = _hip.PbPolicyTerms()
    for name, field, v in (("advantages", "advantages_dev", advantages), ("old_log_probs", "old_log_probs_dev", old_log_probs),
                           ("ref_log_probs", "ref_log_probs_dev", ref_log_probs), ("weights", "weights_dev", weights)):
        if v is not None or name in ("advantages", "old_log_probs"):
            v = _column(name, v, g, dev, torch.float32)
            keep.append(v)
            setattr(t, field, v.data_ptr())
    low, high = _finite("clip[0]", clip[0], 0.0), _finite("clip[1]", clip[1], 0.0)
    t.ratio_min, t.ratio_max = 1.0 - low, 1.0 + high
    t.kl_weight, t.scale = _finite("kl_weight", kl_weight), _finite("scale", scale)
    with _on(dev):
        stats, lp = _empty(3, dev), _empty(g, dev)
        gs = _empty(sets.num_rows, dev, scores.dtype)
        gt = _empty(c.num_buckets, dev) if bias is not None else None
        work, size = sets._workspace(_hip.PB_POLICY, c.num_buckets)
        _hip.check(_hip.load().pb_policy_loss(
            sets._open(), c, t, chosen.data_ptr(), stats.data_ptr(), lp.data_ptr(), gs.data_ptr(), _hip.ptr(gt),
            _hip.ptr(work), size, _hip.stream_ptr()), "pb_policy_loss")
    return PolicyLoss(stats[0], gs, gt, lp, stats[1], stats[2])


def _temperature(v: float) -> float:
    v = float(v)
    if not 2.0 ** -20 <= v <= 2.0 ** 20:
        raise ValueError(f"temperature must lie in [2^-20, 2^20], got {v}")
    return v


def choice_report(scores: torch.Tensor, sets: ChoiceSets, *, chosen: torch.Tensor | None = None, top: int = 0,
                  mask: torch.Tensor | None = None, bias: PositionBias | None = None,
                  temperature: float = 1.0) -> ChoiceReport:
    """What a model says of each set, with p the softmax of its logits over the temperature: the chosen rows'
    log-probabilities (see choice_log_probs), the entropy -sum p log p, the log of the sum of exponentials, and the
    `top` (at most 64) rows of largest logit with their log-probabilities, best first.

    Logits are compared as float32, the bias added; equal ones are listed by index, NaN above all. Masked rows and
    rows of logit -inf are not listed. Sets of more than 2^31 - 1 rows have no lists."""
    c, keep = _scores(scores, sets, mask, bias)
    dev, g, top = sets.device, sets.num_sets, int(top)
    if not 0 <= top <= MAX_TOP:
        raise ValueError(f"top must lie in [0, {MAX_TOP}], got {top}")
    temperature = _temperature(temperature)
    if chosen is not None:
        chosen = _column("chosen", chosen, g, dev, torch.int32)
    with _on(dev):
        lp = None if chosen is None else _empty(g, dev)
        entropy, lse = _empty(g, dev), _empty(g, dev)
        index = torch.empty((g, top), dtype=torch.int32, device=dev) if top else None
        best = torch.empty((g, top), dtype=torch.float32, device=dev) if top else None
        work, size = sets._report_workspace(top, c.num_buckets)
        _hip.check(_hip.load().pb_choice_report(
            sets._open(), c, _hip.ptr(chosen), temperature, top, _hip.ptr(lp), entropy.data_ptr(), lse.data_ptr(),
            _hip.ptr(index), _hip.ptr(best), _hip.ptr(work), size, _hip.stream_ptr()), "pb_choice_report")
    return ChoiceReport(lp, entropy, lse, index, best)


def choice_report_backward(grad_log_probs: torch.Tensor | None, grad_entropy: torch.Tensor | None,
                           scores: torch.Tensor, sets: ChoiceSets, *, chosen: torch.Tensor | None = None,
                           mask: torch.Tensor | None = None, bias: PositionBias | None = None,
                           temperature: float = 1.0) -> tuple[torch.Tensor, torch.Tensor | None]:
    """(gradient of the scores, gradient of the bias table or None) from those of the chosen rows'
    log-probabilities and of the entropies (float32 per set, or None: 0) that `choice_report` gave for the same
    arguments. Masked rows take and give no gradient; steps left out give none through their log-probability. The
    sets' sums are formed anew, so a common offset of the scores does not matter."""
    c, keep = _scores(scores, sets, mask, bias)
    dev, g = sets.device, sets.num_sets
    if grad_log_probs is not None and chosen is None:
        raise ValueError("grad_log_probs need chosen")
    if chosen is not None:
        chosen = _column("chosen", chosen, g, dev, torch.int32)
    if grad_log_probs is not None:
        grad_log_probs = _column("grad_log_probs", grad_log_probs, g, dev, torch.float32)
    if grad_entropy is not None:
        grad_entropy = _column("grad_entropy", grad_entropy, g, dev, torch.float32)
    temperature = _temperature(temperature)
    with _on(dev):
        gs = _empty(sets.num_rows, dev, scores.dtype)
        gt = _empty(c.num_buckets, dev) if bias is not None else None
        work, size = sets._workspace(_hip.PB_REPORT_BACKWARD, c.num_buckets)
        _hip.check(_hip.load().pb_choice_report_backward(
            sets._open(), c, _hip.ptr(chosen), temperature, _hip.ptr(grad_log_probs), _hip.ptr(grad_entropy),
            gs.data_ptr(), _hip.ptr(gt), _hip.ptr(work), size, _hip.stream_ptr()), "pb_choice_report_backward")
    return gs, gt


def _list_of(name: str, t, sets: ChoiceSets, *dtypes: torch.dtype) -> torch.Tensor:
    """t as the kernels read it: a list per set, one after the other."""
    if not isinstance(t, torch.Tensor) or t.device != sets.device:
        raise ValueError(f"{name} must be a tensor on {sets.device}")
    if t.dim() != 2 or t.shape[0] != sets.num_sets or not 1 <= t.shape[1] <= MAX_TOP:
        raise ValueError(f"{name} must have shape [{sets.num_sets}, 1 to {MAX_TOP}], got {tuple(t.shape)}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be {' or '.join(str(d)[6:] for d in dtypes)}, got {str(t.dtype)[6:]}")
    return t.contiguous()


def distillation_loss(scores: torch.Tensor, sets: ChoiceSets, teacher_index: torch.Tensor, teacher_logits: torch.Tensor, *,
                      tail: bool = False, weights: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                      bias: PositionBias | None = None, temperature: float = 1.0,
                      scale: float = 1.0) -> DistillationLoss:
    """The divergence of the scores' softmax from a teacher of which each set's best rows are known, and its gradients.

    teacher_index: int32 [sets, k], k at most 64, rows by their index within the set (outside of it: none);
    teacher_logits [sets, k]: float32, bfloat16 or float16. An entry counts whose row is not masked, of entries
    that name one row the first. With p the student's softmax at the temperature T,

        tail=False   teacher_logits are logits, q their softmax at T within the set's entries that count, rho = 0
        tail=True    teacher_logits are log-probabilities at T (top_log_probs of a choice_report at T), q their
                     exponentials, and rho = 1 - sum q stands against pi, the sum of p over the rows not listed
                     (q / sum q and rho = 0 where there is no such row or the q sum to 1 or more)

        kl = sum q (log q - log p) + rho (log rho - log pi);  loss = scale * T^2 * sum of w * kl

    over the sets. weights (w, default 1) are float32 per set; a set of weight 0 counts for nothing, also where its
    divergence is infinite. A set in which the teacher's entries or the student have no probability is left out; a
    log-probability whose exponential is 0 in 64 bits (below -745) has none."""
    c, keep = _scores(scores, sets, mask, bias)
    dev, g = sets.device, sets.num_sets
    index = _list_of("teacher_index", teacher_index, sets, torch.int32)
    logits = _list_of("teacher_logits", teacher_logits, sets, *_SCORE_TYPES)
    if index.shape != logits.shape:
        raise ValueError(f"teacher_index and teacher_logits differ in shape ({tuple(index.shape)} and {tuple(logits.shape)})")
    t = _hip.PbTeacher()
    t.index_dev, t.logits_dev = index.data_ptr(), logits.data_ptr()
    t.entries, t.logit_type, t.tail = index.shape[1], _SCORE_TYPES[logits.dtype], bool(tail)
    if weights is not None:
        weights = _column("weights", weights, g, dev, torch.float32)
        t.weights_dev = weights.data_ptr()
    t.temperature, t.scale = _temperature(temperature), _finite("scale", scale)
    with _on(dev):
        loss, kl = _empty(1, dev), _empty(g, dev)
        gs = _empty(sets.num_rows, dev, scores.dtype)
        gt = _empty(c.num_buckets, dev) if bias is not None else None
        work, size = sets._workspace(_hip.PB_DISTILL, c.num_buckets)
        _hip.check(_hip.load().pb_distillation_loss(
            sets._open(), c, t, loss.data_ptr(), kl.data_ptr(), gs.data_ptr(), _hip.ptr(gt), _hip.ptr(work), size,
            _hip.stream_ptr()), "pb_distillation_loss")
    return DistillationLoss(loss[0], gs, gt, kl)


def preference_loss(values: torch.Tensor, pairs: PreferencePairs, *, ref_values: torch.Tensor | None = None,
                    weights: torch.Tensor | None = None, beta: float = 0.1, label_smoothing: float = 0.0,
                    scale: float = 1.0) -> PreferenceLoss:
    """The loss of paired log ratios and its gradient with respect to `values`.

    With a = values - ref_values (0 without), summed over each sequence's steps where the pairs name
    sequences, z = beta * (a_winner - a_loser) and s the sigmoid,

        loss = scale * sum of w * (-(1 - label_smoothing) log s(z) - label_smoothing log s(-z)).

    values and ref_values are float32 per value (per step), weights (w, default 1) per pair. Values are
    scores of rows (a reward model) or log-probabilities of steps (choice_log_probs with `chosen`, whose
    backward takes the gradient on); the ref_values those of a reference model. A pair of weight 0 and a
    side of the loss whose factor is 0 count for nothing, also where the margin is infinite."""
    if not isinstance(pairs, PreferencePairs):
        raise ValueError("pairs must be PreferencePairs")
    dev, n = pairs.device, pairs.num_steps
    values = _column("values", values, n, dev, torch.float32)
    if ref_values is not None:
        ref_values = _column("ref_values", ref_values, n, dev, torch.float32)
    if weights is not None:
        weights = _column("weights", weights, pairs.num_pairs, dev, torch.float32)
    beta, scale = _finite("beta", beta), _finite("scale", scale)
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError(f"label_smoothing must lie in [0, 1], got {label_smoothing}")
    with _on(dev):
        loss, grad, margins = _empty(1, dev), _empty(n, dev), _empty(pairs.num_pairs, dev)
        work = _empty(max(16, pairs._work_bytes), dev, torch.uint8)
        _hip.check(_hip.load().pb_preference_loss(
            pairs._open(), values.data_ptr(), _hip.ptr(ref_values), _hip.ptr(weights), beta, float(label_smoothing),
            scale, loss.data_ptr(), grad.data_ptr(), margins.data_ptr(), work.data_ptr(), work.numel(),
            _hip.stream_ptr()), "pb_preference_loss")
    return PreferenceLoss(loss[0], grad, margins)
