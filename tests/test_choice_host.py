"""The choice and preference operators without a GPU: position buckets, the C ABI's refusals and struct
layouts, and the errors of a machine that has none."""

from __future__ import annotations

import ctypes
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parent.parent


def test_position_buckets():
    """One bucket a distance near the reference, then the largest k with (d / e)^m >= (reach / e)^k."""
    from packboost_amd import PositionBuckets

    for num, reach, both in ((32, 128, True), (8, 4, True), (256, 1000, True), (9, 64, False), (4, 2, True)):
        pb = PositionBuckets(num, reach, bidirectional=both)
        side = num // 2 if both else num
        e = side // 2
        m = side - e
        for d in range(0, reach + 3):
            c = min(d, reach)
            want = c if c < e else e + max(k for k in range(m) if c ** m * e ** k >= reach ** k * e ** m)
            assert pb([-d])[0] == want
            assert pb([d])[0] == (want + (side if d > 0 else 0) if both else 0)
        assert pb([-2 ** 31])[0] == side - 1
    for bad in (dict(num_buckets=2), dict(num_buckets=7), dict(num_buckets=258), dict(num_buckets=32, reach=8)):
        with pytest.raises(ValueError):
            PositionBuckets(**bad)


def test_choice_operators_need_the_gpu():
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU is visible")
    from packboost_amd import ChoiceSets, PreferencePairs

    with pytest.raises(RuntimeError):
        ChoiceSets([0, 2])
    with pytest.raises(RuntimeError):
        PreferencePairs([0], [1], num_values=2)
    with pytest.raises(ValueError):
        ChoiceSets([0, 2], device="cpu")


def test_choice_entry_points_refuse():
    """Bad arguments of the choice and preference entry points come back before any device work."""
    from packboost_amd.backends import _hip

    lib = _hip.load()
    out = ctypes.c_void_p()
    for off, code in (([1, 2], -1), ([0, 3, 2], -1)):
        a = np.array(off, np.int64)
        assert lib.pb_sets_create(a.ctypes.data, len(off) - 1, ctypes.byref(out)) == code and not out.value
    assert lib.pb_sets_create(None, 0, ctypes.byref(out)) == -1
    assert lib.pb_sets_create(np.zeros(1, np.int64).ctypes.data, 0, None) == -1
    big = np.array([0, 2 ** 37 + 1], np.int64)
    assert lib.pb_sets_create(big.ctypes.data, 1, ctypes.byref(out)) == -4
    w = np.array([0, 5], np.int64)
    assert lib.pb_pairs_create(w.ctypes.data, w.ctypes.data, 2, 5, None, ctypes.byref(out)) == -2
    assert lib.pb_pairs_create(None, None, 2, 5, None, ctypes.byref(out)) == -1
    assert lib.pb_choice_work_bytes(None, 0, 0) == -1 and lib.pb_preference_work_bytes(None) == -1
    c, t = _hip.PbChoiceScores(), _hip.PbPolicyTerms()
    assert lib.pb_choice_log_probs(None, c, None, None, None, None, 0, None) == -1
    assert lib.pb_choice_log_probs_backward(None, c, None, None, None, None, None, None, 0, None) == -1
    assert lib.pb_policy_loss(None, c, t, None, None, None, None, None, None, 0, None) == -1
    assert lib.pb_preference_loss(None, None, None, None, 1.0, 0.0, 1.0, None, None, None, None, 0, None) == -1
    assert lib.pb_set_gradients(None, None) == -1
    assert lib.pb_last_error().decode()


def test_choice_struct_layouts_match_header():
    """pb_choice_scores and pb_policy_terms against the header, by the host C compiler."""
    import tempfile

    from packboost_amd.backends import _hip

    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no host C compiler")
    probe = ["#include <stdio.h>", "#include <stddef.h>", '#include "packboost_hip.h"', "int main(void) {"]
    want = {}
    for name, cls in (("pb_choice_scores", _hip.PbChoiceScores), ("pb_policy_terms", _hip.PbPolicyTerms)):
        probe.append(f'printf("{name} %zu\\n", sizeof({name}));')
        want[name] = ctypes.sizeof(cls)
        for field, _ in cls._fields_:
            probe.append(f'printf("{name}.{field} %zu\\n", offsetof({name}, {field}));')
            want[f"{name}.{field}"] = getattr(cls, field).offset
    probe.append("return 0; }")
    with tempfile.TemporaryDirectory() as td:
        src, exe = Path(td) / "probe.c", Path(td) / "probe"
        src.write_text("\n".join(probe))
        subprocess.run([cc, "-std=c11", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
        got = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    assert {k: int(v) for k, v in got.items()} == want


def test_build_refuses_spills_of_the_choice_kernels():
    """What the compiler reports of a kernel that spills, and of one that only has a frame reserved."""
    from packboost_amd.build import spilling_kernels

    def remarks(name, scratch, vgprs):
        return "\n".join(f"choice.hip:1:0: remark:     {v} [-Rpass-analysis=kernel-resource-usage]" for v in (
            f"Function Name: {name}", "VGPRs: 96", f"ScratchSize [bytes/lane]: {scratch}", "SGPRs Spill: 40",
            f"VGPRs Spill: {vgprs}", "LDS Size [bytes/block]: 0"))

    wide, tile, other = "_ZN2pb11wide_kernelILi4E", "_ZN2pb11tile_kernelILi3E", "_ZN2pb11join_kernelE"
    assert spilling_kernels("\n".join((remarks(wide, 36, 0), remarks(tile, 0, 0), remarks(other, 64, 3)))) == []
    assert spilling_kernels("\n".join((remarks(tile, 20, 4), remarks(wide, 80, 0)))) == [tile, wide]
    assert spilling_kernels(remarks("_ZN2pb15hist_era_kernelE", 4, 0)) == ["_ZN2pb15hist_era_kernelE"]


def test_objectives_refuse_indices_that_a_cast_would_change():
    """Choices and positions are int32: what int32 does not hold, or what is no whole number, is not cut to fit."""
    from packboost_amd import ChoicePreferenceObjective, PolicyObjective

    off, one = [0, 2, 5], np.ones(2)
    policy = lambda chosen=(0, 1), positions=None: PolicyObjective(off, chosen, one, one, positions=positions)
    sequences = lambda chosen=(0, 1), positions=None: ChoicePreferenceObjective(off, chosen, [0, 1, 2], [0], [1], positions=positions)
    place = np.arange(5)
    for build in (policy, sequences):
        for bad in ([0, 2 ** 32 + 1], [0, -2 ** 31 - 1], [0.0, 1.7], np.array([0.0, 1.0]), np.array([False, True]),
                    np.array([0, 2 ** 64 - 1], dtype=np.uint64)):
            with pytest.raises(ValueError, match="chosen"):
                build(chosen=bad)
        for bad in (place + 2 ** 32, place + 0.5, place.astype(np.float32)):
            with pytest.raises(ValueError, match="positions"):
                build(positions=bad)
        for good in ([-1, 2 ** 31 - 1], np.array([0, 1], dtype=np.uint8), np.array([0, 7], dtype=np.int64)):
            kept = build(chosen=good, positions=place.astype(np.int64))
            assert kept._chosen.dtype == np.int32 and kept._chosen.tolist() == np.asarray(good).tolist()
            assert kept._positions.dtype == np.int32 and kept._positions.tolist() == place.tolist()


@pytest.mark.parametrize("kind", ["policy", "sequences"])
def test_a_bind_that_fails_is_released(monkeypatch, kind):
    """Whatever fails after the sets are laid out (here: memory for the mask) is what the caller hears of, and
    the sets are closed."""
    import torch

    from packboost_amd import ChoicePreferenceObjective, PolicyObjective, objectives

    closed = []

    class Sets:
        def __init__(self, offsets, *, device=None):
            pass

        def close(self):
            closed.append(self)

    def no_memory(device, a):
        raise MemoryError("out of device memory")

    monkeypatch.setattr(objectives, "ChoiceSets", Sets)
    monkeypatch.setattr(objectives, "_to", no_memory)
    one, mask = np.ones(2), np.ones(5, bool)
    obj = (PolicyObjective([0, 2, 5], [0, 1], one, one, mask=mask) if kind == "policy" else
           ChoicePreferenceObjective([0, 2, 5], [0, 1], [0, 1, 2], [0], [1], mask=mask))
    with pytest.raises(MemoryError):
        try:  # as a fit does
            obj.bind(None, 5, torch.device("cpu"))
        finally:
            obj.release()
    assert len(closed) == 1
    obj.release()
    assert len(closed) == 1 and obj.table is None
