"""Reports and distillation without a GPU: the C ABI's refusals, struct layouts, and the objective's checks."""

from __future__ import annotations

import ctypes
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parent.parent


def test_report_entry_points_refuse():
    """Null handles and descriptions come back before any device work."""
    from packboost_amd.backends import _hip

    lib = _hip.load()
    c, t = _hip.PbChoiceScores(), _hip.PbTeacher()
    assert lib.pb_choice_report_work_bytes(None, 1, 0) == -1
    for op in (_hip.PB_REPORT_BACKWARD, _hip.PB_DISTILL):
        assert lib.pb_choice_work_bytes(None, op, 0) == -1
    assert lib.pb_choice_report(None, c, None, 1.0, 0, None, None, None, None, None, None, 0, None) == -1
    assert lib.pb_choice_report_backward(None, c, None, 1.0, None, None, None, None, None, 0, None) == -1
    assert lib.pb_distillation_loss(None, c, t, None, None, None, None, None, 0, None) == -1
    assert lib.pb_last_error().decode()


def test_teacher_struct_matches_header(tmp_path):
    from packboost_amd.backends import _hip

    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no host C compiler")
    fields = [f for f, _ in _hip.PbTeacher._fields_]
    prints = "".join(f'printf("%zu ", offsetof(pb_teacher, {f}));' for f in fields)
    (tmp_path / "probe.c").write_text('#include <stdio.h>\n#include <stddef.h>\n#include "packboost_hip.h"\n'
                                      f'int main(void) {{ printf("%zu ", sizeof(pb_teacher)); {prints} return 0; }}\n')
    exe = tmp_path / "probe"
    subprocess.run([cc, "-std=c11", "-I", str(ROOT / "include"), str(tmp_path / "probe.c"), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(_hip.PbTeacher)] + [getattr(_hip.PbTeacher, f).offset for f in fields]


def test_distillation_objective_checks():
    from packboost_amd import DistillationObjective

    index, logits = np.zeros((2, 3), np.int64), np.zeros((2, 3), np.float32)
    DistillationObjective([0, 4, 9], index, logits)
    for bad in (dict(teacher_index=index[:1]), dict(teacher_logits=logits[:, :2]), dict(teacher_index=index.astype(float)),
                dict(teacher_index=index + 2 ** 31), dict(weights=np.ones(3)), dict(temperature=0.0), dict(temperature=np.nan),
                dict(teacher_index=index[0], teacher_logits=logits[0]),
                dict(teacher_index=np.zeros((2, 65), int), teacher_logits=np.zeros((2, 65))), dict(mask=np.ones(4, bool))):
        with pytest.raises(ValueError):
            DistillationObjective([0, 4, 9], **{**dict(teacher_index=index, teacher_logits=logits), **bad})


def test_objectives_on_choices_need_them():
    """Sets whose choices are None: refused where the objective is made, as any other wrong `chosen`; a distillation has none."""
    from packboost_amd import ChoicePreferenceObjective, DistillationObjective, PolicyObjective

    off, one = [0, 4, 9], np.ones(2)
    with pytest.raises(ValueError, match="chosen"):
        PolicyObjective(off, None, one, one)
    with pytest.raises(ValueError, match="chosen"):
        ChoicePreferenceObjective(off, None, [0, 1, 2], [0], [1])
    DistillationObjective(off, np.zeros((2, 3), int), np.zeros((2, 3)))


def test_build_refuses_spills_of_the_report_kernels():
    from packboost_amd.build import spilling_kernels

    names = ["_ZN2pb12_GLOBAL__N_118report_tile_kernelILb1E", "_ZN2pb12_GLOBAL__N_116soft_wide_kernelILb1E",
             "_ZN2pb12_GLOBAL__N_118report_join_kernelILi0E", "_ZN2pb12_GLOBAL__N_115soft_big_kernelILb1E"]
    remarks = lambda spill: "\n".join(f"x.hip:1:0: remark:     {v} [-Rpass-analysis=kernel-resource-usage]" for n in names for v in
                                      (f"Function Name: {n}", "ScratchSize [bytes/lane]: 0", f"VGPRs Spill: {spill}"))
    assert spilling_kernels(remarks(0)) == []
    assert spilling_kernels(remarks(2)) == names
