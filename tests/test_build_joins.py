"""The build refuses kernels whose listing has vector work in front of a join's exec restore (tests/exec_joins.py says what goes wrong there)."""
import os
import subprocess

import pytest

from rivoli_amd import build
from tests.exec_joins import early_vector_work

BAD = """
	s_and_saveexec_b64 s[56:57], vcc
	s_cbranch_execz .LBB1_2
	v_add_f32 v1, v1, v2
.LBB1_2:                                ;   in Loop
	v_writelane_b32 v255, s62, 7
	v_accvgpr_write_b32 a213, v135
	s_or_b64 exec, exec, s[56:57]
	v_mov_b32 v3, v4
"""
GOOD = BAD.replace("	v_accvgpr_write_b32 a213, v135\n", "")


def test_a_listing_with_work_that_is_skipped_is_refused():
    build.check_joins("mla_attend_tree.hip", GOOD)
    build.check_joins("rope.hip", BAD)                   # (of the kernels that are named alone: elsewhere such work may be meant)
    with pytest.raises(RuntimeError, match="v_accvgpr_write_b32 a213"):
        build.check_joins("mla_attend_tree.hip", BAD)
    assert build.early_vector_work(BAD) == early_vector_work(BAD) and build.early_vector_work(GOOD) == []


def test_the_build_looks_at_the_listing_and_links_nothing_that_fails(monkeypatch, tmp_path):
    ran = []

    def run(cmd, **_):
        ran.append(cmd)
        if "-c" in cmd:
            open(cmd[cmd.index("-o") + 1], "w").close()
        return subprocess.CompletedProcess(cmd, 0, BAD if "-S" in cmd else "", "")

    monkeypatch.setattr(build.subprocess, "run", run)
    monkeypatch.setattr(build, "check_resources", lambda k, report: None)
    csrc = str(tmp_path)
    monkeypatch.setattr(build, "CSRC", csrc)
    with pytest.raises(RuntimeError, match="mla_attend_tree.hip"):
        build.build_kernels()
    assert not any("-shared" in cmd for cmd in ran)
    assert not os.path.exists(os.path.join(csrc, "build", "mla_attend_tree.o")) and os.path.exists(os.path.join(csrc, "build", "rope.o"))
    listed = [cmd for cmd in ran if "-S" in cmd]
    assert [os.path.basename(c[c.index("-S") + 1]) for c in listed] == ["mla_attend_tree.hip"]
    own = build.compile_command("mla_attend_tree.hip")
    assert listed[0][:len(own)] == own, "another program than the one that is shipped"
