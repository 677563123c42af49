"""The tree attention kernel's register budget, held to the build's own resource report, and its plan and scratch."""
import re
import shutil
import subprocess

import pytest

from rivoli_amd import build, hip
from tests.exec_joins import early_vector_work


def test_the_build_refuses_a_kernel_that_spills():
    block = ("remark: Function Name: _ZN2rk22mla_attend_tree_kernelILb1EEEvNS_8TreeArgsE\n ScratchSize [bytes/lane]: %d\n LDS Size [bytes/block]: %d\n")
    build.check_resources("mla_attend_tree.hip", block % (0, 146448))
    for scratch, lds in ((4, 146448), (0, 163841)):
        with pytest.raises(RuntimeError):
            build.check_resources("mla_attend_tree.hip", block % (scratch, lds))
    with pytest.raises(RuntimeError):
        build.check_resources("mla_attend_tree.hip", "")


@pytest.mark.skipif(shutil.which(build.hipcc()) is None, reason="hipcc not found")
def test_the_kernel_keeps_the_register_file_to_itself_and_its_copies_where_lanes_are_enabled(tmp_path):
    listing = tmp_path / "tree.s"
    cmd = build.compile_command("mla_attend_tree.hip") + ["-Rpass-analysis=kernel-resource-usage", "--offload-device-only", "-S",
                                                          f"{build.CSRC}/mla_attend_tree.hip", "-o", str(listing)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-2000:]
    build.check_resources("mla_attend_tree.hip", res.stderr)
    block = next(b for b in re.split(r"remark: Function Name: ", res.stderr)[1:] if "mla_attend_tree_kernel" in b.split()[0])
    assert int(re.search(r"VGPRs: (\d+)", block).group(1)) + int(re.search(r"AGPRs: (\d+)", block).group(1)) <= 512
    assert early_vector_work(listing.read_text()) == []


def test_work_in_front_of_a_restore_is_found():
    listing = """
	s_and_saveexec_b64 s[56:57], vcc
	s_cbranch_execz .LBB1_2
	v_add_f32 v1, v1, v2
.LBB1_2:                                ;   in Loop
	v_writelane_b32 v255, s62, 7
	v_accvgpr_write_b32 a213, v135
	s_or_b64 exec, exec, s[56:57]
	v_mov_b32 v3, v4
"""
    assert early_vector_work(listing) == [(".LBB1_2", "v_accvgpr_write_b32 a213, v135")]
    assert early_vector_work(listing.replace("	v_accvgpr_write_b32 a213, v135\n", "")) == []


def test_scratch_covers_every_record_and_no_more_than_two_a_workgroup():
    record = 64 * (512 + 2)
    # whole blocks: two tiles, and enough blocks of a few
    assert hip.mla_attend_tree_paged_scratch_floats(1, 16, 4, 4, 124) == hip.mla_attend_tree_paged_scratch_floats(32, 16, 128, 4, 508) == 0
    assert hip.mla_attend_tree_paged_scratch_floats(1, 16, 4, 4, 125) == 3 * 2 * record        # one block of three tiles, a workgroup each
    assert hip.mla_attend_tree_paged_scratch_floats(65535, 128, 2 ** 23, 128, 2 ** 31 - 8193) == 0  # too many to count in 32 bits: whole
    assert hip.mla_attend_tree_paged_scratch_floats(32, 64, 256, 8, 32768) == 256 * 2 * record
    small = hip.mla_attend_tree_paged_scratch_floats(1, 16, 4, 4, 2000)
    assert 0 < small < 256 * 2 * record and small % (2 * record) == 0
    for args in ((0, 1, 1, 1, 1), (1, 0, 1, 1, 1), (1, 1, 0, 1, 1), (1, 1, 1, 0, 1), (1, 1, 1, 1, -1)):
        assert hip.mla_attend_tree_paged_scratch_floats(*args) == 0
