"""The tree attention kernel's register budget, held to the build's own resource report, and its plan and scratch."""
import re
import shutil
import subprocess

import pytest

from rivoli_amd import build, hip


def test_the_build_refuses_a_kernel_that_spills():
    block = ("remark: Function Name: _ZN2rk22mla_attend_tree_kernelENS_8TreeArgsE\n ScratchSize [bytes/lane]: %d\n LDS Size [bytes/block]: %d\n")
    build.check_resources("mla_attend_tree.hip", block % (0, 146448))
    for scratch, lds in ((4, 146448), (0, 163841)):
        with pytest.raises(RuntimeError):
            build.check_resources("mla_attend_tree.hip", block % (scratch, lds))
    with pytest.raises(RuntimeError):
        build.check_resources("mla_attend_tree.hip", "")


@pytest.mark.skipif(shutil.which(build.hipcc()) is None, reason="hipcc not found")
def test_the_kernel_keeps_the_whole_register_file_and_no_scratch(tmp_path):
    cmd = build.compile_command("mla_attend_tree.hip") + ["-Rpass-analysis=kernel-resource-usage", "-c", f"{build.CSRC}/mla_attend_tree.hip", "-o",
                                                          str(tmp_path / "m.o")]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-2000:]
    build.check_resources("mla_attend_tree.hip", res.stderr)
    block = next(b for b in re.split(r"remark: Function Name: ", res.stderr)[1:] if "mla_attend_tree_kernel" in b.split()[0])
    assert int(re.search(r"VGPRs: (\d+)", block).group(1)) + int(re.search(r"AGPRs: (\d+)", block).group(1)) <= 512


def test_scratch_covers_every_record_and_no_more_than_two_a_workgroup():
    record = 64 * (512 + 2)
    assert hip.mla_attend_tree_paged_scratch_floats(1, 16, 4, 4, 200) == 0            # whole blocks
    assert hip.mla_attend_tree_paged_scratch_floats(32, 64, 256, 8, 32768) == 256 * 2 * record
    small = hip.mla_attend_tree_paged_scratch_floats(1, 16, 4, 4, 2000)
    assert 0 < small < 256 * 2 * record and small % (2 * record) == 0
    for args in ((0, 1, 1, 1, 1), (1, 0, 1, 1, 1), (1, 1, 0, 1, 1), (1, 1, 1, 0, 1), (1, 1, 1, 1, -1)):
        assert hip.mla_attend_tree_paged_scratch_floats(*args) == 0
