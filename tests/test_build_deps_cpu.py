"""What a change of a public header rebuilds."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "s2pro-native_b200", "csrc")


@pytest.mark.parametrize("target,objects", [("all", "../build/"), ("testlib", "../build_test/")])
@pytest.mark.parametrize("header", ["s2p_b200_abi.h", "s2p_b200_ext.h"])
def test_a_changed_header_rebuilds_every_object(target, objects, header):
    """The kernels take the headers' structs by value: an object that was left as it was would read them wrongly."""
    if shutil.which("make") is None:
        pytest.skip("no make on this machine")
    # (a dry run that takes the header for new)
    told = subprocess.run(["make", "-n", "-W", f"../../include/{header}", target], cwd=CSRC, capture_output=True, text=True, check=True).stdout
    for folder, end in (("cuda", ".cu"), ("host", ".c")):
        for name in sorted(os.listdir(os.path.join(CSRC, folder))):
            if name.endswith(end):
                made = objects + (name + ".o" if end == ".cu" else name[:-1] + "o")
                assert f"-o {made}" in told, made
