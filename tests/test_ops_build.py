"""The build of the training-step operators, without a GPU: their kernels' resources, and that objects
follow the flags they are compiled with."""
import glob
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "msccl_amd", "csrc")


def out_of_date(build, *more):
    """The objects that make would compile."""
    out = subprocess.run(["make", "-n", "-C", CSRC, "BUILD=" + build, "OUT=" + build + "/out.so", *more], check=True,
                         capture_output=True, text=True).stdout
    return sorted(re.findall(r"-c \S+ -o (\S+\.o)", out))


@pytest.mark.skipif(not shutil.which("make"), reason="make missing")
def test_objects_follow_their_flags(tmp_path):
    build = str(tmp_path / "obj")
    every = out_of_date(build)
    assert any(x.endswith("ops_adamw.o") for x in every) and any(x.endswith("/ops.o") for x in every)
    for x in every:   # as if built now
        os.makedirs(os.path.dirname(x), exist_ok=True)
        open(x, "w").close()
    assert out_of_date(build) == [] and out_of_date(build) == []
    kernels = [x for x in every if "/device/kernels_" in x or "/device/ops_" in x]
    assert out_of_date(build, "EXTRA_HIPFLAGS=-DANOTHER") == kernels and len(kernels) < len(every)
    for x in kernels:
        os.utime(x)
    assert out_of_date(build, "EXTRA_HIPFLAGS=-DANOTHER") == []
    assert out_of_date(build) == kernels   # and back


def test_operators_kernels_have_no_scratch():
    """They hold rows and chunks in registers: a spill would be a round trip through memory for each."""
    kernels, name = {}, None
    for f in glob.glob(os.path.join(ROOT, "build", "obj", "device", "ops_*.res")):
        for line in open(f):
            m = re.search(r"Function Name: (\S+)", line)
            if m:
                name = m.group(1)
            m = re.search(r"(VGPRs|ScratchSize \[bytes/lane\]|LDS Size \[bytes/block\]): (\d+)", line)
            if m and name:
                kernels.setdefault(name, {}).setdefault(m.group(1).split()[0], int(m.group(2)))
    if not kernels:
        pytest.skip("no kernel resource reports (run __graft_entry__.build() first)")
    families = ("adamwKernel", "adamwBeginKernel", "squareSumKernel", "sumPartialsKernel", "balanceStatsKernel",
                "balanceFinishKernel", "balanceLossKernel", "balanceBackwardKernel", "tableWriteKernel", "gradWriteKernel")
    for family in families:
        assert any(family in k for k in kernels), family
    for k, v in kernels.items():
        assert v["ScratchSize"] == 0, (k, v)
        assert v["LDS"] <= 65536, (k, v)   # what a launch takes without asking
        # a workgroup of 1024 lanes has 128 registers a lane
        assert v["VGPRs"] <= 128, (k, v)
