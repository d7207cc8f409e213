"""What a change to the build's flags rebuilds (no compiler runs)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "wgpu_morton_code_radix_sort_test_amd", "csrc")


def test_new_flags_reach_every_object():
    """The flags are in the Makefile: objects of an older one are out of date."""
    plan = subprocess.run(["make", "-n", "-W", "Makefile", "all"], cwd=CSRC, capture_output=True, text=True, check=True).stdout
    sources = [f for f in os.listdir(CSRC) if f.endswith(".hip")]
    assert len(sources) > 10
    for name in sources:
        lines = [line for line in plan.splitlines() if "-c %s " % name in line]
        assert lines and all("-packed-fp32-ops" in line for line in lines), name
    assert "-o libmrs.so" in plan and "-o mrs_run" in plan
