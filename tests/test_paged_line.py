"""morello_amd/csrc/paged_line.h, how the attention over pages deals tiles' keys to workgroups.  No GPU needed."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_every_block_is_dealt_once_and_shares_cover_the_line(tmp_path):
    """Random batches, and as many new tokens as there may be over tables of any size: more of them than a table holds made a line that shares of
    32 bits did not cover, and tiles whose pieces would have been sought past the last workgroup's."""
    exe = tmp_path / "paged_line_check"
    cmd = ["g++", "-std=c++17", "-O2", "-Wall", "-Werror", os.path.join(ROOT, "tests", "paged_line_check.cpp"), "-o", str(exe)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True)
    assert run.returncode == 0 and "paged line ok" in run.stdout, run.stdout[-2000:] + run.stderr
