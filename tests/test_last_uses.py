"""What a CTA waits for before it may end (csrc/last_uses.h): the arrivals that other CTAs of its cluster send to its barriers for the last uses, which no
turn of its loops waits for; and the kernels that meet without ordering memory wait for them."""
import os
import re
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "infer_b200", "csrc")


def test_every_use_is_waited_for_once(tmp_path):
    exe = str(tmp_path / "check")
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", CSRC, "-o", exe, os.path.join(HERE, "last_uses_check.cpp")], check=True)
    proc = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert proc.returncode == 0, proc.stdout


def test_no_cta_ends_before_what_is_sent_to_its_barriers():
    """A kernel whose last meeting is relaxed has waited for its free stages and its accumulators, and orders memory where a wait ran out; a relaxed meeting
    stands nowhere else."""
    for name, barriers in (("act_tcgen05.cu", ("empty_bar", "acc_empty_bar")), ("linear_f32_cut.cu", ("empty_bar", "main_empty"))):
        with open(os.path.join(CSRC, name)) as f:
            src = f.read()
        src = re.sub(r"//[^\n]*", "", src)
        ends = [m.start() for m in re.finditer(r"cluster_meet\(\)", src)]
        assert len(ends) == 1 and re.search(r"if \(slots\[1\]\) cluster_sync\(\);\s*else cluster_meet\(\);", src)
        for b in barriers:
            m = re.search(r"last_uses\([^;]*mbar_wait\w*\(%s\(b\), phase\)" % b, src)
            assert m and m.start() < ends[0], f"{name}: {b}"
    with open(os.path.join(CSRC, "linear_f32_cut.cu")) as f:
        assert re.search(r"used >> i & 1\)\) ok = mbar_wait_each\(small_empty\(i\), \(turn >> i & 1\) \^ 1\)", f.read())
