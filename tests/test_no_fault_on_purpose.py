"""CPU: nothing in the tree is made to fault the GPU: no tool reads past a buffer, no library holds the statement that lost a carry, no script loops on either."""
import glob
import os
import subprocess
import sys

from deep_contact_estimator_amd import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_guarded_runs_claim_no_more_than_their_buffers_hold():
    r = subprocess.run([sys.executable, os.path.join(ROOT, "tools", "guard_stress.py"), "--overrun", "1"], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert r.returncode == 2 and "unrecognized arguments" in r.stderr


def test_no_script_asks_for_a_fault():
    found = [p for p in glob.glob(os.path.join(ROOT, "tools", "**", "*"), recursive=True) if os.path.isfile(p) and p.endswith((".sh", ".py", ".hip"))]
    assert found
    for p in found:
        text = open(p, errors="replace").read()
        for word in ("--overrun", "h2sccbug", "h2knospill", "SCC_UNDECLARED", "h2_ksplit=1,h2_fc3=0", "past the end"):
            assert word not in text, (p, word)


def test_the_statement_that_lost_a_carry_is_in_no_library():
    """the host half of a build refuses it (the device half alone is what tests/test_build.py looks through)"""
    cmd = [build._hipcc(), *build.CFLAGS, "-DDCE_EXPERIMENTS=1", "-DH2_SCC_UNDECLARED=1", "--cuda-host-only", "-fsyntax-only", os.path.join(build.CSRC, "fc_gemm_h2.hip")]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=600)
    assert r.returncode != 0 and "no library that can be loaded" in r.stderr, r.stderr[-800:]
    ok = subprocess.run([c for c in cmd if "UNDECLARED" not in c], capture_output=True, text=True, timeout=600)
    assert ok.returncode == 0, ok.stderr[-800:]
