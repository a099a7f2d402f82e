"""CPU: the package and its build where parts of the world are missing."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_everything_that_needs_no_torch_comes_without_it():
    code = ("import sys; sys.modules['torch'] = None\nfrom deep_contact_estimator_amd import *\nassert contact_cnn and load_checkpoint and synth.make_state_dict(1)\n"
            "import deep_contact_estimator_amd as d\n"
            "try: d.ops\nexcept ImportError: print('fine')")
    r = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, PYTHONPATH=ROOT), capture_output=True, text=True, timeout=120, cwd=ROOT)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-800:]
