"""GPU: a context whose dce_finalize_weights failed on the way says so."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# The guard placement of one group of buffers (the 8-bit weights among them) asks for an address range that there is not: the allocation fails on the host.
CODE = """
import ctypes as C
import numpy as np
from deep_contact_estimator_amd import _lib, synth
from deep_contact_estimator_amd.synth import STATE_DICT_SHAPES
lib, ctx, sd = _lib.load(), C.c_void_p(), synth.make_state_dict(1, "uniform")
_lib.check(lib.dce_create_ex(C.byref(ctx), 0, 8, b"guard_alloc=1,guard_mask=256"), None)
for k, _ in STATE_DICT_SHAPES:
    w = sd[k]
    _lib.check(lib.dce_load_weight(ctx, k.encode(), w.ctypes.data_as(C.c_void_p), (C.c_int64 * w.ndim)(*w.shape), w.ndim), ctx)
x = np.random.default_rng(1).standard_normal((5, 150, 54), dtype=np.float32)


def run():
    out = np.empty((5, 16), np.float32)
    rc = lib.dce_forward_windows(ctx, x.ctypes.data_as(C.c_void_p), 5, 0, out.ctypes.data_as(C.c_void_p), None, None)
    return rc, lib.dce_last_error(ctx), out


_lib.check(lib.dce_finalize_weights(ctx, 1), ctx)
rc, _, want = run()
assert rc == 0
rc = lib.dce_finalize_weights(ctx, 4)
assert rc == -2, (rc, lib.dce_last_error(ctx))
rc, said, _ = run()
assert rc == -3 and b"not finalized" in said, (rc, said)
MORE
lib.dce_destroy(ctx)
print("fine")
"""
AGAIN = CODE.replace("MORE\n", """
_lib.check(lib.dce_finalize_weights(ctx, 1), ctx)
rc, said, again = run()
assert rc == 0 and np.array_equal(want, again), (rc, said)
""")


def ends_well(code):
    r = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, PYTHONPATH=ROOT, DCE_GUARD_ALIGN=str(1 << 60)), capture_output=True, text=True, timeout=100, cwd=ROOT)
    assert r.returncode == 0 and "fine" in r.stdout, (r.returncode, r.stdout[-500:], r.stderr[-1500:])


def test_a_failed_finalize_leaves_no_context_that_runs():
    ends_well(CODE.replace("MORE\n", ""))


def test_a_failure_is_reported_once():
    """finalized again, the context serves: the runtime's last error is not taken for one of the launches'"""
    ends_well(AGAIN)
