"""The bounded waits of the product kernel behind linear_cross_entropy: a pipeline that stops making progress ends with a
status, not with a hung GPU.

The self-test build of the library (csrc/build.py: build_selftest) lets the first CTA fill a given number of stages and then
stop: nothing is copied for the stage that is withheld, so no copy is in flight, and every role of that CTA (and of
the one it shares its tiles with) runs into its wait limit, a few milliseconds here.  The kernel drains and returns,
the device's word names the wait, and the next calls are right.  Nothing here faults, traps or spins without a bound.  Runs in a
process of its own because the library variant is chosen when the binding is first loaded.
"""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = r"""
import os, sys, time
sys.path.insert(0, %(root)r)
import torch
from graph_rws_b200 import core
from graph_rws_b200.core import _native
from graph_rws_b200.layers import linear_cross_entropy
lib = _native.lib()
stream = lambda: torch.cuda.current_stream().cuda_stream

def call(x, w, y, backward):
    loss = linear_cross_entropy(x, w, y)
    return [loss.detach()] + (list(torch.autograd.grad(loss, (x, w))) if backward else [])

# a CTA a tile and pairs; 16-bit operands and three planes; the statistics alone, and all three launches
for dtype in (torch.bfloat16, torch.float32):
    for n in (100, 700):
        x = torch.randn(n, 392, device="cuda").to(dtype).requires_grad_(True)
        w = (0.1 * torch.randn(392, 3001, device="cuda")).to(dtype).requires_grad_(True)
        y = torch.randint(0, 3001, (n,), device="cuda")
        good = call(x, w, y, True)
        core.check_device_status()
        for backward in (False, True):
            assert lib.grws_linear_ce_set_wait_limit(8000000) == 0             # about 4 ms of SM clocks per wait
            os.environ["GRWS_CE_WITHHOLD"] = "2"
            t0 = time.perf_counter()
            call(x, w, y, backward)
            torch.cuda.synchronize()                                           # the launches return: no role waits for ever
            elapsed = time.perf_counter() - t0
            assert elapsed < 5.0, elapsed
            st = lib.grws_linear_ce_check(stream())
            assert st == -5, st                                                # GRWS_ERR_DEVICE
            msg = lib.grws_last_error().decode()
            assert "gave up waiting" in msg and "incomplete" in msg, msg
            assert lib.grws_linear_ce_check(stream()) == 0                     # reading the word cleared it
            os.environ["GRWS_CE_WITHHOLD"] = "0"
            assert lib.grws_linear_ce_set_wait_limit(0) == 0
            again = call(x, w, y, True)                                        # the context is intact
            core.check_device_status()
            assert all(torch.equal(a, b) for a, b in zip(again, good))
            print(dtype, n, backward, round(elapsed * 1e3, 1), "ms;", msg)
assert lib.grws_linear_ce_set_wait_limit(-1) == -1
print("TIMEOUT-SELFTEST-OK")
"""


def test_a_withheld_stage_ends_with_a_status_not_a_hang():
    from graph_rws_b200.core import _native
    selftest = os.path.join(os.path.dirname(_native.LIB_PATH), "libgrws_b200_selftest.so")
    if not os.path.exists(selftest):
        pytest.skip("self-test build of the library is missing (graph_rws_b200/csrc/build.py --selftest)")
    env = dict(os.environ, GRWS_LIB_PATH=selftest)
    env.pop("GRWS_CE_WITHHOLD", None)
    out = subprocess.run([sys.executable, "-c", CHILD % {"root": ROOT}], env=env, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout[-2000:] + out.stderr[-4000:]
    assert "TIMEOUT-SELFTEST-OK" in out.stdout
    print(out.stdout)
