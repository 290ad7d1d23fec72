"""Using TVM through the bridge leaves the program's threads on all of its cores."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT
from relax_b200 import backend

pytestmark = pytest.mark.skipif(not backend.have_tvm(), reason="no TVM with Relax importable")

USES_THE_POOL = """
import os
before = os.sched_getaffinity(0)
from relax_b200 import backend
backend.import_tvm().get_global_func("runtime.config_threadpool")(-1, 0)
print(len(before), len(os.sched_getaffinity(0)), os.environ["TVM_BIND_THREADS"])
"""


@pytest.mark.parametrize("given", (None, "0", "1"))
def test_the_pool_does_not_bind_the_caller(given):
    env = {k: v for k, v in os.environ.items() if k != "TVM_BIND_THREADS"}
    if given is not None:
        env["TVM_BIND_THREADS"] = given
    done = subprocess.run([sys.executable, "-c", USES_THE_POOL], cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr
    before, after, says = done.stdout.split()[-3:]
    assert says == (given or "0")                 # who asks for the binding gets it
    if says == "0":
        assert before == after
