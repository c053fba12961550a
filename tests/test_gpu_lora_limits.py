"""Adapters at the limits of what their kernels may have, each as the first call of a process: no larger call has raised a limit before it."""

import subprocess
import sys

import pytest

from tests.conftest import ROOT

pytestmark = pytest.mark.gpu

FIRST_CALL = """
import torch
from tests import test_gpu_lora as tl
t, k, sections, r, adapters = {case}
args = tl.make(t, k, sections, r, adapters, torch.{dtype}, seed=t)
tl.close(tl.call(args, sections), *args, sections)
print("compared")
"""


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize(
    "case",
    [
        # sums and split h of 352 ranks: 49152 bytes beside the static arrays
        (4, 64, [64], 352, 3),
        (5, 64, [64, 32], 176, 3),
        (300, 64, [64, 32, 8, 8], 88, 3),
        # counters of 3060 and 3071 adapters: 48976 and 49152 bytes
        (300, 64, [64], 8, 3060),
        (300, 64, [64], 64, 3071),
    ],
    ids=str,
)
def test_shared_memory_around_the_limit_that_every_kernel_has(case, dtype):
    run = subprocess.run([sys.executable, "-c", FIRST_CALL.format(case=case, dtype=dtype)], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip() == "compared", run.stderr[-2000:]
