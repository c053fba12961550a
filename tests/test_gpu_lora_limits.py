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


def test_an_output_beside_what_is_read():
    """Outputs that touch x or y on either side are other memory; one that is x is refused (y being x or not), one that is y is not."""
    import torch

    from emmy_b200.lib import EmmyqError
    from tests import test_gpu_lora as tl

    for t in (5, 300):
        args = tl.make(t, 64, [64], 8, 3, torch.bfloat16, seed=t)
        want = tl.call(args, [64])
        rows = torch.empty(5 * t, 64, dtype=torch.bfloat16, device="cuda")
        y, x = rows[t : 2 * t], rows[3 * t : 4 * t]
        for first in (0, 2 * t, 4 * t, t):  # before, between and behind them; y itself
            y.copy_(args[0]), x.copy_(args[1])
            out = rows[first : first + t]
            assert tl.call([y, x, *args[2:]], [64], out=out) is out and torch.equal(out, want)
            assert torch.equal(x, args[1]) and (first == t or torch.equal(y, args[0]))
        for args_, out in (((y, x), x), ((x, x), x), ((y, x), rows[2 * t + 1 : 3 * t + 1]), ((y, x), rows[t + 1 : 2 * t + 1])):
            with pytest.raises(EmmyqError, match="EQ_ERR_BAD_ARG"):
                tl.call([*args_, *args[2:]], [64], out=out)
        both = tl.call([x, x, *args[2:]], [64])  # y is x, the result is new
        tl.close(both, x, x, *args[2:], [64])
