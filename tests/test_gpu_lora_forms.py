"""What one form of the adapters' kernels has been shown for, shown for the others: sizes on both sides of the lines between blocks of 16 and of 128 rows."""

import pytest
import torch

from tests import test_gpu_lora as tl

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")], ids=str)
@pytest.mark.parametrize("t,n", [(40, 64), (700, 64), (3000, 4096)])
def test_what_is_not_finite_in_one_section_stays_there(t, n, bad):
    """An adapter whose A overflowed f16 in one section; the other section's sums are far beyond f16's range and its results are not."""
    args = tl.make(t, 256, [n, n], 16, 2, F16, seed=5, ids=torch.zeros(t))
    y, x, a, b, scaling, ids = args
    x *= 2.0**6
    a[:, 1] *= 2.0**12
    b[:, n:] *= 2.0**-14
    a[0, 0, 3, 5] = bad
    got = tl.call(args, [n, n])
    second = [y[:, n:].contiguous(), x, a[:, 1:].contiguous(), b[:, n:].contiguous(), scaling, ids]
    assert (x.double() @ a[0, 1].double().T * scaling[0].item()).abs().amax(1).median() > 65504
    tl.close(got[:, n:].contiguous(), *second, [n])
    assert not torch.isfinite(got[:, :n]).any()
