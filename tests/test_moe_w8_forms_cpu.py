"""Which kernels a call of the FP8 expert layer takes (on 148 SMs, what a machine without a GPU assumes), and that the GPU tests of each form take it."""

import pytest

from emmy_b200 import lib as L
from tests import test_gpu_moe_w8_forms as forms


@pytest.fixture(scope="module")
def kernel():
    from emmy_b200.build import build

    build()
    return lambda t, e, topk, h, i, f16=False: L.load().eq_moe_w8a16_kernel(t, e, topk, h, i, L.EQ_F16 if f16 else L.EQ_BF16).decode()


def test_the_lines_between_the_forms(kernel):
    assert kernel(1, 128, 8, 2048, 768) == forms.OWN and kernel(2, 128, 8, 2048, 768) == kernel(2, 128, 8, 2048, 768, True) == forms.WIDE
    # a CTA of either launch on an SM, f16 activations beside them: 233472 bytes for 199072 and 512 a token
    assert kernel(2, 128, 4, 2048, 768) == forms.OWN and kernel(4, 64, 2, 2048, 1024, True) == forms.DOWN and kernel(3, 64, 2, 2048, 1024, True) == forms.OWN
    assert kernel(3, 64, 2, 2048, 1024) == forms.DOWN and kernel(2, 8, 2, 2048, 2048, True) == forms.OWN and kernel(2, 8, 2, 2048, 2048) == forms.DOWN
    assert kernel(2, 8, 8, 2304, 512, True) == forms.OWN and kernel(2, 8, 8, 2304, 640, True) == forms.DOWN
    # and no more slabs of sixteen channels than SMs
    assert kernel(1, 32, 1, 2304, 512) == forms.OWN and kernel(1, 32, 1, 2432, 512) == kernel(1, 32, 1, 5120, 128, True) == forms.DOWN
    # picks x I / 16 from sixteen an SM on, from four where the layer is 1280 wide
    assert kernel(16, 128, 4, 1152, 576) == forms.DOWN and kernel(16, 128, 4, 1152, 592) == forms.WIDE
    assert kernel(4, 128, 4, 1280, 576) == forms.DOWN and kernel(4, 128, 4, 1280, 592) == forms.WIDE
    # and not with 278 to 296 CTAs in clusters of four
    assert kernel(32, 128, 8, 2176, 768) == kernel(32, 128, 8, 2432, 768) == forms.WIDE and kernel(32, 128, 8, 2304, 768) == forms.DOWN
    assert kernel(32, 256, 1, 512, 256) == forms.DOWN and kernel(33, 256, 1, 512, 256) == kernel(1, 257, 1, 512, 256) == kernel(1, 8, 1, 512, 65664) == forms.EIGHT
    assert kernel(144, 128, 8, 2048, 768) == forms.EIGHT and kernel(145, 128, 8, 2048, 768) == forms.SIXTEEN


@pytest.mark.parametrize("form", list(forms.CASES))
def test_every_case_takes_its_form(kernel, form):
    t, e, topk, h, i = forms.CASES[form]
    assert {kernel(t, e, topk, h, i, f16) for f16 in (False, True)} == {forms.FORM_OF[form]}
