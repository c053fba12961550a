"""Which kernels a call of the adapters takes, and that the GPU tests of each form take it: a line that moves leaves no form untested unseen."""

import pytest

from emmy_b200 import lib as L
from tests import test_gpu_lora_forms as forms


@pytest.fixture(scope="module")
def kernel():
    from emmy_b200.build import build

    build()
    return lambda t, k, n, r, s=1: L.load().eq_lora_kernel(t, k, n, r, s).decode()


def test_the_lines_between_the_forms(kernel):
    assert kernel(1, 4096, 4096, 16) == kernel(256, 5120, 34816, 64, 2) == "lora_rows_kernel"
    # 257 to 2048 rows in blocks of 16: every CTA lists the blocks itself
    assert kernel(257, 1024, 520, 16) == kernel(2048, 128, 136, 16) == "lora_rows_kernel" and kernel(2049, 128, 136, 16) == forms.LIST
    # T (K + 2 N) max(R, 32) = 2e9 with sixteen ranks in all, 8e8 with more
    assert kernel(2048, 1024, 14746, 16) == "lora_rows_kernel" and kernel(2048, 1024, 14748, 16) == forms.TILES
    assert kernel(1000, 1000, 11999, 32) == "lora_rows_kernel" and kernel(1000, 1000, 12000, 32) == forms.TILES
    assert kernel(1000, 1000, 12000, 8, 2) == "lora_rows_kernel" and kernel(1000, 1000, 12000, 8, 3) == forms.TILES
    # ranks that the tiles do not hold
    assert kernel(100000, 4096, 4096, 128, 2) == forms.TILES and kernel(100000, 4096, 4096, 136) == kernel(100000, 4096, 4096, 88, 3) == forms.LIST


@pytest.mark.parametrize("form", list(forms.CASES))
def test_every_case_takes_its_form(kernel, form):
    want = forms.FORM_OF[form]
    for t, k, sections, r, _ in forms.CASES[form].values():
        assert kernel(t, k, sum(sections), r, len(sections)) == want, (form, t, k, sections, r)
