"""Which form of the int8 product takes a call (asked without a GPU), and that the GPU tests reach each of them."""
import pytest

from vtq import probe


@pytest.mark.parametrize("call,form", [
    ((1, 4096, 4096), "rows"), ((4, 11008, 4096), "rows"), ((32, 1024, 1024), "rows"), ((1, 1, 1), "rows"),
    ((1, 4096, 11008), "slices32"), ((8, 4096, 4096), "slices32"), ((19, 11008, 4096), "slices32"),
    ((48, 896, 4864), "slices64"), ((128, 4096, 4096), "slices64"), ((256, 11008, 4096), "slices128"),
    ((192, 4096, 11008), "tiles128"), ((512, 4096, 4096), "tiles128"), ((700, 130, 2049), "pair128"),
    ((512, 4096, 14336), "tiles128x256"), ((4001, 4096, 11008), "tiles256"), ((8192, 8192, 8192), "tiles256")])
def test_forms(call, form):
    assert probe.i8_form(*call) == form


def test_every_size_has_a_form():
    for batch in (1, 2, 5, 16, 17, 33, 64, 65, 127, 129, 300, 1000, 5000, 100000, 2 ** 30):
        for k in (0, 1, 16, 127, 4096, 131071):
            for n in (1, 15, 33, 257, 4096, 4097, 32000, 2 ** 30):
                assert probe.i8_form(batch, k, n) in probe.I8_FORMS


def test_the_product_tests_cover_every_form():
    import test_gpu_i8_linear

    cases = next(m for m in test_gpu_i8_linear.test_product.pytestmark if m.name == "parametrize"
                 and m.args[0] == "m,k,n").args[1]
    assert {probe.i8_form(*c) for c in cases} == set(probe.I8_FORMS)
