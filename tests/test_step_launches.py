"""What the step's calls launch, on the CUDA runtime that records launches (see test_launch_sequence.py)."""
import ctypes

import pytest

from gevva_b200 import step
from tests.test_launch_sequence import recorder  # noqa: F401  (a fixture)

AT = [n << 36 for n in range(1, 14)]


@pytest.fixture(scope="module")
def lib(recorder):  # noqa: F811
    for name in ("gevva_step_plan", "gevva_step_trim", "gevva_step_sample"):
        getattr(recorder.lib, name).argtypes = [ctypes.c_char_p, ctypes.c_void_p]
    return recorder


def sample(lib, rows, vocabulary, f32=1):
    """(CTAs a row, launch) of rows that are one row expanded."""
    args = step._SAMPLE.pack(AT[0], 0, AT[1], 0, 0, 0, 0, AT[2], 0, rows, vocabulary, f32, 0.0)
    assert lib.lib.gevva_step_sample(args, None) == 0
    launch, = lib.launches()
    assert launch["kernel"] == "sample_kernel"
    return launch["grid"] // rows, launch


@pytest.mark.parametrize("rows,vocabulary,f32,ctas", [(1, 262144, 1, 16), (1, 1, 0, 1), (1, 1024, 1, 1), (64, 262144, 0, 4), (256, 50257, 1, 1),
                                                      (2, 5000, 1, 2), (1 << 20, 262144, 0, 1), ((1 << 27) - 1, 7, 1, 1)])
def test_ctas_of_a_row(lib, rows, vocabulary, f32, ctas):
    got, launch = sample(lib, rows, vocabulary, f32)
    assert got == ctas and launch["grid"] == rows * ctas and launch.get("cluster", 1) == ctas


@pytest.mark.parametrize("sequences,tokens,ctas", [(1, 0, 1), (64, 64, 1), (4, 4608, 8), (1000, 100, 1), (16384, 16384, 8), (1, 1 << 30, 8)])
def test_one_cluster_plans(lib, sequences, tokens, ctas):
    args = step._PLAN.pack(*AT[:11], 0, sequences, 4, 4, 1000, 16, tokens)
    assert lib.lib.gevva_step_plan(args, None) == 0
    assert [(x["kernel"], x["grid"], x.get("cluster", 1)) for x in lib.launches()] == [("step_pages_kernel<0>", ctas, ctas)]
    args = step._TRIM.pack(AT[0], AT[1], AT[2], AT[3], AT[4], AT[5], AT[6], 0, sequences, 4, 4, 1000, 16, 0)
    assert lib.lib.gevva_step_trim(args, None) == 0
    assert [(x["kernel"], x["grid"]) for x in lib.launches()] == [("step_pages_kernel<1>", 1 if sequences * 32 <= 1024 else 2 if sequences * 32 <= 2048 else 8)]
