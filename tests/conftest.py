import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (run on the B200 box)")


# These two parameter sets compare with a quotient that is rounded to f32 on the way to e4m3, which in three of their bytes is not
# the nearest e4m3 value (2.12500003611128 becomes 2.125 and then 2; the nearest is 2.25).  They run last, so that a run that stops
# at its first failure has seen every other test; test_gpu_norm_q8_bytes.py has the values in rational arithmetic.
ROUNDED_TWICE = ["test_8_bit_floats_are_the_rounding_of_the_exact_quotient[400-2048-rt0-0]",
                 "test_8_bit_floats_are_the_rounding_of_the_exact_quotient[64-12288-rt3-0]"]


def pytest_collection_modifyitems(items):
    items.sort(key=lambda item: item.name in ROUNDED_TWICE)
