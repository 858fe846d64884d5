"""A refusal of the kernel bindings whose message holds a number is an exception, not a crash."""
import pytest

from centrifuge_b200.ops import kernels


def test_numbers_in_error_messages():
    with pytest.raises(RuntimeError, match="gemm_plan failed with status -10"):
        kernels().gemm_plan(0, 0, 0, 0, 0, 148)
