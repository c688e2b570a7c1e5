"""The same refusals on the GPU."""
import pytest

from tests.test_fp4_arguments_cpu import check_arguments

pytestmark = pytest.mark.gpu


def test_shapes_without_columns():
    check_arguments("cuda")
