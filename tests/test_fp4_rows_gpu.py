"""Ranges of rows of a 4-bit weight on the GPU."""
import pytest

from tests.test_fp4_rows_cpu import check_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_forward_rows_of_a_quantised_layer(fmt, monkeypatch):
    check_rows(fmt, "cuda", monkeypatch)
