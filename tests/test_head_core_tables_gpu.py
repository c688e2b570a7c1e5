"""Tables of other lengths than the sequence in the fused per-head attention core, on the kernels."""
import pytest
import torch

from tests.test_head_core_tables_cpu import check_tables

pytestmark = pytest.mark.gpu


def test_longer_and_shorter_tables():
    check_tables("cuda", torch.bfloat16, 64)
