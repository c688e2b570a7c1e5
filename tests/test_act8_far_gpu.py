"""linear_act8 on the GPU at inputs up to the ends of bf16."""
import pytest

from tests.test_act8_far_cpu import check_far_gelu, check_far_swiglu, far_gelu, far_swiglu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("R,N", [(3, 5), (130, 40), (300, 1024), (20000, 48)])  # whole tiles, and tiles in parts
def test_gelu(R, N):
    check_far_gelu(*far_gelu(R, N, "cuda"))


@pytest.mark.parametrize("R,N", [(3, 5), (130, 40), (300, 1024), (20000, 48)])
def test_swiglu(R, N):
    check_far_swiglu(*far_swiglu(R, N, "cuda"))
