"""nn.GroupedLinear in the "bf16" math mode, whose products stay FP32-accurate: the bounds of the default mode, on every engine that groups have there."""
import pytest

from test_gpu_fused_linear import check_groups, gt  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("counts,I,O,name", [
    ([1, 2, 0, 1] * 4, 256, 128, "silu"),                                        # few rows
    ([200, 0, 3, 150], 128, 96, "gelu"), ([40] * 30, 333, 515, "none"),          # warp-level tiles
    ([900, 30, 2200, 0, 511, 1, 257, 256], 1024, 1408, "silu"),                  # two-SM tiles
    ([2048, 2048], 2048, 2048, "none"), ([1500, 300], 1531, 1601, "gelu")])
def test_bounds_of_the_default_mode(gt, counts, I, O, name):  # noqa: F811
    halves, pairs = gt.lib().THGPUProductCount(1), gt.lib().THGPUProductCount(2)
    gt.set_math_mode("bf16")
    try:
        check_groups(gt, counts, I, O, name)
        assert (gt.lib().THGPUProductCount(1), gt.lib().THGPUProductCount(2)) == (halves, pairs)
    finally:
        gt.set_math_mode("fp32x3")
