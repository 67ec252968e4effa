"""What the layer operators refuse besides test_layer_ops_cpu.py's (no GPU needed)."""
import pytest

import gateddeltanet_b200 as gdn
from test_layer_ops_cpu import norm_args
from test_ops_cpu import lib  # noqa: F401


@pytest.mark.parametrize("eps", [float("inf"), float("-inf")])
def test_norm_with_an_eps_that_is_not_finite(lib, eps):  # noqa: F811
    """Its root would be NaN, not the formula's 0."""
    assert lib.gdn_b200_rms_norm(norm_args(eps=eps)) == -1
    assert "eps" in gdn.last_error()


@pytest.mark.parametrize("eps", [0.0, 1e-45, 3.4e38])
def test_norm_with_any_finite_eps(lib, eps):  # noqa: F811
    assert lib.gdn_b200_rms_norm(norm_args(eps=eps)) == -1
    assert "device" in gdn.last_error()


@pytest.mark.parametrize("ctas,columns,split", [(16, 64, 1), (1, 4096, 1), (1, 64, 65536)])
def test_tiles_out_of_range(lib, ctas, columns, split):  # noqa: F811
    assert lib.gdn_b200_test_linear_tiles(ctas, columns, split) == -1
    assert "no such tiles" in gdn.last_error()
