"""What the group norm's backward asks for, on the CPU."""
import pytest

from test_norm import _lib


@pytest.mark.parametrize("n,s,c,g", [(1 << 19, 1, 4096, 1), (1 << 22, 2, 384, 1), (1 << 20, 1, 1536, 2), (1 << 23, 1, 8192, 8)])
def test_wide_points_need_a_fraction_of_their_tensor(n, s, c, g):
    """Up to 64 samples share a row of 2 c fp32 partial sums: an eighth of a byte a value, and two numbers a group of a sample."""
    need = _lib().pdekan_group_norm_workspace_bytes(n, s, c, g, 1)
    assert 0 < need <= n * s * c // 8 + 8 * n * g
