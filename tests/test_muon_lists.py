"""What a list of matrices asks for, on the CPU."""
import pytest

from test_muon import _lib, _mats


@pytest.mark.parametrize("other", [(300, 300, 1), (60, 1000, 1), (2048, 2048, 1)])
@pytest.mark.parametrize("stack", [(4, 6, 65536), (1, 50, 65536), (64, 64, 5000), (40, 900, 2000), (128, 128, 1000), (1, 70000, 7)])
def test_a_list_needs_about_what_its_entries_need(stack, other):
    """Long stacks beside a larger matrix: tiles take up to three times the workspace of strips, nothing more than that."""
    lib = _lib()
    need = lambda *shapes: lib.pdekan_orthogonalize_workspace_bytes(_mats(*shapes), len(shapes))
    assert 0 < need(stack, other) <= 3 * (need(stack) + need(other))
