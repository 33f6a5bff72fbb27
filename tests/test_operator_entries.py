"""What the library's entries for the operators refuse by addresses: asked for on the host, before anything is launched."""
import pytest

from cbm4gnn_b200 import _lib

GRANT = 1 << 30  # bytes that a workspace is said to have; none of these addresses is ever read


def _refused(name, *args):
    assert getattr(_lib.lib(), name)(*args, None) == 1
    return _lib.lib().cbm_b200_last_error().decode()


@pytest.mark.parametrize("at", [0, 4, 8 + 1])
def test_workspaces_of_norms_lie_at_8_bytes(at):
    n, c, groups, a = 5000, 64, 8, 1 << 20
    ws = at and a + at
    forward = _refused("cbm_b200_group_norm", a, c, 0, n, c, groups, a, 2, 0, a, a, 1, 1e-5, 0, a, c, a, a, ws, GRANT)
    backward = _refused("cbm_b200_group_norm_grad", a, c, a, c, 0, n, c, groups, a, 2, 0, a, a, 1, 1e-5, 0, a, a, a, c, a, a, ws, GRANT)
    for said, who in ((forward, "group_norm"), (backward, "group_norm_grad")):
        assert said == f"{who}: workspace too small, or not at 8 bytes"


def test_statistics_of_class_scores_lie_at_8_bytes():
    a = 1 << 20
    assert "8 bytes" in _refused("cbm_b200_class_log_probs", a, 7, 0, a, 1, 10, 7, 0, a, a, a + 4, a, a)
    assert "8 bytes" in _refused("cbm_b200_class_log_probs_grad", a, 7, 0, a, 1, 10, 7, 0, a + 4, a, a, a, a, a, a, 7)
