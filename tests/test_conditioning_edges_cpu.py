"""What the conditioning operators refuse at the edges of what they take (nothing is launched)."""
from __future__ import annotations

from conftest import dpa_mod
from test_conditioning_cpu import FAKE

L = dpa_mod("_lib")


def test_embedding_gradient_refuses_more_tokens_than_a_grid_has():
    """Its last launch has eight threads to a token."""
    f = L.load().dpa_embedding_bwd
    for n, status in ((1 << 29, -2), ((1 << 31) - 65, -2), ((1 << 29) - 32, -5)):     # (-5: no workspace)
        assert f(FAKE, 0, FAKE, 8, FAKE, 0, n, 10, 8, 1.0, -1, None, 0.0, None, 0, None) == status
