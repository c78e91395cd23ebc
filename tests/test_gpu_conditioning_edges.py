"""The conditioning operators' arguments at the edges of what they take."""
from __future__ import annotations

import pytest
import torch

from conftest import dpa_mod

pytestmark = pytest.mark.gpu

C = dpa_mod("conditioning")


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("pad", [-1, -2, 20, 2**40])
def test_embedding_gradient_refuses_a_padding_outside_the_rows(native, pad, monkeypatch):
    """Both ways to the kernel; None alone means none."""
    g = torch.Generator().manual_seed(1)
    tokens = torch.randint(0, 20, (4, 7), generator=g).cuda()
    grad = torch.randn((4, 7, 24), generator=g).cuda()
    if native:
        assert not isinstance(C._fast(), C._General)
    else:
        monkeypatch.setattr(C, "_FAST", C._General())
    with pytest.raises(ValueError, match="padding_idx"):
        C.embedding_bwd(grad, tokens, 20, padding_idx=pad)
    none, last = C.embedding_bwd(grad, tokens, 20), C.embedding_bwd(grad, tokens, 20, padding_idx=19)
    assert not last[19].any() and torch.equal(none[:19], last[:19])
    assert bool((tokens == 19).any()) and bool(none[19].any())


@pytest.mark.parametrize("c", [1, 3])
def test_embedding_of_more_rows_than_a_grid_has(c):
    """Widths that are no whole 16 B take a wave per row: past 2^26 rows there are more lanes than a launch
    may have."""
    n = (1 << 26) + 3
    w = torch.arange(5 * c, device="cuda").view(5, c).float()
    t = torch.arange(n, device="cuda", dtype=torch.int32) % 5
    out = C.embedding_fwd(t, w)
    for lo in range(0, n, 1 << 24):
        part = t[lo:lo + (1 << 24)].long()
        assert torch.equal(out[lo:lo + (1 << 24)], w[part])
