"""What the conditioning operators refuse at the edges of what they take (nothing is launched)."""
from __future__ import annotations

import pytest
import torch

from conftest import dpa_mod
from test_conditioning_cpu import FAKE, _desc

C = dpa_mod("conditioning")
L = dpa_mod("_lib")


def test_embedding_gradient_refuses_more_tokens_than_a_grid_has():
    """Its last launch has eight threads to a token."""
    f = L.load().dpa_embedding_bwd
    for n, status in ((1 << 29, -2), ((1 << 31) - 65, -2), ((1 << 29) - 32, -5)):     # (-5: no workspace)
        assert f(FAKE, 0, FAKE, 8, FAKE, 0, n, 10, 8, 1.0, -1, None, 0.0, None, 0, None) == status


@pytest.mark.parametrize("kw", [
    dict(b=1 << 20, h=16, g=16, lq=1, lk=8),            # keys in LDS: a workgroup per head
    dict(b=1 << 20, h=16, g=16, lq=40, lk=8),
    dict(b=1 << 20, h=16, g=16, lq=1, lk=200),          # few rows
    dict(b=1 << 10, h=16, g=16, lq=(1 << 17) + 1, lk=200),
])
def test_attention_refuses_more_workgroups_than_a_grid_has(kw):
    lib = L.load()
    room = 1 << 62
    assert lib.dpa_cross_attention_fwd(_desc(**kw), FAKE, room, None) == -2
    assert lib.dpa_cross_attention_bwd(_desc(**kw), FAKE, room, None) == -2


def test_attention_refuses_more_workgroups_of_keys_than_a_grid_has():
    kw = dict(b=1 << 10, h=16, g=16, lq=1, lk=1 << 17)
    assert L.load().dpa_cross_attention_bwd(_desc(**kw), FAKE, 1 << 62, None) == -2


@pytest.mark.parametrize("c", [(1 << 20) + 1, (1 << 32) + 8])
def test_embedding_refuses_wide_rows(c):
    """A width past 32 bits would reach the entry as its lowest 32."""
    wide, tokens = torch.zeros(1).expand(1, c), torch.zeros(1, dtype=torch.int64)
    with pytest.raises(ValueError, match="C up to"):
        C.embedding_fwd(tokens, wide)
    with pytest.raises(ValueError, match="C up to"):
        C.embedding(tokens, wide)
    with pytest.raises(ValueError, match="rows of up to"):
        C.embedding_bwd(wide, tokens, 5)


def test_attention_refuses_scales_that_overflow_in_base_2():
    """The kernels work on scale log2(e): infinite, a score of 0 would be NaN."""
    for s in (2.5e38, 3.3e38):
        with pytest.raises(ValueError, match="scale"):
            C._scale_of(s, 64)
        assert L.load().dpa_cross_attention_fwd(_desc(scale=s), None, 0, None) == -2
    assert C._scale_of(2.2e38, 64) == 2.2e38
