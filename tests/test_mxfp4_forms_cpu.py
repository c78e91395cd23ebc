"""What the MXFP4 product is planned to launch: the sizes that the GPU tests hold against 64 bits take every form."""
from __future__ import annotations

import pytest

from conftest import dpa_mod
from mxfp4_forms import DTYPES, FORMS, PLAN, check_plan, plan


@pytest.mark.parametrize("size", FORMS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_sizes_take_the_form_they_stand_for(size, dtype):
    check_plan(size, dtype)


def test_every_form_is_among_them():
    assert {(s, v, a) for s, v, _, a in FORMS.values()} >= {(256, True, False), (256, True, True), (128, True, True),
                                                            (128, False, True), (64, True, True), (64, False, True)}


def test_few_rows_and_refusals():
    import torch
    assert plan(64, 512, 512, torch.bfloat16)["side"] == 0 and plan(65, 512, 512, torch.bfloat16)["side"] == 64
    assert plan(0, 512, 512, torch.bfloat16)["workgroups"] == 0
    entry, out = dpa_mod("_lib").load().dpa_mxfp4_gemm_plan, bytes(PLAN.size)
    assert entry(1 << 27, 4, 32, 0, out) == -2 and entry(4, 1 << 25, 32, 0, out) == -2
    assert entry(4, 4, 0, 0, out) == -2 and entry(4, 4, 32, 7, out) == -4 and entry(4, 4, 32, 0, None) == 0
