"""Products that between them take every form of the MXFP4 product's kernel, and what each is planned to be."""
from __future__ import annotations

import ctypes
import struct

import torch

from conftest import dpa_mod

DTYPES = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 2}
PLAN = struct.Struct("=4iq")

# (m, n, k): side of the tiles, stores by vectors in 16-bit types and in fp32, whether a workgroup takes more than one tile
FORMS = {
    (4100, 2056, 1536): (256, True, True, False),
    (4096, 8192, 1024): (256, True, True, True),
    (8193, 3000, 1100): (256, True, True, True),        # an odd number of steps, rows and columns that end inside a tile
    (32768, 768, 256): (128, True, True, True),         # one step to a tile, three tiles to a workgroup
    (16640, 520, 264): (128, True, True, True),
    (4400, 4104, 1300): (128, True, True, True),
    (8193, 3002, 1100): (128, False, False, True),      # (planned for the largest tiles)
    (33000, 515, 264): (128, False, False, True),
    (300, 11008, 1300): (64, True, True, True),
    (130, 18952, 2049): (64, True, True, True),
    (300, 11010, 1100): (64, False, False, True),
    (700, 1200, 300): (64, True, True, False),
    (500, 500, 9000): (64, True, True, False),          # split
}


def plan(m: int, n: int, k: int, dtype: torch.dtype) -> dict:
    out = ctypes.create_string_buffer(PLAN.size)
    dpa_mod("_lib").call("dpa_mxfp4_gemm_plan", m, n, k, DTYPES[dtype], out)
    return dict(zip(("side", "vectors", "splits", "workgroups", "tiles"), PLAN.unpack(out.raw)))


def check_plan(size: tuple[int, int, int], dtype: torch.dtype) -> None:
    side, vec16, vec32, again = FORMS[size]
    p = plan(*size, dtype)
    assert p["side"] == side and p["vectors"] == (vec32 if dtype == torch.float32 else vec16), (size, p)
    assert (p["tiles"] > p["workgroups"]) == again, (size, p)
    assert (p["splits"] > 1) == (size[2] == 9000), (size, p)
