"""What the MXFP4 operators refuse, before anything is launched, and the sizes that their C entries report."""
from __future__ import annotations

import ctypes

import pytest
import torch

from conftest import dpa_mod


@pytest.fixture(scope="module")
def M():
    return dpa_mod("mxfp4")


@pytest.fixture(scope="module")
def lib():
    return dpa_mod("_lib").load()


def u8(*shape):
    return torch.zeros(shape, dtype=torch.uint8)


def test_cpu_tensors_are_refused(M):
    x = torch.zeros(4, 64)
    for call in (lambda: M.quantize_mxfp4(x), lambda: M.mxfp4_operand(x), lambda: M.mxfp4_operands(x),
                 lambda: M.linear_mxfp4_fwd(x, x), lambda: M.linear_mxfp4(x, x), lambda: M.linear_mxfp4_train_fwd(x, x),
                 lambda: M.dequantize_mxfp4(M.MXFP4(u8(4, 32), u8(4, 2))),
                 lambda: M.cross_attention_mxfp4_fwd(torch.zeros(1, 2, 2, 64, dtype=torch.bfloat16),
                                                     M.MXFP4(u8(1, 3, 2, 2, 32), u8(1, 3, 2, 2, 2)))):
        with pytest.raises(ValueError, match="expected GPU tensors"):
            call()


def test_quantize_refusals(M):
    for x, why in ((torch.zeros(4, 33), "multiple of 32"), (torch.zeros(()), "multiple of 32"),
                   (torch.zeros(4, 0), "multiple of 32"), (torch.zeros(4, 32, dtype=torch.float64), "bf16, fp16 or fp32"),
                   (torch.zeros(4, 32, dtype=torch.int32), "bf16, fp16 or fp32")):
        with pytest.raises(ValueError, match=why):
            M.quantize_mxfp4(x)
    for q, why in ((M.MXFP4(u8(4, 16), u8(4, 2)), "do not go"), (M.MXFP4(u8(4, 16), u8(3, 1)), "do not go"),
                   (M.MXFP4(u8(4, 16).int(), u8(4, 1)), "uint8")):
        with pytest.raises(ValueError, match=why):
            M.dequantize_mxfp4(q)
    with pytest.raises(ValueError, match="bf16, fp16 or fp32"):
        M.dequantize_mxfp4(M.MXFP4(u8(4, 16), u8(4, 1)), torch.float64)
    for x in (torch.zeros(4), torch.zeros(2, 3, 4), torch.zeros(4, 0)):
        with pytest.raises(ValueError, match="a matrix"):
            M.mxfp4_operand(x)
    with pytest.raises(ValueError, match="bf16, fp16 or fp32"):
        M.mxfp4_operands(torch.zeros(2, 3, dtype=torch.float64))


def test_attention_refusals(M):
    q = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16)

    def kv(b=2, lk=5, two=2, g=2, d=64):
        return M.MXFP4(u8(b, lk, two, g, d // 2), u8(b, lk, two, g, d // 32))
    # (what is refused before the device is looked at)
    with pytest.raises(ValueError, match="do not go together"):
        M.cross_attention_mxfp4_fwd(q, M.MXFP4(u8(2, 5, 2, 2, 32), u8(2, 5, 2, 2, 1)))
    with pytest.raises(ValueError, match="uint8"):
        M.cross_attention_mxfp4_fwd(q, M.MXFP4(u8(2, 5, 2, 2, 32).char(), u8(2, 5, 2, 2, 2)))
    with pytest.raises(ValueError, match="no gradient"):
        M.cross_attention_mxfp4(q.float().requires_grad_(), kv())


def test_c_entries_refuse_before_launch(lib):
    fake, nul, odd = ctypes.c_void_p(0x1000), None, ctypes.c_void_p(0x1004)
    q = lib.dpa_mxfp4_quantize
    assert q(nul, 0, 64, fake, fake, nul) == -1
    assert q(fake, 0, 33, fake, fake, nul) == -2 and q(fake, 0, -32, fake, fake, nul) == -2
    assert q(fake, 0, 1 << 40, fake, fake, nul) == -2           # more workgroups than a launch has
    assert q(fake, 3, 32, fake, fake, nul) == -4
    assert q(odd, 0, 32, fake, fake, nul) == -3
    assert q(nul, 0, 0, nul, nul, nul) == 0
    d = lib.dpa_mxfp4_dequantize
    assert d(fake, nul, fake, 0, 32, nul) == -1 and d(fake, fake, odd, 0, 32, nul) == -3
    assert d(fake, fake, fake, 0, 16, nul) == -2 and d(fake, fake, fake, 7, 32, nul) == -4
    o = lib.dpa_mxfp4_operands
    assert o(fake, 0, 4, 40, 40, nul, nul, nul, nul, nul) == -1          # neither wanted
    assert o(nul, 0, 4, 40, 40, fake, nul, nul, nul, nul) == -1
    assert o(fake, 0, 4, 40, 39, fake, nul, nul, nul, nul) == -2         # rows that overlap
    assert o(fake, 0, 4, 0, 40, fake, nul, nul, nul, nul) == -2
    assert o(fake, 0, -1, 40, 40, fake, nul, nul, nul, nul) == -2
    assert o(fake, 0, 1 << 25, 1 << 12, 1 << 12, fake, nul, nul, nul, nul) == -2
    assert o(fake, 5, 4, 40, 40, fake, nul, nul, nul, nul) == -4
    assert o(fake, 0, 4, 40, 40, odd, nul, nul, nul, nul) == -3
    assert o(fake, 0, 4, 40, 40, nul, odd, nul, nul, nul) == -3
    assert o(fake, 0, 4, 40, 40, fake, nul, nul, odd, nul) == -3         # the seed
    assert o(fake, 0, 4, 40, 40, fake, nul, fake, nul, nul) == -1    # sums without the columns
    assert o(nul, 0, 0, 40, 40, fake, nul, nul, nul, nul) == 0
    g = lib.dpa_mxfp4_gemm
    assert g(fake, nul, nul, fake, 0, 4, 4, 32, nul, 0, nul) == -1
    assert g(fake, fake, nul, fake, 0, 4, 4, 0, nul, 0, nul) == -2
    assert g(fake, fake, nul, fake, 0, 1 << 27, 4, 32, nul, 0, nul) == -2
    assert g(fake, fake, nul, fake, 9, 4, 4, 32, nul, 0, nul) == -4
    assert g(odd, fake, nul, fake, 0, 4, 4, 32, nul, 0, nul) == -3
    assert lib.dpa_mxfp4_gemm_workspace_bytes(100, 64, 16384) > 0
    assert g(fake, fake, nul, fake, 0, 100, 64, 16384, nul, 0, nul) == -5
    assert g(fake, fake, nul, fake, 0, 100, 64, 16384, fake, 16, nul) == -5
    assert g(nul, nul, nul, nul, 0, 0, 4, 32, nul, 0, nul) == 0
    li = lib.dpa_mxfp4_linear
    need = lib.dpa_mxfp4_linear_workspace_bytes(fake, 0, 512, 20, 64, 512)
    assert need >= lib.dpa_mxfp4_operand_bytes(20, 512) > 0
    assert lib.dpa_mxfp4_linear_workspace_bytes(fake, 0, 512, 2, 64, 512) == 0          # within the launch
    assert lib.dpa_mxfp4_linear_workspace_bytes(odd, 0, 512, 2, 64, 512) > 0            # not by vectors
    assert li(fake, 0, 512, fake, nul, fake, 0, 20, 64, 512, fake, need - 1, nul) == -5
    assert li(fake, 0, 511, fake, nul, fake, 0, 20, 64, 512, fake, need, nul) == -2
    assert li(fake, 0, 512, nul, nul, fake, 0, 20, 64, 512, fake, need, nul) == -1
    assert li(fake, 4, 512, fake, nul, fake, 0, 20, 64, 512, fake, need, nul) == -4
    assert li(fake, 0, 512, odd, nul, fake, 0, 20, 64, 512, fake, need, nul) == -3
    assert li(fake, 0, 512, fake, nul, fake, 0, 0, 64, 512, nul, 0, nul) == 0
    c = lib.dpa_column_sum
    assert c(fake, 0, 0, 4, 4, fake, fake, 64, nul) == -2 and c(nul, 0, 4, 4, 4, fake, fake, 64, nul) == -1
    assert c(fake, 0, 4, 4, 4, fake, fake, 15, nul) == -5 and c(fake, 4, 4, 4, 4, fake, fake, 64, nul) == -4
    assert lib.dpa_column_sum_workspace_bytes(129, 10) == 4 * 10 * 4


def test_operand_sizes(lib):
    size = lib.dpa_mxfp4_operand_bytes
    # whole sixteens of rows, and scales of 256 rows behind the last
    assert size(3, 1) == 16 * 128 + (3 + 256) * 16 and size(16, 256) == 16 * 128 + (16 + 256) * 16
    assert size(17, 257) == 32 * 256 + (17 + 256) * 16 and size(3, 513) == 16 * 384 + (2 * 3 + 256) * 16
    assert size(0, 40) == 256 * 16 and size(-1, 40) == 0 and size(3, 0) == 0 and size(1 << 40, 32) == 0


def test_attention_entry_refuses_before_launch(lib, M):
    pack = M._DESC.pack

    def desc(q=0x1000, kd=0x1000, dtype=0, b=1, lq=2, lk=3, h=4, g=2, d=64, scale=0.1, data_stride=16, q_stride=8):
        return pack(q, kd, 0x1001, 0x1000, 0x1001, 0x1000, 0x1000, 0, 0, 0, *(q_stride,) * 3, *(data_stride,) * 3,
                    1, 1, 1, *(data_stride,) * 3, 1, 1, 1, dtype, b, lq, lk, h, g, d, scale)
    f = lib.dpa_cross_attention_mxfp4
    assert f(None, None, 0, None) == -1
    assert f(desc(q=0), None, 0, None) == -1 and f(desc(kd=0), None, 0, None) == -1
    assert f(desc(d=40), None, 0, None) == -4 and f(desc(d=160), None, 0, None) == -4
    assert f(desc(dtype=1), None, 0, None) == -4 and f(desc(g=3), None, 0, None) == -4
    assert f(desc(scale=0.0), None, 0, None) == -2 and f(desc(lq=-1), None, 0, None) == -2
    assert f(desc(data_stride=8), None, 0, None) == -3 and f(desc(q_stride=4), None, 0, None) == -3
    assert f(desc(kd=0x1008), None, 0, None) == -3
    assert f(desc(data_stride=1 << 32), None, 0, None) == -2 and f(desc(data_stride=-16), None, 0, None) == -2
    many = desc(lq=1, lk=100000)
    assert lib.dpa_cross_attention_mxfp4_workspace_bytes(many) > 0
    assert f(many, None, 0, None) == -5
    assert f(desc(b=0), None, 0, None) == 0


def test_text_model_in_four_bits_on_the_cpu(tmp_path):
    """Its parameters are those of the 16-bit one, its file says which it is, and older files still load."""
    T, U, X = (dpa_mod(n) for n in ("trainer", "unet", "text_unet"))
    config = U.UNetConfig(in_channels=3, base_hidden=64, scales=[1, 2], n_heads=2, p_drop=0.1, attn_resolutions=[16],
                          in_resolution=16, n_resblocks=2)
    m = X.TextUNet(config, X.TextConfig(vocab=11, width=24, mxfp4=True))
    plain = X.TextUNet(config, X.TextConfig(vocab=11, width=24))
    plain.load_state_dict(m.state_dict())
    path = tmp_path / "four.pt"
    T.save_checkpoint(m, 2, config.as_dict(), str(path))
    assert T.load_checkpoint(path)[0].text.text.mxfp4
    old = torch.load(path, weights_only=True)
    del old["text"]["mxfp4"]
    torch.save(old, path)
    back = T.load_checkpoint(path)[0]
    assert not back.text.text.mxfp4 and type(back.cross["mid"].q) is torch.nn.Linear
    tokens = torch.zeros(1, 4, dtype=torch.int64)
    with pytest.raises(ValueError, match="16 or 4 bits"):
        m.keep_prompt(tokens, bits=8)
    odd = X.TextUNet(U.UNetConfig(in_channels=3, base_hidden=64, scales=[1, 2], n_heads=4, p_drop=0.1,
                                  attn_resolutions=[16], in_resolution=16, n_resblocks=2),
                     X.TextConfig(vocab=11, width=24))
    with pytest.raises(ValueError, match="multiple of 32"):
        odd.keep_prompt(tokens, bits=4)
