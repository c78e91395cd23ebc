"""Refusals of the conditioning operators: the Python functions' and the C entries' argument checks
(nothing is launched, no GPU needed)."""
from __future__ import annotations

import ctypes
import struct

import pytest
import torch

from conftest import dpa_mod

C = dpa_mod("conditioning")
L = dpa_mod("_lib")

FAKE = 0x1000       # never dereferenced: every call below fails a check first


def _desc(q=FAKE, k=FAKE, v=FAKE, out=FAKE, lse=FAKE, klen=0, mask=0, dout=FAKE, dq=FAKE, dk=FAKE,
          dv=FAKE, strides=(64, 64, 64), k_strides=(64, 64, 64), dtype=0, b=1, lq=1, lk=1, h=1, g=1,
          d=64, scale=0.125):
    return C._DESC.pack(q, k, v, out, lse, klen, mask, dout, dq, dk, dv, 0, *strides, *k_strides,
                        *strides, *strides, *strides, *strides, dtype, b, lq, lk, h, g, d, scale)


@pytest.mark.parametrize("entry", ["dpa_cross_attention_fwd", "dpa_cross_attention_bwd"])
@pytest.mark.parametrize("kw,status", [
    (dict(q=0), -1), (dict(k=0), -1), (dict(out=0), -1), (dict(lse=0), -1),
    (dict(dtype=1), -4), (dict(dtype=7), -4), (dict(b=-1), -2), (dict(lq=-1), -2), (dict(lk=-1), -2),
    (dict(h=0), -2), (dict(g=0), -2), (dict(h=3, g=2), -4), (dict(d=0), -4), (dict(d=12), -4),
    (dict(d=136), -4), (dict(scale=0.0), -2), (dict(scale=-1.0), -2), (dict(scale=float("nan")), -2),
    (dict(scale=float("inf")), -2), (dict(q=FAKE + 2), -3), (dict(v=FAKE + 8), -3),
    (dict(strides=(64, 60, 64)), -3), (dict(k_strides=(63, 64, 64)), -3), (dict(klen=FAKE + 2), -3),
    (dict(b=1 << 20, h=1 << 12, g=1 << 12), -2), (dict(lq=1 << 30), -2), (dict(lk=1 << 30), -2),
])
def test_attention_entry_refuses(entry, kw, status):
    assert getattr(L.load(), entry)(_desc(**kw), None, 0, None) == status


def test_attention_entry_null_and_workspace():
    lib = L.load()
    assert lib.dpa_cross_attention_fwd(None, None, 0, None) == -1
    assert lib.dpa_cross_attention_bwd(None, None, 0, None) == -1
    for kw in (dict(dout=0), dict(dq=0), dict(dk=0), dict(dv=0)):
        assert lib.dpa_cross_attention_bwd(_desc(**kw), None, 0, None) == -1
    # one query over many keys is split: a workspace is needed
    long = _desc(lk=4096)
    need = lib.dpa_cross_attention_fwd_workspace_bytes(long)
    assert need > 0
    assert lib.dpa_cross_attention_fwd(long, None, 0, None) == -5
    assert lib.dpa_cross_attention_fwd(long, FAKE, need - 1, None) == -5
    assert lib.dpa_cross_attention_fwd(long, FAKE + 4, need, None) == -3
    assert lib.dpa_cross_attention_bwd(_desc(), None, 0, None) == -5
    # nothing to do
    assert lib.dpa_cross_attention_fwd(_desc(b=0), None, 0, None) == 0
    assert lib.dpa_cross_attention_fwd(_desc(lq=0), None, 0, None) == 0
    assert lib.dpa_cross_attention_bwd(_desc(b=0), None, 0, None) == 0
    assert lib.dpa_cross_attention_fwd_workspace_bytes(None) == 0
    assert lib.dpa_cross_attention_bwd_workspace_bytes(_desc(d=12)) == 0


def test_descriptor_layout():
    """The packed descriptor has the size and offsets of the header's struct."""
    class S(ctypes.Structure):
        _fields_ = ([(f"p{i}", ctypes.c_void_p) for i in range(11)] + [("mask_stride", ctypes.c_int64)]
                    + [(f"s{i}", ctypes.c_int64 * 3) for i in range(6)]
                    + [(f"n{i}", ctypes.c_int32) for i in range(7)] + [("scale", ctypes.c_float)])
    assert ctypes.sizeof(S) == C._DESC.size
    s = S.from_buffer_copy(_desc(scale=0.5, d=40, lk=7, k_strides=(8, 16, 24)))
    assert s.scale == 0.5 and s.n6 == 40 and s.n3 == 7 and list(s.s1) == [8, 16, 24] and s.p10 == FAKE


def test_dropout_entry_refuses():
    f = L.load().dpa_dropout
    assert f(None, None, FAKE, 0, 8, FAKE, 0.1, None) == -1
    assert f(FAKE, None, None, 0, 8, FAKE, 0.1, None) == -1
    assert f(FAKE, None, FAKE, 0, 8, None, 0.1, None) == -1
    assert f(FAKE, None, FAKE, 0, -1, FAKE, 0.1, None) == -2
    for p in (-0.1, 1.0, float("nan")):
        assert f(FAKE, None, FAKE, 0, 8, FAKE, p, None) == -2
    assert f(FAKE, None, FAKE, 3, 8, FAKE, 0.1, None) == -4
    assert f(FAKE + 1, None, FAKE, 0, 8, FAKE, 0.1, None) == -3
    assert f(FAKE + 2, None, FAKE, 1, 8, FAKE, 0.1, None) == -3
    assert f(FAKE, FAKE + 1, FAKE, 0, 8, FAKE, 0.1, None) == -3
    assert f(FAKE, None, FAKE, 0, 8, FAKE + 4, 0.1, None) == -3
    assert f(None, None, None, 0, 0, None, 0.1, None) == 0


def test_embedding_entry_refuses():
    lib = L.load()

    def fwd(tok=FAKE, tb=8, w=FAKE, wt=0, out=FAKE, ot=0, n=4, v=10, c=8, seed=None, p=0.0):
        return lib.dpa_embedding_fwd(tok, tb, w, wt, out, ot, n, v, c, 1.0, seed, p, None)

    def bwd(g=FAKE, gt=0, tok=FAKE, tb=8, dw=FAKE, wt=0, n=4, v=10, c=8, seed=None, p=0.0, ws=FAKE,
            nb=1 << 20):
        return lib.dpa_embedding_bwd(g, gt, tok, tb, dw, wt, n, v, c, 1.0, -1, seed, p, ws, nb, None)
    for f in (fwd, bwd):
        assert f(tok=None) == -1
        assert f(tb=2) == -4 and f(wt=3) == -4
        assert f(n=-1) == -2 and f(v=0) == -2 and f(c=0) == -2 and f(n=1 << 31) == -2 and f(v=1 << 31) == -2
        assert f(seed=FAKE, p=1.0) == -2 and f(seed=FAKE + 4, p=0.1) == -3
        assert f(tok=FAKE + 4) == -3
    assert fwd(w=None) == -1 and fwd(out=None) == -1 and fwd(n=0, tok=None, w=None, out=None) == 0
    assert bwd(g=None) == -1 and bwd(dw=None) == -1
    need = lib.dpa_embedding_bwd_workspace_bytes(4, 8)
    assert bwd(ws=None) == -5 and bwd(nb=need - 1) == -5
    assert bwd(dw=FAKE + 8) == -3 and bwd(ws=FAKE + 4) == -3
    assert lib.dpa_embedding_bwd_workspace_bytes(0, 8) == 0


def _qkv(b=2, lq=3, lk=5, h=4, g=2, d=16, dtype=torch.bfloat16):
    return (torch.zeros((b, lq, h, d), dtype=dtype), torch.zeros((b, lk, g, d), dtype=dtype),
            torch.zeros((b, lk, g, d), dtype=dtype))


def test_attention_refuses():
    q, k, v = _qkv()
    for args in [(q[0], k, v), (q, k[:1], v[:1]), (q, k, v[:, :4]), (q.float(), k, v),
                 (q.float(), k.float(), v.float()), (q.half(), k, v), (q[..., :12], k[..., :12], v[..., :12]),
                 (q[:, :, :3], k, v), _qkv(d=136), (q[..., :0], k[..., :0], v[..., :0]),
                 (q, k, v)]:          # the last: not on a GPU
        with pytest.raises(ValueError, match="cross attention|GPU"):
            C.cross_attention_fwd(*args)
        with pytest.raises(ValueError, match="cross attention|GPU"):
            C.cross_attention(*args)
    with pytest.raises(ValueError, match="kv is"):
        C.cross_attention_kv(q, k)
    for kw in [dict(key_lengths=torch.zeros(3, dtype=torch.int32)), dict(key_lengths=torch.zeros(2)),
               dict(key_mask=torch.zeros((2, 4), dtype=torch.bool)), dict(key_mask=torch.zeros((2, 5)))]:
        kw = {"key_lengths": None, "key_mask": None, **kw}
        with pytest.raises(ValueError, match="key_lengths|key_mask"):
            C._check_masks(q, k, **kw)
    for s in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale"):
            C._scale_of(s, 64)


def test_dropout_and_embedding_refuse():
    x, seed = torch.zeros(4, 8), torch.zeros(1, dtype=torch.int64)
    for p in (-0.1, 1.0, 1.0 - 1e-12, float("nan")):
        with pytest.raises(ValueError, match="not in"):
            C.dropout_fwd(x, p, seed)
        with pytest.raises(ValueError, match="not in"):
            C.dropout(x, p)
        with pytest.raises(ValueError, match="not in"):
            C.embedding(torch.zeros(3, dtype=torch.int64), x, p_drop=p)
    with pytest.raises(ValueError, match="fp32"):
        C.dropout_fwd(x.double(), 0.1, seed)
    with pytest.raises(ValueError, match="GPU"):
        C.dropout_fwd(x, 0.1, seed)
    with pytest.raises(ValueError, match="seed"):
        C._check_seed(seed.int(), x, "dropout")
    with pytest.raises(ValueError, match="seed"):
        C._check_seed(None, x, "dropout")
    with pytest.raises(ValueError, match="weight"):
        C.embedding_fwd(torch.zeros(3, dtype=torch.int64), x[0])
    with pytest.raises(ValueError, match="tokens"):
        C.embedding_fwd(torch.zeros(3), x)
    with pytest.raises(ValueError, match="fp32"):
        C.embedding_fwd(torch.zeros(3, dtype=torch.int64), x.double())
    with pytest.raises(ValueError, match="GPU"):
        C.embedding_fwd(torch.zeros(3, dtype=torch.int64), x)
    with pytest.raises(ValueError, match="padding_idx"):
        C.embedding(torch.zeros(3, dtype=torch.int64), x, padding_idx=4)
    with pytest.raises(ValueError, match="does not go"):
        C.embedding_bwd(x, torch.zeros(3, dtype=torch.int64), 10)
    # without training they are the identity and refuse nothing of dropout
    assert C.dropout(x, 0.3, training=False) is x and C.dropout(x, 0.0) is x
    assert torch.equal(C.dropout(x, 0.3, training=False, residual=x + 1), x + 1)


def test_p_as_fp32_below_one():
    assert struct.unpack("f", struct.pack("f", 1.0 - 1e-12))[0] == 1.0     # what the check is for
    assert C._check_p(0.999999, "dropout") == 0.999999


def test_text_unet_structure():
    U, X = dpa_mod("unet"), dpa_mod("text_unet")
    cfg = U.UNetConfig(in_channels=3, base_hidden=64, scales=[1, 2, 2], n_heads=2, p_drop=0.1,
                       attn_resolutions=[16], in_resolution=32, n_resblocks=2)
    m = X.TextUNet(cfg, X.TextConfig(vocab=11, width=24))
    base = U.UNet(cfg)
    assert set(base.state_dict()) <= set(m.state_dict())
    assert sorted(m.cross) == ["down1", "mid", "up1"]
    assert m.cross["down1"].q.in_features == 128 and m.cross["up1"].q.in_features == 128
    assert not m.text.weight[0].any() and all(not b.out.weight.any() for b in m.cross.values())
    m.train()
    assert m._dropouts() == base.train()._dropouts() + 4
    assert m.eval()._dropouts() == 0
    # without a prompt it runs as the base model does, on the CPU too
    x, t = torch.randn(1, 3, 32, 32), torch.tensor([3])
    assert torch.equal(m(x, t), base.eval()(x, t))            # (both start at zero)
    with pytest.raises(ValueError, match="cross attention block"):
        X.CrossAttentionBlock(60, X.TextConfig(vocab=11, width=24), 8)
    with pytest.raises(ValueError, match="GPU"):
        m(x, t, torch.ones((1, 5), dtype=torch.int64))


def test_fast_calls_take_plain_gpu_tensors_only():
    """The native calls leave everything else to the general way (None), without touching it."""
    fast = L.fast_calls()
    assert fast is not None
    q, k, v = _qkv()
    x, seed = torch.zeros(4, 8), torch.zeros(1, dtype=torch.int64)
    t = torch.zeros(4, dtype=torch.int64)
    assert fast.attention_fwd(q, k, v, None, None, None) is None
    assert fast.attention_fwd(q, None, v, None, None, None) is None
    assert fast.attention_fwd(q, k) is None and fast.attention_fwd(1, "a", [], {}, (), 0) is None
    assert fast.attention_bwd(q, q, k, v, q, q, None, None, None, True, True) is None
    assert fast.dropout(x, 0.1, seed, None) is None and fast.dropout(x) is None
    assert fast.embedding_fwd(t, x, 1.0, 0.0, None, None) is None
    assert fast.embedding_bwd(x, t, 5, 1.0, -1, 0.0, None, None) is None
