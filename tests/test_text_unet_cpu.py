"""The text-conditioned U-Net's checkpoints."""
from __future__ import annotations

import pytest
import torch

from conftest import dpa_mod

T = dpa_mod("trainer")
U = dpa_mod("unet")
X = dpa_mod("text_unet")


def _config():
    return U.UNetConfig(in_channels=3, base_hidden=64, scales=[1, 2], n_heads=2, p_drop=0.1, attn_resolutions=[16],
                        in_resolution=16, n_resblocks=2)


def _same(a, b):
    a, b = a.state_dict(), b.state_dict()
    assert list(a) == list(b) and all(torch.equal(a[k], b[k]) for k in a)


def test_checkpoint_of_a_text_model(tmp_path):
    """It comes back as one, from the file alone or into a model; a plain model's file is as it was."""
    m = X.TextUNet(_config(), X.TextConfig(vocab=11, width=24, p_drop=0.3, padding_idx=2))
    path = tmp_path / "text.pt"
    T.save_checkpoint(m, 5, m.config.as_dict(), str(path))
    back, step, config = T.load_checkpoint(path)
    assert type(back) is X.TextUNet and step == 5 and config == m.config.as_dict()
    assert back.text.text == m.text.text
    _same(back, m)
    other = X.TextUNet(_config(), X.TextConfig(vocab=11, width=24))
    assert T.load_checkpoint(path, other)[0] is other
    _same(other, m)
    compiled = {"_orig_mod." + k: v for k, v in m.state_dict().items()}
    torch.save({**torch.load(path, weights_only=True), "model_state_dict": compiled}, tmp_path / "c.pt")
    _same(T.load_checkpoint(tmp_path / "c.pt")[0], m)
    with pytest.raises(RuntimeError):
        T.load_checkpoint(path, X.TextUNet(_config(), X.TextConfig(vocab=12, width=24)))

    base = U.UNet(_config())
    T.save_checkpoint(base, 1, base.config.as_dict(), str(tmp_path / "base.pt"))
    assert set(torch.load(tmp_path / "base.pt", weights_only=True)) == set(T.CHECKPOINT_KEYS)
    assert type(T.load_checkpoint(tmp_path / "base.pt")[0]) is U.UNet


def test_checkpoint_of_a_compiled_text_model(tmp_path):
    m = X.TextUNet(_config(), X.TextConfig(vocab=7, width=16))
    T.save_checkpoint(torch.compile(m), 3, m.config.as_dict(), str(tmp_path / "c.pt"))
    _same(T.load_checkpoint(tmp_path / "c.pt")[0], m)
