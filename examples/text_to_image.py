"""Trains a small text-conditioned U-Net on coloured shapes and samples it from prompts.

    python examples/text_to_image.py [--steps 300] [--batch 64] [--prompts "red square" ...]

The images and captions are made here: a square, a disc or a cross of one of four colours on a
grey ground, captioned by its colour and shape in that order, with one caption in ten dropped. One
training step -- token embedding, cross attention at two levels, dropout, the U-Net, loss, AdamW and
EMA -- is captured into a HIP graph and replayed. Sampling projects the prompts' keys and values
once and keeps them over the denoising steps. Needs a gfx950 GPU.
"""
from __future__ import annotations

import argparse
import importlib
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
PKG = "diffusion-profiled_amd"

COLOURS = {"red": (1.0, -1.0, -1.0), "green": (-1.0, 1.0, -1.0), "blue": (-1.0, -1.0, 1.0),
           "yellow": (1.0, 1.0, -1.0)}
SHAPES = ("square", "disc", "cross")
WORDS = ["<pad>", *COLOURS, *SHAPES]
LENGTH = 8


def tokenize(prompts: list[str]) -> torch.Tensor:
    out = torch.zeros((len(prompts), LENGTH), dtype=torch.int64)
    for i, text in enumerate(prompts):
        ids = [WORDS.index(w) for w in text.split()]
        out[i, :len(ids)] = torch.tensor(ids, dtype=torch.int64)
    return out


def draw_batch(n: int, size: int, g: torch.Generator) -> tuple[torch.Tensor, torch.Tensor]:
    """(images [n, 3, size, size], tokens [n, LENGTH])"""
    images = torch.zeros((n, 3, size, size))
    prompts = []
    yy, xx = torch.meshgrid(torch.arange(size), torch.arange(size), indexing="ij")
    names = list(COLOURS)
    for i in range(n):
        colour = names[int(torch.randint(len(names), (1,), generator=g))]
        shape = SHAPES[int(torch.randint(len(SHAPES), (1,), generator=g))]
        r = int(torch.randint(size // 6, size // 3, (1,), generator=g))
        cy, cx = (int(torch.randint(r, size - r, (1,), generator=g)) for _ in range(2))
        dy, dx = (yy - cy).abs(), (xx - cx).abs()
        inside = {"square": (dy <= r) & (dx <= r), "disc": dy**2 + dx**2 <= r * r,
                  "cross": ((dy <= r // 3) & (dx <= r)) | ((dx <= r // 3) & (dy <= r))}[shape]
        images[i] = torch.where(inside, torch.tensor(COLOURS[colour])[:, None, None], images[i])
        dropped = float(torch.rand(1, generator=g)) < 0.1
        prompts.append("" if dropped else f"{colour} {shape}")
    return images, tokenize(prompts)


def main(argv: list[str] | None = None) -> list[float]:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=300)
    ap.add_argument("--batch", type=int, default=64)
    ap.add_argument("--size", type=int, default=16)
    ap.add_argument("--max-t", type=int, default=200)
    ap.add_argument("--prompts", nargs="*", default=["red square", "blue disc"])
    args = ap.parse_args(argv)
    trainer = importlib.import_module(f"{PKG}.trainer")
    unet = importlib.import_module(f"{PKG}.unet")
    text_unet = importlib.import_module(f"{PKG}.text_unet")

    config = unet.UNetConfig(in_channels=3, base_hidden=64, scales=[1, 2], n_heads=2, p_drop=0.1,
                             attn_resolutions=[args.size], in_resolution=args.size, n_resblocks=2)
    text = text_unet.TextConfig(vocab=len(WORDS), width=64)
    state = trainer.TrainState(config, args.batch, lr=1e-3, max_t=args.max_t, text=text,
                               prompt_length=LENGTH, ema_beta=0.99)
    g = torch.Generator().manual_seed(0)
    batches = [draw_batch(args.batch, args.size, g) for _ in range(16)]
    state.set_batch(batches[0][0].cuda(), tokens=batches[0][1].cuda())
    state.capture()
    state.loss_acc.zero_()
    losses = []
    for i in range(args.steps):
        images, tokens = batches[i % len(batches)]
        state.set_batch(images.cuda(), tokens=tokens.cuda())
        state.replay()
        if (i + 1) % 50 == 0 or i + 1 == args.steps:
            n = 50 if (i + 1) % 50 == 0 else (i + 1) % 50
            losses.append(float(state.loss_acc) / n)
            state.loss_acc.zero_()
            print(f"step {i + 1}: mean loss {losses[-1]:.4f}", flush=True)
    model = state.ema_ddpm.model.model
    model.keep_prompt(tokenize(args.prompts).cuda())
    samples = state.ema_ddpm.generate_samples(len(args.prompts))
    model.keep_prompt(None)
    for prompt, image in zip(args.prompts, samples):
        spread = image.flatten(1).amax(1) - image.flatten(1).amin(1)
        print(f"{prompt!r}: channel means {image.mean((1, 2)).tolist()}, spreads {spread.tolist()}")
    return losses


if __name__ == "__main__":
    main()
