"""Trains a sequence encoder through the soft-DTW loss, then encodes a live stream with it.

    python examples/train_encoder.py [--steps 60] [--state-bits 8]

Every step runs this package's operators together as a training program would: layer norm, linear
with its activation and residual, and the gated recurrence in the encoder, soft-DTW on the
features, and AdamW on all weights.  The data are synthetic: noisy, time-warped copies of a few
reference curves; the encoder learns features in which a curve aligns with its own reference
better than with the others.  At the end the same encoder takes the curves frame by frame, with
its states carried along, and gives the features that it gives for whole sequences.
"""

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))  # the package beside this folder

import torchwarp_b200 as torchwarp  # noqa: E402
import torchwarp_b200.functional as TF  # noqa: E402


def curves(batch, frames, classes, generator, device):
    """Warped, noisy copies [batch, frames, 3] of `classes` reference curves, and their classes."""
    label = torch.randint(classes, (batch,), generator=generator, device=device)
    pace = torch.rand(batch, frames, generator=generator, device=device) + 0.2
    time = pace.cumsum(1) / pace.sum(1, keepdim=True)
    angle = 6.28 * time * (1 + label).unsqueeze(1)
    clean = torch.stack([angle.sin(), angle.cos(), (2 * angle).sin()], -1)
    noise = 1.0 * torch.randn(clean.shape, generator=generator, device=device)
    return clean + noise, label


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--state-bits", type=int, default=8, choices=(8, 32))
    args = ap.parse_args()
    device = torch.device("cuda")
    torch.manual_seed(0)
    generator = torch.Generator(device=device).manual_seed(0)
    classes, frames, dim = 4, 64, 64

    encoder = torchwarp.SequenceEncoder(3, dim, layers=2, device=device)
    optimizer = torchwarp.AdamW(encoder.parameters(), lr=2e-3, state_bits=args.state_bits)
    angle = 6.28 * torch.linspace(0, 1, frames, device=device) * torch.arange(
        1, classes + 1, device=device).unsqueeze(1)
    references = torch.stack([angle.sin(), angle.cos(), (2 * angle).sin()], -1)

    def scores(x):
        """[batch, classes]: minus the alignment cost with each reference, a frame and feature."""
        a, b = encoder(x), encoder(references)
        pairs = TF.soft_dtw(a.repeat_interleave(classes, 0), b.repeat(len(a), 1, 1), gamma=1.0)
        return -pairs.view(len(a), classes) / (frames * dim)

    for step in range(args.steps):
        x, label = curves(32, frames, classes, generator, device)
        loss = torch.nn.functional.cross_entropy(scores(x), label)
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        if step % 20 == 0 or step == args.steps - 1:
            print("step {:3d}  loss {:.4f}".format(step, loss.item()))

    x, label = curves(128, frames, classes, generator, device)
    with torch.no_grad():
        right = (scores(x).argmax(1) == label).float().mean().item()
        whole = encoder(x)
        states = encoder.init_state(len(x))
        live = torch.stack([encoder.step(x[:, t], states) for t in range(frames)], 1)
    print("classified {:.0%}; streamed features differ by at most {:.1e}".format(
        right, (live - whole).abs().max().item()))


if __name__ == "__main__":
    main()
