"""A byte-level LUT transformer whose blocks join by norm, gate and counter-based dropout, trained
for a few steps on this package's own sources and asked for a continuation.

    python examples/byte_model.py [--steps N] [--new N]
"""
import argparse
import glob
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
from spiky_amd import LUTTransformer  # noqa: E402


def text():
    files = sorted(glob.glob(os.path.join(ROOT, "spiky_amd", "**", "*.py"), recursive=True))
    return torch.tensor(list(b"".join(open(f, "rb").read() for f in files)), dtype=torch.int64)


def make(device, context=64, seed=1):
    return LUTTransformer(vocab_size=256, embedding_dim=64, context_size=context, positional_dim=4, num_layers=2,
                          num_heads=2, n_detectors=16, n_anchors_per_detector=6, n_anchors_per_detector_attention=4,
                          device=device, seed=seed, dropout=0.05,
                          residual_join=dict(post_norm="rms", pre_norm="rms", gate=0.3))


def train(model, data, steps, batch=16, lr=0.02):
    """The loss of each step."""
    optimizer = torch.optim.Adam(model.parameters(), lr=lr)
    gen = torch.Generator().manual_seed(0)
    S, losses = model.context_size, []
    for _ in range(steps):
        at = torch.randint(0, len(data) - S - 1, (batch,), generator=gen)
        rows = torch.stack([data[i:i + S + 1] for i in at.tolist()]).to(model.device)
        loss = torch.nn.functional.cross_entropy(model(rows[:, :-1]).reshape(-1, 256), rows[:, 1:].reshape(-1))
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


def main():
    parser = argparse.ArgumentParser()
    parser.add_argument("--steps", type=int, default=100)
    parser.add_argument("--new", type=int, default=80)
    args = parser.parse_args()
    device = torch.device("cuda", 0)
    model = make(device)
    losses = train(model, text(), args.steps)
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f} in {args.steps} steps")
    prompt = torch.tensor([list(b"import torch\n")], device=device)
    printable = torch.zeros(256, dtype=torch.bool, device=device)
    printable[[10, *range(32, 127)]] = True
    out = model.generate(prompt, args.new, generator=torch.Generator(device).manual_seed(0), temperature=0.8,
                         repetition_penalty=1.1, frequency_penalty=0.05, mask=printable)
    print(bytes(out[0].tolist()).decode("latin-1"))


if __name__ == "__main__":
    main()
