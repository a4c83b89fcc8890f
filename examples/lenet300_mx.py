"""LeNet-300-100 trained in microscaled 4-bit floating point with AdamW (8-bit moments), then served from 4-bit
weights.  Synthetic digits: ten noisy prototypes of 28 x 28.

    python examples/lenet300_mx.py [--steps 300] [--state-bits 8]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from approxtrain_amd.layers import densemx  # noqa: E402
from approxtrain_amd.optimizers import AdamW  # noqa: E402


def batch(prototypes, n, generator):
    labels = torch.randint(0, 10, (n,), device="cuda", generator=generator)
    return prototypes[labels] + torch.randn((n, 784), device="cuda", generator=generator), labels


def train(steps=300, state_bits=8, rows=128, seed=0):
    """(the trained layers, losses, the accuracy of the layers and of their packed form on fresh digits)"""
    generator = torch.Generator(device="cuda").manual_seed(seed)
    torch.manual_seed(seed)
    prototypes = torch.randn((10, 784), device="cuda", generator=generator) * 0.5
    model = torch.nn.Sequential(densemx(300, "relu", input_dim=784), densemx(100, "relu", input_dim=300), densemx(10, input_dim=100)).cuda()
    optimizer = AdamW(model.parameters(), lr=2e-3, state_bits=state_bits)
    losses = []
    for _ in range(steps):
        x, labels = batch(prototypes, rows, generator)
        optimizer.zero_grad()
        loss = torch.nn.functional.cross_entropy(model(x), labels)
        loss.backward()
        norm = torch.linalg.vector_norm(torch.cat([p.grad.reshape(-1) for p in model.parameters()]))
        optimizer.step(grad_scale=torch.clamp(1.0 / norm, max=1.0))  # (gradients longer than 1 are cut to it)
        losses.append(loss.detach())
    x, labels = batch(prototypes, 2000, generator)
    packed = torch.nn.Sequential(*[layer.pack() for layer in model])
    with torch.no_grad():
        accuracy = [float((m(x).argmax(-1) == labels).float().mean()) for m in (model, packed)]
    return model, packed, torch.stack(losses).tolist(), accuracy


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=300)
    ap.add_argument("--state-bits", type=int, default=8, choices=(8, 32))
    args = ap.parse_args()
    _, packed, losses, (trained, served) = train(args.steps, args.state_bits)
    weights = sum(b.numel() * b.element_size() for b in packed.buffers())
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f} in {args.steps} steps; accuracy {trained:.3f}, served from {weights} bytes of weights and biases {served:.3f}")


if __name__ == "__main__":
    main()
