"""Trains a small sparse autoencoder with the fused loss and the fused optimiser, as a training script uses them together.

The data are sums of K / 2 directions of a hidden dictionary of F / 16.  An encoder picks the K latents of a row with the largest
activations; the hierarchical loss reconstructs the row from every prefix of them, with one backward for the decoder, the
activations and the bias; one optimizer steps everything, with the decoder's rows held at length one, gradients clipped to a
common norm, and moments in 32 or 8 bits.

    python examples/train_sae.py --bits 8 --dtype bf16 --steps 200
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import flexsae_amd as flex  # noqa: E402


class SAE(torch.nn.Module):
    def __init__(self, F, D, K, dtype, device):
        super().__init__()
        decoder = torch.randn(F, D, device=device)
        decoder /= decoder.norm(dim=1, keepdim=True)
        self.K = K
        self.W_dec = torch.nn.Parameter(decoder.to(dtype))
        self.W_enc = torch.nn.Parameter(decoder.to(dtype, copy=True))
        self.b_enc = torch.nn.Parameter(torch.zeros(F, dtype=dtype, device=device))
        self.b_dec = torch.nn.Parameter(torch.zeros(D, dtype=dtype, device=device))

    def loss(self, x):
        activations = (x - self.b_dec.detach()) @ self.W_enc.t() + self.b_enc
        vals, indices = activations.topk(self.K, dim=1)
        return flex.triton_hierarchical_sae_loss(indices, self.W_dec, vals.relu(), self.b_dec, x)


def train(F=4096, D=256, K=32, B=512, steps=100, bits=8, dtype=torch.bfloat16, lr=1e-3, seed=0, device="cuda"):
    """-> the losses of all steps, the model, the optimizer"""
    torch.manual_seed(seed)
    model = SAE(F, D, K, dtype, device)
    opt = flex.AdamW([{"params": [model.W_dec], "unit_rows": True, "weight_decay": 0.0},
                      {"params": [model.W_enc, model.b_enc, model.b_dec]}],
                     lr=lr, weight_decay=1e-4, state_bits=bits, max_norm=1.0)
    hidden = torch.nn.functional.normalize(torch.randn(F // 16, D, device=device), dim=1)
    scale = 65536.0 if dtype == torch.float16 else 1.0  # gradients of about 2 / (B K D) vanish in fp16
    losses = []
    for _ in range(steps):
        which = torch.randint(0, F // 16, (B, K // 2), device=device)
        x = (hidden[which] * torch.rand(B, K // 2, 1, device=device)).sum(1).to(dtype)
        loss = model.loss(x)
        opt.zero_grad(set_to_none=True)
        (loss * scale).backward()
        opt.step(grad_scale=scale)
        losses.append(loss.detach())
    return torch.stack(losses).tolist(), model, opt


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--bits", type=int, choices=(32, 8), default=8, help="of the optimizer's moments")
    ap.add_argument("--dtype", choices=("fp32", "bf16", "fp16"), default="bf16")
    a = ap.parse_args()
    dtype = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}[a.dtype]
    losses, model, opt = train(steps=a.steps, bits=a.bits, dtype=dtype)
    for i in range(0, a.steps, max(1, a.steps // 10)):
        print(f"step {i:5d}  loss {losses[i]:.5f}")
    lengths = model.W_dec.detach().float().norm(dim=1)
    m, v = opt.moments(model.W_dec)
    print(f"last loss {losses[-1]:.5f}, gradient norm {opt.grad_norm.item():.3g}, "
          f"decoder rows of length {lengths.min().item():.4f} to {lengths.max().item():.4f}, "
          f"moments of its first row {m[0].norm().item():.3g} and {v[0].sqrt().norm().item():.3g}")


if __name__ == "__main__":
    main()
