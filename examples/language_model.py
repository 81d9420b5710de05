"""A language model's step from the library's operators, trained and served.

    python examples/language_model.py

Training: embedding rows -> a layer in 8-bit products -> cross entropy, with
the gradients of both tables (torch_embedding, torch_scaled_linear).  Serving:
embedding -> a mixture-of-experts layer -> the output layer stored in 8 bits
(embedding, expert_layer, quantize_blocks, scaled_linear).
"""

from __future__ import annotations

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "ndtensors-rs_b200"))

import ndtensors_b200 as ndt  # noqa: E402


def train_step(table, weight, ids, targets, rate=0.5):
    """One step of gradient descent on the next-id loss, in place; returns the loss before it."""
    hidden = ndt.torch_embedding(table, ids, scale=table.shape[1] ** 0.5)
    logits = ndt.torch_scaled_linear(hidden, weight)
    loss = torch.nn.functional.cross_entropy(logits.float(), targets)
    grads = torch.autograd.grad(loss, (table, weight))
    with torch.no_grad():
        for p, g in zip((table, weight), grads):
            p -= rate * g
    return loss.detach()


class Decoder:
    """The serving form: weights laid out once, one call for each decoding step."""

    def __init__(self, table, router, w_in, w_out, weight, top=2):
        self.table, self.router, self.w_in, self.w_out, self.top = table, router, w_in, w_out, top
        self.weight, self.scales = ndt.quantize_blocks(weight, block_rows=128)

    def logits(self, ids):
        """[tokens] ids -> [tokens, vocabulary]."""
        x = ndt.embedding(self.table, ids, scale=self.table.shape[1] ** 0.5)
        y, _, _ = ndt.expert_layer(x, self.router, self.w_in, self.w_out, self.top)
        return ndt.scaled_linear(x + y, self.weight, self.scales, out_dtype=torch.float32)

    def next_ids(self, ids):
        return self.logits(ids).argmax(1)


def make(vocabulary=1000, dim=256, experts=8, inner=384, dtype=torch.bfloat16, seed=0):
    """Random parameters: (table, router, w_in, w_out, weight)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    return ((normal(vocabulary, dim) * dim ** -0.5).to(dtype), (normal(experts, dim) * dim ** -0.5).to(dtype),
            (normal(experts, 2 * inner, dim) * dim ** -0.5).to(dtype), (normal(experts, dim, inner) * inner ** -0.5).to(dtype),
            (normal(vocabulary, dim) * dim ** -0.5).to(dtype))


def main():
    table, router, w_in, w_out, weight = make()
    v = table.shape[0]
    follow = torch.randperm(v, device="cuda")  # the id that follows each id
    t, w = table.float().requires_grad_(), weight.float().requires_grad_()
    for step in range(30):
        ids = torch.randint(0, v, (2048,), device="cuda")
        loss = train_step(t, w, ids, follow[ids], rate=20.0)
        if step % 10 == 9:
            print(f"step {step + 1}: loss {float(loss):.3f}")
    decoder = Decoder(t.detach().to(torch.bfloat16), router, w_in, w_out, w.detach().to(torch.bfloat16))
    print("next ids:", decoder.next_ids(torch.arange(8, device="cuda")).tolist())


if __name__ == "__main__":
    main()
