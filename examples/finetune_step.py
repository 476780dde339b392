"""Fine-tuning steps of a small RWKV-shaped language model on one GPU, with every
operator of rwkvq.train next to the packed ones.

The table is trained (ScaledEmbedding) and so are the dense receptance gate and the
output projection (LinearAct: sigmoid, and the float32 residual stream added in
the product's output stage) and the dense FFN of the first block (relu^2); the second block's
FFN is frozen in 4 bits with adapters (LoRALinear), the head is frozen in 4 bits.
Every step clips the gradients' global norm.

    python examples/finetune_step.py [--steps 20]
"""
import argparse
import os
import sys

import torch
from torch import nn
from torch.nn import functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "rwkv-metal_amd"))
import rwkvq  # noqa: E402


class Block(nn.Module):
    """h + o(sigmoid(r x) * v x), then h + FFN(x) with relu^2 between its products."""

    def __init__(self, d, packed, **kw):
        super().__init__()
        self.norm1, self.norm2 = nn.LayerNorm(d, **kw), nn.LayerNorm(d, **kw)
        self.r = rwkvq.LinearAct(d, d, activation="sigmoid", **kw)
        self.v = rwkvq.LinearAct(d, d, bias=False, **kw)
        self.o = rwkvq.LinearAct(d, d, bias=False, **kw)
        self.packed = packed
        if packed:
            self.key = rwkvq.LoRALinear(nn.Linear(d, 4 * d, bias=False, **kw), rank=16, quantize_base=4)
            self.value = rwkvq.LoRALinear(nn.Linear(4 * d, d, bias=False, **kw), rank=16, quantize_base=4)
            for m in (self.key, self.value):
                m.linear.requires_grad_(False)
        else:
            self.key = rwkvq.LinearAct(d, 4 * d, bias=False, activation="relu2", **kw)
            self.value = rwkvq.LinearAct(4 * d, d, bias=False, **kw)

    def forward(self, h):
        x = self.norm1(h.to(torch.bfloat16))
        h = self.o(self.r(x) * self.v(x), residual=h)
        x = self.norm2(h.to(torch.bfloat16))
        if self.packed:
            return h + self.value(torch.relu(self.key(x)) ** 2)
        return self.value(self.key(x), residual=h)


class Model(nn.Module):
    def __init__(self, vocab=512, d=256, device="cuda"):
        super().__init__()
        kw = {"device": device, "dtype": torch.bfloat16}
        self.emb = rwkvq.ScaledEmbedding(vocab, d, scale=d ** 0.5, **kw)
        nn.init.normal_(self.emb.weight, std=d ** -0.5)
        self.blocks = nn.ModuleList([Block(d, False, **kw), Block(d, True, **kw)])
        self.norm = nn.LayerNorm(d, **kw)
        self.head = rwkvq.QuantizedLinear.from_linear(nn.Linear(d, vocab, bias=False, **kw))

    def forward(self, idx):
        h = self.emb(idx).float()
        for b in self.blocks:
            h = b(h)
        return self.head(self.norm(h.to(torch.bfloat16)))


def train(steps=20, max_norm=0.5, lr=0.5, seed=0, report=print):
    """The losses and gradient norms of `steps` steps on one batch."""
    torch.manual_seed(seed)
    model = Model()
    params = [p for p in model.parameters() if p.requires_grad]
    opt = torch.optim.SGD(params, lr=lr)
    idx = torch.randint(0, 512, (4, 65), device="cuda")
    losses, norms = [], []
    for step in range(steps):
        logits = model(idx[:, :-1])
        loss = F.cross_entropy(logits.float().reshape(-1, logits.shape[-1]), idx[:, 1:].reshape(-1))
        opt.zero_grad(set_to_none=True)
        loss.backward()
        norm = rwkvq.clip_grad_norm_(params, max_norm)
        opt.step()
        losses.append(loss.item())
        norms.append(norm.item())
        report(f"step {step}: loss {losses[-1]:.4f}, gradient norm {norms[-1]:.3f}")
    return losses, norms


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=20)
    train(ap.parse_args().steps)
