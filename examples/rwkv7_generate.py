"""A small RWKV-7 language model on one GPU: trained on packed sequences, then given a prompt
and asked for tokens.

The time mixing's recurrence is rwkvq.wkv7 over whole sequences (cu_seqlens: packed ones, their
states apart) and rwkvq.wkv7_step over one token of every sequence, with its state updated in
place; rwkvq.sample chooses the tokens.  The projections are dense (LinearAct) for training; `--packed` freezes them
in 4 bits with adapters, as a fine-tuned base has them.

    python examples/rwkv7_generate.py [--steps 20] [--tokens 32] [--packed]
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

D = 64  # channels of a head


class TimeMix(nn.Module):
    """o(g * (norm(y) + (r . (k u)) v)) of the recurrence's y."""

    def __init__(self, d, low=32, packed=False, **kw):
        super().__init__()
        self.heads = d // D
        self.mix = nn.Parameter(torch.rand(6, d, **kw))
        if packed:
            def dense():
                m = rwkvq.LoRALinear(nn.Linear(d, d, bias=False, **kw), rank=16, quantize_base=4)
                m.linear.requires_grad_(False)
                return m
        else:
            def dense():
                return rwkvq.LinearAct(d, d, bias=False, **kw)
        self.r, self.k, self.v, self.o = dense(), dense(), dense(), dense()
        for name in "wag":
            setattr(self, name + "1", nn.Parameter(torch.randn(d, low, **kw) * d ** -0.5))
            setattr(self, name + "2", nn.Parameter(torch.randn(low, d, **kw) * 0.1 * low ** -0.5))
        self.w0 = nn.Parameter(torch.linspace(-3, 1, d, **kw))
        self.a0 = nn.Parameter(torch.zeros(d, **kw))
        self.k_k, self.k_a = nn.Parameter(torch.ones(d, **kw)), nn.Parameter(torch.ones(d, **kw))
        self.bonus = nn.Parameter(torch.randn(self.heads, D, **kw) * 0.1)
        self.norm = nn.GroupNorm(self.heads, d, eps=64e-5, **kw)

    def operands(self, x, last):
        """The recurrence's six, [..., heads, 64], and the gate, from x and the tokens before."""
        xr, xw, xk, xv, xa, xg = (torch.lerp(x, last, m) for m in self.mix)
        heads = (*x.shape[:-1], self.heads, D)
        r, k, v = self.r(xr).view(heads), self.k(xk), self.v(xv).view(heads)
        w = -F.softplus(-(self.w0 + torch.tanh(xw @ self.w1) @ self.w2)) - 0.5
        a = torch.sigmoid(self.a0 + xa @ self.a1 @ self.a2)
        gate = torch.sigmoid(xg @ self.g1) @ self.g2
        kk = F.normalize((k * self.k_k).view(heads), dim=-1)
        k = (k * (1 + (a - 1) * self.k_a)).view(heads)
        return (r, w.view(heads), k, v, -kk, kk * a.view(heads)), gate

    def output(self, y, six, gate):
        r, _, k, v, _, _ = six
        y = self.norm(y.reshape(-1, self.heads * D)).view(y.shape)
        y = y + (r * k * self.bonus).sum(-1, keepdim=True) * v
        return self.o((1 + gate) * y.flatten(-2))

    def forward(self, x, last, state, cu):
        six, gate = self.operands(x, last)
        y, state = rwkvq.wkv7(*six, state, cu)
        return self.output(y, six, gate), state

    def step(self, x, last, state):
        six, gate = self.operands(x, last)
        y, _ = rwkvq.wkv7_step(*six, state, out=state)
        return self.output(y, six, gate)


class Block(nn.Module):
    def __init__(self, d, **kw):
        super().__init__()
        kw = dict(kw)
        self.time = TimeMix(d, packed=kw.pop("packed"), **kw)
        self.norm1, self.norm2 = nn.LayerNorm(d, **kw), nn.LayerNorm(d, **kw)
        self.key = rwkvq.LinearAct(d, 4 * d, bias=False, activation="relu2", **kw)
        self.value = rwkvq.LinearAct(4 * d, d, bias=False, **kw)


class Model(nn.Module):
    def __init__(self, vocab=512, d=128, blocks=2, packed=False, device="cuda", dtype=torch.bfloat16):
        super().__init__()
        kw = {"device": device, "dtype": dtype}
        self.emb = nn.Embedding(vocab, d, **kw)
        self.blocks = nn.ModuleList([Block(d, packed=packed, **kw) for _ in range(blocks)])
        self.norm = nn.LayerNorm(d, **kw)
        self.head = rwkvq.QuantizedLinear.from_linear(nn.Linear(d, vocab, bias=False, **kw))

    def forward(self, idx, state=None, cu=None):
        """(logits, state) of whole sequences, idx [batch, time] or packed [1, time] with their boundaries `cu`.
        The state is a list with (the last token's input, the recurrence's states) of each block, for each
        sequence; a sequence without a token keeps its own."""
        x, after = self.emb(idx), []
        if cu is not None:
            start, end = cu[:-1].long(), cu[1:].long()
            # rows: what the sequences had last, then the tokens.  A token's predecessor is the row before its own, a
            # sequence's first token's what that sequence had last
            seqs, time = torch.arange(start.numel(), device=idx.device), idx.shape[1]
            source = torch.arange(time + 1, device=idx.device) + (len(seqs) - 1)
            source[torch.where(end > start, start, time)] = seqs
            source, left = source[:time], torch.where(end > start, end - 1 + len(seqs), seqs)
        for i, b in enumerate(self.blocks):
            n = b.norm1(x)
            if cu is not None:
                before = n.new_zeros(len(seqs), n.shape[-1]) if state is None else state[i][0]
                rows = torch.cat([before, n[0]])
                last, kept = rows[source][None], rows[left]
            else:
                last = F.pad(n, (0, 0, 1, -1))  # each token's predecessor
                if state is not None:
                    last = torch.cat([state[i][0][:, None], last[:, 1:]], 1)
                kept = n[:, -1]
            y, s = b.time(n, last, None if state is None else state[i][1], cu)
            after.append((kept, s))
            x = x + y
            x = b.value(b.key(b.norm2(x)), residual=x)
        return self.head(self.norm(x)), after

    @torch.no_grad()
    def step(self, idx, state):
        """The logits of one more token of every sequence, idx [batch]; the state is updated in place."""
        x = self.emb(idx)
        for b, (last, s) in zip(self.blocks, state):
            n = b.norm1(x)
            x = x + b.time.step(n, last, s)
            last.copy_(n)
            x = b.value(b.key(b.norm2(x)), residual=x)
        return self.head(self.norm(x))


def train(model, steps, lens=(77, 1, 130, 48), seed=0, report=print):
    """The losses of `steps` steps on one batch of packed sequences."""
    g = torch.Generator().manual_seed(seed)
    idx = torch.randint(0, model.emb.num_embeddings, (1, sum(lens)), generator=g).cuda()
    cu = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32).cuda()
    target = idx.roll(-1, 1)[0]
    target[cu[1:].long() - 1] = -100  # a sequence's last token has no next one
    params = [p for p in model.parameters() if p.requires_grad]
    opt = torch.optim.SGD(params, lr=0.2)
    losses = []
    for step in range(steps):
        logits, _ = model(idx, cu=cu)
        loss = F.cross_entropy(logits[0].float(), target, ignore_index=-100)
        opt.zero_grad(set_to_none=True)
        loss.backward()
        norm = rwkvq.clip_grad_norm_(params, 1.0)
        opt.step()
        losses.append(loss.item())
        report(f"step {step}: loss {losses[-1]:.4f}, gradient norm {norm.item():.3f}")
    return losses


@torch.no_grad()
def generate(model, prompt, tokens, temperature=1.0, top_k=50, top_p=0.95, seed=0):
    """(tokens, their log-probabilities) [batch, tokens] behind a prompt [batch, time]; the decode step runs as a graph."""
    numbers = torch.rand(tokens, prompt.shape[0], generator=torch.Generator().manual_seed(seed)).cuda()
    logits, state = model(prompt)
    token, logprob = rwkvq.sample(logits[:, -1], numbers[0], temperature, top_k, top_p)
    out, scores = [token], [logprob]
    state = [(last.clone(), s) for last, s in state]
    at, u = token.clone(), numbers[0].clone()

    def step():
        return rwkvq.sample(model.step(at, state), u, temperature, top_k, top_p)

    graph = None
    for i in range(1, tokens):
        at.copy_(token)
        u.copy_(numbers[i])
        if i == 1:  # eagerly, on another stream: what capturing wants to have run before
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                token, logprob = step()
            torch.cuda.current_stream().wait_stream(side)
        else:
            if graph is None:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    token, logprob = step()
            graph.replay()
        out.append(token.clone())
        scores.append(logprob.clone())
    return torch.stack(out, 1), torch.stack(scores, 1)


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--tokens", type=int, default=32)
    ap.add_argument("--packed", action="store_true")
    args = ap.parse_args()
    torch.manual_seed(0)
    model = Model(packed=args.packed)
    train(model, args.steps)
    prompt = torch.randint(0, 512, (2, 20)).cuda()
    for row in generate(model, prompt, args.tokens)[0].tolist():
        print(*row)
