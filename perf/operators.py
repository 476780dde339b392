"""The operators of a training step around the packed products, and the work
whose time is measured: the dense products with bias, activation and residual,
the trainable embedding table, and the clip of the global gradient norm.

  linear     y = act(x W^T + b) + r.  x [m, k], W [n, k] and b [n] share a type, r
             and y [m, n] have that type or float32 (a float32 residual stream).
             `train` adds the backward pass: gradients of x, W, b and r.
  embedding  out[i] = scale * W[idx[i]] for the tokens idx[n] and a table [vocab,
             d]; `train` adds the gradient of the table, dense, 0 where no token
             points.  Tokens fall as in text: log-uniform over the vocabulary, a
             few of them in a large share of the places.
  clip       the 2-norm over all gradients of a model, and every gradient times
             min(max_norm / (norm + 1e-6), 1).  `what` says which tensors: the
             adapters of `layers` blocks (A [rank, in] and B [out, rank] of the six
             projections), their dense weights, or those and the embedding
             table.

A block of width d has the projections r, k, v, o [d, d], the FFN key [4d, d] and
the FFN value [d, 4d]; the widths are 768 (0.1B), 2048 (1.5B), 2560 (2.9B) and
4096 (7.2B) with a vocabulary of 65536.  Weights are N(0, 0.02) (the table N(0,
1)), activations N(0, 1), incoming gradients N(0, 1e-2).

`own` False computes the plain form in elementary torch operations, in float32,
rounded once; True calls the package.
"""
import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "fp32": 4}
ACTIVATIONS = ("none", "relu", "relu2", "silu", "gelu", "sigmoid", "tanh")


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # one decode step's low-rank decay branch of the 0.1B model: tanh(x A), launch-bound
        {"name": "linear_0.1b_branch_m1", "op": "linear", "m": 1, "k": 768, "n": 64, "act": "tanh",
         "bias": True, "residual": "", "dtype": "bf16", "train": False},
        # the dense FFN key of a 1.5B decode step over 5 sequences, relu^2
        {"name": "linear_1.5b_key_m5", "op": "linear", "m": 5, "k": 2048, "n": 8192, "act": "relu2",
         "bias": False, "residual": "", "dtype": "bf16", "train": False},
        # the output projection of a 2.9B prompt of odd length, added to a float32 residual stream
        {"name": "linear_2.9b_out_m333", "op": "linear", "m": 333, "k": 2560, "n": 2560,
         "act": "none", "bias": True, "residual": "fp32", "dtype": "bf16", "train": False},
        # a training step through the dense FFN key of the 1.5B model, 8 x 512 tokens
        {"name": "linear_1.5b_key_train", "op": "linear", "m": 4096, "k": 2048, "n": 8192,
         "act": "relu2", "bias": False, "residual": "", "dtype": "bf16", "train": True},
        # a training step at sizes no tile divides, half precision, everything in the epilogue
        {"name": "linear_odd_train", "op": "linear", "m": 1003, "k": 771, "n": 517, "act": "gelu",
         "bias": True, "residual": "f16", "dtype": "f16", "train": True},
        # a training step of a small model kept in float32
        {"name": "linear_fp32_train", "op": "linear", "m": 512, "k": 768, "n": 768, "act": "silu",
         "bias": True, "residual": "", "dtype": "fp32", "train": True},
        # the lookup of one decode token
        {"name": "embedding_0.1b_m1", "op": "embedding", "m": 1, "vocab": 65536, "d": 768,
         "scale": 1.0, "dtype": "bf16", "train": False},
        # lookup and gradient of a 1.5B training step, 8 x 512 tokens
        {"name": "embedding_1.5b_train", "op": "embedding", "m": 4096, "vocab": 65536, "d": 2048,
         "scale": 45.25, "dtype": "bf16", "train": True},
        # lookup and gradient at odd sizes, many repeats of few tokens, float32
        {"name": "embedding_odd_train", "op": "embedding", "m": 30011, "vocab": 5003, "d": 517,
         "scale": 0.5, "dtype": "fp32", "train": True},
        # the adapters of the 1.5B model at rank 16: 288 small tensors
        {"name": "clip_1.5b_adapters", "op": "clip", "what": "adapters", "layers": 24, "d": 2048,
         "rank": 16, "vocab": 65536, "dtype": "bf16", "max_norm": 1.0, "std": 1e-3},
        # every dense weight of a 0.1B model and its table, float32 gradients
        {"name": "clip_0.1b_model", "op": "clip", "what": "model", "layers": 12, "d": 768,
         "rank": 0, "vocab": 65536, "dtype": "fp32", "max_norm": 1.0, "std": 1e-3},
        # the dense weights of 12 blocks of the 1.5B model
        {"name": "clip_1.5b_dense", "op": "clip", "what": "dense", "layers": 12, "d": 2048,
         "rank": 0, "vocab": 65536, "dtype": "bf16", "max_norm": 1.0, "std": 1e-3},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("linear", "linear", "embedding", "clip"))
    if op == "linear":
        train = rng.random() < 0.5
        dtype = rng.choice(("bf16", "bf16", "bf16", "f16", "fp32"))
        while True:
            m = _log_int(rng, 1, 4096)
            k, n = _log_int(rng, 64, 8192), _log_int(rng, 64, 8192)
            if rng.random() < 0.6:   # most weights have whole tiles, some have not
                k, n = max(64, k // 64 * 64), max(64, n // 64 * 64)
            # no more than the largest listed one; float32 runs at a sixteenth of the rate
            if 3072 not in (m, k, n) and m * k * n <= (2 ** 36 if dtype != "fp32" else 2 ** 32):
                break
        return {"op": "linear", "m": m, "k": k, "n": n, "act": rng.choice(ACTIVATIONS),
                "bias": rng.random() < 0.5, "residual": rng.choice(("", "", dtype, "fp32")),
                "dtype": dtype, "train": train}
    if op == "embedding":
        while True:
            m, d = _log_int(rng, 1, 32768), _log_int(rng, 64, 4096)
            vocab = _log_int(rng, 512, 65536)
            if rng.random() < 0.6:
                d = max(64, d // 64 * 64)
            if 3072 not in (m, d, vocab) and m * d <= 2 ** 26:
                break
        return {"op": "embedding", "m": m, "vocab": vocab, "d": d,
                "scale": rng.choice((1.0, 0.5, 45.25)), "dtype": rng.choice(("bf16", "f16", "fp32")),
                "train": rng.random() < 0.7}
    while True:
        what = rng.choice(("adapters", "dense", "model"))
        case = {"op": "clip", "what": what, "layers": rng.randint(1, 24 if what == "adapters" else 6),
                "d": 64 * rng.randint(4, 32),
                "rank": rng.choice((4, 8, 15, 16, 32, 64)) if what == "adapters" else 0,
                "vocab": _log_int(rng, 512, 65536), "dtype": rng.choice(("bf16", "f16", "fp32")),
                "max_norm": rng.choice((0.1, 1.0, 1000.0)), "std": 1e-3}
        if work(case)["bytes"] <= 2 ** 31 and 3072 not in (4 * case["d"], case["vocab"]):
            return case


def _clip_shapes(case):
    d, r = case["d"], case["rank"]
    sides = [(d, d)] * 4 + [(4 * d, d), (d, 4 * d)]
    if case["what"] == "adapters":
        block = [s for n_out, n_in in sides for s in ((r, n_in), (n_out, r))]
    else:
        block = sides
    shapes = block * case["layers"]
    return shapes + [(case["vocab"], d)] if case["what"] == "model" else shapes


def work(case):
    if case["op"] == "linear":
        m, k, n, e = case["m"], case["k"], case["n"], BYTES[case["dtype"]]
        ey = BYTES[case["residual"]] if case["residual"] else e
        b = (m * k + n * k + (n if case["bias"] else 0)) * e + m * n * ey
        b += m * n * ey if case["residual"] else 0
        if case["train"]:
            b += (m * k + n * k + (n if case["bias"] else 0)) * e + m * n * ey
        return {"bytes": b, "flops": (6 if case["train"] else 2) * m * k * n}
    if case["op"] == "embedding":
        m, d, v, e = case["m"], case["d"], case["vocab"], BYTES[case["dtype"]]
        b = 8 * m + 2 * m * d * e
        if case["train"]:
            b += m * d * e + v * d * e
        return {"bytes": b, "flops": m * d * (2 if case["train"] else 1)}
    total = sum(a * b for a, b in _clip_shapes(case))
    return {"bytes": 2 * total * BYTES[case["dtype"]], "flops": 3 * total}


# ----------------------------------------------------------------- the inputs

def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(shape, std, dtype):
        return (torch.randn(shape, generator=g, device=DEVICE) * std).to(dtype)

    dt = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        rdt = DTYPES[case["residual"]] if case["residual"] else dt
        s["x"], s["w"] = normal((m, k), 1.0, dt), normal((n, k), 0.02, dt)
        s["b"] = normal((n,), 0.5, dt) if case["bias"] else None
        s["r"] = normal((m, n), 1.0, rdt) if case["residual"] else None
        s["dy"] = normal((m, n), 1e-2, rdt) if case["train"] else None
        for t in (s["x"], s["w"], s["b"], s["r"]):
            if t is not None:
                t.requires_grad_(case["train"])
    elif case["op"] == "embedding":
        u = torch.rand(case["m"], generator=g, device=DEVICE)
        s["idx"] = (torch.exp(u * math.log(case["vocab"])) - 1).long().clamp_(0, case["vocab"] - 1)
        s["w"] = normal((case["vocab"], case["d"]), 1.0, dt).requires_grad_(case["train"])
        s["dy"] = normal((case["m"], case["d"]), 1e-2, dt) if case["train"] else None
    else:
        shapes = _clip_shapes(case)
        s["grads"] = [normal(sh, case["std"], dt) for sh in shapes]
        # the program's buffer for the clipped gradients, one view a tensor
        s["flat"] = torch.empty(sum(a * b for a, b in shapes), dtype=dt, device=DEVICE)
        s["out"] = [p.view(sh) for p, sh in
                    zip(s["flat"].split([a * b for a, b in shapes]), shapes)]
    return s


# ---------------------------------------------------------------- the passes

def run(state):
    return _run_own(state) if own else _run_plain(state)


_rq = None


def _package():
    global _rq
    if _rq is None:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                            "rwkv-metal_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import rwkvq
        _rq = rwkvq
    return _rq


def _run_own(s):
    rq, case = _package(), s["case"]
    if case["op"] == "linear":
        y = rq.linear_act(s["x"], s["w"], s["b"], None if case["act"] == "none" else case["act"],
                          s["r"])
        out = {"y": y}
        if case["train"]:
            wanted = [n for n in ("x", "w", "b", "r") if s[n] is not None]
            for name, t in zip(wanted, torch.autograd.grad(y, [s[n] for n in wanted], s["dy"])):
                out["d" + name] = t
        return out
    if case["op"] == "embedding":
        y = rq.embedding(s["idx"], s["w"], case["scale"])
        out = {"y": y}
        if case["train"]:
            out["dw"], = torch.autograd.grad(y, [s["w"]], s["dy"])
        return out
    _, norm = rq.clip_grad_norm(s["grads"], case["max_norm"], out=s["out"])
    return {"norm": norm, "clipped": s["flat"]}


def _value_and_slope(act, v, slope):
    """act(v), and act'(v) where `slope` is wanted."""
    if act == "none":
        return v, torch.ones_like(v) if slope else None
    if act == "relu":
        return v.clamp(min=0), (v > 0).to(v.dtype) if slope else None
    if act == "relu2":
        c = v.clamp(min=0)
        return c * c, 2 * c if slope else None
    if act == "tanh":
        t = torch.tanh(v)
        return t, 1 - t * t if slope else None
    if act == "gelu":
        c = 0.5 * (1 + torch.erf(v * math.sqrt(0.5)))
        return v * c, c + v * torch.exp(-0.5 * v * v) * (1 / math.sqrt(2 * math.pi)) if slope else None
    sg = 1 / (1 + torch.exp(-v))
    if act == "sigmoid":
        return sg, sg * (1 - sg) if slope else None
    return v * sg, sg * (1 + v * (1 - sg)) if slope else None


@torch.no_grad()
def _run_plain(s):
    case, dt = s["case"], DTYPES[s["case"]["dtype"]]
    if case["op"] == "linear":
        x, w = s["x"].float(), s["w"].float()
        v = x @ w.t()
        if s["b"] is not None:
            v = v + s["b"].float()
        a, slope = _value_and_slope(case["act"], v, case["train"])
        ydt = dt if s["r"] is None else s["r"].dtype
        out = {"y": (a if s["r"] is None else a + s["r"].float()).to(ydt)}
        if case["train"]:
            gr = s["dy"].float() * slope
            out["dx"], out["dw"] = (gr @ w).to(dt), (gr.t() @ x).to(dt)
            if s["b"] is not None:
                out["db"] = gr.sum(0).to(dt)
            if s["r"] is not None:
                out["dr"] = s["dy"]
        return out
    if case["op"] == "embedding":
        out = {"y": (s["w"][s["idx"]].float() * case["scale"]).to(dt)}
        if case["train"]:
            dw = torch.zeros(s["w"].shape, dtype=torch.float32, device=DEVICE)
            dw.index_add_(0, s["idx"], s["dy"].float())
            out["dw"] = (dw * case["scale"]).to(dt)
        return out
    norm = torch.stack([t.float().square().sum() for t in s["grads"]]).sum().sqrt()
    c = (case["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    for t, o in zip(s["grads"], s["out"]):
        o.copy_(t.float() * c)
    return {"norm": norm, "clipped": s["flat"]}


# ------------------------------------------------------- the definition, 64 bits

@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embedding":
        out = {"y": torch.index_select(s["w"].double(), 0, s["idx"]).mul_(case["scale"])}
        if case["train"]:
            # sums of the rows of equal tokens, in order: sorted, differences of running sums
            # would cancel, so each distinct token's rows are added up by position in its list
            dw = torch.zeros(s["w"].shape, dtype=torch.float64, device=DEVICE)
            token, order = torch.sort(s["idx"], stable=True)
            first = torch.searchsorted(token, token)
            place = torch.arange(token.numel(), device=DEVICE) - first
            # places past the first few repeat for few tokens only
            short = place < 16
            for p in range(16):
                at = place == p
                dw[token[at]] += s["dy"][order[at]].double()
            rest = ~short
            for t in torch.unique(token[rest]).tolist():
                dw[t] += s["dy"][order[rest & (token == t)]].double().sum(0)
            out["dw"] = dw.mul_(case["scale"])
        return out
    if case["op"] == "clip":
        norm = math.sqrt(math.fsum(float(torch.dot(t.double().view(-1), t.double().view(-1)))
                                   for t in s["grads"]))
        c = min(case["max_norm"] / (norm + 1e-6), 1.0)
        flat = torch.empty(s["flat"].numel(), dtype=torch.float64, device=DEVICE)
        at = 0
        for t in s["grads"]:
            flat[at:at + t.numel()] = t.reshape(-1)
            at += t.numel()
        return {"norm": torch.tensor(norm, dtype=torch.float64), "clipped": flat.mul_(c)}
    x, w = s["x"].double(), s["w"].double()
    v = torch.nn.functional.linear(x, w, None if s["b"] is None else s["b"].double())
    act, pos = case["act"], v > 0
    zero = torch.zeros((), dtype=torch.float64, device=DEVICE)
    if act == "relu":
        a, slope = torch.where(pos, v, zero), pos.double()
    elif act == "relu2":
        a, slope = torch.where(pos, v ** 2, zero), torch.where(pos, 2 * v, zero)
    elif act == "tanh":
        a, slope = torch.tanh(v), torch.cosh(v).pow(-2)
    elif act == "sigmoid":
        a = torch.sigmoid(v)
        slope = a * torch.sigmoid(-v)
    elif act == "silu":
        p = torch.sigmoid(v)
        a, slope = v * p, p + v * p * torch.sigmoid(-v)
    elif act == "gelu":
        p = torch.special.ndtr(v)
        a, slope = v * p, p + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    else:
        a, slope = v, torch.ones_like(v)
    out = {"y": a if s["r"] is None else a + s["r"].double()}
    if case["train"]:
        gr = s["dy"].double() * slope
        out["dx"] = torch.matmul(gr, w)
        out["dw"] = torch.matmul(gr.t().contiguous(), x)
        if s["b"] is not None:
            out["db"] = gr.sum(dim=0)
        if s["r"] is not None:
            out["dr"] = s["dy"].double()
    return out
