"""What an RWKV-7 block and its token choice run between the packed products: the
recurrence of the time mixing and the sampler behind the head, and the work whose
time is measured.

  scan    For every head of a sequence, with the state S [64 values, 64 keys] in float32,
              d_t = exp(-exp(w_t))
              S_t = S_{t-1} diag(d_t) + (S_{t-1} a_t) b_t^T + v_t k_t^T
              y_t = S_t r_t
          for r, w, k, v, a, b [batch, time, heads, 64].  It gives y and the last state;
          `state` False starts from 0.  `train` adds the backward pass: the gradients of
          all six and of the first state, from those of y and of the last state.
          `lens` packs sequences of these lengths into a batch of one, each with a state
          of its own; rows behind the last sequence (`rest` of them) belong to none and
          give 0.
  step    One token of every sequence, [batch, heads, 64]: y and the new state.
  sample  One token for each row of logits from a given uniform number u, and the log of
          its probability.  In this order: e_i = exp((l_i - max l) / temperature); the
          top_k largest stay (0: all); of these, from the largest, those before whom less
          than top_p of their sum lies; of these, those with e_i >= min_p.  Equal logits
          rank by index.  The token is the first by index at which the running sum of what
          stays exceeds u times the whole.  `rows` gives each row parameters of its own.

A head has 64 channels; 12, 32, 40 and 64 heads are widths of 768 (0.1B), 2048 (1.5B),
2560 (2.9B) and 4096 (7.2B); the vocabulary is 65536.  r, k and v are N(0, 1); a is the
negative of a unit vector and b the same vector times a gate in (0, 1); w = -softplus(x)
- 0.5, so that decays lie between 0.545 and 1: as the time mixing makes them.  Logits are
N(0, 2.5^2), some of them -inf as a grammar masks them.

`own` False computes the plain form in elementary torch operations, in float32 (the
sampler, whose comparisons decide, in float64), rounded once; True calls the package.
"""
import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "fp32": 4}
D = 64
NAMES = "rwkvab"


# ------------------------------------------------------------------ the cases

def _scan(**more):
    return {"op": "scan", "b": 1, "t": 0, "h": 32, "lens": "", "rest": 0, "state": False,
            "dtype": "bf16", "out": "bf16", "train": False, **more}


def _sample(**more):
    return {"op": "sample", "m": 1, "vocab": 65536, "dtype": "bf16", "temperature": 1.0, "top_k": 0,
            "top_p": 1.0, "min_p": 0.0, "masked": 0.0, "rows": False, **more}


def listed():
    return [
        # one token of one sequence through a 0.1B layer: launch-bound
        {"name": "step_0.1b_b1", "op": "step", "b": 1, "h": 12, "dtype": "bf16", "out": "bf16"},
        # one token of 128 sequences served together by the 1.5B model
        {"name": "step_1.5b_b128", "op": "step", "b": 128, "h": 32, "dtype": "bf16", "out": "bf16"},
        # a prompt of odd length continued from a state, 1.5B
        _scan(name="scan_1.5b_prompt", t=2047, h=32, state=True),
        # prompts of many lengths packed together, a single token and an empty one among them, 2.9B
        _scan(name="scan_2.9b_ragged", h=40, lens="511,1,77,0,1300,16,15,17,203,64,900,31", rest=9,
              state=True, dtype="f16", out="fp32"),
        # a training step of the 1.5B layer, 8 x 512 tokens
        _scan(name="scan_1.5b_train", b=8, t=512, h=32, train=True),
        # documents packed into one row of a training step, float32, odd sizes, through the states
        _scan(name="scan_0.1b_packed_train", h=12, lens="333,7,500,101,1,58", rest=3, state=True,
              dtype="fp32", out="fp32", train=True),
        # a long document in one piece, 0.1B: few heads, many tokens
        _scan(name="scan_0.1b_long_train", b=1, t=8192, h=12, train=True),
        # the token choice of one sequence
        _sample(name="sample_m1", temperature=0.8, top_p=0.9),
        # 128 sequences with everything that a request may set, float32 logits
        _sample(name="sample_m128", m=128, dtype="fp32", temperature=0.7, top_k=50, top_p=0.95,
                min_p=0.02),
        # requests with parameters of their own over a vocabulary of odd size, grammars mask half of it
        _sample(name="sample_odd_rows", m=37, vocab=50021, dtype="f16", masked=0.5, rows=True),
        # every token may come: 512 rollouts of a policy at temperature 1
        _sample(name="sample_m512_full", m=512),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("step", "scan", "scan", "scan", "sample", "sample"))
    dtype = rng.choice(("bf16", "bf16", "f16", "fp32"))
    out = rng.choice((dtype, "fp32"))
    if op == "step":
        return {"op": "step", "b": _log_int(rng, 1, 128), "h": rng.choice((1, 12, 13, 32)), "dtype": dtype,
                "out": out}
    if op == "sample":
        return {"op": "sample", "m": _log_int(rng, 1, 256), "vocab": _log_int(rng, 500, 131072),
                "dtype": dtype, "temperature": rng.choice((0.0, 0.5, 1.0, 1.3)),
                "top_k": rng.choice((0, 0, 1, _log_int(rng, 2, 2000))),
                "top_p": rng.choice((1.0, 0.5, 0.9, 0.97)), "min_p": rng.choice((0.0, 0.0, 0.05)),
                "masked": rng.choice((0.0, 0.2, 0.999)), "rows": rng.random() < 0.3}
    case = _scan(h=rng.choice((1, 5, 12, 32, 40)), dtype=dtype, out=out, state=rng.random() < 0.5,
                 train=rng.random() < 0.5)
    tokens = min(8192, 2 ** 17 // case["h"])   # no more than the largest listed one
    if rng.random() < 0.35:
        case["rest"] = rng.choice((0, 0, 5))
        lens, left = [], tokens - case["rest"]
        for _ in range(rng.randint(1, 24)):
            lens.append(min(left, rng.choice((0, 1, _log_int(rng, 2, 2048)))))
            left -= lens[-1]
        case["lens"] = ",".join(str(n) for n in lens)
        if sum(lens) == 0:
            case["rest"] = 5
    else:
        case["b"] = _log_int(rng, 1, 16)
        case["t"] = _log_int(rng, 1, tokens // case["b"])
    return case


def _lens(case):
    return [int(n) for n in case["lens"].split(",")] if case["lens"] else []


def _tokens(case):
    return sum(_lens(case)) + case["rest"] if case["lens"] else case["b"] * case["t"]


def _states(case):
    return len(_lens(case)) if case["op"] == "scan" and case["lens"] else case["b"]


def work(case):
    if case["op"] == "sample":
        # the logits once; a comparison, an exponential's dozen and two sums for each
        n = case["m"] * case["vocab"]
        return {"bytes": n * BYTES[case["dtype"]] + 16 * case["m"], "flops": 16 * n}
    e, eo, h = BYTES[case["dtype"]], BYTES[case["out"]], case["h"]
    tokens = case["b"] if case["op"] == "step" else _tokens(case)
    state = 4 * D * D * h * _states(case)
    # S a, the three terms of the new state, S r: 9 operations for each of a state's 64 x 64 values
    b, f = tokens * h * D * (6 * e + eo), 9 * D * D * tokens * h
    if case["op"] == "step":
        return {"bytes": b + 2 * state, "flops": f}
    b += state * (2 if case["state"] else 1)
    if case["train"]:
        # dy and the six inputs again, six gradients; the last state's gradient and the first's
        b += tokens * h * D * (12 * e + eo) + state * (2 if case["state"] else 0)
        f *= 3
    return {"bytes": b, "flops": f}


# ----------------------------------------------------------------- the inputs

def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEVICE)

    def uniform(*shape):
        return torch.rand(shape, generator=g, device=DEVICE)

    dt, s = DTYPES[case["dtype"]], {"case": case}
    if case["op"] == "sample":
        m, n = case["m"], case["vocab"]
        logits = normal(m, n) * 2.5
        if case["masked"]:
            gone = uniform(m, n) < case["masked"]
            gone[:, n // 2] = False   # something is left of every row
            logits.masked_fill_(gone, -math.inf)
        s["logits"], s["u"] = logits.to(dt), uniform(m)
        for name in ("temperature", "top_k", "top_p", "min_p"):
            s[name] = case[name]
        if case["rows"]:
            pick = lambda *of: torch.tensor(of, device=DEVICE)[(uniform(m) * len(of)).long()]  # noqa: E731
            s["temperature"], s["top_k"] = pick(0.0, 0.5, 0.7, 1.0, 1.3), pick(0, 0, 1, 20, 100, 1000)
            s["top_p"], s["min_p"] = pick(1.0, 0.5, 0.9, 0.95), pick(0.0, 0.0, 0.02, 0.1)
        return s
    h = case["h"]
    if case["op"] == "step":
        lead = (case["b"], h)
    else:
        lead = (1, _tokens(case), h) if case["lens"] else (case["b"], case["t"], h)
    kk = torch.nn.functional.normalize(normal(*lead, D), dim=-1)
    s["r"], s["k"], s["v"] = (normal(*lead, D).to(dt) for _ in range(3))
    s["w"] = (-torch.nn.functional.softplus(2 * normal(*lead, D)) - 0.5).to(dt)
    s["a"], s["b"] = (-kk).to(dt), (kk * torch.sigmoid(normal(*lead, D))).to(dt)
    first = case["op"] == "step" or case["state"]
    s["state"] = normal(_states(case), h, D, D) if first else None
    if case["op"] == "step":
        s["next"] = torch.empty_like(s["state"])   # the program's other buffer of states
        return s
    s["cu"] = None
    if case["lens"]:
        ends = [0]
        for n in _lens(case):
            ends.append(ends[-1] + n)
        s["cu"], s["longest"] = torch.tensor(ends, dtype=torch.int32, device=DEVICE), max(_lens(case))
    if case["train"]:
        s["dy"] = normal(*lead, D).to(DTYPES[case["out"]])
        s["dstate"] = normal(*s["state"].shape) if first else None
        for name in _leaves(s):
            s[name].requires_grad_()
    return s


def _leaves(s):
    return list(NAMES) + (["state"] if s["state"] is not None else [])


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
    if case["op"] == "sample":
        token, logprob = rq.sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"],
                                   s["min_p"])
        return {"token": token, "logprob": logprob}
    six, out = [s[n] for n in NAMES], DTYPES[case["out"]]
    if case["op"] == "step":
        y, state = rq.wkv7_step(*six, s["state"], out=s["next"], out_dtype=out)
        return {"y": y, "state": state}
    y, state = rq.wkv7(*six, s["state"], cu_seqlens=s["cu"], out_dtype=out)
    return _with_gradients(s, y, state, [s[n] for n in _leaves(s)] if case["train"] else [])


def _with_gradients(s, y, state, leaves):
    """The outputs, and the gradients of `leaves` (in the order of _leaves)."""
    out = {"y": y.detach(), "state": state.detach()}
    if leaves:
        of, by = [y], [s["dy"].to(y.dtype)]
        if s["dstate"] is not None:
            of, by = [y, state], by + [s["dstate"].to(state.dtype)]
        for name, g in zip(_leaves(s), torch.autograd.grad(of, leaves, by)):
            out["d" + name] = g
    return out


def _run_plain(s):
    case = s["case"]
    if case["op"] == "sample":
        return _sample_plain(s)
    out = DTYPES[case["out"]]
    if case["op"] == "step":
        r, w, k, v, a, b = (s[n].float()[..., None, :] for n in NAMES)   # rows [.., 1, 64]
        state = s["state"]
        sa = (state * a).sum(-1, keepdim=True)
        s["next"].copy_(state * torch.exp(-torch.exp(w)) + sa * b + v.transpose(-1, -2) * k)
        return {"y": (s["next"] * r).sum(-1).to(out), "state": s["next"]}
    leaves = [s[n].detach().float().requires_grad_(case["train"]) for n in _leaves(s)]
    state = leaves[6] if s["state"] is not None else torch.zeros(_states(case), case["h"], D, D, device=DEVICE)
    y, state = (_packed if case["lens"] else _chunks)(leaves[:6], state, s)
    got = _with_gradients(s, y, state, leaves if case["train"] else [])
    return {n: t.to(out if n == "y" else torch.float32 if "state" in n else s["r"].dtype)
            for n, t in got.items()}


def _packed(six, state, s):
    """The packed sequences as a padded batch, whose padding leaves the states as they are."""
    n, t, cu = state.shape[0], six[0].shape[1], s["cu"].long()
    if s["longest"] == 0:
        return six[0] * 0, state * 1
    at = cu[:-1, None] + torch.arange(s["longest"], device=DEVICE)
    there = (at < cu[1:, None])[..., None, None]
    zero = torch.zeros((), device=DEVICE)
    at = at.clamp(max=t - 1)
    batch = [torch.where(there, x[0][at], zero - math.inf if name == "w" else zero)
             for name, x in zip(NAMES, six)]
    y, state = _chunks(batch, state, s)
    place = torch.arange(t, device=DEVICE)
    seq = torch.searchsorted(cu, place, right=True).sub_(1)
    y = y[seq.clamp(max=n - 1), (place - cu[seq]).clamp(0, s["longest"] - 1)]
    return torch.where((seq < n)[:, None, None], y, zero)[None], state


def _chunks(six, state, s, size=32):
    """The recurrence over chunks of `size` tokens: within a chunk, with the running sums L of
    the log decays, all tokens at once; from chunk to chunk the state."""
    n, t, h, _ = six[0].shape
    m = -(-t // size)
    pad = lambda x, v: torch.nn.functional.pad(x, (0, 0, 0, 0, 0, m * size - t), value=v)  # noqa: E731
    r, w, k, v, a, b = (pad(x, -math.inf if name == "w" else 0.0).view(n, m, size, h, D).permute(0, 3, 1, 2, 4)
                        for name, x in zip(NAMES, six))
    g = -torch.exp(w)
    run_ = g.cumsum(-2)
    last = run_[..., -1:, :]
    ra, aa = r * torch.exp(run_), a * torch.exp(run_ - g)
    bi, ki = (b * torch.exp(-run_)).transpose(-1, -2), (k * torch.exp(-run_)).transpose(-1, -2)
    bo, ko = b * torch.exp(last - run_), k * torch.exp(last - run_)
    rb, rk = torch.tril(ra @ bi), torch.tril(ra @ ki)
    p, ak = torch.tril(aa @ bi, -1), torch.tril(aa @ ki, -1)
    inv = torch.eye(size, device=DEVICE) + p     # (I - p)^-1, p^size = 0
    for _ in range(int(math.log2(size)) - 1):
        p = p @ p
        inv = inv + inv @ p
    au, vu, kv = inv @ aa, inv @ (ak @ v), v.transpose(-1, -2) @ ko
    decay = torch.exp(last)
    before, sas = [], []
    for j in range(m):
        sa = au[:, :, j] @ state.transpose(-1, -2) + vu[:, :, j]
        before.append(state)
        sas.append(sa)
        state = state * decay[:, :, j] + sa.transpose(-1, -2) @ bo[:, :, j] + kv[:, :, j]
    y = ra @ torch.stack(before, 2).transpose(-1, -2) + rb @ torch.stack(sas, 2) + rk @ v
    return y.permute(0, 2, 3, 1, 4).reshape(n, m * size, h, D)[:, :t], state


def _parameters(s):
    """The parameters as columns of float64 (top_k whole), one row each or one for all."""
    got = []
    for name in ("temperature", "top_k", "top_p", "min_p"):
        x = s[name] if isinstance(s[name], torch.Tensor) else torch.tensor([s[name]], device=DEVICE)
        # the parameters are numbers of 32 bits
        got.append(x.long()[:, None] if name == "top_k" else x.float().double()[:, None])
    return got


@torch.no_grad()
def _sample_plain(s):
    temperature, top_k, top_p, min_p = _parameters(s)
    n = s["logits"].shape[1]
    logits, order = torch.sort(s["logits"].double(), dim=-1, descending=True, stable=True)
    e = torch.exp((logits - logits[:, :1]) / torch.where(temperature > 0, temperature, 1.0))
    rank = torch.arange(n, device=DEVICE)
    kept = (logits > -math.inf) & (rank < torch.where(top_k > 0, top_k, n)) & ((temperature > 0) | (rank < 1))
    e = torch.where(kept, e, 0.0)
    total = e.sum(-1, keepdim=True)
    kept &= (e.cumsum(-1) - e < top_p * total) | (top_p >= 1)
    e = torch.where(kept & (e >= min_p), e, 0.0)
    e = torch.zeros_like(e).scatter_(-1, order, e)
    e_sum = e.cumsum(-1)
    target = s["u"].double()[:, None] * e_sum[:, -1:]
    token = (e_sum > target).to(torch.int8).argmax(-1)
    chosen = e.gather(-1, token[:, None])
    return {"token": token, "logprob": torch.log(chosen / e_sum[:, -1:])[:, 0].float()}


# ------------------------------------------------------- the definition, 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _sample_exact(s)
    six = [s[n].detach().double().requires_grad_(case.get("train", False)) for n in NAMES]
    state = None
    if s["state"] is not None:
        state = s["state"].detach().double().requires_grad_(case.get("train", False))
    start = state if state is not None else torch.zeros(_states(case), case["h"], D, D,
                                                        dtype=torch.float64, device=DEVICE)
    if case["op"] == "step":
        y, last = _by_token([x[:, None] for x in six], start)
        return {"y": y[:, 0], "state": last}
    if case["lens"]:
        ys, lasts, at = [], [], 0
        for i, n in enumerate(_lens(case)):
            y, last = _by_token([x[:, at:at + n] for x in six], start[i:i + 1])
            ys.append(y)
            lasts.append(last)
            at += n
        ys.append(0 * six[0][:, at:])
        y, last = torch.cat(ys, 1), torch.cat(lasts, 0)
    else:
        y, last = _by_token(six, start)
    return _with_gradients(s, y, last, (six + ([] if state is None else [state])) if case["train"] else [])


def _by_token(six, state):
    """The recurrence as it is written, one token after the other."""
    r, w, k, v, a, b = (x.unbind(1) for x in six)
    ys = []
    for t in range(len(r)):
        sa = torch.matmul(state, a[t].unsqueeze(-1))
        state = (state * torch.exp(-torch.exp(w[t])).unsqueeze(-2) + sa * b[t].unsqueeze(-2)
                 + v[t].unsqueeze(-1) * k[t].unsqueeze(-2))
        ys.append(torch.matmul(state, r[t].unsqueeze(-1)).squeeze(-1))
    return torch.stack(ys, 1) if ys else six[0] * 1, state


@torch.no_grad()
def _sample_exact(s):
    """Row by row with thresholds instead of ranks: the probability of the token that the
    running sum reaches."""
    m, out = s["logits"].shape[0], []
    params = [x.expand(m, 1)[:, 0].tolist() for x in _parameters(s)]
    for row, u, temperature, top_k, top_p, min_p in zip(s["logits"].double(), s["u"].double().tolist(), *params):
        index = torch.nonzero(row > -math.inf)[:, 0]
        index = index[torch.sort(-row[index], stable=True).indices]
        if temperature == 0:
            out.append(0.0)
            continue
        if top_k:
            index = index[:int(top_k)]
        p = torch.softmax(row[index] / temperature, 0)
        if top_p < 1:
            below = torch.cumsum(p, 0) < top_p
            index = index[:int(below.sum()) + 1]
        p = torch.softmax(row[index] / temperature, 0)
        index = index[p >= min_p * p[0]]
        index = torch.sort(index).values
        p = torch.softmax(row[index] / temperature, 0)
        at = int((torch.cumsum(p, 0) <= u).sum())
        out.append(float(torch.log(p[min(at, p.numel() - 1)])))
    return {"token": None, "logprob": torch.tensor(out, dtype=torch.float64)}
