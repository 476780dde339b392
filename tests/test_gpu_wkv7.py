"""The recurrence of RWKV-7's time mixing on the GPU against its definition in 64 bits
(bounds: tests/wkv_ref.py)."""
import math

import pytest
import torch

from wkv_ref import D, DT, NAMES, U, U32, bound, close, inputs, reference

pytestmark = pytest.mark.gpu

LEAVES = [*NAMES, "state"]


def run(rq, dev, six, state, dy=None, dstate=None, cu=None, out=None):
    six = [x.to(dev).requires_grad_(dy is not None) for x in six]
    first = None if state is None else state.to(dev).requires_grad_(dy is not None)
    y, last = rq.wkv7(*six, first, cu_seqlens=cu, out_dtype=out)
    got = {"y": y.detach(), "state": last.detach()}
    if dy is not None:
        leaves = six + ([] if first is None else [first])
        of, by = ([y], [dy.to(dev)]) if dstate is None else ([y, last], [dy.to(dev), dstate.to(dev)])
        for name, t in zip(LEAVES, torch.autograd.grad(of, leaves, by)):
            got["d" + name] = t
    return got


def check(rq, dev, seed, b, t, h, dt, out, has_state, train, lens=None, rest=0, w=None, change=None):
    g = torch.Generator().manual_seed(seed)
    if lens is not None:
        b, t = 1, sum(lens) + rest
    seqs = b if lens is None else len(lens)
    six = inputs(g, b, t, h, dtype=DT[dt], w=w)
    if change is not None:
        change(six, g)
    state = torch.randn(seqs, h, D, D, generator=g)
    dy = torch.randn(b, t, h, D, generator=g).to(DT[out]) if train else None
    dstate = torch.randn(seqs, h, D, D, generator=g) if train and has_state else None
    want = reference(six, state if has_state else 0 * state, dy, dstate, lens)
    cu = None
    if lens is not None:
        cu = torch.tensor([sum(lens[:i]) for i in range(seqs + 1)], dtype=torch.int32, device=dev)
    got = run(rq, dev, six, state if has_state else None, dy, dstate, cu, DT[out])
    assert got["y"].dtype == DT[out] and got["state"].dtype == torch.float32
    for name, x in got.items():
        assert x.dtype == (DT[out] if name == "y" else torch.float32 if "state" in name else DT[dt])
        close(x, want[name], name, t)
    if lens is not None and rest:
        assert all((got[n][:, sum(lens):] == 0).all() for n in got if "state" not in n)
    return got


# no token, one, chunks of 16 that are full, begun and just over; one head and several; more
# than 192 heads of sequences, where a block takes a whole head
SHAPES = [(1, 0, 2), (2, 1, 1), (1, 2, 3), (1, 15, 1), (2, 16, 2), (1, 17, 5), (3, 31, 1), (1, 32, 2), (1, 33, 1),
          (2, 100, 3), (1, 257, 2), (65, 21, 3), (0, 5, 2), (97, 1, 2)]


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("dt,out", [("bf16", "bf16"), ("bf16", "fp32"), ("f16", "f16"), ("f16", "fp32"),
                                    ("fp32", "fp32")])
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_sequences(rq, dev, i, dt, out, train):
    b, t, h = SHAPES[i]
    print(f"wkv7 b={b} t={t} h={h} {dt}->{out} train={train}", flush=True)
    check(rq, dev, i, b, t, h, dt, out, i % 2 == 0, train)


LENS = [[5], [16, 16], [1, 1, 1], [0, 3, 0, 40, 0], [17, 15, 1, 33], [100, 0, 7, 64, 2], [0], [0, 0]]


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("i", range(len(LENS)))
def test_packed_sequences(rq, dev, i, dt, train):
    rest = (0, 3, 21)[i % 3]
    print(f"wkv7 lens={LENS[i]} rest={rest} {dt} train={train}", flush=True)
    check(rq, dev, 50 + i, 1, 0, 1 + i % 3, dt, "fp32" if i % 2 else dt, i % 4 != 3, train, LENS[i], rest)


# few heads over many tokens: in segments, whole ones and one of a single token behind them, sequences of
# one segment and of several side by side
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("b,t,h", [(1, 385, 1), (1, 700, 2), (2, 513, 1), (1, 1024, 3)])
def test_segments(rq, dev, b, t, h, dt):
    assert rq._lib.lib().rq_wkv7_workspace_bytes(b, t, h, b, 0) > 0
    print(f"wkv7 segments b={b} t={t} h={h} {dt}", flush=True)
    check(rq, dev, 60 + t, b, t, h, dt, "fp32", t % 2 == 0, True)
    check(rq, dev, 61 + t, b, t, h, dt, dt, t % 2 == 1, False)


@pytest.mark.parametrize("i", range(4))
def test_packed_segments(rq, dev, i):
    lens = [[600, 3, 0, 401], [0, 0, 1, 800], [129, 128, 127, 385, 1, 0], [16, 900]][i]
    rest = (0, 5, 40, 1)[i]
    assert rq._lib.lib().rq_wkv7_workspace_bytes(1, sum(lens) + rest, 2, len(lens), 1) > 0
    check(rq, dev, 90 + i, 1, 0, 2, ("fp32", "bf16", "f16", "fp32")[i], "fp32", i != 3, True, lens, rest)


def test_segments_with_strong_decays_and_equal_directions(rq, dev):
    def change(six, g):
        w = six[1]
        w.copy_(torch.randn(w.shape, generator=g) * 3 - 1)
        w[:, 100:130, :, ::5] = math.inf
    check(rq, dev, 95, 1, 450, 1, "fp32", "fp32", True, True, change=change)

    def change(six, g):
        u = torch.nn.functional.normalize(torch.randn(D, generator=g), dim=-1)
        six[4].copy_(-u.expand_as(six[4]))
        six[5].copy_(u.expand_as(six[5]))
    check(rq, dev, 96, 1, 450, 1, "fp32", "fp32", True, True, change=change, w=-6.0)


def test_wild_boundaries_in_segments(rq, dev):
    """Nothing outside the tensors is touched."""
    g = torch.Generator().manual_seed(97)
    six = [x.to(dev).requires_grad_() for x in inputs(g, 1, 900, 2)]
    wild = torch.tensor([850, 3, 700, -1, 2 ** 31 - 1, 0, 899], dtype=torch.int32, device=dev)
    assert rq._lib.lib().rq_wkv7_workspace_bytes(1, 900, 2, 6, 1) > 0
    y, last = rq.wkv7(*six, cu_seqlens=wild)
    grads = torch.autograd.grad(y.sum() + last.sum(), six)
    torch.cuda.synchronize()
    assert y.shape == six[0].shape and len(grads) == 6


@pytest.mark.parametrize("lens", [None, [600, 3, 0, 401]])
def test_a_state_in_place_in_segments(rq, dev, lens):
    """The C entry point with one buffer for the state before and after: the last segment's block may
    end before the first one's begins."""
    g = torch.Generator().manual_seed(98)
    L, h, t = rq._lib.lib(), 3, 1004
    six = [x.to(dev) for x in inputs(g, 1, t, h)]
    seqs = 1 if lens is None else len(lens)
    cu = None if lens is None else torch.tensor([0, 600, 603, 603, 1004], dtype=torch.int32, device=dev)
    state = torch.randn(seqs, h, D, D, generator=g).to(dev)
    want_y, want_last = rq.wkv7(*six, state, cu_seqlens=cu)
    need = L.rq_wkv7_workspace_bytes(1, t, h, seqs, int(cu is not None))
    assert need > 0
    ws, y = torch.empty(need, dtype=torch.uint8, device=dev), torch.empty_like(six[0])
    rc = L.rq_wkv7(*[x.data_ptr() for x in six], rq._lib.DTYPE_CODE[torch.float32], 1, t, h,
                   0 if cu is None else cu.data_ptr(), seqs, state.data_ptr(), y.data_ptr(),
                   rq._lib.DTYPE_CODE[torch.float32], state.data_ptr(), 0, 0, ws.data_ptr(), need,
                   torch.cuda.current_stream(dev).cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    assert torch.equal(y, want_y) and torch.equal(state, want_last)


def test_many_packed_sequences(rq, dev):
    lens = [(7 * i) % 23 for i in range(200)]
    check(rq, dev, 77, 1, 0, 2, "fp32", "fp32", True, True, lens, 5)


@pytest.mark.parametrize("w", [-math.inf, -20.0, 0.0, 2.0, 3.0, 5.0, 20.0, 100.0, math.inf])
def test_decays_from_none_to_whole(rq, dev, w):
    """Above 2^-32 over a chunk, below it, and 0."""
    check(rq, dev, 101, 2, 37, 2, "fp32", "fp32", True, True, w=w)


def test_decays_of_every_strength_side_by_side(rq, dev):
    def change(six, g):
        w = six[1]
        w.copy_(torch.randn(w.shape, generator=g) * 3 - 1)   # exp(w) from 1e-5 to 1e4 in one chunk
        w[:, 3:9, :, ::5] = math.inf
        w[:, :, :, 1] = -math.inf
    check(rq, dev, 102, 1, 70, 3, "fp32", "fp32", True, True, change=change)
    check(rq, dev, 103, 1, 70, 3, "bf16", "bf16", True, True, change=change)


def test_equal_directions(rq, dev):
    """Every token takes its state's part along one direction away whole: the inverse is far from 1."""
    def change(six, g):
        u = torch.nn.functional.normalize(torch.randn(D, generator=g), dim=-1)
        six[4].copy_(-u.expand_as(six[4]))
        six[5].copy_(u.expand_as(six[5]))
    check(rq, dev, 104, 1, 50, 2, "fp32", "fp32", True, True, change=change, w=-6.0)


def test_gradients_against_differences(rq, dev):
    """Central differences of step h along random directions.  The second-order term is h^2 / 6 times
    a third derivative of the loss's size times small factors: below 1e-3 of the slope for h = 2^-7;
    the loss's own rounding (relative 2e-6 of the terms' norm, over 2 h) stays below 3e-4."""
    g = torch.Generator().manual_seed(7)
    six = inputs(g, 1, 45, 2)
    state = torch.randn(1, 2, D, D, generator=g)
    dy, dstate = torch.randn(1, 45, 2, D, generator=g), torch.randn(1, 2, D, D, generator=g)
    got = run(rq, dev, six, state, dy, dstate)
    h = 2.0 ** -7

    def loss(xs):
        o = run(rq, dev, xs[:6], xs[6])
        return ((o["y"].double().cpu() * dy.double()).sum() + (o["state"].double().cpu() * dstate.double()).sum()).item()

    size = math.sqrt((dy.double() ** 2).sum() + (dstate.double() ** 2).sum())
    for j, name in enumerate(LEAVES):
        xs = [*six, state]
        d = torch.randn(xs[j].shape, generator=g) * (0.1 if name in "ab" else 1.0)
        up, down = list(xs), list(xs)
        up[j], down[j] = xs[j] + h * d, xs[j] - h * d
        slope = (got["d" + name].double().cpu() * d.double()).sum().item()
        diff = (loss(up) - loss(down)) / (2 * h)
        scale = max(abs(slope), got["d" + name].double().norm().item() * d.double().norm().item() / math.sqrt(d.numel()))
        assert abs(diff - slope) <= 1e-3 * scale + 3e-4 * size, (name, diff, slope)


@pytest.mark.parametrize("dt", DT)
def test_steps_follow_the_scan(rq, dev, dt):
    g = torch.Generator().manual_seed(9)
    t = 20
    six = [x.to(dev) for x in inputs(g, 3, t, 5, dtype=DT[dt])]
    state = torch.randn(3, 5, D, D, generator=g).to(dev)
    y, last = rq.wkv7(*six, state, out_dtype=torch.float32)
    s, other = state.clone(), torch.empty_like(state)
    for i in range(t):
        tok = [x[:, i] for x in six]
        if i % 3 == 0:       # in place
            yi, s2 = rq.wkv7_step(*tok, s, out=s, out_dtype=torch.float32)
            assert s2 is s
        elif i % 3 == 1:     # to a buffer
            yi, other = rq.wkv7_step(*tok, s, out=other, out_dtype=torch.float32)
            s, other = other, s
        else:                # to a new one, and as a scan of one token
            y1, s1 = rq.wkv7(*[x[:, None] for x in tok], s, out_dtype=torch.float32)
            yi, s = rq.wkv7_step(*tok, s, out_dtype=torch.float32)
            assert torch.equal(y1[:, 0], yi) and torch.equal(s1, s)
        e = bound("y", torch.float32, t)
        assert (yi.double() - y[:, i].double()).norm() <= 2 * e * y.double().norm() / math.sqrt(t) * 8
    close(s, last.double().cpu(), "state", 2 * t)
    y16, _ = rq.wkv7_step(*[x[:, 0] for x in six], state)
    assert y16.dtype == DT[dt]
    y32, _ = rq.wkv7_step(*[x[:, 0] for x in six], state, out_dtype=torch.float32)
    assert torch.equal(y16, y32.to(DT[dt]))


def test_a_state_carries_over(rq, dev):
    g = torch.Generator().manual_seed(10)
    six = [x.to(dev) for x in inputs(g, 2, 75, 2)]
    y, last = rq.wkv7(*six)
    y1, s = rq.wkv7(*[x[:, :30] for x in six])
    y2, s = rq.wkv7(*[x[:, 30:] for x in six], s)
    close(torch.cat([y1, y2], 1), y.double().cpu(), "y", 75)
    close(s, last.double().cpu(), "state", 75)
    # later tokens change nothing before them
    other = [torch.cat([x[:, :30], x[:, 30:].flip(1)], 1) for x in six]
    assert torch.equal(rq.wkv7(*other)[0][:, :30], y[:, :30])


def test_neutral_tokens_keep_the_state(rq, dev):
    g = torch.Generator().manual_seed(11)
    six = [x.to(dev) for x in inputs(g, 1, 40, 2)]
    state = torch.randn(1, 2, D, D, generator=g).to(dev)
    six[1].fill_(-math.inf)
    six[2].zero_()
    six[5].zero_()
    y, last = rq.wkv7(*six, state)
    assert torch.equal(last, state)
    _, last = rq.wkv7_step(*[x[:, 0] for x in six], state)
    assert torch.equal(last, state)
    # a batch padded at its end: each row's state is that of its own length
    six = [x.to(dev) for x in inputs(g, 3, 40, 2)]
    lens = [40, 1, 23]
    for i, n in enumerate(lens):
        six[1][i, n:] = -math.inf
        six[2][i, n:] = 0
        six[5][i, n:] = 0
    y, last = rq.wkv7(*six)
    for i, n in enumerate(lens):
        yi, si = rq.wkv7(*[x[i:i + 1, :n] for x in six])
        close(last[i:i + 1], si.double().cpu(), "state", 40)
        close(y[i:i + 1, :n], yi.double().cpu(), "y", 40)


def test_what_lies_behind_the_last_sequence_does_not_matter(rq, dev):
    g = torch.Generator().manual_seed(12)
    six = [x.to(dev) for x in inputs(g, 1, 50, 2)]
    cu = torch.tensor([3, 20, 41], dtype=torch.int64, device=dev)
    bad = [x.clone() for x in six]
    for x in bad:
        x[:, :3] = math.nan
        x[:, 41:] = math.inf
    dy = torch.randn(1, 50, 2, D, generator=g).to(dev)
    bad_dy = dy.clone()
    bad_dy[:, 41:] = math.nan
    res = []
    for s, d in ((six, dy), (bad, bad_dy)):
        s = [x.requires_grad_() for x in s]
        y, last = rq.wkv7(*s, cu_seqlens=cu)
        res.append([y, last, *torch.autograd.grad(y, s, d)])
    for x, z in zip(*res):
        assert torch.equal(x, z) and x.isfinite().all()
    assert (res[0][0][:, :3] == 0).all() and (res[0][0][:, 41:] == 0).all()


def test_boundaries_outside_the_batch_stay_inside(rq, dev):
    g = torch.Generator().manual_seed(13)
    six = [x.to(dev) for x in inputs(g, 1, 30, 2)]
    far = torch.tensor([-5, 10, 10, 2 ** 31 - 1], dtype=torch.int32, device=dev)
    near = torch.tensor([0, 10, 10, 30], dtype=torch.int32, device=dev)
    for x, z in zip(rq.wkv7(*six, cu_seqlens=far), rq.wkv7(*six, cu_seqlens=near)):
        assert torch.equal(x, z)
    # boundaries that decrease: nothing outside the tensors is touched, forwards or backwards
    wild = torch.tensor([25, 3, 28, 1, 30, 0], dtype=torch.int32, device=dev)
    s = [x.requires_grad_() for x in six]
    y, last = rq.wkv7(*s, cu_seqlens=wild)
    grads = torch.autograd.grad(y.sum() + last.sum(), s)
    torch.cuda.synchronize()
    assert last.shape == (5, 2, D, D) and len(grads) == 6


def test_nan_and_infinite_inputs_reach_what_depends_on_them(rq, dev):
    g = torch.Generator().manual_seed(14)
    six = [x.to(dev) for x in inputs(g, 2, 40, 2)]
    clean, clean_last = rq.wkv7(*six)
    for j, name in enumerate(NAMES):
        xs = [x.clone() for x in six]
        xs[j][0, 20, 1, 5] = math.nan
        y, last = rq.wkv7(*xs)
        assert torch.equal(y[1], clean[1]) and torch.equal(y[0, :, 0], clean[0, :, 0])
        assert torch.equal(y[0, :16, 1], clean[0, :16, 1])   # the chunks before
        assert y[0, 20, 1].isnan().any(), name
        if name != "r":
            assert last[0, 1].isnan().any(), name


def test_strides_alignment_and_mixed_types(rq, dev):
    g = torch.Generator().manual_seed(15)
    six = inputs(g, 2, 33, 3, dtype=torch.bfloat16)
    want, wlast = rq.wkv7(*[x.to(dev) for x in six])
    # one projection's slices, heads first in memory, an odd offset, every other token of a longer tensor
    odd = []
    for j, x in enumerate(six):
        x = x.to(dev)
        if j % 3 == 0:
            odd.append(x.transpose(1, 2).contiguous().transpose(1, 2))
        elif j % 3 == 1:
            flat = torch.empty(x.numel() + 3, dtype=x.dtype, device=dev)
            odd.append(flat[3:].view(x.shape).copy_(x))
        else:
            long = torch.empty(2, 66, 3, D, dtype=x.dtype, device=dev)
            odd.append(long[:, ::2].copy_(x))
    y, last = rq.wkv7(*odd)
    assert torch.equal(y, want) and torch.equal(last, wlast)
    # another type among them: float32 throughout
    mixed = [x.to(dev) for x in six]
    mixed[1] = mixed[1].float()
    y, _ = rq.wkv7(*mixed)
    assert y.dtype == torch.float32
    assert torch.equal(y, rq.wkv7(*[x.float() for x in mixed])[0])
    state = torch.randn(2, 3, D, D, generator=g).to(dev)
    y1, s1 = rq.wkv7(*mixed, state)
    y2, s2 = rq.wkv7(*mixed, state.transpose(0, 1).contiguous().transpose(0, 1))
    assert torch.equal(y1, y2) and torch.equal(s1, s2)


def test_broadcast_inputs_and_gradients(rq, dev):
    """One a for all heads, one decay for all tokens: their gradients are the sums."""
    g = torch.Generator().manual_seed(16)
    six = [x.to(dev) for x in inputs(g, 2, 20, 3)]
    a = six[4][:, :, :1].clone().requires_grad_()
    w = six[1][:, :1].clone().requires_grad_()
    six[1], six[4] = w.expand(2, 20, 3, D), a.expand(2, 20, 3, D)
    y, _ = rq.wkv7(*six)
    dy = torch.randn(y.shape, generator=g).to(dev)
    dw, da = torch.autograd.grad(y, [w, a], dy)
    full = [x.detach().contiguous().requires_grad_() for x in six]
    gr = torch.autograd.grad(rq.wkv7(*full)[0], full, dy)
    assert dw.shape == w.shape and da.shape == a.shape
    assert torch.allclose(dw, gr[1].sum(1, keepdim=True), rtol=0, atol=40 * U32 * gr[1].abs().sum(1).max().item())
    assert torch.allclose(da, gr[4].sum(2, keepdim=True), rtol=0, atol=6 * U32 * gr[4].abs().sum(2).max().item())


def test_only_what_is_wanted(rq, dev):
    """Gradients of one input, of the state alone, from the last state alone."""
    g = torch.Generator().manual_seed(17)
    six = [x.to(dev) for x in inputs(g, 1, 35, 2)]
    state = torch.randn(1, 2, D, D, generator=g).to(dev)
    dy, ds = torch.randn(1, 35, 2, D, generator=g).to(dev), torch.randn(1, 2, D, D, generator=g).to(dev)
    want = reference(six, state, 0 * dy, ds)
    for j, name in enumerate(LEAVES):
        leaf = [*six, state]
        leaf[j] = leaf[j].clone().requires_grad_()
        _, last = rq.wkv7(*leaf[:6], leaf[6])
        d, = torch.autograd.grad(last, [leaf[j]], ds, allow_unused=True)
        if d is None:
            d = torch.zeros_like(leaf[j])
        close(d, want["d" + name], "d" + name, 35) if want["d" + name].norm() else None
    with pytest.raises(RuntimeError):
        x = [t.clone().requires_grad_() for t in six]
        gr, = torch.autograd.grad(rq.wkv7(*x)[0].sum(), x[:1], create_graph=True)
        torch.autograd.grad(gr.sum(), x)


def test_the_same_bits_and_other_streams(rq, dev):
    g = torch.Generator().manual_seed(18)
    six = [x.to(dev) for x in inputs(g, 4, 90, 3, dtype=torch.bfloat16)]
    dy = torch.randn(4, 90, 3, D, generator=g).to(torch.bfloat16).to(dev)

    def once():
        s = [x.detach().requires_grad_() for x in six]
        y, last = rq.wkv7(*s)
        return [y, last, *torch.autograd.grad(y, s, dy)]

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = once()
    torch.cuda.current_stream().wait_stream(side)
    both = []
    for s in (side, torch.cuda.Stream()):   # two at once
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            both.append(once())
    torch.cuda.synchronize()
    for other in (there, *both, once()):
        for x, z in zip(first, other):
            assert torch.equal(x, z)


def test_captured_and_replayed(rq, dev):
    """Decode steps and a scan in one graph, a training pass in another; replays with eager work
    between them."""
    g = torch.Generator().manual_seed(19)
    six = [x.to(dev) for x in inputs(g, 2, 37, 2, dtype=torch.bfloat16)]
    tok = [x[:, 0].clone() for x in six]
    state = torch.randn(2, 2, D, D, generator=g).to(dev)
    buf = state.clone()

    def serve():
        y, last = rq.wkv7(*six, state)
        rq.wkv7_step(*tok, buf, out=buf)
        y1, _ = rq.wkv7_step(*tok, buf, out=buf)
        return y, last, y1

    leaves = [x.clone().requires_grad_() for x in six]
    dy = torch.randn(2, 37, 2, D, generator=g).to(torch.bfloat16).to(dev)

    def train():
        y, last = rq.wkv7(*leaves)
        return [y, last, *torch.autograd.grad(y, leaves, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        serve()
        train()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for f in (serve, train):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = f()
        graphs.append((graph, out))
    for i in range(4):
        with torch.no_grad():
            for x, z in zip(six, leaves):
                x.copy_(x.roll(1 + i, 1))
                z.copy_(x)
            for x, z in zip(tok, six):
                x.copy_(z[:, i])
        buf.copy_(state * (i + 1))
        for graph, _ in graphs:
            graph.replay()
        after = buf.clone()
        got = [[t.clone() for t in out] for _, out in graphs]
        torch.cuda.synchronize()
        buf.copy_(state * (i + 1))
        want = [serve(), train()]
        assert torch.equal(after, buf)
        for a, b in zip(got, want):
            for x, z in zip(a, b):
                assert torch.equal(x, z)


def test_captured_segments_of_one_pool(rq, dev):
    """Two graphs that share a pool, and with it the memory of their workspaces: each replay behind the other and behind
    eager work gives the eager bits."""
    g = torch.Generator().manual_seed(99)
    six = [x.to(dev) for x in inputs(g, 1, 701, 2, dtype=torch.bfloat16)]
    state = torch.randn(1, 2, D, D, generator=g).to(dev)
    dy = torch.randn(1, 701, 2, D, generator=g).to(torch.bfloat16).to(dev)
    cu = torch.tensor([0, 450, 450, 699], dtype=torch.int32, device=dev)
    states = torch.randn(3, 2, D, D, generator=g).to(dev)
    leaves = [x.clone().requires_grad_() for x in six]

    def train():
        y, last = rq.wkv7(*leaves, state)
        return [y, last, *torch.autograd.grad(y, leaves, dy)]

    def serve():
        return list(rq.wkv7(*six, states, cu_seqlens=cu))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train()
        serve()
    torch.cuda.current_stream().wait_stream(side)
    graphs, pool = [], None
    for f in (train, serve):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            out = f()
        pool = graph.pool()
        graphs.append((graph, out, f))
    for i in range(3):
        with torch.no_grad():
            for x, z in zip(six, leaves):
                x.copy_(x.roll(7 * i + 1, 1))
                z.copy_(x)
        for graph, out, f in (graphs, graphs[::-1])[i % 2]:
            graph.replay()
            got = [x.detach().clone() for x in out]
            torch.cuda.synchronize()
            for x, z in zip(got, f()):
                assert torch.equal(x, z)


def test_offsets_past_32_bits(rq, dev):
    """A packed row of 17 million tokens of one head, 4.35e9 bytes of each tensor and 1.7e10 of states,
    the sequences at its end."""
    n, g = 17_000_003, torch.Generator().manual_seed(20)
    short = [x.to(dev) for x in inputs(g, 1, 70, 1)]
    big = [torch.empty(1, n, 1, D, device=dev) for _ in range(6)]
    for x, s in zip(big, short):
        x[:, n - 72:n - 2] = s
    six = [x.requires_grad_() for x in big]
    cu = torch.tensor([n - 72, n - 40, n - 2], dtype=torch.int32, device=dev)
    y, last = rq.wkv7(*six, cu_seqlens=cu)
    dy = torch.zeros_like(y)
    d = torch.randn(1, 70, 1, D, generator=g).to(dev)
    dy[:, n - 72:n - 2] = d
    grads = torch.autograd.grad(y, six, dy)
    tail = [s.requires_grad_() for s in short]
    cu2 = torch.tensor([0, 32, 70], dtype=torch.int32, device=dev)
    y2, last2 = rq.wkv7(*tail, cu_seqlens=cu2)
    grads2 = torch.autograd.grad(y2, tail, d)
    assert torch.equal(y[:, n - 72:n - 2], y2) and torch.equal(last, last2)
    assert (y[:, :n - 72:4099] == 0).all() and (y[:, n - 2:] == 0).all()
    for x, z in zip(grads, grads2):
        assert torch.equal(x[:, n - 72:n - 2], z)
        assert (x[:, :n - 72:4099] == 0).all() and (x[:, n - 2:] == 0).all()


def test_states_past_32_bits(rq, dev):
    """2^18 + 3 heads of sequences: 4 GB of states."""
    g = torch.Generator().manual_seed(21)
    b = 2 ** 18 + 3
    tok = [x.to(dev) for x in inputs(g, 8, 1, dtype=torch.bfloat16)]
    big = [x.repeat(b // 8 + 1, 1, 1)[:b] for x in tok]
    state = torch.randn(8, 1, D, D, generator=g).to(dev)
    s = state.repeat(b // 8 + 1, 1, 1, 1)[:b]
    y, last = rq.wkv7_step(*big, s)
    y8, last8 = rq.wkv7_step(*tok, state)
    assert torch.equal(y[-3:], y8[[(b - 3 + i) % 8 for i in range(3)]])
    assert torch.equal(last[-3:], last8[[(b - 3 + i) % 8 for i in range(3)]])
    del last
    y, last = rq.wkv7(*[x[:, None].expand(b, 2, 1, D) for x in big], s)
    y8, last8 = rq.wkv7(*[x[:, None].expand(8, 2, 1, D).repeat(30, 1, 1, 1) for x in tok], state.repeat(30, 1, 1, 1))
    assert torch.equal(last[-3:], last8[[(b - 3 + i) % 8 for i in range(3)]])
    assert torch.equal(y[-3:], y8[[(b - 3 + i) % 8 for i in range(3)]])


def test_registered_ops(rq, dev):
    g = torch.Generator().manual_seed(22)
    six = [x.to(dev).requires_grad_() for x in inputs(g, 1, 20, 2)]
    cu = torch.tensor([0, 7, 20], dtype=torch.int32, device=dev)
    state = torch.randn(2, 2, D, D, generator=g).to(dev).requires_grad_()
    checks = ("test_schema", "test_faketensor", "test_autograd_registration")
    torch.library.opcheck(torch.ops.rwkvq.wkv7.default, (*six, state, cu, torch.float32, True), test_utils=checks)
    torch.library.opcheck(torch.ops.rwkvq.wkv7.default, (*[x.detach() for x in six], None, None, torch.float32, False),
                          test_utils=checks)
    # under a dispatch mode the registered op runs: the same bits
    from torch.utils._python_dispatch import TorchDispatchMode

    class Seen(TorchDispatchMode):
        ops = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.ops.append(str(func))
            return func(*args, **(kwargs or {}))

    dy = torch.randn(1, 20, 2, D, generator=g).to(dev)
    y, last = rq.wkv7(*six, state, cu)
    want = torch.autograd.grad(y, [*six, state], dy)
    with Seen():
        y2, last2 = rq.wkv7(*six, state, cu)
        got = torch.autograd.grad(y2, [*six, state], dy)
    assert any("rwkvq.wkv7" in o for o in Seen.ops)
    assert torch.equal(y, y2) and torch.equal(last, last2)
    assert all(torch.equal(x, z) for x, z in zip(want, got))


def test_refusals(rq, dev):
    g = torch.Generator().manual_seed(23)
    six = [x.to(dev) for x in inputs(g, 2, 5, 3)]
    state = torch.zeros(2, 3, D, D, device=dev)
    with pytest.raises(ValueError, match="one shape"):
        rq.wkv7(*six[:5], six[5][:, :4])
    with pytest.raises(ValueError, match="batch, time, heads, 64"):
        rq.wkv7(*[x[..., :32] for x in six])
    with pytest.raises(ValueError, match="bfloat16"):
        rq.wkv7(*[x.double() for x in six])
    with pytest.raises(ValueError, match="state must be"):
        rq.wkv7(*six, state[:1])
    with pytest.raises(ValueError, match="state must be"):
        rq.wkv7(*six, state.bfloat16())
    with pytest.raises(ValueError, match="out_dtype"):
        rq.wkv7(*six, out_dtype=torch.bfloat16)
    cu = torch.tensor([0, 5], dtype=torch.int32, device=dev)
    with pytest.raises(ValueError, match="batch of 1"):
        rq.wkv7(*six, cu_seqlens=cu)
    one = [x[:1] for x in six]
    with pytest.raises(ValueError, match="boundaries"):
        rq.wkv7(*one, cu_seqlens=cu.float())
    with pytest.raises(ValueError, match="no sequence"):
        rq.wkv7(*one, cu_seqlens=cu[:1])
    with pytest.raises((ValueError, RuntimeError)):
        rq.wkv7(*one, cu_seqlens=cu.cpu())
    with pytest.raises((ValueError, RuntimeError)):
        rq.wkv7(*one, state[:1].cpu())
    tok = [x[:, 0] for x in six]
    with pytest.raises(ValueError, match="batch, heads, 64"):
        rq.wkv7_step(*six, state)
    with pytest.raises(ValueError, match="out must be"):
        rq.wkv7_step(*tok, state, out=state[:1])
    with pytest.raises(ValueError, match="contiguous"):
        rq.wkv7_step(*tok, state, out=state.transpose(2, 3))
    pool = torch.zeros(3, 3, D, D, device=dev)
    with pytest.raises(ValueError, match="overlap"):
        rq.wkv7_step(*tok, pool[:2], out=pool[1:])
