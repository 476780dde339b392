"""The precision of the recurrence's gradients, where a norm over the whole tensor or the rounding to 16 bits
would hide its loss."""
import math

import pytest
import torch

from wkv_ref import D, DT, NAMES, bound, inputs, reference

pytestmark = pytest.mark.gpu


def grads(rq, dev, six, state, dy, dstate, cu, out):
    six = [x.to(dev).requires_grad_() for x in six]
    state = state.to(dev).requires_grad_()
    y, last = rq.wkv7(*six, state, cu_seqlens=cu, out_dtype=out)
    return torch.autograd.grad([y, last], [*six, state], [dy.to(dev), dstate.to(dev)])


# one head over a few chunks, several heads, a long one in segments, packed ones with an empty one
SHAPES = [(1, 16, 1, None), (2, 77, 3, None), (1, 1100, 2, None), (1, 90, 2, [33, 0, 1, 50])]


@pytest.mark.parametrize("decays", ["model", "strong", "infinite value"])
@pytest.mark.parametrize("dt,out", [("bf16", "bf16"), ("bf16", "fp32"), ("f16", "f16"), ("f16", "fp32")])
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_gradients_of_16_bit_tensors_are_rounded_once(rq, dev, i, dt, out, decays):
    """Behind the loads nothing depends on the tensors' type: the gradients of 16-bit tensors are those of
    the same numbers in float32, rounded where they are stored."""
    b, t, h, lens = SHAPES[i]
    print(f"wkv7 gradients b={b} t={t} h={h} lens={lens} {dt}->{out} {decays}", flush=True)
    g = torch.Generator().manual_seed(300 + i)
    six = inputs(g, b, t, h, dtype=DT[dt])
    if decays == "strong":
        six[1][:, ::3, :, ::7] = 3.5
    if decays == "infinite value":
        six[3][:, t // 2, 0, 5] = math.inf
    seqs = b if lens is None else len(lens)
    state, dstate = (torch.randn(seqs, h, D, D, generator=g) for _ in range(2))
    dy = torch.randn(b, t, h, D, generator=g).to(DT[out])
    cu = None if lens is None else torch.tensor([0, 33, 33, 34, 84], dtype=torch.int32, device=dev)
    got = grads(rq, dev, six, state, dy, dstate, cu, DT[out])
    want = grads(rq, dev, [x.float() for x in six], state, dy.float(), dstate, cu, torch.float32)
    for name, x, z in zip([*NAMES, "state"], got, want):
        z = z.to(x.dtype)
        assert x.dtype == (torch.float32 if name == "state" else DT[dt])
        same = (x == z) | (x.isnan() & z.isnan())
        assert same.all(), f"d{name}: {(~same).sum().item()} of {x.numel()} differ"


# A token that decays hard among others that hardly do: the pairs of tokens to one side of it are any number of times
# larger than those that pass its decay, and have no part in its dw.  Over chunk, group and segment boundaries; strong enough
# (5: the pairwise form) and not.
LONE = [("first", [0], 3.0, -8.0), ("mid", [7], 3.0, -6.0), ("mid", [9], 3.0, -4.0), ("edge", [0], -0.5, -8.0),
        ("several", [2, 3, 13, 16, 21, 36], 2.5, -7.0), ("strong", [6, 20], 5.0, -8.0), ("chunk's last", [15, 31], 3.0, -8.0)]


@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("i", range(len(LONE)))
def test_decay_gradients_token_by_token(rq, dev, i, dt, given):
    """Every token's dw by its own norm.  The bound is that of a gradient over the whole tensor (wkv_ref): each of
    a token's terms passes the same roundings, and none of it is larger than what it adds to the token's own."""
    name, at, w, others = LONE[i]
    print(f"wkv7 dw {name} w={w} others={others} {dt} state={given}", flush=True)
    t, h = 40, 4
    g = torch.Generator().manual_seed(400 + i)
    six = inputs(g, 1, t, h, dtype=DT[dt], w=others)
    six[1][:, at] = w
    state = torch.randn(1, h, D, D, generator=g) if given else torch.zeros(1, h, D, D)
    dstate = torch.randn(1, h, D, D, generator=g)
    dy = torch.randn(1, t, h, D, generator=g).to(DT[dt])
    want = reference(six, state, dy, dstate)["dw"]
    got = grads(rq, dev, six, state, dy, dstate, None, DT[dt])[1]
    e = bound("dw", DT[dt], t)
    # the smallest steps of the type are not relative: half of one for each value
    least = math.sqrt(h * D) * torch.finfo(DT[dt]).smallest_normal * torch.finfo(DT[dt]).eps / 2
    off = (got.double().cpu() - want).norm(dim=(2, 3))[0]
    norm = want.norm(dim=(2, 3))[0]
    worst = (off / (e * norm + least)).max().item()
    assert worst <= 1, f"{worst:.3g} times the bound at token {(off / (e * norm + least)).argmax().item()}"
    if not given:
        assert (got[:, 0] == 0).all()   # nothing passes the first token's decay


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("i", range(len(LONE)))
def test_everything_token_by_token(rq, dev, i, dt):
    """y and the other gradients by each token's own norm, in the same company."""
    name, at, w, others = LONE[i]
    print(f"wkv7 by tokens {name} w={w} others={others} {dt}", flush=True)
    t, h = 40, 4
    g = torch.Generator().manual_seed(450 + i)
    six = inputs(g, 1, t, h, dtype=DT[dt], w=others)
    six[1][:, at] = w
    state, dstate = torch.randn(1, h, D, D, generator=g), torch.randn(1, h, D, D, generator=g)
    dy = torch.randn(1, t, h, D, generator=g).to(DT[dt])
    want = reference(six, state, dy, dstate)
    got = dict(zip(["d" + n for n in NAMES], grads(rq, dev, six, state, dy, dstate, None, DT[dt])))
    got["y"] = rq.wkv7(*[x.to(dev) for x in six], state.to(dev))[0]
    least = math.sqrt(h * D) * torch.finfo(DT[dt]).smallest_normal * torch.finfo(DT[dt]).eps / 2
    for n, x in got.items():
        off = (x.double().cpu() - want[n]).norm(dim=(2, 3))[0]
        worst = off / (bound(n, DT[dt], t) * want[n].norm(dim=(2, 3))[0] + least)
        assert worst.max() <= 1, f"{n}: {worst.max().item():.3g} times the bound at token {worst.argmax().item()}"
