"""The precision of the recurrence's gradients, where a norm over the whole tensor or the rounding to 16 bits
would hide its loss."""
import math

import pytest
import torch

from wkv_ref import D, DT, NAMES, inputs

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
