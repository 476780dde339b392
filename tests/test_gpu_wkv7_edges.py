"""Calls of the recurrence that its documentation allows and that are easily forgotten: steps whose state something
else still needs, tracing, forward mode, memory around the tensors."""
import math

import pytest
import torch
from torch.autograd import forward_ad

from wkv_ref import D, DT, NAMES, inputs

pytestmark = pytest.mark.gpu


def token(dev, batch=3, heads=2, dt=torch.bfloat16, seed=1):
    g = torch.Generator().manual_seed(seed)
    six = [x.to(dev) for x in inputs(g, batch, heads, dtype=dt)]
    return six, torch.randn(batch, heads, D, D, generator=g).to(dev)


@pytest.mark.parametrize("in_place", [True, False])
def test_a_saved_state_that_is_written_to(rq, dev, in_place):
    """As torch's own operations in place: an error where the old values are needed."""
    six, state = token(dev)
    out = state if in_place else torch.zeros_like(state)
    weight = torch.ones_like(state).requires_grad_()
    loss = (out * weight).sum()       # keeps `out` for weight's gradient
    version = out._version
    rq.wkv7_step(*six, state, out=out)
    assert out._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    view = torch.zeros(2, *state.shape, device=dev)
    version = view._version
    rq.wkv7_step(*six, state, out=view[1])
    assert view._version > version and (view[0] == 0).all()


def test_an_output_that_requires_gradients(rq, dev):
    six, state = token(dev)
    leaf = torch.zeros_like(state).requires_grad_()
    for out in (leaf, leaf * 2):
        with pytest.raises(ValueError, match="gradients"):
            rq.wkv7_step(*six, state, out=out)
    with pytest.raises(ValueError, match="gradients"):
        rq.wkv7_step(*six, leaf, out=leaf)
    want = rq.wkv7_step(*six, state)[1]
    with torch.no_grad():
        rq.wkv7_step(*six, state, out=leaf)
    assert torch.equal(leaf, want)
    with torch.inference_mode():
        mine = state.clone()
        y, new = rq.wkv7_step(*six, mine, out=mine)
    assert torch.equal(new, want)


def test_an_output_over_the_token_is_refused(rq, dev):
    """Before anything is launched; memory side by side is not refused."""
    batch, heads = 3, 2
    size, n = batch * heads * D * D, batch * heads * D
    memory = torch.zeros(size + 6 * n, device=dev)
    state = torch.randn(batch, heads, D, D, device=dev)
    out = memory[:size].view(state.shape)
    beside = [memory[size + i * n:size + (i + 1) * n].view(batch, heads, D) for i in range(6)]
    want, _ = rq.wkv7_step(*beside, state)
    got, new = rq.wkv7_step(*beside, state, out=out)
    assert torch.equal(got, want) and new is out
    inside = memory[size - n // 2:size + n // 2].view(batch, heads, D)   # its first half
    for i in range(6):
        six = [inside if j == i else x for j, x in enumerate(beside)]
        with pytest.raises(ValueError, match="overlap"):
            rq.wkv7_step(*six, state, out=out)
        with pytest.raises(ValueError, match="overlap"):
            rq.wkv7_step(*six, out, out=out)
    # a strided one is copied first
    apart = memory[:2 * n].view(n, 2)[:, 0].view(batch, heads, D)
    rq.wkv7_step(apart, *beside[1:], state, out=out)
    for x in rq.wkv7_step(*[x[:0] for x in beside], state[:0], out=out[:0]):
        assert x.numel() == 0


def test_boundaries_of_64_bits(rq, dev):
    """Moved into the batch by their value, whatever their low 32 bits say."""
    g = torch.Generator().manual_seed(2)
    six = [x.to(dev).requires_grad_() for x in inputs(g, 1, 30, 2)]
    dy = torch.randn(1, 30, 2, D, generator=g).to(dev)
    far = torch.tensor([-2 ** 32, 10, 10, 2 ** 32 + 12], device=dev)
    near = torch.tensor([0, 10, 10, 30], dtype=torch.int32, device=dev)
    got, want = [], []
    for cu, res in ((far, got), (near, want)):
        y, last = rq.wkv7(*six, cu_seqlens=cu)
        res += [y, last, *torch.autograd.grad(y, six, dy)]
    for x, z in zip(got, want):
        assert torch.equal(x, z)
    far = torch.tensor([2 ** 33, 2 ** 33 + 5, 2 ** 40], device=dev)   # all behind the end
    y, last = rq.wkv7(*six, cu_seqlens=far)
    assert (y == 0).all() and (last == 0).all()
