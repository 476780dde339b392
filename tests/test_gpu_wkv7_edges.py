"""Calls of the recurrence that its documentation allows and that are easily forgotten: steps whose state something
else still needs, tracing, forward mode, memory around the tensors."""

import pytest
import torch
from torch.autograd import forward_ad

from wkv_ref import D, NAMES, close, inputs, reference

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


def test_what_is_not_reached_has_no_gradient(rq, dev):
    """r reads states and changes none: the last state's gradient leaves dr at 0, exactly; and nothing is left out."""
    g = torch.Generator().manual_seed(3)
    six = [x.to(dev).requires_grad_() for x in inputs(g, 2, 35, 2)]
    state = torch.randn(2, 2, D, D, generator=g).to(dev).requires_grad_()
    ds = torch.randn(2, 2, D, D, generator=g).to(dev)
    _, last = rq.wkv7(*six, state)
    grads = torch.autograd.grad(last, [*six, state], ds)
    for name, x in zip([*NAMES, "state"], grads):
        assert (x == 0).all() if name == "r" else x.norm() > 0, name
    # and y's gradient of a sequence's last token alone reaches none behind it
    y, _ = rq.wkv7(*six, state)
    dy = torch.zeros_like(y)
    dy[:, 20] = torch.randn(2, 2, D, generator=g).to(dev)
    for name, x in zip(NAMES, torch.autograd.grad(y, six, dy)):
        assert (x[:, 21:] == 0).all(), name
        assert x[:, 20].norm() > 0, name


def test_shapes_on_both_sides_of_the_plan(rq, dev):
    """The first length of one head that runs in segments, and the one before it, forwards and backwards."""
    L = rq._lib.lib()
    for query in (L.rq_wkv7_workspace_bytes, L.rq_wkv7_backward_workspace_bytes):
        for heads in (1, 3):
            time = next(t for t in range(16, 4000, 16) if query(1, t, heads, 1, 0) > 0)
            for t in (time - 16, time - 15, time, time + 1):
                g = torch.Generator().manual_seed(t)
                six = [x.to(dev).requires_grad_() for x in inputs(g, 1, t, heads)]
                dy = torch.randn(1, t, heads, D, generator=g).to(dev)
                y, last = rq.wkv7(*six)
                grads = torch.autograd.grad(y, six, dy)
                want = reference(six, torch.zeros(1, heads, D, D), dy)
                close(y.detach(), want["y"], "y", t)
                close(last.detach(), want["state"], "state", t)
                for name, x in zip(NAMES, grads):
                    close(x, want["d" + name], "d" + name, t)


def test_saved_tensor_hooks(rq, dev):
    """What is kept goes through the hooks: on the host meanwhile, the same gradients."""
    g = torch.Generator().manual_seed(4)
    six = [x.to(dev).requires_grad_() for x in inputs(g, 2, 35, 2, dtype=torch.bfloat16)]
    dy = torch.randn(2, 35, 2, D, generator=g).to(torch.bfloat16).to(dev)
    want = torch.autograd.grad(rq.wkv7(*six)[0], six, dy)
    with torch.autograd.graph.save_on_cpu():
        y, _ = rq.wkv7(*six)
    for x, z in zip(torch.autograd.grad(y, six, dy), want):
        assert torch.equal(x, z)
    # the kept boundaries that are overwritten before the backward pass: an error
    one = [x.detach()[:1].requires_grad_() for x in six]
    cu = torch.tensor([0, 11, 35], dtype=torch.int32, device=dev)
    y, _ = rq.wkv7(*one, cu_seqlens=cu)
    cu.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, one, dy[:1])


def test_registered_steps(rq, dev):
    six, state = token(dev)
    checks = ("test_schema", "test_faketensor")
    torch.library.opcheck(torch.ops.rwkvq.wkv7_step.default, (*six, state, torch.float32), test_utils=checks)
    torch.library.opcheck(torch.ops.rwkvq.wkv7_step_out.default, (*six, state, torch.zeros_like(state), torch.bfloat16),
                          test_utils=checks)
    torch.library.opcheck(torch.ops.rwkvq.wkv7_step_out.default, (*six, None, state.clone(), torch.bfloat16), test_utils=checks)
    want, new = rq.wkv7_step(*six, state)

    traced = torch.jit.trace(lambda *t: rq.wkv7_step(*t), (*[x * 0 for x in six], state * 0), check_trace=False)
    compiled = torch.compile(lambda *t: rq.wkv7_step(*t), backend="aot_eager", fullgraph=True)
    for f in (traced, compiled):
        y, s = f(*six, state)
        assert torch.equal(y, want) and torch.equal(s, new)
    in_place = torch.compile(lambda *t: rq.wkv7_step(*t, out=t[6])[0], backend="aot_eager", fullgraph=True)
    for f in (in_place, torch.jit.trace(lambda *t: rq.wkv7_step(*t, out=t[6])[0], (*six, state.clone()), check_trace=False)):
        mine = state.clone()
        version = mine._version
        assert torch.equal(f(*six, mine), want) and torch.equal(mine, new) and mine._version > version
    buffer = torch.compile(lambda o, *t: rq.wkv7_step(*t, out=o)[0], backend="aot_eager", fullgraph=True)
    other = torch.zeros_like(state)
    assert torch.equal(buffer(other, *six, state), want) and torch.equal(other, new)


def test_compiled_scan_and_sampler(rq, dev):
    g = torch.Generator().manual_seed(5)
    six = [x.to(dev).requires_grad_() for x in inputs(g, 1, 50, 2)]
    state = torch.randn(2, 2, D, D, generator=g).to(dev).requires_grad_()
    cu = torch.tensor([0, 17, 50], dtype=torch.int32, device=dev)
    dy = torch.randn(1, 50, 2, D, generator=g).to(dev)
    compiled = torch.compile(lambda *t: rq.wkv7(*t, cu_seqlens=cu), backend="aot_eager", fullgraph=True)
    res = []
    for f in (lambda *t: rq.wkv7(*t, cu_seqlens=cu), compiled):
        y, last = f(*six, state)
        res.append([y, last, *torch.autograd.grad([y, last], [*six, state], [dy, torch.ones_like(last)])])
    for x, z in zip(*res):
        assert torch.equal(x, z)
    logits, u = torch.randn(4, 301, generator=g).to(dev), torch.rand(4, generator=g).to(dev)
    kw = {"temperature": 0.7, "top_k": 20, "top_p": 0.9}
    want = rq.sample(logits, u, **kw)
    for f in (torch.compile(lambda l, v: rq.sample(l, v, **kw), backend="aot_eager", fullgraph=True),
              torch.jit.trace(lambda l, v: rq.sample(l, v, **kw), (logits * 0, u * 0), check_trace=False)):
        token, logprob = f(logits, u)
        assert torch.equal(token, want[0]) and torch.equal(logprob, want[1])


def test_forward_mode_is_refused_on_the_gpu(rq, dev):
    six, state = token(dev)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(six[2], torch.ones_like(six[2]))
        with pytest.raises(NotImplementedError):
            rq.wkv7_step(*six[:2], dual, *six[3:], state)
        with pytest.raises(NotImplementedError):
            rq.wkv7(*[x[:, None] for x in (*six[:2], dual, *six[3:])], state)
        y, _ = rq.wkv7_step(*six, state)
    assert torch.equal(y, rq.wkv7_step(*six, state)[0])
