"""Refusals and host logic of rwkvq.train at its edges, without a GPU: nothing
here reaches a launch."""
import ctypes

import pytest
import torch

P = 0x1000  # never dereferenced: validation fails first


@pytest.fixture(scope="module")
def L():
    from rwkvq import _lib
    return _lib.lib()


def err(L):
    return L.rq_last_error().decode()


def clip(L, *entries):
    """rq_clip_grads of (g, out, elements[, dtype]) with a workspace that is too
    small, which is the check behind the one of shared memory."""
    from rwkvq._lib import RqGrad
    a = (RqGrad * len(entries))(*[RqGrad(e[0], e[1], e[2], e[3] if len(e) > 3 else 2, 0) for e in entries])
    assert L.rq_clip_grads(ctypes.addressof(a), len(entries), 1.0, 1e-6, P, P, 0, None) == -1
    return err(L)


def test_clip_refuses_outputs_that_share_memory(L):
    a, b, c = 0x10000, 0x20000, 0x30000
    for entries in (
            [(a, a, 100), (a + 40, a + 40, 100)],               # in place, one inside the other
            [(a + 40, a + 40, 100), (a, a, 11)],
            [(a, c, 100), (b, c, 100)],                         # two gradients, one output
            [(a, a, 100), (b, a, 100)],
            [(a, a, 100), (a, a, 99)],                          # the same place, another size or type
            [(a, a, 100), (a, a, 100, 0)],
            [(a, a + 4, 100)],                                  # shifted onto itself
            [(a, b, 100), (b, a, 100)],                         # exchanged
            [(a, b, 100), (b, c, 100), (c, a, 100)],
            [(b, c, 100), (a, b, 100), (c + 200, c + 4000, 100), (c + 4000, a, 9)]):
        assert "overlap" in clip(L, *entries), entries


def test_clip_takes_what_has_an_order(L):
    a, b, c = 0x10000, 0x20000, 0x30000
    for entries in (
            [(a, a, 100), (a, a, 100)],                         # tied weights
            [(b, b, 100), (a, a, 100), (b, b, 100), (a, a, 100)],
            [(a, b, 100), (a, b, 100)],
            [(a, b, 100), (a, c, 100)],                         # one gradient, two outputs
            [(a, a, 100), (a + 40, b, 10)],                     # one reads what another scales in place
            [(a + 40, b, 10), (a, a, 100), (a + 80, c, 10)],
            [(c, c, 5), (b, b, 0), (a, a, 100), (b, b, 7)],     # in place in any order of addresses
            [(a, a, 100), (a + 400, a + 400, 100)],             # side by side
            [(a, c, 100), (b, c + 400, 100), (c + 1000, c + 800, 50)]):
        assert "workspace" in clip(L, *entries), entries


def meta(*shape, dt=torch.bfloat16):
    return torch.empty(*shape, dtype=dt, device="meta")


def test_fake_gradients_have_the_strides_that_the_kernels_write(rq):
    """Row-major, also where an operand is a transposed view."""
    x, w = meta(2, 16, 6).transpose(1, 2), meta(16, 5).t()
    dx, dw, db = torch.ops.rwkvq.linear_act_backward(meta(2, 6, 5), x, w, None, 0, 0, True, torch.bfloat16)
    assert dx.shape == x.shape and dx.is_contiguous()
    assert dw.shape == w.shape and dw.is_contiguous() and db.shape == (5,)
    y, _ = torch.ops.rwkvq.linear_act(x, w, None, None, 0)
    assert y.is_contiguous()
    x.requires_grad_(), w.requires_grad_()
    y = rq.linear_act(x, w, None, "gelu")
    dx, dw = torch.autograd.grad(y, (x, w), meta(5, 2, 6).permute(1, 2, 0))
    assert dx.is_contiguous() and dw.is_contiguous()
    table = meta(4, 9).t().requires_grad_()
    de, = torch.autograd.grad(rq.embedding(meta(3, dt=torch.int64), table), table, meta(4, 3).t())
    assert de.shape == (9, 4) and de.is_contiguous()


def test_compiled_calls_are_recorded_whole(rq):
    """One graph, without a break, forward and backward."""
    def step(idx, table, x, w):
        h = rq.embedding(idx, table, 2.0)
        return rq.linear_act(x.transpose(0, 1), w.t(), None, "silu", h)

    args = [meta(7, dt=torch.int64), meta(9, 5), meta(6, 7), meta(6, 5)]
    for t in args[1:]:
        t.requires_grad_()
    y = torch.compile(step, backend="aot_eager", fullgraph=True)(*args)
    grads = torch.autograd.grad(y, args[1:], meta(7, 5))
    # row-major gradients of the transposed views, seen from behind the transposition
    assert [g.stride() for g in grads] == [(5, 1), (1, 6), (1, 6)]


def test_the_recorded_op_keeps_slopes_only_for_gradients_that_take_them(rq, monkeypatch):
    seen = []
    op = rq.train._linear_op
    monkeypatch.setattr(rq.train, "_linear_op", lambda *a: seen.append(op(*a)) or seen[-1])
    x, w, b, r = meta(6, 8), meta(5, 8), meta(5), meta(6, 5)

    def slopes(grads=()):
        for t in (x, w, b, r):
            t.requires_grad_(any(t is g for g in grads))
        y = rq.linear_act(x, w, b, "silu", r)
        return y, seen[-1][1].numel()

    assert slopes()[1] == 0 and slopes([r])[1] == 0
    for t in (x, w, b):
        assert slopes([t])[1] == 30
    with torch.no_grad():
        assert slopes([x, w])[1] == 0
    y, _ = slopes([r])
    assert torch.autograd.grad(y, r, meta(6, 5))[0].shape == (6, 5)
    y, _ = op(x, w.requires_grad_(), b, r, 3, False)
    with pytest.raises(RuntimeError, match="want_slope"):
        torch.autograd.grad(y, w, meta(6, 5))


def test_the_recorded_op_materialises_no_gradient_of_its_slopes(rq):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Calls(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            names.append(str(func))
            return func(*args, **(kwargs or {}))

    names = []
    w = meta(5, 8).requires_grad_()
    y, slope = torch.ops.rwkvq.linear_act(meta(6, 8), w, None, None, 3)
    assert slope.numel() == 30
    with Calls():
        torch.autograd.grad(y, w, meta(6, 5))
    assert any("linear_act_backward" in n for n in names) and not any("zeros" in n for n in names), names


def kept(fn):
    """What a call saves for its backward pass."""
    ts = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: ts.append(t) or t, lambda t: t):
        y = fn()
    return y, ts


def test_only_what_the_gradients_read_is_kept_by_the_recorded_op(rq):
    x, w, b = meta(6, 8), meta(5, 8), meta(5)
    for needs, shapes in (((x,), {(5, 8), (6, 5)}), ((w,), {(6, 8), (6, 5)}), ((b,), {(6, 5)}),
                          ((x, w, b), {(5, 8), (6, 8), (6, 5)})):
        for t in (x, w, b):
            t.requires_grad_(any(t is n for n in needs))
        for name in ("silu", "relu"):       # slopes, and y
            y, ts = kept(lambda: rq.linear_act(x, w, b, name))
            assert {tuple(t.shape) for t in ts} == shapes and len(ts) == len(shapes)
            grads = torch.autograd.grad(y, needs, meta(6, 5))
            assert [g.shape for g in grads] == [t.shape for t in needs]
        y, ts = kept(lambda: rq.linear_act(x, w, b))
        assert {tuple(t.shape) for t in ts} == shapes - {(6, 5)}
        torch.autograd.grad(y, needs[:1], meta(6, 5))


def test_the_largest_vocabulary_of_a_table_gradient(L):
    assert L.rq_embed_grad_workspace_bytes(1, 2 ** 30, 8) > 0
    assert L.rq_embed_grad_workspace_bytes(1, 2 ** 30 + 1, 8) == -1 and "2^30" in err(L)
    assert L.rq_embed_grad(P, 8, 1, P, 0, 2 ** 30 + 1, 8, 1.0, -1, P, P, 1 << 40, None) == -1 and "2^30" in err(L)


def test_embedding_over_a_table_that_is_there(rq):
    """The constructor of nn.Embedding that the module inherits."""
    t = torch.randn(10, 4, dtype=torch.bfloat16)
    e = rq.ScaledEmbedding.from_pretrained(t, padding_idx=-1, scale=3.0)
    assert type(e) is rq.ScaledEmbedding and e.scale == 3.0 and e.padding_idx == 9
    assert e.weight.data_ptr() == t.data_ptr() and not e.weight.requires_grad
    assert rq.ScaledEmbedding.from_pretrained(t, freeze=False).weight.requires_grad
    with pytest.raises(ValueError, match="2-D"):
        rq.ScaledEmbedding.from_pretrained(t[0])
