"""What tracing and compiling record of the recurrence and the sampler, on tensors without storage."""
import pytest
import torch


def meta(*shape, dt=torch.bfloat16):
    return torch.empty(*shape, dtype=dt, device="meta")


def token(batch=3, heads=2):
    return [meta(batch, heads, 64) for _ in range(6)], meta(batch, heads, 64, 64, dt=torch.float32)


def names(graph):
    return [n.kind() for n in graph.nodes() if n.kind().startswith("rwkvq::")]


def test_traced_steps_are_recorded(rq):
    six, state = token()
    f = torch.jit.trace(lambda *t: rq.wkv7_step(*t), (*six, state), check_trace=False)
    assert names(f.inlined_graph) == ["rwkvq::wkv7_step"]
    f = torch.jit.trace(lambda *t: rq.wkv7_step(*t, out=t[6])[0], (*six, state), check_trace=False)
    assert names(f.inlined_graph) == ["rwkvq::wkv7_step_out"]
    other = torch.empty_like(state)
    f = torch.jit.trace(lambda *t: rq.wkv7_step(*t[:7], out=t[7])[0], (*six, state, other), check_trace=False)
    assert names(f.inlined_graph) == ["rwkvq::wkv7_step_out"]


def test_shapes_and_types_of_recorded_steps(rq):
    six, state = token()
    y, new = rq.wkv7_step(*six, state)
    assert y.shape == (3, 2, 64) and y.dtype == torch.bfloat16 and new.shape == state.shape and new is not state
    y, new = rq.wkv7_step(*six, state, out=state, out_dtype=torch.float32)
    assert y.dtype == torch.float32 and new is state
    six[2] = six[2].float()
    assert rq.wkv7_step(*six, state)[0].dtype == torch.float32
    # without gradients
    six = [x.requires_grad_() for x in token()[0]]
    y, new = rq.wkv7_step(*six, state)
    assert not y.requires_grad and not new.requires_grad


def test_compiled_decoding_is_recorded_whole(rq):
    """A prompt, a step in place, one to a new state and a token in one graph, without a break."""
    def decode(prompt, tok, state, logits, u):
        y, last = rq.wkv7(*prompt, state)
        y1, _ = rq.wkv7_step(*tok, last, out=last)
        y2, new = rq.wkv7_step(*tok, last)
        t, lp = rq.sample(logits, u, temperature=0.8, top_k=5)
        return y + y1[:, None] + y2[:, None], new, t, lp

    tok, state = token()
    prompt = [meta(3, 7, 2, 64) for _ in range(6)]
    args = (prompt, tok, state, meta(3, 99), meta(3, dt=torch.float32))
    with torch.no_grad():
        y, new, t, lp = torch.compile(decode, backend="aot_eager", fullgraph=True)(*args)
    assert y.shape == (3, 7, 2, 64) and new.shape == state.shape and t.dtype == torch.int64 and lp.shape == (3,)


def test_compiled_updates_reach_the_state(rq):
    """In place on an argument: the graph writes it back."""
    tok, state = token()
    f = torch.compile(lambda s: rq.wkv7_step(*tok, s, out=s)[0], backend="aot_eager", fullgraph=True)
    before = state._version
    with torch.no_grad():
        assert f(state).shape == (3, 2, 64)
    assert state._version > before
    other = torch.empty_like(state)
    f = torch.compile(lambda s, o: rq.wkv7_step(*tok, s, out=o)[0], backend="aot_eager", fullgraph=True)
    with torch.no_grad():
        f(state, other)
    assert other._version > 0


def test_compiled_training_is_recorded_whole(rq):
    six = [meta(1, 20, 2, 64).requires_grad_() for _ in range(6)]
    state, cu = meta(2, 2, 64, 64, dt=torch.float32).requires_grad_(), meta(3, dt=torch.int32)
    y, last = torch.compile(lambda s, *t: rq.wkv7(*t, s, cu), backend="aot_eager", fullgraph=True)(state, *six)
    grads = torch.autograd.grad([y, last], [*six, state], [meta(*y.shape), meta(*last.shape, dt=torch.float32)])
    assert [g.shape for g in grads] == [t.shape for t in [*six, state]]
    assert [g.dtype for g in grads] == [t.dtype for t in [*six, state]]


def test_refusals_of_recorded_steps(rq):
    six, state = token()
    with pytest.raises(ValueError, match="out must be"):
        rq.wkv7_step(*six, state, out=state[:2])
    with pytest.raises(ValueError, match="batch, heads, 64"):
        rq.wkv7_step(*[x[0] for x in six], state)
    with pytest.raises(RuntimeError, match="only on a ROCm GPU"):
        rq.wkv7_step(*[torch.zeros(1, 1, 64)] * 6, torch.zeros(1, 1, 64, 64))


def test_forward_mode_is_refused(rq):
    """Of an operand with a tangent, whether or not anything requires gradients; the others run."""
    from torch.autograd import forward_ad
    six, state = token()
    seq = [meta(1, 9, 2, 64) for _ in range(6)]
    first, logits, u = meta(1, 2, 64, 64, dt=torch.float32), meta(3, 50), meta(3, dt=torch.float32)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.empty_like(t))

        for needs in (False, True):
            for i in (0, 1, 5):
                args = [x.detach().requires_grad_(needs) for x in seq]
                args[i] = dual(args[i])
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    rq.wkv7(*args)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            rq.wkv7(*seq, dual(first))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            rq.wkv7_step(*six[:3], dual(six[3]), *six[4:], state)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            rq.wkv7_step(*six, dual(state))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            rq.wkv7_step(*six, state, out=dual(torch.empty_like(state)))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            rq.sample(dual(logits), u)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            rq.sample(logits, u, temperature=dual(u))
        rq.wkv7(*seq, first)
        rq.wkv7_step(*six, state)
        rq.sample(logits, u)


def test_top_k_is_a_whole_number(rq, monkeypatch):
    logits, u = meta(3, 50), meta(3, dt=torch.float32)
    seen = []
    monkeypatch.setattr(rq.rwkv7, "_sample_op", lambda *a: seen.append(a[7]) or (u, u))
    for x, want in ((5, 5), (5.0, 5), (True, 1), (2 ** 80, 2 ** 62), (-3, -1), (-2 ** 80, -1)):
        rq.sample(logits, u, top_k=x)
        assert seen[-1] == want
    for x in (2.5, 0.9):
        with pytest.raises(ValueError, match="top_k must be an integer"):
            rq.sample(logits, u, top_k=x)
