"""The recurrence's C entry points between guards: nothing around the tensors is written to, and what is written is what the
Python entry points give."""
import pytest
import torch

from wkv_ref import D, DT, inputs

pytestmark = pytest.mark.gpu

GUARD = 4096   # bytes on either side


class Guarded:
    """Tensors in one allocation each, between bytes that are looked at afterwards."""

    def __init__(self, dev):
        self.dev, self.all = dev, []

    def __call__(self, shape, dtype):
        n = torch.Size(shape).numel() * dtype.itemsize
        memory = torch.full((n + 2 * GUARD,), 0xa5, dtype=torch.uint8, device=self.dev)
        self.all.append((memory, n))
        return memory[GUARD:GUARD + n].view(dtype).view(shape)

    def whole(self):
        return all((m[:GUARD] == 0xa5).all() and (m[GUARD + n:] == 0xa5).all() for m, n in self.all)


# boundaries that decrease, lie outside, repeat; and orderly ones; whole and in segments
CASES = [(30, 2, [25, 3, 28, 1, 30, 0]), (30, 2, [-5, 10, 10, 2 ** 31 - 1]), (900, 2, [850, 3, 700, -1, 2 ** 31 - 1, 0, 899]),
         (900, 1, [899, 0, 900]), (900, 2, [0, 900, 0, 900]), (901, 2, [0, 450, 450, 901]), (37, 3, [2, 20, 33]), (1024, 1, None),
         (17, 3, None), (1, 2, None), (385, 1, [384, 385, 384])]


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("i", range(len(CASES)))
def test_nothing_around_the_tensors_is_touched(rq, dev, i, dt):
    time, heads, cu = CASES[i]
    print(f"wkv7 guards time={time} heads={heads} cu={cu} {dt}", flush=True)
    L, code, one = rq._lib.lib(), rq._lib.DTYPE_CODE[DT[dt]], DT[dt]
    g, at = torch.Generator().manual_seed(500 + i), Guarded(dev)
    seqs = 1 if cu is None else len(cu) - 1
    six = [at(x.shape, one).copy_(x) for x in inputs(g, 1, time, heads, dtype=one)]
    state, dlast = (at((seqs, heads, D, D), torch.float32).copy_(torch.randn(seqs, heads, D, D, generator=g)) for _ in range(2))
    dy = at((1, time, heads, D), one).copy_(torch.randn(1, time, heads, D, generator=g))
    bounds = None if cu is None else at((len(cu),), torch.int32).copy_(torch.tensor(cu, dtype=torch.int32))
    chunks = L.rq_wkv7_chunks(1, time, seqs, int(cu is not None))
    y, last = at((1, time, heads, D), one), at((seqs, heads, D, D), torch.float32)
    states, sa = at((chunks, heads, D, D), torch.float32), at((chunks, heads, 16, D), torch.float32)
    need = L.rq_wkv7_workspace_bytes(1, time, heads, seqs, int(cu is not None))
    ws = at((need,), torch.uint8)
    stream = torch.cuda.current_stream(dev).cuda_stream
    cup = 0 if cu is None else bounds.data_ptr()

    def p(x):
        return x.data_ptr() if x.numel() else 0

    inputs_before = [x.clone() for x in (*six, state, dlast, dy)]
    rc = L.rq_wkv7(*map(p, six), code, 1, time, heads, cup, seqs, p(state), p(y), code, p(last), p(states), p(sa), p(ws), need, stream)
    assert rc == 0, L.rq_last_error()
    need = L.rq_wkv7_backward_workspace_bytes(1, time, heads, seqs, int(cu is not None))
    ws = at((need,), torch.uint8)
    grads, dstate = [at(x.shape, one) for x in six], at(state.shape, torch.float32)
    rc = L.rq_wkv7_backward(*map(p, six), code, 1, time, heads, cup, seqs, p(states), p(sa), p(dy), code, p(dlast),
                            *map(p, grads), p(dstate), p(ws), need, stream)
    assert rc == 0, L.rq_last_error()
    torch.cuda.synchronize()
    assert at.whole()
    for x, z in zip((*six, state, dlast, dy), inputs_before):
        assert torch.equal(x, z)
    inside = [0, time] if cu is None else [min(max(x, 0), time) for x in cu]
    if inside == sorted(inside):   # else the results are undefined
        leaves = [x.clone().requires_grad_() for x in (*six, state)]
        want_y, want_last = rq.wkv7(*leaves[:6], leaves[6], cu_seqlens=bounds)
        want = torch.autograd.grad([want_y, want_last], leaves, [dy, dlast])
        assert torch.equal(y, want_y) and torch.equal(last, want_last)
        for x, z in zip((*grads, dstate), want):
            assert torch.equal(x, z)


def test_a_step_between_guards(rq, dev):
    L, g = rq._lib.lib(), torch.Generator().manual_seed(9)
    for dt in DT.values():
        at, code = Guarded(dev), rq._lib.DTYPE_CODE[dt]
        six = [at(x.shape, dt).copy_(x) for x in inputs(g, 5, 3, dtype=dt)]
        state, last = at((5, 3, D, D), torch.float32).fill_(0.25), at((5, 3, D, D), torch.float32)
        y = at((5, 3, D), dt)
        rc = L.rq_wkv7_step(*[x.data_ptr() for x in six], code, 5, 3, state.data_ptr(), y.data_ptr(), code, last.data_ptr(),
                            torch.cuda.current_stream(dev).cuda_stream)
        assert rc == 0
        torch.cuda.synchronize()
        assert at.whole()
        want, new = rq.wkv7_step(*six, state)
        assert torch.equal(y, want) and torch.equal(last, new)
