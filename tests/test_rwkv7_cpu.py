"""Argument checks of the C entry points of the recurrence and the sampler, without a GPU: nothing here reaches a
launch."""
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 0x1000  # never dereferenced: validation fails first


@pytest.fixture(scope="module")
def L():
    from rwkvq import _lib
    return _lib.lib()


def err(L):
    return L.rq_last_error().decode()


def test_every_declared_entry_point_is_exported_and_bound(L):
    from rwkvq import _lib
    text = open(os.path.join(ROOT, "include", "rwkvq_rwkv7.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    names = set(re.findall(r"^\s*\w+\s+(rq_\w+)\s*\(", text, flags=re.M))
    assert names == {"rq_wkv7", "rq_wkv7_backward", "rq_wkv7_step", "rq_wkv7_chunks",
                     "rq_wkv7_workspace_bytes", "rq_wkv7_backward_workspace_bytes", "rq_sample"}
    for name in names:
        assert hasattr(L, name) and name in _lib.SIGNATURES


def test_chunks_and_workspaces(L):
    assert L.rq_wkv7_chunks(3, 33, 3, 0) == 9 and L.rq_wkv7_chunks(1, 33, 4, 1) == 6
    assert L.rq_wkv7_chunks(2, 33, 4, 1) == -1 and L.rq_wkv7_chunks(2, 33, 3, 0) == -1
    assert L.rq_wkv7_chunks(-1, 33, -1, 0) == -1 and "negative" in err(L)
    assert L.rq_wkv7_chunks(0, 5, 0, 0) == 0
    assert L.rq_wkv7_backward_workspace_bytes(1, 16, 2, 1, 0) == 0
    assert L.rq_wkv7_backward_workspace_bytes(1, 2 ** 30, 64, 1, 0) == -1 and "heads of chunks" in err(L)
    # few heads over many tokens run in segments, which take room for 3 states each; many heads do not
    one = 3 * 4 * 64 * 64
    assert L.rq_wkv7_workspace_bytes(1, 16, 12, 1, 0) == 0 and L.rq_wkv7_workspace_bytes(8, 512, 32, 8, 0) == 0
    for args in ((1, 8192, 12, 1, 0), (1, 2047, 32, 1, 0), (1, 8192, 12, 3, 1)):
        n = L.rq_wkv7_workspace_bytes(*args)
        assert n > 0 and n % (one * args[2]) == 0
    assert L.rq_wkv7_workspace_bytes(2, 1, 1, 1, 0) == -1


def test_packed_sequences_never_share_a_chunk():
    """Sequence n begins at chunk start / 16 + n: its chunks end before the next one's."""
    g = torch.Generator().manual_seed(0)
    for _ in range(300):
        lens = torch.randint(0, 40, (int(torch.randint(1, 12, (1,), generator=g)),), generator=g).tolist()
        start, free = 0, 0
        for n, length in enumerate(lens):
            first = start // 16 + n
            assert first >= free
            free = first + -(-length // 16)
            start += length
        assert free <= start // 16 + len(lens)


def test_scan_refusals(L):
    def fwd(x=P, dt=0, batch=1, time=4, heads=2, cu=0, seqs=1, state=0, y=P, ydt=0, so=0, st=0, sa=0, w=P, ws=0, nb=0):
        return L.rq_wkv7(x, w, x, x, x, x, dt, batch, time, heads, cu, seqs, state, y, ydt, so, st, sa, ws, nb, None)

    for kw, text in (({"dt": 3}, "dtype"), ({"ydt": 1}, "y must have"), ({"time": -1}, "negative"), ({"x": 0}, "NULL"),
                     ({"y": 0}, "NULL"), ({"w": 0}, "NULL"), ({"seqs": 2}, "seqs"), ({"cu": P, "batch": 2}, "batch of 1"),
                     ({"cu": P, "seqs": 0}, "no sequence"), ({"st": P}, "together"), ({"sa": P}, "together"),
                     ({"time": 2 ** 31}, "2^31"), ({"batch": 2 ** 20, "seqs": 2 ** 20, "heads": 64}, "heads of sequences"),
                     ({"time": 2 ** 30, "heads": 64, "st": P, "sa": P}, "heads of chunks"),
                     ({"time": 2 ** 16}, "workspace"), ({"time": 2 ** 16, "ws": P, "nb": 64}, "workspace")):
        assert fwd(**kw) == -1 and text in err(L), (kw, err(L))
    for kw in ({"x": P + 2}, {"w": P + 8}, {"y": P + 4}, {"state": P + 8}, {"so": P + 4}, {"st": P + 4, "sa": P}, {"ws": P + 8},
               {"cu": P + 2}):
        assert fwd(**kw) == -2 and "aligned" in err(L), kw
    assert fwd(heads=0) == 0 and fwd(batch=0, seqs=0) == 0


def test_backward_refusals(L):
    need = L.rq_wkv7_backward_workspace_bytes(1, 4000, 2, 1, 0)
    assert need > 0

    def bwd(x=P, dt=0, batch=1, time=4000, heads=2, cu=0, seqs=1, st=P, sa=P, dy=P, ydt=0, dso=0, g=P, ds=0, ws=P, nb=need):
        return L.rq_wkv7_backward(x, x, x, x, x, x, dt, batch, time, heads, cu, seqs, st, sa, dy, ydt, dso, g, g, g, g,
                                  g, g, ds, ws, nb, None)

    for kw, text in (({"dt": -1}, "dtype"), ({"ydt": 1}, "y must have"), ({"heads": -1}, "negative"), ({"x": 0}, "NULL"),
                     ({"st": 0}, "NULL"), ({"sa": 0}, "NULL"), ({"dy": 0}, "NULL"), ({"ws": 0}, "workspace"),
                     ({"nb": need - 1}, "workspace"), ({"cu": P, "seqs": 0}, "no sequence")):
        assert bwd(**kw) == -1 and text in err(L), (kw, err(L))
    for kw in ({"x": P + 2}, {"g": P + 2}, {"dso": P + 8}, {"ds": P + 4}, {"ws": P + 4}):
        assert bwd(**kw) == -2 and "aligned" in err(L), kw
    assert bwd(heads=0) == 0


def test_step_refusals(L):
    def step(x=P, dt=0, batch=1, heads=2, state=P, y=P, ydt=0, so=P):
        return L.rq_wkv7_step(x, x, x, x, x, x, dt, batch, heads, state, y, ydt, so, None)

    for kw, text in (({"dt": 7}, "dtype"), ({"ydt": 1}, "y must have"), ({"batch": -1}, "negative"), ({"x": 0}, "NULL"),
                     ({"y": 0}, "NULL"), ({"batch": 2 ** 21, "heads": 2}, "heads of sequences")):
        assert step(**kw) == -1 and text in err(L), (kw, err(L))
    for kw in ({"x": P + 2}, {"state": P + 8}, {"so": P + 8}, {"y": P + 2}):
        assert step(**kw) == -2 and "aligned" in err(L), kw
    assert step(batch=0) == 0


def test_sampler_refusals(L):
    def call(x=P, dt=0, rows=2, vocab=10, u=P, t=0, ta=1.0, k=0, ka=0, p=0, pa=1.0, m=0, ma=0.0, token=P, lp=0):
        return L.rq_sample(x, dt, rows, vocab, u, t, ta, k, ka, p, pa, m, ma, token, lp, None)

    nan = float("nan")
    for kw, text in (({"dt": 3}, "dtype"), ({"rows": -1}, "negative"), ({"vocab": -1}, "negative"), ({"vocab": 0}, "without a logit"),
                     ({"vocab": 2 ** 20 + 1}, "vocabulary"), ({"rows": 2 ** 21 + 1}, "rows"), ({"ta": -0.5}, "temperature"),
                     ({"ta": nan}, "temperature"), ({"ka": -1}, "top_k"), ({"pa": 0.0}, "top_p"), ({"pa": 1.25}, "top_p"),
                     ({"pa": nan}, "top_p"), ({"ma": -1.0}, "min_p"), ({"ma": 1.5}, "min_p"), ({"x": 0}, "NULL"),
                     ({"u": 0}, "NULL"), ({"token": 0}, "NULL")):
        assert call(**kw) == -1 and text in err(L), (kw, err(L))
    for kw in ({"x": P + 1}, {"x": P + 2, "dt": 2}, {"u": P + 2}, {"t": P + 1}, {"k": P + 4}, {"p": P + 2}, {"m": P + 2},
               {"token": P + 4}, {"lp": P + 2}):
        assert call(**kw) == -2 and "aligned" in err(L), kw
    assert call(rows=0, x=0, u=0, token=0) == 0


def test_no_cpu_path():
    import rwkvq
    six = [torch.zeros(1, 2, 1, 64) for _ in range(6)]
    with pytest.raises(RuntimeError, match="no CPU"):
        rwkvq.wkv7(*six)
    with pytest.raises(RuntimeError, match="no CPU"):
        rwkvq.wkv7_step(*[x[:, 0] for x in six], torch.zeros(1, 1, 64, 64))
    with pytest.raises(RuntimeError, match="no CPU"):
        rwkvq.sample(torch.zeros(2, 5), torch.zeros(2))
