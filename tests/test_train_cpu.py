"""Host logic of rwkvq.train and the argument checks of its C entry points,
without a GPU: nothing here reaches a launch."""
import ctypes
import os
import re

import pytest
import torch

from train_ref import act

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
    text = open(os.path.join(ROOT, "include", "rwkvq_train.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    names = set(re.findall(r"^\s*\w+\s+(rq_\w+)\s*\(", text, flags=re.M))
    assert names == {"rq_linear_slope", "rq_linear_workspace_bytes", "rq_linear",
                     "rq_linear_backward_workspace_bytes", "rq_linear_backward", "rq_embed", "rq_embed_grad_workspace_bytes",
                     "rq_embed_grad", "rq_grad_norm_workspace_bytes", "rq_grad_norm", "rq_clip_grads"}
    for name in names:
        assert hasattr(L, name) and name in _lib.SIGNATURES
    assert ctypes.sizeof(_lib.RqGrad) == 32


def test_linear_refusals(L):
    def fwd(x=P, w=P, b=0, dt=0, r=0, ydt=0, m=4, n=8, k=16, a=0, y=P, s=0, ws=0, nb=0):
        return L.rq_linear(x, w, b, dt, r, ydt, m, n, k, a, y, s, ws, nb, None)

    for kw, text in (({"dt": 3}, "dtype"), ({"ydt": 1}, "y must have"), ({"m": -1}, "negative"),
                     ({"a": 7}, "activation"), ({"x": 0}, "NULL"), ({"w": 0}, "NULL"), ({"y": 0}, "NULL"),
                     ({"s": P}, "keeps no slopes"), ({"s": P, "a": 1}, "keeps no slopes"),
                     ({"n": 2 ** 40}, "more than")):
        assert fwd(**kw) == -1 and text in err(L), (kw, err(L))
    for name in ("x", "w", "b", "r", "y"):
        assert fwd(**{name: P + 2}) == -2 and "aligned" in err(L)
    assert fwd(m=0, x=0, w=0, y=0) == 0 and fwd(n=0, y=0) == 0
    def bwd(dy=P, ydt=0, s=0, kind=0, a=0, x=P, w=P, dt=0, m=4, n=8, k=16, dx=P, dw=P, db=0, ws=0, nb=0):
        return L.rq_linear_backward(dy, ydt, s, kind, a, x, w, dt, m, n, k, dx, dw, db, ws, nb, None)

    for kw, text in (({"dt": 3}, "dtype"), ({"ydt": 1}, "dy must have"), ({"m": -1}, "negative"),
                     ({"a": -1}, "activation"), ({"kind": 5}, "slope kind"), ({"kind": 1, "s": P, "a": 3}, "slope of"),
                     ({"kind": 2, "a": 3}, "NULL"), ({"dy": 0}, "NULL"), ({"x": 0}, "NULL"), ({"w": 0}, "NULL"),
                     ({"db": P}, "workspace"), ({"kind": 2, "s": P, "a": 3}, "workspace"), ({"ydt": 2}, "workspace")):
        assert bwd(**kw) == -1 and text in err(L), (kw, err(L))
    for name in ("dy", "x", "w", "dx", "dw", "db"):
        assert bwd(**{name: P + 8}) == -2
    assert bwd(dx=0, dw=0) == 0 and bwd(n=0, dx=0) == 0 and bwd(k=0) == 0
    need = L.rq_linear_backward_workspace_bytes(100, 33, 64, 0, 2, 0, 1, 1, 1)
    assert need >= 100 * 33 * 2 + 4 * 33 * 4     # g and the four partial sums of db
    assert L.rq_linear_backward_workspace_bytes(64, 64, 64, 0, 0, 0, 1, 0, 0) == 0
    assert L.rq_linear_backward_workspace_bytes(64, 64, 64, 0, 1, 0, 1, 0, 0) == -1
    assert L.rq_linear_workspace_bytes(-1, 1, 1, 0) == -1


def test_where_the_backward_pass_takes_the_slope_from(L):
    none, of_y, f16, f32, wide16 = range(5)
    for dt in range(3):
        assert L.rq_linear_slope(0, dt, 1) == none
        assert L.rq_linear_slope(1, dt, 0) == of_y
        assert L.rq_linear_slope(2, dt, 0) == (wide16, f32, of_y)[dt]
        assert L.rq_linear_slope(2, dt, 1) == (wide16, f32, f32)[dt]
        for a in (1, 3, 4, 5, 6):
            assert L.rq_linear_slope(a, dt, 1) == (f16 if dt == 0 else f32)
    assert L.rq_linear_slope(7, 0, 0) == -1 and L.rq_linear_slope(0, 9, 0) == -1


def test_embedding_refusals(L):
    assert L.rq_embed(P, 3, 1, P, 0, 5, 8, 1.0, P, None) == -1 and "4 or 8 bytes" in err(L)
    assert L.rq_embed(P, 8, 1, P, 3, 5, 8, 1.0, P, None) == -1
    assert L.rq_embed(P, 8, -1, P, 0, 5, 8, 1.0, P, None) == -1 and "negative" in err(L)
    assert L.rq_embed(0, 8, 1, P, 0, 5, 8, 1.0, P, None) == -1 and "NULL" in err(L)
    assert L.rq_embed(P, 8, 1, 0, 0, 5, 8, 1.0, P, None) == -1
    assert L.rq_embed(P, 8, 1, P + 1, 0, 5, 8, 1.0, P, None) == -2
    assert L.rq_embed(P + 4, 8, 1, P, 0, 5, 8, 1.0, P, None) == -2
    assert L.rq_embed(0, 8, 0, 0, 0, 5, 8, 1.0, 0, None) == 0
    need = L.rq_embed_grad_workspace_bytes(100, 5, 8)
    assert need > 800
    assert L.rq_embed_grad(P, 8, 100, P, 0, 5, 8, 1.0, -1, P, P, need - 1, None) == -1 and "workspace" in err(L)
    assert L.rq_embed_grad(P, 8, 100, P, 0, 5, 8, 1.0, -1, 0, P, need, None) == -1 and "NULL" in err(L)
    assert L.rq_embed_grad(P, 8, 100, P, 0, 5, 8, 1.0, -1, P, P + 8, need, None) == -2
    assert L.rq_embed_grad(P, 8, 2 ** 31, P, 0, 5, 8, 1.0, -1, P, P, need, None) == -1
    assert L.rq_embed_grad(P, 8, 100, P, 0, 0, 8, 1.0, -1, 0, 0, 0, None) == 0
    assert L.rq_embed_grad_workspace_bytes(-1, 5, 8) == -1
    assert L.rq_embed_grad_workspace_bytes(1, 2 ** 31, 8) == -1


def test_clip_refusals(L):
    from rwkvq._lib import RqGrad
    ok = RqGrad(P, P, 100, 0, 0)

    def clip(*ts, norm=P, ws=P, nb=1 << 20, top=1.0, eps=0.0, count=None):
        a = (RqGrad * max(1, len(ts)))(*ts)
        return L.rq_clip_grads(ctypes.addressof(a), len(ts) if count is None else count, top, eps, norm,
                               ws, nb, None)

    assert clip(RqGrad(P, P, 100, 3, 0)) == -1 and "dtype" in err(L)
    assert clip(RqGrad(P, P, -1, 0, 0)) == -1 and "negative" in err(L)
    assert clip(RqGrad(0, P, 1, 0, 0)) == -1 and clip(RqGrad(P, 0, 1, 0, 0)) == -1 and "NULL" in err(L)
    assert clip(ok, RqGrad(P + 2, P, 1, 2, 0)) == -2 and "tensor 1" in err(L)
    assert clip(ok, count=-1) == -1
    assert clip(ok, norm=0) == -1 and clip(ok, norm=P + 2) == -2
    assert clip(ok, nb=7) == -1 and "8 bytes" in err(L)
    assert clip(ok, top=-1.0) == -1 and clip(ok, top=float("nan")) == -1 and clip(ok, eps=-1.0) == -1
    a = (RqGrad * 2)(ok, RqGrad(P, P, 16384 * 5000, 2, 0))
    assert L.rq_grad_norm_workspace_bytes(ctypes.addressof(a), 2) == 8 * 1024
    assert L.rq_grad_norm_workspace_bytes(0, 0) == 0 and L.rq_grad_norm_workspace_bytes(0, 1) == -1


def meta(*shape, dt=torch.bfloat16):
    return torch.empty(*shape, dtype=dt, device="meta")


def test_python_refusals(rq):
    x, w = torch.zeros(3, 8), torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="GPU"):
        rq.linear_act(x, w)
    with pytest.raises(RuntimeError, match="GPU"):
        rq.embedding(torch.zeros(3, dtype=torch.int64), w)
    with pytest.raises(RuntimeError, match="GPU"):
        rq.clip_grad_norm([x], 1.0)
    with pytest.raises(RuntimeError, match="GPU"):
        rq.grad_norm([x])
    for bad, text in (((x, w, None, "swish"), "activation"), ((x, meta(4, 9)), "inner dimension"),
                      ((x, meta(8)), "2-D"), ((x.int(), w), "bfloat16"), ((x, w, meta(5)), "bias"),
                      ((x, w, None, None, meta(3, 5)), "residual"), ((x, w, None, None, meta(4)), "residual")):
        with pytest.raises(ValueError, match=text):
            rq.linear_act(*bad)
    with pytest.raises(ValueError, match="integer"):
        rq.embedding(x, w)
    with pytest.raises(ValueError, match="2-D"):
        rq.embedding(torch.zeros(3, dtype=torch.int64), meta(4))
    with pytest.raises(ValueError, match="padding_idx"):
        rq.embedding(torch.zeros(3, dtype=torch.int64), w, padding_idx=4)
    with pytest.raises(ValueError, match="negative"):
        rq.clip_grad_norm([x], -1.0)
    with pytest.raises(ValueError, match="negative"):
        rq.clip_grad_norm_([], float("nan"))
    with pytest.raises(ValueError, match="2 tensors for 1"):
        rq.clip_grad_norm([x], 1.0, out=[x, x])
    with pytest.raises(ValueError, match="bfloat16"):
        rq.grad_norm([x.int()])
    with pytest.raises(ValueError, match="tensors"):
        rq.train._check_grads([1.0])
    with pytest.raises(ValueError, match="activation"):
        rq.LinearAct(4, 4, activation="elu")


def test_shapes_and_dtypes_on_meta_tensors(rq):
    y = rq.linear_act(meta(2, 3, 8), meta(5, 8), meta(5), "gelu", meta(2, 3, 5, dt=torch.float32))
    assert y.shape == (2, 3, 5) and y.dtype == torch.float32
    assert rq.linear_act(meta(8), meta(5, 8)).dtype == torch.bfloat16
    assert rq.linear_act(meta(3, 8, dt=torch.float16), meta(5, 8)).dtype == torch.float32
    assert rq.embedding(meta(2, 3, dt=torch.int64), meta(7, 4), 2.0).shape == (2, 3, 4)
    _, slope = torch.ops.rwkvq.linear_act(meta(3, 8), meta(5, 8), None, None, 4)
    assert slope.shape == (3, 5) and slope.dtype == torch.float16


def test_no_gradients(rq):
    assert rq.grad_norm([]).item() == 0
    assert rq.clip_grad_norm([], 1.0)[0] == []
    assert rq.clip_grad_norm_([torch.nn.Parameter(torch.ones(3))], 1.0).item() == 0


def test_dense_memory_in_any_order(rq):
    from rwkvq.train import _dense
    t = torch.zeros(4, 6, 8)
    assert _dense(t) and _dense(t.permute(2, 0, 1)) and _dense(t[:1].transpose(1, 2))
    assert not _dense(t[:, ::2]) and not _dense(t[:, :, :5]) and not _dense(torch.zeros(1).expand(4))
    assert _dense(torch.zeros(0, 4)) and _dense(torch.zeros(()))


def test_modules(rq):
    lin = torch.nn.Linear(8, 6, bias=False)
    m = rq.LinearAct.from_linear(lin, "tanh")
    assert m.weight is lin.weight and m.bias is None and "tanh" in repr(m)
    assert set(rq.LinearAct(8, 6).state_dict()) == {"weight", "bias"}
    e = rq.ScaledEmbedding(10, 4, scale=2.0, padding_idx=3)
    assert "scale=2.0" in repr(e) and set(e.state_dict()) == {"weight"}


@pytest.mark.parametrize("name", (None, "relu", "relu2", "silu", "gelu", "sigmoid", "tanh"))
def test_the_reference_slopes_against_differences(name):
    v = torch.linspace(-6, 6, 4001, dtype=torch.float64) + 1e-3
    h = 1e-5
    up, down = act(name, v + h)[0], act(name, v - h)[0]
    assert ((up - down) / (2 * h) - act(name, v)[1]).abs().max() < 1e-8
