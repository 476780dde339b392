"""The training-step operators on the GPU at their edges: shared memory,
saturated and non-finite values, parameters and modules, very long inputs.  The
bounds are those of tests/train_ref.py unless a test derives its own."""
import math

import pytest
import torch

from train_ref import U, U32, act, close

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "fp32": torch.float32}


# --------------------------------------------------------- dense products

def test_transposed_operands_under_compile(rq, dev):
    """A traced training step over transposed views: the planned strides are those
    that the kernels write."""
    g = torch.Generator().manual_seed(3)
    h = torch.randn(2, 64, 24, generator=g).to(torch.bfloat16).to(dev).requires_grad_()
    wt = (torch.randn(64, 40, generator=g) * 0.1).to(torch.bfloat16).to(dev).requires_grad_()
    dy = torch.randn(2, 24, 40, generator=g).to(torch.bfloat16).to(dev)

    def step(h, wt):
        y = rq.linear_act(h.transpose(1, 2), wt.t(), None, "silu")
        return y * 2

    want = torch.autograd.grad(step(h, wt), (h, wt), dy)
    traced = torch.compile(step, backend="aot_eager", fullgraph=True)
    for got, w in zip(torch.autograd.grad(traced(h, wt), (h, wt), dy), want):
        assert torch.equal(got, w)


def act64(name, v):
    """act(v) and act'(v); gelu's tail by erfc, which keeps its precision where the
    distribution function of torch.special.ndtr has become 0 (v below -8.3)."""
    if name != "gelu":
        return act(name, v)
    p = 0.5 * torch.special.erfc(-v / math.sqrt(2))
    return v * p, p + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)


def slopes_of(rq, dev, name, v):
    """act'(v) times 2^20 as one product with w = 1 gives it back: the slope's, g's and
    dx's roundings, and 64 fp32 units for the functions where their parts do not cancel."""
    x = v.to(torch.bfloat16)[:, None].to(dev).requires_grad_()
    w = torch.ones(1, 1, dtype=torch.bfloat16, device=dev)
    r = torch.zeros(len(v), 1, dtype=torch.float32, device=dev)
    dx, = torch.autograd.grad(rq.linear_act(x, w, None, name, r), x, torch.full_like(r, 2.0 ** 20))
    want = act64(name, x.detach().double().cpu())[1] * 2.0 ** 20
    return dx.double().cpu(), want, (3 * U[torch.bfloat16] + 64 * U32) * want.abs()


@pytest.mark.parametrize("name,lo,hi", [("sigmoid", -80, 80), ("tanh", -40, 40), ("silu", -80, -3), ("gelu", -13, -1.5)])
def test_slopes_of_saturated_values_beside_bf16(rq, dev, name, lo, hi):
    """Far below float16's range they keep bf16's precision."""
    got, want, bound = slopes_of(rq, dev, name, torch.linspace(lo, hi, 1000))
    close(got, want, bound, "slope")
    assert (want.abs() < 2.0 ** -20 * 2.0 ** -24).any()


def test_the_tail_of_gelu_in_float32(rq, dev):
    """v Phi(v) and its slope for negative v to fp32's relative precision: the tail is a
    product of factors that are each a few units off (24 in all); in the slope, for
    v < -1.5, its parts cancel by at most a factor of two."""
    for m in (3, 1000):    # both output stages
        v = torch.linspace(-13, -1.5, m)
        x = v[:, None].expand(m, 16).contiguous().to(dev).requires_grad_()
        y = rq.linear_act(x, torch.eye(16, device=dev), None, "gelu")
        dx, = torch.autograd.grad(y, x, torch.ones_like(y))
        a, s = act64("gelu", x.detach().double().cpu())
        close(y, a, 24 * U32 * a.abs(), "y")
        close(dx, s, 64 * U32 * s.abs(), "slope")


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("residual", ("", "fp32"))
@pytest.mark.parametrize("name", ("relu", "relu2"))
def test_nan_in_front_of_relu(rq, dev, name, residual, dt):
    """As through torch's relu: the gradient goes on through relu, and is NaN behind its
    square; rows without a NaN do not see it."""
    g = torch.Generator().manual_seed(5)
    for m, n in ((6, 40), (300, 136)):
        x, w = torch.randn(m, 64, generator=g), torch.randn(n, 64, generator=g)
        b, dy = torch.randn(n, generator=g), torch.randn(m, n, generator=g)
        x[2, 3] = float("nan")
        leaves = [t.to(DT[dt]).to(dev).requires_grad_() for t in (x, w, b)]
        r = torch.zeros(m, n, device=dev) if residual else None
        y = rq.linear_act(*leaves, name, r)
        got = torch.autograd.grad(y, leaves, dy.to(y.dtype).to(dev))
        plain = [t.detach().float().cpu().requires_grad_() for t in leaves]
        c = torch.relu(plain[0] @ plain[1].t() + plain[2])
        want = torch.autograd.grad(c if name == "relu" else c * c, plain, dy.to(y.dtype).float())
        for p, q in zip(got, want):
            assert torch.equal(p.isnan().cpu(), q.isnan())
        assert bool(got[0][2].isnan().all()) == (name == "relu2") and not got[0][3:].isnan().any()
        assert name == "relu2" or (got[0][2] != 0).any()


# ---------------------------------------------------------- gradient clip

@pytest.mark.parametrize("dt", DT)
def test_clip_scales_a_gradient_listed_twice_once(rq, dev, dt):
    """Tied weights: twice in the norm, one factor on the gradient."""
    print(f"clip of a gradient listed twice {dt}", flush=True)
    g = torch.Generator().manual_seed(1)
    tied = torch.randn(700, 333, generator=g).to(DT[dt]).to(dev)
    other = torch.randn(5000, generator=g).to(DT[dt]).to(dev)
    kept = [tied.clone(), other.clone()]
    want, same = rq.clip_grad_norm([*kept, kept[0].clone()], 2.0)   # three tensors of their own
    n = math.sqrt(2 * (tied.double() ** 2).sum().item() + (other.double() ** 2).sum().item())
    out, norm = rq.clip_grad_norm([tied, other, tied], 2.0, out=[tied, other, tied])
    assert abs(norm.item() - n) <= 2 * U32 * n and torch.equal(norm, same)
    for o, k in zip(out, want):
        assert torch.equal(o, k)
    p, q = torch.nn.Parameter(kept[0].clone()), torch.nn.Parameter(kept[0].clone())
    p.grad = q.grad = kept[0].clone()
    rq.clip_grad_norm_([p, q], 2.0)
    assert torch.equal(p.grad, rq.clip_grad_norm([kept[0], kept[0].clone()], 2.0)[0][0])


def test_clip_reads_a_gradient_before_it_is_scaled_in_place(rq, dev):
    g = torch.Generator().manual_seed(2)
    flat = torch.randn(300000, generator=g).to(dev)
    ts = [flat, flat[1000:2000], flat[250000:]]
    kept = [t.clone() for t in ts]
    want, _ = rq.clip_grad_norm(kept, 1.0)
    out, _ = rq.clip_grad_norm(ts, 1.0, out=[flat, torch.empty_like(kept[1]), torch.empty_like(kept[2])])
    for o, k in zip(out, want):
        assert torch.equal(o, k)
    with pytest.raises(ValueError, match="overlap"):
        rq.clip_grad_norm(ts, 1.0, out=ts)


# --------------------------------------------------- parameters and modules

def test_module_without_gradients_writes_only_its_output(rq, dev):
    """No slopes: the forward under no_grad allocates y, and so does one where only
    the residual has a gradient."""
    m = rq.LinearAct(64, 4096, activation="silu", device=dev, dtype=torch.float16)
    x = torch.randn(2048, 64, device=dev).to(torch.float16)
    r = torch.randn(2048, 4096, device=dev).to(torch.float16).requires_grad_()

    def peak(fn):
        fn()
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        y = fn()
        return torch.cuda.max_memory_allocated() - before, y

    with torch.no_grad():
        assert peak(lambda: m(x))[0] == 2 * 2048 * 4096
        assert peak(lambda: torch.ops.rwkvq.linear_act(x, m.weight, m.bias, None, 3, False)[0])[0] < 2.1 * 2048 * 4096
    m.requires_grad_(False)
    used, y = peak(lambda: m(x, r))
    assert used == 2 * 2048 * 4096
    dy = torch.ones_like(y)
    assert torch.equal(torch.autograd.grad(y, r, dy)[0], dy)


def test_parameters_take_the_direct_path(rq, dev, monkeypatch):
    """Modules and calls on their weights run the same code as plain tensors, not the
    registered ops; other subclasses do not."""
    class Other(torch.Tensor):
        pass

    g = torch.Generator().manual_seed(4)
    lin = rq.LinearAct(64, 40, activation="tanh", device=dev, dtype=torch.bfloat16)
    emb = rq.ScaledEmbedding(30, 64, scale=3.0, device=dev, dtype=torch.bfloat16)
    idx = torch.randint(0, 30, (2, 7), generator=g).to(dev)
    dy = torch.randn(2, 7, 40, generator=g).to(torch.bfloat16).to(dev)

    def step(w, b, table):
        y = rq.linear_act(rq.embedding(idx, table, 3.0), w, b, "tanh")
        return [y, *torch.autograd.grad(y, (w, b, table), dy)]

    want = step(*[t.detach().clone().requires_grad_() for t in (lin.weight, lin.bias, emb.weight)])

    def refuse(*a):
        raise AssertionError("the registered op was called")

    for name in ("_linear_op", "_embed_op", "_embed_grad_op", "_linear_backward_op"):
        monkeypatch.setattr(rq.train, name, refuse)
    for got in (step(lin.weight, lin.bias, emb.weight), [lin(emb(idx))]):
        for p, q in zip(got, want):
            assert torch.equal(p, q)
    with torch.no_grad():
        assert torch.equal(lin(emb(idx)), want[0])
    with pytest.raises(AssertionError, match="registered"):
        rq.embedding(idx, emb.weight.detach().as_subclass(Other))


@pytest.mark.parametrize("name", (None, "relu", "silu"))
def test_a_frozen_layer_keeps_no_activations(rq, dev, name):
    """Only what the gradients wanted read is kept, and the gradients are the same."""
    g = torch.Generator().manual_seed(6)
    x, w, b = [torch.randn(s, generator=g).to(torch.bfloat16).to(dev) for s in ((50, 64), (40, 64), (40,))]
    dy = torch.randn(50, 40, generator=g).to(torch.bfloat16).to(dev)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(rq.linear_act(*leaves, name), leaves, dy)
    for needs in ((0,), (1,), (2,), (0, 1), (0, 2), (1, 2)):
        ts, kept = [t.detach().clone().requires_grad_(i in needs) for i, t in enumerate(leaves)], []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t.shape) or t, lambda t: t):
            y = rq.linear_act(*ts, name)
        shapes = [(50, 64)] * (1 in needs) + [(40, 64)] * (0 in needs) + [(50, 40)] * (name is not None)
        assert sorted(kept) == sorted(shapes)
        for i, got in zip(needs, torch.autograd.grad(y, [ts[i] for i in needs], dy)):
            assert torch.equal(got, want[i])


def test_no_workspace_outlives_its_call(rq, dev):
    """The backward pass's g (64 MB here), the table gradient's and the clip's scratch
    memory go back to the allocator."""
    x = torch.zeros(8192, 64, dtype=torch.bfloat16, device=dev)
    w = torch.zeros(4096, 64, dtype=torch.bfloat16, device=dev, requires_grad=True)
    table = torch.zeros(500, 64, device=dev, requires_grad=True)
    idx = torch.arange(9000, device=dev) % 500

    def step():
        rq.linear_act(x, w, None, "silu").sum().backward()
        rq.embedding(idx, table).sum().backward()
        rq.clip_grad_norm_([w, table], 1.0)
        w.grad = table.grad = None

    torch.ones(8, device=dev).sum()
    before = torch.cuda.memory_allocated()
    step()
    assert torch.cuda.memory_allocated() == before


@pytest.mark.parametrize("to", ("bf16", "f16"))
def test_linear_act_under_autocast(rq, dev, to):
    """float32 parameters compute in autocast's dtype, as nn.Linear's do, and get float32
    gradients; a float32 residual stream stays one."""
    T = DT[to]
    g = torch.Generator().manual_seed(7)
    lin = torch.nn.Linear(64, 40, device=dev)
    m = rq.LinearAct.from_linear(lin, "silu")
    x = torch.randn(3, 9, 64, generator=g).to(dev).requires_grad_()
    r = torch.randn(3, 9, 40, generator=g).to(dev)
    for res in (None, r):
        with torch.autocast("cuda", dtype=T):
            y, plain = m(x, res), lin(x)
        assert plain.dtype == T and y.dtype == (T if res is None else torch.float32)
        cast = [t.detach().to(T).requires_grad_() for t in (x, lin.weight, lin.bias)]
        want = rq.linear_act(*cast, "silu", res)
        assert torch.equal(y, want)
        dy = torch.randn(3, 9, 40, generator=g).to(dev).to(y.dtype)
        for p, q in zip(torch.autograd.grad(y, (x, lin.weight, lin.bias), dy),
                        torch.autograd.grad(want, cast, dy)):
            assert p.dtype == torch.float32 and torch.equal(p, q.float())
    with torch.autocast("cuda", dtype=T, enabled=False):
        assert m(x).dtype == torch.float32


# --------------------------------------------------------------- embedding

def test_lookup_of_more_rows_than_a_grid_holds(rq, dev):
    """2^26 + 5 tokens: 64 threads each are past the 2^32 of one launch."""
    n = 2 ** 26 + 5
    idx = torch.arange(n, dtype=torch.int32, device=dev) % 251
    w = torch.arange(251 * 8, device=dev).view(251, 8).to(torch.bfloat16)
    out = rq.embedding(idx, w)
    for a in range(0, n, 2 ** 23):
        assert torch.equal(out[a:a + 2 ** 23], w[idx[a:a + 2 ** 23].long()])
