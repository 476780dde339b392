"""linear_act and its backward pass on the GPU against the formulas in 64 bits,
within the bounds of tests/train_ref.py, and its gradients against differences."""
import pytest
import torch

from train_ref import Linear, U32, close

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "fp32": torch.float32}
ACTS = (None, "relu", "relu2", "silu", "gelu", "sigmoid", "tanh")

# (m, n, k): single elements, one token, fewer rows than a tile, one past a
# tile in each direction, rows that are not whole 16-byte lines, whole tiles,
# long contractions with few outputs, many rows with a short contraction
SIZES = [(1, 1, 1), (1, 64, 768), (2, 96, 200), (5, 17, 33), (16, 128, 64), (17, 48, 320), (31, 515, 96),
         (65, 129, 72), (64, 64, 2056), (130, 72, 771), (256, 256, 128), (257, 384, 264), (300, 257, 100),
         (512, 1024, 512), (1025, 136, 40), (3, 2048, 4096), (700, 8, 1032)]


def make(dev, m, n, k, dt, bias, residual, seed):
    g = torch.Generator().manual_seed(seed)
    T = DT[dt]
    x = torch.randn(m, k, generator=g).to(T)
    w = (torch.randn(n, k, generator=g) * (1.5 / max(k, 1) ** 0.5)).to(T)
    b = torch.randn(n, generator=g).to(T) if bias else None
    r = torch.randn(m, n, generator=g).to(DT[residual]) if residual else None
    dy = torch.randn(m, n, generator=g).to(r.dtype if r is not None else T)
    return [None if t is None else t.to(dev) for t in (x, w, b, r, dy)]


def check(rq, dev, m, n, k, dt, name, bias, residual, seed=0):
    x, w, b, r, dy = make(dev, m, n, k, dt, bias, residual, 31 * m + 7 * n + k + seed)
    print(f"linear_act m={m} n={n} k={k} {dt} {name} bias={bias} residual={residual}", flush=True)
    ref = Linear(x, w, b, r, name, dy)
    y0 = rq.linear_act(x, w, b, name, r)
    leaves = [t.requires_grad_() for t in (x, w, b, r) if t is not None]
    y = rq.linear_act(x, w, b, name, r)
    assert torch.equal(y0, y.detach()) or y0.isnan().any(), "with and without slopes"
    close(y, ref.y, ref.ey, "y")
    grads = dict(zip([i for i, t in enumerate((x, w, b, r)) if t is not None],
                     torch.autograd.grad(y, leaves, dy)))
    close(grads[0], ref.dx, ref.edx, "dx")
    close(grads[1], ref.dw, ref.edw, "dw")
    assert grads[0].dtype == grads[1].dtype == x.dtype
    if b is not None:
        close(grads[2], ref.db, ref.edb, "db")
    if r is not None:
        assert torch.equal(grads[3], dy)
    again = torch.autograd.grad(rq.linear_act(x, w, b, name, r), leaves, dy)
    for p, q in zip(again, grads.values()):
        assert torch.equal(p, q), "the same inputs give the same bits"


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("i", range(len(SIZES)))
def test_sizes(rq, dev, dt, i):
    m, n, k = SIZES[i]
    residual = ("", dt, "fp32")[i % 3]
    check(rq, dev, m, n, k, dt, ACTS[i % 7], i % 2 == 0, residual)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("name", ACTS)
def test_activations(rq, dev, dt, name):
    for residual in ("", dt, "fp32"):
        check(rq, dev, 70, 136, 64, dt, name, True, residual)
        check(rq, dev, 4, 136, 64, dt, name, False, residual)


def test_large_tiles(rq, dev):
    """Whole and ragged tiles of the large products, every order of the operands."""
    check(rq, dev, 1024, 768, 1024, "bf16", "gelu", True, "fp32")
    check(rq, dev, 777, 1288, 520, "bf16", "relu2", False, "")
    check(rq, dev, 777, 1288, 520, "f16", "silu", True, "f16")
    check(rq, dev, 1100, 640, 600, "fp32", "tanh", True, "")


def test_largest_tiles(rq, dev):
    """Enough outputs that the 256 x 256 tiles are the cheapest, whole and ragged,
    with a contraction that is not whole stages; the gradients' long contractions."""
    check(rq, dev, 4096, 4096, 136, "bf16", "relu2", False, "")
    check(rq, dev, 3000, 5000, 72, "f16", "silu", True, "fp32")


def test_many_rows_of_few_columns(rq, dev):
    """More rows than a grid's second dimension has blocks, a gradient of one tile
    over a contraction of as many."""
    check(rq, dev, 70000, 8, 64, "bf16", "tanh", True, "")


def test_empty(rq, dev):
    for m, n, k in ((0, 8, 8), (4, 0, 8), (4, 8, 0)):
        x, w, b, r, dy = make(dev, m, n, k, "bf16", True, "fp32", 1)
        for t in (x, w, b):
            t.requires_grad_()
        y = rq.linear_act(x, w, b, "silu", r)
        ref = Linear(x, w, b, r, "silu", dy)
        close(y, ref.y, ref.ey, "y")
        dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
        close(dx, ref.dx, ref.edx, "dx")
        close(dw, ref.dw, ref.edw, "dw")
        close(db, ref.db, ref.edb, "db")


def test_leading_dimensions_strides_and_alignment(rq, dev):
    g = torch.Generator().manual_seed(3)
    base = torch.randn(6, 50, 130, generator=g).to(torch.bfloat16).to(dev)
    wt = (torch.randn(128, 72, generator=g) * 0.1).to(torch.bfloat16).to(dev)
    x, w = base[1:5, ::2, 1:129], wt.t()     # rows apart, off alignment; columns apart
    r = torch.randn(25, 4, 72, generator=g).to(dev).transpose(0, 1)
    b = torch.randn(144, generator=g).to(torch.bfloat16).to(dev)[::2]
    y = rq.linear_act(x, w, b, "tanh", r)
    assert y.shape == (4, 25, 72) and y.dtype == torch.float32
    ref = Linear(x, w, b, r, "tanh")
    close(y, ref.y, ref.ey, "y")
    xr, wr = x.detach().requires_grad_(), w.detach().requires_grad_()
    out = rq.linear_act(xr, wr, None, "relu2")
    dy = torch.ones((), dtype=out.dtype, device=dev).expand(out.shape)   # of out.sum()
    ref = Linear(x, w, None, None, "relu2", dy)
    dx, dw = torch.autograd.grad(out.sum(), (xr, wr))
    close(dx, ref.dx, ref.edx, "dx")
    close(dw, ref.dw, ref.edw, "dw")


def test_some_gradients_only(rq, dev):
    x, w, b, r, dy = make(dev, 40, 64, 72, "bf16", True, "bf16", 5)
    ref = Linear(x, w, b, r, "gelu", dy)
    for want in ((0,), (1,), (2,), (3,), (0, 2), (1, 3)):
        ts = [t.detach().clone() for t in (x, w, b, r)]
        for i in want:
            ts[i].requires_grad_()
        y = rq.linear_act(ts[0], ts[1], ts[2], "gelu", ts[3])
        got = torch.autograd.grad(y, [ts[i] for i in want], dy)
        for i, t in zip(want, got):
            val, e = ((ref.dx, ref.edx), (ref.dw, ref.edw), (ref.db, ref.edb),
                      (dy.double().cpu(), torch.zeros(40, 64)))[i]
            close(t, val, e, f"gradient {i}")


def test_mixed_dtypes_compute_in_float32(rq, dev):
    x, w, b, r, dy = make(dev, 33, 40, 64, "fp32", True, "", 6)
    wb = w.to(torch.bfloat16).requires_grad_()
    y = rq.linear_act(x, wb, b, "silu")
    assert y.dtype == torch.float32
    ref = Linear(x, wb.detach().float(), b, None, "silu", dy)
    close(y, ref.y, ref.ey, "y")
    dw, = torch.autograd.grad(y, (wb,), dy)
    assert dw.dtype == torch.bfloat16
    close(dw, ref.dw, ref.edw + 2.0 ** -8 * (ref.dw.abs() + ref.edw), "dw")


def test_values_that_are_not_finite_stay_in_their_rows(rq, dev):
    for m in (4, 70, 300):
        x, w, b, _, _ = make(dev, m, 136, 264, "bf16", True, "", 8)
        x[1, 3], x[2, 200] = float("inf"), float("nan")
        y = rq.linear_act(x, w, b, None).double().cpu()
        want = x.double().cpu() @ w.double().cpu().t() + b.double().cpu()
        assert torch.equal(y[1], want[1]) and y[2].isnan().all()
        keep = [i for i in range(m) if i not in (1, 2)]
        assert y[keep].isfinite().all()
        y = rq.linear_act(x, w, b, "relu").double().cpu()
        assert torch.equal(y[1], want[1].clamp(min=0)) and y[2].isnan().all()


def test_on_another_stream(rq, dev):
    x, w, b, r, dy = make(dev, 200, 264, 128, "bf16", True, "fp32", 9)
    ref = Linear(x, w, b, r, "silu", dy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        leaves = [t.requires_grad_() for t in (x, w, b)]
        y = rq.linear_act(x, w, b, "silu", r)
        got = torch.autograd.grad(y, leaves, dy)
    torch.cuda.current_stream().wait_stream(s)
    close(y, ref.y, ref.ey, "y")
    for t, (v, e) in zip(got, ((ref.dx, ref.edx), (ref.dw, ref.edw), (ref.db, ref.edb))):
        close(t, v, e, "gradient on another stream")


@pytest.mark.parametrize("m", (3, 40, 520))
def test_in_a_hip_graph(rq, dev, m):
    x, w, b, r, dy = make(dev, m, 264, 1024, "bf16", True, "fp32", 10)
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def step():
        y = rq.linear_act(x, w, b, "silu", r)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for replay in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(replay)).to(x))
        want = step()
        for t in got:
            t.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(got, want):
            assert torch.equal(p, q), f"replay {replay}"


@pytest.mark.parametrize("name", ACTS[3:])
def test_gradients_against_differences(rq, dev, name):
    """<gradient, d> against the central difference of <dy, y> along d.  The
    difference is off by at most h^2 / 6 times the third derivative along d (the
    activations' third derivatives are below 3) and by the rounding of y over h."""
    x, w, b, _, dy = make(dev, 24, 40, 48, "fp32", True, "", 11)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(rq.linear_act(x, w, b, name), leaves, dy)
    g = torch.Generator().manual_seed(12)
    h = 2.0 ** -7
    for i, (t, grad) in enumerate(zip(leaves, grads)):
        d = torch.randn(t.shape, generator=g).to(dev)

        def loss(step):
            ts = [p.detach().clone() for p in leaves]
            ts[i] += step * d
            return (rq.linear_act(*ts, name).double() * dy.double()).sum().item(), ts

        (up, ts), (down, _) = loss(h), loss(-h)
        ref = Linear(x, w, b, None, name, dy)
        X, W = x.detach().double().cpu(), w.detach().double().cpu()
        dv = (d.double().cpu() @ W.t() if i == 0 else X @ d.double().cpu().t() if i == 1
              else d.double().cpu().expand(24, 40))
        D = dy.double().cpu().abs()
        third = h * h / 6 * (D * 3 * dv.abs() ** 3).sum()
        rounding = (D * 2 * ref.ey).sum() / h + (D * 1.2).sum() * U32 * 8 / h
        ownd = ((ref.edx, ref.edw, ref.edb)[i] * d.double().cpu().abs()).sum()
        slope = (grad.double() * d.double()).sum().item()
        assert abs((up - down) / (2 * h) - slope) <= float(third + rounding + ownd)


def test_module(rq, dev):
    lin = torch.nn.Linear(64, 48, device=dev, dtype=torch.bfloat16)
    m = rq.LinearAct.from_linear(lin, "sigmoid")
    assert m.weight is lin.weight and m.bias is lin.bias
    x = torch.randn(3, 5, 64, device=dev, dtype=torch.bfloat16)
    r = torch.randn(3, 5, 48, device=dev)
    y = m(x, r)
    ref = Linear(x, lin.weight, lin.bias, r, "sigmoid", r)
    close(y, ref.y, ref.ey, "y")
    y.backward(r)
    close(lin.weight.grad, ref.dw, ref.edw, "weight.grad")
    close(lin.bias.grad, ref.db, ref.edb, "bias.grad")


def test_registered_op_and_its_gradients(rq, dev):
    """What torch.compile and tracing record: the same results."""
    x, w, b, r, dy = make(dev, 37, 72, 64, "bf16", True, "fp32", 13)
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    code = ACTS.index("gelu")
    y, _ = torch.ops.rwkvq.linear_act(x, w, b, r, code)
    assert torch.equal(y, rq.linear_act(x, w, b, "gelu", r))
    want = torch.autograd.grad(rq.linear_act(x, w, b, "gelu", r), leaves, dy)
    for p, q in zip(torch.autograd.grad(y, leaves, dy), want):
        assert torch.equal(p, q)


def test_slopes_of_relu2_over_the_whole_range_of_bf16(rq, dev):
    """2 v from far below float16's range to far above it, through one weight."""
    v = torch.logspace(-30, 15, 512, base=10.0, dtype=torch.float64)
    x = v.to(torch.bfloat16)[:, None].to(dev).requires_grad_()
    w = torch.ones(1, 1, dtype=torch.bfloat16, device=dev)
    r = torch.zeros(512, 1, dtype=torch.float32, device=dev)
    dx, = torch.autograd.grad(rq.linear_act(x, w, None, "relu2", r), x, torch.full_like(r, 2.0 ** -10))
    want = 2 * x.detach().double() * 2.0 ** -10
    # the slope's rounding (bf16 at worst), g's and dx's (both exact to bf16)
    assert ((dx.double() - want).abs() <= 3 * 2.0 ** -8 * want).all()


def test_second_derivatives_are_refused(rq, dev):
    x, w, _, _, dy = make(dev, 8, 16, 16, "fp32", False, "", 14)
    x.requires_grad_()
    dx, = torch.autograd.grad(rq.linear_act(x, w, None, "silu"), x, dy, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.sum(), x)
    e = torch.randn(9, 4, device=dev, requires_grad=True)
    g = torch.randn(3, 4, device=dev, requires_grad=True)
    de, = torch.autograd.grad(rq.embedding(torch.tensor([1, 2, 1], device=dev), e), e, g, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(de.sum(), g)


# (m, n, k): each at which one of the three products takes a form that the sizes
# above do not reach -- large and small tiles, shallow and deep stages, odd widths
# in large tiles, few rows by groups of 16, 32 and 64, shares of the contraction
FORM_SIZES = [(5432, 2192, 64), (8720, 208, 64), (8376, 200, 456), (65, 8992, 72), (2831, 2196, 65),
              (5619, 64, 2216), (195, 64, 8200), (202, 632, 8200), (8936, 64, 72), (8584, 66, 734),
              (64, 1320, 8928), (64, 8720, 200), (68, 3818, 1654), (40, 200, 136), (40, 77, 131)]


@pytest.mark.parametrize("i", range(len(FORM_SIZES)))
def test_forms(rq, dev, i):
    m, n, k = FORM_SIZES[i]
    check(rq, dev, m, n, k, ("bf16", "f16")[i % 2], ACTS[1 + i % 6], i % 3 == 0, ("", "fp32")[i % 2])


@pytest.mark.parametrize("size", [(6999, 392, 8), (461, 8, 6208), (1, 336, 8216), (50, 96, 1000)])
def test_forms_of_float32(rq, dev, size):
    check(rq, dev, *size, "fp32", "silu", True, "")


def test_offsets_past_32_bits(rq, dev):
    """70000 x 32768 outputs: the last rows' byte offsets pass 2^32."""
    g = torch.Generator().manual_seed(15)
    m, n, k = 70000, 32768, 64
    x = torch.randn(m, k, generator=g).to(torch.bfloat16).to(dev).requires_grad_()
    w = (torch.randn(n, k, generator=g) * 0.2).to(torch.bfloat16).to(dev)
    r = torch.zeros(m, n, dtype=torch.bfloat16, device=dev)
    r[-3:] = 1
    y = rq.linear_act(x, w, None, "sigmoid", r)
    rows = torch.tensor([0, 1, 33000, 65535, m - 3, m - 2, m - 1], device=dev)
    ref = Linear(x.detach()[rows], w, None, r[rows], "sigmoid", torch.ones(7, n, dtype=torch.bfloat16))
    close(y.detach()[rows], ref.y, ref.ey, "y")
    dx, = torch.autograd.grad(y, x, torch.ones((), dtype=torch.bfloat16, device=dev).expand(m, n))
    close(dx[rows], ref.dx, ref.edx, "dx")
