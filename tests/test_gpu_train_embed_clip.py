"""The trainable table's lookup and gradient, and the gradient norm and clip, on
the GPU against the formulas in 64 bits (bounds: tests/train_ref.py)."""
import math

import pytest
import torch

from train_ref import TINY, U, U32, close, embedding_grad

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "fp32": torch.float32}


# --------------------------------------------------------------- embedding

def tokens(n, vocab, kind, g):
    if kind == "uniform":
        return torch.randint(0, vocab, (n,), generator=g)
    if kind == "text":   # log-uniform: a few ids hold a large share
        return (torch.exp(torch.rand(n, generator=g) * math.log(vocab)) - 1).long().clamp(0, vocab - 1)
    if kind == "one":
        return torch.full((n,), vocab // 2)
    if kind == "runs":   # long runs of neighbouring ids
        return torch.arange(n) * 3 % max(1, min(vocab, 7)) + max(0, vocab - 7)
    return torch.arange(n) % vocab


# (n, vocab, dim): no token, one, shares of one and of several sorted tokens,
# rows of odd width and of several tiles, small and odd vocabularies, more ids
# than one block of 256 counts
SHAPES = [(0, 300, 24, "uniform"), (1, 65536, 768, "uniform"), (7, 5, 1, "uniform"), (8, 9, 64, "one"),
          (9, 1, 40, "one"), (64, 1000, 515, "text"), (333, 257, 129, "text"), (1000, 512, 72, "one"),
          (2048, 4096, 520, "text"), (4099, 50, 33, "text"), (9001, 131075, 20, "text"),
          (20000, 3000, 136, "runs"), (8200, 700, 8, "one"), (3000, 6000, 2056, "cycle")]


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_embedding(rq, dev, dt, i):
    n, vocab, dim, kind = SHAPES[i]
    print(f"embedding n={n} vocab={vocab} dim={dim} {dt} {kind}", flush=True)
    g = torch.Generator().manual_seed(i)
    idx = tokens(n, vocab, kind, g)
    if i % 2:
        idx = idx.to(torch.int32)
    T, scale = DT[dt], (1.0, 0.5, 45.25, -3.0)[i % 4]
    w = torch.randn(vocab, dim, generator=g).to(T).to(dev).requires_grad_()
    idx_d = idx.to(dev)
    out = rq.embedding(idx_d, w, scale)
    want = w.detach().double().cpu()[idx.long()] * scale
    close(out, want, U[T] * want.abs() + TINY[T], "lookup")
    dout = torch.randn(n, dim, generator=g).to(T).to(dev)
    dw, = torch.autograd.grad(out, w, dout)
    ref, e = embedding_grad(idx, dout, vocab, scale, None)
    close(dw, ref, e, "gradient")
    dw2, = torch.autograd.grad(rq.embedding(idx_d, w, scale), w, dout)
    assert torch.equal(dw, dw2), "the same inputs give the same bits"


def test_embedding_shapes_padding_and_outside(rq, dev):
    g = torch.Generator().manual_seed(5)
    w = torch.randn(40, 24, generator=g).to(dev).requires_grad_()
    idx = torch.randint(0, 40, (3, 4, 5), generator=g)
    idx[0, 0, 0], idx[1, 2, 3], idx[2, 0, 1], idx[2, 0, 2] = -1, 40, 7, 2 ** 40
    out = rq.embedding(idx.to(dev), w, 2.0, padding_idx=7)
    ok = (idx >= 0) & (idx < 40)
    assert out.shape == (3, 4, 5, 24) and out[~ok.to(dev)].isnan().all()
    assert torch.equal(out.detach().cpu()[ok], w.detach().cpu()[idx[ok]] * 2)
    dout = torch.randn(3, 4, 5, 24, generator=g).to(dev)
    dw, = torch.autograd.grad(out, w, dout)
    ref, e = embedding_grad(idx, dout, 40, 2.0, 7)
    close(dw, ref, e, "gradient")
    assert (dw[7] == 0).all()
    # padding_idx from the end, strided indices, a broadcast gradient, an offset table
    odd = torch.randn(41 * 24 + 1, generator=g).to(torch.bfloat16).to(dev)
    w2 = odd[1:1 + 40 * 24].view(40, 24).requires_grad_()
    out = rq.embedding(idx.to(dev)[:, ::2], w2, 1.0, padding_idx=-33)
    dw, = torch.autograd.grad(out.nan_to_num().sum(), w2)
    keep = idx[:, ::2]
    ref, e = embedding_grad(keep, torch.ones(*keep.shape, 24, dtype=torch.bfloat16), 40, 1.0, 7)
    close(dw, ref, e, "gradient of a sum")


def test_embedding_gradient_keeps_values_that_are_not_finite(rq, dev):
    idx = torch.tensor([3, 1, 3, 2, 1], device=dev)
    w = torch.zeros(5, 16, device=dev, requires_grad=True)
    dout = torch.ones(5, 16, device=dev)
    dout[1, 2], dout[2, 3] = float("inf"), float("nan")
    dw, = torch.autograd.grad(rq.embedding(idx, w), w, dout)
    assert dw[1, 2] == float("inf") and dw[3, 3].isnan()
    dw[1, 2] = dw[3, 3] = 2
    assert torch.equal(dw.sum(1).cpu(), torch.tensor([0., 32, 16, 32, 0]))


def test_embedding_against_differences(rq, dev):
    """The lookup is linear in the table: the difference quotient is exact up to
    the rounding of the outputs."""
    g = torch.Generator().manual_seed(6)
    idx = torch.randint(0, 30, (50,), generator=g).to(dev)
    w = torch.randn(30, 20, generator=g).to(dev).requires_grad_()
    dout, d = torch.randn(50, 20, generator=g).to(dev), torch.randn(30, 20, generator=g).to(dev)
    dw, = torch.autograd.grad(rq.embedding(idx, w, 3.0), w, dout)
    up = (rq.embedding(idx, w.detach() + d, 3.0).double() * dout.double()).sum().item()
    down = (rq.embedding(idx, w.detach() - d, 3.0).double() * dout.double()).sum().item()
    _, e = embedding_grad(idx, dout, 30, 3.0, None)
    mag = 3.0 * ((w.detach().abs() + d.abs()).double()[idx] * dout.abs().double()).sum().item()
    slope = (dw.double() * d.double()).sum().item()
    assert abs((up - down) / 2 - slope) <= 4 * U32 * mag + (e * d.double().cpu().abs()).sum().item()


def test_embedding_module_and_registered_op(rq, dev):
    g = torch.Generator().manual_seed(7)
    m = rq.ScaledEmbedding(50, 32, scale=5.0, padding_idx=0, device=dev, dtype=torch.bfloat16)
    idx = torch.randint(0, 50, (4, 9), generator=g).to(dev)
    out = m(idx)
    dout = torch.randn(4, 9, 32, generator=g).to(torch.bfloat16).to(dev)
    out.backward(dout)
    ref, e = embedding_grad(idx, dout, 50, 5.0, 0)
    close(m.weight.grad, ref, e, "weight.grad")
    w = m.weight.detach().clone().requires_grad_()
    y = torch.ops.rwkvq.embedding(idx, w, 5.0, 0)
    assert torch.equal(y, out)
    assert torch.equal(torch.autograd.grad(y, w, dout)[0], m.weight.grad)


# -------------------------------------------------------- gradient norm, clip

def grads(dev, shapes, dt, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * std).to(DT[dt] if isinstance(dt, str) else DT[dt[i % len(dt)]]).to(dev)
            for i, s in enumerate(shapes)]


def norm64(ts):
    return math.sqrt(math.fsum((t.double() ** 2).sum().item() for t in ts))


SETS = {
    "one element": [(1,)],
    "empty ones": [(0,), (3, 0), (5,), ()],
    "odd": [(7, 13), (1,), (513,), (3, 5, 7)],
    "adapters": [(16, 2048), (2048, 16)] * 150,
    "past a chunk": [(8192,), (8193,), (4095,), (16385,), (2, 100003)],
    "large": [(2048, 2051), (3000, 1000), (1,)],
    "many": [(i % 5 + 1,) for i in range(700)],
}


@pytest.mark.parametrize("dt", ["bf16", "f16", "fp32", ("fp32", "bf16", "f16")])
@pytest.mark.parametrize("kind", SETS)
def test_clip(rq, dev, dt, kind):
    print(f"clip {kind} {dt}", flush=True)
    ts = grads(dev, SETS[kind], dt, 1)
    n = norm64(ts)
    # exact squares and sums in fp64 (2^-53 each), one rounding to fp32
    assert abs(rq.grad_norm(ts).item() - n) <= 2 * U32 * n
    for factor in (0.1, 1.5):
        top = factor * n
        out, norm = rq.clip_grad_norm(ts, top)
        assert abs(norm.item() - n) <= 2 * U32 * n and norm.dtype == torch.float32
        c = min(top / (n + 1e-6), 1.0)
        kept = [t.clone() for t in ts]
        again = rq.clip_grad_norm(ts, top, out=ts)[0]
        assert all(a is t for a, t in zip(again, ts))
        for o, k, t in zip(out, kept, ts):
            assert o.dtype == k.dtype and o.shape == k.shape
            want = k.double().cpu() * c
            # the factor: three fp32 roundings and the norm's
            close(o, want, (U[k.dtype] + 8 * U32) * want.abs() + TINY[k.dtype], "clipped")
            assert torch.equal(o, t), "in place"
            if factor > 1:
                assert torch.equal(o, k), "within max_norm: unchanged"
            t.copy_(k)


def test_clip_parameters_in_place(rq, dev):
    ps = [torch.nn.Parameter(torch.zeros(s, device=dev)) for s in ((40, 24), (24,), (8, 8), (6, 5, 4))]
    src = grads(dev, [(40, 24), (24,), (8, 8), (6, 5, 4)], "fp32", 2)
    ps[0].grad, ps[1].grad = src[0].clone(), src[1].clone()
    ps[3].grad = src[3].clone().permute(0, 1, 2)
    wide = torch.zeros(40, 40, device=dev)
    ps.append(torch.nn.Parameter(torch.zeros(24, 40, device=dev).t()))
    ps[4].grad = wide[:, :24]                 # rows apart: copied, clipped, written back
    wide[:, :24] = 3.0
    ps.append(torch.nn.Parameter(torch.zeros(24, 40, device=dev).t()))
    ps[5].grad = torch.full((24, 40), 2.0, device=dev).t()
    kept = [None if p.grad is None else p.grad.clone() for p in ps]
    n = norm64([k for k in kept if k is not None])
    norm = rq.clip_grad_norm_(ps, 2.0)
    assert abs(norm.item() - n) <= 2 * U32 * n
    for p, k in zip(ps, kept):
        if k is None:
            assert p.grad is None
        else:
            want = k.double().cpu() * (2.0 / (n + 1e-6))
            close(p.grad, want, 16 * U32 * want.abs(), "grad")
    assert (wide[:, 24:] == 0).all()
    one = torch.nn.Parameter(torch.ones(3, device=dev))
    one.grad = torch.full((3,), 4.0, device=dev)
    rq.clip_grad_norm_(one, 100.0)
    assert (one.grad == 4).all()
    assert rq.clip_grad_norm_([torch.nn.Parameter(torch.ones(2, device=dev))], 1.0).item() == 0


def test_clip_values_past_fp32_squares_and_not_finite(rq, dev):
    big = [torch.full((1000,), 3e30, device=dev), torch.full((10,), 1e-30, device=dev)]
    n = norm64(big)
    assert abs(rq.grad_norm(big).item() - n) <= 2 * U32 * n
    out, _ = rq.clip_grad_norm(big, 1.0)
    want = 3e30 / n
    assert (out[0].double() - want).abs().max().item() <= 16 * U32 * want
    small = [torch.full((9,), 1e-30, device=dev)]
    assert abs(rq.grad_norm(small).item() - 3e-30) <= 4 * U32 * 3e-30
    for bad in (float("nan"), float("inf")):
        ts = [torch.ones(20, device=dev), torch.tensor([1.0, bad], device=dev)]
        out, norm = rq.clip_grad_norm(ts, 1.0)
        if math.isnan(bad):
            assert norm.isnan() and all(o.isnan().all() for o in out)
        else:
            assert norm.isinf() and (out[0] == 0).all() and out[1][0] == 0 and out[1][1].isnan()
    zero = [torch.zeros(30, device=dev)]
    out, norm = rq.clip_grad_norm(zero, 1.0)
    assert norm.item() == 0 and (out[0] == 0).all()
    out, _ = rq.clip_grad_norm([torch.ones(5, device=dev)], 0.0)
    assert (out[0] == 0).all()


def test_clip_offset_views(rq, dev):
    flat = torch.randn(5000, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).to(dev)
    ts = [flat[1:2000], flat[2001:4003], flat[4003:4004]]
    n = norm64(ts)
    out, norm = rq.clip_grad_norm(ts, 1.0)
    assert abs(norm.item() - n) <= 2 * U32 * n
    for o, t in zip(out, ts):
        want = t.double().cpu() / (n + 1e-6)
        close(o, want, (2.0 ** -8 + 8 * U32) * want.abs(), "clipped")


def test_embedding_gradient_and_clip_in_a_hip_graph(rq, dev):
    g = torch.Generator().manual_seed(10)
    idx = torch.randint(0, 900, (600,), generator=g).to(dev)
    w = torch.randn(900, 72, generator=g).to(dev).requires_grad_()
    dout = torch.randn(600, 72, generator=g).to(dev)
    other = torch.randn(70000, generator=g).to(dev)

    def step():
        dw, = torch.autograd.grad(rq.embedding(idx, w, 2.0), w, dout)
        out, norm = rq.clip_grad_norm([dw, other], 1.0)
        return [dw, norm, *out]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for replay in range(3):
        idx.copy_(torch.randint(0, 900, (600,), generator=g))
        want = step()
        for t in got:
            t.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(got, want):
            assert torch.equal(p, q), f"replay {replay}"


def test_offsets_past_32_bits(rq, dev):
    """A table and a gradient of 70000 x 32768: byte offsets pass 2^32."""
    vocab, dim = 70000, 32768
    w = torch.zeros(vocab, dim, dtype=torch.bfloat16, device=dev)
    w[-2:] = torch.arange(dim, device=dev) % 256
    w.requires_grad_()
    idx = torch.tensor([vocab - 1, 0, vocab - 2, vocab - 1, vocab], device=dev)
    out = rq.embedding(idx, w, 2.0)
    assert torch.equal(out[0].float(), 2.0 * (torch.arange(dim, device=dev) % 256)) and (out[1] == 0).all()
    assert torch.equal(out[0], out[2]) and out[4].isnan().all()
    dw, = torch.autograd.grad(out, w, torch.ones_like(out))
    assert (dw[vocab - 1] == 4).all() and (dw[vocab - 2] == 2).all() and (dw[0] == 2).all()
    assert int(torch.count_nonzero(dw[1:vocab - 2])) == 0
    clipped, norm = rq.clip_grad_norm([dw, dw[:1]], 1.0, out=[dw, torch.empty_like(dw[:1])])
    n = math.sqrt(dim * (16 + 4 + 4 + 4))
    assert abs(norm.item() - n) <= 2 * U32 * n
    want = torch.tensor(4 / (n + 1e-6), dtype=torch.float64)
    assert (clipped[0][vocab - 1].double().cpu() - want).abs().max() <= 2.0 ** -7 * want
