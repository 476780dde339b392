"""The sampler on the GPU against its definition by sorting in float64.

Tokens have to be equal.  A log-probability is rounded once from float64, where the terms' rounding to
2^-36 shifts the sum by at most n 2^-37 of a sum of at least 1: 2^-20 for the largest n here, half
that on average over many; so it is held to 2^-24 of its value plus n 2^-37."""
import math

import pytest
import torch

from sample_ref import sample as want_of

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "fp32": torch.float32}


def check(rq, logits, u, **kw):
    dev = logits.device
    token, logprob = rq.sample(logits, u, **kw)
    assert token.dtype == torch.int64 and logprob.dtype == torch.float32
    assert token.shape == logprob.shape == u.shape and token.device == dev
    want, wlog = want_of(logits, u, **kw)
    bad = (token.cpu() != want).nonzero()
    assert not len(bad), f"{len(bad)} tokens of {u.numel()} differ, first at {bad[0].tolist()}"
    off = (logprob.double().cpu() - wlog).abs()
    e = 2.0 ** -24 * wlog.abs() + logits.shape[-1] * 2.0 ** -37
    assert ((off <= e) | (wlog.isnan() & logprob.cpu().isnan())).all(), off.max()
    return token, logprob


PARAMS = [{}, {"temperature": 0.7}, {"top_k": 1}, {"top_k": 5}, {"top_k": 50, "temperature": 1.5}, {"top_p": 0.9},
          {"top_p": 0.3, "temperature": 0.5}, {"min_p": 0.1}, {"top_k": 40, "top_p": 0.95, "min_p": 0.02},
          {"temperature": 0.0}, {"top_p": 1e-6}, {"min_p": 1.0}, {"top_k": 10 ** 6}, {"temperature": 100.0, "top_p": 0.5},
          {"temperature": 1e-3}]


@pytest.mark.parametrize("vocab", [1, 2, 7, 64, 511, 513, 8191, 8200])
@pytest.mark.parametrize("dt", DT)
def test_every_rule_at_small_vocabularies(rq, dev, dt, vocab):
    for i, kw in enumerate(PARAMS):
        print(f"sample vocab={vocab} {dt} {kw}", flush=True)
        g = torch.Generator().manual_seed(1000 * vocab + i)
        logits = (torch.randn(9, vocab, generator=g) * 2.5).to(DT[dt]).to(dev)
        check(rq, logits, torch.rand(9, generator=g).to(dev), **kw)


@pytest.mark.parametrize("vocab", [50021, 65536, 65537, 131072, 200003, 2 ** 20])
def test_large_vocabularies(rq, dev, vocab):
    for i, (dt, kw) in enumerate(zip(("bf16", "f16", "fp32", "bf16", "fp32"),
                                     ({}, {"top_p": 0.9}, {"top_k": 100, "top_p": 0.8}, {"top_k": 2000}, {"min_p": 0.01}))):
        print(f"sample vocab={vocab} {dt} {kw}", flush=True)
        g = torch.Generator().manual_seed(vocab + i)
        logits = (torch.randn(3, vocab, generator=g) * 2.5).to(DT[dt]).to(dev)
        check(rq, logits, torch.rand(3, generator=g).to(dev), **kw)


def test_equal_logits_rank_by_index(rq, dev):
    """Sums of equal terms are exact: every border is met on the point."""
    logits = torch.zeros(8, 8, device=dev)
    u = torch.arange(8, device=dev) / 8
    assert rq.sample(logits, u)[0].tolist() == list(range(8))
    below = torch.nextafter(u[1:], torch.zeros(7, device=dev))
    assert rq.sample(logits[1:], below)[0].tolist() == list(range(7))
    assert rq.sample(logits, u, top_p=0.5)[0].tolist() == [0, 0, 1, 1, 2, 2, 3, 3]
    assert rq.sample(logits, u, top_k=2)[0].tolist() == [0] * 4 + [1] * 4
    assert rq.sample(logits, u, top_k=4, top_p=0.5)[0].tolist() == [0] * 4 + [1] * 4
    token, logprob = rq.sample(logits, u, min_p=1.0)
    assert token.tolist() == list(range(8)) and torch.equal(logprob, torch.full((8,), -math.log(8), device=dev))
    # -0 and 0 are one value
    logits[:, 1::2] = -0.0
    assert rq.sample(logits, u, top_k=2)[0].tolist() == [0] * 4 + [1] * 4


@pytest.mark.parametrize("vocab", [37, 700, 20000])
def test_many_ties(rq, dev, vocab):
    """Logits of a few values: the borders of top_k and top_p fall among equal ones."""
    g = torch.Generator().manual_seed(vocab)
    logits = torch.randint(-2, 3, (40, vocab), generator=g).to(torch.float16).to(dev)
    u = torch.rand(40, generator=g).to(dev)
    for kw in ({"top_k": vocab // 3}, {"top_p": 0.7}, {"top_k": vocab // 2, "top_p": 0.6}, {"top_k": vocab // 7 + 1, "top_p": 0.999},
               {"top_k": vocab // 4 + 1, "top_p": 0.9, "min_p": 0.3}, {"min_p": 0.2}):
        check(rq, logits, u, **kw)


def test_more_ties_than_a_bin_of_float_holds(rq, dev):
    """Sums of 60000 equal terms, as one class and beside larger ones."""
    n = 100003
    g = torch.Generator().manual_seed(3)
    logits = torch.zeros(4, n)
    logits[1, torch.randperm(n, generator=g)[:500]] = 1.0
    logits[2] = torch.randint(0, 2, (n,), generator=g).float()
    logits[3] = torch.randint(0, 3, (n,), generator=g).float() * 0.5
    logits, u = logits.to(dev), torch.rand(4, generator=g).to(dev)
    for kw in ({"top_k": 60000, "top_p": 0.9}, {"top_p": 0.7}, {"top_k": 90000}, {"top_k": 60000, "top_p": 0.999, "temperature": 2.0},
               {"temperature": 50.0, "top_p": 0.3}):
        for dt in DT.values():
            check(rq, logits.to(dt), u, **kw)


def test_rows_with_parameters_of_their_own(rq, dev):
    g = torch.Generator().manual_seed(4)
    m, vocab = 60, 3001
    logits = (torch.randn(m, vocab, generator=g) * 3).to(torch.bfloat16).to(dev)
    u = torch.rand(m, generator=g).to(dev)

    def pick(*of):
        return torch.tensor(of)[torch.randint(0, len(of), (m,), generator=g)].to(dev)

    kw = {"temperature": pick(0.0, 0.5, 1.0, 2.0), "top_k": pick(0, 1, 7, 100, 5000), "top_p": pick(1.0, 0.2, 0.9),
          "min_p": pick(0.0, 0.05, 1.0)}
    token, logprob = check(rq, logits, u, **kw)
    # each row as a call of its own, in other shapes and types
    for i in range(0, m, 7):
        one = {n: x[i].item() for n, x in kw.items()}
        t, lp = rq.sample(logits[i], u[i], **one)
        assert t.shape == () and t == token[i] and torch.equal(lp, logprob[i])
    kw["top_k"] = kw["top_k"].to(torch.int32)
    kw["temperature"] = kw["temperature"].double()
    shaped = {n: x.view(3, 20) for n, x in kw.items()}
    t, lp = rq.sample(logits.view(3, 20, vocab), u.view(3, 20), **shaped)
    assert torch.equal(t.view(m), token) and torch.equal(lp.view(m), logprob)
    t, _ = rq.sample(logits, u, top_k=torch.tensor(3, device=dev))
    assert torch.equal(t, rq.sample(logits, u, top_k=3)[0])


def test_masked_infinite_and_nan_logits(rq, dev):
    g = torch.Generator().manual_seed(5)
    inf = math.inf
    logits = torch.randn(12, 1000, generator=g)
    logits[0] = -inf
    logits[1, 5] = math.nan
    logits[2] = -inf
    logits[2, 777] = -3.0
    logits[3, 10] = logits[3, 20] = inf
    logits[4, torch.rand(1000, generator=g) < 0.99] = -inf
    logits[5] = torch.finfo(torch.float32).min            # a mask of the type's lowest value
    logits[5, 3:9] = torch.randn(6, generator=g)
    logits[6] = torch.finfo(torch.float32).min            # everywhere
    logits[7, 0], logits[7, 1:] = torch.finfo(torch.float32).max, torch.finfo(torch.float32).min
    logits[8] = -inf
    logits[8, 999] = inf
    logits[9, 0] = -math.nan
    logits = logits.to(dev)
    u = torch.rand(12, generator=g).to(dev)
    for kw in ({}, {"top_k": 3}, {"top_p": 0.8}, {"top_k": 600, "top_p": 0.9, "min_p": 0.01}, {"temperature": 0.0},
               {"temperature": 1e-30}, {"temperature": inf}, {"temperature": inf, "top_p": 0.5}):
        token, logprob = check(rq, logits, u, **kw)
        assert token[[0, 1, 9]].tolist() == [-1] * 3 and logprob[[0, 1, 9]].isnan().all()
        assert token[2] == 777 and logprob[2] == 0 and token[8] == 999
        assert token[3].item() in (10, 20)
        if kw.get("temperature") != inf:   # there every finite logit has the same share, the lowest value too
            assert 3 <= token[5] < 9
    # a token that stands for none looks up a row of NaN
    assert rq.embedding(token[:1], torch.ones(5, 8, device=dev)).isnan().all()


def test_numbers_at_and_past_their_borders(rq, dev):
    g = torch.Generator().manual_seed(6)
    logits = (torch.randn(7, 999, generator=g) * 2).to(dev)
    u = torch.tensor([0.0, -0.0, 1.0 - 2.0 ** -24, 1.0, 7.0, -1.0, math.nan], device=dev)
    for kw in ({}, {"top_k": 9}, {"top_p": 0.5}, {"min_p": 0.3}):
        check(rq, logits, u, **kw)
    # values on the device that a number could not have
    m = len(u)
    weird = [{"temperature": torch.full((m,), x, device=dev)} for x in (-1.0, math.nan)]
    for kw in weird:
        assert torch.equal(rq.sample(logits, u, **kw)[0], logits.argmax(-1))
    assert torch.equal(rq.sample(logits, u, top_k=torch.full((m,), -4, device=dev))[0], rq.sample(logits, u)[0])
    for x in (2.0, math.nan):
        assert torch.equal(rq.sample(logits, u, top_p=torch.full((m,), x, device=dev))[0], rq.sample(logits, u)[0])
    assert torch.equal(rq.sample(logits, u, top_p=torch.full((m,), -1.0, device=dev))[0], logits.argmax(-1))
    for x in (-1.0, math.nan):
        assert torch.equal(rq.sample(logits, u, min_p=torch.full((m,), x, device=dev))[0], rq.sample(logits, u)[0])
    assert torch.equal(rq.sample(logits, u, min_p=torch.full((m,), 5.0, device=dev))[0], logits.argmax(-1))


def test_a_flat_row_reaches_every_token(rq, dev):
    """u = (i + 1/2) / n over n equal logits gives token i."""
    n = 4099
    u = ((torch.arange(n, dtype=torch.float64) + 0.5) / n).float().to(dev)
    token, _ = rq.sample(torch.full((n, n), 3.0, dtype=torch.bfloat16, device=dev), u)
    assert torch.equal(token, torch.arange(n, device=dev))


def test_strides_and_alignment(rq, dev):
    g = torch.Generator().manual_seed(7)
    for dt in DT.values():
        logits = torch.randn(6, 1001, generator=g).to(dt).to(dev)
        u = torch.rand(6, generator=g).to(dev)
        want = rq.sample(logits, u, top_p=0.9)
        flat = torch.empty(logits.numel() + 1, dtype=dt, device=dev)
        odd = flat[1:].view(6, 1001).copy_(logits)
        wide = torch.empty(6, 1501, dtype=dt, device=dev)
        wide[:, 200:1201] = logits
        for x in (odd, wide[:, 200:1201], logits.t().contiguous().t()):
            for a, b in zip(want, rq.sample(x, u, top_p=0.9)):
                assert torch.equal(a, b)
        a, b = rq.sample(logits, torch.stack([u, u], 1)[:, 0], top_p=torch.full((12,), 0.9, device=dev)[::2])
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])
        for x in rq.sample(logits[:0], u[:0]):
            assert x.numel() == 0


def test_other_streams_graphs_and_the_same_bits(rq, dev):
    g = torch.Generator().manual_seed(8)
    logits = (torch.randn(20, 7001, generator=g) * 2).to(torch.bfloat16).to(dev)
    u = torch.rand(20, generator=g).to(dev)
    kw = {"top_k": torch.full((20,), 500, device=dev), "top_p": 0.9}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = rq.sample(logits, u, **kw)
    torch.cuda.current_stream().wait_stream(side)
    here = rq.sample(logits, u, **kw)
    assert torch.equal(there[0], here[0]) and torch.equal(there[1], here[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rq.sample(logits, u, **kw)
    for i in range(4):
        logits.copy_(logits.roll(i + 1, 0))
        u.copy_(u.flip(0) * 0.9)
        graph.replay()
        got = [x.clone() for x in out]
        torch.cuda.synchronize()
        want = rq.sample(logits, u, **kw)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_offsets_past_32_bits(rq, dev):
    m, vocab = 36000, 65537     # 4.7e9 bytes
    logits = torch.full((m, vocab), -1.0, dtype=torch.bfloat16, device=dev)
    at = torch.arange(m, device=dev) * 7919 % vocab
    logits.scatter_(1, at[:, None], 30.0)
    token, _ = rq.sample(logits, torch.full((m,), 0.5, device=dev))
    assert torch.equal(token, at)


def test_registered_op(rq, dev):
    logits, u = torch.randn(3, 50, device=dev), torch.rand(3, device=dev)
    torch.library.opcheck(torch.ops.rwkvq.sample.default,
                          (logits, u, torch.ones(3, device=dev), None, None, None, 1.0, 5, 0.9, 0.0),
                          test_utils=("test_schema", "test_faketensor"))


def test_refusals(rq, dev):
    logits, u = torch.zeros(3, 10, device=dev), torch.zeros(3, device=dev)
    for kw, text in (({"temperature": -1.0}, "temperature"), ({"temperature": math.nan}, "temperature"), ({"top_k": -1}, "top_k"),
                     ({"top_p": 0.0}, "top_p"), ({"top_p": 1.5}, "top_p"), ({"min_p": -0.1}, "min_p"), ({"min_p": 2.0}, "min_p"),
                     ({"top_k": torch.ones(3, device=dev)}, "top_k"), ({"top_p": torch.ones(3, device=dev).int()}, "top_p"),
                     ({"min_p": torch.ones(3, 1, device=dev)}, "min_p")):
        with pytest.raises(ValueError, match=text):
            rq.sample(logits, u, **kw)
    with pytest.raises(ValueError, match="u must be"):
        rq.sample(logits, u[:2])
    with pytest.raises(ValueError, match="u must be"):
        rq.sample(logits, u.double())
    with pytest.raises(ValueError, match="logits"):
        rq.sample(logits.long(), u)
    with pytest.raises(ValueError, match="without a logit"):
        rq.sample(logits[:, :0], u)
    with pytest.raises(ValueError, match="vocabulary"):
        rq.sample(torch.zeros(1, 2 ** 20 + 1, device=dev), u[:1])
    with pytest.raises((ValueError, RuntimeError)):
        rq.sample(logits, u.cpu())
    with pytest.raises((ValueError, RuntimeError)):
        rq.sample(logits, u, top_p=torch.ones(3))
