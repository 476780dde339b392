"""The sampler on rows whose logits lie closer together, or further apart, than its bins and quanta."""
import math

import pytest
import torch

from sample_ref import sample as want_of

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "fp32": torch.float32}


@pytest.mark.parametrize("spread", [1e-37, 3e-36, 5e-36, 7e-36, 1e-30, 1e-40, 1e-44])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_logits_closer_than_a_bin_can_be(rq, dev, dt, spread):
    """All terms are 1 in float64: what stays is counted, and every border lies between two counts."""
    g = torch.Generator().manual_seed(1)
    for vocab in (2, 3, 7, 100, 512, 1024, 5000, 5120):
        rows = torch.stack([torch.where(torch.arange(vocab) % 3 == 1, 0.0, -spread),            # two values
                            -spread * torch.rand(vocab, generator=g),                          # many
                            torch.where(torch.arange(vocab) == vocab - 1, 0.0, -spread),       # the largest last
                            -spread * (torch.arange(vocab) == 0).float()])                     # all equal but one
        logits = rows.to(DT[dt]).repeat_interleave(4, 0).to(dev)
        u = torch.tensor([0.0, 0.31, 0.617, 0.993], device=dev).repeat(4)
        for kw in ({"top_p": 0.5}, {"top_p": 0.9}, {"top_p": 0.03}, {"top_p": 0.9, "min_p": 0.5}, {"top_k": 2, "top_p": 0.9},
                   {"top_k": vocab - 1 if vocab > 1 else 1, "top_p": 0.77}, {}, {"top_p": 0.9, "temperature": 1e4}):
            print(f"sample spread={spread} {dt} vocab={vocab} {kw}", flush=True)
            token, logprob = rq.sample(logits, u, **kw)
            want, wlog = want_of(logits, u, **kw)
            assert torch.equal(token.cpu(), want), kw
            # terms of 1: no rounding but the logarithm's own
            assert ((logprob.double().cpu() - wlog).abs() <= 2.0 ** -24 * wlog.abs() + 2.0 ** -40).all()


def test_temperatures_next_to_nothing(rq, dev):
    """26 temperatures below the largest logit, where the last bin ends, lie closer than a bin can be."""
    g = torch.Generator().manual_seed(2)
    logits, u = torch.randn(5, 999, generator=g).to(dev), torch.rand(5, generator=g).to(dev)
    for t in (1e-36, 1e-37, 1e-38, 1e-44):
        for kw in ({"top_p": 0.9}, {"top_p": 0.9, "top_k": 40}, {"min_p": 0.1}):
            token, logprob = rq.sample(logits, u, temperature=t, **kw)
            assert torch.equal(token, logits.argmax(-1)) and (logprob == 0).all(), (t, kw)


@pytest.mark.parametrize("vocab", [70000, 131072, 131073, 2 ** 20])
def test_terms_next_to_the_quantum(rq, dev, vocab):
    """A term is rounded to whole quanta of 2^-36, past 2^17 logits 2^-33: tokens below half of one never come, and the sums
    and the log-probabilities are those of the rounded terms."""
    bits = 36 if vocab <= 2 ** 17 else 33
    at = vocab // 3
    u = torch.tensor([0.0, 0.5, 1 - 2.0 ** -10, 1 - 2.0 ** -24], device=dev)
    for quanta in (0.4, 0.6, 1.4, 2.6):
        logits = torch.full((len(u), vocab), math.log(quanta * 2.0 ** -bits))
        logits[:, at] = 0.0
        logits = logits.to(dev)
        tail = round(quanta)
        term = torch.full((vocab,), tail, dtype=torch.int64)
        term[at] = 2 ** bits
        upto = term.cumsum(0).double()   # below 2^53: exact
        whole = int(upto[-1])
        want = [min(int((upto <= min(x * whole, whole - 1)).sum()), vocab - 1) for x in u.double().tolist()]
        if tail == 0:
            assert want == [at] * len(u)
        for kw in ({}, {"top_p": 1 - 2.0 ** -24}) if tail == 0 else ({},):
            token, logprob = rq.sample(logits, u, **kw)
            assert token.tolist() == want, (quanta, kw)
            z = torch.where(token.cpu() == at, 0.0, logits[0, at - 1].double().cpu().item())
            share = z - math.log(whole / 2 ** bits)
            assert ((logprob.double().cpu() - share).abs() <= 2.0 ** -24 * share.abs() + 2.0 ** -45).all()
