"""The sampler on rows whose logits lie closer together than its bins."""
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
