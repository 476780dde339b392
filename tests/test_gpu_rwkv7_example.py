"""The recurrence, its single-token form and the sampler together, as the example's model has
them: training on packed sequences, a prompt, and decoding by a captured step."""
import importlib.util
import math
import os

import pytest
import torch
from torch.nn import functional as F

import sample_ref
import wkv_ref

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "rwkv7_generate.py")


@pytest.fixture(scope="module")
def example(rq, dev):
    spec = importlib.util.spec_from_file_location("rwkv7_generate", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("packed", [False, True])
def test_example_runs(example, packed):
    torch.manual_seed(1)
    model = example.Model(packed=packed)
    losses = example.train(model, 3, report=lambda s: print(s, flush=True))
    assert all(map(math.isfinite, losses)) and abs(losses[0] - math.log(512)) < 1.0
    prompt = torch.randint(0, 512, (2, 20)).cuda()
    tokens, scores = example.generate(model, prompt, 9)
    assert tokens.shape == scores.shape == (2, 9)
    assert tokens.min() >= 0 and tokens.max() < 512 and (scores <= 0).all()
    again, _ = example.generate(model, prompt, 9)
    assert torch.equal(tokens, again)
    print("ok", flush=True)


def close(got, want, tol, what):
    got, want = got.double().cpu(), want.double().cpu()
    assert (got - want).norm() <= tol * want.norm(), (what, ((got - want).norm() / want.norm()).item())


# The model's other parts are the same code on both sides.  An element of the recurrence is off by at most a
# few hundred roundings of its terms (a sum of 64 products in each of up to 130 tokens, whose decays and unit directions
# amplify nothing: 130 * 64 * 2^-24 = 5e-4 of the terms' size if every rounding went the same way; they are
# independent, so that the square root of their number, 91 * 2^-24 = 5.4e-6, is the norm's).  Two blocks, with a norm and
# three products each behind it, may turn that into ten times as much: 5.4e-5.
TOL = 5.4e-5

# The packed head rounds its float32 input to bf16 over more than 16 rows and does not for three: elements off by 2^-8 of
# themselves at most.  Its random [512, 128] matrix stretches no vector more than (sqrt(512) + sqrt(128)) /
# (sqrt(512) - sqrt(128)) = 3 times as much as another.
HEAD = 3 * 2.0 ** -8


def test_training_gradients(example, monkeypatch):
    """Every parameter's gradient through two blocks and packed sequences, against the same model
    with a plain recurrence in 64 bits."""
    torch.manual_seed(2)
    model = example.Model(dtype=torch.float32)
    lens = (77, 1, 130, 16)
    idx = torch.randint(0, 512, (1, sum(lens))).cuda()
    cu = torch.tensor([0, 77, 78, 208, 224], dtype=torch.int32).cuda()
    weight = torch.randn(1, sum(lens), 512).cuda()
    params = {n: p for n, p in model.named_parameters() if p.requires_grad}

    def grads():
        logits, _ = model(idx, cu=cu)
        return logits.detach(), torch.autograd.grad((logits * weight).sum(), list(params.values()))

    logits, got = grads()

    def plain(r, w, k, v, a, b, state, cu):
        six = [x.double() for x in (r, w, k, v, a, b)]
        zero = torch.zeros(len(lens), r.shape[2], 64, 64, dtype=torch.float64, device=r.device)
        y, last = wkv_ref.packed(six, zero, lens)
        return y.to(r.dtype), last.float()

    monkeypatch.setattr(example.rwkvq, "wkv7", plain)
    want_logits, want = grads()
    close(logits, want_logits, TOL, "logits")
    for (name, _), x, z in zip(params.items(), got, want):
        close(x, z, TOL, name)


def test_prompt_and_steps_follow_the_whole(example):
    """A prompt and single steps behind it give the logits of one scan over all, and the sampler
    the tokens that follow from them in 64 bits."""
    torch.manual_seed(3)
    model = example.Model(dtype=torch.float32)
    idx = torch.randint(0, 512, (3, 53)).cuda()
    with torch.no_grad():
        whole, last = model(idx)
        logits, state = model(idx[:, :37])
        close(logits, whole[:, :37], TOL, "prompt")
        more, carried = model(idx[:, 37:], state)
        close(more, whole[:, 37:], TOL, "continued prompt")
        state = [(x.clone(), s.clone()) for x, s in state]
        for t in range(37, 53):
            logits = model.step(idx[:, t], state)
            close(logits, whole[:, t], TOL + HEAD, t)
        for (x, s), (x1, s1), (x2, s2) in zip(state, last, carried):
            close(x, x1, TOL, "last input")
            close(s, s1, TOL, "state")
            close(s2, s1, TOL, "carried state")
    u = torch.tensor([0.1, 0.5, 0.9]).cuda()
    token, logprob = example.rwkvq.sample(logits, u, 0.8, 50, 0.95)
    want, scores = sample_ref.sample(logits, u, 0.8, 50, 0.95, 0.0)
    assert torch.equal(token.cpu(), want.cpu())
    assert (logprob.cpu().double() - scores.cpu().double()).abs().max() < 1e-5
