"""The example's model over packed sequences that go on from a state: each as if it were alone."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "rwkv7_generate.py")

# As in test_gpu_rwkv7_example.py: a recurrence off by 5.4e-6 of its norm behind ten times as much of a model, and a head
# that rounds its input to bf16 over more than 16 rows, by a matrix that stretches no vector more than 3 times as another.
TOL, HEAD = 5.4e-5, 3 * 2.0 ** -8


@pytest.fixture(scope="module")
def example(rq, dev):
    spec = importlib.util.spec_from_file_location("rwkv7_generate", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def close(got, want, tol, what):
    got, want = got.double().cpu(), want.double().cpu()
    assert got.shape == want.shape and (got - want).norm() <= tol * want.norm(), what


def boundaries(lens):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32).cuda()


@pytest.mark.parametrize("first,then", [([7, 3, 12, 1], [5, 3, 1, 4]), ([7, 0, 12, 1], [5, 3, 0, 4]),
                                        ([0, 4, 9, 0], [2, 0, 0, 6]), ([5, 30, 2, 0], [1, 1, 1, 0])])
def test_packed_sequences_go_on(example, first, then):
    torch.manual_seed(4)
    model = example.Model(dtype=torch.float32)
    d = model.emb.embedding_dim
    whole = [torch.randint(0, 512, (1, a + b)).cuda() for a, b in zip(first, then)]
    one = torch.cat([x[:, :a] for x, a in zip(whole, first)], 1)
    two = torch.cat([x[:, a:] for x, a in zip(whole, first)], 1)
    with torch.no_grad():
        logits1, state = model(one, cu=boundaries(first))
        assert all(x.shape == (4, d) and s.shape == (4, 2, 64, 64) for x, s in state)
        logits2, state = model(two, state, boundaries(then))
        at1 = at2 = 0
        for i, x in enumerate(whole):
            a, b = first[i], then[i]
            mine = [logits1[0, at1:at1 + a], logits2[0, at2:at2 + b]]
            at1, at2 = at1 + a, at2 + b
            if not x.numel():
                assert all((last[i] == 0).all() and (s[i] == 0).all() for last, s in state)
                continue
            logits, alone = model(x)
            close(torch.cat(mine), logits[0], TOL + HEAD, f"logits of {i}")
            for (last, s), (last1, s1) in zip(state, alone):
                close(last[i], last1[0], TOL, f"last input of {i}")
                close(s[i], s1[0], TOL, f"state of {i}")
        # and by single tokens, all sequences at once
        tok = torch.randint(0, 512, (4,)).cuda()
        state = [(last.clone(), s.clone()) for last, s in state]
        got = model.step(tok, state)
        for i, x in enumerate(whole):
            want, _ = model(torch.cat([x, tok[i:i + 1, None]], 1))
            close(got[i], want[0, -1], TOL + HEAD, f"step of {i}")
