"""Which decode steps of an engine take the route for shared prefixes, and what their plan has."""
import pytest
import torch

from conftest import load
from test_serving_step_gpu import _engine, _weights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    return load("ops")


def _start(cuda, n_asks, system=96, **kw):
    w, _, _ = _weights()
    g = torch.Generator().manual_seed(3)
    text = torch.randint(0, 1000, (system,), generator=g).tolist()
    asks = [torch.randint(0, 1000, (k,), generator=g).tolist() for k in n_asks]
    eng = _engine(w, cuda, **kw)
    eng.prefix_least = 0
    return eng, text, asks


def test_steps_that_share_nothing_stay_as_they_were(ops, cuda):
    """A pair of sequences shares a prefix; eager, captured and session steps of the others run as without it, bit for bit."""
    got = []
    for forks in (False, True):
        eng, text, asks = _start(cuda, (9, 20, 3))
        for i, a in enumerate(asks):
            eng.kv.add_sequence(i)
        tok = eng.extend(range(3), asks)[1].tolist()
        if forks:
            eng.kv.add_sequence(50)
            eng.extend([50], [text])
            eng.kv.fork(51, 50)
        out = [eng.decode(range(3), tok, [-1] * 3)[0].clone()]
        tok = eng.next_tok[:3].tolist()
        graph = eng.capture_decode([0, 1, 2], [-1] * 3, reserve_tokens=4, feed_back=False)
        eng.tokens[:3].copy_(torch.tensor(tok, dtype=torch.int32))
        graph.replay()
        out.append(eng.logits[:3].clone())
        tok = eng.next_tok[:3].tolist()
        said = load("model").DecodeSession(eng, [0, 1, 2], [-1] * 3, tok, [5, 3, 6]).run()
        assert eng.prefix_plan is None and eng.step_seqs is None
        got.append((out, said))
    for a, b in zip(got[0][0], got[1][0]):
        assert torch.equal(a, b)
    assert got[0][1] == got[1][1]
