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


def _tiles(plan):
    """Of a plan: {(first entry of the list of rows, rows, slot that is read)}, and the list."""
    t = plan.table.cpu().tolist()
    first = 8 + 4 * plan.max_rows
    items = first + (plan.max_rows + 3) // 4 * 4
    tiles = {(t[items + 8 * i + 4], t[items + 8 * i + 5], t[items + 8 * i]) for i in range(t[2])}
    assert len(tiles) == t[1]
    return tiles, t[first:first + sum(n for _, n, _ in tiles)]


def test_padding_joins_no_group(ops, cuda):
    """Rows of padding have the slot of a sequence and position -1: no part of its group, whatever they would save."""
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)
    pid, plen = i32([5, 5, 5, -1, 8]), i32([1024, 1024, 1024, 0, 512])
    plan = ops.PrefixPlan(32, 32, 8, cuda, least=0)
    slots, pos = [1, 4, 2] + [0] * 13, [1030, 600, 1100] + [-1] * 13
    ops.prefix_plan(i32(slots), pid, plen, plan, i32(pos))
    assert _tiles(plan) == ({(0, 2, 1)}, [0, 2])
    ops.prefix_plan(i32([0] * 20), pid, plen, plan, i32([-1] * 19 + [1030]))  # a live row and padding
    assert _tiles(plan) == (set(), [])
    ops.prefix_plan(i32(slots), pid, plen, plan)  # (a caller without padding: every row counts)
    assert {n for _, n, _ in _tiles(plan)[0]} == {15}
    with pytest.raises(ValueError, match="row_pos"):
        ops.prefix_plan(i32(slots), pid, plen, plan, i32(pos[:-1]))


def test_a_session_whose_bucket_is_part_padding(ops, cuda):
    """The sequence in the cache's first slot has a prefix; the last steps have three live rows and one of padding."""
    eng, text, asks = _start(cuda, (4, 7, 2, 9, 3))
    eng.kv.add_sequence(0)  # slot 0
    assert eng.kv.slot(0) == 0
    eng.extend([0], [text])
    rest = [text[eng.kv.fork(i, 0):] + a for i, a in enumerate(asks, 1)]
    tok = eng.extend(range(1, 6), rest)[1].tolist()
    session = load("model").DecodeSession(eng, list(range(1, 6)), [-1] * 5, tok, [9, 3, 9, 9, 2])
    got = session.run()
    assert [len(x) for x in got] == [9, 3, 9, 9, 2] and 4 in session._graphs
    assert _tiles(eng.prefix_plan) == ({(0, 3, eng.kv.slot(1))}, [0, 1, 2])
    eng.check_status()


@pytest.mark.parametrize("length", [2 ** 31 - 1, 2 ** 31 - 127, 4096])
def test_a_prefix_longer_than_the_block_table_is_cut(ops, cuda, length):
    """Rows that end inside what their slots call a prefix: all of their tokens are the prefix's, whatever its length is said to be."""
    from test_shared_attention_gpu import _call, _case, _want

    c = _case(8, 2, 64, 16, [(0, 320, 319), (0, 320, 319), (0, 320, 200)], seed=6)
    c["table"] = c["table"][:, :20].contiguous()
    want, bound = _want(c, 8, 2, 64)
    c["rows"] = [(0, length, p) for _, _, p in c["rows"]]
    got, plan = _call(ops, c, 8, 2, cuda)
    assert _tiles(plan)[1] == [0, 1, 2]
    err = (got.cpu().double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
