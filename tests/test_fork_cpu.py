"""Sequences that share pages: who holds a page, when it is free again, and what the tables say."""
import numpy as np
import pytest

from conftest import load


@pytest.fixture
def kv():
    return load("kv_cache").PagedKVCache(1, 2, 64, 6, 960, 64, 16, "cpu", max_seq_len=320)


def _grow(kv, sid, n):
    kv.begin_rows([sid], [n])
    slot = kv.slot(sid)
    kv._len_host[slot] += n
    kv._pending = None


def _pages(kv, sid):
    return kv._bt_host[kv.slot(sid), :kv._n_pages_of[sid]].tolist()


def test_a_fork_shares_whole_pages(kv):
    free = len(kv._free)
    kv.add_sequence(10)
    _grow(kv, 10, 70)
    assert kv.fork(11, 10) == 64 and kv.fork(12, 10, 40) == 32 and kv.fork(13, 10, 15) == 0
    assert _pages(kv, 11) == _pages(kv, 10)[:4] and _pages(kv, 12) == _pages(kv, 10)[:2] and _pages(kv, 13) == []
    assert (kv.length(11), kv.length(12), kv.length(13)) == (64, 32, 0)
    assert len(kv._free) == free - 5  # (a fork takes no page)
    assert kv.block_table[kv.slot(11), :4].tolist() == _pages(kv, 11)
    _grow(kv, 11, 20)
    assert _pages(kv, 11)[:4] == _pages(kv, 10)[:4] and _pages(kv, 11)[4:] != _pages(kv, 10)[4:]
    # the group is what the first fork shared; one that shares less stays outside
    ids = {s: int(kv.prefix_id[kv.slot(s)]) for s in (10, 11, 12, 13)}
    assert ids[10] == ids[11] >= 0 and ids[12] == ids[13] == -1
    assert int(kv.prefix_len[kv.slot(10)]) == int(kv.prefix_len[kv.slot(11)]) == 64


@pytest.mark.parametrize("order", [(10, 11, 12), (12, 11, 10), (11, 10, 12), (10, 12, 11)])
def test_the_last_holder_frees_a_page(kv, order):
    free = sorted(kv._free)
    kv.add_sequence(10)
    _grow(kv, 10, 100)
    kv.fork(11, 10)
    _grow(kv, 11, 30)
    kv.fork(12, 11, 110)
    held = {s: set(_pages(kv, s)) for s in (10, 11, 12)}
    for i, s in enumerate(order):
        kv.remove_sequence(s)
        still = set().union(*(held[x] for x in order[i + 1:])) if i < 2 else set()
        assert not still & set(kv._free) and len(kv._free) == len(set(kv._free))
    assert sorted(kv._free) == free and not kv._more_holders and not kv._shared_tokens and not kv.shares_prefixes
    assert (kv.prefix_id == -1).all()


def test_a_fork_of_a_fork_joins_the_group(kv):
    kv.add_sequence(0)
    _grow(kv, 0, 64)
    kv.fork(1, 0)
    kv.remove_sequence(0)
    _grow(kv, 1, 40)
    assert kv.fork(2, 1) == 96
    assert int(kv.prefix_id[kv.slot(2)]) == int(kv.prefix_id[kv.slot(1)]) and int(kv.prefix_len[kv.slot(2)]) == 64
    other = kv.add_sequence(3)
    assert int(kv.prefix_id[other]) == -1  # (a slot that changed hands)


def test_refusals(kv):
    kv.add_sequence(0)
    _grow(kv, 0, 50)
    with pytest.raises(ValueError):
        kv.fork(1, 0, 51)
    with pytest.raises(KeyError):
        kv.fork(1, 7)
    with pytest.raises(ValueError):
        kv.fork(0, 0)
    assert kv.length(0) == 50 and len(kv._slot_of) == 1
    kv.fork(1, 0)
    for sid in (0, 1):  # shared tokens stay where they are
        with pytest.raises(ValueError):
            kv.begin_rows([sid], [-(kv.length(sid) - 47)])
    kv.begin_rows([0], [-2])
    for s in (2, 3, 4, 5):
        kv.fork(s, 0)
    with pytest.raises(RuntimeError):
        kv.fork(6, 0)
    assert np.array_equal(kv._bt_host[kv.slot(5), :3], kv._bt_host[kv.slot(0), :3])
