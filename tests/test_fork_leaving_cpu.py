"""What is left of sharing when sequences leave: who may take tokens back, and whether a decode step has rows that share a prefix."""
import pytest

from conftest import load


@pytest.fixture
def kv():
    return load("kv_cache").PagedKVCache(1, 2, 64, 6, 1600, 64, 16, "cpu", max_seq_len=320)


def _grow(kv, sid, n):
    kv.begin_rows([sid], [n])
    kv._len_host[kv.slot(sid)] += n
    kv._pending = None


def test_the_only_holder_takes_tokens_back(kv):
    kv.add_sequence(0)
    _grow(kv, 0, 100)
    kv.fork(1, 0)         # 96 tokens
    kv.fork(2, 0, 40)     # 32
    _grow(kv, 1, 10)
    with pytest.raises(ValueError, match="take back"):
        kv.begin_rows([0], [-5])
    kv.begin_rows([0], [-4])
    kv._pending = None
    kv.remove_sequence(1)
    _grow(kv, 0, -5)      # (page 5 is the source's alone again)
    _grow(kv, 0, -60)
    assert kv.length(0) == 35
    for sid in (0, 2):    # the first two pages are still shared
        with pytest.raises(ValueError, match="take back"):
            kv.begin_rows([sid], [31 - kv.length(sid)])
    kv.begin_rows([0], [-3])
    kv._pending = None
    kv.remove_sequence(0)
    _grow(kv, 2, -32)     # (a fork whose source has gone)
    assert kv.length(2) == 0
    kv.remove_sequence(2)
    assert not kv._more_holders and len(kv._free) == kv.n_pages


def test_pages_that_changed_hands(kv):
    """A sequence that never shared is not asked about the pages that its slot or its numbers had before."""
    kv.add_sequence(0)
    _grow(kv, 0, 64)
    kv.fork(1, 0)
    kv.remove_sequence(1)
    kv.remove_sequence(0)
    kv.add_sequence(1)
    _grow(kv, 1, 64)
    kv.add_sequence(5)
    kv.fork(6, 1, 16)
    _grow(kv, 1, -48)
    with pytest.raises(ValueError, match="take back"):
        kv.begin_rows([1], [-1])
    kv.begin_rows([5], [0])


def test_a_prefix_that_one_sequence_is_left_with(kv):
    """A cache shares prefixes while two sequences begin with one; the one that is left can begin a group of fewer tokens."""
    for sid in (0, 9):
        kv.add_sequence(sid)
        _grow(kv, sid, 200)
    kv.fork(1, 0)
    assert kv.shares_prefixes
    kv.remove_sequence(1)
    assert not kv.shares_prefixes
    kv.fork(2, 0, 100)
    assert kv.shares_prefixes
    one, two = (kv.slot(s) for s in (0, 2))
    assert int(kv.prefix_id[one]) == int(kv.prefix_id[two]) >= 0 and int(kv.prefix_len[one]) == int(kv.prefix_len[two]) == 96
    kv.fork(3, 9, 32)
    assert int(kv.prefix_id[kv.slot(3)]) == int(kv.prefix_id[kv.slot(9)]) != int(kv.prefix_id[one])
    kv.fork(4, 0, 64)  # (while others are in the group, one that shares fewer stays outside)
    assert int(kv.prefix_id[kv.slot(4)]) == -1 and int(kv.prefix_len[one]) == 96
    kv.remove_sequence(0)
    assert kv.shares_prefixes  # (3 and 9)
    kv.remove_sequence(9)
    assert not kv.shares_prefixes
    assert int(kv.prefix_id[two]) >= 0  # (a graph captured earlier finds no second row with it)


def test_steps_whose_rows_share_nothing(kv):
    """The engine takes the route for shared prefixes only where two sequences of the step begin with one."""
    engine = load("model").Engine
    eng = engine.__new__(engine)
    eng.kv, eng.shared_rows, eng.step_seqs, eng.prefix_least = kv, 256, None, 0
    for sid in (0, 7, 8):
        kv.add_sequence(sid)
        _grow(kv, sid, 100)
    kv.fork(1, 0)
    kv.fork(2, 0)
    kv.fork(9, 8)
    assert kv.shared_by([0, 7, 1]) and kv.shared_by([1, 2]) and not kv.shared_by([0, 7]) and not kv.shared_by([0, 8, 7]) and not kv.shared_by([])
    for seqs, shares in (([7, 8, 0], False), ([2, 9], False), ([1, 2, 7], True), ([9, 1, 8], True)):
        kv.begin_rows(seqs, [1] * len(seqs))  # (an eager step)
        assert eng._shares_prefixes(len(seqs), True) == shares and not eng._shares_prefixes(len(seqs), False)
        kv._pending = None
        eng.step_seqs = seqs  # (a captured one)
        assert eng._shares_prefixes(len(seqs), True) == shares
        eng.step_seqs = None
        assert eng._shares_prefixes(len(seqs), True)  # (a caller's own: any sequences of the cache)


def test_steps_whose_groups_are_not_worth_a_plan():
    """Groups that the plan would leave to their rows: the engine does not make one."""
    kv = load("kv_cache").PagedKVCache(1, 8, 64, 8, 20000, 64, 16, "cpu", max_seq_len=4000)
    engine = load("model").Engine
    eng = engine.__new__(engine)
    eng.kv, eng.shared_rows, eng.prefix_least = kv, 256, -1
    for sid, n in ((0, 2000), (10, 900)):
        kv.add_sequence(sid)
        _grow(kv, sid, n)
    for sid in (1, 2, 3):
        kv.fork(sid, 0)
    kv.fork(11, 10)
    for least, shares in ((-1, [True, False, False, False]), (0, [True, True, True, False]), (40000, [True, False, False, False])):
        eng.prefix_least = least
        for seqs, want in zip(([0, 1, 2, 3], [3, 1, 2], [10, 11], [0, 10]), shares):
            eng.step_seqs = seqs
            assert eng._shares_prefixes(len(seqs), True) == want, (least, seqs)
    together = load("ops").prefix_together
    assert together(4, 1024, 1) and not together(3, 32768, 40) and not together(4, 1023, 8) and together(32, 208, 32) and not together(32, 192, 32)
    assert together(2, 64, 1, 64) and not together(2, 64, 1, 65) and not together(2, 63, 1, 0) and not together(1, 4096, 8, 0)


@pytest.mark.parametrize("rows,tokens,kv_heads", [(-1, 64, 8), (4, -1, 8), (4, 1024, 0)])
def test_groups_of_no_size_are_refused(rows, tokens, kv_heads):
    with pytest.raises(load("_lib").MloraError, match="bad sizes"):
        load("ops").prefix_together(rows, tokens, kv_heads)
