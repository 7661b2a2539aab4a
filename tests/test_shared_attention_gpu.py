"""Decode attention of a batch that shares prefixes, against the formula in 64 bits.

Bound of an output's error, with A = sum over the keys of softmax * |v|: half a step of bf16 of the output itself (2^-8 |o|); half a step of
bf16 of every probability of the prefix's keys (2^-8 A), whose sum is taken before that rounding; and what 32-bit sums of `dim` products
do to the scores and so to the probabilities (twice dim 2^-24 scale max sum |q k|, and 2^-20 for the other 32-bit steps)."""
import pytest
import torch

from conftest import load

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    return load("ops")


def _case(heads, kv_heads, dim, page, rows, seed=0, in_order=False, scale_q=2.0):
    """``rows``: (prefix id or -1, prefix length, last position or -1).  Every place of the pages that no row's token lies in is NaN.
    Returns the call's tensors on the CPU and, per row, its keys and values."""
    g = torch.Generator().manual_seed(seed)
    R = len(rows)
    max_pages = max(max(p // page + 1 for _, _, p in rows), 1) + 1
    shared_pages = {}
    lens = {}
    for pid, n, _ in rows:
        if pid >= 0:
            lens[pid] = n
    need = sum(n // page for n in lens.values()) + sum(p // page + 1 for _, _, p in rows if p >= 0) + 4
    order = list(range(need)) if in_order else torch.randperm(need, generator=g).tolist()
    it = iter(order)
    for pid, n in lens.items():
        shared_pages[pid] = [next(it) for _ in range(n // page)]  # (whole pages; what is left of the prefix is each row's own copy)
    text = {pid: torch.randn(2, n, kv_heads, dim, generator=g).bfloat16() for pid, n in lens.items()}
    kv = torch.full((2, need, kv_heads, page, dim), float("nan"), dtype=torch.bfloat16)
    table = torch.zeros(R, max_pages, dtype=torch.int32)
    per_row = []
    for t, (pid, n, pos) in enumerate(rows):
        own = torch.randn(2, max(pos + 1, 0), kv_heads, dim, generator=g).bfloat16()
        ids = []
        if pid >= 0:
            m = min(n, pos + 1)
            own[:, :m] = text[pid][:, :m]
            ids = list(shared_pages[pid])
            for i, pg in enumerate(ids):
                kv[:, pg] = text[pid][:, i * page:(i + 1) * page].transpose(1, 2)
        while len(ids) * page < pos + 1:
            pg = next(it)
            i = len(ids)
            part = own[:, i * page:(i + 1) * page]
            kv[:, pg, :, :part.shape[1]] = part.transpose(1, 2)
            ids.append(pg)
        if pid >= 0 and n % page and pos + 1 < n:
            raise AssertionError("a row that ends before its prefix needs a prefix of whole pages")
        table[t, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
        per_row.append(own)
    q = (scale_q * torch.randn(R, heads * dim, generator=g)).bfloat16()
    return dict(q=q, k=kv[0], v=kv[1], table=table, rows=rows, per_row=per_row)


def _want(c, heads, kv_heads, dim):
    out, bound = [], []
    for t, own in enumerate(c["per_row"]):
        if own.shape[1] == 0:
            out.append(torch.zeros(heads * dim, dtype=torch.float64))
            bound.append(torch.zeros(heads * dim, dtype=torch.float64))
            continue
        q = c["q"][t].double().view(kv_heads, -1, dim)
        k, v = own.double().permute(0, 2, 1, 3)
        s = q @ k.mT / dim ** 0.5
        p = torch.softmax(s, -1)
        o, a = p @ v, p @ v.abs()
        e = 2 * dim * 2.0 ** -24 * (q.abs() @ k.abs().mT).amax(-1, keepdim=True) / dim ** 0.5 + 2.0 ** -20
        out.append(o.reshape(-1))
        bound.append((2.0 ** -8 * (o.abs() + a) + e * a).reshape(-1))
    return torch.stack(out), torch.stack(bound)


def _call(ops, c, heads, kv_heads, cuda, work=None, slots=None, max_rows=None, out=None, least=0):
    R = len(c["rows"])
    slots = torch.arange(R, dtype=torch.int32) if slots is None else slots
    n = int(slots.max()) + 1
    pid, plen = torch.full((n,), -1, dtype=torch.int32), torch.zeros(n, dtype=torch.int32)
    table = torch.zeros(n, c["table"].shape[1], dtype=torch.int32)
    for t, (i, m, _) in enumerate(c["rows"]):
        pid[slots[t]], plen[slots[t]] = i, m
        table[slots[t]] = c["table"][t]
    d = lambda x: x.to(cuda)
    plan = ops.PrefixPlan(max_rows or R, heads, kv_heads, cuda, least=least)
    ops.prefix_plan(d(slots), d(pid), d(plen), plan)
    pos = torch.tensor([p for _, _, p in c["rows"]], dtype=torch.int32)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    got = ops.paged_attention_shared(d(c["q"]), d(c["k"]), d(c["v"]), d(table), d(slots), d(pos), plan, heads, out=out, work=work, status=status)
    assert int(status) == 0
    return got, plan


SHAPES = [  # heads, key heads, dim, page
    (8, 8, 128, 16), (8, 2, 128, 16), (4, 4, 64, 16), (16, 1, 64, 32), (6, 2, 128, 32), (20, 1, 128, 16), (40, 1, 64, 16)]


@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
@pytest.mark.parametrize("in_order", [False, True])
def test_groups_of_all_kinds(ops, cuda, heads, kv_heads, dim, page, in_order):
    """Two prefixes (one of them no multiple of a page or of a block), rows without any, a prefix of one row, a short one, an empty row, a
    row that ends inside its prefix, and a row that ends right behind it."""
    w = 128 // page * page
    rows = [(0, 5 * w, 5 * w + 40), (1, 200 + page // 2, 300), (-1, 0, 70), (0, 5 * w, 5 * w), (7, 256, 400), (9, 32, 50), (9, 32, 33), (-1, 0, -1),
            (0, 5 * w, 3 * w + 5), (1, 200 + page // 2, 200 + page // 2 - 1), (-1, 0, 0), (0, 5 * w, 5 * w + 700), (0, 5 * w, -1)]
    c = _case(heads, kv_heads, dim, page, rows, seed=heads + dim, in_order=in_order)
    got, plan = _call(ops, c, heads, kv_heads, cuda)
    want, bound = _want(c, heads, kv_heads, dim)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound.clamp(min=1e-30)).max())
    assert int(plan.table[1]) >= 2  # tiles: both prefixes were read together


@pytest.mark.parametrize("heads,kv_heads,n", [(8, 2, 70), (4, 4, 140), (32, 1, 11), (8, 8, 257)])
def test_more_pairs_than_a_tile(ops, cuda, heads, kv_heads, n):
    rows = [(0, 272, 272 + (t * 37) % 90) for t in range(n)] + [(3, 96, 100), (3, 96, 130)]
    c = _case(heads, kv_heads, 128, 16, rows, seed=n)
    got, plan = _call(ops, c, heads, kv_heads, cuda)
    want, bound = _want(c, heads, kv_heads, 128)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
    rt = 128 // (heads // kv_heads)
    assert int(plan.table[1]) == -(-n // rt) + 1


def test_long_own_parts_are_split_and_joined(ops, cuda):
    """Few rows with long texts of their own: several CTAs a row, the last one joins them; the counters are zero again after it."""
    rows = [(0, 128, 4000), (0, 128, 129), (-1, 0, 2111)]
    c = _case(4, 2, 128, 16, rows, seed=3)
    want, bound = _want(c, 4, 2, 128)
    work = ops.new_workspace(ops.paged_attention_shared_workspace(3, 4, 2, 128), cuda)
    first, _ = _call(ops, c, 4, 2, cuda, work=work)
    assert not bool(work[:4096].any())
    err = (first.cpu().double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
    again, _ = _call(ops, c, 4, 2, cuda, work=work)
    assert torch.equal(first, again)


def test_peaked_rows_and_far_scores(ops, cuda):
    """One key far above the others, in the prefix or behind it; scores of some thousands."""
    rows = [(0, 512, 600), (0, 512, 700)]
    c = _case(4, 4, 64, 16, rows, seed=5, scale_q=400.0)
    got, _ = _call(ops, c, 4, 4, cuda)
    want, bound = _want(c, 4, 4, 64)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


def test_slots_in_any_order_and_a_larger_plan(ops, cuda):
    """Slots are not row numbers, the plan has room for more rows, one scratch buffer serves calls of several sizes, and only the given
    columns of the result are written."""
    work = ops.new_workspace(max(ops.paged_attention_shared_workspace(n, 8, 4, 128) for n in (2, 5, 9)), cuda)
    for n in (5, 2, 9):
        rows = [(2 if t % 3 else 5, 160 if t % 3 else 80, 170 + 11 * t) for t in range(n)]
        c = _case(8, 4, 128, 16, rows, seed=n)
        slots = torch.randperm(n + 3, generator=torch.Generator().manual_seed(n))[:n].int()
        whole = torch.full((n + 1, 8 * 128 + 8), 7.0, dtype=torch.bfloat16, device=cuda)
        got, _ = _call(ops, c, 8, 4, cuda, work=work, slots=slots, max_rows=64, out=whole[:n, :1024])
        want, bound = _want(c, 8, 4, 128)
        err = (got.cpu().double() - want).abs()
        assert bool((err <= bound).all()), float((err / bound).max())
        assert bool((whole[n] == 7).all()) and bool((whole[:, 1024:] == 7).all())


def test_small_groups_are_left_to_their_rows(ops, cuda):
    rows = [(0, 512, 512 + t) for t in range(5)]
    c = _case(4, 2, 64, 16, rows, seed=8)
    want, bound = _want(c, 4, 2, 64)
    for least, tiles in ((4 * 512 * 2, 1), (4 * 512 * 2 + 1, 0), (-1, 0)):
        got, plan = _call(ops, c, 4, 2, cuda, least=least)
        assert int(plan.table[1]) == tiles
        err = (got.cpu().double() - want).abs()
        assert bool((err <= bound).all()), float((err / bound).max())


def test_captured_and_replayed_with_other_rows(ops, cuda):
    """A captured step follows its tables: other slots, positions and groups, the same graph."""
    heads, kv_heads, dim, n = 8, 2, 128, 6
    a = [(0, 256, 256 + 9 * t) for t in range(n)]
    b = [(-1, 0, 30), (4, 64, 64), (4, 64, 90), (5, 160, 333), (5, 160, 170), (-1, 0, -1)]
    ca, cb = (_case(heads, kv_heads, dim, 16, r, seed=s) for s, r in enumerate((a, b)))
    pages = max(ca["k"].shape[0], cb["k"].shape[0])
    width = max(ca["table"].shape[1], cb["table"].shape[1])
    z = lambda *s, **k: torch.zeros(*s, device=cuda, **k)
    k, v = (z(pages, kv_heads, 16, dim, dtype=torch.bfloat16) for _ in range(2))
    q, table, pos = z(n, heads * dim, dtype=torch.bfloat16), z(n, width, dtype=torch.int32), z(n, dtype=torch.int32)
    pid, plen, slots = z(n, dtype=torch.int32), z(n, dtype=torch.int32), torch.arange(n, dtype=torch.int32, device=cuda)
    plan, out = ops.PrefixPlan(n, heads, kv_heads, cuda, least=0), z(n, heads * dim, dtype=torch.bfloat16)
    work = ops.new_workspace(ops.paged_attention_shared_workspace(n, heads, kv_heads, dim), cuda)

    def put(c):
        k[:c["k"].shape[0]].copy_(c["k"])
        v[:c["v"].shape[0]].copy_(c["v"])
        q.copy_(c["q"])
        table[:, :c["table"].shape[1]].copy_(c["table"])
        pos.copy_(torch.tensor([r[2] for r in c["rows"]]))
        pid.copy_(torch.tensor([r[0] for r in c["rows"]]))
        plen.copy_(torch.tensor([r[1] for r in c["rows"]]))

    def step():
        ops.prefix_plan(slots, pid, plen, plan)
        ops.paged_attention_shared(q, k, v, table, slots, pos, plan, heads, out=out, work=work)

    put(ca)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for c in (cb, ca, cb):
        put(c)
        for _ in range(2):
            graph.replay()
        want, bound = _want(c, heads, kv_heads, dim)
        err = (out.cpu().double() - want).abs()
        assert bool((err <= bound).all()), float((err / bound.clamp(min=1e-30)).max())


def test_refusals(ops, cuda):
    c = _case(4, 2, 64, 16, [(0, 64, 70), (0, 64, 80)])
    z = lambda *s, **k: torch.zeros(*s, device=cuda, **k)
    i32 = dict(dtype=torch.int32)
    slots, pos, pid = z(2, **i32), z(2, **i32), z(2, **i32)
    q, k, v, table = (c[n].to(cuda) for n in ("q", "k", "v", "table"))
    plan = ops.prefix_plan(slots, pid, pid, ops.PrefixPlan(2, 4, 2, cuda))
    good = dict(q=q, k_pages=k, v_pages=v, block_table=table, row_slot=slots, row_pos=pos, plan=plan, Hq=4)
    bad = [dict(q=q.float()), dict(q=q[:1]), dict(Hq=2), dict(v_pages=v[:1]), dict(row_pos=pos.long()), dict(block_table=table.t()),
           dict(q=q[:, :128]), dict(k_pages=k.transpose(1, 2)), dict(row_slot=slots.cpu()), dict(out=z(2, 255, dtype=torch.bfloat16))]
    for b in bad:
        with pytest.raises(ValueError):
            ops.paged_attention_shared(**{**good, **b})
    err = load("_lib").MloraError
    with pytest.raises(err, match="scratch"):
        ops.paged_attention_shared(**good, work=z(256, dtype=torch.uint8))
    with pytest.raises(err, match="head_dim"):
        wide = ops.prefix_plan(slots, pid, pid, ops.PrefixPlan(2, 4, 2, cuda))
        ops.paged_attention_shared(**{**good, "plan": wide, "k_pages": z(1, 2, 16, 80, dtype=torch.bfloat16), "v_pages": z(1, 2, 16, 80, dtype=torch.bfloat16),
                                      "q": z(2, 320, dtype=torch.bfloat16)})
    with pytest.raises(ValueError):
        ops.PrefixPlan(2000, 4, 2, cuda)
    with pytest.raises(err, match="bad sizes"):
        ops.prefix_plan(slots, pid, pid, ops.PrefixPlan(1, 4, 2, cuda))
    with pytest.raises(err, match="bad sizes"):
        ops.prefix_plan(slots, pid, pid, ops.PrefixPlan(2, 64, 1, cuda))


@pytest.mark.parametrize("heads,kv_heads,dim", [(40, 40, 64), (32, 16, 128), (64, 32, 128)])
def test_many_rows_and_key_heads(ops, cuda, heads, kv_heads, dim):
    """Enough pairs of rows and key heads for the smaller CTAs of the rows' own parts."""
    n = 2100 // kv_heads + 3
    rows = [(t % 3, (96, 160, 272)[t % 3], (96, 160, 272)[t % 3] + (t * 13) % 60) if t % 5 else (-1, 0, t % 40 - 1) for t in range(n)]
    c = _case(heads, kv_heads, dim, 16, rows, seed=n)
    got, plan = _call(ops, c, heads, kv_heads, cuda)
    want, bound = _want(c, heads, kv_heads, dim)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound.clamp(min=1e-30)).max())
    assert int(plan.table[1]) >= 3


def test_slots_that_disagree_share_the_shortest(ops, cuda):
    """One prefix of which the slots give different lengths: the rows still see every token once."""
    rows = [(0, 256, 300), (0, 160, 310), (0, 200, 290)]
    c = _case(4, 2, 64, 16, [(0, 256, p) for _, _, p in rows], seed=11)
    c["rows"] = rows
    got, plan = _call(ops, c, 4, 2, cuda)
    want, bound = _want(c, 4, 2, 64)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= bound).all()) and int(plan.table[1]) == 1, float((err / bound).max())
