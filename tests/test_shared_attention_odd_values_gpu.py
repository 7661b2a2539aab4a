"""Keys that a row does not see or a head scores -inf, with values that are infinite or none, and infinite values that a row does see.

The formula leaves such keys out; what it gives for the others, in 64 bits, is wanted: the same numbers within the bound of
test_shared_attention_gpu.py, the same infinities, and NaN where it has NaN."""
import math

import pytest
import torch

from conftest import load
from test_shared_attention_gpu import _call, _case

pytestmark = pytest.mark.gpu

INF, NAN = math.inf, math.nan


@pytest.fixture(scope="module")
def ops():
    return load("ops")


def _put(c, t, key, k=None, v=None, head=None, col=None):
    """Overwrites a key or a value of row t's sequence (and so of whoever shares its page)."""
    page = c["k"].shape[2]
    at = (int(c["table"][t, key // page]), slice(None) if head is None else head, key % page)
    for pages, x in ((c["k"], k), (c["v"], v)):
        if x is not None:
            pages[at + ((slice(None),) if col is None else (col,))] = x


def _check(ops, c, heads, kv_heads, dim, cuda):
    page = c["k"].shape[2]
    out = torch.full((len(c["rows"]), heads * dim), 5.0, dtype=torch.bfloat16, device=cuda)
    got = _call(ops, c, heads, kv_heads, cuda, out=out)[0].cpu().double()
    finite = 0
    for t, (_, _, pos) in enumerate(c["rows"]):
        if pos < 0:
            assert not bool(got[t].any())
            continue
        ids = c["table"][t, :pos // page + 1].long()
        k, v = (x[ids].double().transpose(0, 1).flatten(1, 2)[:, :pos + 1] for x in (c["k"], c["v"]))  # [key head, key, dim]
        q = c["q"][t].double().view(kv_heads, -1, dim)
        for kh in range(kv_heads):
            for h in range(q.shape[1]):
                s = (q[kh, h] * k[kh]).sum(-1) / dim ** 0.5
                keep = s != -INF
                s, kk, vv = s[keep], k[kh][keep], v[kh][keep]
                p = torch.softmax(s, 0)
                o, a = (p[:, None] * vv).sum(0), (p[:, None] * vv.abs()).sum(0)
                e = 2 * dim * 2.0 ** -24 * float((q[kh, h].abs() * kk.abs()).sum(-1).max()) / dim ** 0.5 + 2.0 ** -20 if len(s) else 0.0
                g = got[t].view(kv_heads, -1, dim)[kh, h]
                ok = torch.where(o.isfinite(), (g - o).abs() <= 2.0 ** -8 * (o.abs() + a) + e * a, torch.where(o.isnan(), g.isnan(), g == o))
                assert bool(ok.all()), (t, kh, h, g[~ok][:4].tolist(), o[~ok][:4].tolist())
                finite += int(o.isfinite().sum())
    return finite


SHAPES = [(8, 2, 128, 16, 5), (6, 2, 64, 32, 6), (7, 1, 64, 16, 5), (32, 32, 64, 16, 65)]


def _rows(n):
    """Ends inside the prefix, behind it, no prefix, and an empty row; the first two of a group see 300 tokens."""
    return [[(0, 288, 300), (0, 288, 420), (0, 288, 150), (-1, 0, 70), (0, 288, 287), (-1, 0, -1)][t % 6] for t in range(n)]


@pytest.mark.parametrize("heads,kv_heads,dim,page,n", SHAPES)
@pytest.mark.parametrize("what", [INF, -INF, NAN])
def test_values_behind_a_row_that_ends_in_the_prefix(ops, cuda, heads, kv_heads, dim, page, n, what):
    """In the same block of keys and in a later one; the rows that see them have them in those columns."""
    c = _case(heads, kv_heads, dim, page, _rows(n), seed=1)
    _put(c, 0, 151, v=what, col=3)
    _put(c, 0, 170, v=what, head=kv_heads - 1, col=9)
    _put(c, 0, 280, v=what, col=5)
    assert _check(ops, c, heads, kv_heads, dim, cuda)


@pytest.mark.parametrize("heads,kv_heads,dim,page,n", SHAPES)
def test_keys_behind_a_row_that_ends_in_the_prefix(ops, cuda, heads, kv_heads, dim, page, n):
    c = _case(heads, kv_heads, dim, page, _rows(n), seed=2)
    _put(c, 0, 200, k=NAN, v=NAN, head=kv_heads - 1)
    assert _check(ops, c, heads, kv_heads, dim, cuda)


@pytest.mark.parametrize("heads,kv_heads,dim,page,n", SHAPES)
@pytest.mark.parametrize("what", [INF, NAN])
def test_keys_that_are_scored_minus_infinity(ops, cuda, heads, kv_heads, dim, page, n, what):
    """In the prefix and behind it, one of a row without a prefix, a whole block, and all tokens behind the prefix of one row."""
    c = _case(heads, kv_heads, dim, page, _rows(n), seed=3)
    c["q"].view(n, heads, dim)[:, :, 0] = 1.0
    for key in [7, 140] + list(range(256, 288)):
        _put(c, 0, key, k=-INF, col=0)
        _put(c, 0, key, v=what)
    for t, keys in ((0, range(288, 301)), (1, (290, 400)), (3, (0, 33))):
        for key in keys:
            _put(c, t, key, k=-INF, col=0)
            _put(c, t, key, v=what, col=2)
    assert _check(ops, c, heads, kv_heads, dim, cuda)


@pytest.mark.parametrize("heads,kv_heads,dim,page,n", SHAPES)
def test_a_row_that_scores_everything_minus_infinity(ops, cuda, heads, kv_heads, dim, page, n):
    """Nothing is left: zeros, and the other rows as they are."""
    c = _case(heads, kv_heads, dim, page, _rows(n), seed=4)
    c["q"].view(n, heads, dim)[:, :, 0] = 0.0
    c["k"][:, :, :, 0] = torch.where(c["k"][:, :, :, 0].isnan(), c["k"][:, :, :, 0], torch.tensor(-3e38).bfloat16())
    c["q"].view(n, heads, dim)[[0, 3], :, 0] = 3e38
    c["v"][:, :, ::3, 1] = torch.where(c["v"][:, :, ::3, 1].isnan(), c["v"][:, :, ::3, 1], torch.tensor(2.0).bfloat16())
    got = _call(ops, c, heads, kv_heads, cuda)[0].cpu()
    assert not bool(got[[0, 3]].any()) and bool(got[1].isfinite().all())


@pytest.mark.parametrize("heads,kv_heads,dim,page,n", SHAPES)
def test_infinite_values_that_are_seen(ops, cuda, heads, kv_heads, dim, page, n):
    """One sign in a column: that infinity; both: NaN."""
    c = _case(heads, kv_heads, dim, page, _rows(n), seed=5, scale_q=0.5)
    _put(c, 0, 20, v=INF, col=1)
    _put(c, 0, 260, v=-INF, col=2)
    _put(c, 0, 30, v=INF, col=4)
    _put(c, 0, 31, v=-INF, col=4)
    _put(c, 0, 295, v=-INF, col=6)
    _put(c, 3, 11, v=INF, col=dim - 1)
    assert _check(ops, c, heads, kv_heads, dim, cuda)
