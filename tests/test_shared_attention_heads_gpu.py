"""Attention behind shared prefixes for every number of query heads that a CTA of the rows' own parts can have, against the formula in
64 bits with the bound of test_shared_attention_gpu.py.  The result begins as NaN: a head that is not written shows."""
import pytest
import torch

from conftest import load
from test_shared_attention_gpu import _call, _case, _want

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    return load("ops")


@pytest.mark.parametrize("kv_heads,n", [(2, 5), (64, 33)])  # either size of the CTAs (2048 rows x key heads)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rep", [1, 2, 3, 4, 5, 6, 7, 8, 9, 13, 14, 15])
def test_every_head_is_written(ops, cuda, rep, dim, kv_heads, n):
    heads = rep * kv_heads
    rows = [(-1, 0, 20 * t % 47) if t % 4 == 3 else (0, 64, 64 + 7 * t % 30) for t in range(n)]
    c = _case(heads, kv_heads, dim, 16, rows, seed=rep)
    out = torch.full((n, heads * dim), float("nan"), dtype=torch.bfloat16, device=cuda)
    got, plan = _call(ops, c, heads, kv_heads, cuda, out=out)
    want, bound = _want(c, heads, kv_heads, dim)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= bound).all()), (got.cpu().view(n, heads, dim).isnan().any(-1).sum(0).tolist(), float((err / bound).nan_to_num(0).max()))
    assert int(plan.table[1]) >= 1


@pytest.mark.parametrize("rep,splits", [(7, True), (14, False)])
def test_heads_of_64_with_long_own_parts(ops, cuda, rep, splits):
    """The join of several CTAs' ranges, and of more prefix ranges than one pass over the factors has."""
    rows = [(0, 16384, 16384 + 3000), (0, 16384, 16384 + 1), (-1, 0, 2111)] if splits else [(0, 128, 400 + t) for t in range(60)]
    c = _case(rep * 2, 2, 64, 16, rows, seed=rep)
    out = torch.full((len(rows), rep * 128), float("nan"), dtype=torch.bfloat16, device=cuda)
    got, _ = _call(ops, c, rep * 2, 2, cuda, out=out)
    want, bound = _want(c, rep * 2, 2, 64)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).nan_to_num(9).max())
