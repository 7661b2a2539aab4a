"""Into how many key ranges a plan cuts a prefix, and their join."""
import pytest
import torch

from conftest import load
from test_shared_attention_gpu import _call, _case, _want

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    return load("ops")


@pytest.mark.parametrize("rows,tokens,kv_heads,rep", [(2, 32768, 1, 8), (16, 32768, 1, 8), (8, 16384, 2, 7), (4, 8192, 2, 4), (2, 256, 8, 4), (128, 32768, 8, 4)])
def test_a_long_prefix_is_not_cut_into_single_blocks(ops, cuda, rows, tokens, kv_heads, rep):
    """A row joins its ranges one after the other: with few tiles a prefix is cut into fewer than there are SMs for."""
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)
    plan = ops.PrefixPlan(rows, kv_heads * rep, kv_heads, cuda, least=0)
    ops.prefix_plan(i32(list(range(rows))), i32([3] * rows), i32([tokens] * rows), plan)
    head = plan.table[:4].tolist()
    blocks, tiles = -(-tokens // 128), -(-rows // (128 // rep))
    ranges, left = divmod(head[2], tiles * kv_heads)
    assert head[1] == tiles and not left and head[3] == rows * ranges
    assert 1 <= ranges <= min(blocks, 4 * blocks ** 0.5 + 2)


@pytest.mark.parametrize("dim,kv_heads,rep", [(64, 1, 8), (128, 1, 3), (64, 2, 5)])
def test_many_ranges_of_the_prefix_and_of_the_rows_own_tokens(ops, cuda, dim, kv_heads, rep):
    """More than one pass over the factors of the join has: ranges of the prefix behind those of a long text of the row's own."""
    rows = [(0, 32768, 32768 + 9000), (0, 32768, 32768), (0, 32768, 32768 + 300)]
    c = _case(kv_heads * rep, kv_heads, dim, 16, rows, seed=rep)
    out = torch.full((3, kv_heads * rep * dim), float("nan"), dtype=torch.bfloat16, device=cuda)
    got, plan = _call(ops, c, kv_heads * rep, kv_heads, cuda, out=out)
    assert int(plan.table[3]) // 3 >= 32  # (and up to 32 of the row's own)
    want, bound = _want(c, kv_heads * rep, kv_heads, dim)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).nan_to_num(9).max())


@pytest.mark.parametrize("rows,tokens,kv_heads,together", [(2, 8192, 8, False), (2, 65536, 32, False), (3, 32768, 8, False), (4, 1024, 1, True), (4, 1023, 8, False),
                                                           (8, 512, 8, False), (32, 512, 32, True), (32, 208, 32, True),  # (31 x 208 x 32 = 206336)
                                                           (32, 192, 32, False), (128, 64, 32, True)])
def test_which_groups_are_taken_together(ops, cuda, rows, tokens, kv_heads, together):
    """Where the caller does not say what a group has to save: rows enough, and a long prefix or many reads."""
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)
    plan = ops.PrefixPlan(rows + 1, kv_heads, kv_heads, cuda)
    ops.prefix_plan(i32(list(range(rows + 1))), i32([-1] + [3] * rows), i32([0] + [tokens] * rows), plan)
    assert bool(int(plan.table[1])) == together
