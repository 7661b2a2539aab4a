"""How exactly the values are weighted: answers that are small differences of large parts, against the formula in 64 bits.

Half of the keys have weight 1 and value 1, the other half weight c and value -1, so that o = (1 - c) / (1 + c), some 0.001, while A = sum of
softmax |v| is 1.  A weight has 16 bits: 2^-15 A; the result's own rounding 2^-8 |o|; 32-bit scores and sums as in
test_shared_attention_gpu.py.  (c rounded to bf16 would be off by up to 2^-9, more than the whole result.)"""
import pytest
import torch

from conftest import load
from test_shared_attention_gpu import _call

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    return load("ops")


def _second_key(dim):
    """A bf16 number k with exp(-2 k / sqrt(dim)) below 1 and as far from bf16 as it gets."""
    k = torch.linspace(0.005, 0.06, 2000).bfloat16().unique().double()
    c = torch.exp(-2.0 * k / dim ** 0.5)
    return float(k[(c - c.bfloat16().double()).abs().mul(c > 0.996).argmax()])


@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 64), (8, 2, 128), (32, 2, 128)])
@pytest.mark.parametrize("later", [False, True])
def test_small_differences_of_large_parts(ops, cuda, heads, kv_heads, dim, later):
    """``later``: the last block of the prefix has scores that are 4 (2^5.8) larger, which the reference does not follow."""
    page, prefix, rows = 16, 384, [(0, 384, 384 + 20 * t + 1) for t in range(5)]
    last = max(p for _, _, p in rows)
    key = _second_key(dim)
    k, v = torch.zeros(last + 1, kv_heads, dim), torch.ones(last + 1, kv_heads, dim)
    k[1::2, :, 0], v[1::2] = -key, -1.0
    if later:
        k[256:384, :, 1] = 1.0
    q = torch.zeros(len(rows), heads, dim)
    q[:, :, 0], q[:, :, 1] = 2.0, 4.0 * dim ** 0.5 if later else 0.0
    n = prefix // page
    own = -(-(last + 1 - prefix) // page)
    table = torch.tensor([list(range(n)) + [n + t * own + i for i in range(own)] for t in range(len(rows))], dtype=torch.int32)
    pages = torch.zeros(2, n + len(rows) * own, kv_heads, page, dim, dtype=torch.bfloat16)
    padded = torch.zeros(2, (n + own) * page, kv_heads, dim, dtype=torch.bfloat16)
    padded[:, :last + 1] = torch.stack([k, v]).bfloat16()
    for t in range(len(rows)):
        pages[:, table[t].long()] = padded.view(2, n + own, page, kv_heads, dim).transpose(2, 3)
    c = dict(q=q.reshape(len(rows), -1).bfloat16(), k=pages[0], v=pages[1], table=table, rows=rows)
    got, plan = _call(ops, c, heads, kv_heads, cuda)
    assert int(plan.table[1]) >= 1
    for t, (_, _, pos) in enumerate(rows):
        kt, vt = (padded[i, :pos + 1].double().permute(1, 0, 2) for i in (0, 1))
        qt = c["q"][t].double().view(kv_heads, -1, dim)
        o = (torch.softmax(qt @ kt.mT / dim ** 0.5, -1) @ vt).reshape(-1)
        e = 2 * dim * 2.0 ** -24 * float((qt.abs() @ kt.abs().mT).max()) / dim ** 0.5 + 2.0 ** -20
        err = (got[t].cpu().double() - o).abs()
        assert bool((err <= 2.0 ** -8 * o.abs() + 2.0 ** -15 + e).all()), (float(err.max()), float(o.abs().max()))
