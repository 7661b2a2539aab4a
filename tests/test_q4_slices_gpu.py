"""4-bit projections with adapters of more rows than one slice of 512: what follows the first slice, and the scratch that slices share.
Bounds as in test_q4_gpu.py."""
import pytest
import torch

from conftest import load
from test_q4_gpu import _bound, _packed, _weights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    return load("ops")


def _adapters(T, N, rank, n, offs, seed):
    """(B, u, slots, scales) and what they add to [T, N], with its bound, in 64 bits."""
    g = torch.Generator().manual_seed(seed)
    n_mod = len(offs) - 1
    B, u = (torch.randn(n, N, rank, generator=g) * 0.2).bfloat16(), torch.randn(T, rank * n_mod, generator=g)
    slots, scales = torch.randint(-1, n + 1, (T,), generator=g).int(), torch.linspace(0.5, 2, n)
    add, bound = torch.zeros(T, N, dtype=torch.float64), torch.zeros(T, N, dtype=torch.float64)
    for i in range(n):
        rows = (slots == i).nonzero()[:, 0]
        for m in range(n_mod):
            cols = slice(offs[m], offs[m + 1])
            um, b = u[rows, m * rank:(m + 1) * rank].double(), B[i, cols].double()
            add[rows, cols] = scales[i].double() * (um @ b.T)
            bound[rows, cols] = (rank + 4) * 2.0 ** -23 * scales[i].double() * (um.abs() @ b.abs().T)
    return B, u, slots, scales, add, bound


@pytest.mark.parametrize("T", [512, 513, 515, 524, 529, 540, 1100])
@pytest.mark.parametrize("rank,n_mod,packed", [(16, 3, True), (16, 1, False), (8, 3, False)])
def test_rows_behind_the_first_slice(ops, cuda, T, rank, n_mod, packed):
    K, N, n = 256, 384, 5
    q, s, z, w = _weights(N, K, 64, True, seed=rank)
    g = torch.Generator().manual_seed(T)
    wide = torch.full((T, K + 8), float("nan"), dtype=torch.bfloat16)
    wide[:, :K] = torch.randn(T, K, generator=g).bfloat16()
    x = wide[:, :K]
    offs = (0, 128, 256, 384) if n_mod == 3 else (0, N)
    B, u, slots, scales, add, bound = _adapters(T, N, rank, n, offs, T + rank)
    want = x.double() @ w.T + add
    limit = _bound(x, w, K) + bound + 2.0 ** -23 * (want.abs() + 1)
    st = ops.LoraStack(torch.zeros(n, rank * n_mod, K, dtype=torch.bfloat16, device=cuda), B.to(cuda),
                       torch.full((n,), rank, dtype=torch.int32, device=cuda), scales.to(cuda), rank, n_mod, offs)
    if packed:
        st.pack_b()
    W = _packed(ops, q, s, z, 64, cuda)
    work = ops.new_workspace(ops.q4_linear_workspace(T, K, N), cuda)
    call = lambda out, flags: ops.linear(wide.to(cuda)[:, :K], W, st, slots.to(cuda), u=u.to(cuda), flags=flags, out=out, work=work)
    out = torch.full((T + 1, N + 12), 7.0, device=cuda)
    got = call(out[:T, :N], ops.OUT_F32)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= limit).all()), float((err / limit).max())
    assert bool((out[T] == 7).all()) and bool((out[:, N:] == 7).all())
    half = torch.full((T + 1, N + 8), 7.0, dtype=torch.bfloat16, device=cuda)
    got = call(half[:T, :N], 0)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= limit + 2.0 ** -8 * want.abs()).all()), float((err / (limit + 2.0 ** -8 * want.abs())).max())
    assert bool((half[T] == 7).all()) and bool((half[:, N:] == 7).all())
    assert torch.equal(got, call(None, 0)) and ops.status_word(work) == 0


@pytest.mark.parametrize("T", [515, 524, 700])
def test_gate_and_up_behind_the_first_slice(ops, cuda, T):
    """silu(g) u as in test_q4_gpu.py: the slope of silu is at most 1.1, __expf and the fast division add 2^-20 of the result."""
    K, N, n, rank = 320, 272, 3, 16
    q, s, z, w = _weights(N, K, 32, False, seed=N)
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(T)).bfloat16()
    B, u, slots, scales, add, bound = _adapters(T, N, 2 * rank, n, (0, N), T)
    pre = x.double() @ w.T + add
    limit = _bound(x, w, K) + bound + 2.0 ** -23 * pre.abs()
    st = ops.LoraStack(torch.zeros(n, 2 * rank, K, dtype=torch.bfloat16, device=cuda), B.to(cuda), torch.full((n,), rank, dtype=torch.int32, device=cuda),
                       scales.to(cuda), rank, 2, (0, N // 2, N))
    gate, up = pre.view(T, -1, 2, 8).unbind(2)
    eg, eu = limit.view(T, -1, 2, 8).unbind(2)
    act = gate * torch.sigmoid(gate)
    want = (act * up).reshape(T, N // 2)
    limit = (1.1 * eg * (up.abs() + eu) + act.abs() * eu + 2.0 ** -20 * (act * up).abs() + 2.0 ** -24).reshape(T, N // 2) + 2.0 ** -23 * want.abs()
    out = torch.full((T + 1, N // 2 + 3), 7.0, device=cuda)
    got = ops.linear(x.to(cuda), _packed(ops, q, s, z, 32, cuda), st, slots.to(cuda), u=u.to(cuda), flags=ops.SILU_MUL | ops.OUT_F32, out=out[:T, :N // 2])
    err = (got.cpu().double() - want).abs()
    assert bool((err <= limit).all()), float((err / limit).max())
    assert bool((out[T] == 7).all()) and bool((out[:, N // 2:] == 7).all())
