"""Projections with 4-bit weights, against the formula in 64 bits.

The integers q - z are exact and the sums are 32-bit, so with S = sum over k of |x W| an output is off by at most half a step of its own
type, and what 32-bit sums cost: 2^-23 S for every one of the about 16 + in / 16 additions in a row that a term goes through (tensor
cores may drop what they should round, hence a whole step of 2^-23; the scaled groups and the joined shares count as additions too).
An adapter's share has products of r terms more, an activation the steps of its own formula (written at the test)."""
import pytest
import torch

from conftest import load

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    return load("ops")


def _weights(N, K, group, zeros, seed, extremes=False):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(0, 16, (N, K), generator=g, dtype=torch.uint8)
    if extremes:
        q[:, ::2], q[:, 1::2] = 0, 15
    s = ((0.5 + torch.rand(N, K // group, generator=g)) * K ** -0.5 / 4).bfloat16()
    z = torch.randint(0, 16, (N, K // group), generator=g, dtype=torch.uint8) if zeros else None
    w = (q.double() - (8.0 if z is None else z.double().repeat_interleave(group, 1))) * s.double().repeat_interleave(group, 1)
    return q, s, z, w


def _bound(x, w, K):
    return (16 + K / 16) * 2.0 ** -23 * (x.double().abs() @ w.abs().T)


def _packed(ops, q, s, z, group, cuda):
    return ops.QuantWeight.from_integers(q.to(cuda), s.to(cuda), None if z is None else z.to(cuda), group=group)


CASES = [  # rows, in, out
    (1, 32, 1), (1, 4096, 4096), (2, 96, 500), (3, 160, 130), (5, 11008, 257), (8, 512, 16), (9, 544, 48), (16, 4096, 2100), (13, 352, 9500),
    (17, 32, 1), (17, 4096, 128), (31, 96, 300), (33, 2080, 1000), (64, 512, 4096), (65, 160, 130), (101, 5120, 1100), (128, 96, 129), (129, 544, 260),
    (300, 1024, 513), (40, 11008, 130),
    (5, 96, 60000), (33, 160, 40000), (70, 96, 60000), (130, 160, 20001)]  # (inputs that end inside a block, many tiles per CTA)


@pytest.mark.parametrize("T,K,N", CASES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_against_the_formula(ops, cuda, T, K, N, group, zeros):
    K = -(-K // group) * group
    q, s, z, w = _weights(N, K, group, zeros, seed=T + K + N)
    g = torch.Generator().manual_seed(T)
    wide = torch.full((T, K + 8), float("nan"), dtype=torch.bfloat16)
    wide[:, :K] = torch.randn(T, K, generator=g).bfloat16()
    wide[:, 0] *= 64  # (one input far above the others)
    x = wide[:, :K]
    W = _packed(ops, q, s, z, group, cuda)
    want, b32 = x.double() @ w.T, _bound(x, w, K)
    xd = wide.to(cuda)[:, :K]  # (behind a row lies what is no input)
    out = torch.full((T + 1, N + 5), 7.0, device=cuda)
    got = ops.linear(xd, W, flags=ops.OUT_F32, out=out[:T, :N])
    err = (got.cpu().double() - want).abs()
    assert bool((err <= b32 + 2.0 ** -24 * want.abs()).all()), float((err / b32).max())
    assert bool((out[T] == 7).all()) and bool((out[:, N:] == 7).all())
    got = ops.linear(xd, W)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= b32 + 2.0 ** -8 * want.abs()).all()), float((err / (b32 + 2.0 ** -8 * want.abs())).max())
    assert torch.equal(got, ops.linear(xd, W))  # (the same bits again)


@pytest.mark.parametrize("T", [1, 8, 16, 17, 100, 200])
@pytest.mark.parametrize("rank,packed,n_mod", [(8, False, 1), (16, False, 3), (16, True, 3), (32, True, 1), (64, True, 3), (64, False, 1), (40, False, 1)])
def test_with_adapters(ops, cuda, T, rank, packed, n_mod):
    """Rows without an adapter, with one that does not exist, neighbours that share one; modules that own ranges of the outputs."""
    K, N, n = 256, 384, 5
    q, s, z, w = _weights(N, K, 64, True, seed=rank)
    g = torch.Generator().manual_seed(T + rank)
    x = torch.randn(T, K, generator=g).bfloat16()
    offs = (0, 128, 256, 384) if n_mod == 3 else (0, N)
    A = (torch.randn(n, rank * n_mod, K, generator=g) * K ** -0.5).bfloat16()
    B = (torch.randn(n, N, rank, generator=g) * 0.2).bfloat16()
    u = torch.randn(T, rank * n_mod, generator=g)
    scales = torch.linspace(0.5, 2, n)
    slots = torch.randint(-1, n + 1, (T,), generator=g).sort().values.int() if T > 20 else torch.randint(-1, n + 1, (T,), generator=g).int()
    want, bound = x.double() @ w.T, _bound(x, w, K)
    for t in range(T):
        i = int(slots[t])
        if 0 <= i < n:
            for m in range(n_mod):
                lo, hi = offs[m], offs[m + 1]
                um = u[t, m * rank:(m + 1) * rank].double()
                want[t, lo:hi] += scales[i].double() * (B[i, lo:hi].double() @ um)
                bound[t, lo:hi] += (rank + 4) * 2.0 ** -23 * scales[i].double() * (B[i, lo:hi].double().abs() @ um.abs())
    st = ops.LoraStack(A.to(cuda), B.to(cuda), torch.full((n,), rank, dtype=torch.int32, device=cuda), scales.to(cuda), rank, n_mod, offs)
    if packed:
        st.pack_b()
    W = _packed(ops, q, s, z, 64, cuda)
    got = ops.linear(x.to(cuda), W, st, slots.to(cuda), u=u.to(cuda), flags=ops.OUT_F32)
    err = (got.cpu().double() - want).abs()
    limit = bound + 2.0 ** -23 * (want.abs() + 1)
    assert bool((err <= limit).all()), float((err / limit).max())
    shrunk = ops.linear(x.to(cuda), W, st, slots.to(cuda), flags=ops.OUT_F32)  # (with the shrink in the call)
    again = ops.linear(x.to(cuda), W, st, slots.to(cuda), u=ops.lora_shrink(x.to(cuda), st, slots.to(cuda)), flags=ops.OUT_F32, with_shrink=True)
    assert torch.equal(shrunk, again)


@pytest.mark.parametrize("T,N", [(1, 16), (7, 1040), (16, 4096), (30, 272), (128, 640), (150, 96)])
@pytest.mark.parametrize("rank", [0, 16])
def test_gate_and_up(ops, cuda, T, N, rank):
    """silu(g) u with g and u off by their bounds: the slope of silu is at most 1.1, __expf and the fast division add 2^-20 of the result."""
    K, n = 320, 3
    q, s, z, w = _weights(N, K, 32, False, seed=N)
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, K, generator=g).bfloat16()
    pre, bound = x.double() @ w.T, _bound(x, w, K)
    st = u = slots = None
    if rank:
        B = (torch.randn(n, N, 2 * rank, generator=g) * 0.2).bfloat16()
        u, slots, scales = torch.randn(T, 2 * rank, generator=g), torch.randint(-1, n, (T,), generator=g).int(), torch.tensor([1.0, 0.5, 2.0])
        for t in range(T):
            i = int(slots[t])
            if i >= 0:
                pre[t] += scales[i].double() * (B[i].double() @ u[t].double())
                bound[t] += (2 * rank + 4) * 2.0 ** -23 * scales[i].double() * (B[i].double().abs() @ u[t].double().abs())
        st = ops.LoraStack(torch.zeros(n, 2 * rank, K, dtype=torch.bfloat16, device=cuda), B.to(cuda), torch.full((n,), rank, dtype=torch.int32, device=cuda),
                           scales.to(cuda), rank, 2, (0, N // 2, N))
        u, slots = u.to(cuda), slots.to(cuda)
    bound += 2.0 ** -23 * pre.abs()
    v, e = pre.view(T, -1, 2, 8), bound.view(T, -1, 2, 8)
    gate, up = v[:, :, 0], v[:, :, 1]
    silu = gate * torch.sigmoid(gate)
    want = (silu * up).reshape(T, -1)
    limit = (1.1 * e[:, :, 0] * (up.abs() + e[:, :, 1]) + silu.abs() * e[:, :, 1]).reshape(T, -1) + (2.0 ** -8 + 2.0 ** -20) * want.abs()
    got = ops.linear(x.to(cuda), _packed(ops, q, s, z, 32, cuda), st, slots, u=u, flags=ops.SILU_MUL)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= limit).all()), float((err / limit).max())


@pytest.mark.parametrize("T", [3, 50])
def test_activations(ops, cuda, T):
    """relu(y)^2 and gelu(y): slopes of at most 2 |y| and 1.13."""
    K, N = 128, 200
    q, s, z, w = _weights(N, K, 128, True, seed=1)
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(T)).bfloat16()
    y, b = x.double() @ w.T, _bound(x, w, K)
    W = _packed(ops, q, s, z, 128, cuda)
    for flag, want, slope in ((ops.ACT_RELU2, y.clamp(min=0) ** 2, 2 * y.abs() + 2 * b), (ops.ACT_GELU, 0.5 * y * (1 + torch.erf(y / 2 ** 0.5)), 1.13)):
        got = ops.linear(x.to(cuda), W, flags=flag | ops.OUT_F32)
        err = (got.cpu().double() - want).abs()
        limit = slope * b + 2.0 ** -21 * (want.abs() + y.abs())
        assert bool((err <= limit).all()), float((err / limit).max())


@pytest.mark.parametrize("T", [4, 40])
def test_extreme_integers(ops, cuda, T):
    """0 and 15 in turn, all inputs alike: sums that cancel, and sums that do not."""
    K, N = 1024, 256
    q, s, z, w = _weights(N, K, 128, False, seed=2, extremes=True)
    x = torch.ones(T, K).bfloat16()
    x[1::2] = torch.tensor([1.0, -1.0]).repeat(K // 2).bfloat16()
    want, b = x.double() @ w.T, _bound(x, w, K)
    got = ops.linear(x.to(cuda), _packed(ops, q, s, z, 128, cuda), flags=ops.OUT_F32)
    assert bool(((got.cpu().double() - want).abs() <= b + 2.0 ** -24 * want.abs()).all())


@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True), (128, False)])
def test_quantising(ops, cuda, group, zeros):
    """Every weight goes to its nearest value: at most half a scale off, one and a half where rounding the scale (2^-8) cut the range; an
    identity shows the weights that a projection sees."""
    N, K = 70, 256
    g = torch.Generator().manual_seed(group)
    W = (torch.randn(N, K, generator=g) * 0.05).bfloat16()
    W[3] = 0
    W[4, :group] = W[4, :group].abs()
    W[5, :group] = -W[5, :group].abs()
    Q = ops.QuantWeight(W.to(cuda), group, zeros)
    seen = torch.cat([ops.linear(torch.eye(K)[i:i + 16].bfloat16().to(cuda), Q, flags=ops.OUT_F32) for i in range(0, K, 16)]).T.cpu().double()
    again = ops.linear(torch.eye(K).bfloat16().to(cuda), Q, flags=ops.OUT_F32).T.cpu().double()
    assert torch.equal(seen, again)  # (both kernels: one term per sum)
    v = W.double().view(N, -1, group)
    lo, hi = v.amin(-1).clamp(max=0), v.amax(-1).clamp(min=0)
    scale = (hi - lo) / 15 if zeros else torch.maximum(hi, -lo) / 7
    err = (seen.view(N, -1, group) - v).abs()
    # a value at the edge of the range loses 15 steps of the scale's rounding (2^-8 each) and half a step of the zero point's
    limit = scale[..., None] * (0.5 * (1 + 2.0 ** -8) + 15 * 2.0 ** -8 + (0.5 if zeros else 0.0)) + 1e-9
    assert bool((err <= limit).all()), float((err / limit.clamp(min=1e-30)).max())
    assert not bool(seen[3].any())


def test_one_scratch_for_all_shapes_and_captured(ops, cuda):
    g = torch.Generator().manual_seed(0)
    shapes = [(40, 512, 2000), (100, 4096, 300), (17, 64, 40), (300, 256, 700)]
    work = ops.new_workspace(max(ops.q4_linear_workspace(*s) for s in shapes), cuda)
    calls = []
    for T, K, N in shapes:
        q, s, z, w = _weights(N, K, 64, True, seed=N)
        x = torch.randn(T, K, generator=g).bfloat16()
        calls.append((x.to(cuda), _packed(ops, q, s, z, 64, cuda), torch.empty(T, N, device=cuda)))
    run = lambda: [ops.linear(x, W, flags=ops.OUT_F32, out=y, work=work) for x, W, y in calls]
    want = [y.clone() for y in run()]
    assert ops.status_word(work) == 0 and not bool(work[256:256 + 2048].any())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for _, _, y in calls:
        y.zero_()
    for _ in range(3):
        graph.replay()
    assert all(torch.equal(y, v) for (_, _, y), v in zip(calls, want))


def test_empty_and_refusals(ops, cuda):
    q, s, z, _ = _weights(64, 128, 64, True, seed=0)
    W = _packed(ops, q, s, z, 64, cuda)
    x = torch.zeros(20, 128, dtype=torch.bfloat16, device=cuda)
    assert ops.linear(x[:0], W).shape == (0, 64)
    u8 = lambda *n: torch.zeros(*n, dtype=torch.uint8, device=cuda)
    sc = torch.ones(64, 2, dtype=torch.bfloat16, device=cuda)
    for bad in (lambda: ops.QuantWeight(torch.zeros(64, 100, dtype=torch.bfloat16, device=cuda), 64), lambda: ops.QuantWeight(x.float(), 64),
                lambda: ops.QuantWeight(x, 48), lambda: ops.QuantWeight.from_integers(u8(64, 128) + 16, sc, group=64),
                lambda: ops.QuantWeight.from_integers(u8(64, 128), sc.float(), group=64), lambda: ops.QuantWeight.from_integers(u8(64, 128), sc, group=128),
                lambda: ops.QuantWeight.from_integers(u8(64, 128), sc, u8(64, 1), group=64), lambda: ops.linear(x.float(), W),
                lambda: ops.linear(x[:, :64], W), lambda: ops.linear(x, W, out=torch.empty(20, 64, device=cuda)),
                lambda: ops.linear(x, W, work=u8(256)), lambda: ops.linear(x.t(), W)):
        with pytest.raises(ValueError):
            bad()
    err = load("_lib").MloraError
    with pytest.raises(err, match="alignment"):
        ops.linear(torch.zeros(21 * 128, dtype=torch.bfloat16, device=cuda)[1:1 + 2560].view(20, 128), W)
    with pytest.raises(err, match="sixteens"):
        q2, s2, z2, _ = _weights(40, 128, 64, True, seed=0)
        ops.linear(x, _packed(ops, q2, s2, z2, 64, cuda), flags=ops.SILU_MUL)


def test_paths_without_integers_refuse_them(ops, cuda):
    """The folded norm and the one-launch layer read bf16 weights: packed integers are refused before a launch."""
    q, s, z, _ = _weights(64, 128, 64, True, seed=0)
    W = _packed(ops, q, s, z, 64, cuda)
    x = torch.zeros(4, 128, dtype=torch.bfloat16, device=cuda)
    y = torch.zeros(4, 64, dtype=torch.bfloat16, device=cuda)
    with pytest.raises(ValueError, match="bf16 weights"):
        ops.linear_norm(x, W, res=torch.zeros(4, 64, device=cuda), norm_w=y[0], sumsq_out=torch.zeros(32, device=cuda))
    with pytest.raises(ValueError, match="PackedWeight"):
        ops.decode_chain([ops.ChainStep(x=x, W=W, y=y)], None, None, None, 0, ops.new_workspace(1 << 20, cuda))
