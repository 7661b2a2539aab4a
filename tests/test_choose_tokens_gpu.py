"""The next token under penalties, biases and masks.  The rules are a fixed order of single 32-bit operations, so the logits after them
have the bits of the same operations in numpy, and the tokens are equal."""
import numpy as np
import pytest
import torch

from conftest import load

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    return load("ops")


def _plain(logits, src, rep=None, freq=None, pres=None, prompts=None, answers=None, biases=None, allowed=None):
    """(tokens, logits after the rules), row by row in numpy's 32-bit arithmetic."""
    l = logits.copy()
    tok = []
    for t, s in enumerate(src):
        row = l[t]
        if 0 <= s < 10 ** 6:
            p, a = (prompts[s] if prompts else []), (answers[s] if answers else [])
            f = lambda v, d: np.float32(d if v is None else v[s])
            r, fr, pr = f(rep, 1), f(freq, 0), f(pres, 0)
            for v in sorted(set(p) | set(a)):
                if not 0 <= v < row.size:
                    continue
                x = row[v] / r if row[v] > 0 else row[v] * r
                x = np.float32(x - np.float32(fr * np.float32(a.count(v))))
                row[v] = np.float32(x - pr) if v in a else x
            for v, b in sorted((biases[s] or {}).items() if biases else []):
                row[v] = np.float32(row[v] + np.float32(b))
            if allowed and allowed[s] is not None:
                keep = np.zeros(row.size, bool)
                keep[list(allowed[s])] = True
                row[~keep] = -np.inf
        clean = np.where(np.isnan(row), -np.inf, row)
        tok.append(int(clean.argmax()) if clean.max() > -np.inf else -1)
    return tok, l


def _rules(ops, cuda, V, n, rep, freq, pres, prompts, answers, biases, allowed):
    r = ops.LogitRules.build(V, n, cuda, rep, freq, pres, prompts, biases, allowed)
    if answers is not None:
        width = max([len(a) for a in answers] + [1])
        r.answer = torch.tensor([a + [0] * (width - len(a)) for a in answers], dtype=torch.int32, device=cuda)
        r.answer_len = torch.tensor([len(a) for a in answers], dtype=torch.int32, device=cuda)
    return r


def _random(seed, V, n):
    g = np.random.default_rng(seed)
    text = lambda m: [int(x) for x in (V * g.random(m) ** 2).astype(int)]
    prompts = [text(int(g.integers(0, 3000))) for _ in range(n)]
    answers = [text(int(g.integers(0, 900))) for _ in range(n)]
    rep, freq, pres = (g.choice(v, n).astype(np.float32) for v in ([1.0, 1.2, 0.8], [0.0, 0.3, -0.1], [0.0, 0.6]))
    sets = [{int(v): float(b) for v, b in zip(g.integers(0, V, 50), g.normal(size=50) * 4)} for _ in range(3)] + [None]
    biases = [sets[i] for i in g.integers(0, 4, n)]
    masks = [sorted({int(v) for v in g.integers(0, V, m)}) for m in (1, 40, max(V // 2, 1))] + [None, []]
    allowed = [masks[i] for i in g.integers(0, 5, n)]
    logits = (g.normal(size=(n, V)) * 3).astype(np.float32)
    logits[:, :: 7] = np.round(logits[:, :: 7])  # (ties)
    return logits, rep, freq, pres, prompts, answers, biases, allowed


@pytest.mark.parametrize("V,n", [(1, 3), (31, 2), (33, 5), (1000, 4), (4096, 2), (4097, 3), (32000, 9), (65537, 2), (128000, 3)])
@pytest.mark.parametrize("which", ["all", "penalties", "biases", "masks", "none"])
def test_every_rule(ops, cuda, V, n, which):
    logits, rep, freq, pres, prompts, answers, biases, allowed = _random(V + n, V, n)
    pen, bi, ma = which in ("all", "penalties"), which in ("all", "biases"), which in ("all", "masks")
    a = dict(rep=rep if pen else None, freq=freq if pen else None, pres=pres if pen else None, prompts=prompts if pen else None,
             answers=answers if pen else None, biases=biases if bi else None, allowed=allowed if ma else None)
    rules = _rules(ops, cuda, V, n, **a)
    tok, after = _plain(logits, range(n), **a)
    x = torch.from_numpy(logits).to(cuda)
    kept = torch.full((n, V + 3), 5.0, device=cuda)  # (an odd pitch, and columns that are not the call's)
    got = ops.choose_tokens(x, rules, logits_out=kept[:, :V])
    assert got.tolist() == tok
    assert np.array_equal(kept[:, :V].cpu().numpy(), after) and bool((kept[:, V:] == 5).all())
    assert torch.equal(x.cpu(), torch.from_numpy(logits))
    assert ops.choose_tokens(x, rules).tolist() == tok
    assert ops.choose_tokens(x, rules, logits_out=x).tolist() == tok and np.array_equal(x.cpu().numpy(), after)  # in place


def test_rows_of_requests_and_padding(ops, cuda):
    """Rows name their requests in any order, twice too; a row of padding has no rules; rows of a column slice."""
    V, n = 5000, 4
    logits, rep, freq, pres, prompts, answers, biases, allowed = _random(1, V, n)
    a = dict(rep=rep, freq=freq, pres=pres, prompts=prompts, answers=answers, biases=biases, allowed=allowed)
    src = [2, -1, 0, 2, 10 ** 7, 3]
    wide = np.random.default_rng(2).normal(size=(6, V + 9)).astype(np.float32)
    tok, after = _plain(wide[:, 2:V + 2].copy(), src, **a)
    x = torch.from_numpy(wide).to(cuda)[:, 2:V + 2]
    kept = torch.empty(6, V, device=cuda)
    got = ops.choose_tokens(x, _rules(ops, cuda, V, n, **a), row_src=torch.tensor(src, dtype=torch.int32, device=cuda), logits_out=kept)
    assert got.tolist() == tok and np.array_equal(kept.cpu().numpy(), after)


def test_infinities_and_nan(ops, cuda):
    V = 300
    x = np.zeros((6, V), np.float32)
    x[0] = -np.inf
    x[1], x[1, 7] = np.nan, -5.0
    x[2, 9], x[2, 200] = np.inf, np.inf
    x[3] = np.nan
    x[4, 0], x[4, 1:] = -0.0, -1.0
    x[4, 50] = 0.0
    x[5, 3] = np.nan  # masked: gone
    allowed = [None] * 5 + [[5, 6]]
    rules = ops.LogitRules.build(V, 6, cuda, allowed=allowed)
    kept = torch.empty(6, V, device=cuda)
    assert ops.choose_tokens(torch.from_numpy(x).to(cuda), rules, logits_out=kept).tolist() == [-1, 7, 9, -1, 0, 5]
    assert bool((kept[5] == -np.inf).sum() == V - 2) and not bool(kept[5].isnan().any())


def test_tables_out_of_range_are_no_rules(ops, cuda):
    """Texts with tokens outside the vocabulary, lengths beyond the tables, sets and masks that do not exist."""
    V, n = 100, 2
    x = torch.linspace(-1, 1, V, device=cuda).repeat(n, 1).contiguous()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)
    f32 = lambda v: torch.tensor(v, device=cuda)
    r = ops.LogitRules(repetition=f32([2.0, 2.0]), frequency=f32([0.5, 0.5]), presence=f32([0.25, 0.25]), prompt=i32([[99, -4, 400], [7, 7, 7]]),
                       prompt_len=i32([10 ** 6, -3]), answer=i32([[98, 98], [1, 1]]), answer_len=i32([2, 0]), bias_set=i32([5, 0]), bias_start=i32([0, 2]),
                       bias_token=i32([4, 4]), bias_value=f32([1.5, 1.25]), mask_of=i32([9, -7]), masks=i32([[0] * 4]))
    kept = torch.empty_like(x)
    tok = ops.choose_tokens(x, r, logits_out=kept).tolist()
    want = x.clone()
    want[0, 99] /= 2
    want[0, 98] = want[0, 98] / 2 - 0.5 * 2 - 0.25
    want[1, 4] += 2.75
    assert torch.equal(kept, want) and tok == want.argmax(1).tolist()


def test_a_decode_loop_captured(ops, cuda):
    """The answer grows between replays of one graph: every step sees the tokens before it."""
    V, n, steps = 700, 3, 6
    g = torch.Generator().manual_seed(0)
    x = torch.randn(n, V, generator=g).to(cuda)
    r = ops.LogitRules.build(V, n, cuda, repetition=1.5, frequency=0.75, presence=0.5, prompts=[[1, 2], [], [5]])
    r.answer, r.answer_len = torch.zeros(n, steps, dtype=torch.int32, device=cuda), torch.zeros(n, dtype=torch.int32, device=cuda)
    out = torch.empty(n, dtype=torch.int32, device=cuda)
    ops.choose_tokens(x, r, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.choose_tokens(x, r, out=out)
    said = [[] for _ in range(n)]
    for i in range(steps):
        graph.replay()
        want, _ = _plain(x.cpu().numpy(), range(n), [1.5] * n, [0.75] * n, [0.5] * n, [[1, 2], [], [5]], said)
        assert out.tolist() == want
        for s, t in zip(said, want):
            s.append(t)
        r.answer[:, i] = out
        r.answer_len += 1


def test_refusals(ops, cuda):
    V, n = 64, 2
    x = torch.zeros(n, V, device=cuda)
    r = ops.LogitRules.build(V, n, cuda, repetition=1.5, prompts=[[1], [2]], biases=[{3: 1.0}, None], allowed=[[1], None])
    import dataclasses
    bad = [dict(repetition=r.repetition.double()), dict(prompt=r.prompt.long()), dict(prompt_len=None), dict(bias_value=r.bias_value.double()),
           dict(masks=r.masks[:, :1].contiguous()), dict(mask_of=r.mask_of.cpu()), dict(presence=torch.zeros(5, device=cuda)), dict(bias_token=None)]
    for b in bad:
        with pytest.raises(ValueError):
            ops.choose_tokens(x, dataclasses.replace(r, **b))
    with pytest.raises(ValueError):
        ops.choose_tokens(x.half(), r)
    with pytest.raises(ValueError):
        ops.choose_tokens(torch.zeros(n + 1, V, device=cuda), r)  # (three rows, rules of two requests)
    with pytest.raises(ValueError):
        ops.choose_tokens(x, r, out=torch.zeros(n, device=cuda))
    for kw in (dict(biases=[{V: 1.0}, None]), dict(allowed=[[V], None]), dict(allowed=[[-1], None]), dict(prompts=[[1]]), dict(repetition=[1.0, 2.0, 3.0])):
        with pytest.raises(ValueError):
            ops.LogitRules.build(V, n, cuda, **kw)


def test_a_table_that_grows_in_place(ops, cuda):
    """Rules whose answers' buffer is resized in place between calls are read from where it lies then."""
    V = 500
    rules = ops.LogitRules(frequency=torch.full((2,), 100.0, device=cuda), answer=torch.full((2, 4), 7, dtype=torch.int32, device=cuda),
                           answer_len=torch.tensor([1, 1], dtype=torch.int32, device=cuda))
    logits = torch.zeros(2, V, device=cuda)
    logits[:, 7], logits[:, 9], logits[:, 11] = 3.0, 2.0, 1.0
    assert ops.choose_tokens(logits, rules).tolist() == [9, 9]
    rules.answer.resize_(2, 100000)
    rules.answer.zero_()
    rules.answer[:, 0], rules.answer[:, 1], rules.answer[:, 2] = 7, 9, 5
    rules.answer_len.fill_(3)
    assert ops.choose_tokens(logits, rules).tolist() == [11, 11]
