"""4-bit weights, shared prefixes and token rules together, as a serving step uses them."""
import dataclasses

import pytest
import torch

from conftest import load
from oracle import llama as ollama

pytestmark = pytest.mark.gpu

CFG = dict(name="small", hidden_size=256, intermediate_size=704, num_attention_heads=8, num_hidden_layers=2, num_key_value_heads=2, head_dim=64,
           rms_norm_eps=1e-5, vocab_size=1000, rope_theta=10000.0)


@pytest.fixture(scope="module")
def ops():
    return load("ops")


def _weights():
    synth = load("synth")
    w = {k: v.bfloat16() for k, v in synth.base_weights(CFG).items()}
    ads = [{k: v.bfloat16() for k, v in a.items()} for a in synth.lora_adapters(CFG, 3, 8)]
    return w, ads, [2.0, 1.0, 0.5]


def _as_seen(ops, cuda, w, group, zeros):
    """The weights that the quantised projections multiply, as 32-bit matrices: a projection of the identity gives them exactly."""
    out = {}
    for name, t in w.items():
        out[name] = t
        if "proj" in name:
            q = ops.QuantWeight(t.to(cuda), group, zeros)
            eye = torch.eye(t.shape[1], dtype=torch.bfloat16, device=cuda)
            out[name] = torch.cat([ops.linear(eye[i:i + 16].contiguous(), q, flags=ops.OUT_F32) for i in range(0, t.shape[1], 16)]).T.cpu().contiguous()
    return out


def _engine(weights, cuda, ads=(), scales=(), max_batch=8, **kw):
    model = load("model").PackedLlama(CFG, weights, ads, scales, device=cuda, **kw)
    kv = model.new_cache(max_batch, 4096, 256, 16, max_seq_len=512)
    return model.new_engine(kv, 256)


@pytest.mark.parametrize("group,zeros", [(64, True), (32, False)])
def test_quantised_llama_against_the_oracle(ops, cuda, group, zeros):
    """The quantised model is the full one with the rounded weights: prompts (tensor-core kernel) and decode steps, with adapters."""
    w, ads, scales = _weights()
    seen = _as_seen(ops, cuda, w, group, zeros)
    prompts = load("synth").prompts(4, 40, CFG["vocab_size"])
    ids = [0, 2, -1, 1]
    want_tok, want = ollama.OracleLlama(CFG, seen, ads, scales).greedy([list(p) for p in prompts], ids, 3)
    eng = _engine(w, cuda, ads, scales, weight_bits=4, weight_group=group, weight_zeros=zeros)
    assert eng.m.weight_bytes() < 0.5 * load("model").PackedLlama(CFG, w, device=cuda).weight_bytes() + 2 * 2 * 1000 * 256
    for s in range(4):
        eng.kv.add_sequence(s)
    lg, _ = eng.prefill([0, 1, 2, 3], [list(p) for p in prompts], ids)
    torch.testing.assert_close(lg.cpu(), want[0], atol=2e-2, rtol=1e-2)
    for step in (1, 2):
        lg, _ = eng.decode([0, 1, 2, 3], want_tok[:, step - 1].tolist(), ids)
        torch.testing.assert_close(lg.cpu(), want[step], atol=2e-2, rtol=1e-2)
    eng.check_status()


@pytest.mark.parametrize("bits", [16, 4])
def test_forked_sequences_decode_like_separate_ones(ops, cuda, bits):
    """One prompt run once and forked, against every sequence with a prompt of its own: eager steps and a captured one."""
    w, _, _ = _weights()
    g = torch.Generator().manual_seed(0)
    system = torch.randint(0, 1000, (150,), generator=g).tolist()
    asks = [torch.randint(0, 1000, (n,), generator=g).tolist() for n in (5, 17, 1, 30)]
    kw = dict(weight_bits=4, weight_group=64) if bits == 4 else {}
    a, b = _engine(w, cuda, **kw), _engine(w, cuda, **kw)
    a.prefix_least = 0
    a.kv.add_sequence(99)
    a.extend([99], [system])
    rest = []
    for i, q in enumerate(asks):
        n = a.kv.fork(i, 99)
        assert n == 144
        rest.append(system[n:] + q)
        b.kv.add_sequence(i)
    la, ta = a.extend(range(4), rest)
    lb, tb = b.extend(range(4), [system + q for q in asks])
    torch.testing.assert_close(la, lb, atol=2e-2, rtol=1e-2)
    toks = tb.tolist()
    a.kv.remove_sequence(99)  # (the pages stay while a fork holds them)
    for _ in range(3):
        la, _ = a.decode(range(4), toks, [-1] * 4)
        lb, tb = b.decode(range(4), toks, [-1] * 4)
        torch.testing.assert_close(la, lb, atol=2e-2, rtol=1e-2)
        toks = tb.tolist()
    assert int(a.prefix_plan.table[1]) == 1  # (one tile: the prefix was read once)
    ga, gb = (e.capture_decode(range(4), [-1] * 4, reserve_tokens=8, feed_back=False) for e in (a, b))
    for _ in range(4):
        for e in (a, b):
            e.tokens[:4].copy_(torch.tensor(toks, dtype=torch.int32))
        ga.replay()
        gb.replay()
        torch.testing.assert_close(a.logits[:4], b.logits[:4], atol=2e-2, rtol=1e-2)
        toks = b.next_tok[:4].tolist()
    a.check_status()


def test_everything_in_one_session(ops, cuda):
    """Quantised weights, adapters, a forked prompt and rules: the session's tokens are those of a loop on the host that applies the rules
    to the same logits, and they keep the rules; a request whose grammar allows nothing ends with its first token."""
    w, ads, scales = _weights()
    g = torch.Generator().manual_seed(1)
    system = torch.randint(0, 1000, (96,), generator=g).tolist()
    asks = [torch.randint(0, 1000, (n,), generator=g).tolist() for n in (3, 20, 9, 1, 12)]
    n, steps = len(asks), 12
    words = sorted(torch.randperm(1000, generator=g)[:40].tolist())
    allowed = [None, words, words, [], None]
    kw = dict(repetition=[1.3, 1.0, 1.1, 1.2, 1.0], frequency=0.2, presence=[0.0, 0.4, 0.1, 0.0, 0.0], biases=[None, {words[3]: 4.0}, None, None, {7: 9.0}],
              allowed=allowed)

    def start():
        eng = _engine(w, cuda, ads, scales, weight_bits=4, weight_group=64)
        eng.prefix_least = 0
        eng.kv.add_sequence(99)
        eng.extend([99], [system], [1])
        texts = [system + q for q in asks]
        rest = [t[eng.kv.fork(i, 99):] for i, t in enumerate(texts)]
        lg, _ = eng.extend(range(n), rest, [1] * n)
        return eng, lg, ops.LogitRules.build(1000, n, cuda, prompts=texts, **kw)

    eng, lg, rules = start()
    first = ops.choose_tokens(lg, rules).tolist()
    assert first[3] == -1
    first[3] = 5
    session = load("model").DecodeSession(eng, list(range(n)), [1] * n, first, [steps] * n, rules=rules)
    got = session.run()
    eng.check_status()
    assert rules.answer is None and len(got[3]) == 1 and all(len(t) == steps for i, t in enumerate(got) if i != 3)
    assert set(got[1]) | set(got[2]) <= set(words)

    eng, lg, rules = start()
    said = [[t] for t in first]
    live = [0, 1, 2, 4]
    eng.kv.reserve(0, 1)
    for step in range(steps - 1):
        rows = list(range(n)) if step == 0 else live  # (the session's first step has all of them)
        lg, _ = eng.decode(rows, [said[i][-1] for i in rows], [1] * len(rows))
        r = dataclasses.replace(rules, answer=torch.tensor([s + [0] * (steps - len(s)) for s in said], dtype=torch.int32, device=cuda),
                                answer_len=torch.tensor([len(s) for s in said], dtype=torch.int32, device=cuda))
        tok = ops.choose_tokens(lg.contiguous(), r, row_src=torch.tensor(rows, dtype=torch.int32, device=cuda)).tolist()
        for i, t in zip(rows, tok):
            if i != 3:
                said[i].append(t)
    # the same kernels on the same values; batches of other sizes take other orders of sums, so a near tie may fall the other way: the
    # sequences agree up to there, and most do to the end
    same = [next((k for k, (x, y) in enumerate(zip(a, b)) if x != y), steps) for a, b in zip(got, said)]
    assert sum(same[i] == steps for i in live) >= 3 and all(same[i] >= 2 for i in live)


def test_session_refusals(ops, cuda):
    w, _, _ = _weights()
    eng = _engine(w, cuda)
    eng.kv.add_sequence(0)
    eng.extend([0], [[1, 2, 3]])
    rules = ops.LogitRules.build(1000, 2, cuda, repetition=1.5)
    with pytest.raises(ValueError):
        load("model").DecodeSession(eng, [0], [-1], [4], [3], rules=rules)
    model = load("model").PackedLlama
    for kw in (dict(weight_bits=8), dict(weight_bits=4, weight_group=128), dict(weight_bits=4, weight_group=48)):
        with pytest.raises(ValueError):
            model(CFG, w, device=cuda, **kw)
    registry = load("registry")
    with pytest.raises(ValueError):
        registry.build_model(CFG, w, device=cuda, nonsense=1)
    assert registry.build_model(CFG, w, device=cuda, weight_bits=4, weight_group=64).weight_bits == 4


def test_the_cache_after_a_session_with_rules(ops, cuda):
    """The host's lengths are the device's when a session ends, whichever way its sequences did, and a continuation gives the logits of the
    whole text run at once."""
    w, _, _ = _weights()
    texts = [[5, 17, 3, 8], [9, 2, 40]]

    def start():
        eng = _engine(w, cuda)
        for i, t in enumerate(texts):
            eng.kv.add_sequence(i)
        return eng, eng.extend(range(2), texts)[0]

    eng, _ = start()
    rules = ops.LogitRules.build(1000, 2, cuda, allowed=[None, []])
    with pytest.raises(ValueError, match="first token"):
        load("model").DecodeSession(eng, [0, 1], [-1, -1], [4, -1], [3, 3], rules=rules)
    got = load("model").DecodeSession(eng, [0, 1], [-1, -1], [4, 7], [3, 3], rules=rules).run()
    assert [len(g) for g in got] == [3, 1] and got[1] == [7]
    lengths = eng.kv.seq_lens.cpu().tolist()
    held = [eng.kv.length(i) for i in range(2)]
    assert held == [lengths[eng.kv.slot(i)] for i in range(2)] == [4 + 2, 3 + 1]
    more = [got[0][-1:] + [11], [11]]
    a = eng.extend(range(2), more)[0].clone()
    eng, _ = start()
    b = eng.extend(range(2), [got[0][:-1] + more[0], got[1] + more[1]])[0]
    torch.testing.assert_close(a, b, atol=2e-2, rtol=1e-2)
