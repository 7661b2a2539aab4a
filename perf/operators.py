"""Operators of a serving step: projections with 4-bit weights and adapters, attention of a batch that shares long prefixes, and
the choice of the next tokens under penalties, biases and masks.

Widths, heads, feed-forwards, ranks and vocabularies are those of ``synth.py``'s Llama configurations (7B- and 13B-shaped) and of the
benchmark's workloads, or generic ones.  Inputs are random, from the seed.
"""
from __future__ import annotations

import importlib
import math

import torch

own = False  # True: the framework's operators; False: the same in elementary torch operations

PKG = "tensor-program-optimization-with-auto-batching_b200"


def _ops():
    return importlib.import_module(PKG + ".ops")


def listed():
    return [
        # the output projection of one user's request: a step's latency is the time between two tokens
        _proj("q4 1 row 4096-4096", rows=1, k=4096, n=4096, group=128),
        # the down projection of a few requests with adapters, fine groups with zero points
        _proj("q4 7 rows 11008-4096 adapters", rows=7, k=11008, n=4096, group=32, zeros=True, rank=16, adapters=16),
        # gate and up of the ordinary decode batch: the largest weights of a layer
        _proj("q4 32 rows 4096-22016 gate up", rows=32, k=4096, n=22016, group=128, silu=True),
        # the 13B feed-forward of a busy server, an odd number of rows, 32-bit results
        _proj("q4 101 rows 5120-13824", rows=101, k=5120, n=13824, group=64, zeros=True, f32=True),
        # a prompt of 512 tokens through the same weights
        _proj("q4 512 rows 4096-11008", rows=512, k=4096, n=11008, group=128),
        # four requests behind one short instruction: latency
        _attn("prefix 4 x 512", rows=4, heads=32, kv_heads=8, groups=1, prefix=512, prefix_short=512, tail=48, tail_short=17),
        # the ordinary decode batch behind one long system prompt, every head with keys of its own
        _attn("prefix 32 x 4096", rows=32, heads=32, kv_heads=32, groups=1, prefix=4096, prefix_short=4096, tail=576, tail_short=64),
        # several tenants with prompts of their own (13B heads), ragged, and requests without any
        _attn("prefix 4 groups 13B", rows=72, heads=40, kv_heads=40, groups=4, prefix=6000, prefix_short=700, tail=900, tail_short=1, alone=8),
        # many answers over one long document, query heads that share keys
        _attn("prefix 128 x 32768", rows=128, heads=32, kv_heads=8, groups=1, prefix=32768, prefix_short=32768, tail=300, tail_short=20),
        # one constrained answer: every launch is latency
        _tokens("tokens 1", rows=1, vocab=32000, prompt=600, answer=40, bias=8, masks=1),
        # the ordinary decode batch under all rules
        _tokens("tokens 32", rows=32, vocab=32000, prompt=1200, answer=400, bias=64, masks=8),
        # a large batch over a large vocabulary, the processed scores kept for a sampler
        _tokens("tokens 256 kept", rows=256, vocab=128000, prompt=2000, answer=800, bias=300, masks=16, keep=True),
    ]


def _proj(name, rows, k, n, group, zeros=False, rank=0, adapters=0, silu=False, f32=False):
    c = {"kind": "projection", "rows": rows, "in": k, "out": n, "group": group, "zeros": zeros, "rank": rank, "adapters": adapters,
         "silu": silu, "f32": f32}
    return dict(c, name=name) if name else c


def _attn(name, rows, heads, kv_heads, groups, prefix, prefix_short, tail, tail_short, dim=128, page=16, alone=0):
    c = {"kind": "attention", "rows": rows, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "groups": groups, "prefix": prefix,
         "prefix_short": prefix_short, "tail": tail, "tail_short": tail_short, "alone": alone}
    return dict(c, name=name) if name else c


def _tokens(name, rows, vocab, prompt, answer, bias, masks, keep=False):
    c = {"kind": "tokens", "rows": rows, "vocab": vocab, "prompt": prompt, "answer": answer, "bias": bias, "masks": masks, "keep": keep}
    return dict(c, name=name) if name else c


def draw(rng):
    spread = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    kind = rng.choice(("projection", "attention", "tokens"))
    if kind == "projection":
        group = rng.choice((32, 64, 128))
        silu = rng.random() < 0.3
        n = spread(500, 14000)
        return _proj(None, rows=spread(1, 512), k=group * max(2, spread(512, 11008) // group), n=-(-n // 16) * 16 if silu else n, group=group,
                     zeros=rng.random() < 0.5, rank=0 if silu else rng.choice((0, 8, 16, 64)), adapters=spread(1, 32), silu=silu,
                     f32=not silu and rng.random() < 0.3)
    if kind == "attention":
        kv, rep = rng.choice(((1, 8), (8, 1), (8, 4), (32, 1), (5, 3), (16, 2), (4, 16)))
        groups, longest = rng.randint(1, 5), spread(300, 8000)
        rows = spread(3, 128)
        return _attn(None, rows=rows, heads=kv * rep, kv_heads=kv, groups=groups, prefix=longest, prefix_short=spread(100, longest),
                     tail=spread(1, 900), tail_short=1, dim=rng.choice((64, 128, 128)), page=rng.choice((16, 32)), alone=rng.randint(0, rows // 3))
    return _tokens(None, rows=spread(1, 256), vocab=spread(1000, 128000), prompt=spread(1, 4000), answer=spread(1, 1500), bias=spread(1, 300),
                   masks=rng.randint(1, 16), keep=rng.random() < 0.5)


def prepare(case, seed):
    st = {"projection": _proj_inputs, "attention": _attn_inputs, "tokens": _token_inputs}[case["kind"]](case, seed)
    if own:
        {"projection": _proj_handles, "attention": _attn_handles, "tokens": _token_handles}[case["kind"]](case, st)
    return st


def run(state):
    if own:
        return state["call"]()
    return {"projection": _proj_plain, "attention": _attn_plain, "tokens": _token_plain}[state["case"]["kind"]](state)


def work(case):
    return {"projection": _proj_work, "attention": _attn_work, "tokens": _token_work}[case["kind"]](case)


def exact(case, seed):
    return {"projection": _proj_exact, "attention": _attn_exact, "tokens": _token_exact}[case["kind"]](case, seed)


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


# ---------------------------------------------------------------- projections with 4-bit weights
# W[o, k] = (q[o, k] - zero[o, k / group]) scale[o, k / group] with q, zero in 0 .. 15 (zero 8 where there are none);
# y = x W^T + alpha B[slot] (A[slot] x); gate and up in one matrix (rows in turns of 8): y = silu(gate) up
def _proj_inputs(case, seed):
    g, T, K, N, G = _generator(seed), case["rows"], case["in"], case["out"], case["group"]
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x = rnd(T, K)
    x[:, torch.randint(0, K, (max(K // 512, 1),), generator=g, device="cuda")] *= 8.0  # (a few channels carry most of the energy)
    # what rounding normal weights to a grid over 15 steps of about 0.4 standard deviations gives
    q = (rnd(N, K) * 2.5 + 7.5).round_().clamp_(0, 15).to(torch.uint8)
    st = {"case": dict(case), "x": x.bfloat16(), "q": q[:, 0::2] | (q[:, 1::2] << 4),  # two a byte, the even column in the low half
          "scale": ((0.6 + 0.8 * torch.rand(N, K // G, generator=g, device="cuda")) * 0.4 * K ** -0.5).bfloat16(),
          "zero": torch.randint(5, 11, (N, K // G), generator=g, device="cuda").to(torch.uint8) if case["zeros"] else None}
    if case["rank"]:
        n, r = case["adapters"], case["rank"]
        st["A"], st["B"] = (rnd(n, r, K) * K ** -0.5).bfloat16(), (rnd(n, N, r) * 0.3).bfloat16()
        st["slots"] = torch.randint(-1, n, (T,), generator=g, device="cuda", dtype=torch.int32)
        st["alpha"] = 0.5 + torch.rand(n, generator=g, device="cuda")
    return st


def _unpacked(q):
    return torch.stack([q & 15, q >> 4], -1).flatten(-2)


def _proj_handles(case, st):
    ops = _ops()
    W = ops.QuantWeight.from_integers(_unpacked(st["q"]), st["scale"], st["zero"], group=case["group"])
    flags = (ops.SILU_MUL if case["silu"] else 0) | (ops.OUT_F32 if case["f32"] else 0)
    stack = None
    if case["rank"]:
        n, r = case["adapters"], case["rank"]
        stack = ops.LoraStack(st["A"], st["B"], torch.full((n,), r, dtype=torch.int32, device="cuda"), st["alpha"], r, 1, (0, case["out"]))
    st["call"] = lambda: ops.linear(st["x"], W, stack, st.get("slots"), flags=flags)


def _proj_plain(st):
    c = st["case"]
    G, N, K = c["group"], c["out"], c["in"]
    w = _unpacked(st["q"]).float().view(N, K // G, G)
    w = ((w - (8.0 if st["zero"] is None else st["zero"].float()[..., None])) * st["scale"].float()[..., None]).view(N, K)
    x = st["x"].float()
    y = x @ w.T
    if c["rank"]:
        s = st["slots"].long()
        u = torch.einsum("tk,trk->tr", x, st["A"].float()[s.clamp(min=0)])
        d = torch.einsum("tr,tnr->tn", u, st["B"].float()[s.clamp(min=0)]) * st["alpha"][s.clamp(min=0)][:, None]
        y = torch.where(s[:, None] < 0, y, y + d)
    if c["silu"]:
        v = y.view(y.shape[0], N // 16, 2, 8)
        y = (v[:, :, 0] / (1 + torch.exp(-v[:, :, 0])) * v[:, :, 1]).reshape(y.shape[0], N // 2)
    return y if c["f32"] else y.bfloat16()


def _proj_exact(case, seed):
    st, G = _proj_inputs(case, seed), case["group"]
    q = torch.empty(case["out"], case["in"], dtype=torch.float64, device="cuda")
    q[:, 0::2], q[:, 1::2] = (st["q"] & 15).double(), (st["q"] >> 4).double()
    zero = torch.full_like(st["scale"], 8.0).double() if st["zero"] is None else st["zero"].double()
    q = (q - zero.repeat_interleave(G, 1)) * st["scale"].double().repeat_interleave(G, 1)
    x = st["x"].double()
    y = torch.matmul(x, q.t())
    if case["rank"]:
        for t, s in enumerate(st["slots"].tolist()):
            if s >= 0:
                y[t] += st["alpha"][s].double() * (st["B"][s].double() @ (st["A"][s].double() @ x[t]))
    if case["silu"]:
        cols = torch.arange(case["out"], device="cuda")
        gate, up = y[:, cols % 16 < 8], y[:, cols % 16 >= 8]
        y = gate * torch.sigmoid(gate) * up
    return y


def _proj_work(case):
    T, K, N, G = case["rows"], case["in"], case["out"], case["group"]
    cols = N // 2 if case["silu"] else N
    b = N * K // 2 + N * (K // G) * (3 if case["zeros"] else 2) + 2 * T * K + (4 if case["f32"] else 2) * T * cols
    f = 2 * T * K * N
    if case["rank"]:
        b += min(T, case["adapters"]) * 2 * case["rank"] * (K + N) + 4 * T
        f += 2 * T * case["rank"] * (K + N)
    return {"bytes": b, "flops": f}


# ---------------------------------------------------------------- attention of a batch that shares prefixes
# o[t, h] = softmax over the tokens 0 .. pos[t] of (q[t, h] . k / sqrt(dim)) v; the first tokens of the rows of a group are the
# same pages of the cache
def _lengths(case):
    """(prefix length of every group, group of every row or -1, length of every row)."""
    page, G, R = case["page"], case["groups"], case["rows"]
    lo, hi = case["prefix_short"], case["prefix"]
    pre = [max(1, round(lo * (hi / lo) ** (g / max(G - 1, 1))) // page) * page for g in range(G)]
    shared = R - case["alone"]
    group = [t % G if t < shared else -1 for t in range(R)]
    tail = [case["tail_short"] + (case["tail"] - case["tail_short"]) * (t * 7919 % R) // max(R - 1, 1) for t in range(R)]
    return pre, group, [(pre[g] if g >= 0 else 0) + n for g, n in zip(group, tail)]


def _attn_inputs(case, seed):
    g, page, R, D = _generator(seed), case["page"], case["rows"], case["dim"]
    pre, group, length = _lengths(case)
    pages = lambda n: -(-n // page)
    need = sum(pages(p) for p in pre) + sum(pages(n) - (pages(pre[k]) if k >= 0 else 0) for k, n in zip(group, length))
    free = iter(torch.randperm(need, generator=g, device="cuda").tolist())
    shared = [[next(free) for _ in range(pages(p))] for p in pre]
    table = torch.zeros(R, pages(max(length)), dtype=torch.int32)
    for t, (k, n) in enumerate(zip(group, length)):
        ids = list(shared[k]) if k >= 0 else []
        ids += [next(free) for _ in range(pages(n) - len(ids))]
        table[t, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
    kv = torch.randn(2, need, case["kv_heads"], page, D, generator=g, device="cuda").bfloat16()
    q = 2.0 * torch.randn(R, case["heads"] * D, generator=g, device="cuda")  # (scores of two standard deviations)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    return {"case": dict(case), "q": q.bfloat16(), "k": kv[0], "v": kv[1], "table": table.cuda(), "pos": i32([n - 1 for n in length]),
            "slot": i32(list(range(R))), "group": i32(group), "prefix": i32([pre[k] if k >= 0 else 0 for k in group])}


def _attn_handles(case, st):
    ops, out = _ops(), torch.empty_like(st["q"])
    plan = ops.PrefixPlan(case["rows"], case["heads"], case["kv_heads"], "cuda")
    ops.prefix_plan(st["slot"], st["group"], st["prefix"], plan)  # (once for all layers of a step)
    st["call"] = lambda: ops.paged_attention_shared(st["q"], st["k"], st["v"], st["table"], st["slot"], st["pos"], plan, case["heads"], out=out)


def _attn_plain(st):
    c = st["case"]
    R, Hkv, D, page = c["rows"], c["kv_heads"], c["dim"], c["page"]
    pre, group, length = _lengths(c)
    q = st["q"].float().view(R, Hkv, -1, D) / math.sqrt(D)
    out = torch.empty_like(q)
    dense = lambda pages, ids: pages[ids.long()].float().transpose(-4, -3).flatten(-3, -2)  # [..., Hkv, keys, D]
    for k in [-1] + list(range(c["groups"])):  # a group's prefix is read once, its rows' own tokens row by row
        rows = [t for t in range(R) if group[t] == k]
        if not rows:
            continue
        t = torch.tensor(rows, device="cuda")
        first = pre[k] // page if k >= 0 else 0
        last = max(-(-length[i] // page) for i in rows)
        kt, vt = (dense(st[n], st["table"][t, first:last]) for n in ("k", "v"))
        s = torch.einsum("bhgd,bhkd->bhgk", q[t], kt)
        hidden = first * page + torch.arange(kt.shape[2], device="cuda") > st["pos"][t][:, None]
        s = s.masked_fill(hidden[:, None, None], -math.inf)
        vt = vt.masked_fill(hidden[:, None, :, None], 0.0)
        m = s.amax(-1, keepdim=True)
        if k >= 0:
            kp, vp = (dense(st[n], st["table"][rows[0], :first]) for n in ("k", "v"))
            sp = torch.einsum("bhgd,hkd->bhgk", q[t], kp)
            m = torch.maximum(m, sp.amax(-1, keepdim=True))
            sp = torch.exp(sp - m)
        s = torch.exp(s - m)
        total, o = s.sum(-1, keepdim=True), torch.einsum("bhgk,bhkd->bhgd", s, vt)
        if k >= 0:
            total, o = total + sp.sum(-1, keepdim=True), o + torch.einsum("bhgk,hkd->bhgd", sp, vp)
        out[t] = o / total
    return out.reshape(R, -1).bfloat16()


def _attn_exact(case, seed):
    st = _attn_inputs(case, seed)
    R, Hkv, D, page = case["rows"], case["kv_heads"], case["dim"], case["page"]
    out = []
    for t, n in enumerate((st["pos"] + 1).tolist()):
        ids = st["table"][t, :-(-n // page)].long()
        k, v = (st[x][ids].double().permute(1, 0, 2, 3).reshape(Hkv, -1, D)[:, :n] for x in ("k", "v"))
        qt = st["q"][t].double().view(Hkv, -1, D)
        out.append((torch.softmax(qt @ k.mT / D ** 0.5, -1) @ v).reshape(-1))
    return torch.stack(out)


def _attn_work(case):
    pre, group, length = _lengths(case)
    keys = sum(pre) + sum(n - (pre[k] if k >= 0 else 0) for k, n in zip(group, length))
    return {"bytes": 4 * keys * case["kv_heads"] * case["dim"] + 4 * case["rows"] * case["heads"] * case["dim"],
            "flops": 4 * case["heads"] * case["dim"] * sum(length)}


# ---------------------------------------------------------------- next tokens under rules
# for every token v that row t has seen in its prompt or its answer: l = l / r where l > 0, else l r; then, with c = how often the
# answer has it: l -= frequency c; l -= presence where c > 0; then l += bias of the row's set; then -inf where the row's mask does not
# allow v.  The token: the first one of the largest l, -1 where none is allowed.
def _token_lengths(case, t):
    R = max(case["rows"] - 1, 1)
    return 1 + (case["prompt"] - 1) * (t * 7919 % case["rows"]) // R, 1 + (case["answer"] - 1) * (t * 104729 % case["rows"]) // R


def _token_inputs(case, seed):
    g, R, V, n_sets = _generator(seed), case["rows"], case["vocab"], 4
    rand = lambda *s: torch.rand(*s, generator=g, device="cuda")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    logits = 2.0 * torch.randn(R, V, generator=g, device="cuda")
    text = lambda n: (V * rand(R, n) ** 3).int().clamp_(max=V - 1)  # (few tokens make up most of a text)
    lengths = [_token_lengths(case, t) for t in range(R)]
    st = {"case": dict(case), "logits": logits, "prompt": text(case["prompt"]), "answer": text(case["answer"]),
          "prompt_len": i32([p for p, _ in lengths]), "answer_len": i32([a for _, a in lengths])}
    pick = lambda *v: torch.tensor(v, device="cuda")[torch.randint(0, len(v), (R,), generator=g, device="cuda")]
    st["repetition"], st["frequency"], st["presence"] = pick(1.0, 1.1, 1.3), pick(0.0, 0.2, 0.7), pick(0.0, 0.5, -0.3)
    n = min(case["bias"], V)
    st["bias_tokens"] = torch.stack([torch.randperm(V, generator=g, device="cuda")[:n].sort().values for _ in range(n_sets)]).int()
    st["bias_values"] = 3.0 * torch.randn(n_sets, n, generator=g, device="cuda")
    st["bias_set"] = torch.randint(-1, n_sets, (R,), generator=g, device="cuda", dtype=torch.int32)
    # grammars: one that allows nearly everything, others only a few words
    allowed = rand(case["masks"], V) < torch.logspace(0, -2.5, case["masks"], device="cuda")[:, None] * 0.9
    words = -(-V // 32)
    bits = torch.zeros(case["masks"], words * 32, dtype=torch.int64, device="cuda")
    bits[:, :V] = allowed
    bits = (bits.view(case["masks"], words, 32) << torch.arange(32, device="cuda")).sum(-1)
    st["masks"] = torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).int()  # bit v % 32 of word v / 32
    st["mask_of"] = torch.randint(-1, case["masks"], (R,), generator=g, device="cuda", dtype=torch.int32)
    return st


def _token_handles(case, st):
    ops = _ops()
    n_sets, n = st["bias_tokens"].shape
    start = torch.arange(n_sets + 1, dtype=torch.int32, device="cuda") * n
    rules = ops.LogitRules(repetition=st["repetition"], frequency=st["frequency"], presence=st["presence"], prompt=st["prompt"],
                           prompt_len=st["prompt_len"], answer=st["answer"], answer_len=st["answer_len"], bias_set=st["bias_set"],
                           bias_start=start, bias_token=st["bias_tokens"].reshape(-1), bias_value=st["bias_values"].reshape(-1),
                           mask_of=st["mask_of"], masks=st["masks"])
    out = torch.empty(case["rows"], dtype=torch.int32, device="cuda")
    kept = torch.empty_like(st["logits"]) if case["keep"] else None

    def call():
        ops.choose_tokens(st["logits"], rules, out=out, logits_out=kept)
        return [out, kept] if case["keep"] else [out]

    st["call"] = call


def _token_plain(st):
    c = st["case"]
    R, V = c["rows"], c["vocab"]
    place = lambda n: torch.arange(n, device="cuda")[None]
    count, seen = torch.zeros(R, V + 1, device="cuda"), torch.zeros(R, V + 1, device="cuda")  # (column V: no token)
    for name, into in (("prompt", (seen,)), ("answer", (seen, count))):
        text = st[name].long()
        text = torch.where(place(text.shape[1]) < st[name + "_len"][:, None], text, V)
        for a in into:
            a.scatter_add_(1, text, torch.ones_like(text, dtype=torch.float32))
    count, seen = count[:, :V], seen[:, :V] > 0
    l, r = st["logits"], st["repetition"][:, None]
    l = torch.where(seen, torch.where(l > 0, l / r, l * r), l)
    l = l - st["frequency"][:, None] * count
    l = torch.where(count > 0, l - st["presence"][:, None], l)
    bias = torch.zeros(st["bias_tokens"].shape[0], V, device="cuda").scatter_(1, st["bias_tokens"].long(), st["bias_values"])
    has = st["bias_set"][:, None] >= 0
    l = torch.where(has, l + bias[st["bias_set"].long().clamp(min=0)], l)
    bit = (st["masks"].long()[:, :, None] >> torch.arange(32, device="cuda")) & 1
    allowed = bit.flatten(1)[:, :V].bool()[st["mask_of"].long().clamp(min=0)] | (st["mask_of"][:, None] < 0)
    l = torch.where(allowed, l, -math.inf)
    best = l.amax(1)
    token = torch.where(l == best[:, None], place(V), V).amin(1)
    token = torch.where(best == -math.inf, -1, token).int()
    return [token, l] if c["keep"] else [token]


def _token_exact(case, seed):
    st, V = _token_inputs(case, seed), case["vocab"]
    rows, tokens, sure = [], [], True
    words = st["masks"].cpu().tolist()
    as_bits = {-1: torch.ones(V, dtype=torch.bool, device="cuda")}
    for i, w in enumerate(words):
        as_bits[i] = torch.tensor([(x >> b) & 1 for x in w for b in range(32)][:V], dtype=torch.bool, device="cuda")
    for t in range(case["rows"]):
        l = st["logits"][t].double()
        prompt, answer = st["prompt"][t, :st["prompt_len"][t]].long(), st["answer"][t, :st["answer_len"][t]].long()
        seen = torch.cat([prompt, answer]).unique()
        r = st["repetition"][t].double()
        l[seen] = torch.where(l[seen] > 0, l[seen] / r, l[seen] * r)
        said, times = answer.unique(return_counts=True)
        l[said] -= st["frequency"][t].double() * times + st["presence"][t].double()
        if int(st["bias_set"][t]) >= 0:
            l[st["bias_tokens"][st["bias_set"][t]].long()] += st["bias_values"][st["bias_set"][t]].double()
        l[~as_bits[int(st["mask_of"][t])]] = -math.inf
        two = l.topk(min(2, V)).values.tolist()
        tokens.append(-1 if two[0] == -math.inf else int(l.argmax()))
        sure = sure and (two[0] == -math.inf or two[0] - two[-1] > 1e-5 * (1 + abs(two[0])))  # (32 bits may see a tie there)
        rows.append(l)
    token = torch.tensor(tokens, dtype=torch.int32, device="cuda") if sure else None
    return [token, torch.stack(rows)] if case["keep"] else [token]


def _token_work(case):
    R, V = case["rows"], case["vocab"]
    text = sum(sum(_token_lengths(case, t)) for t in range(R))
    return {"bytes": 4 * R * V * (2 if case["keep"] else 1) + 4 * text + case["masks"] * V // 8 + 32 * case["bias"] + 4 * R,
            "flops": 4 * R * V}
