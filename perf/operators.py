"""Packed attention with grouped heads and a learned relative position bias, forward and backward: the cases that are timed, their
inputs, the operators in plain torch and their values in 64 bits.

Layout: q, out, dq [tokens][heads][head_dim]; k, v, dk, dv [tokens][kv_heads][head_dim]; sequences back to back, sequence i being
rows offsets[i] .. offsets[i + 1].  A padded case holds [sequences][longest] rows each and a key mask instead of offsets."""
import math

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _case(name, op, dtype, sequences, shortest, longest, heads, kv_heads, head_dim, causal, buckets=0, max_distance=0, padded=False):
    c = dict(op=op, dtype=dtype, sequences=sequences, shortest=shortest, longest=longest, heads=heads, kv_heads=kv_heads,
             head_dim=head_dim, causal=causal, buckets=buckets, max_distance=max_distance, padded=padded)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one user's query through the bi-encoder's layer (12 heads of 32): latency is all that counts
        _case("query", "forward", "bf16", 1, 17, 17, 12, 12, 32, False, 32, 128),
        # a bulk embedding pass: 64K-token budget, chunks of 32 to 256 tokens, packed, relative bias
        _case("chunks_packed", "forward", "bf16", 400, 32, 256, 12, 12, 32, False, 32, 128),
        # a rerank batch as a padded call makes it: (query, passage) pairs up to 512 tokens under a key mask
        _case("pairs_padded", "forward", "fp16", 64, 61, 512, 12, 12, 64, False, 32, 128, True),
        # a serving step: prompts of very different lengths, from a single token on, causal, grouped heads
        _case("prompts", "forward", "bf16", 13, 1, 2039, 32, 8, 128, True),
        # a long document, causal with one-sided bias
        _case("document_bias", "forward", "bf16", 2, 2500, 4099, 8, 8, 64, True, 32, 128),
        # the longest prompt, few key heads
        _case("long_prompt", "forward", "fp16", 1, 16384, 16384, 16, 2, 128, True),
        # fine-tuning steps (forward and backward): a handful of short queries
        _case("tune_queries", "train", "bf16", 8, 5, 31, 12, 12, 32, False, 32, 128),
        # ... a batch of chunks with the bias table's gradient
        _case("tune_chunks", "train", "bf16", 96, 40, 256, 12, 12, 32, False, 32, 128),
        # ... passages with wider heads, fp16, two-sided bias
        _case("tune_passages", "train", "fp16", 24, 100, 511, 12, 12, 64, False, 32, 128),
        # ... prompts of different lengths, causal, grouped heads
        _case("tune_prompts", "train", "bf16", 9, 33, 2048, 16, 4, 128, True),
        # ... a long document
        _case("tune_long", "train", "bf16", 1, 8191, 8191, 8, 2, 128, True),
        # ... a long document with one-sided bias
        _case("tune_long_bias", "train", "bf16", 1, 4000, 4000, 8, 8, 64, True, 32, 128),
    ]


def _lengths(case):
    """The sequences' lengths: spread over the logarithm from shortest to longest, in a fixed shuffled order."""
    n = case["sequences"]
    if n == 1:
        return [case["longest"]]
    step = math.log(case["longest"] / case["shortest"]) / (n - 1)
    lens = [round(case["shortest"] * math.exp(step * i)) for i in range(n)]
    lens[-1] = case["longest"]
    return [lens[i] for i in np.random.default_rng(n).permutation(n)]


def _pairs(case):
    """Attended (query, key) pairs of one head."""
    lens = _lengths(case)
    rows = [case["longest"]] * len(lens) if case["padded"] else lens
    if not case["causal"]:
        return sum(r * x for r, x in zip(rows, lens))
    return sum(x * (x + 1) // 2 + (r - x) * x for r, x in zip(rows, lens))


def _tokens(case):
    return case["sequences"] * case["longest"] if case["padded"] else sum(_lengths(case))


def draw(rng):
    most = max(listed(), key=lambda c: work(c)["flops"])
    limit_flops, limit_cells = work(most)["flops"], most["heads"] * most["longest"] ** 2
    while True:
        train = rng.random() < 0.5
        longest = round(math.exp(rng.uniform(math.log(2), math.log(16000))))
        shortest = max(1, round(longest * math.exp(-rng.uniform(0, 4))))
        sequences = round(math.exp(rng.uniform(0, math.log(300))))
        group = rng.choice((1, 2, 4, 8))
        kv_heads = rng.choice((1, 2, 3, 4, 8, 12))
        head_dim = rng.choice((32, 64, 64, 96, 128, 128))
        causal = rng.random() < 0.5
        biased = rng.random() < 0.5
        buckets = 2 * rng.randint(4, 24) if biased else 0
        max_distance = rng.randint(buckets + 1, 320) if biased else 0
        padded = rng.random() < 0.25
        case = _case("", "train" if train else "forward", rng.choice(("bf16", "fp16")), sequences, shortest, longest, kv_heads * group,
                     kv_heads, head_dim, causal, buckets, max_distance, padded)
        cells = sequences * kv_heads * group * longest ** 2
        # a handful of tokens has gradients that cancel to nothing; the plain form's score matrices have to fit the card
        if _tokens(case) >= 16 and longest >= 8 and cells * (3 if train else 1) <= limit_cells and work(case)["flops"] <= limit_flops:
            return case


def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def prepare(case, seed):
    dev = _device()
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dt = _TYPES[case["dtype"]]
    lens, D = _lengths(case), case["head_dim"]
    lead = (case["sequences"], case["longest"]) if case["padded"] else (sum(lens),)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32)

    state = {"case": dict(case), "offsets": None, "key_mask": None, "table": None}
    state["q"] = normal(*lead, case["heads"], D).to(dt)
    state["k"] = normal(*lead, case["kv_heads"], D).to(dt)
    state["v"] = normal(*lead, case["kv_heads"], D).to(dt)
    if case["op"] == "train":
        state["dout"] = normal(*lead, case["heads"], D).to(dt)
    if case["buckets"]:
        state["table"] = normal(case["buckets"], case["heads"])
    lens_t = torch.tensor(lens, dtype=torch.int32, device=dev)
    if case["padded"]:
        state["key_mask"] = (torch.arange(case["longest"], device=dev, dtype=torch.int32)[None, :] < lens_t[:, None]).to(torch.int32)
    else:
        state["offsets"] = torch.zeros(len(lens) + 1, dtype=torch.int32, device=dev)
        state["offsets"][1:] = lens_t.cumsum(0)
    return state


def _buckets(L, case, dev):
    """bucket(j - i) for j - i = -(L - 1) .. L - 1.  The borders between the logarithmic buckets are found in 64 bits, with room for
    their rounding: a border that is a whole number belongs to the upper bucket."""
    two_sided = not case["causal"]
    n = case["buckets"] // 2 if two_sided else case["buckets"]
    m = n // 2
    t = torch.arange(1, n - m, dtype=torch.float64, device=dev)
    border = m * torch.exp(t / (n - m) * math.log(case["max_distance"] / m))
    border = torch.ceil(border * (1 - 1e-11))
    r = torch.arange(-(L - 1), L, device=dev)
    d = r.abs() if two_sided else (-r).clamp(min=0)
    far = m + (d[:, None].to(torch.float64) >= border).sum(1)
    return torch.where(d < m, d, far) + (torch.where(r > 0, n, 0) if two_sided else 0)


def _plain(state):
    case, dev = state["case"], state["q"].device
    L, Hq, Hk, D = case["longest"], case["heads"], case["kv_heads"], case["head_dim"]
    G, scale, dt = Hq // Hk, 1 / math.sqrt(D), state["q"].dtype
    at = torch.arange(L, device=dev)
    if case["padded"]:
        attended = (state["key_mask"] != 0)[:, None, :].expand(-1, L, -1)
        pad = lambda x: x.float()                                                    # noqa: E731
        pack = lambda x: x                                                           # noqa: E731
    else:
        lens = state["offsets"][1:] - state["offsets"][:-1]
        inside = at[None, :] < lens[:, None]
        rows = (state["offsets"][:-1, None] + at[None, :]).clamp(max=state["q"].shape[0] - 1)
        attended = inside[:, None, :] & inside[:, :, None]
        pad = lambda x: x[rows].float().masked_fill(~inside[:, :, None, None], 0.0)   # noqa: E731
        pack = lambda x: x[inside]                                                   # noqa: E731
    if case["causal"]:
        attended = attended & (at[None, :] <= at[:, None])
    attended = attended[:, None, None]                                               # [B][1][1][L][L]
    B = attended.shape[0]
    q = pad(state["q"]).view(B, L, Hk, G, D).permute(0, 2, 3, 1, 4)                   # [B][Hk][G][L][D]
    k = pad(state["k"]).permute(0, 2, 1, 3)[:, :, None]                               # [B][Hk][1][L][D]
    v = pad(state["v"]).permute(0, 2, 1, 3)[:, :, None]
    s = torch.matmul(q, k.transpose(-1, -2)) * scale
    if state["table"] is not None:
        bucket = _buckets(L, case, dev)
        s += state["table"][bucket].t()[:, (at[None, :] - at[:, None]) + L - 1].view(Hk, G, L, L)
    s.masked_fill_(~attended, -math.inf)
    top = s.amax(-1, keepdim=True)
    top.masked_fill_(top == -math.inf, 0.0)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    p /= total.masked_fill_(total == 0, 1.0)
    o = torch.matmul(p, v)
    back = lambda x, H: pack(x.reshape(B, H, L, D).permute(0, 2, 1, 3)).to(dt)        # noqa: E731
    out = back(o, Hq)
    if case["op"] == "forward":
        return out
    do = pad(state["dout"]).view(B, L, Hk, G, D).permute(0, 2, 3, 1, 4)
    dv = torch.matmul(p.transpose(-1, -2), do).sum(2)
    ds = torch.matmul(do, v.transpose(-1, -2))
    ds -= (p * ds).sum(-1, keepdim=True)
    ds *= p
    dq = torch.matmul(ds, k) * scale
    dk = torch.matmul(ds.transpose(-1, -2), q).sum(2) * scale
    grads = (out, back(dq, Hq), back(dk, Hk), back(dv, Hk))
    if state["table"] is None:
        return grads
    # sums over the diagonals: with j reversed they are the sums over i + j, which rows of 2 L columns, read again as rows of
    # 2 L - 1, put below each other
    wide = torch.zeros(Hq, L, 2 * L, device=dev)
    wide[:, :, :L] = ds.sum(0).view(Hq, L, L).flip(-1)
    sums = wide.view(Hq, -1)[:, :L * (2 * L - 1)].view(Hq, L, 2 * L - 1).sum(1, dtype=torch.float64).flip(-1)
    one_hot = (bucket[:, None] == torch.arange(case["buckets"], device=dev)).to(torch.float64)
    return (*grads, torch.matmul(sums, one_hot).t().float().contiguous())


def exact(case, seed):
    state = prepare(case, seed)
    dev, D, Hk = state["q"].device, case["head_dim"], case["kv_heads"]
    G, L, train = case["heads"] // Hk, case["longest"], case["op"] == "train"
    lens = _lengths(case)
    rows = [(i * L, L, n) for i, n in enumerate(lens)] if case["padded"] else []
    if not rows:
        ends = np.cumsum(lens)
        rows = [(int(e) - n, n, n) for e, n in zip(ends, lens)]
    names = ("q", "k", "v") + (("dout",) if train else ())
    x = {n: state[n].reshape(-1, state[n].shape[-2], D) for n in names}
    y = {n: torch.zeros(x[m].shape, dtype=torch.float64, device=dev) for n, m in (("out", "q"), ("dq", "q"), ("dk", "k"), ("dv", "v"))}
    biased = case["buckets"] > 0
    if biased:
        table = state["table"].double()
        dtable = torch.zeros_like(table)
        number = torch.tensor([_bucket_of(r, case) for r in range(-L + 1, L)], device=dev)
    for start, n, valid in rows:
        at, keys = torch.arange(n, device=dev), torch.arange(valid, device=dev)
        rel = keys[None, :] - at[:, None]
        for g0 in range(0, Hk, Hk if n * n * Hk * G < 1 << 28 else 1):                 # key heads at a time
            g1 = Hk if n * n * Hk * G < 1 << 28 else g0 + 1
            h = slice(g0 * G, g1 * G)
            part = {m: x[m][start:start + n, h if m in ("q", "dout") else slice(g0, g1)].double().transpose(0, 1) for m in names}
            q = part["q"].reshape(g1 - g0, G * n, D)
            k, v = part["k"][:, :valid], part["v"][:, :valid]
            s = (torch.bmm(q, k.transpose(1, 2).contiguous()) / D ** 0.5).view(-1, n, valid)
            if biased:
                s += table[number[rel + L - 1], h].permute(2, 0, 1)
            if case["causal"]:
                s.masked_fill_(rel > 0, -math.inf)
            p = torch.softmax(s, -1)
            pg = p.view(g1 - g0, G * n, valid)
            y["out"][start:start + n, h] = torch.bmm(pg, v).view(-1, n, D).transpose(0, 1)
            if not train:
                continue
            do = part["dout"].reshape(g1 - g0, G * n, D)
            dp = torch.bmm(do, v.transpose(1, 2).contiguous()).view(-1, n, valid)
            ds = p * (dp - (dp * p).sum(-1, keepdim=True))
            dg = ds.view(g1 - g0, G * n, valid)
            y["dq"][start:start + n, h] = (torch.bmm(dg, k.contiguous()) / D ** 0.5).view(-1, n, D).transpose(0, 1)
            y["dk"][start:start + valid, g0:g1] = (torch.bmm(dg.transpose(1, 2).contiguous(), q) / D ** 0.5).transpose(0, 1)
            y["dv"][start:start + valid, g0:g1] = torch.bmm(pg.transpose(1, 2).contiguous(), do).transpose(0, 1)
            if biased:
                for b in torch.unique(number[rel + L - 1]).tolist():
                    dtable[b, h] += (ds * (number[rel + L - 1] == b)).sum((1, 2))
    y = {n: t.view(state[{"out": "q", "dq": "q", "dk": "k", "dv": "v"}[n]].shape) for n, t in y.items()}
    if not train:
        return y["out"]
    return (y["out"], y["dq"], y["dk"], y["dv"]) + ((dtable,) if biased else ())


def _bucket_of(r, case):
    """bucket(r) in whole numbers: d is in or above logarithmic bucket t when (d / m)^(n - m) >= (M / m)^t."""
    M, n, d, first = case["max_distance"], case["buckets"], -r if r < 0 else 0, 0
    if not case["causal"]:
        n, d, first = n // 2, abs(r), n // 2 if r > 0 else 0
    m = n // 2
    if d < m:
        return first + d
    if d >= M:
        return first + n - 1
    return first + m + sum(d ** (n - m) >= M ** t * m ** (n - m - t) for t in range(1, n - m))


def _kwargs(state):
    case = state["case"]
    kw = dict(offsets=state["offsets"], causal=case["causal"], key_mask=state["key_mask"])
    if case["buckets"]:
        kw.update(bias_table=state["table"], max_distance=case["max_distance"], bidirectional=not case["causal"])
    return kw


def run(state):
    if not own:
        return _plain(state)
    from rag_amd.attention import packed_attention, packed_attention_backward
    q, k, v, kw = state["q"], state["k"], state["v"], _kwargs(state)
    if state["case"]["op"] == "forward":
        return packed_attention(q, k, v, **kw)
    out, lse = packed_attention(q, k, v, return_lse=True, **kw)
    grads = packed_attention_backward(state["dout"], q, k, v, out, lse, **kw)
    return (out, *(g for g in grads if g is not None))


def work(case):
    D, tokens, pairs = case["head_dim"], _tokens(case), _pairs(case)
    q_rows, k_rows = 2 * D * tokens * case["heads"], 2 * D * tokens * case["kv_heads"]
    table = 4 * case["buckets"] * case["heads"]
    if case["op"] == "forward":
        return {"bytes": 2 * q_rows + 2 * k_rows + table, "flops": 4 * D * pairs * case["heads"]}
    # reads q, k, v, dout, writes out, dq, dk, dv; two products forward, five backward
    return {"bytes": 4 * q_rows + 4 * k_rows + 2 * table, "flops": 14 * D * pairs * case["heads"]}
