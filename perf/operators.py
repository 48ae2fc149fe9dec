"""Measured cases of the batched-serving operators: the paged, quantised KV
cache (written with RoPE, read back), the attention of packed prompts and of
single tokens over it, and the sampler.

`run` goes through one operator.  Where `own` is false it computes the
operator's plain form from elementary torch operations in fp32; where it is
true it makes the calls a user of guanaco_b200 makes.  `exact` is the same
definition in 64 bits.

Cache layout (per pool, K and V alike): page, KV head, then for F16 the rows
[page_size][head_dim] of halves; for Q8_0 the codes [page_size][head_dim] of
int8 followed by the scales [page_size][head_dim / 32] of halves.  Token t of
sequence s (cu[s] <= t < cu[s + 1]) sits at position kv_len[s] - (cu[s + 1] - t).
"""
import random

import numpy as np
import torch

own = False

ROPE_THETA = 500000.0


# ------------------------------------------------------------------ the cases
def _cache(name, **k):
    return dict(op="cache", name=name, **k)


def _attn(name, op, **k):
    return dict(op=op, name=name, **k)


def listed():
    return [
        # one new token of one sequence, TinyLlama heads: the smallest write, a decode step's latency
        _cache("cache_token", act="f32", cache="q8_0", heads=32, kv=4, hd=64, page=16, n_seq=1, q_lo=1, q_hi=1,
               past_lo=700, past_hi=700, mix=1),
        # one new token for each of 61 sequences of a decode batch, Llama-3.1-8B heads
        _cache("cache_batch", act="f16", cache="f16", heads=32, kv=8, hd=128, page=32, n_seq=61, q_lo=1, q_hi=1,
               past_lo=0, past_hi=4096, mix=2),
        # the prompts of five requests, about 16 thousand tokens, quantised as they are written
        _cache("cache_prompts", act="f32", cache="q8_0", heads=32, kv=8, hd=128, page=64, n_seq=5, q_lo=1500, q_hi=4096,
               past_lo=0, past_hi=512, mix=3),
        # decode of a few short chats on a TinyLlama: latency
        _attn("decode_short", "decode", act="f32", cache="q8_0", heads=32, kv=4, hd=64, page=16, n_seq=7, q_lo=1, q_hi=1,
              past_lo=0, past_hi=300, mix=4),
        # one long context, batch 1: 8193 positions, as the fp32 cache's attention is measured
        _attn("decode_long", "decode", act="f32", cache="f16", heads=32, kv=8, hd=128, page=64, n_seq=1, q_lo=1, q_hi=1,
              past_lo=8192, past_hi=8192, mix=5),
        # a full decode batch with contexts from a few tokens to 8192
        _attn("decode_batch", "decode", act="f16", cache="q8_0", heads=32, kv=8, hd=128, page=32, n_seq=96, q_lo=1,
              q_hi=1, past_lo=16, past_hi=8191, mix=6),
        # a handful of short prompts of odd lengths (TinyLlama), one of them a single token
        _attn("prefill_short", "prefill", act="f32", cache="f16", heads=32, kv=4, hd=64, page=16, n_seq=6, q_lo=1,
              q_hi=130, past_lo=0, past_hi=0, mix=7),
        # ragged prompts after cached prefixes, fp32 activations over the 8-bit cache
        _attn("prefill_ragged", "prefill", act="f32", cache="q8_0", heads=32, kv=8, hd=128, page=32, n_seq=5, q_lo=200,
              q_hi=2048, past_lo=0, past_hi=700, mix=8),
        # one prompt of 8192 tokens, fp16 activations and cache: the largest
        _attn("prefill_long", "prefill", act="f16", cache="f16", heads=32, kv=8, hd=128, page=64, n_seq=1, q_lo=8192,
              q_hi=8192, past_lo=0, past_hi=0, mix=9),
        # one row of a small vocabulary, every filter on: a batch-1 step
        dict(op="sample", name="sample_one", rows=1, vocab=32000, filters="all"),
        # a decode batch on the Llama-3.1-8B vocabulary, requests with different settings
        dict(op="sample", name="sample_mixed", rows=61, vocab=128256, filters="mixed"),
        # a large batch, nucleus sampling
        dict(op="sample", name="sample_top_p", rows=256, vocab=128256, filters="top_p"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["cache", "decode", "prefill", "sample"])
    if op == "sample":
        return dict(op=op, rows=_log_int(rng, 1, 256), vocab=_log_int(rng, 32000, 128256),
                    filters=rng.choice(["all", "mixed", "top_p", "none"]))
    case = dict(op=op, act=rng.choice(["f32", "f16"]), cache=rng.choice(["q8_0", "f16"]), hd=rng.choice([64, 128]),
                page=rng.choice([16, 32, 64, 128]), mix=rng.randrange(1 << 20))
    case["kv"] = rng.choice([1, 2, 4, 8])
    case["heads"] = case["kv"] * rng.choice([1, 2, 4, 5, 7, 8])
    if (case["heads"] + 2 * case["kv"]) * case["hd"] == 3072:   # keep the projection's width generic
        case["hd"] = 64 if case["hd"] == 128 else 128
    if op == "decode":
        n = _log_int(rng, 1, 96)
        case.update(n_seq=n, q_lo=1, q_hi=1, past_lo=0, past_hi=_log_int(rng, 64, 8191))
    elif op == "cache":
        if rng.random() < 0.5:
            case.update(n_seq=_log_int(rng, 1, 128), q_lo=1, q_hi=1, past_lo=0, past_hi=_log_int(rng, 64, 4096))
        else:
            n = rng.randint(1, 6)
            hi = _log_int(rng, 8, 2700)
            case.update(n_seq=n, q_lo=max(1, hi // 3), q_hi=hi, past_lo=0, past_hi=512)
    else:
        # the plain form holds n_seq * heads * q_hi * (q_hi + past_hi) scores
        hi = _log_int(rng, 16, 4096)
        n = max(1, min(_log_int(rng, 1, 16), 8192 // hi))
        past = rng.choice([0, _log_int(rng, 16, 1024)])
        case["heads"] = min(case["heads"], 32 // case["kv"] * case["kv"])
        case.update(n_seq=n, q_lo=max(1, hi // 4), q_hi=hi, past_lo=0, past_hi=past)
    return case


def _lengths(case):
    """(new tokens, tokens already cached) of each sequence: the case's alone."""
    r = random.Random(case["mix"])
    q = [r.randint(case["q_lo"], case["q_hi"]) for _ in range(case["n_seq"])]
    past = [r.randint(case["past_lo"], case["past_hi"]) for _ in range(case["n_seq"])]
    return q, past


def _row_bytes(case):
    return case["hd"] * 2 if case["cache"] == "f16" else case["hd"] + case["hd"] // 16


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4.0 * n + 24.0 * case["rows"], "flops": 4.0 * n}
    q, past = _lengths(case)
    tokens, act = sum(q), 4 if case["act"] == "f32" else 2
    qd, kvd = case["heads"] * case["hd"], case["kv"] * case["hd"]
    if case["op"] == "cache":   # q in and out, k and v in, rows written, rows read, values out
        rows = 2 * tokens * case["kv"] * _row_bytes(case)
        return {"bytes": float(tokens * (2 * qd + 4 * kvd) * act + 2 * rows + tokens * case["hd"] * 4),
                "flops": float(3 * tokens * (qd + 3 * kvd))}
    kv_rows = sum(a + b for a, b in zip(q, past))
    pairs = sum(a * b + a * (a + 1) // 2 for a, b in zip(q, past))
    return {"bytes": float(2 * kv_rows * case["kv"] * _row_bytes(case) + 2 * tokens * qd * act),
            "flops": 4.0 * pairs * qd}


# ------------------------------------------------------------------ the inputs
def _quantise(x, one27):
    """Q8_0 of the last dimension: codes (int8) and scales (half)."""
    b = x.float().unflatten(-1, (-1, 32))
    d = (b.abs().amax(-1) / one27).clamp(max=65504.0).half()
    df = d.float().unsqueeze(-1)
    code = torch.where(df > 0, (b / df).round().clamp(-127, 127), torch.zeros_like(b))
    return code.to(torch.int8).flatten(-2), d


def _make_pool(case, n_pages, gen):
    """A pool of filled pages, [n_pages][kv][bytes of a page's rows of a head] as bytes."""
    kv, hd, page = case["kv"], case["hd"], case["page"]
    chan = torch.exp(0.4 * torch.randn(kv, 1, hd, device="cuda", generator=gen)).half()
    x = torch.randn(n_pages, kv, page, hd, device="cuda", generator=gen, dtype=torch.float16) * chan
    if case["cache"] == "f16":
        return x.reshape(n_pages, kv, page * hd).view(torch.uint8)
    pool = torch.empty(n_pages, kv, page * (hd + hd // 16), device="cuda", dtype=torch.uint8)
    codes, scales = _quantise(x, torch.full((), 127.0, device="cuda"))
    pool[..., : page * hd] = codes.reshape(n_pages, kv, page * hd).view(torch.uint8)
    pool[..., page * hd:] = scales.reshape(n_pages, kv, page * hd // 32).view(torch.uint8)
    return pool


def _prepare_sample(case, gen):
    rows, vocab, f = case["rows"], case["vocab"], case["filters"]
    dev = dict(device="cuda")
    # a bell of unlikely tokens, a power-law head of likely ones
    logits = torch.randn(rows, vocab, generator=gen, **dev) * 1.7
    head = torch.rand(rows, vocab, generator=gen, **dev).topk(300, dim=-1).indices
    rank = torch.arange(1, 301, **dev).float()
    logits.scatter_(1, head, (12.0 - 1.3 * torch.log(rank)).expand(rows, 300).contiguous())
    # a grammar's mask on every fourth row
    mask = torch.rand(rows, vocab, generator=gen, **dev) < 0.3
    mask &= (torch.arange(rows, **dev) % 4 == 3)[:, None]
    logits.masked_fill_(mask, float("-inf"))
    r = torch.arange(rows, **dev)
    temperature = torch.full((rows,), 0.8, **dev)
    top_k = torch.zeros(rows, dtype=torch.int32, **dev)
    top_p = torch.ones(rows, **dev)
    min_p = torch.zeros(rows, **dev)
    if f in ("all", "mixed"):
        top_k[:] = 40
        top_p[:] = 0.95
        min_p[:] = 0.05
    if f == "top_p":
        top_p[:] = 0.9
        temperature[:] = 1.0
    if f == "mixed":   # greedy, unfiltered, top-k alone, nucleus alone, all
        temperature[r % 5 == 0] = 0.0
        top_k[(r % 5 == 1) | (r % 5 == 3)] = 0
        top_p[(r % 5 == 1) | (r % 5 == 2)] = 1.0
        min_p[r % 5 != 4] = 0.0
    u = torch.rand(rows, generator=gen, **dev)
    return dict(case=case, logits=logits, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, u=u,
                out=torch.empty(rows, dtype=torch.int32, **dev))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    if case["op"] == "sample":
        return _prepare_sample(case, gen)
    heads, kv, hd, page = case["heads"], case["kv"], case["hd"], case["page"]
    q_len, past = _lengths(case)
    kv_len = [a + b for a, b in zip(q_len, past)]
    need = [-(-n // page) for n in kv_len]
    n_pages = sum(need) + sum(need) // 16 + 3   # some pages are free
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((case["n_seq"], max(need) + 1), -1, dtype=torch.int32)   # unused entries: -1
    host, at = order.cpu(), 0
    for s, n in enumerate(need):
        table[s, :n] = host[at: at + n]
        at += n
    act = torch.float32 if case["act"] == "f32" else torch.float16
    tokens = sum(q_len)
    cu = [0]
    for n in q_len:
        cu.append(cu[-1] + n)
    st = dict(case=case, k_pool=_make_pool(case, n_pages, gen), v_pool=_make_pool(case, n_pages, gen),
              n_pages=n_pages, table=table.cuda(), kv_len=torch.tensor(kv_len, dtype=torch.int32, device="cuda"),
              cu=torch.tensor(cu, dtype=torch.int32, device="cuda"), max_q=max(q_len), max_kv=max(kv_len),
              tokens=tokens, one27=torch.full((), 127.0, device="cuda"))
    if case["op"] == "cache":
        # q, k and v are columns of one projection's output
        width = (heads + 2 * kv) * hd
        st["qkv"] = torch.randn(tokens, width, generator=gen, device="cuda").to(act)
        ang = torch.arange(st["max_kv"], dtype=torch.float64)[:, None] * \
            (ROPE_THETA ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd))[None, :]
        st["rope"] = torch.stack([ang.cos(), ang.sin()], -1).float().reshape(st["max_kv"], hd).cuda()
        st["q_out"] = torch.empty(tokens, heads * hd, dtype=act, device="cuda")
        st["k_out"] = torch.empty(tokens, kv * hd, dtype=act, device="cuda")
        st["v_out"] = torch.empty(tokens, kv * hd, dtype=act, device="cuda")
    else:
        st["q"] = (1.5 * torch.randn(tokens, heads * hd, generator=gen, device="cuda")).to(act)
        st["out"] = torch.empty(tokens, heads * hd, dtype=act, device="cuda")
    return st


# ------------------------------------------------------------------ plain forms
def _places(st):
    """Each token's sequence, position, page and row."""
    t = torch.arange(st["tokens"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(st["cu"][1:], t, right=True)
    pos = st["kv_len"][seq] - (st["cu"][seq + 1] - t)
    page = st["table"][seq, torch.div(pos, st["case"]["page"], rounding_mode="floor").long()]
    return pos.long(), page.long(), (pos % st["case"]["page"]).long()


def _parts(st, pool):
    """A pool's rows: halves [pages][kv][page][hd], or codes and scales."""
    c = st["case"]
    n, kv, page, hd = st["n_pages"], c["kv"], c["page"], c["hd"]
    if c["cache"] == "f16":
        return pool.view(torch.float16).view(n, kv, page, hd), None
    codes = pool[..., : page * hd].view(torch.int8).unflatten(-1, (page, hd))
    return codes, pool[..., page * hd:].view(torch.float16).unflatten(-1, (page, hd // 32))


def _values(st, x, s):
    """fp32 values of gathered rows."""
    if s is None:
        return x.float()
    return (x.float().unflatten(-1, (-1, 32)) * s.float().unsqueeze(-1)).flatten(-2)


def _rope(x, cs):
    """Rotates the pairs of x [tokens][heads][hd] by cs [tokens][hd / 2][2]."""
    a, b = x.unflatten(-1, (-1, 2)).unbind(-1)
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    return torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)


def _plain_cache(st):
    c = st["case"]
    heads, kv, hd = c["heads"], c["kv"], c["hd"]
    act = st["qkv"].dtype
    pos, page, row = _places(st)
    q, k, v = st["qkv"].float().split([heads * hd, kv * hd, kv * hd], dim=1)
    cs = st["rope"][pos].unflatten(-1, (-1, 2))
    q = _rope(q.unflatten(-1, (heads, hd)), cs).flatten(1).to(act)
    k = _rope(k.unflatten(-1, (kv, hd)), cs)
    v = v.unflatten(-1, (kv, hd))

    def through(pool, x):
        rows, scales = _parts(st, pool)
        if scales is None:
            rows[page, :, row] = x.half()
            return rows[page, :, row].to(act).flatten(1)
        codes, d = _quantise(x, st["one27"])
        rows[page, :, row] = codes
        scales[page, :, row] = d
        return _values(st, rows[page, :, row], scales[page, :, row]).to(act).flatten(1)

    return [q, through(st["k_pool"], k), through(st["v_pool"], v)]


def _plain_attention(st):
    """Every sequence padded to the longest: gather, scores, softmax, sum."""
    c = st["case"]
    heads, kv, hd, page, n = c["heads"], c["kv"], c["hd"], c["page"], c["n_seq"]
    max_q, max_kv = st["max_q"], st["max_kv"]
    dev = st["q"].device
    key = torch.arange(max_kv, device=dev)
    pages = st["table"][:, torch.div(key, page, rounding_mode="floor")].clamp(min=0).long()   # [n][max_kv]
    row = key % page

    def gather(pool):
        rows, scales = _parts(st, pool)
        x = _values(st, rows[pages, :, row], None if scales is None else scales[pages, :, row])
        return x.permute(0, 2, 1, 3)   # [n][kv][max_kv][hd]

    i = torch.arange(max_q, device=dev)
    q_len = st["cu"][1:] - st["cu"][:-1]
    token = (st["cu"][:-1, None] + i).clamp(max=st["tokens"] - 1).long()      # [n][max_q]
    live = i < q_len[:, None]
    pos = st["kv_len"][:, None] - q_len[:, None] + i                          # [n][max_q]
    q = st["q"].float()[token].view(n, max_q, kv, heads // kv, hd).permute(0, 2, 3, 1, 4)
    q = q.reshape(n, kv, heads // kv * max_q, hd)
    s = torch.matmul(q, gather(st["k_pool"]).transpose(-1, -2)).mul_(hd ** -0.5)
    s = s.view(n, kv, heads // kv, max_q, max_kv)
    hidden = (key > pos[:, :, None])[:, None, None]
    s = s.masked_fill_(hidden, float("-inf"))
    s = s.sub_(s.amax(-1, keepdim=True)).exp_()
    total = s.sum(-1)
    o = torch.matmul(s.view(n, kv, -1, max_kv), gather(st["v_pool"])).view(n, kv, heads // kv, max_q, hd)
    o = (o / total.unsqueeze(-1)).permute(0, 3, 1, 2, 4).reshape(n, max_q, heads * hd)
    return o[live].to(st["q"].dtype)


def _share(total, part):
    """floor(total * part / 2^24) for integers, part <= 2^24."""
    return (total >> 24) * part + (((total & 0xFFFFFF) * part) >> 24)


def _plain_sample(st):
    logits = st["logits"]
    rows, vocab = logits.shape
    x, index = torch.sort(logits, dim=-1, descending=True, stable=True)
    hot = st["temperature"] > 0
    t = torch.where(hot, st["temperature"], torch.ones_like(st["temperature"]))
    e = torch.exp((x - x[:, :1]) / t[:, None])
    w = (e * 2.0 ** 40).round().to(torch.int64)
    rank = torch.arange(vocab, device=x.device)
    k = torch.where(st["top_k"] > 0, st["top_k"].long(), vocab)
    w = w * (rank < k[:, None])
    before = w.cumsum(-1) - w
    total = before[:, -1] + w[:, -1]
    p24 = (st["top_p"].clamp(0, 1) * 2.0 ** 24).round().to(torch.int64)
    kept = (before < _share(total, p24)[:, None]) | (rank == 0)
    w = w * (kept & (e >= st["min_p"][:, None]))
    w = torch.zeros_like(w).scatter_(1, index, w)   # by index again
    upto = w.cumsum(-1)
    u24 = (st["u"] * 2.0 ** 24).floor().to(torch.int64)
    target = _share(upto[:, -1], u24)
    token = (upto > target[:, None]).to(torch.uint8).argmax(-1)
    return torch.where(hot, token, index[:, 0]).to(torch.int32)


# ------------------------------------------------------------------ the framework's calls
def _handles(st, gb):
    """The cache, batch and workspace that a program keeps from step to step."""
    if "cache_h" not in st:
        c = st["case"]
        st["cache_h"] = gb.KVCache(gb.DT_F16 if c["cache"] == "f16" else gb.DT_Q8_0, c["kv"], c["hd"], c["page"],
                                   st["n_pages"], st["k_pool"], st["v_pool"])
        one = st["max_q"] == 1   # a decode batch: one token per sequence
        st["batch_h"] = gb.KVBatch(c["n_seq"], st["tokens"], st["kv_len"], st["table"], None if one else st["cu"])
        st["ws"] = torch.zeros(gb.paged_workspace_bytes(c["heads"], c["kv"], c["hd"], c["n_seq"]), dtype=torch.uint8,
                               device="cuda")
    return st["cache_h"], st["batch_h"], st["ws"]


def run(st):
    c = st["case"]
    if not own:
        if c["op"] == "cache":
            return _plain_cache(st)
        return _plain_sample(st) if c["op"] == "sample" else _plain_attention(st)
    import guanaco_b200 as gb
    if c["op"] == "sample":
        gb.sample(st["logits"], st["out"], st["u"], temperature=st["temperature"], top_k=st["top_k"],
                  top_p=st["top_p"], min_p=st["min_p"])
        return st["out"]
    cache, batch, ws = _handles(st, gb)
    if c["op"] == "cache":
        qd, kvd = c["heads"] * c["hd"], c["kv"] * c["hd"]
        qkv = st["qkv"]
        gb.kv_append(cache, batch, qkv[:, qd: qd + kvd], qkv[:, qd + kvd:], q=qkv[:, :qd], q_out=st["q_out"],
                     rope_cs=st["rope"])
        gb.kv_read(cache, batch, st["k_out"], st["v_out"])
        return [st["q_out"], st["k_out"], st["v_out"]]
    attend = gb.paged_attention_decode if c["op"] == "decode" else gb.paged_attention_prefill
    attend(cache, batch, st["q"], st["out"], ws)
    return st["out"]


# ------------------------------------------------------------------ 64 bits
def _exact_rows(st, pool, seq, n):
    """Sequence seq's first n rows of a pool as float64 [kv][n][hd]."""
    c = st["case"]
    kv, page, hd = c["kv"], c["page"], c["hd"]
    ids = st["table"][seq, : -(-n // page)].long()
    raw = pool[ids]
    if c["cache"] == "f16":
        x = raw.view(torch.float16).reshape(len(ids), kv, page, hd).double()
    else:
        code = raw[..., : page * hd].view(torch.int8).reshape(len(ids), kv, page, hd // 32, 32).double()
        d = raw[..., page * hd:].view(torch.float16).reshape(len(ids), kv, page, hd // 32, 1).double()
        x = (code * d).reshape(len(ids), kv, page, hd)
    return x.transpose(0, 1).reshape(kv, -1, hd)[:, :n]


def _exact_attention(st):
    c = st["case"]
    kv, hd, group = c["kv"], c["hd"], c["heads"] // c["kv"]
    q_len, past = _lengths(c)
    out, t0 = [], 0
    for s, (n, p) in enumerate(zip(q_len, past)):
        k, v = _exact_rows(st, st["k_pool"], s, n + p), _exact_rows(st, st["v_pool"], s, n + p)
        q = st["q"][t0: t0 + n].double().reshape(n, kv, group, hd)
        t0 += n
        o = torch.empty(n, kv, group, hd, dtype=torch.float64, device="cuda")
        seen = torch.arange(n + p, device="cuda")[None, :] <= torch.arange(p, p + n, device="cuda")[:, None]
        for g in range(kv):
            for j in range(group):
                score = (q[:, g, j] @ k[g].T) / hd ** 0.5
                o[:, g, j] = torch.softmax(score.masked_fill(~seen, float("-inf")), -1) @ v[g]
        out.append(o.reshape(n, -1))
    return torch.cat(out)


def _exact_cache(st):
    c = st["case"]
    heads, kv, hd = c["heads"], c["kv"], c["hd"]
    q_len, past = _lengths(c)
    pos = np.concatenate([np.arange(p, p + n) for n, p in zip(q_len, past)])
    x = st["qkv"].double().reshape(-1, heads + 2 * kv, hd // 2, 2)
    turn = torch.view_as_complex(st["rope"].double()[torch.from_numpy(pos).cuda()].reshape(-1, 1, hd // 2, 2))
    turned = torch.view_as_real(torch.view_as_complex(x[:, : heads + kv].contiguous()) * turn)

    def stored(y):
        y = y.reshape(-1, kv * hd)
        if c["cache"] == "f16":
            return y.half().double()
        b = y.reshape(len(y), -1, 32)
        d = (b.abs().amax(-1, keepdim=True) / 127).half().double()
        return torch.where(d > 0, (b / d).round().clamp(-127, 127) * d, torch.zeros_like(b)).reshape(len(y), -1)

    return [turned[:, :heads].reshape(-1, heads * hd), stored(turned[:, heads:]), stored(x[:, heads + kv:])]


def exact(case, seed):
    if case["op"] == "sample":
        return None   # tokens are whole numbers
    st = prepare(case, seed)
    return _exact_cache(st) if case["op"] == "cache" else _exact_attention(st)
