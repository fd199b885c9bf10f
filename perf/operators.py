"""The operators of the 8-bit integer KV cache: what is measured, in plain torch and through the framework.

A pool of dtype "int8" holds K and V as 8-bit codes with one scale for each (token, kv head) row, written as the token
is appended.  For a row x of head_dim values: amax = min(max(max |x|, 2^-40), 2^64), scale = amax / 127,
code = round_half_even(127 x / amax) clamped to [-127, 127]; the row stands for code * scale.  Four operators:

  write   quantise the rows of a step's new tokens into their pages, and read those rows back
  read    rows of token ranges of several sequences, dequantised into contiguous tensors
  decode  quantise one new token per sequence and attend from it to the whole sequence
  chunk   quantise a chunk of new tokens per sequence and attend from each of them to the tokens up to its own

Attention: out = softmax(q k / sqrt(head_dim)) v over the tokens up to the query's own, `heads / kv_heads` query heads
to a kv head, tokens stored 16 to a page, pages anywhere in the pool.
"""
import math
import random

import torch

own = False

PAGE = 16


def listed():
    return [
        # 64 sequences write one new token each at the 8B head shape: the smallest write, all latency
        dict(name="write_step", op="write", io="bf16", heads=32, kv_heads=8, dim=128, seqs=64, ctx_lo=1024, ctx_hi=2048, new_lo=1, new_hi=1),
        # 64 prompts of 512 tokens enter the cache in one step (the append step that the benchmark times)
        dict(name="write_prompts", op="write", io="bf16", heads=32, kv_heads=8, dim=128, seqs=64, ctx_lo=0, ctx_hi=0, new_lo=512, new_hi=512),
        # a few ragged ranges of a small model's cache (head_dim 64, fp16), as a prefix is exported
        dict(name="read_ranges", op="read", io="fp16", heads=8, kv_heads=2, dim=64, seqs=5, ctx_lo=33, ctx_hi=701, new_lo=1, new_hi=601),
        # 32 whole sequences leave the cache for another machine
        dict(name="read_sequences", op="read", io="bf16", heads=32, kv_heads=8, dim=128, seqs=32, ctx_lo=2048, ctx_hi=6144, new_lo=2048, new_hi=6144),
        # one short sequence of the tiny configuration decodes: the smallest attention
        dict(name="decode_tiny", op="decode", io="fp16", heads=8, kv_heads=2, dim=64, seqs=1, ctx_lo=164, ctx_hi=164, new_lo=1, new_hi=1),
        # the benchmark's batch: 64 sequences of 1024 to 8192 tokens, 32 query heads on 8 kv heads
        dict(name="decode_batch", op="decode", io="bf16", heads=32, kv_heads=8, dim=128, seqs=64, ctx_lo=1024, ctx_hi=8192, new_lo=1, new_hi=1),
        # one long sequence, fp16: the work is split along the context
        dict(name="decode_long", op="decode", io="fp16", heads=32, kv_heads=8, dim=128, seqs=1, ctx_lo=65535, ctx_hi=65535, new_lo=1, new_hi=1),
        # the benchmark's 8-bit batch: 64 query heads on 8 kv heads, 32 sequences of 32768 tokens
        dict(name="decode_wide", op="decode", io="bf16", heads=64, kv_heads=8, dim=128, seqs=32, ctx_lo=32768, ctx_hi=32768, new_lo=1, new_hi=1),
        # verification of four drafted tokens per sequence
        dict(name="chunk_verify", op="chunk", io="bf16", heads=32, kv_heads=8, dim=128, seqs=64, ctx_lo=1024, ctx_hi=8192, new_lo=4, new_hi=4),
        # sequences with a prompt chunk of any length, one token among them, head_dim 64
        dict(name="chunk_ragged", op="chunk", io="fp16", heads=16, kv_heads=4, dim=64, seqs=9, ctx_lo=0, ctx_hi=1500, new_lo=1, new_hi=517),
        # prompt chunks of 1024 tokens on contexts of up to 4096
        dict(name="chunk_prompts", op="chunk", io="bf16", heads=32, kv_heads=8, dim=128, seqs=8, ctx_lo=0, ctx_hi=4096, new_lo=1024, new_hi=1024),
        # one fresh prompt of 8192 tokens, 64 query heads on 8 kv heads
        dict(name="chunk_fresh", op="chunk", io="fp16", heads=64, kv_heads=8, dim=128, seqs=1, ctx_lo=0, ctx_hi=0, new_lo=8192, new_hi=8192),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["write", "read", "decode", "chunk"])
    kv = rng.choice([1, 2, 3, 4, 8])
    c = dict(op=op, io=rng.choice(["bf16", "fp16"]), heads=kv * rng.choice([1, 2, 4, 8, 16]), kv_heads=kv, dim=rng.choice([64, 128, 128]),
             seqs=_log(rng, 1, 64))
    room = 200000 // c["seqs"]                              # tokens a sequence may hold at most
    hi = _log(rng, 1, min(room, 32768))
    c["ctx_hi"] = hi if op != "read" else max(hi, 2)
    c["ctx_lo"] = rng.randint(0 if op in ("write", "chunk") else 1, c["ctx_hi"])
    if op == "decode":
        c["new_lo"] = c["new_hi"] = 1
    elif op == "read":
        c["new_hi"] = _log(rng, 1, c["ctx_hi"])
        c["new_lo"] = rng.randint(1, c["new_hi"])
    elif op == "write":
        c["new_hi"] = _log(rng, 1, min(room, 4096))
        c["new_lo"] = rng.randint(1, c["new_hi"])
    else:
        # (query head, position) pairs stay below those of the largest listed chunk, padded to the longest row
        c["ctx_hi"] = min(c["ctx_hi"], 16384)
        c["ctx_lo"] = min(c["ctx_lo"], c["ctx_hi"])
        cap = 1000000000 // (c["seqs"] * c["heads"])
        most = max(1, int((-c["ctx_hi"] + math.sqrt(c["ctx_hi"] ** 2 + 4 * cap)) / 2))
        c["new_hi"] = _log(rng, 1, min(most, 4096))
        c["new_lo"] = rng.randint(1, c["new_hi"])
    return c


# ---- sizes and inputs of a case ------------------------------------------------------------------------------

def _lengths(c):
    """(tokens held before the call, new tokens or tokens to read, first token to read) of each sequence: the case's own."""
    r = random.Random("%(seqs)d %(ctx_lo)d %(ctx_hi)d %(new_lo)d %(new_hi)d" % c)
    ctx = [r.randint(c["ctx_lo"], c["ctx_hi"]) for _ in range(c["seqs"])]
    new = [r.randint(c["new_lo"], c["new_hi"]) for _ in range(c["seqs"])]
    if c["op"] == "read":
        new = [min(n, x) for n, x in zip(new, ctx)]
        return ctx, new, [r.randint(0, x - n) for n, x in zip(new, ctx)]
    return ctx, new, ctx


def _type(c):
    return torch.bfloat16 if c["io"] == "bf16" else torch.float16


def _rows(gen, n, c):
    """K and V rows of n tokens: keys with a few strong channels, values whose size differs from token to token."""
    h, d, dev = c["kv_heads"], c["dim"], "cuda"
    strong = torch.where(torch.rand(h, d, device=dev, generator=gen) < 0.03, 6.0, 1.0)
    k = torch.randn(n, h, d, device=dev, generator=gen) * strong
    v = torch.randn(n, h, d, device=dev, generator=gen) * torch.exp(0.5 * torch.randn(n, h, 1, device=dev, generator=gen))
    return k.to(_type(c)), v.to(_type(c))


def _inputs(c, seed):
    ctx, new, _ = _lengths(c)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    old_k, old_v = _rows(gen, sum(ctx), c)
    k, v = _rows(gen, 0 if c["op"] == "read" else sum(new), c)
    q = torch.randn(k.shape[0], c["heads"], c["dim"], device="cuda", generator=gen).to(_type(c))
    return old_k, old_v, k, v, q


def work(c):
    ctx, new, _ = _lengths(c)
    h, d, n = c["kv_heads"], c["dim"], sum(new)
    row = 2 * h * (d + 4)                                   # a token's K and V in the cache: codes and scales
    io = 2 * h * d * 2                                      # ... and outside it
    if c["op"] == "read":
        return {"bytes": n * (row + io), "flops": n * 2 * h * d}
    if c["op"] == "write":
        return {"bytes": n * (io + row + io), "flops": n * 2 * h * d * 4}
    seen = sum(t * x + t * (t + 1) // 2 for x, t in zip(ctx, new))
    return {"bytes": (sum(ctx) + n) * row + n * io + 2 * n * c["heads"] * d * 2, "flops": 4 * d * c["heads"] * seen}


# ---- the plain forms ------------------------------------------------------------------------------------------

def _quantise(x):
    """Rows [..., D] -> (codes as int8, scales)."""
    x = x.float()
    amax = x.abs().amax(-1, keepdim=True).clamp(2.0 ** -40, 2.0 ** 64)
    return torch.round(127.0 * x / amax).clamp(-127, 127).to(torch.int8), (amax / 127.0).squeeze(-1)


def _write(s, k, v, page, row):
    s["k"][page, row], s["ks"][page, row] = _quantise(k)
    s["v"][page, row], s["vs"][page, row] = _quantise(v)


def _attend(s, q):
    """Every new token of every sequence against its sequence's pages, sequences and chunks padded to the longest."""
    b, t = s["pad"].shape
    h, d = s["ks"].shape[2], q.shape[-1]
    g = q.shape[1] // h
    keys = (s["k"][s["table"]].float() * s["ks"][s["table"]][..., None]).reshape(b, -1, h, d).permute(0, 2, 3, 1)
    scores = q[s["pad"]].float().reshape(b, t, h, g, d).permute(0, 2, 1, 3, 4).reshape(b, h, t * g, d) @ keys
    del keys
    scores = scores.view(b, h, t, g, -1).mul_(1.0 / math.sqrt(d))
    scores.masked_fill_((s["place"][None, None, :] > s["last"][:, :, None])[:, None, :, None, :], -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1, keepdim=True)
    values = (s["v"][s["table"]].float() * s["vs"][s["table"]][..., None]).reshape(b, -1, h, d).transpose(1, 2)
    out = (scores.view(b, h, t * g, -1) @ values).view(b, h, t, g, d) / total
    return out.permute(0, 2, 1, 3, 4).reshape(b, t, h * g, d)[s["of"], s["nth"]].to(q.dtype)


def _read(s):
    kind = s["io"]
    return ((s["k"][s["page"], s["row"]].float() * s["ks"][s["page"], s["row"]][..., None]).to(kind),
            (s["v"][s["page"], s["row"]].float() * s["vs"][s["page"], s["row"]][..., None]).to(kind))


def _prepare_plain(c, seed):
    ctx, new, start = _lengths(c)
    old_k, old_v, k, v, q = _inputs(c, seed)
    dev = "cuda"
    held = [x if c["op"] == "read" else x + n for x, n in zip(ctx, new)]
    pages = [(x + PAGE - 1) // PAGE for x in held]
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed + 1)
    free = torch.randperm(sum(pages), device=dev, generator=gen)
    table = torch.nn.utils.rnn.pad_sequence(list(free.split(pages)), batch_first=True)

    def places(first, count):                               # (sequence, index in its run, position) of runs of tokens
        count_t, first_t = torch.tensor(count, device=dev), torch.tensor(first, device=dev)
        of = torch.repeat_interleave(torch.arange(len(count), device=dev), count_t)
        nth = torch.arange(of.numel(), device=dev) - (count_t.cumsum(0) - count_t)[of]
        return of, nth, first_t[of] + nth

    h, d, p = c["kv_heads"], c["dim"], sum(pages)
    s = {"op": c["op"], "io": _type(c), "table": table, "new": (k, v, q)}
    for name in ("k", "v"):
        s[name] = torch.zeros(p, PAGE, h, d, dtype=torch.int8, device=dev)
        s[name + "s"] = torch.zeros(p, PAGE, h, device=dev)
    of, _, pos = places([0] * len(ctx), ctx)
    _write(s, old_k, old_v, table[of, pos // PAGE], pos % PAGE)
    of, nth, pos = places(start, new)
    s["page"], s["row"], s["of"], s["nth"] = table[of, pos // PAGE], pos % PAGE, of, nth
    first = torch.tensor(new, device=dev).cumsum(0) - torch.tensor(new, device=dev)
    step = torch.minimum(torch.arange(max(new), device=dev)[None, :], torch.tensor(new, device=dev)[:, None] - 1)
    s["pad"] = first[:, None] + step                        # row of q of each (sequence, new token), the last one repeated
    s["last"] = torch.tensor(start, device=dev)[:, None] + step
    s["place"] = torch.arange(table.shape[1] * PAGE, device=dev)
    return s


def _run_plain(s):
    k, v, q = s["new"]
    if s["op"] == "read":
        return _read(s)
    _write(s, k, v, s["page"], s["row"])
    return _read(s) if s["op"] == "write" else _attend(s, q)


# ---- the framework's --------------------------------------------------------------------------------------------

def _prepare_own(c, seed):
    from titan_engine_b200 import PagedKVCache
    ctx, new, start = _lengths(c)
    old_k, old_v, k, v, q = _inputs(c, seed)
    held = [x if c["op"] == "read" else x + n for x, n in zip(ctx, new)]
    pages = [(x + PAGE - 1) // PAGE for x in held]
    slice_ = 16384
    cache = PagedKVCache(1, c["heads"], c["kv_heads"], c["dim"], sum(pages), len(ctx), max(pages), dtype="int8", io_dtype=c["io"],
                         max_step_tokens=max(slice_, sum(new)))
    seqs = [cache.seq_alloc() for _ in ctx]
    at = 0
    for sid, n in zip(seqs, ctx):
        for lo in range(0, n, slice_):
            m = min(slice_, n - lo)
            cache.step_begin([sid], [m])
            cache.append(0, old_k[at:at + m], old_v[at:at + m])
            at += m
    return {"op": c["op"], "cache": cache, "seqs": seqs, "start": start, "count": new, "new": (k, v, q)}


def _run_own(s):
    """A step from its beginning: pages for the new tokens, the plan and its upload, then the layer's call."""
    cache, (k, v, q) = s["cache"], s["new"]
    if s["op"] == "read":
        return cache.read(0, s["seqs"], s["start"], s["count"])
    cache.step_begin(s["seqs"], s["count"])
    if s["op"] == "write":
        cache.append(0, k, v)
        out = cache.read(0, s["seqs"], s["start"], s["count"])
    elif s["op"] == "decode":
        out = cache.append_decode(0, k, v, q)
    else:
        out = cache.append_decode_multi(0, k, v, q)
    for seq, held in zip(s["seqs"], s["start"]):            # the step is taken back, so that the next pass finds what this one found
        cache.truncate(seq, held)
    return out


def prepare(case, seed):
    return _prepare_own(case, seed) if own else _prepare_plain(case, seed)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definition in 64 bits ------------------------------------------------------------------------------------

def _stands_for(x):
    """What rows stand for once they are in the cache, in 64 bits."""
    x = x.double()
    amax = torch.linalg.vector_norm(x, math.inf, dim=-1, keepdim=True).clamp(2.0 ** -40, 2.0 ** 64)
    unit = amax / 127
    return (x * 127 / amax).round().clamp(-127, 127) * unit


def exact(case, seed):
    ctx, new, start = _lengths(case)
    old_k, old_v, k, v, q = _inputs(case, seed)
    if case["op"] == "write":
        return _stands_for(k), _stands_for(v)
    if case["op"] == "read":
        begin, rows = 0, []
        for n, lo, count in zip(ctx, start, new):
            rows.append(torch.arange(begin + lo, begin + lo + count, device="cuda"))
            begin += n
        rows = torch.cat(rows)
        return _stands_for(old_k[rows]), _stands_for(old_v[rows])
    group = case["heads"] // case["kv_heads"]
    outs, a, b = [], 0, 0
    for n, t in zip(ctx, new):
        keys = _stands_for(torch.cat([old_k[a:a + n], k[b:b + t]]))
        vals = _stands_for(torch.cat([old_v[a:a + n], v[b:b + t]]))
        query = q[b:b + t].double() / math.sqrt(case["dim"])
        a, b = a + n, b + t
        out = torch.empty(t, case["heads"], case["dim"], dtype=torch.float64, device="cuda")
        for head in range(case["heads"]):
            logits = query[:, head] @ keys[:, head // group].T
            logits += torch.full_like(logits, -math.inf).triu_(n + 1)
            weights = torch.softmax(logits, -1)
            out[:, head] = weights @ vals[:, head // group]
        outs.append(out)
    return torch.cat(outs)
