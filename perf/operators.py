"""Operators of a serving step around the attention of a layer, each in its plain form and as the framework's call.

  rotary    rotary_embedding: rotary positions of q and k, half or interleaved layout, whole heads or part of them
  append    quantize_and_scatter: new K/V rows into the 8-bit paged cache (e4m3 codes, one scale per 16 tokens and head)
  attend    paged_attention_8bit: attention over that cache: one query token per sequence, a few, or prompt chunks
  plan      plan_step: block tables, slot map, positions and lengths of a step from the requests' lengths
  release   release_blocks: the blocks of ended requests back on the stack of free blocks

`own` says which of the two run() computes.  The plain forms are elementary torch operations in 32 bits, rounded once.
"""
import math
import os
import sys

import torch

sys.path.insert(0, os.path.abspath("turboquant-amd_b200"))   # imported with the repository's root as working folder

own = False

DEV = "cuda:0"
PAGE = 16                      # tokens that share a scale
E4M3_MAX = 448.0
MIN_EXPONENT = -100
OUTLIER_CHANNELS = [5, 23, 50]
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
ITEM = {"fp16": 2, "bf16": 2}
POSITIONS = 131072


def listed():
    return [
        # q and k of one decode step of 64 sequences: the smallest call, once per layer.
        dict(op="rotary", rows=64, q_heads=64, kv_heads=8, head_dim=128, rotary_dim=128, interleaved=False, scaling="llama3",
             inverse=False, dtype="fp16", name="rotary 64 half fp16"),
        # A batch of prompts in one call, half of each head rotated, interleaved, context stretched by YaRN; ragged length.
        dict(op="rotary", rows=16411, q_heads=32, kv_heads=8, head_dim=128, rotary_dim=64, interleaved=True, scaling="yarn",
             inverse=False, dtype="bf16", name="rotary 16411 part bf16"),
        # The new tokens of a decode step: pages partly filled, some scales grow.
        dict(op="append", lens="ones:64", kv_heads=8, head_dim=128, block_size=16, dtype="fp16", name="append 64"),
        # Prompts of 24 sequences of mixed lengths, some continuing a page; K and V are views of the fused projection.
        dict(op="append", lens="lognormal:24:2048:0.8:1:8192", kv_heads=8, head_dim=128, block_size=32, dtype="bf16",
             name="append 24 prompts bf16"),
        # One interactive user with a 4096-token context: latency.
        dict(op="attend", queries="ones:1", context="fixed:4095", q_heads=32, kv_heads=8, head_dim=128, block_size=16,
             dtype="fp16", name="attend 1x4096"),
        # Batched serving at a common length: the shape of the default benchmark.
        dict(op="attend", queries="ones:64", context="fixed:8191", q_heads=64, kv_heads=8, head_dim=128, block_size=16,
             dtype="fp16", name="attend 64x8192"),
        # A serving batch of mixed lengths, from one token to long contexts.
        dict(op="attend", queries="ones:64", context="lognormal:64:2048:1.0:0:16000", q_heads=32, kv_heads=8, head_dim=128,
             block_size=32, dtype="bf16", name="attend 64 mixed bf16"),
        # Prompt chunks that continue cached contexts of different lengths.
        dict(op="attend", queries="uniform:4:700:1024", context="uniform:4:1000:7168", q_heads=32, kv_heads=8, head_dim=128,
             block_size=16, dtype="bf16", name="attend 4 chunks bf16"),
        # The tables of one decode step of 64 requests, tables as wide as the longest allowed context.
        dict(op="plan", queries="ones:64", context="uniform:64:1:8192", block_size=16, width=2048, name="plan 64"),
        # A step of 1000 requests, prompts among them.
        dict(op="plan", queries="lognormal:1000:40:1.5:0:4000", context="lognormal:1000:1500:1.0:0:16000", block_size=16,
             width=2048, name="plan 1000"),
        # Three of 64 requests end.
        dict(op="release", context="uniform:64:1:8192", ended=3, block_size=16, width=2048, name="release 3 of 64"),
        # A batch job ends: 900 of 1000 requests.
        dict(op="release", context="lognormal:1000:1500:1.0:0:16000", ended=900, block_size=16, width=2048,
             name="release 900 of 1000"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["rotary", "rotary", "append", "append", "attend", "attend", "attend", "plan", "release"])
    if op == "rotary":
        dim = rng.choice([64, 80, 96, 128, 128, 192, 256])
        hq, hk = rng.choice([(1, 1), (8, 1), (12, 4), (28, 4), (32, 8), (64, 8)])
        most = 16411 * 40 * 128 // ((hq + hk) * dim)
        return dict(op=op, rows=_log(rng, 1, most), q_heads=hq, kv_heads=hk, head_dim=dim,
                    rotary_dim=rng.choice([dim, dim, dim // 2, dim // 4]), interleaved=rng.random() < 0.4,
                    scaling=rng.choice(["none", "linear", "yarn", "llama3"]), inverse=rng.random() < 0.2,
                    dtype=rng.choice(["fp16", "bf16", "bf16"]))
    if op == "append":
        if rng.random() < 0.4:
            lens = "ones:%d" % _log(rng, 1, 2048)
        else:
            n = _log(rng, 1, 64)
            lens = "lognormal:%d:%d:0.8:1:%d" % (n, _log(rng, 4, 40000 // n), 49152 // n)
        return dict(op=op, lens=lens, kv_heads=rng.choice([1, 2, 4, 8]), head_dim=rng.choice([64, 128, 128]),
                    block_size=rng.choice([16, 16, 32]), dtype=rng.choice(["fp16", "bf16"]))
    if op == "attend":
        hk, dim = rng.choice([1, 2, 4, 8, 8]), rng.choice([64, 128, 128])
        hq = hk * rng.choice([1, 2, 4, 5, 8, 8, 16] if hk < 8 else [1, 4, 7, 8])
        kind = rng.choice(["decode", "decode", "few", "chunks"])
        if kind == "chunks":
            n, most = _log(rng, 1, 8), rng.choice([64, 256, 700, 1024])
            longest = max(16, min(16384, (1 << 30) // (n * hq * most)) - most)
            return dict(op=op, queries="uniform:%d:1:%d" % (n, most), context="uniform:%d:0:%d" % (n, longest), q_heads=hq, kv_heads=hk,
                        head_dim=dim, block_size=rng.choice([16, 32]), dtype=rng.choice(["fp16", "bf16"]))
        n = _log(rng, 1, 256)
        longest = _log(rng, 32, max(32, min(32768, (1 << 29) // (n * hk * dim))))
        context = rng.choice(["fixed:%d" % longest, "uniform:%d:0:%d" % (n, longest),
                              "lognormal:%d:%d:1.0:0:%d" % (n, max(1, longest // 4), longest)])
        return dict(op=op, queries="ones:%d" % n if kind == "decode" else "uniform:%d:1:%d" % (n, rng.choice([2, 4, 8])),
                    context=context, q_heads=hq, kv_heads=hk, head_dim=dim, block_size=rng.choice([16, 16, 32]),
                    dtype=rng.choice(["fp16", "bf16"]))
    n = _log(rng, 1, 1000)
    context = "lognormal:%d:%d:1.0:0:16000" % (n, _log(rng, 10, 4000))
    if op == "plan":
        queries = rng.choice(["ones:%d" % n, "lognormal:%d:%d:1.0:0:4000" % (n, _log(rng, 1, 60))])
        return dict(op=op, queries=queries, context=context, block_size=rng.choice([16, 32]), width=rng.choice([1250, 2048]))
    return dict(op=op, context=context, ended=rng.randint(0, n), block_size=rng.choice([16, 32]), width=rng.choice([1000, 2048]))


# ---- inputs ------------------------------------------------------------------------------------
def _lengths(spec, n=None, salt=0):
    """Lengths of a batch: a property of the case, the same for every seed."""
    kind, *a = spec.split(":")
    g = torch.Generator().manual_seed(1234 + salt)
    if kind == "ones":
        return torch.ones(int(a[0]), dtype=torch.int64)
    if kind == "fixed":
        return torch.full((n,), int(a[0]), dtype=torch.int64)
    if kind == "uniform":
        return torch.randint(int(a[1]), int(a[2]) + 1, (int(a[0]),), generator=g)
    z = torch.randn(int(a[0]), generator=g) * float(a[2]) + math.log(float(a[1]))
    return z.exp().round().clamp(float(a[3]), float(a[4])).to(torch.int64)


def _vectors(g, dtype, *shape):
    x = torch.randn(*shape, generator=g, device=DEV, dtype=DTYPES[dtype])
    for ch in OUTLIER_CHANNELS:
        x[..., ch] *= 10
    return x


def _inverse_frequencies(dim, scaling):
    """fp64 angular frequencies of the `dim` / 2 pairs and the factor on cos and sin."""
    i = torch.arange(0, dim, 2, dtype=torch.float64)
    base = 10000.0 if scaling in ("none", "linear") else 500000.0
    f = base ** (-i / dim)
    if scaling == "linear":
        return f / 4.0, 1.0
    if scaling == "llama3":      # low frequencies divided by 8, a ramp between wavelengths of 8192 / 4 and 8192
        turns = 8192.0 * f / (2 * math.pi)
        ramp = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return f / 8.0 * (1 - ramp) + f * ramp, 1.0
    if scaling == "yarn":        # a ramp over the pairs between 32 and 1 turns in 8192 positions, factor 16
        at = lambda turns: dim * math.log(8192 / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), dim - 1)
        ramp = ((torch.arange(dim // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
        return f / 16.0 * ramp + f * (1 - ramp), 0.1 * math.log(16.0) + 1.0
    return f, 1.0


def _prepare_rotary(case, g):
    T, hq, hk, dim = case["rows"], case["q_heads"], case["kv_heads"], case["head_dim"]
    f, factor = _inverse_frequencies(case["rotary_dim"], case["scaling"])
    angle = torch.arange(POSITIONS, device=DEV, dtype=torch.float64)[:, None] * f.to(DEV)
    table = torch.cat([angle.cos() * factor, angle.sin() * factor], 1).float()
    qkv = _vectors(g, case["dtype"], T, hq + 2 * hk, dim)           # views of one fused projection
    start = torch.randint(0, POSITIONS - T, (1,), generator=g, device=DEV)
    pos = start + torch.arange(T, device=DEV) if T > 256 else torch.randint(0, POSITIONS, (T,), generator=g, device=DEV)
    return dict(q=qkv[:, :hq], k=qkv[:, hq:hq + hk], positions=pos, table=table, interleaved=case["interleaved"], inverse=case["inverse"],
                dim=case["rotary_dim"])


def _exponent(amax):
    """Smallest e with amax <= 448 * 2^e."""
    m, x = torch.frexp(amax)
    return torch.where(amax > 0, x - 9 + (m > 0.875).to(x.dtype), MIN_EXPONENT).clamp(min=MIN_EXPONENT)


def _empty_cache(blocks, bs, heads, dim):
    """The cache and its two views: codes [blocks, heads, pages, K/V, 16, dim] and scales [blocks, heads, pages, K/V]."""
    page = 2 * PAGE * dim + 32
    cache = torch.zeros(blocks, heads, bs // PAGE * page, dtype=torch.uint8, device=DEV)
    by_page = cache.view(blocks, heads, bs // PAGE, page)
    codes = by_page[..., :2 * PAGE * dim].unflatten(-1, (2, PAGE, dim)).view(torch.float8_e4m3fn)
    scales = by_page[..., 2 * PAGE * dim:2 * PAGE * dim + 8].view(torch.float32)
    return cache, codes, scales


def _fill(g, codes, scales):
    """Pages as quantize_and_scatter leaves them, filled with K/V of N(0, 1) and outlier channels."""
    for a in range(0, codes.shape[0], 8192):
        x = _vectors(g, "fp32", *codes[a:a + 8192].shape)
        e = _exponent(x.abs().amax((-1, -2)))
        scales[a:a + 8192] = torch.ldexp(torch.ones_like(scales[a:a + 8192]), e)
        codes[a:a + 8192] = torch.ldexp(x, -e[..., None, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def _tables(g, lens, bs, width=0):
    blocks = (lens + bs - 1) // bs
    n = max(1, int(blocks.sum()))
    start = (torch.cumsum(blocks, 0) - blocks).to(DEV)
    perm = torch.randperm(n, generator=g, device=DEV)
    col = torch.arange(max(1, int(blocks.max()), width), device=DEV)
    at = (start[:, None] + col).clamp(max=n - 1)
    return torch.where(col < blocks.to(DEV)[:, None], perm[at], 0).to(torch.int32), n


def _rows(query):
    """(sequence, index within it) of every row."""
    seq = torch.repeat_interleave(torch.arange(len(query)), query)
    return seq, torch.arange(int(query.sum())) - (torch.cumsum(query, 0) - query)[seq]


def _values(codes):
    """The values of codes, which are indexed as bytes."""
    return codes.view(torch.float8_e4m3fn)


def _prepare_append(case, g):
    query, H, dim, bs = _lengths(case["lens"]), case["kv_heads"], case["head_dim"], case["block_size"]
    n, T = len(query), int(query.sum())
    ctx = _lengths("uniform:%d:0:%d" % (n, 3 * bs), salt=5)                 # tokens that the sequences have already
    tables, blocks = _tables(g, ctx + query, bs)
    cache, codes, scales = _empty_cache(blocks, bs, H, dim)
    _fill(g, codes, scales)
    seq, j = (t.to(DEV) for t in _rows(query))
    pos = ctx.to(DEV)[seq] + j
    slots = tables[seq, pos // bs].to(torch.int64) * bs + pos % bs
    kv = _vectors(g, case["dtype"], T, 2 * H, dim) * 1.3
    kv *= torch.randn(T, 1, 1, generator=g, device=DEV).mul(0.4).exp().to(kv.dtype)     # tokens differ in size
    return dict(key=kv[:, :H], value=kv[:, H:], cache=cache, codes=codes, scales=scales, slots=slots, block_size=bs)


def _prepare_attend(case, g):
    query = _lengths(case["queries"])
    n, dim, bs = len(query), case["head_dim"], case["block_size"]
    lens = _lengths(case["context"], n, salt=9) + query
    tables, blocks = _tables(g, lens, bs)
    cache, codes, scales = _empty_cache(blocks, bs, case["kv_heads"], dim)
    _fill(g, codes, scales)
    T = int(query.sum())
    q = torch.randn(T, case["q_heads"], dim, generator=g, device=DEV, dtype=DTYPES[case["dtype"]])
    start = torch.nn.functional.pad(torch.cumsum(query, 0), (1, 0)).to(DEV, torch.int32)
    return dict(q=q, cache=cache, codes=codes, scales=scales, tables=tables, lens=lens.to(DEV, torch.int32), start=start, block_size=bs,
                most_queries=int(query.max()), longest=int(lens.max()))


def _prepare_plan(case, g):
    ctx, bs = _lengths(case["context"], salt=9), case["block_size"]
    n = len(ctx)
    tables, blocks = _tables(g, ctx, bs, case["width"])
    s = dict(context=ctx.to(DEV, torch.int32), tables=tables, block_size=bs, n=n)
    if case["op"] == "plan":
        query = _lengths(case["queries"])
        pool = int(query.sum()) // bs + 2 * n
        s |= dict(query=query.to(DEV, torch.int32), rows=int(query.sum()),
                  free=(torch.randperm(pool, generator=g, device=DEV) + blocks).to(torch.int32),
                  count=torch.tensor([pool], dtype=torch.int32, device=DEV))
    else:
        pool = 1000
        s |= dict(free=torch.nn.functional.pad((torch.randperm(pool, generator=g, device=DEV) + blocks).to(torch.int32), (0, blocks)),
                  count=torch.tensor([pool], dtype=torch.int32, device=DEV),
                  ended=torch.rand(n, generator=g, device=DEV).argsort() < case["ended"])
    return s


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    make = {"rotary": _prepare_rotary, "append": _prepare_append, "attend": _prepare_attend, "plan": _prepare_plan,
            "release": _prepare_plan}[case["op"]]
    return dict(make(case, g), op=case["op"])


# ---- one pass ----------------------------------------------------------------------------------
def _rotate(x, cos, sin, dim, interleaved):
    x32 = x.float()
    if interleaved:
        a, b = x32[..., 0:dim:2], x32[..., 1:dim:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x32[..., :dim // 2], x32[..., dim // 2:dim]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y.to(x.dtype), x[..., dim:]], -1)


def _run_rotary(s):
    if own:
        from turboquant.kernels.rotary import rotary_embedding
        return rotary_embedding(s["q"], s["k"], s["positions"], s["table"], interleaved=s["interleaved"], inverse=s["inverse"])
    rows = s["table"][s["positions"]][:, None]
    cos, sin = rows[..., :s["dim"] // 2], rows[..., s["dim"] // 2:]
    sin = -sin if s["inverse"] else sin
    return tuple(_rotate(x, cos, sin, s["dim"], s["interleaved"]) for x in (s["q"], s["k"]))


def _run_append(s):
    if own:
        from turboquant.kernels.paged_8bit import quantize_and_scatter
        quantize_and_scatter(s["key"], s["value"], s["cache"], s["slots"], s["block_size"])
        return s["codes"], s["scales"]
    codes, scales, bs = s["codes"].view(torch.uint8), s["scales"], s["block_size"]
    H = codes.shape[1]
    x = torch.stack([s["key"], s["value"]], 2).float()                       # [T, H, 2, D]
    page, at = s["slots"] // PAGE, s["slots"] % PAGE
    first = torch.ones_like(page, dtype=torch.bool)
    first[1:] = page[1:] != page[:-1]
    begin = first.nonzero()[:, 0]                                            # first row of every page that is written
    run = torch.cumsum(first, 0) - 1
    size = x.abs().amax(-1)
    new = _exponent(torch.zeros(len(begin), H, 2, device=x.device).index_reduce_(0, run, size, "amax"))
    b, p, live = page[begin] // (bs // PAGE), page[begin] % (bs // PAGE), at[begin]
    old = _exponent(scales[b, :, p] * E4M3_MAX)
    e = torch.where((live == 0)[:, None, None], new, torch.maximum(old, new))
    kept = _values(codes[b, :, p]).float()                                            # [runs, H, 2, 16, D]
    kept = torch.where((torch.arange(PAGE, device=x.device) < live[:, None])[:, None, None, :, None],
                       torch.ldexp(kept, (old - e)[..., None, None]), kept)
    codes[b, :, p] = kept.to(torch.float8_e4m3fn).view(torch.uint8)
    scales[b, :, p] = torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)
    y = torch.ldexp(x, -e[run][..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    codes[page // (bs // PAGE), :, page % (bs // PAGE), :, at] = y.view(torch.uint8)
    return s["codes"], scales


def _dense(s, dtype):
    """K and V of every sequence, [n, H, longest, D], and the tokens' indices."""
    codes, scales, bs = s["codes"].view(torch.uint8), s["scales"], s["block_size"]
    n, tokens = s["tables"].shape[0], torch.arange(s["longest"], device=s["q"].device)
    b, p, at = s["tables"].to(torch.int64)[:, tokens // bs], tokens % bs // PAGE, tokens % PAGE
    p, at = p.expand(n, -1), at.expand(n, -1)
    kv = _values(codes[b, :, p, :, at]).to(dtype) * scales[b, :, p].to(dtype)[..., None]        # [n, longest, H, 2, D]
    return kv[..., 0, :].transpose(1, 2), kv[..., 1, :].transpose(1, 2), tokens


def _run_attend(s):
    q, lens, start = s["q"], s["lens"], s["start"]
    if own:
        from turboquant.kernels.paged_8bit import paged_attention_8bit
        more = {} if s["most_queries"] == 1 else dict(query_start_loc=start, max_query_len=s["most_queries"])
        return paged_attention_8bit(q, s["cache"], s["tables"], lens, s["block_size"], max_seq_len=s["longest"], **more)
    n, H, dim = len(lens), s["codes"].shape[1], q.shape[-1]
    k, v, tokens = _dense(s, torch.float32)
    count = (start[1:] - start[:-1]).to(torch.int64)
    j = torch.arange(s["most_queries"], device=q.device)
    row = (start[:-1].to(torch.int64)[:, None] + j).clamp(max=len(q) - 1)              # [n, most_queries]
    qs = q[row].float().unflatten(2, (H, -1)).permute(0, 2, 3, 1, 4).flatten(2, 3)     # [n, H, G * most, D]
    limit = lens.to(torch.int64)[:, None] - count[:, None] + j + 1                     # tokens that a row sees
    seen = (tokens < limit[..., None])[:, None, None]
    score = (qs @ k.transpose(-1, -2)).mul_(dim ** -0.5).unflatten(2, (-1, len(j)))
    score.masked_fill_(~seen, -math.inf)
    weight = (score - score.amax(-1, keepdim=True)).exp_()
    out = (weight.flatten(2, 3) @ torch.where((tokens < lens[:, None])[:, None, :, None], v, 0)).unflatten(2, (-1, len(j)))
    out = out / weight.sum(-1, keepdim=True)
    out = out.permute(0, 3, 1, 2, 4).flatten(2, 3)[j < count[:, None]]                  # the rows that are there, in order
    return out.to(q.dtype)


def _run_plan(s):
    if own:
        from turboquant.kernels.block_plan import plan_step
        plan = plan_step(s["query"], s["context"], s["tables"], s["free"], s["count"], s["block_size"], s["rows"])
        return plan.slot_mapping, plan.positions, plan.seq_lens, plan.query_start_loc, plan.free_count, s["tables"]
    ctx, query, bs, count = s["context"].to(torch.int64), s["query"].to(torch.int64), s["block_size"], s["count"].to(torch.int64)
    held, total = (ctx + bs - 1) // bs, (ctx + query + bs - 1) // bs
    wide = total <= s["tables"].shape[1]
    need = torch.where(wide, total - held, 0)
    last = torch.cumsum(need, 0)
    served = wide & ((need == 0) | (last <= count))
    ends = torch.cumsum(query, 0)
    row = torch.arange(s["rows"], device=ctx.device)
    seq = torch.searchsorted(ends, row, right=True)
    pos = ctx[seq] + row - (ends - query)[seq]
    at = pos // bs
    fresh = at >= held[seq]
    block = s["free"][(count - 1 - ((last - need)[seq] + at - held[seq])).clamp(0, len(s["free"]) - 1)]
    block = torch.where(fresh, block, s["tables"][seq, at.clamp(max=s["tables"].shape[1] - 1)])
    keep = (served[seq] & fresh & (pos % bs == 0)).nonzero()[:, 0]
    s["tables"][seq[keep], at[keep]] = block[keep]
    slots = torch.where(served[seq], block.to(torch.int64) * bs + pos % bs, -1)
    start = torch.nn.functional.pad(ends, (1, 0)).to(torch.int32)
    taken = torch.where(served & (need > 0), last, 0).amax()
    return slots, pos, torch.where(served, ctx + query, ctx).to(torch.int32), start, (count - taken).to(torch.int32), s["tables"]


def _run_release(s):
    if own:
        from turboquant.kernels.block_plan import release_blocks
        lens, count = release_blocks(s["ended"], s["context"], s["tables"], s["free"], s["count"], s["block_size"])
        return lens, count, s["free"]
    ctx = s["context"].to(torch.int64)
    held = torch.where(s["ended"], (ctx + s["block_size"] - 1) // s["block_size"], 0)
    col = torch.arange(s["tables"].shape[1], device=ctx.device)
    given = s["tables"][col < held[:, None]]                                            # by request, then by position
    s["free"].index_copy_(0, s["count"].to(torch.int64) + torch.arange(len(given), device=ctx.device), given)
    return torch.where(s["ended"], 0, s["context"]), s["count"] + len(given), s["free"]


def run(state):
    return {"rotary": _run_rotary, "append": _run_append, "attend": _run_attend, "plan": _run_plan, "release": _run_release}[state["op"]](state)


def work(case):
    op = case["op"]
    if op == "rotary":
        values = case["rows"] * (case["q_heads"] + case["kv_heads"])
        return {"bytes": 2 * values * case["head_dim"] * ITEM[case["dtype"]] + case["rows"] * (8 + 4 * case["rotary_dim"]),
                "flops": 3 * values * case["rotary_dim"]}
    if op == "append":
        T = int(_lengths(case["lens"]).sum())
        values = T * case["kv_heads"] * 2 * case["head_dim"]
        return {"bytes": values * (ITEM[case["dtype"]] + 1) + T * 8, "flops": 3 * values}
    if op == "attend":
        query = _lengths(case["queries"])
        ctx = _lengths(case["context"], len(query), salt=9)
        row = case["q_heads"] * case["head_dim"]
        pages = (ctx + query + PAGE - 1) // PAGE
        kv = int((ctx + query).sum()) * 2 * case["head_dim"] + int(pages.sum()) * 8
        return {"bytes": kv * case["kv_heads"] + 2 * int(query.sum()) * row * ITEM[case["dtype"]] + int(pages.sum()) * 4,
                "flops": 4 * row * int((query * ctx + query * (query + 1) // 2).sum())}
    ctx = _lengths(case["context"], salt=9)
    if op == "plan":
        query = _lengths(case["queries"])
        new = int(((ctx + query + case["block_size"] - 1) // case["block_size"] - (ctx + case["block_size"] - 1) // case["block_size"]).sum())
        return {"bytes": len(ctx) * 16 + int(query.sum()) * 16 + new * 8, "flops": 10 * int(query.sum())}
    share = case["ended"] / len(ctx)
    return {"bytes": int(len(ctx) * 9 + share * float(ctx.sum()) / case["block_size"] * 8), "flops": 4 * len(ctx)}


# ---- the definition in 64 bits ------------------------------------------------------------------
def _e4m3(x):
    """fp64 values rounded to the nearest value of e4m3, ties to even, saturating at 448."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))).clamp(min=-6) - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def _exact_rotary(case, s):
    f, factor = _inverse_frequencies(case["rotary_dim"], case["scaling"])
    angle = (s["positions"].double()[:, None] * f.to(DEV))[:, None]
    turn = torch.polar(torch.full_like(angle, factor), -angle if case["inverse"] else angle)
    out = []
    for x in (s["q"].double(), s["k"].double()):
        r = x[..., :case["rotary_dim"]]
        pairs = r.unflatten(-1, (-1, 2)) if case["interleaved"] else r.unflatten(-1, (2, -1)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        z = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
        out.append(torch.cat([z, x[..., case["rotary_dim"]:]], -1))
    return tuple(out)


def _exact_append(case, s):
    codes, scales, bs = s["codes"].double(), s["scales"].double(), s["block_size"]
    x = torch.stack([s["key"], s["value"]], 2).double()
    slots = s["slots"].tolist()
    runs = []
    for i, t in enumerate(slots):
        if i and t == slots[i - 1] + 1 and t % PAGE:
            runs[-1][1] = i + 1
        else:
            runs.append([i, i + 1])
    for a, b in runs:
        block, page, at = slots[a] // bs, slots[a] % bs // PAGE, slots[a] % PAGE
        # 1e-12: log2 of a power of two may come out a last bit too large; inputs of 11 bits are never that close to one
        e = torch.ceil(torch.log2((x[a:b].abs().amax((0, -1)) / E4M3_MAX).clamp(min=2.0 ** MIN_EXPONENT)) - 1e-12)     # [H, 2]
        if at:
            before = scales[block, :, page]
            e = torch.maximum(e, torch.log2(before.clamp(min=2.0 ** MIN_EXPONENT)))
            codes[block, :, page, :, :at] = _e4m3(codes[block, :, page, :, :at] * (before / torch.exp2(e))[..., None, None])
        scales[block, :, page] = torch.exp2(e)
        codes[block, :, page, :, at:at + b - a] = _e4m3(x[a:b] / torch.exp2(e)[..., None]).permute(1, 2, 0, 3)
    return codes, scales


def _exact_attend(case, s):
    codes, scales, bs, out = s["codes"].view(torch.uint8), s["scales"], s["block_size"], []
    H, G, dim = case["kv_heads"], case["q_heads"] // case["kv_heads"], case["head_dim"]
    lens, start = s["lens"].tolist(), s["start"].tolist()
    for i, L in enumerate(lens):
        a, b = start[i], start[i + 1]
        blocks = s["tables"][i, :-(-L // bs)].long()
        kv = (_values(codes[blocks]).double() * scales[blocks].double()[..., None, None]).permute(3, 1, 0, 2, 4, 5).reshape(2, H, -1, dim)[:, :, :L]
        for h in range(H):
            q = s["q"][a:b, h * G:(h + 1) * G].double()
            score = torch.einsum("jgd,kd->jgk", q, kv[0, h]) / math.sqrt(dim)
            hidden = torch.arange(L, device=DEV) > torch.arange(L - (b - a), L, device=DEV)[:, None]
            out.append(torch.softmax(score.masked_fill_(hidden[:, None], -math.inf), -1) @ kv[1, h])
    rows = [torch.cat(out[i * H:(i + 1) * H], 1) for i in range(len(lens))]
    return torch.cat(rows)


def exact(case, seed):
    if case["op"] in ("plan", "release"):
        return None                                                    # whole numbers, no roundings
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(case, s)
    if case["op"] == "append":
        runs = sum(-(-int(q) // PAGE) + 1 for q in _lengths(case["lens"]))
        return _exact_append(case, s) if runs < 10000 and s["codes"].numel() < 1 << 29 else None
    if len(s["lens"]) * case["kv_heads"] > 2100:
        return None
    return _exact_attend(case, s)
