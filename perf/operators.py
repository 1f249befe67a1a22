"""The attention step between two quantized projections, over a cache held in 4 bits: cases, plain forms, exact values.

Four operators of pfng_b200 that a serving step calls one after the other:

  kv_plan          block table, slot map, positions and lengths of a step from the requests' lengths
  qk_norm_rope     RMS norm of every query and key head and the position rotation, in one pass
  kv_append_q4_0   keys and values quantized to q4_0 into the pages of the cache
  attention_q4_0   attention over the q4_0 cache: single tokens, a few tokens, prompts and chunks of prompts

`own` chooses between the plain forms (elementary torch operations in 32 bits) and the library's kernels.

The cache: K and V are uint8 buffers of [pages][heads_kv][page_size / 16] groups.  A group holds 16 tokens of one head:
16 rows of D / 2 bytes of nibbles, then 16 rows of D / 32 fp16 scales.  Byte i (0..15) of a q4_0 block holds value i in
its low and value i + 16 in its high nibble; a value is scale * (nibble - 8).  The bytes of a token's D / 32 blocks are
interleaved: byte 4 t + e of block b stands at t * (D / 8) + 4 b + e in a K row, byte 2 g + e of block b at
g * (D / 16) + 2 b + e in a V row.
"""
import math
import pathlib
import sys

import torch

own = False
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # four chats that each take one token: the call is a few hundred bytes, latency is all of it
        {"name": "plan-step-4", "op": "plan", "requests": 4, "max_kv": 900, "max_q": 1, "page": 16},
        # a full scheduler step: 1000 requests, single tokens and prompt chunks mixed
        {"name": "plan-step-1000", "op": "plan", "requests": 1000, "max_kv": 16000, "max_q": 160, "page": 64},
        # one decode token of a 4096-wide layer with 32 heads, straight from the fp32 projection
        {"name": "rope-decode-1", "op": "rope", "tokens": 1, "heads_q": 32, "heads_k": 32, "dim": 128, "rot": 128,
         "interleaved": False, "norm": False, "fmt_in": "f32", "fmt_out": "bf16"},
        # a prompt step with grouped heads, bf16 throughout
        {"name": "rope-prompt-8192", "op": "rope", "tokens": 8192, "heads_q": 32, "heads_k": 8, "dim": 128, "rot": 128,
         "interleaved": False, "norm": True, "fmt_in": "bf16", "fmt_out": "bf16"},
        # a decode step's keys and values: 64 requests, one row each, scattered over the pages
        {"name": "append-decode-64", "op": "append", "tokens": 64, "heads_kv": 8, "dim": 128, "page": 16, "run": 1,
         "fmt_k": "bf16", "fmt_v": "f32"},
        # a prompt step's keys and values: long runs of slots
        {"name": "append-prompt-16384", "op": "append", "tokens": 16384, "heads_kv": 8, "dim": 128, "page": 64,
         "run": 1024, "fmt_k": "bf16", "fmt_v": "bf16"},
        # one chat, one token, a short odd context, a head of keys for every head of queries
        {"name": "attn-decode-1x777", "op": "attn", "requests": 1, "min_kv": 777, "max_kv": 777, "min_q": 1,
         "max_q": 1, "heads_q": 32, "heads_kv": 32, "dim": 128, "page": 16, "window": 0, "fmt": "bf16"},
        # a server's decode step: 48 requests of very different lengths, grouped heads
        {"name": "attn-decode-48x8000", "op": "attn", "requests": 48, "min_kv": 64, "max_kv": 8000, "min_q": 1,
         "max_q": 1, "heads_q": 32, "heads_kv": 8, "dim": 128, "page": 64, "window": 0, "fmt": "bf16"},
        # few requests with very long contexts
        {"name": "attn-decode-8x100000", "op": "attn", "requests": 8, "min_kv": 60000, "max_kv": 100000, "min_q": 1,
         "max_q": 1, "heads_q": 32, "heads_kv": 8, "dim": 128, "page": 64, "window": 0, "fmt": "bf16"},
        # a few tokens a request (drafted tokens being checked), small heads, fp16
        {"name": "attn-draft-16x5000", "op": "attn", "requests": 16, "min_kv": 500, "max_kv": 5000, "min_q": 1,
         "max_q": 4, "heads_q": 16, "heads_kv": 4, "dim": 64, "page": 32, "window": 0, "fmt": "f16"},
        # chunks of prompts on top of what is cached, ragged, a sliding window
        {"name": "attn-chunk-5x1400", "op": "attn", "requests": 5, "min_kv": 1500, "max_kv": 7000, "min_q": 300,
         "max_q": 1400, "heads_q": 32, "heads_kv": 8, "dim": 128, "page": 16, "window": 4096, "fmt": "bf16"},
        # one whole prompt
        {"name": "attn-prompt-8192", "op": "attn", "requests": 1, "min_kv": 8192, "max_kv": 8192, "min_q": 8192,
         "max_q": 8192, "heads_q": 32, "heads_kv": 8, "dim": 128, "page": 64, "window": 0, "fmt": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["plan", "rope", "append", "attn", "attn", "attn"])
    page = rng.choice([16, 32, 64, 128])
    if op == "plan":
        return {"op": op, "requests": _log(rng, 1, 1000), "max_kv": _log(rng, 1, 16000), "max_q": _log(rng, 1, 160),
                "page": page}
    dim = rng.choice([64, 128, 128])
    if op == "rope":
        heads_k = rng.choice([1, 2, 4, 8])
        return {"op": op, "tokens": _log(rng, 1, 8192), "heads_q": heads_k * rng.choice([1, 3, 4]), "heads_k": heads_k,
                "dim": dim, "rot": rng.choice([dim, dim // 2]), "interleaved": rng.random() < 0.3,
                "norm": rng.random() < 0.7, "fmt_in": rng.choice(["f32", "f16", "bf16"]),
                "fmt_out": rng.choice(["f32", "f16", "bf16"])}
    if op == "append":
        tokens = _log(rng, 1, 16384)
        return {"op": op, "tokens": tokens, "heads_kv": rng.choice([1, 2, 4, 8]), "dim": dim, "page": page,
                "run": rng.choice([1, min(tokens, 37), tokens]), "fmt_k": rng.choice(["f32", "f16", "bf16"]),
                "fmt_v": rng.choice(["f32", "f16", "bf16"])}
    heads_kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 3, 4, 4])
    kind = rng.choice(["decode", "decode", "draft", "chunk"])
    case = {"op": op, "heads_q": heads_kv * group, "heads_kv": heads_kv, "dim": dim, "page": page,
            "window": rng.choice([0, 0, 0, _log(rng, 100, 4096)])}
    if kind == "chunk":
        max_q = _log(rng, 20, 4000)
        max_kv = _log(rng, max_q, 16000)
        fit = max(1, 30_000_000 // (max_q * max_kv))
        return {**case, "requests": _log(rng, 1, min(8, fit)), "min_kv": 1 + max_kv // 4, "max_kv": max_kv,
                "min_q": 1 + max_q // 4, "max_q": max_q, "fmt": "bf16"}
    max_kv = _log(rng, 1, 100000)
    most = max(1, 700_000 // max_kv)
    return {**case, "requests": _log(rng, 1, min(64, most)), "min_kv": 1 + max_kv // 3, "max_kv": max_kv, "min_q": 1,
            "max_q": 1 if kind == "decode" else min(max_kv, rng.choice([2, 3, 4])),
            "fmt": rng.choice(["bf16", "f16"]) if kind == "decode" else "bf16"}


# ------------------------------------------------------------------------------------------------ inputs
def _ints(gen, lo, hi, n):
    """n whole numbers of lo..hi, the largest of them among them."""
    v = torch.randint(lo, hi + 1, (n,), generator=gen)
    v[int(torch.randint(0, n, (1,), generator=gen))] = hi
    return v


def _lengths(case):
    """kv (cached and new) and q lengths of an attention case.  They belong to the case: every seed has the same work."""
    gen = torch.Generator().manual_seed(case["requests"] * 1000003 + case["max_kv"] * 101 + case["max_q"])
    seq = _ints(gen, case["min_kv"], case["max_kv"], case["requests"])
    q = torch.minimum(_ints(gen, case["min_q"], case["max_q"], case["requests"]), seq)
    return seq, q


def _plan_lengths(case):
    gen = torch.Generator().manual_seed(case["requests"] * 7919 + case["max_kv"])
    kv = _ints(gen, 0, case["max_kv"], case["requests"])
    q = _ints(gen, 1, case["max_q"], case["requests"])
    return kv, torch.where(torch.rand(case["requests"], generator=gen) < 0.5, torch.ones_like(q), q)


def _quantize(x):
    """q4_0 of x [..., D] in 32 bits: (nibbles [..., D / 32, 32], scales fp16 [..., D / 32])."""
    x = x.float().unflatten(-1, (-1, 32))
    size = x.abs()
    top = size.amax(-1, keepdim=True)
    at = torch.arange(32, device=x.device).expand_as(x)
    first = torch.where(size == top, at, 32).amin(-1, keepdim=True)
    d = x.gather(-1, first) / -8.0
    inv = torch.where(d != 0, 1.0 / d, torch.zeros_like(d))
    n = torch.clamp((x * inv + 8.5).to(torch.int32), max=15)
    return n, d.squeeze(-1).to(torch.float16)


def _rows(n, is_k):
    """The bytes of a cache row from the nibbles [..., blocks, 32] of one token."""
    b = n[..., :16] | (n[..., 16:] << 4)
    b = b.unflatten(-1, (4, 4) if is_k else (8, 2))  # [..., block, t, e]
    return b.transpose(-3, -2).flatten(-3).to(torch.uint8)


def _parts(cache, pages, heads, page, dim):
    """Views of a cache's nibble rows [pages, heads, page / 16, 16, dim / 2] and scale bytes [..., 16, dim / 16]."""
    c = cache.view(pages, heads, page // 16, 16 * (dim // 2 + dim // 16))
    return c[..., :8 * dim].unflatten(-1, (16, dim // 2)), c[..., 8 * dim:].unflatten(-1, (16, dim // 16))


def _write(cache, x, is_k, page_ids, offsets, pages, page):
    """Rows x [tokens, heads, dim] quantized into the cache at (page, offset)."""
    nib, sc = _parts(cache, pages, x.shape[1], page, x.shape[2])
    n, d = _quantize(x)
    nib[page_ids, :, offsets // 16, offsets % 16] = _rows(n, is_k)
    sc[page_ids, :, offsets // 16, offsets % 16] = d.view(torch.uint8)


def _cache_bytes(pages, heads, page, dim):
    return pages * heads * page * (dim // 2 + dim // 16)


def _filled_cache(gen, pages, heads, page, dim, is_k, spread):
    """A cache whose every slot holds a quantized row, as a server's does after a while."""
    cache = torch.empty(_cache_bytes(pages, heads, page, dim), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 26) // (heads * page * dim))
    nib, sc = _parts(cache, pages, heads, page, dim)
    for p in range(0, pages, step):
        count = min(step, pages - p)
        x = torch.randn(count, heads, page // 16, 16, dim, generator=gen, device="cuda") * spread
        n, d = _quantize(x)
        nib[p:p + count] = _rows(n, is_k)
        sc[p:p + count] = d.view(torch.uint8)
    return cache


def _library():
    root = pathlib.Path(__file__).resolve().parent.parent
    path = str(root / "qgemm-perf-framework-ng_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import pfng_b200
    return pfng_b200


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    s = dict(case)
    page = case.get("page")
    if case["op"] == "plan":
        kv, q = _plan_lengths(case)
        have, need = (kv + page - 1) // page, (kv + q + page - 1) // page
        used, new = int(have.sum()), int((need - have).sum())
        ids = torch.randperm(used + new + 7, generator=cpu).to(torch.int32)
        s["max_pages"] = int(need.max()) + 3
        table = torch.full((case["requests"], s["max_pages"]), -1, dtype=torch.int32)
        owned = torch.arange(s["max_pages"])[None] < have[:, None]
        table[owned] = ids[:used]
        s["tokens"] = int(q.sum())
        s["table"], s["free"] = table.cuda(), ids[used:].cuda()
        s["kv_len"], s["q_len"] = kv.to(torch.int32).cuda(), q.to(torch.int32).cuda()
    elif case["op"] == "rope":
        heads = case["heads_q"] + 2 * case["heads_k"]  # the row of a Q/K/V projection; the values are not touched
        x = torch.randn(case["tokens"], heads * case["dim"], generator=gen, device="cuda") * 1.3
        s["x"] = x.to(DTYPES[case["fmt_in"]])
        positions = 16384
        inv = 10000.0 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64) / case["rot"])
        angle = torch.arange(positions, dtype=torch.float64)[:, None] * inv
        s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).float().cuda()
        first = int(torch.randint(0, positions - case["tokens"], (1,), generator=cpu))
        s["positions"] = torch.arange(first, first + case["tokens"], dtype=torch.int32, device="cuda")
        s["wq"] = s["wk"] = None
        if case["norm"]:
            s["wq"] = 1 + 0.2 * torch.randn(case["dim"], generator=gen, device="cuda")
            s["wk"] = 1 + 0.2 * torch.randn(case["dim"], generator=gen, device="cuda")
    elif case["op"] == "append":
        width = case["heads_kv"] * case["dim"]
        for name in ("k", "v"):
            x = torch.randn(case["tokens"], width, generator=gen, device="cuda")
            s[name] = x.to(DTYPES[case["fmt_" + name]])
        # runs of consecutive slots, each on pages of its own, the pages in no order
        runs = -(-case["tokens"] // case["run"])
        each = -(-case["run"] // page) + 1
        s["pages"] = runs * each + 3
        ids = torch.randperm(s["pages"], generator=cpu)
        token = torch.arange(case["tokens"])
        run, at = token // case["run"], token % case["run"] + torch.randint(0, page, (runs,), generator=cpu)[token // case["run"]]
        s["slots"] = (ids[run * each + at // page] * page + at % page).cuda()
        size = _cache_bytes(s["pages"], case["heads_kv"], page, case["dim"])
        s["k_cache"] = torch.zeros(size, dtype=torch.uint8, device="cuda")
        s["v_cache"] = torch.zeros(size, dtype=torch.uint8, device="cuda")
    else:
        seq, q = _lengths(case)
        need = (seq + page - 1) // page
        s["pages"] = int(need.sum()) + 2
        s["max_pages"] = int(need.max())
        ids = torch.randperm(s["pages"], generator=cpu).to(torch.int32)
        table = torch.full((case["requests"], s["max_pages"]), -1, dtype=torch.int32)
        owned = torch.arange(s["max_pages"])[None] < need[:, None]
        table[owned] = ids[:int(need.sum())]
        s["table"] = table.cuda()
        s["seq_len"] = seq.to(torch.int32).cuda()
        s["cu_q"] = torch.cat([torch.zeros(1, dtype=torch.int64), q.cumsum(0)]).to(torch.int32).cuda()
        s["tokens"], s["max_q_len"], s["max_seq_len"] = int(q.sum()), int(q.max()), int(seq.max())
        s["q"] = (torch.randn(s["tokens"], case["heads_q"] * case["dim"], generator=gen, device="cuda") * 1.5).to(
            DTYPES[case["fmt"]])
        s["k_cache"] = _filled_cache(gen, s["pages"], case["heads_kv"], page, case["dim"], True, 1.0)
        s["v_cache"] = _filled_cache(gen, s["pages"], case["heads_kv"], page, case["dim"], False, 0.7)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_plan(s):
    page = s["page"]
    kv, q, table = s["kv_len"], s["q_len"], s["table"]
    seq = kv + q
    have, need = (kv + page - 1) // page, (seq + page - 1) // page
    taken = (need - have).cumsum(0)
    first = taken - (need - have)
    col = torch.arange(s["max_pages"], device="cuda", dtype=torch.int32)[None]
    is_new = (col >= have[:, None]) & (col < need[:, None])
    at = (first[:, None] + col - have[:, None]).clamp(0, s["free"].numel() - 1)
    table.copy_(torch.where(is_new, s["free"][at.long()], table))
    ends = q.cumsum(0)
    cu_q = torch.cat([torch.zeros_like(ends[:1]), ends]).to(torch.int32)
    token = torch.arange(s["tokens"], device="cuda")
    r = torch.searchsorted(ends, token, right=True)
    pos = kv[r] + (token - cu_q[r])
    slots = table[r, (pos // page).long()].long() * page + pos % page
    counts = torch.stack([ends[-1], taken[-1], torch.zeros_like(ends[-1])]).to(torch.int32)
    return {"table": table, "seq_len": seq, "cu_q": cu_q, "positions": pos.to(torch.int32), "slots": slots,
            "counts": counts}


def _plain_rope(s):
    dim, rot, heads_q, heads_k = s["dim"], s["rot"], s["heads_q"], s["heads_k"]
    cs = s["cos_sin"][s["positions"].long()][:, None]
    cos, sin = cs[..., :rot // 2], cs[..., rot // 2:]

    def part(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        turn, rest = x[..., :rot], x[..., rot:]
        if s["interleaved"]:
            a, b = turn[..., 0::2], turn[..., 1::2]
            turn = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = turn[..., :rot // 2], turn[..., rot // 2:]
            turn = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([turn, rest], -1).flatten(-2).to(DTYPES[s["fmt_out"]])

    x = s["x"].unflatten(-1, (-1, dim))
    return {"q": part(x[:, :heads_q], s["wq"]), "k": part(x[:, heads_q:heads_q + heads_k], s["wk"])}


def _plain_append(s):
    page = s["page"]
    pages, offsets = s["slots"] // page, s["slots"] % page
    for name in ("k", "v"):
        x = s[name].unflatten(-1, (s["heads_kv"], s["dim"]))
        _write(s[name + "_cache"], x, name == "k", pages, offsets, s["pages"], page)
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _gathered(s, cache, is_k, table):
    """The rows of every request's pages in 32 bits: [requests, heads_kv, padded length, dim]."""
    dim = s["dim"]
    nib, sc = _parts(cache, s["pages"], s["heads_kv"], s["page"], dim)
    nib = nib[table].unflatten(-1, (4, dim // 32, 4) if is_k else (8, dim // 32, 2))  # [R, NP, H, G, 16, t, block, e]
    n = torch.stack([nib & 15, nib >> 4], -4).permute(0, 2, 1, 3, 4, 7, 5, 6, 8)  # [R, H, NP, G, 16, block, half, t, e]
    d = sc[table].contiguous().view(torch.float16).permute(0, 2, 1, 3, 4, 5)
    x = (n.flatten(-3).float() - 8.0) * d.float().unsqueeze(-1)
    return x.flatten(-2).flatten(2, 4)


def _plain_attn(s):
    dim, hk, page = s["dim"], s["heads_kv"], s["page"]
    group = s["heads_q"] // hk
    r_count, mq = s["requests"], s["max_q_len"]
    table = s["table"].clamp(min=0).long()
    k, v = _gathered(s, s["k_cache"], True, table), _gathered(s, s["v_cache"], False, table)
    length = k.shape[2]
    cu = s["cu_q"].long()
    q_len = cu[1:] - cu[:-1]
    i = torch.arange(mq, device="cuda")
    rows = (cu[:-1, None] + i).clamp(max=s["tokens"] - 1)
    q = s["q"].float()[rows].unflatten(-1, (hk, group, dim)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    score = torch.matmul(q, k.transpose(-1, -2)).mul_(dim ** -0.5).unflatten(2, (group, mq))
    pos = (s["seq_len"].long() - q_len)[:, None] + i
    j = torch.arange(length, device="cuda")
    seen = (j <= pos[..., None]) & (j < s["seq_len"].long()[:, None, None])
    if s["window"]:
        seen &= j > pos[..., None] - s["window"]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = score.sum(-1, keepdim=True)
    o = torch.matmul(score.flatten(2, 3), v).unflatten(2, (group, mq))
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    token = torch.arange(s["tokens"], device="cuda")
    r = torch.searchsorted(cu[1:].contiguous(), token, right=True)
    o = o.permute(0, 3, 1, 2, 4)[r, token - cu[r]]
    return {"out": o.flatten(1).to(DTYPES[s["fmt"]])}


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    if not own:
        return {"plan": _plain_plan, "rope": _plain_rope, "append": _plain_append, "attn": _plain_attn}[s["op"]](s)
    pb = _library()
    if s["op"] == "plan":
        p = pb.kv_plan(s["kv_len"], s["q_len"], s["table"], s["free"], s["page"], s["tokens"])
        return {"table": s["table"], "seq_len": p.seq_len, "cu_q": p.cu_q, "positions": p.positions, "slots": p.slots,
                "counts": p.counts}
    if s["op"] == "rope":
        q, k = pb.qk_norm_rope(s["x"], s["positions"], s["cos_sin"], s["heads_q"], s["heads_k"], s["dim"],
                               q_weight=s["wq"], k_weight=s["wk"], eps=EPS, interleaved=s["interleaved"],
                               out_format=s["fmt_out"])
        return {"q": q, "k": k}
    if s["op"] == "append":
        pb.kv_append_q4_0(s["k"], s["v"], s["slots"], s["k_cache"], s["v_cache"], s["heads_kv"], s["dim"], s["page"])
        return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    out = pb.attention_q4_0(s["q"], s["k_cache"], s["v_cache"], s["table"], s["seq_len"], s["cu_q"], s["heads_q"],
                            s["heads_kv"], s["dim"], s["page"], max_q=s["max_q_len"], max_kv=s["max_seq_len"],
                            causal=True, window=s["window"], out_format=s["fmt"])
    return {"out": out}


# ------------------------------------------------------------------------------------------------ least work
def _size(fmt):
    return 4 if fmt == "f32" else 2


def work(case):
    if case["op"] == "plan":
        kv, q = _plan_lengths(case)
        page = case["page"]
        new = int(((kv + q + page - 1) // page - (kv + page - 1) // page).sum())
        tokens, r = int(q.sum()), case["requests"]
        touched = int(((kv + page - 1) // page > kv // page).sum())  # requests whose last page has room left
        return {"bytes": 8 * r + 4 * touched + 8 * new + 4 * r + 4 * (r + 1) + 12 * tokens + 12, "flops": 6 * tokens}
    if case["op"] == "rope":
        heads = case["heads_q"] + case["heads_k"]
        values = case["tokens"] * heads * case["dim"]
        io = values * (_size(case["fmt_in"]) + _size(case["fmt_out"]))
        return {"bytes": io + case["tokens"] * (4 + 4 * case["rot"]) + 8 * case["dim"] * case["norm"],
                "flops": values * (4 * case["norm"] + 3)}
    if case["op"] == "append":
        values = case["tokens"] * case["heads_kv"] * case["dim"]
        return {"bytes": values * (_size(case["fmt_k"]) + _size(case["fmt_v"])) + 2 * values * 18 // 32
                + 8 * case["tokens"], "flops": 8 * values}
    seq, q = _lengths(case)
    keys = pairs = 0
    for n, m in zip(seq.tolist(), q.tolist()):
        w = case["window"] or n
        keys += min(n, w + m - 1)
        first = n - m  # the position of the first new token
        full = max(0, min(m, n - max(first, w - 1)))  # rows that see a whole window
        lo = m - full  # rows first .. first + lo - 1 see position + 1 keys
        pairs += full * w + lo * (first + 1) + lo * (lo - 1) // 2
    tokens = int(q.sum())
    row = case["heads_kv"] * case["dim"] * 18 // 32
    return {"bytes": 2 * keys * row + 2 * tokens * case["heads_q"] * case["dim"] * _size(case["fmt"])
            + 4 * sum(-(-int(n) // case["page"]) for n in seq) + 8 * case["requests"],
            "flops": 4 * pairs * case["heads_q"] * case["dim"]}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_rows(s, cache, is_k, pages):
    """Rows of one request in 64 bits, from the bytes: [heads_kv, length of its pages, dim]."""
    dim, blocks = s["dim"], s["dim"] // 32
    raw = cache.view(s["pages"], s["heads_kv"], s["page"] // 16, -1)[pages].transpose(0, 1)  # [H, NP, G, bytes]
    nib = raw[..., :8 * dim].reshape(*raw.shape[:3], 16, dim // 2)
    sc = raw[..., 8 * dim:].contiguous().view(torch.float16).reshape(*raw.shape[:3], 16, blocks).double()
    at = torch.arange(dim, device=cache.device)
    block, i = at // 32, at % 16
    if is_k:
        byte = (i // 4) * (4 * blocks) + 4 * block + i % 4
    else:
        byte = (i // 2) * (2 * blocks) + 2 * block + i % 2
    n = (nib[..., byte].int() >> torch.where(at % 32 < 16, 0, 4).int()) & 15
    return ((n.double() - 8) * sc[..., block]).flatten(1, 3)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return None
    if case["op"] == "append":  # bytes: they have to be equal
        return None
    if case["op"] == "rope":
        dim, rot = case["dim"], case["rot"]
        half = rot // 2
        x = s["x"].double().reshape(case["tokens"], -1, dim)
        cs = s["cos_sin"].double()[s["positions"].long()]
        c, z = cs[:, None, :half], cs[:, None, half:]
        lo = torch.arange(half, device="cuda") * (2 if case["interleaved"] else 1)
        hi = lo + 1 if case["interleaved"] else lo + half
        found = {}
        for name, a, b, w in (("q", 0, case["heads_q"], s["wq"]),
                              ("k", case["heads_q"], case["heads_q"] + case["heads_k"], s["wk"])):
            y = x[:, a:b].clone()
            if w is not None:
                y = y / (y.pow(2).sum(-1, keepdim=True) / dim + EPS).sqrt() * w.double()
            out = y.clone()
            out[..., lo] = y[..., lo] * c - y[..., hi] * z
            out[..., hi] = y[..., lo] * z + y[..., hi] * c
            found[name] = out.flatten(1)
        return found
    dim, group = case["dim"], case["heads_q"] // case["heads_kv"]
    out = torch.zeros(s["tokens"], case["heads_q"], dim, dtype=torch.float64, device="cuda")
    seq, q_len = _lengths(case)
    start = 0
    for r, (n, m) in enumerate(zip(seq.tolist(), q_len.tolist())):
        pages = s["table"][r, :-(-n // case["page"])].long()
        k = _exact_rows(s, s["k_cache"], True, pages)[:, :n]
        v = _exact_rows(s, s["v_cache"], False, pages)[:, :n]
        for first in range(0, m, 512):
            last = min(m, first + 512)
            q = s["q"][start + first:start + last].double().reshape(last - first, case["heads_kv"], group, dim)
            a = torch.einsum("ihgd,hjd->hgij", q, k) / math.sqrt(dim)
            pos = torch.arange(n - m + first, n - m + last, device="cuda")[:, None]
            j = torch.arange(n, device="cuda")[None]
            hidden = j > pos
            if case["window"]:
                hidden = hidden | (j <= pos - case["window"])
            p = torch.softmax(a.masked_fill(hidden, -math.inf), -1)
            out[start + first:start + last] = torch.einsum("hgij,hjd->ihgd", p, v).flatten(1, 2)
        start += m
    return {"out": out.flatten(1)}
