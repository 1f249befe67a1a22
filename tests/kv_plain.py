"""Plain 64-bit forms of the attention step's operators (test infrastructure), written from include/pfng_b200.h.

A cache is handled here as values [pages][heads_kv][page_size][D] (float64) or as block_q4_0 fields; pack() and
unpack() are the only places that know the byte layout.
"""
import math

import torch


def row_positions(dim: int, is_k: bool) -> torch.Tensor:
    """Position in a row's bytes of byte i of block b: [blocks][16]."""
    blocks = dim // 32
    b, i = torch.arange(blocks)[:, None], torch.arange(16)[None]
    if is_k:
        return (i // 4) * 4 * blocks + 4 * b + i % 4
    return (i // 2) * 2 * blocks + 2 * b + i % 2


def unpack(cache, pages, page, heads, dim, is_k):
    """(nibbles int [pages][heads][page][D / 32][32], scales float16 [...][D / 32]) of a cache's bytes."""
    raw = cache.cpu().reshape(pages, heads, page // 16, 9 * dim)
    rows = raw[..., :8 * dim].reshape(pages, heads, page, dim // 2)
    scales = raw[..., 8 * dim:].contiguous().view(torch.float16).reshape(pages, heads, page, dim // 32)
    by = rows[..., row_positions(dim, is_k).reshape(-1)].reshape(pages, heads, page, dim // 32, 16).to(torch.int32)
    return torch.cat([by & 15, by >> 4], -1), scales


def pack(nibbles, scales, is_k):
    """The inverse of unpack: uint8 bytes."""
    pages, heads, page, blocks, _ = nibbles.shape
    dim = 32 * blocks
    by = (nibbles[..., :16] | (nibbles[..., 16:] << 4)).to(torch.uint8).reshape(pages, heads, page, -1)
    rows = torch.empty(pages, heads, page, dim // 2, dtype=torch.uint8)
    rows[..., row_positions(dim, is_k).reshape(-1)] = by
    raw = torch.empty(pages, heads, page // 16, 9 * dim, dtype=torch.uint8)
    raw[..., :8 * dim] = rows.reshape(pages, heads, page // 16, 8 * dim)
    raw[..., 8 * dim:] = scales.contiguous().view(torch.uint8).reshape(pages, heads, page // 16, dim)
    return raw.reshape(-1)


def values(cache, pages, page, heads, dim, is_k):
    """float64 [pages][heads][page][D]."""
    n, d = unpack(cache, pages, page, heads, dim, is_k)
    return ((n.double() - 8) * d.double()[..., None]).flatten(-2)


def plan(kv_len, q_len, table, free, page, max_tokens):
    """kv_plan with Python numbers; table is a list of lists, changed in place."""
    seq, cu, positions, slots = [], [0], [], []
    taken = lost = 0
    for r, (kv, q) in enumerate(zip(kv_len, q_len)):
        kv, q = max(kv, 0), max(q, 0)
        have, need = -(-kv // page), -(-(kv + q) // page)
        for at in range(have, need):
            if at < len(table[r]) and cu[-1] + at * page - kv < max_tokens:
                table[r][at] = free[taken + at - have] if taken + at - have < len(free) else -1
        got = min(have + max(0, min(len(free) - taken, need - have)), len(table[r]))
        lost += min(q, max(0, kv + q - got * page))
        for i in range(q):
            at, pos = (kv + i) // page, kv + i
            entry = table[r][at] if at < len(table[r]) and len(positions) < max_tokens else -1
            if at >= have and taken + at - have >= len(free):
                entry = -1
            if len(positions) < max_tokens:
                positions.append(pos)
                slots.append(-1 if entry < 0 else entry * page + pos % page)
        taken += need - have
        seq.append(kv + q)
        cu.append(cu[-1] + q)
    positions += [-1] * (max_tokens - len(positions))
    slots += [-1] * (max_tokens - len(slots))
    return seq, cu, positions, slots, [cu[-1], taken, lost]


def norm_rope(x, weight, eps, positions, cos_sin, rot, interleaved):
    """x [tokens][heads][D] in float64 -> (y, |a| + |b| of each value's pair, for error bounds)."""
    y = x.double()
    if weight is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    cs = cos_sin.double()[positions.long()][:, None]
    c, s = cs[..., :rot // 2], cs[..., rot // 2:]
    out, size = y.clone(), y.abs()
    lo = torch.arange(rot // 2) * (2 if interleaved else 1)
    hi = lo + (1 if interleaved else rot // 2)
    a, b = y[..., lo], y[..., hi]
    out[..., lo], out[..., hi] = a * c - b * s, b * c + a * s
    size[..., lo] = size[..., hi] = a.abs() + b.abs()
    return out, size


def attention(q, k, v, table, seq_len, cu_q, page, scale, causal, window):
    """q [tokens][heads][D] float64; k, v [pages][heads_kv][page][D] float64.  Returns (out, lse, spread, reach): spread is
    sum_j p_j |v_j|, reach max_j scale sum_i |q_i k_ji|, the quantities that operand roundings scale with."""
    tokens, heads, dim = q.shape
    pages, heads_kv = k.shape[0], k.shape[1]
    out, spread = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full((tokens, heads), -math.inf, dtype=torch.float64)
    reach = torch.zeros(tokens, heads, dtype=torch.float64)
    for r in range(len(seq_len)):
        n = max(0, min(seq_len[r], len(table[r]) * page))
        m = cu_q[r + 1] - cu_q[r]
        ids = [table[r][j // page] for j in range(n)]
        held = torch.tensor([0 <= p < pages for p in ids], dtype=torch.bool)
        at = torch.tensor([p if 0 <= p < pages else 0 for p in ids], dtype=torch.long)
        off = torch.arange(n) % page
        kr, vr = k[at, :, off].transpose(0, 1), v[at, :, off].transpose(0, 1)  # [heads_kv][n][D]
        for i in range(m):
            row, pos = cu_q[r] + i, n - m + i
            j = torch.arange(n)
            seen = held & (j <= pos) if causal else held
            if window:
                seen = seen & (j > pos - window)
            if not bool(seen.any()):
                continue
            for h in range(heads):
                g = h // (heads // heads_kv)
                ks, vs = kr[g][seen], vr[g][seen]
                s = scale * (ks @ q[row, h])
                p = torch.softmax(s, 0)
                out[row, h], spread[row, h] = p @ vs, p @ vs.abs()
                lse[row, h] = torch.logsumexp(s, 0)
                reach[row, h] = (scale * (ks.abs() @ q[row, h].abs())).max()
    return out, lse, spread, reach


def attention_tolerance(out, spread, reach, out_format, operand_bits):
    """Elementwise bound on a kernel's error: the output's own rounding; probabilities and values rounded to
    `operand_bits` bits each (relative 2^-bits) move a sum of p v by at most that share of sum p |v|; a score off by e
    changes every probability by at most a factor (1 + 2 e), e = 2^-bits reach for a rounded key; fp32 work (exp, sums)
    is within 2^-17 (1 + reach) of that sum at the lengths tested."""
    unit = 2.0 ** -operand_bits
    fp32 = 2.0 ** -17
    rounding = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[out_format]
    r = reach[..., None]
    tol = (2 * unit + 2 * unit * r + fp32 * (1 + r)) * spread
    return tol + rounding * (out.abs() + tol) + 1e-7
