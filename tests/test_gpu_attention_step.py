"""The attention step over a q4_0 cache on the GPU: kv_plan, qk_norm_rope, kv_append_q4_0, attention_q4_0.

Each operator against its plain form in 64 bits (tests/kv_plain.py); plans and cache bytes have to be equal.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
import kv_plain  # noqa: E402
import pfng_b200 as pb  # noqa: E402

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    yield
    pb.check_kernel_error()


# --------------------------------------------------------------------------- kv_plan
def run_plan(kv, q, page, max_pages, num_free, max_tokens, holes=False, seed=0):
    rng = np.random.default_rng(seed)
    have = [-(-max(k, 0) // page) for k in kv]
    ids = list(map(int, rng.permutation(sum(have) + num_free + 5)))
    table, at = [], 0
    for h in have:
        row = ids[at:at + h][:max_pages]
        at += h
        table.append(row + [-1] * (max_pages - len(row)))
    if holes and table and have[0]:
        table[0][0] = -7
    free = ids[sum(have):sum(have) + num_free]
    t = torch.tensor(table, dtype=torch.int32).reshape(len(kv), max_pages).cuda()
    got = pb.kv_plan(torch.tensor(kv, dtype=torch.int32).cuda(), torch.tensor(q, dtype=torch.int32).cuda(), t,
                     torch.tensor(free, dtype=torch.int32).cuda(), page, max_tokens)
    want = kv_plain.plan(kv, q, table, free, page, max_tokens)
    for name, g, w in zip(got._fields, got, want):
        assert g.cpu().tolist() == w, name
    assert t.cpu().reshape(-1).tolist() == [x for row in table for x in row]


@pytest.mark.parametrize("kv,q", [([0], [1]), ([15, 16, 17, 0], [1, 1, 1, 1]), ([5, 0, 40, 3], [0, 0, 7, 100]),
                                  ([0, 0], [0, 0]), ([-3, 9], [2, -1]), ([1000], [2000])])
@pytest.mark.parametrize("page", [16, 48, 64])
def test_plan_small(kv, q, page):
    total = sum(max(v, 0) for v in q)
    run_plan(kv, q, page, 200, 300, total)
    run_plan(kv, q, page, 200, 300, total + 600)        # a fixed capacity, padded
    run_plan(kv, q, page, 200, 300, max(0, total - 3))  # too small a capacity


@pytest.mark.parametrize("requests", [511, 512, 513, 1700])
def test_plan_many_requests(requests):
    rng = np.random.default_rng(requests)
    kv, q = rng.integers(0, 300, requests).tolist(), rng.integers(0, 40, requests).tolist()
    run_plan(kv, q, 16, 24, 6000, sum(q), seed=requests)


def test_plan_short_of_pages():
    run_plan([10, 20, 30], [50, 60, 70], 16, 20, 4, 180)            # free list too short
    run_plan([10, 20, 30], [50, 60, 70], 16, 4, 40, 180)            # table rows too short
    run_plan([10, 20, 30], [50, 60, 70], 16, 20, 0, 180)            # no free page at all
    run_plan([100, 20], [5, 6], 16, 20, 9, 11, holes=True)          # an entry of the table that is no page
    run_plan([], [], 16, 4, 4, 5)


# ---------------------------------------------------------------------- qk_norm_rope
def rope_table(max_pos, rot):
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))
    a = torch.arange(max_pos, dtype=torch.float64)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], 1).float()


def rope_tolerance(y, size, fmt):
    """fp32: a mean of up to 512 squares, a square root, a division and four products and a sum, each within 2^-23 and the
    sum's tree within 10 roundings: 2^-19 of |a| + |b|; then the rounding of the output."""
    unit = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[fmt]
    tol = 2.0 ** -19 * size
    return tol + unit * (y.abs() + tol) + (2.0 ** -25 if fmt == "f16" else 0)


def check_rope(tokens, hq, hk, dim, rot, interleaved, norm, fmt_in, fmt_out, pad=0, offset=0):
    g = torch.Generator().manual_seed(tokens * 31 + dim + rot)
    width = (hq + 2 * hk) * dim + pad
    flat = (torch.randn(tokens * width + offset, generator=g) * 1.7).to(DT[fmt_in])
    x = flat[offset:].reshape(tokens, width)
    pos = torch.randint(0, 500, (tokens,), generator=g, dtype=torch.int32)
    table = rope_table(500, rot)
    wq, wk = (1 + torch.randn(2, dim, generator=g) * 0.3) if norm else (None, None)
    xd = flat.cuda()[offset:].reshape(tokens, width)
    q, k = pb.qk_norm_rope(xd, pos.cuda(), table.cuda(), hq, hk, dim, q_weight=None if wq is None else wq.cuda(),
                           k_weight=None if wk is None else wk.cuda(), eps=1e-5, interleaved=interleaved,
                           out_format=fmt_out)
    heads = x[:, :(hq + hk) * dim].reshape(tokens, hq + hk, dim)
    for got, part, w in ((q, heads[:, :hq], wq), (k, heads[:, hq:], wk)):
        y, size = kv_plain.norm_rope(part, w, 1e-5, pos, table, rot, interleaved)
        err = (got.cpu().double().reshape(y.shape) - y).abs()
        tol = rope_tolerance(y, size, fmt_out)
        assert bool((err <= tol).all()), f"worst {float((err / tol).max())} of the tolerance"


@pytest.mark.parametrize("dim,rot", [(128, 128), (128, 64), (64, 64), (64, 32), (96, 96), (256, 128), (512, 512),
                                     (32, 6), (34, 34), (2, 2), (128, 0), (80, 20)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_shapes(dim, rot, interleaved):
    check_rope(5, 3, 2, dim, rot, interleaved, True, "f32", "f32")
    check_rope(3, 1, 1, dim, rot, interleaved, False, "bf16", "f16")


@pytest.mark.parametrize("fmt_in", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("fmt_out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("norm", [False, True])
def test_rope_types(fmt_in, fmt_out, norm):
    check_rope(67, 8, 2, 128, 128, False, norm, fmt_in, fmt_out)
    check_rope(9, 4, 4, 64, 64, True, norm, fmt_in, fmt_out, pad=3)              # odd row stride
    check_rope(4, 2, 1, 128, 128, False, norm, fmt_in, fmt_out, pad=8, offset=1)  # misaligned rows
    check_rope(1, 1, 0, 128, 128, False, norm, fmt_in, fmt_out)                  # no key heads
    check_rope(0, 2, 2, 128, 128, False, norm, fmt_in, fmt_out)


def test_rope_padding_positions_and_in_place():
    x = torch.randn(6, 5 * 64, device="cuda")
    pos = torch.tensor([0, -1, 7, 500, 499, -5], dtype=torch.int32, device="cuda")
    table = rope_table(500, 64).cuda()
    q, k = pb.qk_norm_rope(x, pos, table, 3, 2, 64, out_format="f32")
    for t in (q, k):
        assert bool((t[[1, 5]] == 0).all()) and bool(t[3].isnan().all()) and bool(t[[0, 2, 4]].isfinite().all())
    y = x.clone()
    pb.qk_norm_rope(y, pos, table, 3, 2, 64, q_out=y[:, :192], k_out=y[:, 192:])
    assert torch.equal(torch.nan_to_num(y[:, :192]), torch.nan_to_num(q))
    assert torch.equal(torch.nan_to_num(y[:, 192:]), torch.nan_to_num(k))


# -------------------------------------------------------------------- kv_append_q4_0
def check_append(oracle, tokens, heads, dim, page, pages, fmt_k, fmt_v, pad=0, offset=0, skip=(), special=False):
    g = torch.Generator().manual_seed(tokens + heads * 7 + dim)
    width = heads * dim + pad
    x, xd = {}, {}
    for name, fmt in (("k", fmt_k), ("v", fmt_v)):
        flat = (torch.randn(tokens * width + offset, generator=g) * 2).to(DT[fmt])
        if special:  # ties of magnitude, zeros, a block of zeros, tiny and large values
            rows = flat[offset:].reshape(tokens, width)
            rows[0, :32] = 0
            rows[1, :32] = torch.tensor([-1.5, 1.5] * 16).to(DT[fmt])
            rows[2, :32] = torch.tensor([1.5, -1.5, 0.75, 0.09375] * 8).to(DT[fmt])
            rows[3, :32] = (rows[3, :32].float() * 1e-6).to(DT[fmt])
            rows[4, :32] = (rows[4, :32].float() * 5e3).to(DT[fmt])
        x[name] = flat[offset:].reshape(tokens, width)[:, :heads * dim]
        xd[name] = flat.cuda()[offset:].reshape(tokens, width)[:, :heads * dim]
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    slots[list(skip)] = torch.tensor([-1, pages * page, -5, pages * page + 99][:len(skip)], dtype=torch.int64)
    size = pb.kv_cache_bytes(pages, page, heads, dim)
    caches = {n: torch.full((size,), 0xA5, dtype=torch.uint8, device="cuda") for n in "kv"}
    pb.kv_append_q4_0(xd["k"], xd["v"], slots.cuda(), caches["k"], caches["v"], heads, dim, page)
    for name in "kv":
        want = torch.full((size,), 0xA5, dtype=torch.uint8)
        n, d = kv_plain.unpack(want, pages, page, heads, dim, name == "k")
        keep = [t for t in range(tokens) if t not in skip]
        if keep:
            blocks = oracle.quantize("q4_0", x[name].float().reshape(tokens, heads * dim).numpy())
            qs = torch.from_numpy(blocks["qs"].copy()).reshape(tokens, heads, dim // 32, 16).to(torch.int32)
            dd = torch.from_numpy(blocks["d"].copy().view(np.float16)).reshape(tokens, heads, dim // 32)
            at = slots[keep]
            n[at // page, :, at % page] = torch.cat([qs & 15, qs >> 4], -1)[keep]
            d[at // page, :, at % page] = dd[keep]
        assert torch.equal(caches[name].cpu(), kv_plain.pack(n, d, name == "k")), name


@pytest.mark.parametrize("fmt_k", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("fmt_v", ["f32", "f16", "bf16"])
def test_append_types(oracle, fmt_k, fmt_v):
    check_append(oracle, 37, 2, 128, 16, 6, fmt_k, fmt_v, special=True)
    check_append(oracle, 20, 3, 64, 32, 2, fmt_k, fmt_v, pad=5)               # odd row stride
    check_append(oracle, 11, 1, 96, 48, 1, fmt_k, fmt_v, pad=8, offset=1)     # misaligned rows


@pytest.mark.parametrize("tokens,heads,dim,page,pages", [(1, 1, 32, 16, 1), (1, 8, 128, 64, 3), (128, 8, 128, 64, 2),
                                                         (300, 4, 256, 16, 40), (7, 2, 512, 16, 1), (33, 5, 160, 80, 1)])
def test_append_shapes(oracle, tokens, heads, dim, page, pages):
    check_append(oracle, tokens, heads, dim, page, pages, "bf16", "f32")
    if tokens > 4:
        check_append(oracle, tokens, heads, dim, page, pages, "f32", "bf16", skip=(0, 2, 3, 4))  # slots outside


# -------------------------------------------------------------------- attention_q4_0
class Case:
    """A cache with ragged requests on scattered pages; slots that no request owns hold NaN scales."""

    def __init__(self, seq, q_len, hq, hk, dim, page, fmt="f16", seed=0, spread=1.0, extra_rows=0, pad=0):
        g = torch.Generator().manual_seed(seed + sum(seq) + dim)
        need = [-(-n // page) for n in seq]
        self.seq, self.q_len, self.hq, self.hk, self.dim, self.page = seq, q_len, hq, hk, dim, page
        self.pages = sum(need) + 3
        ids = torch.randperm(self.pages, generator=g).tolist()
        self.max_pages = max(need + [0]) + 2
        self.table, at = [], 0
        for n in need:
            self.table.append(ids[at:at + n] + [-1] * (self.max_pages - n))
            at += n
        self.cu = [0]
        for m in q_len:
            self.cu.append(self.cu[-1] + m)
        self.caches, self.vals = {}, {}
        for name in "kv":
            shape = (self.pages, hk, page, dim // 32)
            n = torch.randint(0, 16, (*shape, 32), generator=g, dtype=torch.int32)
            d = (torch.rand(shape, generator=g) * 0.3 * spread + 0.01).half()
            used = torch.zeros(self.pages, page, dtype=torch.bool)
            for row, length in zip(self.table, seq):
                for j in range(length):
                    used[row[j // page], j % page] = True
            d = torch.where(used[:, None, :, None], d, torch.full_like(d, math.nan))
            raw = kv_plain.pack(n, d, name == "k")
            self.caches[name] = raw.cuda()
            self.vals[name] = kv_plain.values(raw, self.pages, page, hk, dim, name == "k")
        rows = self.cu[-1] + extra_rows
        self.q = torch.randn(rows, hq * dim + pad, generator=g).to(DT[fmt])

    def run(self, out_format="bf16", path="auto", causal=True, window=0, scale=None, max_q=None, max_kv=None):
        rows = self.q.shape[0]
        out = torch.full((rows, self.hq * self.dim), 77.0, dtype=DT[out_format], device="cuda")
        lse = torch.full((rows, self.hq), 77.0, device="cuda")
        pb.attention_q4_0(self.q.cuda()[:, :self.hq * self.dim], self.caches["k"], self.caches["v"],
                          torch.tensor(self.table, dtype=torch.int32).reshape(len(self.seq), -1).cuda(),
                          torch.tensor(self.seq, dtype=torch.int32).cuda(),
                          torch.tensor(self.cu, dtype=torch.int32).cuda(), self.hq, self.hk, self.dim, self.page,
                          max_q=max(self.q_len + [0]) if max_q is None else max_q,
                          max_kv=max(self.seq + [0]) if max_kv is None else max_kv, scale=scale, causal=causal,
                          window=window, out=out, lse=lse, path=path)
        return out.cpu(), lse.cpu()

    def check(self, out_format="bf16", path="auto", causal=True, window=0, scale=None, **more):
        got, lse = self.run(out_format, path, causal, window, scale, **more)
        q = self.q[:, :self.hq * self.dim].double().reshape(-1, self.hq, self.dim)
        want, want_lse, spread, reach = kv_plain.attention(
            q, self.vals["k"], self.vals["v"], self.table, self.seq, self.cu, self.page,
            self.dim ** -0.5 if scale is None else scale, causal, window)
        n = self.cu[-1]
        assert bool((got[n:] == 77).all()) and bool((lse[n:] == 77).all())  # rows of no request stay as they were
        # the SIMPLE path keeps fp32 operands, the others round them to fp16 (2^-11)
        tol = kv_plain.attention_tolerance(want, spread, reach, out_format, 24 if path == "simple" else 11)
        err = (got.double().reshape(-1, self.hq, self.dim) - want)[:n].abs()
        assert bool((err <= tol[:n]).all()), f"worst {float((err / tol[:n]).nan_to_num(9e9).max())} of the tolerance"
        empty = want_lse[:n] == -math.inf
        assert torch.equal(lse[:n] == -math.inf, empty)
        # ln of the sum moves by at most the error of a score
        unit = 2.0 ** -24 if path == "simple" else 2.0 ** -11
        off = (lse[:n].double() - want_lse[:n]).abs()[~empty]
        bound = ((unit + 2.0 ** -17) * (1 + reach[:n]) + 2.0 ** -20 * want_lse[:n].abs())[~empty]
        assert bool((off <= bound).all()), f"lse {float((off / bound).max())}"


PATHS = ["simple", "gemv", "mma", "auto"]


@pytest.mark.parametrize("path", PATHS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("hq,hk", [(1, 1), (4, 4), (8, 2), (6, 2), (8, 1), (16, 1)])
def test_attention_single_tokens(path, dim, hq, hk):
    Case([1, 2, 15, 16, 17, 33, 64, 129], [1] * 8, hq, hk, dim, 16).check(path=path)
    Case([300, 1, 1025], [1] * 3, hq, hk, dim, 64, "bf16").check("f32", path=path)


@pytest.mark.parametrize("path", PATHS)
@pytest.mark.parametrize("dim", [32, 96, 160, 256])
def test_attention_other_head_dims(path, dim):
    if path == "auto":
        Case([70, 3], [1, 1], 4, 2, dim, 16).check("f16")
    if path in ("gemv", "mma"):  # no such kernel for these
        with pytest.raises(pb.PfngError) as e:
            Case([70, 40], [5, 40], 4, 2, dim, 32).run("f16", path)
        assert e.value.status == -7
        return
    Case([70, 40], [5, 40], 4, 2, dim, 32).check("f16", path=path)


@pytest.mark.parametrize("path", PATHS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 48, 64, 256])
def test_attention_ragged_prompts(path, dim, page):
    Case([40, 7, 200, 0, 131], [40, 1, 130, 0, 3], 4, 2, dim, page).check(path=path)


@pytest.mark.parametrize("path", PATHS)
@pytest.mark.parametrize("window", [1, 5, 16, 100, 4000])
def test_attention_window(path, window):
    Case([90, 300, 16], [20, 1, 16], 4, 2, 64, 16).check(path=path, window=window)
    Case([300, 200], [1, 1], 4, 4, 128, 32).check(path=path, window=window)


@pytest.mark.parametrize("path", PATHS)
def test_attention_rows_without_keys(path):
    # more new tokens than keys: the first rows stand before the first key; a request without any key
    Case([3, 0, 5, 1], [5, 2, 5, 3], 4, 2, 64, 16, extra_rows=3).check(path=path)
    Case([0, 0], [1, 1], 4, 2, 128, 16).check(path=path)
    Case([20, 4], [0, 4], 2, 2, 128, 16, extra_rows=2).check(path=path)


@pytest.mark.parametrize("path", PATHS)
def test_attention_not_causal(path):
    Case([50, 3, 0, 130], [7, 10, 2, 1], 6, 3, 128, 16).check(path=path, causal=False)
    Case([200], [1], 8, 2, 64, 16).check(path=path, causal=False)


@pytest.mark.parametrize("path", PATHS)
@pytest.mark.parametrize("fmt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
def test_attention_types(path, fmt, out):
    Case([77, 21], [1, 1], 8, 2, 128, 16, fmt, pad=3).check(out, path=path)
    Case([77, 21], [30, 2], 8, 2, 64, 16, fmt, pad=8).check(out, path=path)


@pytest.mark.parametrize("path", PATHS)
def test_attention_scales_and_outliers(path):
    Case([100, 260], [1, 1], 4, 2, 128, 16, spread=4.0).check(path=path, scale=0.3)   # one key takes all
    Case([100, 260], [9, 1], 4, 2, 128, 16, spread=0.001).check("f16", path=path)     # tiny values
    c = Case([120], [60], 4, 2, 128, 16)
    c.q[:, :32] *= 40
    c.check(path=path)


@pytest.mark.parametrize("path", PATHS)
def test_attention_pages_outside_the_cache(path):
    c = Case([100, 40], [1, 30], 4, 2, 128, 16)
    c.table[0][2], c.table[0][4], c.table[1][0] = -1, c.pages, 1 << 30
    c.check(path=path)


@pytest.mark.parametrize("path", PATHS)
def test_attention_bounds_may_be_generous_and_results_repeat(path):
    c = Case([500, 30, 7], [1, 1, 1], 8, 2, 128, 16)
    c.check(path=path, max_q=3, max_kv=4000)
    a, b = c.run(path=path)[0], c.run(path=path)[0]
    assert torch.equal(a, b)


def test_attention_on_another_stream():
    c = Case([300, 40], [1, 20], 4, 2, 128, 16)
    want = c.run()[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = c.run()[0]
    assert torch.equal(want, got)


@pytest.mark.parametrize("path", PATHS)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("which", ["k", "v"])
def test_attention_scales_that_are_not_finite(path, bad, which):
    """A key with such a scale changes the rows that see it, and no other."""
    c = Case([200, 70], [180, 1], 4, 2, 128, 16)
    window, key = 60, 90
    want = c.run("f32", path, window=window)[0]
    raw = c.caches[which].cpu()
    n, d = kv_plain.unpack(raw, c.pages, c.page, c.hk, c.dim, which == "k")
    d[c.table[0][key // c.page], :, key % c.page] = bad
    c.caches[which] = kv_plain.pack(n, d, which == "k").cuda()
    got = c.run("f32", path, window=window)[0]
    pos = torch.arange(180) + 20
    sees = torch.cat([(pos >= key) & (pos - key < window), torch.zeros(1, dtype=torch.bool)])
    assert torch.equal(got[~sees], want[~sees])
    heads = got[sees].reshape(-1, c.hq, c.dim)
    assert bool((~heads.isfinite()).any(-1).all())


@pytest.mark.parametrize("path", PATHS)
def test_attention_output_rows_apart(path):
    """An output with a row stride of its own, aligned and not; what lies between the rows stays."""
    c = Case([150, 40], [30, 2], 4, 2, 64, 16)
    want = c.run(path=path)[0]
    for pad, offset in ((64, 0), (3, 0), (5, 1)):
        width = c.hq * c.dim + pad
        flat = torch.full((c.q.shape[0] * width + offset,), 5.0, dtype=torch.bfloat16, device="cuda")
        rows = flat[offset:].reshape(-1, width)
        pb.attention_q4_0(c.q.cuda(), c.caches["k"], c.caches["v"], torch.tensor(c.table, dtype=torch.int32).cuda(),
                          torch.tensor(c.seq, dtype=torch.int32).cuda(), torch.tensor(c.cu, dtype=torch.int32).cuda(),
                          c.hq, c.hk, c.dim, c.page, max_q=30, max_kv=150, out=rows[:, :c.hq * c.dim], path=path)
        assert torch.equal(rows[:, :c.hq * c.dim].cpu(), want) and bool((rows[:, c.hq * c.dim:] == 5).all())


@pytest.mark.parametrize("path,q_len", [("gemv", 1), ("mma", 40), ("simple", 2)])
def test_cache_past_32_bits(path, q_len):
    """Pages whose bytes lie past 4 GB: the same bits as on the first pages."""
    heads, dim, page, n = 8, 128, 64, 150
    per_page = pb.kv_cache_bytes(1, page, heads, dim)
    pages = (1 << 32) // per_page + 40
    g = torch.Generator("cuda").manual_seed(1)
    k = torch.randn(n, heads * dim, generator=g, device="cuda").bfloat16()
    v = torch.randn(n, heads * dim, generator=g, device="cuda")
    q = torch.randn(q_len, 2 * heads * dim, generator=g, device="cuda").bfloat16()
    outs = []
    for count, ids in ((3, [2, 0, 1]), (pages, [pages - 1, pages - 30, pages - 2])):
        caches = [torch.empty(count * per_page, dtype=torch.uint8, device="cuda") for _ in range(2)]
        table = torch.tensor([ids], dtype=torch.int32, device="cuda")
        slots = torch.tensor([ids[j // page] * page + j % page for j in range(n)], device="cuda")
        pb.kv_append_q4_0(k, v, slots, *caches, heads, dim, page)
        outs.append(pb.attention_q4_0(q, *caches, table, torch.tensor([n], dtype=torch.int32, device="cuda"),
                                      torch.tensor([0, q_len], dtype=torch.int32, device="cuda"), 2 * heads, heads, dim,
                                      page, max_q=q_len, max_kv=n, path=path))
    assert torch.equal(outs[0], outs[1]) and bool(outs[0].isfinite().all())


def test_step_in_a_graph():
    """Plan, rotation, append and attention captured once and replayed on new values."""
    c = Case([100, 33, 260], [1, 1, 1], 8, 2, 128, 16)
    table = torch.tensor(c.table, dtype=torch.int32).cuda()
    seq = torch.tensor(c.seq, dtype=torch.int32).cuda()
    cu = torch.tensor(c.cu, dtype=torch.int32).cuda()
    q = c.q.cuda()
    call = lambda: pb.attention_q4_0(q, c.caches["k"], c.caches["v"], table, seq, cu, 8, 2, 128, 16, max_q=1, max_kv=260)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = call()
    q.mul_(-1.5)
    graph.replay()
    torch.cuda.synchronize()
    got = out.clone()
    assert torch.equal(got, call())


@pytest.mark.parametrize("dim", [64, 128])
def test_attention_pieces_are_joined(dim):
    """Few blocks of rows over many keys (keys cut into pieces), ragged, on both tensor-core paths."""
    for path in ("gemv", "mma"):
        Case([3000, 700, 1], [20, 3, 1], 4, 2, dim, 64).check(path=path)
        Case([2500], [70], 4, 1, dim, 16).check("f32", path=path, window=900)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("requests,hq,hk,most_q,most_kv", [(90, 8, 4, 90, 400), (60, 8, 2, 150, 300), (400, 2, 2, 5, 60)])
def test_attention_more_blocks_than_run_at_once(dim, requests, hq, hk, most_q, most_kv):
    """Blocks of rows that a CTA takes one after the other: of one and two row tiles, without keys, without rows."""
    rng = np.random.default_rng(requests + dim)
    q_len = rng.integers(0, most_q + 1, requests)
    seq = rng.integers(0, most_kv + 1, requests)
    seq[::3] = np.maximum(seq[::3], q_len[::3])
    q_len[::7] = 0
    seq[5], q_len[5], q_len[8] = 1500, most_q, 1
    c = Case(seq.tolist(), q_len.tolist(), hq, hk, dim, 16, "bf16", extra_rows=2)
    c.check(path="mma")
    c.check("f32", path="mma", window=70)
    c.check("f16", path="mma", causal=False)
    assert all(torch.equal(x, y) for x, y in zip(c.run(path="mma"), c.run(path="mma")))


def test_example_runs():
    import importlib.util
    import pathlib
    path = pathlib.Path(__file__).resolve().parent.parent / "examples" / "quantized_attention.py"
    spec = importlib.util.spec_from_file_location("quantized_attention", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    layer, table, held, q, a, out = m.run(steps=3)
    off, size = m.check(layer, table, held, q, a)
    # fp32 output: d P rounded to fp16 (2^-11 at most) of a mean of values of this size
    assert bool(out.isfinite().all()) and off <= 2 ** -10 * 4 * size


# ------------------------------------------------------------------- the step as a whole
def test_step_of_a_layer_over_two_steps():
    """Plan, rotate, append, attend for a prompt step and a decode step; against 64 bits on the cache's own values."""
    hq, hk, dim, page, pages = 8, 2, 128, 16, 40
    width = (hq + 2 * hk) * dim
    g = torch.Generator("cuda").manual_seed(4)
    size = pb.kv_cache_bytes(pages, page, hk, dim)
    kc, vc = (torch.zeros(size, dtype=torch.uint8, device="cuda") for _ in range(2))
    table = torch.full((3, 12), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(pages, device="cuda").to(torch.int32)
    kv = torch.zeros(3, dtype=torch.int32, device="cuda")
    cs = rope_table(256, dim).cuda()
    w = torch.ones(dim, device="cuda")
    taken = 0
    for lens in ([33, 1, 70], [1, 1, 1]):
        total = sum(lens)
        plan = pb.kv_plan(kv, torch.tensor(lens, dtype=torch.int32, device="cuda"), table, free[taken:], page, total)
        x = torch.randn(total, width, generator=g, device="cuda")
        q, k = pb.qk_norm_rope(x, plan.positions, cs, hq, hk, dim, q_weight=w, k_weight=w)
        pb.kv_append_q4_0(k, x[:, (hq + hk) * dim:], plan.slots, kc, vc, hk, dim, page)
        seq = plan.seq_len.tolist()
        out = pb.attention_q4_0(q, kc, vc, table, plan.seq_len, plan.cu_q, hq, hk, dim, page, max_q=max(lens),
                                max_kv=max(seq), out_format="bf16")
        want, _, spread, reach = kv_plain.attention(
            q.cpu().double().reshape(total, hq, dim), kv_plain.values(kc, pages, page, hk, dim, True),
            kv_plain.values(vc, pages, page, hk, dim, False), table.tolist(), seq, plan.cu_q.tolist(), page,
            dim ** -0.5, True, 0)
        tol = kv_plain.attention_tolerance(want, spread, reach, "bf16", 11)
        assert bool(((out.cpu().double().reshape(want.shape) - want).abs() <= tol).all())
        taken += plan.counts.tolist()[1]
        assert plan.counts.tolist()[2] == 0
        kv = plan.seq_len
