"""Paged 8-bit cache and beam selection against a plain implementation in 64 bits.

Tolerances of attention (``bound``), per output value, from the arithmetic:
  * the result is rounded to 16 bits once: half a step of its type, relative to the value (bf16 2^-8, fp16 2^-11);
  * a score is a sum of 128 exact products in fp32: off by at most 128 * 2^-23 * sum |q k| scale, a capped one by another
    2^-21 cap, the bias and the multiplication by log2 e by 2^-22 of the magnitudes; exponential and sums by 2^-20;
    an error d of the scores changes a normalised weight by at most 2 d of itself;
  * the weights enter the product with the values with at least fp16's half step, 2^-11 of themselves;
  weights' errors reach the result through sum p |v|, which the reference computes.
Codes, scales, tails, tables, references, parents and tokens are exact.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

D = 128
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


# ------------------------------------------------------------------ the plain implementation

def encode(x, fmt):
    """x [H, page, 128] fp64 -> the values that the page stands for, by the definition of the format."""
    top = 448.0 if fmt == "e4m3" else 127.0
    out = torch.empty_like(x)
    for h in range(x.shape[0]):
        if not bool(torch.isfinite(x[h]).all()):
            out[h] = math.nan
            continue
        amax = float(x[h].abs().max())
        e = 0
        if amax > 0:
            e = math.frexp(amax / top)[1]
            while e > -126 and amax <= top * 2.0 ** (e - 1):
                e -= 1
            while e < -126 or amax > top * 2.0 ** e:
                e += 1
        y = x[h] / 2.0 ** e
        if fmt == "int8":
            code = torch.round(y)
            under = torch.trunc(y)
        else:
            a = y.abs()
            step = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0 ** -20))).clamp_min(-6) - 3)
            code = torch.round(y / step) * step
            under = torch.trunc(y / step) * step
        out[h] = torch.where((code * 2.0 ** e).abs() < 2.0 ** 128, code, under) * 2.0 ** e      # values stay in fp32's range
    return out


class Plain:
    """The tokens of every sequence as they came; what the cache stands for is computed from them."""

    def __init__(self, L, N, H, page, fmt, dtype):
        self.L, self.N, self.H, self.page, self.fmt, self.dtype = L, N, H, page, fmt, dtype
        self.k = [[torch.zeros(H, 0, D, dtype=torch.float64) for _ in range(N)] for _ in range(L)]
        self.v = [[torch.zeros(H, 0, D, dtype=torch.float64) for _ in range(N)] for _ in range(L)]
        self.new = [0] * N

    def begin(self, new):
        self.new = list(new)

    def append(self, layer, k, v):
        for n in range(self.N):
            self.k[layer][n] = torch.cat([self.k[layer][n], k[n, :, : self.new[n]].double().cpu()], dim=1)
            self.v[layer][n] = torch.cat([self.v[layer][n], v[n, :, : self.new[n]].double().cpu()], dim=1)

    def fork(self, parents):
        W = parents.shape[1]
        src = [b * W + int(parents[b, w]) for b in range(parents.shape[0]) for w in range(W)]
        for x in (self.k, self.v):
            for layer in range(self.L):
                x[layer] = [x[layer][s] for s in src]
        self.new = [self.new[s] for s in src]

    def free(self, leave):
        for n in range(self.N):
            if leave[n]:
                self.new[n] = 0
                for x in (self.k, self.v):
                    for layer in range(self.L):
                        x[layer][n] = x[layer][n][:, :0]

    def stored(self, layer, n):
        out = []
        for x in (self.k, self.v):
            t = x[layer][n].clone()
            for p in range(t.shape[1] // self.page):
                t[:, p * self.page:(p + 1) * self.page] = encode(t[:, p * self.page:(p + 1) * self.page], self.fmt)
            out.append(t)
        return out

    def attention(self, layer, q, scale=None, softcap=0.0, slopes=None):
        return dense_attention([self.stored(layer, n) for n in range(self.N)], self.new, q, scale, softcap, slopes)


def dense_attention(stored, new, q, scale=None, softcap=0.0, slopes=None):
    """(want, bound, lse, lse_bound) in fp64 on the device of q; stored[n]: keys and values [H, tokens, 128]."""
    N, Hq, Tq, _ = q.shape
    dev = q.device
    scale = D ** -0.5 if scale is None else scale
    want = torch.zeros(N, Hq, Tq, D, dtype=torch.float64, device=dev)
    bound = torch.zeros_like(want)
    lse = torch.full((N, Hq, Tq), -math.inf, dtype=torch.float64, device=dev)
    lse_bound = torch.zeros_like(lse)
    for n in range(N):
        K, V = (t.to(dev) for t in stored[n])
        H, total = K.shape[0], K.shape[1]
        if new[n] == 0 or total == 0:
            continue
        G = Hq // H
        qn = q[n, :, : new[n]].double().view(H, G, -1, D)
        dist = (torch.arange(total, device=dev)[None, :] - (total - new[n] + torch.arange(qn.shape[2], device=dev))[:, None]).double()
        s = torch.einsum("hgtd,hkd->hgtk", qn, K) * scale
        mags = torch.einsum("hgtd,hkd->hgtk", qn.abs(), K.abs()) * abs(scale)
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        if slopes is not None:
            s = s + slopes.double().view(H, G, 1, 1) * dist
            mags = mags + 0 * s + (slopes.double().view(H, G, 1, 1) * dist).abs() * 2.0 ** (16 - 21)
        hidden = dist > 0
        s = s.masked_fill(hidden, -math.inf)
        mags = mags.masked_fill(hidden, 0)
        d = mags.amax(-1) * 2.0 ** -16 + 2.0 ** -21 * softcap + 2.0 ** -20
        p = torch.softmax(s, -1)
        rows = slice(0, qn.shape[2])
        want[n, :, rows] = torch.einsum("hgtk,hkd->hgtd", p, V).reshape(Hq, -1, D)
        spread = torch.einsum("hgtk,hkd->hgtd", p, V.abs())
        bound[n, :, rows] = ((2 * d + 2.0 ** -11)[..., None] * spread).reshape(Hq, -1, D) + HALF[q.dtype] * want[n, :, rows].abs()
        lse[n, :, rows] = torch.logsumexp(s, -1).reshape(Hq, -1)
        lse_bound[n, :, rows] = (d + 2.0 ** -20 * (1 + torch.logsumexp(s, -1).abs())).reshape(Hq, -1)
    bound = bound + (2.0 ** -25 if q.dtype == torch.float16 else 2.0 ** -134)      # below the normal numbers the step is fixed
    return want, bound, lse, lse_bound


def check_attention(got, lse, ref, what=""):
    want, bound, wlse, lbound = ref
    assert torch.isfinite(got).all() or torch.isnan(want).any(), what
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), (what, float((off / bound).max()))
    if lse is not None:
        empty = wlse == -math.inf
        assert bool((lse[empty] == -math.inf).all()), what
        assert bool(((lse.double() - wlse).abs()[~empty] <= lbound[~empty]).all()), what


def tokens(g, *shape, dtype, keys):
    x = torch.randn(*shape, D, generator=g)
    if keys:
        x[..., 5::32] *= 10.0
    return x.to(dtype).cuda()


def check_cache(cache, ref):
    """Everything the cache holds, exactly; references against the table."""
    total = (cache.lens + cache.new_lens).tolist()
    for layer in range(ref.L):
        for n in range(ref.N):
            assert total[n] == ref.k[layer][n].shape[1]
            got = cache.materialize(layer, n)
            for a, b in zip(got, ref.stored(layer, n)):
                b = b.cuda()
                assert torch.equal(torch.isnan(a), torch.isnan(b))
                assert torch.equal(a.double().nan_to_num(), b.nan_to_num())
    table = cache.table.cpu()
    assert int(table.max()) < cache.num_pages
    for n in range(ref.N):
        full = total[n] // cache.page
        assert bool((table[n, :full] >= 0).all()) and bool((table[n, full:] == -1).all())
    held = table[table >= 0].long()
    assert torch.equal(torch.bincount(held, minlength=cache.num_pages), cache.refs.cpu().long())


def make(pkg, L, N, H, page, max_tokens, fmt="e4m3", dtype=torch.bfloat16, pages=None):
    pages = N * (max_tokens // page + 1) if pages is None else pages
    return (pkg.BlockKVCache.allocate(L, N, H, pages, max_tokens, page, dtype, fmt), Plain(L, N, H, page, fmt, dtype))


def step(cache, ref, g, new, H=None):
    """begin + append in all layers, with the newest tokens' keys and values."""
    new = [int(x) for x in new]
    T = max(new)
    cache.begin(torch.tensor(new, dtype=torch.int32, device="cuda"))
    ref.begin(new)
    for layer in range(ref.L):
        k = tokens(g, ref.N, ref.H, T, dtype=ref.dtype, keys=True)
        v = tokens(g, ref.N, ref.H, T, dtype=ref.dtype, keys=False)
        cache.append(layer, k, v)
        ref.append(layer, k, v)


# ------------------------------------------------------------------ append

@pytest.mark.parametrize("fmt,dtype", [("e4m3", torch.bfloat16), ("int8", torch.float16), ("e4m3", torch.float16), ("int8", torch.bfloat16)])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_append_ragged_steps(pkg, cuda, page, fmt, dtype):
    g = torch.Generator().manual_seed(page)
    cache, ref = make(pkg, 2, 4, 2, page, 4 * page + 40, fmt, dtype)
    for new in ([1, 0, page, 2 * page + 3], [page - 1, 5, 0, 1], [1, 1, 1, 1], [0, page - 5, 3, page], [2, page, 1, 0]):
        step(cache, ref, g, new)
        check_cache(cache, ref)
    cache.check()


def test_append_takes_any_strides(pkg, cuda):
    g = torch.Generator().manual_seed(3)
    cache, ref = make(pkg, 1, 2, 3, 16, 64)
    big = tokens(g, 2, 20, 3 + 4, dtype=torch.bfloat16, keys=True)               # [N, T, H', 128]: a slice of a joint projection
    k, v = big[:, :, 1:4].transpose(1, 2), big[:, :, 4:7].transpose(1, 2)
    cache.begin(20)
    ref.begin([20, 20])
    cache.append(0, k, v)
    ref.append(0, k, v)
    check_cache(cache, ref)
    flat = torch.zeros(2 * 3 * 7 * D + 1, dtype=torch.bfloat16, device=cuda)[1:]     # two bytes off the 16-byte boundary
    flat.copy_(tokens(g, 2 * 3 * 7, dtype=torch.bfloat16, keys=False).view(-1))
    odd = flat.view(2, 3, 7, D)
    cache.begin(7)
    ref.begin([7, 7])
    cache.append(0, odd, odd)
    ref.append(0, odd, odd)
    check_cache(cache, ref)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_append_special_values(pkg, cuda, fmt, dtype):
    """Zeros, the type's extremes, numbers below the normal ones, ties at half a step; infinities and NaN poison their page only."""
    g = torch.Generator().manual_seed(5)
    cache, ref = make(pkg, 1, 6, 1, 16, 48, fmt, dtype)
    x = tokens(g, 6, 1, 32, dtype=dtype, keys=False)
    x[0, 0, :16] = 0.0
    x[1] *= torch.finfo(dtype).max / 8
    x[1, 0, 3, 7] = -torch.finfo(dtype).max
    x[2] = x[2] * (2.0 ** -132 if dtype == torch.bfloat16 else 2.0 ** -20)
    x[3, 0, 2, 9], x[3, 0, 20, 1] = math.inf, -math.inf
    x[4, 0, 17, 0] = math.nan
    ties = torch.arange(-64, 64, device=cuda).to(torch.float32)
    x[5] = (ties * 0.5 + 0.25).to(dtype)
    x[5, 0, 0, 0] = 127.0 if fmt == "int8" else 448.0
    cache.begin(32)
    ref.begin([32] * 6)
    cache.append(0, x, x)
    ref.append(0, x, x)
    check_cache(cache, ref)


# ------------------------------------------------------------------ attention

CASES = [
    # N, H, G, page, fmt, dtype, before, Tq
    (1, 1, 1, 16, "e4m3", torch.bfloat16, [0], 1),
    (3, 2, 4, 16, "e4m3", torch.float16, [0, 15, 16], 1),
    (3, 2, 4, 64, "int8", torch.bfloat16, [63, 127, 200], 1),
    (4, 4, 7, 32, "int8", torch.bfloat16, [1, 31, 500, 333], 1),
    (2, 1, 8, 128, "e4m3", torch.bfloat16, [127, 1000], 1),
    (2, 2, 12, 64, "e4m3", torch.float16, [77, 640], 1),
    (1, 1, 16, 16, "int8", torch.float16, [2000], 1),
    (2, 8, 3, 64, "e4m3", torch.bfloat16, [3000, 5], 1),
    (1, 2, 5, 64, "e4m3", torch.bfloat16, [0], 130),          # a prompt from nothing
    (2, 2, 4, 64, "e4m3", torch.bfloat16, [100, 700], 37),
    (2, 1, 8, 16, "int8", torch.float16, [5, 400], 3),
    (3, 1, 1, 32, "e4m3", torch.float16, [0, 64, 300], 65),
    (1, 2, 4, 128, "int8", torch.bfloat16, [1100], 257),
    (1, 1, 33, 64, "e4m3", torch.bfloat16, [90], 2),
]


@pytest.mark.parametrize("N,H,G,page,fmt,dtype,before,Tq", CASES)
@pytest.mark.parametrize("softcap,slopes", [(0.0, False), (20.0, True)])
def test_attention(pkg, cuda, N, H, G, page, fmt, dtype, before, Tq, softcap, slopes):
    g = torch.Generator().manual_seed(sum(before) + Tq)
    cache, ref = make(pkg, 1, N, H, page, max(before) + Tq, fmt, dtype)
    if max(before):
        step(cache, ref, g, before)
    step(cache, ref, g, [Tq] * N)
    q = torch.randn(N, H * G, Tq, D, generator=g).to(dtype).cuda()
    sl = torch.exp2(-torch.arange(1, H * G + 1).float() * 8 / (H * G)).cuda() if slopes else None
    out, lse = cache.attention(0, q, softcap=softcap, slopes=sl, return_lse=True)
    check_attention(out, lse, ref.attention(0, q, softcap=softcap, slopes=sl))
    again = cache.attention(0, q, softcap=softcap, slopes=sl)
    assert torch.equal(out, again)                                   # the same call gives the same bits


@pytest.mark.parametrize("Tq", [1, 6, 40])
def test_attention_padded_batch(pkg, cuda, Tq):
    """Fewer running tokens than rows, sequences without any, an empty sequence: the rows behind are zeros."""
    g = torch.Generator().manual_seed(Tq)
    cache, ref = make(pkg, 1, 5, 2, 32, 400)
    step(cache, ref, g, [100, 0, 350, 0, 64])
    new = [min(Tq, x) for x in (1, 0, Tq, Tq, 0)]
    step(cache, ref, g, new)
    q = torch.randn(5, 8, Tq, D, generator=g).to(torch.bfloat16).cuda()
    q[1] = math.nan                                                  # padding is not read
    out, lse = cache.attention(0, q, return_lse=True)
    for n in range(5):
        assert bool((out[n, :, new[n]:] == 0).all())
        q[n, :, new[n]:] = 0
    check_attention(out, lse, ref.attention(0, q))


def test_attention_strided_query_and_scale(pkg, cuda):
    g = torch.Generator().manual_seed(11)
    cache, ref = make(pkg, 1, 2, 2, 16, 120)
    step(cache, ref, g, [90, 33])
    step(cache, ref, g, [9, 9])
    q = torch.randn(2, 9, 8, D, generator=g).to(torch.bfloat16).cuda().transpose(1, 2)
    check_attention(cache.attention(0, q, scale=0.31), None, ref.attention(0, q, scale=0.31))
    check_attention(cache.attention(0, q, scale=-0.05), None, ref.attention(0, q, scale=-0.05))
    check_attention(cache.attention(0, q, scale=0.0), None, ref.attention(0, q, scale=0.0))


@pytest.mark.parametrize("heads", [4, 16])                             # 20 and 80 rows: the step and the tile kernel
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_wide_ranges(pkg, cuda, dtype, heads):
    """Pages whose values differ by 2^20 in size, large queries, scores of hundreds: nothing overflows on the way."""
    g = torch.Generator().manual_seed(12)
    cache, ref = make(pkg, 1, 1, 1, 16, 200, "e4m3", dtype)
    size = torch.exp2(torch.tensor([0, 10, -10, 5, -4, 8, 2, 0, -8, 9, 1, 3]).float()).repeat_interleave(16)
    k = (torch.randn(1, 1, 192, D, generator=g) * 3).to(dtype).cuda()
    v = (torch.randn(1, 1, 192, D, generator=g) * size[:, None]).to(dtype).cuda()
    cache.begin(192), ref.begin([192])
    cache.append(0, k, v), ref.append(0, k, v)
    step(cache, ref, g, [5])
    for mul in (1.0, 30.0, 2.0 ** -12):
        q = (torch.randn(1, heads, 5, D, generator=g) * mul).to(dtype).cuda()
        out, lse = cache.attention(0, q, return_lse=True)
        check_attention(out, lse, ref.attention(0, q), mul)
    if dtype == torch.bfloat16:                                       # beyond fp16's range
        q = (torch.randn(1, heads, 5, D, generator=g) * 2.0 ** 20).to(dtype).cuda()
        out, lse = cache.attention(0, q, scale=2.0 ** -24, return_lse=True)
        check_attention(out, lse, ref.attention(0, q, scale=2.0 ** -24))
        cache2, ref2 = make(pkg, 1, 1, 1, 16, 40, "e4m3", dtype)
        k = tokens(g, 1, 1, 23, dtype=dtype, keys=False)
        v = (torch.randn(1, 1, 23, D, generator=g) * 2.0 ** 100).to(dtype).cuda()
        cache2.begin(23), ref2.begin([23])
        cache2.append(0, k, v), ref2.append(0, k, v)
        q = torch.randn(1, heads, 23, D, generator=g).to(dtype).cuda()
        check_attention(cache2.attention(0, q), None, ref2.attention(0, q))
    # values near the lower end of the type, in pages and in the tail, and all zeros in either
    for tiny, zero_tail in ((2.0 ** -110 if dtype == torch.bfloat16 else 2.0 ** -10, False), (1.0, True), (0.0, False)):
        cache3, ref3 = make(pkg, 1, 1, 1, 16, 40, "int8", dtype)
        k = tokens(g, 1, 1, 38, dtype=dtype, keys=False)
        v = (torch.randn(1, 1, 38, D, generator=g) * tiny).to(dtype).cuda()
        if zero_tail:
            v[:, :, 32:] = 0.0
        cache3.begin(38), ref3.begin([38])
        cache3.append(0, k, v), ref3.append(0, k, v)
        q = torch.randn(1, heads, 38, D, generator=g).to(dtype).cuda()
        want, bound, _, _ = ref3.attention(0, q)
        got = cache3.attention(0, q).double()
        assert bool(((got - want).abs() <= bound).all()), (tiny, zero_tail)


def test_attention_poisoned_page_and_garbage_behind_the_tail(pkg, cuda):
    """A NaN in a page reaches the rows that see it and no other; what lies behind the last token is never used."""
    g = torch.Generator().manual_seed(13)
    cache, ref = make(pkg, 1, 2, 1, 16, 100)
    k = tokens(g, 2, 1, 70, dtype=torch.bfloat16, keys=True)
    v = tokens(g, 2, 1, 70, dtype=torch.bfloat16, keys=False)
    k[0, 0, 20] = math.nan
    cache.k_tail.fill_(math.nan)
    cache.v_tail.fill_(math.inf)
    cache.k_codes.view(torch.uint8).fill_(0x7f)                        # NaN in e4m3
    cache.begin(70), ref.begin([70, 70])
    cache.append(0, k, v), ref.append(0, k, v)
    q = torch.randn(2, 2, 70, D, generator=g).to(torch.bfloat16).cuda()
    out = cache.attention(0, q)
    assert bool(torch.isnan(out[0, :, 20:]).all())
    want, bound, _, _ = ref.attention(0, q)
    seen = torch.cat([out[0, :, :16].double() - want[0, :, :16], out[1].double() - want[1]], dim=1).abs()
    assert bool((seen <= torch.cat([bound[0, :, :16], bound[1]], dim=1)).all())


@pytest.mark.parametrize("Tq,G", [(12, 1), (12, 3), (70, 4)])
def test_attention_infinities_in_the_tail(pkg, cuda, Tq, G):
    """NaN and infinities among the running tokens reach the rows that see them, and those only."""
    g = torch.Generator().manual_seed(14)
    cache, ref = make(pkg, 1, 1, 1, 128, 300)
    step(cache, ref, g, [40])
    k = tokens(g, 1, 1, Tq, dtype=torch.bfloat16, keys=True)
    v = tokens(g, 1, 1, Tq, dtype=torch.bfloat16, keys=False)
    v[0, 0, 5, 3], v[0, 0, 7, 90], v[0, 0, 9, 3] = math.inf, math.nan, -math.inf
    k[0, 0, Tq - 1, 2] = math.nan
    cache.begin(Tq), ref.begin([Tq])
    cache.append(0, k, v), ref.append(0, k, v)
    q = torch.randn(1, G, Tq, D, generator=g).to(torch.bfloat16).cuda()
    out = cache.attention(0, q)
    want, bound, _, _ = ref.attention(0, q)
    for j in range(Tq - 1):
        row, w = out[0, :, j].double(), want[0, :, j]
        bad = torch.zeros(D, dtype=torch.bool, device=cuda)
        if j >= 5:
            bad[3] = True
            assert bool((torch.isinf(row[:, 3]) if j < 9 else torch.isnan(row[:, 3])).all())
        if j >= 7:
            bad[90] = True
            assert bool(torch.isnan(row[:, 90]).all())
        clean = ref_row_without(ref, q, j, bad)
        assert bool(((row - clean[0]).abs() <= clean[1])[:, ~bad].all()), j
    assert bool(torch.isnan(out[0, :, Tq - 1]).all())


def ref_row_without(ref, q, j, bad):
    """Row j's result and bound with only the tokens it sees, infinite coordinates left out."""
    k, v = ref.stored(0, 0)
    seen = k.shape[1] - ref.new[0] + j + 1
    v = v[:, :seen].clone()
    v[..., bad.cpu()] = 0.0
    want, bound, _, _ = dense_attention([(k[:, :seen], v)], [1], q[:, :, j:j + 1])
    return want[0, :, 0], bound[0, :, 0]


def test_attention_long_and_deep_offsets(pkg, cuda):
    """Pages beyond 4 GB of codes, and a sequence of 40 000 tokens whose pages lie in any order."""
    H, page, pages = 8, 64, 70000                                     # 70000 * 65536 bytes = 4.6 GB a side
    N, ctx = 2, 40000
    width = ctx // page + 1
    codes = [torch.zeros(1, pages, H, page, D, dtype=torch.int8, device=cuda) for _ in range(2)]
    scale = [torch.ones(1, pages, H, device=cuda) for _ in range(2)]
    g = torch.Generator().manual_seed(2)
    order = torch.randperm(3 * N * width, generator=g)[: N * (ctx // page)] + pages - 3 * N * width
    table = torch.full((N, width), -1, dtype=torch.int32)
    table[:, : ctx // page] = order.view(N, -1).to(torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    refs[order] = 1
    at = order.cuda()
    for c, s in zip(codes, scale):
        c[0, at] = torch.randint(-127, 128, (at.numel(), H, page, D), generator=g, dtype=torch.int8).cuda()
        s[0, at] = torch.exp2(torch.randint(-8, -4, (at.numel(), H), generator=g).float()).cuda()
    tail = [torch.zeros(1, N, H, page, D, dtype=torch.bfloat16, device=cuda) for _ in range(2)]
    lens = torch.tensor([ctx - 1, ctx // 3], dtype=torch.int32, device=cuda)
    cache = pkg.BlockKVCache(*codes, *scale, *tail, table.cuda(), lens, torch.ones_like(lens), refs.cuda())
    cache.table[1, (ctx // 3 + 1) // page:] = -1
    q = torch.randn(N, H * 4, 1, D, generator=g).to(torch.bfloat16).cuda()
    out, lse = cache.attention(0, q, return_lse=True)
    check_attention(out, lse, dense_attention([[t.double() for t in cache.materialize(0, n)] for n in range(N)], [1, 1], q))


def test_attention_on_a_side_stream_and_in_a_graph(pkg, cuda):
    """A captured step of two layers, replayed as the sequences grow past pages, equals the eager one; two graphs that share
    the allocator's pool do not disturb each other."""
    g = torch.Generator().manual_seed(21)
    N, H, L = 3, 2, 2
    cache, ref = make(pkg, L, N, H, 16, 100)
    step(cache, ref, g, [14, 0, 33])
    k = torch.zeros(L, N, H, 1, D, dtype=torch.bfloat16, device=cuda)
    v, q = torch.zeros_like(k), torch.zeros(L, N, 4 * H, 1, D, dtype=torch.bfloat16, device=cuda)

    def run():
        cache.begin(1)
        outs = []
        for layer in range(L):
            cache.append(layer, k[layer], v[layer])
            outs.append(cache.attention(layer, q[layer]))
        return torch.stack(outs)

    import copy
    saved = copy.deepcopy(cache)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()                                                          # warm up, on the side stream
    torch.cuda.current_stream().wait_stream(side)
    names = ("k_codes", "v_codes", "k_scale", "v_scale", "k_tail", "v_tail", "table", "lens", "new_lens", "refs", "status")

    def restore():
        for x in names:
            getattr(cache, x).view(torch.uint8).copy_(getattr(saved, x).view(torch.uint8))

    restore()
    pool = torch.cuda.graph_pool_handle()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, pool=pool):
            out = run()
        graphs.append((gr, out))
    restore()
    for i in range(20):
        k.copy_(tokens(g, L, N, H, 1, dtype=torch.bfloat16, keys=True))
        v.copy_(tokens(g, L, N, H, 1, dtype=torch.bfloat16, keys=False))
        q.copy_(torch.randn(q.shape, generator=g))
        gr, out = graphs[i % 2]
        gr.replay()
        ref.begin([1] * N)
        for layer in range(L):
            ref.append(layer, k[layer], v[layer])
            check_attention(out[layer], None, ref.attention(layer, q[layer]), (i, layer))
    check_cache(cache, ref)
    cache.check()


def test_dimensions_of_one_with_any_stride(pkg, cuda):
    """One token, one head or one sequence out of a larger tensor: the stride of a dimension of one means nothing."""
    g = torch.Generator().manual_seed(17)
    cache, ref = make(pkg, 1, 1, 1, 16, 64)
    step(cache, ref, g, [30])
    big = torch.randn(9 * D, generator=g).to(torch.bfloat16).cuda()
    k = big.as_strided((1, 1, 1, D), (5, 3, 7, 1), D)
    v = big.as_strided((1, 1, 1, D), (1, 1, 1, 1), 2 * D)
    q = big.as_strided((1, 3, 1, D), (3, 2 * D, 11, 1), 3 * D)
    cache.begin(1), ref.begin([1])
    cache.append(0, k, v), ref.append(0, k, v)
    check_cache(cache, ref)
    check_attention(cache.attention(0, q), None, ref.attention(0, q))


@pytest.mark.parametrize("Tq", [1, 50])
@pytest.mark.parametrize("hole", [-1, 10 ** 6])
def test_attention_over_a_hole_in_the_table(pkg, cuda, Tq, hole):
    """A table entry without a page gives NaN to the sequence, and to no other."""
    g = torch.Generator().manual_seed(18)
    cache, ref = make(pkg, 1, 2, 2, 16, 400)
    step(cache, ref, g, [300, 200])
    step(cache, ref, g, [Tq, Tq])
    q = torch.randn(2, 4, Tq, D, generator=g).to(torch.bfloat16).cuda()
    want = ref.attention(0, q)
    cache.table[0, 7] = hole
    out = cache.attention(0, q)
    assert bool(torch.isnan(out[0]).all())
    check_attention(out[1:], None, tuple(t[1:] for t in want))


def test_captured_chunks_follow_the_lengths(pkg, cuda):
    """A captured chunk of 40 tokens (the tile kernel), replayed as the sequences grow and with fewer tokens in some."""
    g = torch.Generator().manual_seed(22)
    N, H, T = 2, 1, 40
    cache, ref = make(pkg, 1, N, H, 32, 600)
    step(cache, ref, g, [10, 100])
    k = torch.zeros(N, H, T, D, dtype=torch.bfloat16, device=cuda)
    v, q = torch.zeros_like(k), torch.zeros(N, 4, T, D, dtype=torch.bfloat16, device=cuda)
    new = torch.zeros(N, dtype=torch.int32, device=cuda)

    def run():
        cache.begin(new)
        cache.append(0, k, v)
        return cache.attention(0, q)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()                                                          # warm up: a step without tokens
    torch.cuda.current_stream().wait_stream(side)
    ref.begin([0, 0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for more in ([40, 40], [0, 40], [40, 3], [40, 39], [17, 40], [0, 0]):
        new.copy_(torch.tensor(more, dtype=torch.int32))
        k.copy_(tokens(g, N, H, T, dtype=torch.bfloat16, keys=True))
        v.copy_(tokens(g, N, H, T, dtype=torch.bfloat16, keys=False))
        q.copy_(torch.randn(q.shape, generator=g))
        graph.replay()
        ref.begin(more)
        ref.append(0, k, v)
        clean = q.clone()
        for n in range(N):
            clean[n, :, more[n]:] = 0
        check_attention(out, None, ref.attention(0, clean), more)
    check_cache(cache, ref)


# ------------------------------------------------------------------ pages

def test_begin_refuses_what_does_not_fit(pkg, cuda):
    g = torch.Generator().manual_seed(1)
    cache, ref = make(pkg, 1, 4, 1, 16, 64, pages=5)
    step(cache, ref, g, [20, 16, 3, 0])                                # two pages taken
    cache.check()
    cache.begin(torch.tensor([32, 64, 16, 28], dtype=torch.int32, device=cuda))     # 2 pages, 4 (a row holds 4 in all), 1, 1
    assert cache.new_lens.tolist() == [32, 0, 16, 0] and cache.lens.tolist() == [20, 16, 3, 0]
    assert int(cache.status) == pkg._lib.PAGES_EXHAUSTED | pkg._lib.PAGES_TABLE_FULL
    with pytest.raises(pkg.OdmkvError):
        cache.check()


def test_begin_grants_in_order(pkg, cuda):
    """Three free pages: sequence 0 needs two, 1 needs three, 2 needs one, 3 needs one: 0 and 2 go on."""
    cache, _ = make(pkg, 1, 4, 1, 16, 160, pages=3)
    cache.begin(torch.tensor([40, 48, 16, 17], dtype=torch.int32, device=cuda))
    assert cache.new_lens.tolist() == [40, 0, 16, 0]
    assert cache.table[:, 0].tolist() == [0, -1, 2, -1] and cache.table[0, 1] == 1
    assert int(cache.status) == pkg._lib.PAGES_EXHAUSTED
    assert cache.free_pages() == 0
    cache.begin(torch.tensor([8, 15, 15, 300], dtype=torch.int32, device=cuda))      # 48 tokens: a third page, and there is none
    assert cache.lens.tolist() == [40, 0, 16, 0] and cache.new_lens.tolist() == [0, 15, 15, 0]
    assert int(cache.status) == pkg._lib.PAGES_EXHAUSTED | pkg._lib.PAGES_TABLE_FULL


def test_begin_over_many_sequences_and_pages(pkg, cuda):
    """More sequences and pages than one pass of the block holds; lowest free page first."""
    N, page, pages = 1500, 16, 9000
    cache, _ = make(pkg, 1, N, 1, page, 96, pages=pages)
    g = torch.Generator().manual_seed(8)
    busy = torch.rand(pages, generator=g) < 0.3
    cache.refs.copy_(busy.to(torch.int32))
    new = torch.randint(0, 90, (N,), generator=g, dtype=torch.int32)
    cache.begin(new.cuda())
    need = (new // page).long()
    assert int(need.sum()) < int((~busy).sum())
    free = torch.nonzero(~busy).view(-1)
    want = torch.full((N, cache.width), -1, dtype=torch.int64)
    at = 0
    for n in range(N):
        want[n, : need[n]] = free[at: at + need[n]]
        at += int(need[n])
    assert torch.equal(cache.table.cpu().long(), want)
    refs = busy.to(torch.int32)
    refs[free[:at]] = 1
    assert torch.equal(cache.refs.cpu(), refs) and torch.equal(cache.new_lens.cpu(), new)
    cache.check()


@pytest.mark.parametrize("W", [1, 2, 4, 5, 8, 16, 32])
def test_fork_any_parents(pkg, cuda, W):
    """Permutations, cycles, one parent for all; then the beams grow apart and are forked again."""
    g = torch.Generator().manual_seed(W)
    B = 2
    N = B * W
    cache, ref = make(pkg, 2, N, 2, 16, 120)
    step(cache, ref, g, [17 + (5 * n) % 23 for n in range(N)])
    for r in range(4):
        if r == 0:
            parents = torch.stack([torch.randperm(W, generator=g) for _ in range(B)])
        elif r == 1:
            parents = torch.full((B, W), W - 1)
        else:
            parents = torch.randint(0, W, (B, W), generator=g)
        cache.fork(parents.cuda())
        ref.fork(parents)
        check_cache(cache, ref)
        step(cache, ref, g, [(7 * n + r) % 19 for n in range(N)])
        check_cache(cache, ref)
    q = torch.randn(N, 4, 18, D, generator=g).to(torch.bfloat16).cuda()
    got = cache.attention(0, q)
    for n in range(N):
        q[n, :, ref.new[n]:] = 0
    check_attention(got, None, ref.attention(0, q))
    cache.check()
    cache.free(torch.ones(N, dtype=torch.bool, device=cuda))
    assert cache.free_pages() == cache.num_pages


def test_fork_leaves_unused_slots_and_reports_bad_parents(pkg, cuda):
    g = torch.Generator().manual_seed(4)
    cache, ref = make(pkg, 1, 4, 1, 16, 64)
    step(cache, ref, g, [3, 9, 20, 0])
    before = cache.k_tail.clone()
    parents = torch.tensor([[1, 1], [0, 0]])
    cache.fork(parents.cuda())
    ref.fork(parents)
    check_cache(cache, ref)
    assert torch.equal(cache.k_tail[0, 0, :, 9:], before[0, 0, :, 9:]) and torch.equal(cache.k_tail[0, 3, :, 4:], before[0, 3, :, 4:])
    cache.fork(torch.tensor([[-1, 2], [0, 1]], device=cuda))            # outside: the beam itself
    check_cache(cache, ref)
    assert int(cache.status) == pkg._lib.PAGES_BAD_PARENT
    with pytest.raises(pkg.OdmkvError, match="parent"):
        cache.check()


def test_free_and_admit(pkg, cuda):
    g = torch.Generator().manual_seed(6)
    cache, ref = make(pkg, 1, 4, 2, 16, 100, pages=14)
    step(cache, ref, g, [50, 50, 33, 0])
    cache.fork(torch.tensor([[0, 0], [0, 1]], device=cuda))
    ref.fork(torch.tensor([[0, 0], [0, 1]]))
    check_cache(cache, ref)
    leave = torch.tensor([True, False, True, False], device=cuda)
    cache.free(leave)
    ref.free(leave.tolist())
    check_cache(cache, ref)
    cache.free(leave)                                                   # twice: nothing more to give
    check_cache(cache, ref)
    step(cache, ref, g, [64, 1, 0, 40])
    check_cache(cache, ref)
    cache.check()


def test_compact(pkg, cuda):
    g = torch.Generator().manual_seed(7)
    cache, ref = make(pkg, 2, 6, 2, 16, 120, pages=60)
    step(cache, ref, g, [100, 40, 119, 5, 64, 16])
    cache.fork(torch.tensor([[0, 0, 2], [0, 1, 2]], device=cuda))
    ref.fork(torch.tensor([[0, 0, 2], [0, 1, 2]]))
    leave = torch.tensor([False, False, True, True, False, True], device=cuda)
    cache.free(leave)
    ref.free(leave.tolist())
    order = torch.unique(cache.table[cache.table >= 0])
    moved = cache.compact()
    assert moved.num_pages == order.numel() and moved.free_pages() == 0
    check_cache(moved, ref)
    assert torch.equal(moved.k_codes.view(torch.uint8), cache.k_codes.view(torch.uint8)[:, order.long()])
    # into a larger pool with tensors of its own, and back to work
    other, _ = make(pkg, 2, 6, 2, 16, 120, pages=80)
    keep = other.k_codes.view(torch.uint8)[:, order.numel():].fill_(3).clone()
    moved.compact_into(other)
    check_cache(other, ref)
    assert torch.equal(other.k_codes.view(torch.uint8)[:, order.numel():], keep)
    step(other, ref, g, [10, 20, 30, 40, 50, 60])
    check_cache(other, ref)
    # too small: refused, and empty
    small, _ = make(pkg, 2, 6, 2, 16, 120, pages=order.numel() - 1)
    cache.compact_into(small)
    assert int(small.status) == pkg._lib.PAGES_POOL_SMALL and small.lens.tolist() == [0] * 6
    assert bool((small.table == -1).all()) and small.free_pages() == small.num_pages
    with pytest.raises(ValueError):
        cache.compact(order.numel() - 1)


# ------------------------------------------------------------------ beam selection

def beam_reference(logits, scores, K, done=None, pad=0):
    """In fp64 on the CPU; equal scores by the lower index."""
    B, W, V = logits.shape
    top = torch.finfo(logits.dtype).max
    x = logits.double().cpu()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x.clamp_max(top))
    s = scores.double().cpu()
    out = []
    for b in range(B):
        cand = []
        for w in range(W):
            if done is not None and bool(done[b, w]):
                row = torch.full((V,), -math.inf, dtype=torch.float64)
                row[pad] = s[b, w]
            elif bool((x[b, w] == -math.inf).all()):
                row = torch.full((V,), -math.inf, dtype=torch.float64)
            else:
                row = s[b, w] + (x[b, w] - torch.logsumexp(x[b, w], 0))
            cand.append(row)
        flat = torch.cat(cand).nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf)
        val, at = torch.sort(flat, descending=True, stable=True)
        out.append((val[:K], at[:K] // V, at[:K] % V))
    return [torch.stack(t) for t in zip(*out)]


def check_beam(pkg, logits, scores, K, done=None, pad=0):
    best, parents, toks = pkg.ops.beam_select(logits, scores, K, done=done, pad_token=pad)
    w_best, w_parents, w_toks = beam_reference(logits, scores, K, done, pad)
    assert torch.equal(parents.cpu(), w_parents) and torch.equal(toks.cpu(), w_toks)
    finite = torch.isfinite(w_best)
    assert torch.equal(torch.isfinite(best.cpu()), finite)
    # one rounding to fp32 of a value within 1e-12
    assert bool(((best.cpu().double() - w_best).abs()[finite] <= w_best.abs()[finite] * 2.0 ** -24 + 1e-11).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,W,V,K", [(1, 1, 1, 1), (1, 4, 7, 28), (3, 2, 100, 4), (2, 4, 32000, 4), (1, 1, 5003, 64), (2, 3, 40001, 33),
                                     (5, 8, 2048, 16), (1, 16, 152064, 32), (1, 1024, 50, 4), (2, 700, 9, 64), (1, 3, 70001, 64)])
def test_beam_select(pkg, cuda, dtype, B, W, V, K):
    g = torch.Generator().manual_seed(V)
    logits = (torch.randn(B, W, V, generator=g) * 3).to(dtype).cuda()
    scores = (-torch.rand(B, W, generator=g) * 5).cuda()
    check_beam(pkg, logits, scores, K)
    done = (torch.rand(B, W, generator=g) < 0.4).cuda()
    check_beam(pkg, logits, scores, K, done, pad=V - 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [999, 4096, 20001])
def test_beam_select_ties(pkg, cuda, dtype, V):
    """Equal logits, equal beams (rows at different alignments), all logits equal, ascending and descending rows."""
    g = torch.Generator().manual_seed(1)
    row = torch.randint(-4, 5, (V,), generator=g).to(dtype)
    logits = row.expand(2, 5, V).contiguous().cuda()
    check_beam(pkg, logits, torch.zeros(2, 5, device=cuda), 20)
    check_beam(pkg, torch.zeros(2, 5, V, dtype=dtype, device=cuda), torch.zeros(2, 5, device=cuda), 64)
    up = (torch.arange(V) / 64.0).to(dtype).expand(1, 3, V).contiguous().cuda()
    check_beam(pkg, up, torch.tensor([[0.0, -1.0, 2.0]], device=cuda), 40)
    check_beam(pkg, up.flip(-1).contiguous(), torch.tensor([[0.0, -1.0, 2.0]], device=cuda), 40)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_beam_select_masks(pkg, cuda, dtype):
    """-inf and the type's lowest value as masks, rows without a token, NaN, +inf, unused beams, fewer continuations than K."""
    g = torch.Generator().manual_seed(2)
    V = 700
    x = torch.randn(4, 4, V, generator=g)
    x[0, 0] = -math.inf
    x[0, 1, 5:] = -math.inf
    x[1, 0] = torch.finfo(dtype).min
    x[1, 1, ::2] = torch.finfo(dtype).min
    x[1, 2] = torch.finfo(dtype).max
    x[2, 0, 3], x[2, 1, 9], x[2, 2] = math.nan, math.inf, math.nan
    x[3] = -math.inf
    x[3, 1, 17] = 0.5
    scores = torch.tensor([[0.0, -1.0, -2.0, -0.5]] * 4)
    scores[2, 3] = -math.inf
    check_beam(pkg, x.to(dtype).cuda(), scores.cuda(), 8)
    first = torch.full((4, 4), -math.inf)
    first[:, 0] = 0.0                                                  # the first step of a search
    check_beam(pkg, x.to(dtype).cuda(), first.cuda(), 8)
    check_beam(pkg, x.to(dtype).cuda(), torch.full((4, 4), -math.inf, device=cuda), 8)
    check_beam(pkg, x.to(dtype).cuda(), scores.cuda(), 8, torch.ones(4, 4, dtype=torch.bool, device=cuda), pad=3)


def test_beam_select_wide_values(pkg, cuda):
    """Logits hundreds and thousands apart, the largest last or first: the sum's reference moves with them."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 3, 9000, generator=g) * 400
    x[0, 0] = torch.linspace(-3000, 3000, 9000)
    x[0, 1] = torch.linspace(3000, -3000, 9000)
    check_beam(pkg, x.cuda(), torch.zeros(2, 3, device=cuda), 12)


def test_beam_select_close_scores(pkg, cuda):
    """Beams whose continuations differ by 1e-9 at scores of -50: closer than fp32 can tell."""
    V = 4000
    x = torch.zeros(1, 2, V)
    x[0, 0, 7] = x[0, 1, 9] = 3.0
    x[0, 1, 100:140] = 2.0 ** -20                                      # raises beam 1's normaliser by 40 * 2^-20 / (V + 19)
    scores = torch.tensor([[-50.0, -50.0]])
    _, parents, toks = pkg.ops.beam_select(x.cuda(), scores.cuda(), 2)
    assert parents.tolist() == [[0, 1]] and toks.tolist() == [[7, 9]]
    _, parents, _ = pkg.ops.beam_select(x.flip(1).contiguous().cuda(), scores.cuda(), 2)
    assert parents.tolist() == [[1, 0]]


def test_beam_select_strides(pkg, cuda):
    """The last position of a model's output, and a transposed batch."""
    g = torch.Generator().manual_seed(5)
    full = torch.randn(6, 3, 1001, generator=g).to(torch.bfloat16).cuda()
    check_beam(pkg, full[:, -1].view(2, 3, 1001), torch.zeros(2, 3, device=cuda), 5)
    check_beam(pkg, full.transpose(0, 1), torch.zeros(3, 6, device=cuda), 5)
    check_beam(pkg, full[:, :, 1:].transpose(1, 2)[:, :, :2].transpose(1, 2), torch.zeros(6, 2, device=cuda), 5)
    check_beam(pkg, full[:, :, ::2], torch.zeros(6, 3, device=cuda), 5)


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("fmt,page", [("e4m3", 16), ("int8", 32)])
def test_beam_search_over_the_cache(pkg, cuda, fmt, page):
    """A beam search of a small random model (keys, values and logits are functions of the token): prompt, steps with selection
    and reordering, a sequence that ends and another that takes its place, a move into another pool."""
    g = torch.Generator().manual_seed(31)
    L, B, W, H, G, V = 2, 2, 3, 2, 2, 50
    N = B * W
    dtype = torch.bfloat16
    emb = [[torch.randn(V, H, D, generator=g).to(dtype).cuda() for _ in range(2)] for _ in range(L)]
    qs = torch.randn(L, V, H * G, D, generator=g).to(dtype).cuda()
    head = (torch.randn(D, V, generator=g) * 2).cuda()
    cache, ref = make(pkg, L, N, H, page, 150, fmt, dtype, pages=N * (150 // page + 1))
    prompt = torch.randint(0, V, (B, 37), generator=g).repeat_interleave(W, 0).cuda()

    def forward(ids, new):
        cache.begin(torch.tensor(new, dtype=torch.int32, device=cuda))
        ref.begin(new)
        for layer in range(L):
            k, v = (e[ids].transpose(1, 2).contiguous() for e in emb[layer])
            cache.append(layer, k, v)
            ref.append(layer, k, v)
            q = qs[layer][ids].transpose(1, 2).contiguous()
            out = cache.attention(layer, q)
            for n in range(N):
                q[n, :, new[n]:] = 0
            check_attention(out, None, ref.attention(layer, q))
        return (out[:, 0, -1].float() @ head).view(B, W, V)

    logits = forward(prompt, [37] * N)
    scores = torch.full((B, W), -math.inf, device=cuda)
    scores[:, 0] = 0.0
    for t in range(12):
        w_best, w_parents, w_toks = beam_reference(logits, scores, W)
        scores, parents, toks = pkg.ops.beam_select(logits, scores)
        assert torch.equal(parents.cpu(), w_parents) and torch.equal(toks.cpu(), w_toks)
        cache.fork(parents)
        ref.fork(w_parents)
        check_cache(cache, ref)
        if t == 6:                                                     # the second search ends, a new prompt takes its place
            leave = torch.tensor([False] * W + [True] * W, device=cuda)
            cache.free(leave)
            ref.free(leave.tolist())
            ids = torch.zeros(N, 21, dtype=torch.int64, device=cuda)
            ids[:W, 0] = toks[0]
            ids[W:] = torch.randint(0, V, (1, 21), generator=g).cuda()
            forward(ids, [1] * W + [21] * W)
            scores[1] = -math.inf
            scores[1, 0] = 0.0
            logits = torch.randn(B, W, V, generator=g).cuda()
        else:
            logits = forward(toks.view(N, 1), [1] * N)
        if t == 8:
            cache = cache.compact(cache.num_pages)
            check_cache(cache, ref)
    cache.check()


# ------------------------------------------------------------------ refusals

def test_refusals(pkg, cuda):
    cache, _ = make(pkg, 2, 4, 2, 16, 64)
    z = torch.zeros(4, 2, 3, D, dtype=torch.bfloat16, device=cuda)
    for bad in (lambda: cache.append(2, z, z), lambda: cache.append(-1, z, z), lambda: cache.append(0, z, z[:, :, :2]),
                lambda: cache.append(0, z[:3], z[:3]), lambda: cache.append(0, z.half(), z.half()), lambda: cache.append(0, z[:, :1], z[:, :1]),
                lambda: cache.attention(2, z), lambda: cache.attention(0, z[:, :1]), lambda: cache.attention(0, z.half()),
                lambda: cache.attention(0, z[:3]), lambda: cache.attention(0, z, softcap=-1.0), lambda: cache.attention(0, z, softcap=math.nan),
                lambda: cache.attention(0, z, slopes=torch.zeros(3, device=cuda)), lambda: cache.attention(0, z[..., :64]),
                lambda: cache.attention(0, z, slopes=torch.zeros(2, dtype=torch.float64, device=cuda)),
                lambda: cache.begin(-1), lambda: cache.begin(torch.zeros(4, dtype=torch.int64, device=cuda)),
                lambda: cache.begin(torch.zeros(3, dtype=torch.int32, device=cuda)),
                lambda: cache.fork(torch.zeros(2, 2, dtype=torch.int32, device=cuda)), lambda: cache.fork(torch.zeros(3, 1, dtype=torch.int64, device=cuda)),
                lambda: cache.free(torch.zeros(4, dtype=torch.uint8, device=cuda)), lambda: cache.free(torch.zeros(5, dtype=torch.bool, device=cuda)),
                lambda: cache.compact_into(cache), lambda: cache.compact_into(make(pkg, 2, 4, 2, 32, 64)[0]),
                lambda: cache.compact_into(make(pkg, 2, 4, 2, 16, 64, "int8")[0])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(pkg.OdmkvError):
        cache.append(0, z.cpu(), z.cpu())
    with pytest.raises(pkg.OdmkvError):
        cache.begin(torch.zeros(4, dtype=torch.int32))
    x, s = torch.zeros(2, 3, 10, device=cuda), torch.zeros(2, 3, device=cuda)
    for bad in (lambda: pkg.ops.beam_select(x, s, 0), lambda: pkg.ops.beam_select(x, s, 31), lambda: pkg.ops.beam_select(x[0], s),
                lambda: pkg.ops.beam_select(x, s[:1]), lambda: pkg.ops.beam_select(x, s.double()), lambda: pkg.ops.beam_select(x.double(), s),
                lambda: pkg.ops.beam_select(x, s, pad_token=10), lambda: pkg.ops.beam_select(x, s, done=s),
                lambda: pkg.ops.beam_select(torch.zeros(1, 2, 100, device=cuda), s[:1, :2], 65)):
        with pytest.raises(ValueError):
            bad()
    cache.append(0, z[:, :, :0], z[:, :, :0])                            # no tokens: nothing to do
    assert cache.attention(0, z[:, :, :0]).shape == (4, 2, 0, D)
    cache.check()
