"""Paged 8-bit cache and beam selection at the ends of their ranges.

Bounds as in ``test_block_cache_gpu.py``: an output is rounded once to its type; an error d of the scores (2^-16 of the sum of
|q k| scale, of the bias, and 2^-19 of a capped score) moves a weight by at most 2 d of itself; weights enter with fp16's half step.
Where values of very different sizes meet (``page`` given): a weight enters as w = p s / max(p s), or up to 2^15 times that, s its page's
scale (the tile kernel takes the largest scale of 128 tokens, at most 2^10 times the page's, for a lift of 2^10), in fp16 whose smallest
step is 2^-24, so w is off by up to 2^-25 beside its half step; times the code, at most 2 max|v| / s: 2^-24 max(p max|v|) for each token
that the row sees, max|v| the largest of the token's page (of the token itself in the tail).
"""
import math

import pytest
import torch

from test_block_cache_gpu import D, HALF, check_attention, check_beam, make, step, tokens

pytestmark = pytest.mark.gpu


def reference(stored, new, q, softcap=0.0, page=0, slopes=None):
    """(want, bound, lse, lse_bound) in fp64; no term of the bound grows with the cap or with keys that a row does not see."""
    N, Hq, Tq, _ = q.shape
    want = torch.zeros(N, Hq, Tq, D, dtype=torch.float64, device=q.device)
    bound, lse = torch.zeros_like(want), torch.full((N, Hq, Tq), -math.inf, dtype=torch.float64, device=q.device)
    lse_bound = torch.zeros_like(lse)
    for n in range(N):
        K, V = (t.to(q.device) for t in stored[n])
        H, total = K.shape[0], K.shape[1]
        if not new[n]:
            continue
        qn = q[n, :, : new[n]].double().view(H, Hq // H, -1, D)
        hidden = torch.arange(total, device=q.device)[None, :] > (total - new[n] + torch.arange(new[n], device=q.device))[:, None]
        s = torch.einsum("hgtd,hkd->hgtk", qn, K) * D ** -0.5
        mags = torch.einsum("hgtd,hkd->hgtk", qn.abs(), K.abs()) * D ** -0.5
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        if slopes is not None:                                             # two roundings of the bias and one of the sum: 2^-21 of it
            far = torch.arange(total, device=q.device)[None, :] - (total - new[n] + torch.arange(new[n], device=q.device))[:, None]
            bias = slopes.double().view(H, -1, 1, 1) * far
            s, mags = s + bias, mags + bias.abs() * 2.0 ** (16 - 21)
        s, mags = s.masked_fill(hidden, -math.inf), mags.masked_fill(hidden, 0)
        d = mags.amax(-1) * (2.0 ** -16 + 2.0 ** -19) + 2.0 ** -20
        p = torch.softmax(s, -1)
        rows = slice(0, new[n])
        low = 0.0
        if page:
            amax, full = V.abs().amax(-1), total // page * page
            amax[:, :full] = amax[:, :full].unflatten(1, (-1, page)).amax(-1).repeat_interleave(page, 1)
            low = ((p * amax[:, None, None]).amax(-1) * (~hidden).sum(-1) * 2.0 ** -24)[..., None].expand(*p.shape[:3], D).reshape(Hq, -1, D)
        want[n, :, rows] = torch.einsum("hgtk,hkd->hgtd", p, V).reshape(Hq, -1, D)
        spread = torch.einsum("hgtk,hkd->hgtd", p, V.abs())
        bound[n, :, rows] = ((2 * d + 2.0 ** -11)[..., None] * spread).reshape(Hq, -1, D) + HALF[q.dtype] * want[n, :, rows].abs() + low
        lse[n, :, rows] = torch.logsumexp(s, -1).reshape(Hq, -1)
        lse_bound[n, :, rows] = (d + 2.0 ** -20 * (1 + torch.logsumexp(s, -1).abs())).reshape(Hq, -1)
    return want, bound + (2.0 ** -25 if q.dtype == torch.float16 else 2.0 ** -134), lse, lse_bound


def filled(pkg, page, fmt, dtype, k, v, running):
    """A cache of one layer that holds k, v [N, H, T, 128], the last ``running`` tokens running."""
    N, H, T, _ = k.shape
    cache, ref = make(pkg, 1, N, H, page, T + 1, fmt, dtype)
    for lo, hi in ((0, T - running), (T - running, T)):
        if hi > lo:
            cache.begin(hi - lo), ref.begin([hi - lo] * N)
            cache.append(0, k[:, :, lo:hi], v[:, :, lo:hi]), ref.append(0, k[:, :, lo:hi], v[:, :, lo:hi])
    return cache, ref


# ------------------------------------------------------------------ large caps

@pytest.mark.parametrize("cap", [1e-40, 0.5, 30.0, 1e3, 1e5, 1e7, 1e9, 1e30])
@pytest.mark.parametrize("rows", [8, 80])                              # the step and the tile kernel
@pytest.mark.parametrize("fmt,dtype", [("e4m3", torch.bfloat16), ("int8", torch.float16)])
def test_caps_of_any_size(pkg, cuda, cap, rows, fmt, dtype):
    g = torch.Generator().manual_seed(rows)
    T = 150
    k, v = tokens(g, 1, 2, T, dtype=dtype, keys=True), tokens(g, 1, 2, T, dtype=dtype, keys=False)
    cache, ref = filled(pkg, 32, fmt, dtype, k, v, rows // 4)
    q = torch.randn(1, 8, rows // 4, D, generator=g).to(dtype).cuda()
    out, lse = cache.attention(0, q, softcap=cap, return_lse=True)
    check_attention(out, lse, reference([ref.stored(0, 0)], ref.new, q, cap), cap)


# ------------------------------------------------------------------ scores and scales far apart

@pytest.mark.parametrize("heads", [1, 4])
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_scores_near_the_lowest_number(pkg, cuda, heads, fmt):
    """Equal scores of -1e35: the mean of the values, as with any other equal scores."""
    g = torch.Generator().manual_seed(4)
    k = torch.full((1, 1, 100, D), -2.0 ** 55).bfloat16().cuda()
    v = tokens(g, 1, 1, 100, dtype=torch.bfloat16, keys=False)
    cache, ref = filled(pkg, 64, fmt, torch.bfloat16, k, v, 20)
    q = torch.full((1, heads, 20, D), 2.0 ** 58).bfloat16().cuda()
    out, lse = cache.attention(0, q, return_lse=True)
    values = ref.stored(0, 0)[1][0].cuda()
    for j in range(20):
        seen = values[: 81 + j]
        want, spread = seen.mean(0), seen.abs().mean(0)
        bound = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -18) * spread
        assert bool(((out[0, :, j].double() - want).abs() <= bound).all()), j
    assert bool((lse < -1e34).all()) and bool(torch.isfinite(lse).all())


@pytest.mark.parametrize("heads", [1, 4])
@pytest.mark.parametrize("page", [16, 128])
def test_scores_near_the_largest_number(pkg, cuda, heads, page):
    """Scores of 2^120 to 2^122, exact, from keys of 2^118 to 2^120: the mean of the values whose score is the largest."""
    g = torch.Generator().manual_seed(15)
    T = 100
    k = torch.zeros(1, 1, T, D)
    k[0, 0, :, 0] = 2.0 ** torch.randint(118, 121, (T,), generator=g).float()
    k[0, 0, :, 1] = 2.0 ** 119
    v = torch.randn(1, 1, T, D, generator=g).bfloat16().cuda()
    cache, ref = filled(pkg, page, "e4m3", torch.bfloat16, k.bfloat16().cuda(), v, 20)
    q = torch.zeros(1, heads, 20, D)
    q[..., 0], q[..., 1] = 4.0, -4.0                                        # (-2^121 everywhere)
    out = cache.attention(0, q.bfloat16().cuda(), scale=1.0)
    keys, values = (t[0].cuda() for t in ref.stored(0, 0))
    for j in range(20):
        seen = slice(0, T - 19 + j)
        of = values[seen][keys[seen, 0] == keys[seen, 0].max()]
        bound = 2.0 ** -8 * of.mean(0).abs() + (2.0 ** -11 + 2.0 ** -18) * of.abs().mean(0)
        assert bool(((out[0, :, j].double() - of.mean(0)).abs() <= bound).all()), j


@pytest.mark.parametrize("heads", [1, 4])
@pytest.mark.parametrize("size", [2.0 ** -30, 1.0, 2.0 ** 30])
def test_scores_beside_which_a_scale_is_nothing(pkg, cuda, heads, size):
    """Scores of 2^30 to 2^32, exact and equal or far apart: the mean of the values whose score is the largest."""
    g = torch.Generator().manual_seed(5)
    T = 300
    k = torch.zeros(1, 1, T, D)
    k[0, 0, :, 0] = 2.0 ** torch.randint(14, 17, (T,), generator=g).float()
    v = (torch.randn(1, 1, T, D, generator=g) * size).bfloat16().cuda()
    cache, ref = filled(pkg, 16, "e4m3", torch.bfloat16, k.bfloat16().cuda(), v, 30)
    q = torch.zeros(1, heads, 30, D)
    q[..., 0] = 2.0 ** 16
    out = cache.attention(0, q.bfloat16().cuda(), scale=1.0)
    keys, values = (t[0].cuda() for t in ref.stored(0, 0))
    for j in range(30):
        seen = slice(0, T - 29 + j)
        of = values[seen][keys[seen, 0] == keys[seen, 0].max()]
        bound = 2.0 ** -8 * of.mean(0).abs() + (2.0 ** -11 + 2.0 ** -18) * of.abs().mean(0)
        assert bool(((out[0, :, j].double() - of.mean(0)).abs() <= bound).all()), j


@pytest.mark.parametrize("heads", [1, 4])
@pytest.mark.parametrize("small,large,gap", [(2.0 ** -110, 2.0 ** 30, 140.0), (2.0 ** -118, 2.0 ** 120, 0.0), (2.0 ** -118, 2.0 ** 120, 60.0),
                                             (2.0 ** 120, 2.0 ** -118, 0.0), (2.0 ** 30, 2.0 ** -110, 140.0), (2.0 ** -118, 1.0, 110.0)])
def test_values_at_both_ends_of_the_type(pkg, cuda, heads, small, large, gap):
    """Half of the tokens ``small``, the other half ``large`` and ``gap`` powers of two below in their weights: finite, and right;
    enough sequences that a warp goes over both."""
    g = torch.Generator().manual_seed(3)
    N, T, new = 24, 2048, 10
    k, v = torch.zeros(N, 1, T, D), torch.randn(N, 1, T, D, generator=g)
    k[:, 0, :1024, 0] = gap * math.log(2.0) * D ** 0.5 / 8.0
    v[:, 0, :1024] *= small
    v[:, 0, 1024:] *= large
    cache, ref = filled(pkg, 128, "e4m3", torch.bfloat16, k.bfloat16().cuda(), v.bfloat16().cuda(), new)
    q = torch.zeros(N, heads, new, D)
    q[..., 0] = 8.0
    q = q.bfloat16().cuda()
    out, lse = cache.attention(0, q, return_lse=True)
    check_attention(out, lse, reference([ref.stored(0, n) for n in range(N)], ref.new, q))


@pytest.mark.parametrize("page,fmt", [(16, "e4m3"), (64, "int8"), (128, "e4m3")])
@pytest.mark.parametrize("heads", [1, 4])                              # up to 32 rows, and more
@pytest.mark.parametrize("side", ["k", "v", "both"])
@pytest.mark.parametrize("size", [2.0 ** 22, 2.0 ** 40, 2.0 ** 100, 2.0 ** -30, 2.0 ** -100])
def test_later_tokens_of_another_size(pkg, cuda, page, fmt, heads, side, size):
    """Tokens whose keys or values are far larger or smaller than their neighbours': rows in front of them (of their page, where
    they share one) do not notice."""
    g = torch.Generator().manual_seed(page + heads)
    dtype, T = torch.bfloat16, 2 * 128 + 100
    k, v = tokens(g, 1, 1, T, dtype=dtype, keys=False), tokens(g, 1, 1, T, dtype=dtype, keys=False)
    for at in (slice(128 + 64, 128 + 80), slice(2 * 128 + 90, 2 * 128 + 93)):
        if side != "v":
            k[:, :, at] *= size
        if side != "k":
            v[:, :, at] *= size
    new = 30 if heads == 1 else 200
    cache, ref = filled(pkg, page, fmt, dtype, k, v, new)
    q = torch.randn(1, heads, new, D, generator=g).to(dtype).cuda()
    out, lse = cache.attention(0, q, return_lse=True)
    check_attention(out, lse, reference([ref.stored(0, 0)], ref.new, q, page=page), (page, size))


@pytest.mark.parametrize("heads", [1, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_lowest_value_in_a_later_token(pkg, cuda, heads, dtype):
    """The type's lowest and largest values in a running token: the rows in front of it are as without it."""
    g = torch.Generator().manual_seed(heads)
    new = 30
    k, v = tokens(g, 1, 1, 60, dtype=dtype, keys=False), tokens(g, 1, 1, 60, dtype=dtype, keys=False)
    k[0, 0, 50], v[0, 0, 50] = torch.finfo(dtype).max, torch.finfo(dtype).min
    cache, ref = filled(pkg, 128, "e4m3", dtype, k, v, new)
    q = torch.randn(1, heads, new, D, generator=g).to(dtype).cuda()
    out = cache.attention(0, q)[:, :, :20]
    keys, values = ref.stored(0, 0)
    want, bound, _, _ = reference([(keys[:, :50], values[:, :50])], [20], q[:, :, :20])
    assert bool(((out.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("heads", [1, 4])
@pytest.mark.parametrize("page", [16, 32])
@pytest.mark.parametrize("apart", [9, 14, 19, 30])
def test_many_small_weights_beside_large_pages(pkg, cuda, heads, page, apart):
    """One token with 2^16 times the weight of each other, which together weigh as much, and in every 128 tokens a page of values
    2^apart times as large that hardly counts: the others keep their share."""
    g = torch.Generator().manual_seed(6)
    T, new = 40000, 10
    k, v = torch.zeros(1, 1, T, D), torch.randn(1, 1, T, D, generator=g) + 1.0
    unit = math.log(2.0) * D ** 0.5 / 8.0                                  # a score of one power of two
    large = torch.arange(T) % 128 // page == 1
    k[0, 0, large, 0] = -80.0 * unit
    v[0, 0, large] *= 2.0 ** apart
    k[0, 0, 5, 0] = 15.0 * unit
    cache, ref = filled(pkg, page, "e4m3", torch.bfloat16, k.bfloat16().cuda(), v.bfloat16().cuda(), new)
    q = torch.zeros(1, heads, new, D)
    q[..., 0] = 8.0
    q = q.bfloat16().cuda()
    out, lse = cache.attention(0, q, return_lse=True)
    check_attention(out, lse, reference([ref.stored(0, 0)], ref.new, q, page=page))


@pytest.mark.parametrize("heads", [1, 4])
def test_negative_scores_before_the_largest_key(pkg, cuda, heads):
    """Rows whose scores are all equal and negative, in front of a key of the type's largest value: the mean of the values."""
    g = torch.Generator().manual_seed(19)
    new = 30
    k, v = torch.full((1, 1, 60, D), -1.0), torch.randn(1, 1, 60, D, generator=g)
    k[0, 0, 55] = torch.finfo(torch.bfloat16).max
    cache, ref = filled(pkg, 128, "e4m3", torch.bfloat16, k.bfloat16().cuda(), v.bfloat16().cuda(), new)
    out = cache.attention(0, torch.full((1, heads, new, D), 8.0, dtype=torch.bfloat16, device=cuda))
    values = ref.stored(0, 0)[1][0].cuda()
    for j in range(25):
        seen = values[: 31 + j]
        bound = 2.0 ** -8 * seen.mean(0).abs() + (2.0 ** -11 + 2.0 ** -18) * seen.abs().mean(0)
        assert bool(((out[0, :, j].double() - seen.mean(0)).abs() <= bound).all()), j


@pytest.mark.parametrize("heads", [1, 4])
@pytest.mark.parametrize("fmt,page", [("e4m3", 16), ("int8", 64), ("e4m3", 128)])
@pytest.mark.parametrize("size", [2.0 ** -25, 2.0 ** -40, 2.0 ** -100])
def test_zeros_among_tiny_values(pkg, cuda, heads, fmt, page, size):
    """Zeros (of either sign) have a scale of 1, which does not count beside smaller ones: in single pages, in whole blocks, in the tail."""
    g = torch.Generator().manual_seed(9)
    N, T, new = 16, 1500, 30
    k = tokens(g, N, 1, T, dtype=torch.bfloat16, keys=False)
    v = (torch.randn(N, 1, T, D, generator=g) * size).bfloat16().cuda()
    zero = torch.arange(T, device=cuda)
    zero = (zero // page % 5 == 3) | (zero // 128 % 4 == 1) | (zero > T - 20)
    v = torch.where(zero[:, None], -torch.zeros_like(v), v)
    cache, ref = filled(pkg, page, fmt, torch.bfloat16, k, v, new)
    q = torch.randn(N, heads, new, D, generator=g).to(torch.bfloat16).cuda()
    out, lse = cache.attention(0, q, return_lse=True)
    check_attention(out, lse, reference([ref.stored(0, n) for n in range(N)], ref.new, q))


@pytest.mark.parametrize("page,fmt", [(64, "e4m3"), (16, "int8"), (32, "e4m3")])
@pytest.mark.parametrize("large", [2.0 ** 90, 2.0 ** 20, 2.0 ** -60])
def test_zeros_in_front_of_larger_tokens(pkg, cuda, page, fmt, large):
    """Rows that see zeros in a block whose later tokens, hidden from them, are far larger than all that they see: tile kernel."""
    g = torch.Generator().manual_seed(16)
    T, new = 224, 150
    k, v = tokens(g, 2, 1, T, dtype=torch.bfloat16, keys=False), tokens(g, 2, 1, T, dtype=torch.bfloat16, keys=False)
    v[:, :, :64] *= large * 2.0 ** -40
    v[:, :, 64:192] = 0
    v[0, :, 192:] *= large
    v[1, :, 192:208] = 0
    v[1, :, 208:] *= large
    cache, ref = filled(pkg, page, fmt, torch.bfloat16, k, v, new)
    q = torch.randn(2, 4, new, D, generator=g).to(torch.bfloat16).cuda()
    out, lse = cache.attention(0, q, return_lse=True)
    check_attention(out, lse, reference([ref.stored(0, n) for n in range(2)], ref.new, q, page=page))


@pytest.mark.parametrize("heads", [1, 4])
@pytest.mark.parametrize("page", [64, 128])
@pytest.mark.parametrize("dtype,usual,large", [(torch.bfloat16, 1.0, 2.0 ** 30), (torch.bfloat16, 2.0 ** -40, 2.0 ** 80),
                                               (torch.bfloat16, 2.0 ** -105, 2.0 ** 20), (torch.float16, 2.0 ** -11, 2.0 ** 13),
                                               (torch.float16, 1.0, 2.0 ** 12)])
def test_large_tokens_in_the_tail(pkg, cuda, heads, page, dtype, usual, large):
    """Running tokens in the tail whose values are far larger, hidden from the rows before them, or seen with next to no weight;
    enough sequences that a warp goes from the tail to several pages."""
    g = torch.Generator().manual_seed(18)
    N, T, new = 32, 1024 + 50, 30
    k = tokens(g, N, 1, T, dtype=dtype, keys=False)
    v = (torch.randn(N, 1, T, D, generator=g) * usual).to(dtype).cuda()
    v[:, :, T - 10] = large
    v[:, :, T - 40] = large * 2.0 ** -4
    k[:, :, T - 40, 0] = -300.0                                            # (hardly any weight)
    q = torch.randn(N, heads, new, D, generator=g)
    q[..., 0] = 8.0
    q = q.to(dtype).cuda()
    cache, ref = filled(pkg, page, "e4m3", dtype, k, v, new)
    out, lse = cache.attention(0, q, return_lse=True)
    check_attention(out, lse, reference([ref.stored(0, n) for n in range(N)], ref.new, q, page=page))


@pytest.mark.parametrize("page,fmt", [(16, "e4m3"), (64, "int8")])
@pytest.mark.parametrize("heads", [1, 4])
@pytest.mark.parametrize("cap,biased,scale", [(30.0, False, 1.0), (0.0, True, 1.0), (1e4, True, 1.0), (0.0, True, 2.0 ** 20)])
def test_cap_and_bias_beside_large_tokens(pkg, cuda, page, fmt, heads, cap, biased, scale):
    """The slower form of a step does all that the fast one does: caps, distance biases, scores of 2^20 and more."""
    g = torch.Generator().manual_seed(20)
    T, new = 300, 30 if heads == 1 else 170
    k, v = tokens(g, 2, 2, T, dtype=torch.bfloat16, keys=False), tokens(g, 2, 2, T, dtype=torch.bfloat16, keys=False)
    v[:, :, 160:176] *= 2.0 ** 30
    v[:, :, 290:] *= 2.0 ** -30
    k[:, :, 64:80] *= 2.0 ** -40
    cache, ref = filled(pkg, page, fmt, torch.bfloat16, k * scale, v, new)
    q = torch.randn(2, 2 * heads, new, D, generator=g).to(torch.bfloat16).cuda()
    slopes = torch.exp2(-torch.arange(1, 2 * heads + 1).float()).cuda() if biased else None
    out, lse = cache.attention(0, q, softcap=cap, slopes=slopes, return_lse=True)
    check_attention(out, lse, reference([ref.stored(0, n) for n in range(2)], ref.new, q, cap, page, slopes))


# ------------------------------------------------------------------ many sequences

@pytest.mark.parametrize("N,Tq", [(129, 1), (300, 1), (1500, 1), (129, 7), (449, 9), (700, 9)])
def test_more_sequences_than_threads(pkg, cuda, N, Tq):
    """Ragged, some long, many and whole runs of them without running tokens."""
    g = torch.Generator().manual_seed(N)
    cache, ref = make(pkg, 1, N, 1, 16, 1300, pages=N * 4 + 400)
    before = torch.randint(0, 50, (N,), generator=g)
    before[[3, N // 2, N - 1]] = torch.tensor([1000, 333, 1200])
    step(cache, ref, g, before.tolist())
    new = torch.randint(0, Tq + 1, (N,), generator=g)
    new[5:5 + 100] = 0
    if N > 400:
        new[128:256] = 0
    new[[3, N // 2, N - 1]] = Tq
    step(cache, ref, g, new.tolist())
    cache.check()
    q = torch.randn(N, 4, Tq, D, generator=g).to(torch.bfloat16).cuda()
    out, lse = cache.attention(0, q, return_lse=True)
    for n in range(N):
        q[n, :, ref.new[n]:] = 0
        assert bool((out[n, :, ref.new[n]:] == 0).all())
    check_attention(out, lse, reference([ref.stored(0, n) for n in range(N)], ref.new, q))


# ------------------------------------------------------------------ append

@pytest.mark.parametrize("T", [0, 10, 99])
def test_append_of_too_few_tokens(pkg, cuda, T):
    """The sequence whose step is longer than the tensors is left alone and reported; the others are stored."""
    g = torch.Generator().manual_seed(T)
    cache, ref = make(pkg, 1, 3, 2, 16, 200)
    step(cache, ref, g, [20, 7, 0])
    cache.begin(torch.tensor([100, min(T, 3), T], dtype=torch.int32, device=cuda))
    before = [getattr(cache, x).clone() for x in ("k_codes", "k_tail", "v_tail")]
    k, v = tokens(g, 3, 2, T, dtype=torch.bfloat16, keys=True), tokens(g, 3, 2, T, dtype=torch.bfloat16, keys=False)
    cache.append(0, k, v)
    mine = cache.table[0, :7].long()
    assert torch.equal(cache.k_codes.view(torch.uint8)[0, mine], before[0].view(torch.uint8)[0, mine])
    assert torch.equal(cache.k_tail[0, 0], before[1][0, 0]) and torch.equal(cache.v_tail[0, 0], before[2][0, 0])
    ref.begin([0, min(T, 3), T])
    ref.append(0, k, v)
    for n in (1, 2):
        for a, b in zip(cache.materialize(0, n), ref.stored(0, n)):
            assert torch.equal(a.double(), b.cuda())
    assert int(cache.status) == pkg._lib.APPEND_SHORT
    with pytest.raises(pkg.OdmkvError, match="fewer tokens"):
        cache.check()


# ------------------------------------------------------------------ pages

@pytest.mark.parametrize("live,room", [(6000, 5999), (6000, 4500), (4097, 4096), (130, 100), (9000, 1)])
def test_refused_compaction_of_large_pools(pkg, cuda, live, room):
    """More live pages than the new pool holds, spread over many warps and passes: the new cache is empty, every time."""
    g = torch.Generator().manual_seed(room)
    cache, _ = make(pkg, 1, 4, 1, 16, 16 * live, pages=live + 500)
    order = torch.randperm(live + 500, generator=g)[:live]
    cache.table[0, :live] = order.to(torch.int32).cuda()
    cache.refs[order.cuda()] = 1
    cache.lens[0] = 16 * live
    small, _ = make(pkg, 1, 4, 1, 16, 16 * live, pages=room)
    for _ in range(20):
        small.refs.fill_(7), small.table.fill_(3), small.lens.fill_(5), small.new_lens.fill_(1), small.status.zero_()
        cache.compact_into(small)
        assert int(small.status) == pkg._lib.PAGES_POOL_SMALL
        assert bool((small.refs == 0).all()) and bool((small.table == -1).all())
        assert small.lens.tolist() == [0] * 4 and small.new_lens.tolist() == [0] * 4
    assert int(cache.refs.sum()) == live and cache.lens.tolist() == [16 * live, 0, 0, 0]
    step_after = cache.compact(live)
    assert step_after.free_pages() == 0 and bool((step_after.refs == 1).all())


def test_compaction_with_shared_lengths(pkg, cuda):
    """A move that could be refused needs lengths of its own; ``compact`` makes them."""
    cache, _ = make(pkg, 1, 2, 1, 16, 64, pages=8)
    cache.begin(40)

    def pool(pages):
        other, _ = make(pkg, 1, 2, 1, 16, 64, pages=pages)
        names = ("k_codes", "v_codes", "k_scale", "v_scale", "table", "refs")
        return pkg.BlockKVCache(**{x: getattr(other, x) for x in names}, k_tail=cache.k_tail, v_tail=cache.v_tail, lens=cache.lens,
                                new_lens=cache.new_lens)

    with pytest.raises(ValueError):
        cache.compact_into(pool(7))
    same = pool(8)
    cache.compact_into(same)
    assert same.new_lens.tolist() == [40, 40] and same.table[:, :2].tolist() == [[0, 1], [2, 3]]
    moved = cache.compact()
    assert moved.num_pages == 4 and moved.new_lens.tolist() == [40, 40]
    moved.free(torch.ones(2, dtype=torch.bool, device=cuda))
    assert cache.new_lens.tolist() == [40, 40] and moved.new_lens.tolist() == [0, 0]


# ------------------------------------------------------------------ beam selection

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [37, 9000, 70001])
def test_zeros_of_either_sign_are_equal(pkg, cuda, dtype, V):
    g = torch.Generator().manual_seed(V)
    x = torch.randn(2, 4, V, generator=g).clamp_max(0.0)
    x = torch.where(torch.rand(2, 4, V, generator=g) < 0.3, -torch.zeros(()), x)
    x = torch.where(torch.rand(2, 4, V, generator=g) < 0.3, torch.zeros(()), x).to(dtype).cuda()
    scores = torch.zeros(2, 4, device=cuda)
    check_beam(pkg, x, scores, 20)
    check_beam(pkg, x[:, :1].expand(2, 4, V).contiguous(), scores, 33)
    # finished beams whose scores are zeros of either sign, beside continuations of score 0
    sure = torch.full((2, 4, V), -math.inf)
    sure[..., V // 2] = 0.0
    done = torch.tensor([[True, False, True, False], [False, True, False, True]], device=cuda)
    zeros = torch.tensor([[-0.0, 0.0, 0.0, -0.0], [0.0, 0.0, -0.0, -0.0]], device=cuda)
    check_beam(pkg, sure.to(dtype).cuda(), zeros, 3, done, pad=1)


@pytest.mark.parametrize("at", [(10, 20), (20, 10), (10, 69990), (69990, 10), (30000, 69990)])
def test_a_beams_own_order_is_that_of_its_logits(pkg, cuda, at):
    """Logits so close that the scores are equal as fp64 numbers, in one stretch of the row or in two: the larger logit first."""
    x = torch.full((1, 2, 70001), -30.0)
    x[0, 1, at[0]], x[0, 1, at[1]] = 2e-20, 1e-20
    x[0, 0, 5] = -1e-20
    for k in (1, 2, 3):
        _, parents, toks = pkg.ops.beam_select(x.cuda(), torch.tensor([[-60.0, -50.0]], device=cuda), k)
        assert parents.tolist()[0] == [1, 1, 0][:k] and toks.tolist()[0] == [at[0], at[1], 5][:k]
    # the first of them is the lower beam's where beams tie
    y = x[:, 1:].expand(1, 2, 70001).contiguous().cuda()
    _, parents, toks = pkg.ops.beam_select(y, torch.tensor([[-50.0, -50.0]], device=cuda), 4)
    assert parents.tolist() == [[0, 0, 1, 1]] and toks.tolist() == [[at[0], at[1], at[0], at[1]]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K", [1, 16, 32, 33, 64])
@pytest.mark.parametrize("B,W,V", [(16, 8, 40000), (2, 256, 9001), (2, 64, 128256)])
def test_rising_rows_over_many_passes(pkg, cuda, dtype, K, B, W, V):
    """Every pass over a stretch beats the bound of the one before: the lists are cut down again and again."""
    g = torch.Generator().manual_seed(K)
    up = torch.arange(V) / 8.0 if dtype == torch.float32 else torch.arange(V) // 64 / 4.0
    blocks = torch.arange(V) // 1000 * 3.0 + torch.randn(V, generator=g)
    scores = (torch.randn(B, W, generator=g) * 3).cuda()
    for row in (up, blocks, up // 100):
        x = (row.expand(B, W, V) * (torch.rand(B, W, 1, generator=g) + 0.5)).to(dtype).cuda()
        check_beam(pkg, x, scores, K)
