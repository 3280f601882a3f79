"""The operators of a paged 8-bit key/value cache, as they are measured.

A cache holds, per layer, pages of ``page`` tokens x H heads x 128 coordinates in 8 bits (e4m3 or int8) with one
power-of-two scale per page and head, and the tokens behind the last full page of every sequence in 16 bits (the
"tail").  Four kinds of work go over it: appending tokens, attention, turning pages over (fork, free, admit, compact)
and a beam search's selection, whose parents the fork takes.

``run`` computes each in elementary torch operations, or with ``own`` through the package's operators.
"""
import math

import torch

own = False

D = 128
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


# --------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one decode step of a serving batch: every sequence gets one token, a few complete a page
        dict(name="append_step", kind="append", N=64, H=8, T=1, ctx=1024, page=64, dtype="bf16", fmt="e4m3", ragged=True),
        # admission of four prompts of different lengths
        dict(name="append_prompt", kind="append", N=4, H=8, T=16384, ctx=0, page=64, dtype="bf16", fmt="int8", ragged=True),
        # one chat at its beginning, one token: the latency of a call
        dict(name="attn_step_short", kind="attn", N=1, H=8, G=4, Tq=1, ctx=611, page=64, dtype="fp16", fmt="e4m3", softcap=0.0,
             slopes=False, ragged=False),
        # a serving batch of chats from one token to 8192, seven query heads to a key head, capped scores
        dict(name="attn_step_ragged", kind="attn", N=64, H=4, G=7, Tq=1, ctx=8192, page=32, dtype="bf16", fmt="int8", softcap=30.0,
             slopes=False, ragged=True),
        # eight long documents, one token each
        dict(name="attn_step_long", kind="attn", N=8, H=8, G=4, Tq=1, ctx=131072, page=64, dtype="bf16", fmt="e4m3", softcap=0.0,
             slopes=False, ragged=False),
        # a short question to each of four documents, distance-biased scores
        dict(name="attn_question", kind="attn", N=4, H=8, G=4, Tq=37, ctx=32768, page=64, dtype="bf16", fmt="e4m3", softcap=0.0,
             slopes=True, ragged=True),
        # one chunk of a long prompt over what the cache holds of it already
        dict(name="attn_chunk", kind="attn", N=1, H=8, G=4, Tq=1024, ctx=32768, page=64, dtype="bf16", fmt="e4m3", softcap=0.0,
             slopes=False, ragged=False),
        # a beam search's reordering over the 32 layers of a model: four searches of four beams
        dict(name="fork_beams", kind="fork", L=32, B=4, W=4, H=8, ctx=4096, page=64, dtype="bf16", fmt="e4m3"),
        # a scheduler's turn: some sequences end, others take their places and pages
        dict(name="turnover", kind="turnover", N=256, H=1, ctx=8192, page=64, dtype="bf16", fmt="e4m3"),
        # a pool that is about half empty moves into a new one, its pages side by side
        dict(name="compact_pool", kind="compact", L=4, N=32, H=8, ctx=4096, page=64, dtype="bf16", fmt="e4m3"),
        # one search of four beams
        dict(name="beam_one", kind="beam", B=1, W=4, K=4, V=32000, dtype="fp32", done=False),
        # sixteen searches of eight beams, some of them finished, twice as many candidates as beams
        dict(name="beam_batch", kind="beam", B=16, W=8, K=16, V=128256, dtype="bf16", done=True),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["append", "append", "attn", "attn", "attn", "attn", "fork", "turnover", "compact", "beam", "beam"])
    page, dtype, fmt = rng.choice([16, 32, 64, 128]), rng.choice(["bf16", "fp16"]), rng.choice(["e4m3", "int8"])
    if kind == "append":
        if rng.random() < 0.5:
            return dict(kind=kind, N=log(1, 128), H=rng.choice([1, 2, 4, 8]), T=1, ctx=log(1, 1024), page=page, dtype=dtype, fmt=fmt,
                        ragged=True)
        N = log(1, 16)
        return dict(kind=kind, N=N, H=rng.choice([1, 2, 4, 8]), T=log(1, max(2, 65536 // N)), ctx=0, page=page, dtype=dtype, fmt=fmt,
                    ragged=rng.random() < 0.5)
    if kind == "attn":
        H, G = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16])
        if rng.random() < 0.6:
            N, Tq = log(1, 128), 1
            ctx = log(1, max(2, min(131072, 8 * 8 * 131072 // (N * H))))
        else:
            N, Tq = log(1, 8), log(2, 512)
            ctx = log(1, max(2, min(32768, 1024 * 32 * 32768 // (N * H * G * Tq))))
        return dict(kind=kind, N=N, H=H, G=G, Tq=Tq, ctx=ctx, page=page, dtype=dtype, fmt=fmt,
                    softcap=rng.choice([0.0, 0.0, 30.0, 50.0]), slopes=rng.random() < 0.3, ragged=rng.random() < 0.7)
    if kind == "fork":
        L, B, W = log(1, 32), log(1, 8), rng.choice([2, 3, 4, 5, 8])
        return dict(kind=kind, L=L, B=min(B, max(1, 16 // W)), W=W, H=rng.choice([1, 2, 4, 8]), ctx=log(1, 4096), page=page, dtype=dtype,
                    fmt=fmt)
    if kind == "turnover":
        return dict(kind=kind, N=log(1, 256), H=1, ctx=log(1, 8192), page=rng.choice([64, 128]), dtype=dtype, fmt=fmt)
    if kind == "compact":
        return dict(kind=kind, L=log(1, 4), N=log(1, 32), H=rng.choice([1, 2, 4, 8]), ctx=log(16, 4096), page=page, dtype=dtype, fmt=fmt)
    B, W, V = log(1, 16), rng.choice([1, 2, 3, 4, 5, 8]), log(100, 128256)
    return dict(kind=kind, B=B, W=W, K=W * rng.choice([1, 2]), V=V, dtype=rng.choice(["bf16", "fp16", "fp32"]), done=rng.random() < 0.5)


# --------------------------------------------------------------------------------------------- inputs

def _rng(case, seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 17)


def _tokens(g, *shape, keys):
    """Keys with four channels ten times as large as the others, as models have them; values without."""
    x = torch.randn(*shape, D, generator=g, device="cuda")
    if keys:
        x[..., 5::32] *= 10.0
    return x


def _scale(amax, fmt):
    """The smallest power of two s (at least 2^-126) with amax <= top * s; 1 where all is zero."""
    m, e = torch.frexp(amax)
    top, bits = (0.875, 9) if fmt == "e4m3" else (127.0 / 128.0, 7)
    e = (e - bits + (m > top)).clamp_min(-126)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e), torch.ones_like(amax))


def _encode(x, fmt):
    """x [..., page, 128] in 32 bits -> codes, scale [...]"""
    s = _scale(x.abs().amax(dim=(-2, -1)), fmt)
    y = x / s[..., None, None]
    return (y if fmt == "e4m3" else torch.round(y)).to(CODES[fmt]), s


def _pool(case, g, L, pages, filled=True):
    """Pages with tokens in them (or empty ones): codes [L, pages, H, page, 128] and scales [L, pages, H]."""
    H, P, fmt = case["H"], case["page"], case["fmt"]
    out = []
    for keys in (True, False):
        if filled:
            c = torch.empty(L, pages, H, P, D, dtype=CODES[fmt], device="cuda")
            s = torch.empty(L, pages, H, device="cuda")
            for layer in range(L):
                c[layer], s[layer] = _encode(_tokens(g, pages, H, P, keys=keys), fmt)
        else:
            c = torch.zeros(L, pages, H, P, D, dtype=torch.uint8, device="cuda").view(CODES[fmt])
            s = torch.ones(L, pages, H, device="cuda")
        out.append((c, s))
    return out


def _lengths(case, g, N, ragged, low=1):
    ctx = case["ctx"]
    if not ragged or ctx <= low:
        return torch.full((N,), ctx, dtype=torch.int64, device="cuda")
    u = torch.rand(N, generator=g, device="cuda")
    lens = (low + u * (ctx - low + 1)).floor().clamp(low, ctx).to(torch.int64)
    lens[0] = ctx
    return lens


def _state(case, g, L, N, lens, new, most, spare=0, filled=True):
    """A cache of N sequences of up to ``most`` tokens that hold lens committed and new running ones; the pages lie in
    the pool in any order."""
    P, H, dt = case["page"], case["H"], DTYPES[case["dtype"]]
    need = (lens + new) // P
    width = max(1, most // P)
    pages = N * width + spare
    order = torch.randperm(pages, generator=g, device="cuda")
    slot = torch.arange(width, device="cuda")[None, :]
    start = torch.cumsum(need, 0) - need
    held = slot < need[:, None]
    table = torch.where(held, order[(start[:, None] + slot).clamp_max(pages - 1)], -torch.ones_like(order[:1]))
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[order[: int(need.sum())]] = 1
    (kc, ks), (vc, vs) = _pool(case, g, L, pages, filled)
    st = dict(k_codes=kc, v_codes=vc, k_scale=ks, v_scale=vs, table=table.to(torch.int32), lens=lens.to(torch.int32),
              new_lens=new.to(torch.int32), refs=refs)
    there = (torch.arange(P, device="cuda")[None, :] < ((lens + new) % P)[:, None])[None, :, None, :, None]
    for name, keys in (("k_tail", True), ("v_tail", False)):
        st[name] = (_tokens(g, L, N, H, P, keys=keys) * there).to(dt)
    return st


def prepare(case, seed):
    g = _rng(case, seed)
    kind = case["kind"]
    st = dict(case=dict(case))
    if kind == "append":
        N, H, T, P, dt = case["N"], case["H"], case["T"], case["page"], DTYPES[case["dtype"]]
        if T == 1:
            lens = _lengths(case, g, N, True) - 1
            ends = lens // P * P + P - 1
            sel = (torch.arange(N, device="cuda") % 7 == 0) & (ends < case["ctx"])
            lens = torch.where(sel, ends, lens)               # these complete a page
            new = torch.ones_like(lens)
        else:
            lens = torch.zeros(N, dtype=torch.int64, device="cuda")
            new = _lengths(dict(ctx=T), g, N, case["ragged"])
        st.update(_state(case, g, 1, N, lens, new, case["ctx"] if T == 1 else T, filled=False))
        old = (torch.arange(P, device="cuda")[None, :] < (lens % P)[:, None])[None, :, None, :, None]
        st["k_tail"] = (_tokens(g, 1, N, H, P, keys=True) * old).to(dt)
        st["v_tail"] = (_tokens(g, 1, N, H, P, keys=False) * old).to(dt)
        st["k"], st["v"] = _tokens(g, N, H, T, keys=True).to(dt), _tokens(g, N, H, T, keys=False).to(dt)
        blocks = int(((lens % P + new) // P).max())
        done = torch.arange(blocks, device="cuda")[None, :] < ((lens % P + new) // P)[:, None]
        st["blocks"], st["completed"] = blocks, done.nonzero()       # the (sequence, block) pairs that this call completes
    elif kind == "attn":
        N, H, Tq = case["N"], case["H"], case["Tq"]
        total = _lengths(case, g, N, case["ragged"])
        if Tq == 1:
            lens, new = total - 1, torch.ones_like(total)
        else:
            lens = total
            new = _lengths(dict(ctx=Tq), g, N, case["ragged"])
        st.update(_state(case, g, 1, N, lens, new, case["ctx"] + (Tq if Tq > 1 else 0)))
        st["q"] = torch.randn(N, H * case["G"], Tq, D, generator=g, device="cuda").to(DTYPES[case["dtype"]])
        Hq = H * case["G"]
        st["slopes"] = torch.exp2(-8.0 * torch.arange(1, Hq + 1, device="cuda") / Hq) if case["slopes"] else None
    elif kind == "fork":
        B, W = case["B"], case["W"]
        lens = _lengths(case, g, B, True).repeat_interleave(W)
        st.update(_state(case, g, case["L"], B * W, lens, torch.zeros_like(lens), case["ctx"]))
        # the beams of a search share all pages but the last few
        P = case["page"]
        full = (lens // P).view(B, W)[:, :1]
        col = torch.arange(st["table"].shape[1], device="cuda")
        t = st["table"].view(B, W, -1)
        t.copy_(torch.where((col < full - 2)[:, None, :], t[:, :1], t))
        held = t.reshape(-1)
        st["refs"].zero_().index_add_(0, held.clamp_min(0).long(), (held >= 0).to(torch.int32))
        # surviving beams stay in their places, the others become copies of one of them
        stay = torch.rand(B, W, generator=g, device="cuda") < 0.5
        stay[torch.arange(B, device="cuda"), torch.randint(W, (B,), generator=g, device="cuda")] = True
        pick = (torch.rand(B, W, W, generator=g, device="cuda") * stay[:, None, :]).argmax(-1)
        st["parents"] = torch.where(stay, torch.arange(W, device="cuda")[None, :], pick)
    elif kind == "turnover":
        N, P = case["N"], case["page"]
        lens = _lengths(case, g, N, True)
        st.update(_state(dict(case, H=1), g, 1, N, lens, torch.zeros_like(lens), case["ctx"], spare=N, filled=False))
        leave = torch.rand(N, generator=g, device="cuda") < 0.25
        leave[0] = True
        st["leave"] = leave
        st["admit"] = (torch.rand(N, generator=g, device="cuda") * (lens + 1)).floor().to(torch.int32) * leave
    elif kind == "compact":
        N, L, P = case["N"], case["L"], case["page"]
        lens = _lengths(case, g, N, True)
        st.update(_state(case, g, L, N, lens, torch.zeros_like(lens), case["ctx"]))
        pages = st["refs"].shape[0]
        (kc, ks), (vc, vs) = _pool(case, g, L, pages, filled=False)
        st["into"] = dict(k_codes=kc, v_codes=vc, k_scale=ks, v_scale=vs, table=torch.empty_like(st["table"]),
                          refs=torch.empty(pages, dtype=torch.int32, device="cuda"))
    else:
        B, W, V = case["B"], case["W"], case["V"]
        x = torch.randn(B, W, V, generator=g, device="cuda") * 2.5
        x[..., : max(1, V // 100)] += 3.0                                # frequent tokens
        st["logits"] = x.to(DTYPES[case["dtype"]])
        st["scores"] = -40.0 * torch.rand(B, W, generator=g, device="cuda") ** 2 * 0.25
        st["done"] = torch.rand(B, W, generator=g, device="cuda") < 0.2 if case["done"] else None
    return st


# --------------------------------------------------------------------------------------------- plain forms

def _plain_append(st):
    case = st["case"]
    P, fmt, nb = case["page"], case["fmt"], st["blocks"]
    lens, new, table = st["lens"].long(), st["new_lens"].long(), st["table"].long()
    o = lens % P
    last = (o + new) // P                                                # pages completed
    pos = torch.arange((nb + 1) * P, device="cuda")[None, :]
    where = torch.where(pos < o[:, None], pos, P + pos - o[:, None]).clamp_max(P + case["T"] - 1)
    n, b = st["completed"].unbind(1)
    slot = torch.arange(P, device="cuda")[None, :]
    fresh = slot < ((o + new) % P)[:, None]
    out = {}
    for x in ("k", "v"):
        both = torch.cat([st[x + "_tail"][0], st[x]], dim=2)
        seq = both.gather(2, where[:, None, :, None].expand(-1, both.shape[1], -1, D))
        codes, s = _encode(seq[:, :, : nb * P].unflatten(2, (nb, P)).float(), fmt)
        page = table[n, lens[n] // P + b]
        st[x + "_codes"][0].view(torch.uint8).index_copy_(0, page, codes.view(torch.uint8)[n, :, b])
        st[x + "_scale"][0].index_copy_(0, page, s[n, :, b])
        tail = seq.gather(2, (last[:, None] * P + slot)[:, None, :, None].expand(-1, both.shape[1], -1, D))
        st[x + "_tail"][0].copy_(torch.where(fresh[:, None, :, None], tail, st[x + "_tail"][0]))
        out.update({x + "_codes": st[x + "_codes"], x + "_scale": st[x + "_scale"], x + "_tail": st[x + "_tail"]})
    return out


def _plain_attn(st):
    case = st["case"]
    N, H, G, Tq, P = case["N"], case["H"], case["G"], case["Tq"], case["page"]
    lens, new, table = st["lens"].long(), st["new_lens"].long(), st["table"].long()
    full = (lens + new) // P
    slot, col = torch.arange(P, device="cuda")[None, :], torch.arange(table.shape[1] * P, device="cuda")[None, :]
    kpos = torch.cat([col.expand(N, -1), full[:, None] * P + slot], dim=1)
    there = torch.cat([col < (full * P)[:, None], slot < ((lens + new) % P)[:, None]], dim=1)
    qpos = lens[:, None] + torch.arange(Tq, device="cuda")[None, :]
    real = torch.arange(Tq, device="cuda")[None, :] < new[:, None]
    seen = there[:, None, :] & (kpos[:, None, :] <= qpos[:, :, None]) & real[:, :, None]

    def dense(x):
        pages = st[x + "_codes"][0][table.clamp_min(0)].float() * st[x + "_scale"][0][table.clamp_min(0)][..., None, None]
        return torch.cat([pages.transpose(1, 2).flatten(2, 3), st[x + "_tail"][0].float()], dim=2)      # [N, H, keys, 128]

    q = st["q"].float().view(N, H, G * Tq, D)
    s = ((q @ dense("k").transpose(2, 3)) * (D ** -0.5)).view(N, H, G, Tq, -1)
    if case["softcap"]:
        s = case["softcap"] * torch.tanh(s / case["softcap"])
    if st["slopes"] is not None:
        far = (kpos[:, None, :] - qpos[:, :, None]).float()
        s = s + st["slopes"].view(1, H, G, 1, 1) * far[:, None, None]
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    e = torch.exp(s - top)
    w = e.sum(-1, keepdim=True)
    p = e / torch.where(w > 0, w, torch.ones_like(w))
    return (p.view(N, H, G * Tq, -1) @ dense("v")).view(N, H * G, Tq, D).to(st["q"].dtype)


def _plain_fork(st):
    case = st["case"]
    B, W, P, L = case["B"], case["W"], case["page"], case["L"]
    src = (torch.arange(B, device="cuda")[:, None] * W + st["parents"]).view(-1)
    for x in ("table", "lens", "new_lens"):
        st[x].copy_(st[x][src])
    held = st["table"].reshape(-1)
    st["refs"].zero_().index_add_(0, held.clamp_min(0).long(), (held >= 0).to(torch.int32))
    keep = torch.arange(P, device="cuda")[None, :] < ((st["lens"] + st["new_lens"]) % P)[:, None]
    for x in ("k_tail", "v_tail"):
        st[x].copy_(torch.where(keep[None, :, None, :, None], st[x][:, src], st[x]))
    return {x: st[x] for x in ("table", "lens", "new_lens", "refs", "k_tail", "v_tail")}


def _plain_turnover(st):
    P, leave, admit = st["case"]["page"], st["leave"], st["admit"]
    table, refs, lens, new = st["table"], st["refs"], st["lens"], st["new_lens"]
    held = table.reshape(-1)
    given = ((table >= 0) & leave[:, None]).reshape(-1).to(torch.int32)
    refs.index_add_(0, held.clamp_min(0).long(), -given)
    table.masked_fill_(leave[:, None], -1)
    lens.copy_(torch.where(leave, torch.zeros_like(lens), lens + new))
    new.copy_(admit)
    first, need = lens // P, (lens + admit) // P - lens // P
    start = torch.cumsum(need, 0) - need
    free = torch.argsort((refs > 0).to(torch.uint8), stable=True)       # free pages, lowest first
    col = torch.arange(table.shape[1], device="cuda")[None, :]
    take = (col >= first[:, None]) & (col < (first + need)[:, None])
    page = free[(start[:, None] + col - first[:, None]).clamp(0, refs.shape[0] - 1)]
    table.copy_(torch.where(take, page.to(torch.int32), table))
    rank = torch.empty_like(free).index_copy_(0, free, torch.arange(free.shape[0], device="cuda"))
    refs.copy_(torch.where((refs == 0) & (rank < need.sum()), torch.ones_like(refs), refs))
    return {"table": table, "refs": refs, "lens": lens, "new_lens": new}


def _plain_compact(st):
    into, live = st["into"], st["refs"] > 0
    pages = into["refs"].shape[0]
    order = torch.argsort((~live).to(torch.uint8), stable=True)[:pages]
    full = torch.arange(pages, device="cuda") < live.sum()
    for x in ("k_codes", "v_codes"):
        a, b = into[x].view(torch.uint8), st[x].view(torch.uint8)
        a.copy_(torch.where(full[None, :, None, None, None], b[:, order], a))
    for x in ("k_scale", "v_scale"):
        into[x].copy_(torch.where(full[None, :, None], st[x][:, order], into[x]))
    rank = torch.cumsum(live, 0) - 1
    t = st["table"]
    into["table"].copy_(torch.where(t >= 0, rank[t.clamp_min(0).long()].to(torch.int32), t))
    into["refs"].copy_(torch.where(full, st["refs"][order], torch.zeros_like(into["refs"])))
    return dict(into)


def _plain_beam(st):
    case = st["case"]
    B, W, V, K = case["B"], case["W"], case["V"], case["K"]
    x = st["logits"].double()                      # candidates of different beams can be closer than 32 bits tell apart
    top = x.amax(-1, keepdim=True)
    s = st["scores"].double()[..., None] + (x - top) - torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    if st["done"] is not None:                     # a finished beam goes on as itself, with the padding token 0
        first = torch.arange(V, device="cuda") == 0
        s = torch.where(st["done"][..., None], torch.where(first, st["scores"].double()[..., None], -math.inf), s)
    best, at = torch.sort(s.view(B, W * V), dim=-1, descending=True, stable=True)
    return {"scores": best[:, :K].float(), "parents": at[:, :K] // V, "tokens": at[:, :K] % V}


# --------------------------------------------------------------------------------------------- the package's operators

def _package():
    import importlib
    return importlib.import_module("odm-kv_b200")


def _handle(st):
    """The cache object that a program keeps beside its tensors."""
    if "handle" not in st:
        cls = _package().block_cache.BlockKVCache
        names = ("k_codes", "v_codes", "k_scale", "v_scale", "k_tail", "v_tail", "table", "lens", "new_lens", "refs")
        st["handle"] = cls(**{x: st[x] for x in names})
        if "into" in st:
            shared = {x: st[x] for x in ("k_tail", "v_tail", "lens", "new_lens")}
            st["into_handle"] = cls(**st["into"], **shared)
    return st["handle"]


def _own(st):
    case = st["case"]
    if case["kind"] == "beam":
        best, parents, tokens = _package().ops.beam_select(st["logits"], st["scores"], case["K"], done=st["done"])
        return {"scores": best, "parents": parents, "tokens": tokens}
    cache = _handle(st)
    if case["kind"] == "append":
        cache.append(0, st["k"], st["v"])
        return {x: st[x] for x in ("k_codes", "k_scale", "k_tail", "v_codes", "v_scale", "v_tail")}
    if case["kind"] == "attn":
        return cache.attention(0, st["q"], softcap=case["softcap"], slopes=st["slopes"])
    if case["kind"] == "fork":
        cache.fork(st["parents"])
        return {x: st[x] for x in ("table", "lens", "new_lens", "refs", "k_tail", "v_tail")}
    if case["kind"] == "turnover":
        cache.free(st["leave"])
        cache.begin(st["admit"])
        return {x: st[x] for x in ("table", "refs", "lens", "new_lens")}
    cache.compact_into(st["into_handle"])
    return dict(st["into"])


def run(state):
    if own:
        return _own(state)
    plain = dict(append=_plain_append, attn=_plain_attn, fork=_plain_fork, turnover=_plain_turnover, compact=_plain_compact,
                 beam=_plain_beam)
    return plain[state["case"]["kind"]](state)


# --------------------------------------------------------------------------------------------- work

def work(case):
    kind = case["kind"]
    if kind == "beam":
        size = 4 if case["dtype"] == "fp32" else 2
        live = 0.8 if case["done"] else 1.0
        n = case["B"] * case["W"] * case["V"] * live
        return {"bytes": n * size + case["B"] * (case["W"] * 4 + case["K"] * 20), "flops": 4 * n}
    P = case["page"]
    mean = 0.5 if case.get("ragged", True) else 1.0
    if kind == "append":
        vals = 2 * case["N"] * case["H"] * D
        if case["T"] == 1:      # a token in and into its tail; one sequence in seven reads its tail and writes a page
            return {"bytes": vals * (4 + (2 * P + P) / 7), "flops": 3 * vals * P / 7}
        tokens = case["T"] * mean
        return {"bytes": vals * tokens * 3, "flops": 3 * vals * tokens}
    if kind == "attn":
        keys = case["N"] * case["ctx"] * mean + case["N"] * (case["Tq"] * mean if case["Tq"] > 1 else 0)
        rows = case["G"] * (case["Tq"] * mean if case["Tq"] > 1 else 1)
        tail = case["N"] * P / 2
        q = case["N"] * case["H"] * case["G"] * case["Tq"] * D * 2
        pairs = (case["ctx"] * mean + (case["Tq"] * mean / 2 if case["Tq"] > 1 else 0)) * case["N"] * case["H"] * rows
        return {"bytes": 2 * case["H"] * D * (keys + 2 * tail) + 2 * q, "flops": 4 * D * pairs}
    if kind == "fork":
        # about half of the beams are written, from half as many that are read; half of the slots of a tail are in use
        N = case["B"] * case["W"]
        tail = 2 * case["L"] * case["H"] * D * 2 * P / 2
        table = 4 * N * (case["ctx"] / P / 2 + 2)
        return {"bytes": tail * (N / 2 + N / 4) + 2 * table, "flops": N}
    if kind == "turnover":
        pages = case["N"] * (case["ctx"] / P / 2 + 1)
        return {"bytes": 4 * pages + 4 * pages / 4 * 4 + 16 * case["N"], "flops": pages}
    pages = case["N"] * case["ctx"] / P / 2
    return {"bytes": pages * (2 * 2 * case["L"] * case["H"] * (P * D + 4) + 24), "flops": pages}


# --------------------------------------------------------------------------------------------- in 64 bits

def _exact_codes(x, fmt):
    """x [..., page, 128] in 64 bits -> the values of the codes, and the scale, by their definition."""
    amax = x.abs().amax(dim=(-2, -1))
    top = 448.0 if fmt == "e4m3" else 127.0
    e = torch.ceil(torch.log2(torch.where(amax > 0, amax, torch.full_like(amax, top)) / top))
    e = torch.where(amax > top * torch.exp2(e), e + 1, e)
    e = torch.where(amax <= top * torch.exp2(e - 1), e - 1, e).clamp_min(-126)
    s = torch.where(amax > 0, torch.exp2(e), torch.ones_like(e))
    y = x / s[..., None, None]
    if fmt == "int8":
        return torch.round(y), s
    a = y.abs()
    binade = torch.floor(torch.log2(torch.where(a > 0, a, torch.ones_like(a)))).clamp_min(-6)
    binade = torch.where(torch.exp2(binade) > a, (binade - 1).clamp_min(-6), binade)
    step = torch.exp2(binade - 3)
    return torch.round(y / step) * step, s


def exact(case, seed):
    kind = case["kind"]
    if kind in ("fork", "turnover", "compact"):
        return None                                   # whole numbers and copies
    st = prepare(case, seed)
    if kind == "beam":
        s = torch.log_softmax(st["logits"].double(), dim=-1) + st["scores"].double()[..., None]
        if st["done"] is not None:
            s[st["done"]] = -math.inf
            s[..., 0] = torch.where(st["done"], st["scores"].double(), s[..., 0])
        flat = s.flatten(1)
        got = [sorted(((-float(v), int(i)) for v, i in zip(*torch.topk(row, min(4 * case["K"], row.numel()))))) for row in flat]
        at = torch.tensor([[i for _, i in r[: case["K"]]] for r in got], device="cuda")
        return {"scores": flat.gather(1, at), "parents": at // case["V"], "tokens": at % case["V"]}
    P, N, fmt = case["page"], case["N"], case["fmt"]
    if kind == "append":
        out = {}
        for x in ("k", "v"):
            codes, scale = st[x + "_codes"].double(), st[x + "_scale"].double()
            tail = st[x + "_tail"].double()
            for n in range(N):
                have, more = int(st["lens"][n]), int(st["new_lens"][n])
                o = have % P
                seq = torch.cat([tail[0, n, :, :o], st[x][n, :, :more].double()], dim=1)
                blocks = seq.shape[1] // P
                if blocks:
                    c, s = _exact_codes(seq[:, : blocks * P].unflatten(1, (blocks, P)), fmt)
                    page = st["table"][n, have // P: have // P + blocks].long()
                    codes[0, page], scale[0, page] = c.transpose(0, 1), s.transpose(0, 1)
                rest = seq[:, blocks * P:]
                tail[0, n, :, : rest.shape[1]] = rest
            out.update({x + "_codes": codes if fmt == "e4m3" else codes.to(torch.int8), x + "_scale": scale, x + "_tail": tail})
        return out
    H, G, Tq = case["H"], case["G"], case["Tq"]
    out = torch.zeros(N, H * G, Tq, D, dtype=torch.float64, device="cuda")
    for n in range(N):
        have, more = int(st["lens"][n]), int(st["new_lens"][n])
        blocks, rest = (have + more) // P, (have + more) % P
        page = st["table"][n, :blocks].long()
        for h in range(H):
            k, v = (torch.cat([(st[x + "_codes"][0, page, h].double() * st[x + "_scale"][0, page, h].double()[:, None, None]).reshape(-1, D),
                               st[x + "_tail"][0, n, h, :rest].double()]) for x in ("k", "v"))
            far = torch.arange(have + more, device="cuda")[None, :] - (have + torch.arange(more, device="cuda"))[:, None]
            for g in range(h * G, (h + 1) * G):
                s = st["q"][n, g, :more].double() @ k.T / math.sqrt(D)
                if case["softcap"]:
                    s = case["softcap"] * torch.tanh(s / case["softcap"])
                if st["slopes"] is not None:
                    s = s + st["slopes"][g].double() * far
                out[n, g, :more] = torch.softmax(s.masked_fill(far > 0, -math.inf), dim=-1) @ v
    return out
