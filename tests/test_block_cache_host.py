"""Paged 8-bit cache and beam selection: what is refused before anything is launched (no GPU)."""
import ctypes

import pytest
import torch


def struct(pkg, **changes):
    """A cache description whose pointers are never followed: every call below is refused on the host."""
    c = pkg._lib.BlockCache()
    for name, _ in pkg._lib.BlockCache._fields_[:11]:
        setattr(c, name, 0x1000)
    c.L, c.N, c.H, c.page, c.pages, c.width, c.code_format, c.tail_dtype = 2, 4, 2, 64, 8, 4, 0, 1
    for name, value in changes.items():
        setattr(c, name, value)
    return c


def calls(pkg, c):
    L = pkg._lib.lib()
    r, p = ctypes.byref(c), ctypes.c_void_p(0x1000)
    st = (ctypes.c_int64 * 3)(1024, 512, 128)
    return {
        "append": lambda layer=0, k=p, strides=st, T=1: L.odmkv_block8_append(r, layer, k, p, strides, st, T, None),
        "attn": lambda layer=0, q=p, strides=st, G=4, Tq=1, cap=0.0, ws=p, n=1 << 40: L.odmkv_block8_attn(
            r, layer, q, strides, G, Tq, 1.0, cap, None, p, None, ws, n, None),
        "fork": lambda parents=p, W=2: L.odmkv_pages_fork(r, parents, W, None),
        "free": lambda leave=p: L.odmkv_pages_free(r, leave, None),
        "begin": lambda lens=p, every=0: L.odmkv_pages_begin(r, lens, every, None),
        "compact": lambda other=None, ws=p, n=1 << 30: L.odmkv_pages_compact(r, ctypes.byref(other or c), ws, n, None),
    }


@pytest.mark.parametrize("change,status", [(dict(page=48), -2), (dict(page=0), -2), (dict(N=0), -2), (dict(L=0), -2), (dict(H=-1), -2),
                                           (dict(pages=0), -2), (dict(width=0), -2), (dict(code_format=2), -4), (dict(tail_dtype=2), -4),
                                           (dict(N=8194), -5), (dict(H=40000), -5), (dict(width=1 << 30), -5), (dict(table=None), -1),
                                           (dict(status=None), -1), (dict(lens=None), -1), (dict(refs=None), -1)])
def test_bad_caches(pkg, change, status):
    c = calls(pkg, struct(pkg, **change))
    for name in ("append", "attn", "fork", "free", "begin", "compact"):
        assert c[name]() == status, name


def test_bad_arguments(pkg):
    c = calls(pkg, struct(pkg))
    odd = (ctypes.c_int64 * 3)(1024, 512, 130)
    off = ctypes.c_void_p(0x1002)
    assert c["append"](layer=2) == -2 and c["append"](layer=-1) == -2 and c["append"](T=-1) == -2
    assert c["append"](k=None) == -1 and c["append"](k=off) == -1 and c["append"](strides=odd) == -1
    assert c["attn"](layer=2) == -2 and c["attn"](G=0) == -2 and c["attn"](Tq=-1) == -2
    assert c["attn"](q=None) == -1 and c["attn"](q=off) == -1 and c["attn"](strides=odd) == -1
    assert c["attn"](cap=-1.0) == -1 and c["attn"](cap=float("nan")) == -1
    assert c["attn"](ws=None) == -3 and c["attn"](n=16) == -3 and c["attn"](ws=ctypes.c_void_p(0x1010)) == -3
    assert c["fork"](W=3) == -2 and c["fork"](W=0) == -2 and c["fork"](parents=None) == -1
    assert calls(pkg, struct(pkg, N=128))["fork"](W=64) == -5
    assert c["free"](leave=None) == -1 and c["begin"](lens=None, every=-1) == -2
    assert c["compact"]() == -1                                            # a cache into itself
    other = struct(pkg, pages=9)
    for i, (name, _) in enumerate(pkg._lib.BlockCache._fields_[:11]):
        setattr(other, name, 0x100000 * (i + 1))
    for name in ("L", "N", "H", "width"):
        bad = struct(pkg)
        ctypes.pointer(bad)[0] = other
        setattr(bad, name, getattr(other, name) * 2)
        assert c["compact"](bad) == -2, name
    assert c["compact"](other, n=8) == -3 and c["compact"](other, ws=None) == -3
    assert calls(pkg, struct(pkg, k_codes=None))["append"]() == -1


def test_beam_arguments(pkg):
    L = pkg._lib.lib()
    p, st = ctypes.c_void_p(0x1000), (ctypes.c_int64 * 2)(100, 10)

    def call(logits=p, dtype=0, B=1, W=2, V=10, K=2, pad=0, ws=p, n=1 << 30):
        return L.odmkv_beam_select(logits, dtype, st, p, None, B, W, V, K, pad, p, p, p, ws, n, None)

    assert call(logits=None) == -1 and call(dtype=3) == -4 and call(pad=10) == -1 and call(pad=-1) == -1
    assert call(B=0) == -2 and call(K=21) == -2 and call(V=100, K=65) == -5 and call(W=2000, V=10) == -5 and call(B=40000) == -5
    assert call(ws=None) == -3 and call(n=8) == -3
    assert L.odmkv_beam_select_workspace_bytes(1, 2, 10, 0) == 0
    assert L.odmkv_beam_select_workspace_bytes(1, 2, 10, 2) > 0


def test_cache_wants_the_gpu_and_right_tensors(pkg):
    with pytest.raises(pkg.OdmkvError):
        pkg.BlockKVCache.allocate(1, 2, 2, 8, 100, device="cpu")
    with pytest.raises(ValueError):
        pkg.BlockKVCache.allocate(1, 2, 2, 8, 100, fmt="e5m2", device="cpu")
    with pytest.raises(ValueError):
        pkg.BlockKVCache.allocate(1, 2, 2, 8, 100, page=48, device="cpu")
    with pytest.raises(ValueError):
        pkg.BlockKVCache.allocate(1, 9000, 2, 8, 100, device="cpu")
    with pytest.raises(pkg.OdmkvError):
        pkg.ops.beam_select(torch.zeros(1, 2, 10), torch.zeros(1, 2))


def test_struct_mirror(pkg):
    assert ctypes.sizeof(pkg._lib.BlockCache) == 11 * 8 + 8 * 4
