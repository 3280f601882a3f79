"""Paged 8-bit cache: refusals at the ends of the ranges, before anything is launched (no GPU)."""
import pytest
import torch

from test_block_cache_host import calls, struct


def test_shared_lengths_need_a_pool_that_cannot_refuse(pkg):
    import ctypes
    c, other = struct(pkg, pages=8), struct(pkg, pages=7)
    for i, name in enumerate(("k_codes", "v_codes", "k_scale", "v_scale", "table", "refs")):
        setattr(other, name, 0x100000 * (i + 1))
    L, ws = pkg._lib.lib(), ctypes.c_void_p(0x1000)
    assert L.odmkv_pages_compact(ctypes.byref(c), ctypes.byref(other), ws, 1 << 30, None) == -1
    other.pages = 8                                                        # (what comes next in the call: its workspace)
    assert L.odmkv_pages_compact(ctypes.byref(c), ctypes.byref(other), None, 0, None) == -3
    assert calls(pkg, c)["compact"](other, n=8) == -3


@pytest.mark.parametrize("change", [dict(N=4096, width=1 << 19, page=16), dict(N=2, width=(1 << 30) - 1, page=16), dict(N=1, width=0x7fffffff),
                                    dict(N=1, width=0x7fffffff, page=16), dict(N=3000, width=800000)])
def test_counts_stay_in_32_bits(pkg, change):
    """Sums of pages over the sequences, and positions: a table that could overflow them is refused."""
    c = calls(pkg, struct(pkg, **change))
    for name in ("append", "attn", "fork", "free", "begin", "compact"):
        if name != "fork" or change["N"] % 2 == 0:
            assert c[name]() == -5, name
    assert calls(pkg, struct(pkg, N=4096, width=(1 << 19) - 1, page=16))["begin"](lens=None, every=-1) == -2      # just within


def test_cache_refuses_such_tables(pkg):
    def meta(shape, dtype):
        return torch.empty(shape, dtype=dtype, device="meta")

    codes, scale, tail = meta((1, 8, 1, 16, 128), torch.int8), meta((1, 8, 1), torch.float32), meta((1, 4096, 1, 16, 128), torch.float16)
    table, lens, refs = meta((4096, 1 << 19), torch.int32), meta((4096,), torch.int32), meta((8,), torch.int32)
    with pytest.raises(ValueError, match="32 bits"):
        pkg.BlockKVCache(codes, codes, scale, scale, tail, tail, table, lens, lens, refs)
