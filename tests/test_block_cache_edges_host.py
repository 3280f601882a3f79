"""Paged 8-bit cache: refusals at the ends of the ranges, before anything is launched (no GPU)."""
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
