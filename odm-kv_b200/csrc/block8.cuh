// Paged 8-bit cache: what its kernels share (block8_append.cu, block8_attn.cu, pages.cu).
#pragma once
#include "common.cuh"

#include <cuda_fp8.h>

namespace odmkv {

// the largest magnitude of a code: 448 = 0.875 * 2^9 (e4m3), 127 = 0.9921875 * 2^7 (int8)
__host__ __device__ inline int code_top_exp(int fmt) { return fmt == ODMKV_CODE_E4M3 ? 9 : 7; }

inline bool block_page_ok(int page) { return page == 16 || page == 32 || page == 64 || page == 128; }

// argument check of every entry point that takes a cache; `data`: its pages and tails are used too
inline int block_cache_check(const odmkv_block_cache *c, bool data) {
    if (!c || !c->table || !c->lens || !c->new_lens || !c->refs || !c->status) return ODMKV_ERR_ARG;
    if (data && (!c->k_codes || !c->v_codes || !c->k_scale || !c->v_scale || !c->k_tail || !c->v_tail)) return ODMKV_ERR_ARG;
    if (c->L <= 0 || c->N <= 0 || c->H <= 0 || c->pages <= 0 || c->width <= 0 || !block_page_ok(c->page)) return ODMKV_ERR_SHAPE;
    if (c->code_format != ODMKV_CODE_E4M3 && c->code_format != ODMKV_CODE_INT8) return ODMKV_ERR_UNSUPPORTED;
    if (c->tail_dtype != kF16 && c->tail_dtype != kBF16) return ODMKV_ERR_UNSUPPORTED;
    if (c->N > ODMKV_BLOCK_MAX_SEQS || (long long)c->H * 2 > 65535) return ODMKV_ERR_LIMIT;
    if (((long long)c->width + 1) * c->page > 0x7fffffffLL) return ODMKV_ERR_LIMIT;      // positions are 32-bit
    if ((long long)c->N * c->width > 0x7fffffffLL) return ODMKV_ERR_LIMIT;               // and so are sums of pages over the sequences
    return ODMKV_OK;
}

}  // namespace odmkv
