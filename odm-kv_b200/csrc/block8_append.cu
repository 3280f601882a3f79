// Paged 8-bit cache: storing tokens (sm_100a).
//
// Per page, head and side:  s = 2^e, the smallest with max|x| <= top * s;  code = rn(x / s).  With s a power of two both
// x / s and code * s are exact in fp32, so a code is the input rounded once, to the grid of e4m3 or int8, and an
// evaluation in any wider precision gives the same code (a free scale amax / top would round twice and leave ties to
// the last bit of a division); it costs int8 up to one bit against the free scale and e4m3 nothing but range.
// Tokens are rounded when their page is complete and not before: a page filled token by token with a scale that grows
// would have to be rounded again and again.
// Bound: HBM, 2 bytes read and 1 written per value.  Four prompts of up to 16384 tokens, 8 heads: 44 us (201 MB by the mean of
// the lengths drawn, 4.6 TB/s); one token to 64 sequences: 6.5 us, launch and two dependent loads.
#include "block8.cuh"

namespace odmkv {

namespace {

constexpr int kAppThreads = 256;

struct AppendArgs {
    odmkv_block_cache c;
    const void *k, *v;
    long long ks[3], vs[3];
    int layer, T;
};

__device__ __forceinline__ float2 pair_f32(uint32_t w, bool bf16) {
    if (bf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    return __half22float2(*reinterpret_cast<__half2 *>(&w));
}

// One CTA: one page of one head and side.  A row of 128 values is 16 lanes x 16 bytes; a thread holds C = page / 16 such
// pieces (rows threadIdx / 16 + 16 i) in registers between the maximum and the rounding, so the input is read once.
// blockIdx.x counts the pages that this call completes; CTA 0, the only one that reads the tail, also writes the tokens
// behind the last full page into it, after a barrier.
template <int C>
__global__ void __launch_bounds__(kAppThreads) append_kernel(const __grid_constant__ AppendArgs a) {
    constexpr int P = C * 16;
    const odmkv_block_cache &c = a.c;
    const int n = blockIdx.z, h = blockIdx.y >> 1, side = blockIdx.y & 1, blk = blockIdx.x;
    const int have = max(c.lens[n], 0), more = max(c.new_lens[n], 0);
    if (more > a.T) {                            // positions and pages are those of all running tokens: none can be left out
        if (threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0) atomicOr(c.status, ODMKV_APPEND_SHORT);
        return;
    }
    const int o = have % P, first = have / P;
    const int nfull = (o + more) / P, rest = (o + more) % P;
    if (more == 0 || (blk >= nfull && blk != 0)) return;
    const bool bf16 = c.tail_dtype == kBF16;
    const unsigned char *src = reinterpret_cast<const unsigned char *>(side ? a.v : a.k);
    const long long *st = side ? a.vs : a.ks;
    src += 2 * (n * st[0] + h * st[1]);
    const long long row_bytes = 2 * st[2];
    unsigned char *tail = reinterpret_cast<unsigned char *>(side ? c.v_tail : c.k_tail) +
                          (((size_t)a.layer * c.N + n) * c.H + h) * (size_t)(P * kD * 2);
    const int r0 = threadIdx.x >> 4, piece = threadIdx.x & 15;
    // token i of the stretch that begins with the page of the first new token
    auto token = [&](int i) -> const unsigned char * {
        return (i < o ? tail + (size_t)i * (kD * 2) : src + (long long)(i - o) * row_bytes) + piece * 16;
    };
    if (blk < nfull) {
        uint4 x[C];
#pragma unroll
        for (int i = 0; i < C; ++i) x[i] = *reinterpret_cast<const uint4 *>(token(blk * P + r0 + 16 * i));
        // 16-bit magnitudes order as integers; infinities and NaN lie above every finite one
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < C; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t w = (&x[i].x)[j] & 0x7fff7fffu;
                top = max(top, max(w & 0xffffu, w >> 16));
            }
        top = __reduce_max_sync(0xffffffffu, top);
        __shared__ uint32_t tops[kAppThreads / 32];
        if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kAppThreads / 32; ++i) top = max(top, tops[i]);
        const bool bad = top >= (bf16 ? 0x7f80u : 0x7c00u);
        const float amax = pair_f32(top, bf16).x;
        // amax = m 2^e with m in [0.5, 1); s = 2^(e - k), one more when m is above the code's largest mantissa
        const int k = code_top_exp(c.code_format);
        const uint32_t u = __float_as_uint(amax);
        const uint32_t over = c.code_format == ODMKV_CODE_E4M3 ? 0x600000u : 0x7e0000u;
        int e = (int)(u >> 23) - 126 - k + ((u & 0x7fffffu) > over ? 1 : 0);
        e = max(e, -126);                       // (an amax below the normal numbers ends here too)
        if (amax == 0.f) e = 0;
        const float s = __uint_as_float((uint32_t)(e + 127) << 23), inv = __uint_as_float((uint32_t)(127 - e) << 23);
        // an input that would round up to 2^128, out of fp32's range, takes the code below (bf16 only: |x| >= 0.97 * 2^128)
        const int last = c.code_format == ODMKV_CODE_E4M3 ? 120 : 122;
        const bool huge = e == last;
        const float most = c.code_format == ODMKV_CODE_E4M3 ? 240.f : 63.f;
        const int page = first + blk < c.width ? c.table[(size_t)n * c.width + first + blk] : -1;
        if (page >= 0 && page < c.pages) {
            const size_t head = ((size_t)a.layer * c.pages + page) * c.H + h;
            uint8_t *dst = (side ? c.v_codes : c.k_codes) + head * (size_t)(P * kD) + r0 * kD + piece * 8;
#pragma unroll
            for (int i = 0; i < C; ++i) {
                uint32_t out[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float2 p = pair_f32((&x[i].x)[2 * j], bf16), q = pair_f32((&x[i].x)[2 * j + 1], bf16);
                    p = make_float2(p.x * inv, p.y * inv);
                    q = make_float2(q.x * inv, q.y * inv);
                    if (huge) {
                        p = make_float2(fminf(fmaxf(p.x, -most), most), fminf(fmaxf(p.y, -most), most));
                        q = make_float2(fminf(fmaxf(q.x, -most), most), fminf(fmaxf(q.y, -most), most));
                    }
                    if (c.code_format == ODMKV_CODE_E4M3) {
                        const uint32_t lo = __nv_cvt_float2_to_fp8x2(p, __NV_SATFINITE, __NV_E4M3);
                        const uint32_t hi = __nv_cvt_float2_to_fp8x2(q, __NV_SATFINITE, __NV_E4M3);
                        out[j] = lo | (hi << 16);
                    } else {
                        out[j] = (uint32_t)(__float2int_rn(p.x) & 0xff) | (uint32_t)(__float2int_rn(p.y) & 0xff) << 8 |
                                 (uint32_t)(__float2int_rn(q.x) & 0xff) << 16 | (uint32_t)(__float2int_rn(q.y) & 0xff) << 24;
                    }
                }
                *reinterpret_cast<uint2 *>(dst + (size_t)i * 16 * kD) = bad ? make_uint2(0, 0) : make_uint2(out[0], out[1]);
            }
            if (threadIdx.x == 0) (side ? c.v_scale : c.k_scale)[head] = bad ? __uint_as_float(0x7fc00000u) : s;
        }
    }
    if (blk == 0) {
        __syncthreads();       // the tail's old tokens are in registers
        for (int r = r0 + (nfull == 0 ? o / 16 * 16 : 0); r < rest; r += 16) {
            const int i = nfull * P + r;
            if (i >= o) *reinterpret_cast<uint4 *>(tail + (size_t)r * (kD * 2) + piece * 16) = *reinterpret_cast<const uint4 *>(token(i));
        }
    }
}

}  // namespace
}  // namespace odmkv

using namespace odmkv;

extern "C" {

int odmkv_block8_append(const odmkv_block_cache *cache, int layer, const void *k, const void *v, const int64_t *k_strides,
                        const int64_t *v_strides, int T, void *stream) {
    const int rc = block_cache_check(cache, true);
    if (rc != ODMKV_OK) return rc;
    if (layer < 0 || layer >= cache->L || T < 0) return ODMKV_ERR_SHAPE;
    if (T > 0 && (!k || !v)) return ODMKV_ERR_ARG;
    if (!k_strides || !v_strides) return ODMKV_ERR_ARG;
    if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)cache->k_tail | (uintptr_t)cache->v_tail | (uintptr_t)cache->k_codes |
         (uintptr_t)cache->v_codes) & 15)
        return ODMKV_ERR_ARG;
    AppendArgs a;
    a.c = *cache;
    a.k = k;
    a.v = v;
    a.layer = layer;
    a.T = T;
    for (int i = 0; i < 3; ++i) {
        if ((k_strides[i] | v_strides[i]) & 7) return ODMKV_ERR_ARG;
        a.ks[i] = k_strides[i];
        a.vs[i] = v_strides[i];
    }
    const dim3 grid(max(1, (int)(((long long)cache->page - 1 + T) / cache->page)), 2 * cache->H, cache->N);
    cudaStream_t st = (cudaStream_t)stream;
    switch (cache->page) {
        case 16: append_kernel<1><<<grid, kAppThreads, 0, st>>>(a); break;
        case 32: append_kernel<2><<<grid, kAppThreads, 0, st>>>(a); break;
        case 64: append_kernel<4><<<grid, kAppThreads, 0, st>>>(a); break;
        default: append_kernel<8><<<grid, kAppThreads, 0, st>>>(a); break;
    }
    return launch_status();
}

}  // extern "C"
