// What the two kernels of block-8 attention share (block8_attn.cu: few query rows a key head; block8_tile.cu: many).
#pragma once
#include "block8.cuh"

#include <atomic>

namespace odmkv {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNone = -3.402823466e38f;  // running maximum of a row that has seen nothing: no finite score lies below it
constexpr float kLift = 10.f, kSlack = 5.f;    // weights of at most 2^(kLift + kSlack) enter as fp16
constexpr float kApart = 90.f;             // values' scales this many powers of two apart: no factor between score and weight fits fp32

struct BlockAttnArgs {
    odmkv_block_cache c;
    const void *q;
    long long qs[3];
    const float *slopes;
    void *out;
    float *lse;
    int layer, G, Tq, tile, tiles;         // rows of a tile; tiles of a (sequence, key head)
    float scale, softcap, cap2, icap2;     // cap2 = softcap log2 e, icap2 its reciprocal
    int slot_rows;                         // rows of a partial result
    float *part;                           // [2 * CTAs, slot_rows, 128]
    float4 *part_ml;                       // [2 * CTAs, slot_rows] (m, l, D, -)
    int2 *meta;                            // [2 * CTAs]: .x used, .y: even slot 1 = the unit ends here, odd slot the unit
    int *pieces;                           // [1]
};

__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }    // -126 <= e <= 127

// c tanh(x / c) of a log2-score x, with c = cap log2 e and icap = 1 / c.  1 - 2 / (1 + e^2t) alone has an error of c 2^-23
// however small x is, which a cap of 10^4 and more makes a wrong weight: below |t| = 1/4 the odd series up to t^9 stands in its
// place (remainder 9e-9 of the value), so the error is 2^-20 of the capped score for any cap.
__device__ __forceinline__ float capped(float x, float c, float icap) {
    const float t = x * icap, z = t * t, y = t * (2.f * kLog2e);
    const float far = c - 2.f * c * __fdividef(1.f, 1.f + ex2(y > 126.f ? 126.f : y));
    float p = fmaf(z, 62.f / 2835.f, -17.f / 315.f);
    p = fmaf(z, p, 2.f / 15.f);
    p = fmaf(z, p, -1.f / 3.f);
    return fabsf(t) < 0.25f ? fmaf(x * z, p, x) : far;
}

// four codes -> two pairs of fp16
template <int FMT> __device__ __forceinline__ void codes_f16(uint32_t w, uint32_t &lo, uint32_t &hi) {
    if constexpr (FMT == ODMKV_CODE_E4M3) {
        asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}\n" : "=r"(lo), "=r"(hi) : "r"(w));
    } else {
        // 1024 + (code + 128) has the biased code in its low mantissa bits
        const uint32_t u = w ^ 0x80808080u;
        const __half2 off = __float2half2_rn(1152.f);
        uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
        const __half2 x = __hsub2(*reinterpret_cast<__half2 *>(&a), off), y = __hsub2(*reinterpret_cast<__half2 *>(&b), off);
        lo = *reinterpret_cast<const uint32_t *>(&x);
        hi = *reinterpret_cast<const uint32_t *>(&y);
    }
}

// Zeros have scale 1 whatever lies beside them, so values of a scale of 1 are looked at: those of zeros must not count as the
// largest.  Bits that are set in a word of four codes other than zeros:
template <int FMT> __device__ __forceinline__ uint32_t not_zeros(uint32_t w) { return FMT == ODMKV_CODE_E4M3 ? w & 0x7f7f7f7fu : w; }

template <bool BF> __device__ __forceinline__ uint32_t pack2(float x, float y) {
    if constexpr (BF) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&v);
    } else {
        const __half2 v = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
}
template <bool BF> __device__ __forceinline__ float2 unpack2(uint32_t w) {
    if constexpr (BF) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    else return __half22float2(*reinterpret_cast<__half2 *>(&w));
}

// what a sequence has to do
struct Seq {
    int have, more, full;                  // finished and running tokens, full pages
};
__device__ __forceinline__ Seq seq_of(const BlockAttnArgs &a, int n) {
    Seq s;
    s.have = max(a.c.lens[n], 0);
    s.more = min(max(a.c.new_lens[n], 0), a.Tq);
    s.full = min((int)(((long long)s.have + max(a.c.new_lens[n], 0)) / a.c.page), a.c.width);
    return s;
}
// keys that row tile rt looks at
__device__ __forceinline__ int keys_of(const BlockAttnArgs &a, const Seq &s, int rt) {
    if (rt * a.tile / a.G >= s.more) return 0;
    return min(s.have + min((rt * a.tile + a.tile - 1) / a.G, s.more - 1) + 1, (s.full + 1) * a.c.page);
}

// A row has two running maxima: m of the scores, and m + D of the scores + log2 of the values' scale.  D is kept by itself: beside
// scores of 2^24 and more the scale's exponent would be lost in their sum.
__device__ __forceinline__ float2 join_tops(float2 p, float2 q) {      // (m, D) of two parts
    const float m = fmaxf(p.x, q.x);
    return make_float2(m, fmaxf(p.y + (p.x - m), q.y + (q.x - m)));
}

// o / l with its two powers of two taken off one after the other (2^D alone may be near the ends of fp32)
template <bool BF>
__device__ __forceinline__ void finish(void *out, size_t at, float4 o, float D, float l) {
    const float f = (1.f / (1 << (int)kLift)) / l, e = ex2(D);
    store4<BF ? kBF16 : kF16>(out, at, make_float4(o.x * f * e, o.y * f * e, o.z * f * e, o.w * f * e));
}

// Rows behind a sequence's running tokens are zeros.
template <int THREADS>
__device__ __forceinline__ void clear_padding(const BlockAttnArgs &a) {
    const odmkv_block_cache &c = a.c;
    const int tid = threadIdx.x, Hq = c.H * a.G;
    for (int n = blockIdx.x; n < c.N; n += gridDim.x) {
        const int more = min(max(c.new_lens[n], 0), a.Tq);
        for (int i = tid; i < Hq * (a.Tq - more) * 16; i += THREADS) {
            const int r = i >> 4;
            const size_t row = ((size_t)n * Hq + r / (a.Tq - more)) * a.Tq + more + r % (a.Tq - more);
            reinterpret_cast<uint4 *>(a.out)[row * 16 + (i & 15)] = make_uint4(0, 0, 0, 0);
            if (a.lse && !(i & 15)) a.lse[row] = -INFINITY;
        }
    }
}

// A CTA's piece of all work.  A unit is (sequence, key head, row tile); its keys count in blocks of KEYS, and COST blocks
// more for its beginning and its end.  All units laid end to end are cut into equal pieces of at least LEAST.
struct Piece {
    int me, pieces;                        // pieces <= me: nothing to do
    int n, h, rt, at;                      // the first unit, and the block in it
    long long left;                        // blocks (and costs) to go
};
struct PieceScratch {
    long long sums[16], found_at;
    int found_n;
};

template <int THREADS, int KEYS, int COST, int LEAST>
__device__ __forceinline__ Piece take_piece(const BlockAttnArgs &a, PieceScratch &sh) {
    const odmkv_block_cache &c = a.c;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    static_assert(THREADS / 32 <= 16, "one sum a warp");
    auto blocks = [&](const Seq &s, int rt) {
        const int keys = keys_of(a, s, rt);
        return keys ? (keys + KEYS - 1) / KEYS + COST : 0;
    };
    auto weight = [&](int n) {
        if (n >= c.N) return 0LL;
        const Seq s = seq_of(a, n);
        long long w = 0;
        for (int rt = 0; rt < a.tiles; ++rt) w += blocks(s, rt);
        return w * c.H;
    };
    auto block_sum = [&](long long v, long long *before) {
        long long x = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 31) sh.sums[warp] = x;
        __syncthreads();
        long long total = 0, b = x - v;
#pragma unroll
        for (int w = 0; w < THREADS / 32; ++w) {
            if (w < warp) b += sh.sums[w];
            total += sh.sums[w];
        }
        *before = b;
        return total;
    };
    const long long w0 = weight(tid);
    long long before0, mine = w0;
    for (int n = tid + THREADS; n < c.N; n += THREADS) mine += weight(n);
    const long long all = block_sum(mine, &before0);        // (with up to THREADS sequences before0 is what lies in front of tid)
    Piece p;
    p.me = blockIdx.x;
    p.pieces = (int)min((long long)gridDim.x, (all + LEAST - 1) / LEAST);
    if (p.me == 0 && tid == 0) *a.pieces = p.pieces;
    if (p.me >= p.pieces) return p;
    const long long each = all / p.pieces, more_by_one = all - each * p.pieces;
    const long long from = each * p.me + min((long long)p.me, more_by_one);
    p.left = each + (p.me < more_by_one);
    if (tid == 0) {
        a.meta[2 * p.me] = make_int2(0, 0);
        a.meta[2 * p.me + 1] = make_int2(0, 0);
    }
    if (c.N <= THREADS) {
        if (from >= before0 && from < before0 + w0) {
            sh.found_n = tid;
            sh.found_at = before0;
        }
    } else {
        long long carry = 0;
        for (int base = 0; base < c.N && carry <= from; base += THREADS) {
            const long long w = weight(base + tid);
            long long before;
            const long long total = block_sum(w, &before);
            if (from >= carry + before && from < carry + before + w) {
                sh.found_n = base + tid;
                sh.found_at = carry + before;
            }
            carry += total;
        }
    }
    __syncthreads();
    p.n = sh.found_n;
    long long at = from - sh.found_at;
    const Seq s = seq_of(a, p.n);
    long long per_head = 0;
    for (int rt = 0; rt < a.tiles; ++rt) per_head += blocks(s, rt);
    p.h = (int)(at / per_head);
    at -= p.h * per_head;
    for (p.rt = 0;; ++p.rt) {
        const int w = blocks(s, p.rt);
        if (at < w) break;
        at -= w;
    }
    p.at = (int)at;
    return p;
}

// Allows a kernel its dynamic shared memory, once on each device (the attribute is the device's; 2 us of the host a call).
template <class Kernel>
inline int allow_smem(Kernel *kernel, int bytes, std::atomic<unsigned long long> &done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    const unsigned long long bit = 1ull << (dev & 63);
    if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return 0;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev < 64) done.fetch_or(bit, std::memory_order_relaxed);
    return (int)e;
}

// block8_tile.cu
size_t block8_tile_workspace_bytes();
int block8_tile_launch(BlockAttnArgs a, void *workspace, cudaStream_t st);
// block8_attn.cu: joins the partial results of `ctas` pieces
void block8_join_launch(const BlockAttnArgs &a, int ctas, cudaStream_t st);

}  // namespace odmkv
