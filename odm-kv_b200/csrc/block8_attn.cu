// Paged 8-bit cache: causal attention of the running tokens over everything stored (sm_100a).
//
//   o_r = sum_j w_rj v_j / sum_j w_rj,   w_rj = exp(cap(scale q_r.k_j) + slope (j - pos_r)),   j <= pos_r
//
// with k_j = sk kc_j, v_j = sv vc_j for the tokens of a page (codes kc, vc; powers of two sk, sv) and 16-bit k_j, v_j in
// the tail.  This file serves few query rows per key head (a decode step, a handful of tokens): every byte of the cache is
// used by up to 8 rows, so HBM is the bound (256 bytes per token and key head).
//
// Rows: row r = j G + g of a (sequence, key head) is token j, query head g; 8 rows are a tile.  A unit is (sequence, key
// head, row tile); its keys are taken in groups of 16 tokens, which never cross a page.  The groups of all units laid end
// to end are cut into equal pieces, one per CTA, from the lengths in device memory: a batch of any raggedness fills the
// device, and a captured call follows the lengths as they grow.  A unit inside one piece is written at once; a unit that
// is cut leaves one partial result per piece, which a second kernel joins in a fixed order (no atomics).
//
// Inside a CTA its warps take the groups in turn, each with a ring of cp.async stages of its own: a lane copies exactly
// the 16-byte pieces that it consumes, so no barrier stands between copy and use.  Both products run on mma.sync
// m16n8k16 with fp32 accumulators, directly from the token-major bytes, because the order of the contraction index is
// free as long as both operands share it, and the output columns may be any permutation of the coordinates:
//   S = Q K^T: lane (g, t) holds coordinates 16 t .. 16 t + 15 and 64 + 16 t .. of token g (and g + 8);
//   O = P V:   lane (g, t) holds coordinates 16 g .. 16 g + 15 of tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9, whose bytes are
//              interleaved in registers; column m of tile m is coordinate 16 g + m.
// e4m3 and int8 codes convert to fp16 exactly.  Queries are scaled by a power of two per row so that bf16 fits fp16
// (8 bits of 11; what is below 2^-26 of the row's largest magnitude loses bits).  The weights enter as two fp16 limbs in
// the two halves of the 16 rows (22 bits): their rounding does not show beside the output's.
#include "block8.cuh"

namespace odmkv {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNone = -1.0e30f;          // running maximum of a row that has seen nothing
constexpr int kStepWarps = 4, kStepThreads = kStepWarps * 32;
constexpr int kStages = 4;                 // ring depth in groups
constexpr int kGroup = 16;                 // tokens
constexpr int kStageBytes = 2 * kGroup * kD + 256;        // codes of 16 tokens, both sides; the two scales for every lane
constexpr int kStepSmem = kStepWarps * kStages * kStageBytes;
constexpr int kRowTile = 8;
constexpr int kStepCtas = 148 * 3;         // three CTAs of 66 KB and 168 registers a thread on an SM
constexpr float kLift = 10.f, kSlack = 5.f;    // weights of at most 2^(kLift + kSlack) enter as fp16

struct BlockAttnArgs {
    odmkv_block_cache c;
    const void *q;
    long long qs[3];
    const float *slopes;
    void *out;
    float *lse;
    int layer, G, Tq, tiles;               // tiles: row tiles of a (sequence, key head)
    float scale, softcap;
    float *part;                           // [2 * kStepCtas, 8, 128]
    float4 *part_ml;                       // [2 * kStepCtas, 8] (m, l, M, -)
    int2 *meta;                            // [2 * kStepCtas]: .x used, .y: even slot 1 = the unit ends here, odd slot the unit
    int *pieces;                           // [1]
};

__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }    // -126 <= e <= 127

__device__ __forceinline__ void cp16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint4 lds16(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ float lds4(uint32_t a) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];\n" : "=f"(v) : "r"(a));
    return v;
}

template <bool BF>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (BF)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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
// groups of 16 keys that row tile rt looks at: those of pages, then those of the tail
__device__ __forceinline__ int2 groups_of(const BlockAttnArgs &a, const Seq &s, int rt) {
    const int j0 = rt * kRowTile / a.G;
    if (j0 >= s.more) return make_int2(0, 0);
    const int keys = s.have + min((rt * kRowTile + kRowTile - 1) / a.G, s.more - 1) + 1;
    const int paged = s.full * a.c.page;
    return make_int2((min(keys, paged) + kGroup - 1) / kGroup, (min(max(keys - paged, 0), a.c.page) + kGroup - 1) / kGroup);
}

// State of one row tile in a warp: lane (g, t) has row g's statistics (the same in the four lanes t) and the columns
// 32 t + m and 32 t + 16 + m of row g (o[m][0], o[m][1]: upper limb of the weights; [2], [3]: lower limb).
struct RowState {
    float o[16][4];
    float m, M, l;                         // running maxima of the scores and of scores + log2 sv, sum of 2^(score - m)
};

// Weights of 16 tokens and their product with the values.  s[i][e]: log2-scores of tokens 8 i + 2 t + e (masked: -inf).
// o holds sum 2^(score - M + log2 sv + kLift) vc (ev = log2 sv): M moves with the values' scale, so that neither large
// values overflow the fp16 weights nor small ones beside large ones vanish; l has a maximum of its own.  `raise` keeps
// the weights of very large values that much lower.
template <bool BF, class Frag>
__device__ __forceinline__ void weigh(RowState &st, float (&s)[2][2], float ev, float raise, Frag &&frag) {
    float top = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // the maxima move only when they are exceeded by 2^kSlack, for all rows of the warp at once
    if (__any_sync(0xffffffffu, top > st.m + kSlack || top + ev + raise > st.M + kSlack)) {
        const float m = fmaxf(st.m, top), M = fmaxf(st.M, top + ev + raise);
        st.l *= ex2(st.m - m);
        const float f = ex2(st.M - M);
        st.m = m;
        st.M = M;
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) st.o[i][e] *= f;
    }
    // (a row that sees none of the tokens takes nothing, not even from a page whose scale is NaN)
    const float lift = top == -INFINITY ? 0.f : ex2(st.m - st.M + (ev + kLift));
    uint32_t hi[2], lo[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float p = ex2(s[i][0] - st.m), q = ex2(s[i][1] - st.m);
        st.l += p + q;
        hi[i] = pack2<BF>(p * lift, q * lift);
        const float2 back = unpack2<BF>(hi[i]);
        lo[i] = pack2<BF>(p * lift - back.x, q * lift - back.y);
    }
#pragma unroll
    for (int m = 0; m < 16; ++m) {
        uint32_t b0, b1;
        frag(m, b0, b1);
        mma<BF>(st.o[m], hi[0], lo[0], hi[1], lo[1], b0, b1);
    }
}

// raw products of a row with tokens -> log2-scores; MOD: cap and bias
template <bool MOD>
__device__ __forceinline__ float score(const BlockAttnArgs &a, float raw, float mult, float slope2, int dist) {
    float s = raw * mult;                                   // mult: scale, the scales of query and page, log2 e
    if constexpr (MOD) {
        if (a.softcap > 0.f) {
            const float cap = a.softcap * kLog2e;           // tanh y = 1 - 2 / (1 + e^2y)
            const float y = s * (2.f / a.softcap);
            s = cap - 2.f * cap * __fdividef(1.f, 1.f + ex2(y > 126.f ? 126.f : y));
        }
        s += slope2 * (float)dist;
    }
    return s;
}

template <int FMT, bool BF, bool MOD>
__global__ void __launch_bounds__(kStepThreads, 3) block8_step_kernel(const __grid_constant__ BlockAttnArgs a) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ long long sums[kStepWarps];
    __shared__ long long found_at;
    __shared__ int found_n;
    __shared__ float3 stat[kStepWarps][kRowTile];
    const odmkv_block_cache &c = a.c;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int Hq = c.H * a.G;

    // rows behind a sequence's running tokens
    for (int n = blockIdx.x; n < c.N; n += gridDim.x) {
        const int more = min(max(c.new_lens[n], 0), a.Tq);
        for (int i = tid; i < Hq * (a.Tq - more) * 16; i += kStepThreads) {
            const int r = i >> 4;
            const size_t row = ((size_t)n * Hq + r / (a.Tq - more)) * a.Tq + more + r % (a.Tq - more);
            reinterpret_cast<uint4 *>(a.out)[row * 16 + (i & 15)] = make_uint4(0, 0, 0, 0);
            if (a.lse && !(i & 15)) a.lse[row] = -INFINITY;
        }
    }

    // this CTA's piece of all groups
    auto weight = [&](int n) {
        if (n >= c.N) return 0LL;
        const Seq s = seq_of(a, n);
        long long w = 0;
        for (int rt = 0; rt < a.tiles; ++rt) {
            const int2 x = groups_of(a, s, rt);
            w += x.x + x.y;
        }
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
        if (lane == 31) sums[warp] = x;
        __syncthreads();
        long long total = 0, b = x - v;
#pragma unroll
        for (int w = 0; w < kStepWarps; ++w) {
            if (w < warp) b += sums[w];
            total += sums[w];
        }
        if (before) *before = b;
        return total;
    };
    long long mine = 0;
    for (int n = tid; n < c.N; n += kStepThreads) mine += weight(n);
    const long long all = block_sum(mine, nullptr);
    // pieces of at least one group per warp
    const int pieces = (int)min((long long)gridDim.x, (all + kStepWarps - 1) / kStepWarps);
    if (blockIdx.x == 0 && tid == 0) *a.pieces = pieces;
    if ((int)blockIdx.x >= pieces) return;
    const int me = blockIdx.x;
    const long long from = all * me / pieces, to = all * (me + 1) / pieces;
    if (tid == 0) {
        a.meta[2 * me] = make_int2(0, 0);
        a.meta[2 * me + 1] = make_int2(0, 0);
    }
    long long carry = 0;
    for (int base = 0; base < c.N; base += kStepThreads) {
        const long long w = weight(base + tid);
        long long before;
        const long long total = block_sum(w, &before);
        if (from >= carry + before && from < carry + before + w) {
            found_n = base + tid;
            found_at = carry + before;
        }
        carry += total;
        if (carry > from) break;
    }
    __syncthreads();
    int n = found_n;
    Seq sq = seq_of(a, n);
    long long left = to - from, at = from - found_at;
    int h, rt = 0;
    {
        const long long per_head = weight(n) / c.H;
        h = (int)(at / per_head);
        at -= h * per_head;
        for (;; ++rt) {
            const int2 x = groups_of(a, sq, rt);
            if (at < x.x + x.y) break;
            at -= x.x + x.y;
        }
    }
    int g0 = (int)at;                                       // first group of the unit that is this CTA's

    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * (kStages * kStageBytes);
    const int lg = c.page == 16 ? 0 : c.page == 32 ? 1 : c.page == 64 ? 2 : 3;       // groups of a page, log2
    const size_t page_bytes = (size_t)c.H * c.page * kD;

    while (left > 0) {
        const int2 ng = groups_of(a, sq, rt);
        const int groups = ng.x + ng.y;
        if (groups > 0) {
            const int g1 = (int)min((long long)groups, g0 + left);
            // ---- queries: row g of the tile, scaled by a power of two into fp16 -------------------------------------
            const int row = rt * kRowTile + g, j = row / a.G, hq = h * a.G + row % a.G;
            const bool real = j < sq.more;
            uint32_t qa[16];
            float rs = 0.f;
            {
                uint4 raw[4] = {};
                if (real) {
                    const unsigned char *qp = reinterpret_cast<const unsigned char *>(a.q) + 2 * (n * a.qs[0] + hq * a.qs[1] + j * a.qs[2]) + 32 * t;
                    raw[0] = *reinterpret_cast<const uint4 *>(qp);
                    raw[1] = *reinterpret_cast<const uint4 *>(qp + 16);
                    raw[2] = *reinterpret_cast<const uint4 *>(qp + 128);
                    raw[3] = *reinterpret_cast<const uint4 *>(qp + 144);
                }
                float top = 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float2 x = unpack2<BF>((&raw[i >> 2].x)[i & 3]);
                    top = fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y)));
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const int e = top > 0.f ? max((int)(__float_as_uint(top) >> 23) - 127 - 12, -126) : 0;
                const float inv = pow2i(-e);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float2 x = unpack2<BF>((&raw[i >> 2].x)[i & 3]);
                    qa[i] = pack2<false>(x.x * inv, x.y * inv);
                }
                rs = a.scale * pow2i(e) * kLog2e;
            }
            const int lim = real ? sq.have + j : -1;         // last key that the row sees
            const float slope2 = MOD && a.slopes && real ? a.slopes[hq] * kLog2e : 0.f;
            RowState st;
#pragma unroll
            for (int i = 0; i < 16; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) st.o[i][e] = 0.f;
            st.m = st.M = kNone;
            st.l = 0.f;

            // ---- pages ----------------------------------------------------------------------------------------------
            const int first = g0 + warp;
            const int nk = first < min(g1, ng.x) ? (min(g1, ng.x) - first + kStepWarps - 1) / kStepWarps : 0;
            const size_t head0 = (size_t)a.layer * c.pages * c.H + h;
            const unsigned char *kp = c.k_codes + head0 * ((size_t)c.page * kD), *vp = c.v_codes + head0 * ((size_t)c.page * kD);
            int ids = 0;
            auto issue = [&](int k) {
                if (k < nk) {
                    if ((k & 31) == 0) {
                        const int gi = first + (k + lane) * kStepWarps;
                        ids = k + lane < nk ? c.table[(size_t)n * c.width + (gi >> lg)] : -1;
                    }
                    const int id = __shfl_sync(0xffffffffu, ids, k & 31);
                    const bool there = id >= 0 && id < c.pages;
                    const int gi = first + k * kStepWarps;
                    const size_t off = (there ? id : 0) * page_bytes + (size_t)((gi & ((1 << lg) - 1)) * kGroup * kD);
                    const uint32_t dst = ring + (k % kStages) * kStageBytes + lane * 16;
                    const unsigned char *ks = kp + off + g * kD + 16 * t, *vs = vp + off + 2 * t * kD + 16 * g;
                    cp16(dst, ks);
                    cp16(dst + 512, ks + 64);
                    cp16(dst + 1024, ks + 8 * kD);
                    cp16(dst + 1536, ks + 8 * kD + 64);
                    cp16(dst + 2048, vs);
                    cp16(dst + 2560, vs + kD);
                    cp16(dst + 3072, vs + 8 * kD);
                    cp16(dst + 3584, vs + 9 * kD);
                    const uint32_t sd = ring + (k % kStages) * kStageBytes + 4096 + lane * 4;
                    const size_t hd = head0 + (size_t)(there ? id : 0) * c.H;
                    if (there) {
                        cp4(sd, c.k_scale + hd);
                        cp4(sd + 128, c.v_scale + hd);
                    } else {                                 // a hole in the table: NaN, as a poisoned page
                        asm volatile("st.shared.f32 [%0], %1;\nst.shared.f32 [%0 + 128], %1;\n" ::"r"(sd), "f"(__uint_as_float(0x7fc00000u)) : "memory");
                    }
                }
                cp_commit();
            };
#pragma unroll
            for (int k = 0; k < kStages - 1; ++k) issue(k);
            for (int k = 0; k < nk; ++k) {
                cp_wait<kStages - 2>();
                issue(k + kStages - 1);                      // into the stage that the last round consumed
                const uint32_t src = ring + (k % kStages) * kStageBytes + lane * 16;
                const uint32_t sd = ring + (k % kStages) * kStageBytes + 4096 + lane * 4;
                const float ks = lds4(sd), vs = lds4(sd + 128);
                float raw[2][4] = {};
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint4 x = lds16(src + half * 512), y = lds16(src + 1024 + half * 512);
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        uint32_t b0, b1;
                        const uint32_t a0 = qa[half * 8 + 2 * w], a2 = qa[half * 8 + 2 * w + 1];
                        codes_f16<FMT>((&x.x)[w], b0, b1);
                        mma<false>(raw[0], a0, 0u, a2, 0u, b0, b1);
                        codes_f16<FMT>((&y.x)[w], b0, b1);
                        mma<false>(raw[1], a0, 0u, a2, 0u, b0, b1);
                    }
                }
                const int key = (first + k * kStepWarps) * kGroup + 2 * t;
                const float mult = rs * ks;
                float s[2][2];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int pos = key + 8 * i + e;
                        s[i][e] = score<MOD>(a, raw[i][e], mult, slope2, pos - lim);
                        if (pos > lim) s[i][e] = -INFINITY;
                    }
                const uint4 v0 = lds16(src + 2048), v1 = lds16(src + 2560), v2 = lds16(src + 3072), v3 = lds16(src + 3584);
                const float ev = (float)((int)(__float_as_uint(vs) >> 23) - 127) + (vs != vs ? vs : 0.f);
                uint32_t b[2][4];
                weigh<false>(st, s, ev, 0.f, [&](int m, uint32_t &b0, uint32_t &b1) {
                    if ((m & 3) == 0) {
                        const uint32_t w0 = (&v0.x)[m >> 2], w1 = (&v1.x)[m >> 2], w2 = (&v2.x)[m >> 2], w3 = (&v3.x)[m >> 2];
                        codes_f16<FMT>(__byte_perm(w0, w1, 0x5140), b[0][0], b[0][1]);
                        codes_f16<FMT>(__byte_perm(w0, w1, 0x7362), b[0][2], b[0][3]);
                        codes_f16<FMT>(__byte_perm(w2, w3, 0x5140), b[1][0], b[1][1]);
                        codes_f16<FMT>(__byte_perm(w2, w3, 0x7362), b[1][2], b[1][3]);
                    }
                    b0 = b[0][m & 3];
                    b1 = b[1][m & 3];
                });
            }
            cp_wait<0>();

            // ---- tail: 16-bit rows, products in their own type ------------------------------------------------------
            const int rest = min(max(sq.have + max(c.new_lens[n], 0) - sq.full * c.page, 0), c.page);       // tokens in the tail
            const size_t tail0 = (((size_t)a.layer * c.N + n) * c.H + h) * (size_t)(c.page * kD * 2);
            for (int gi = max(g0, ng.x); gi < g1; ++gi) {
                if ((gi - g0) % kStepWarps != warp) continue;
                const int slot = (gi - ng.x) * kGroup;
                const unsigned char *kt = reinterpret_cast<const unsigned char *>(c.k_tail) + tail0, *vt = reinterpret_cast<const unsigned char *>(c.v_tail) + tail0;
                float raw[2][4] = {};
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int tok = slot + 8 * i + g;
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint4 x = {}, y = {};
                        if (tok < rest) {
                            const unsigned char *p = kt + (size_t)tok * 256 + half * 128 + 32 * t;
                            x = *reinterpret_cast<const uint4 *>(p);
                            y = *reinterpret_cast<const uint4 *>(p + 16);
                        }
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            uint32_t a0 = qa[half * 8 + 2 * w], a2 = qa[half * 8 + 2 * w + 1];
                            if constexpr (BF) {              // the scaled queries, back in their own type
                                const float2 p = unpack2<false>(a0), q = unpack2<false>(a2);
                                a0 = pack2<true>(p.x, p.y);
                                a2 = pack2<true>(q.x, q.y);
                            }
                            const uint4 &z = w < 2 ? x : y;
                            mma<BF>(raw[i], a0, 0u, a2, 0u, (&z.x)[2 * w & 3], (&z.x)[(2 * w & 3) + 1]);
                        }
                    }
                }
                const int key = sq.full * c.page + slot + 2 * t;
                float s[2][2];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int pos = key + 8 * i + e;
                        s[i][e] = score<MOD>(a, raw[i][e], rs, slope2, pos - lim);
                        if (pos > lim) s[i][e] = -INFINITY;
                    }
                uint4 v[4][2];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int tok = slot + 2 * t + (i & 1) + 8 * (i >> 1);
                    v[i][0] = v[i][1] = make_uint4(0, 0, 0, 0);
                    if (tok < rest) {
                        const unsigned char *p = vt + (size_t)tok * 256 + 32 * g;
                        v[i][0] = *reinterpret_cast<const uint4 *>(p);
                        v[i][1] = *reinterpret_cast<const uint4 *>(p + 16);
                    }
                }
                // infinities and NaN leave the product, where a weight of 0 would not hold them back, and go to the rows that
                // see their token below
                bool odd = false;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int w = 0; w < 8; ++w) {
                        uint32_t &x = (&v[i][w >> 2].x)[w & 3];
                        const uint32_t top = BF ? 0x7f80u : 0x7c00u;
                        const bool l = (x & top) == top, u = (x >> 16 & top) == top;
                        if (l) x &= 0xffff0000u;
                        if (u) x &= 0xffffu;
                        odd |= l || u;
                    }
                // bf16 values may be as large as 2^128: their weights stay below 1
                weigh<BF>(st, s, 0.f, BF ? kLift + kSlack : 0.f, [&](int m, uint32_t &b0, uint32_t &b1) {
                    const int w = (m >> 1) & 3, hv = m >> 3;
                    const uint32_t sel = m & 1 ? 0x7632 : 0x5410;
                    b0 = __byte_perm((&v[0][hv].x)[w], (&v[1][hv].x)[w], sel);
                    b1 = __byte_perm((&v[2][hv].x)[w], (&v[3][hv].x)[w], sel);
                });
                if (__any_sync(0xffffffffu, odd)) {
                    for (int tok = slot; tok < min(slot + kGroup, rest); ++tok) {
                        if (sq.full * c.page + tok > lim) break;
                        const unsigned char *p = vt + (size_t)tok * 256 + 64 * t;
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float x = Elem<BF ? kBF16 : kF16>::to_f32(reinterpret_cast<const typename Elem<BF ? kBF16 : kF16>::T *>(p)[i]);
                            const float y = Elem<BF ? kBF16 : kF16>::to_f32(reinterpret_cast<const typename Elem<BF ? kBF16 : kF16>::T *>(p)[16 + i]);
                            if (!(fabsf(x) < INFINITY)) st.o[i][0] += x;
                            if (!(fabsf(y) < INFINITY)) st.o[i][1] += y;
                        }
                    }
                }
            }

            // ---- the warps' states, joined --------------------------------------------------------------------------
            st.l += __shfl_xor_sync(0xffffffffu, st.l, 1);
            st.l += __shfl_xor_sync(0xffffffffu, st.l, 2);
            __syncwarp();
            constexpr int kPad = 144;                        // floats of a row in shared memory, 36 per lane t: no conflicts
            float *mine_o = reinterpret_cast<float *>(smem + warp * (kStages * kStageBytes)) + g * kPad + t * 36;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                *reinterpret_cast<float4 *>(mine_o + 4 * i) = make_float4(st.o[4 * i][0] + st.o[4 * i][2], st.o[4 * i + 1][0] + st.o[4 * i + 1][2],
                                                                          st.o[4 * i + 2][0] + st.o[4 * i + 2][2], st.o[4 * i + 3][0] + st.o[4 * i + 3][2]);
                *reinterpret_cast<float4 *>(mine_o + 16 + 4 * i) = make_float4(st.o[4 * i][1] + st.o[4 * i][3], st.o[4 * i + 1][1] + st.o[4 * i + 1][3],
                                                                               st.o[4 * i + 2][1] + st.o[4 * i + 2][3], st.o[4 * i + 3][1] + st.o[4 * i + 3][3]);
            }
            if (t == 0) stat[warp][g] = make_float3(st.m, st.l, st.M);
            __syncthreads();
            const bool begins = g0 == 0, ends = g1 == groups;
            const int slot = 2 * me + (begins ? 1 : 0);
            for (int r = warp; r < kRowTile; r += kStepWarps) {
                const int row_r = rt * kRowTile + r, jr = row_r / a.G;
                if (jr >= sq.more) continue;                 // (uniform in the warp)
                float m = kNone, M = kNone, l = 0.f;
#pragma unroll
                for (int w = 0; w < kStepWarps; ++w) {
                    m = fmaxf(m, stat[w][r].x);
                    M = fmaxf(M, stat[w][r].z);
                }
                float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kStepWarps; ++w) {
                    const float3 x = stat[w][r];
                    l += x.y * ex2(x.x - m);
                    const float f = ex2(x.z - M);
                    const float4 y = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(smem + w * (kStages * kStageBytes)) + r * kPad + (lane >> 3) * 36 + (lane & 7) * 4);
                    o = make_float4(o.x + f * y.x, o.y + f * y.y, o.z + f * y.z, o.w + f * y.w);
                }
                if (begins && ends) {
                    const size_t orow = ((size_t)n * Hq + h * a.G + row_r % a.G) * a.Tq + jr;
                    const float f = ex2(M - m - kLift) / l;
                    store4<BF ? kBF16 : kF16>(a.out, orow * kD + lane * 4, make_float4(o.x * f, o.y * f, o.z * f, o.w * f));
                    if (a.lse && lane == 0) a.lse[orow] = (m + log2f(l)) * 0.69314718055994531f;
                } else {
                    *reinterpret_cast<float4 *>(a.part + ((size_t)slot * kRowTile + r) * kD + lane * 4) = o;
                    if (lane == 0) a.part_ml[slot * kRowTile + r] = make_float4(m, l, M, 0.f);
                }
            }
            if (!(begins && ends) && tid == 0) a.meta[slot] = make_int2(1, begins ? (n * c.H + h) * a.tiles + rt : (int)ends);
            __syncthreads();
            left -= g1 - g0;
        }
        g0 = 0;
        if (++rt == a.tiles) {
            rt = 0;
            if (++h == c.H) {
                h = 0;
                if (++n >= c.N) break;
                sq = seq_of(a, n);
                if (sq.more == 0)                            // nothing to do for this sequence
                    h = c.H - 1, rt = a.tiles - 1;
            }
        }
    }
}

// The partial results of a unit that was cut: it begins in piece blockIdx.x and goes on through the pieces behind it.
// One CTA per row; its warps take the partials in turn, and their sums are added in the order of the warps.
template <bool BF>
__global__ void __launch_bounds__(128) block8_join_kernel(const __grid_constant__ BlockAttnArgs a) {
    __shared__ float4 acc[4][32];
    __shared__ float2 top[4];
    __shared__ float den[4];
    const int me = blockIdx.x, r = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int pieces = *a.pieces;
    if (me >= pieces) return;
    const int2 head = a.meta[2 * me + 1];
    if (!head.x) return;
    const int rt = head.y % a.tiles, h = head.y / a.tiles % a.c.H, n = head.y / a.tiles / a.c.H;
    const int row = rt * kRowTile + r, j = row / a.G;
    if (j >= min(max(a.c.new_lens[n], 0), a.Tq)) return;
    int count = 1;                                           // partials: slot 2 me + 1, then the even slots up to the end
    for (int base = me + 1;; base += 32) {
        const bool end = base + lane < pieces && a.meta[2 * (base + lane)].y;
        const unsigned ends = __ballot_sync(0xffffffffu, end);
        if (ends) {
            count += base - me - 1 + __ffs(ends);
            break;
        }
        if (base + 32 >= pieces) return;                     // (cannot be: the last group of all belongs to the last piece)
    }
    auto slot = [&](int i) { return i == 0 ? 2 * me + 1 : 2 * (me + i); };
    float m = kNone, M = kNone;
    for (int i = threadIdx.x; i < count; i += 128) {
        const float4 x = a.part_ml[slot(i) * kRowTile + r];
        m = fmaxf(m, x.x);
        M = fmaxf(M, x.z);
    }
    m = warp_max(m);
    M = warp_max(M);
    if (lane == 0) top[warp] = make_float2(m, M);
    __syncthreads();
    for (int w = 0; w < 4; ++w) {
        m = fmaxf(m, top[w].x);
        M = fmaxf(M, top[w].y);
    }
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = warp; i < count; i += 4) {
        const float4 x = a.part_ml[slot(i) * kRowTile + r];
        const float4 y = *reinterpret_cast<const float4 *>(a.part + ((size_t)slot(i) * kRowTile + r) * kD + lane * 4);
        l += x.y * ex2(x.x - m);
        const float f = ex2(x.z - M);
        o = make_float4(o.x + f * y.x, o.y + f * y.y, o.z + f * y.z, o.w + f * y.w);
    }
    acc[warp][lane] = o;
    if (lane == 0) den[warp] = l;
    __syncthreads();
    if (warp) return;
    l = den[0] + den[1] + den[2] + den[3];
    for (int w = 1; w < 4; ++w) {
        const float4 y = acc[w][lane];
        o = make_float4(o.x + y.x, o.y + y.y, o.z + y.z, o.w + y.w);
    }
    const size_t orow = ((size_t)n * a.c.H * a.G + h * a.G + row % a.G) * a.Tq + j;
    const float f = ex2(M - m - kLift) / l;
    store4<BF ? kBF16 : kF16>(a.out, orow * kD + lane * 4, make_float4(o.x * f, o.y * f, o.z * f, o.w * f));
    if (a.lse && lane == 0) a.lse[orow] = (m + log2f(l)) * 0.69314718055994531f;
}

constexpr size_t kPartBytes = (size_t)2 * kStepCtas * kRowTile * kD * 4;
constexpr size_t kMlBytes = (size_t)2 * kStepCtas * kRowTile * 16;
constexpr size_t kMetaBytes = (size_t)2 * kStepCtas * 8;

template <int FMT, bool BF, bool MOD>
int launch_step(const BlockAttnArgs &a, cudaStream_t st) {
    static_assert(kStepSmem >= kStepWarps * kRowTile * 144 * 4, "the joined rows lie in the rings");
    const cudaError_t e = cudaFuncSetAttribute(block8_step_kernel<FMT, BF, MOD>, cudaFuncAttributeMaxDynamicSharedMemorySize, kStepSmem);
    if (e != cudaSuccess) return (int)e;
    block8_step_kernel<FMT, BF, MOD><<<kStepCtas, kStepThreads, kStepSmem, st>>>(a);
    block8_join_kernel<BF><<<dim3(kStepCtas, min(kRowTile, a.G * a.Tq)), 128, 0, st>>>(a);
    return launch_status();
}

}  // namespace
}  // namespace odmkv

using namespace odmkv;

extern "C" {

size_t odmkv_block8_attn_workspace_bytes(int N, int H, int G, int Tq, int width, int page) {
    if (N <= 0 || H <= 0 || G <= 0 || Tq < 0 || width <= 0 || !block_page_ok(page)) return 0;
    return kPartBytes + kMlBytes + kMetaBytes + 256;
}

int odmkv_block8_attn(const odmkv_block_cache *cache, int layer, const void *q, const int64_t *q_strides, int G, int Tq,
                      float scale, float softcap, const float *slopes, void *out, float *lse, void *workspace,
                      size_t workspace_bytes, void *stream) {
    const int rc = block_cache_check(cache, true);
    if (rc != ODMKV_OK) return rc;
    if (layer < 0 || layer >= cache->L || G <= 0 || Tq < 0) return ODMKV_ERR_SHAPE;
    if (Tq == 0) return ODMKV_OK;
    if (!q || !q_strides || !out || !(softcap >= 0.f)) return ODMKV_ERR_ARG;
    if (!workspace || workspace_bytes < odmkv_block8_attn_workspace_bytes(cache->N, cache->H, G, Tq, cache->width, cache->page) ||
        ((uintptr_t)workspace & 255))
        return ODMKV_ERR_WORKSPACE;
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)cache->k_tail | (uintptr_t)cache->v_tail | (uintptr_t)cache->k_codes |
         (uintptr_t)cache->v_codes) & 15)
        return ODMKV_ERR_ARG;
    const long long rows = (long long)G * Tq, tiles = (rows + kRowTile - 1) / kRowTile;
    if ((long long)cache->N * cache->H * rows > 0x7fffffffLL / 16) return ODMKV_ERR_LIMIT;
    BlockAttnArgs a;
    a.c = *cache;
    a.q = q;
    for (int i = 0; i < 3; ++i) {
        if (q_strides[i] & 7) return ODMKV_ERR_ARG;
        a.qs[i] = q_strides[i];
    }
    a.slopes = slopes;
    a.out = out;
    a.lse = lse;
    a.layer = layer;
    a.G = G;
    a.Tq = Tq;
    a.tiles = (int)tiles;
    a.scale = scale;
    a.softcap = softcap;
    unsigned char *ws = reinterpret_cast<unsigned char *>(workspace);
    a.part = reinterpret_cast<float *>(ws);
    a.part_ml = reinterpret_cast<float4 *>(ws + kPartBytes);
    a.meta = reinterpret_cast<int2 *>(ws + kPartBytes + kMlBytes);
    a.pieces = reinterpret_cast<int *>(ws + kPartBytes + kMlBytes + kMetaBytes);
    cudaStream_t st = (cudaStream_t)stream;
    const bool mod = softcap > 0.f || slopes;
    const int which = (cache->code_format == ODMKV_CODE_INT8 ? 4 : 0) | (cache->tail_dtype == kBF16 ? 2 : 0) | (mod ? 1 : 0);
    switch (which) {
        case 0: return launch_step<ODMKV_CODE_E4M3, false, false>(a, st);
        case 1: return launch_step<ODMKV_CODE_E4M3, false, true>(a, st);
        case 2: return launch_step<ODMKV_CODE_E4M3, true, false>(a, st);
        case 3: return launch_step<ODMKV_CODE_E4M3, true, true>(a, st);
        case 4: return launch_step<ODMKV_CODE_INT8, false, false>(a, st);
        case 5: return launch_step<ODMKV_CODE_INT8, false, true>(a, st);
        case 6: return launch_step<ODMKV_CODE_INT8, true, false>(a, st);
        default: return launch_step<ODMKV_CODE_INT8, true, true>(a, st);
    }
}

}  // extern "C"
