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
// Inside a CTA its warps take the groups in turn, each with a ring of cp.async stages of its own (neighbouring lanes copy
// neighbouring 16 bytes: pieces copied in the order of their use fetched every sector twice, 506 us instead of 387 us for one
// token over 8 x 131072, which takes 328 to 357 us now, 6.0 to 6.6 TB/s).  Both products run on mma.sync
// m16n8k16 with fp32 accumulators and the query rows as the 8 columns, directly from the token-major bytes, because the
// order of the contraction index is free as long as both operands share it, and the rows of the second product may be any
// permutation of the coordinates:
//   S^T = K Q^T (16 tokens x 8): lane (g, t) holds coordinates 16 t .. 16 t + 15 and 64 + 16 t .. of tokens g and g + 8;
//   O^T = V^T P^T (128 x 8):     lane (g, t) holds coordinates 16 g .. 16 g + 15 of tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9,
//                                whose bytes are interleaved in registers; rows g and g + 8 of tile m are coordinates
//                                16 g + 2 m and 16 g + 2 m + 1.  The weights change sides by movmatrix.
// e4m3 and int8 codes convert to fp16 exactly.  Queries are scaled by a power of two per row so that bf16 fits fp16
// (8 bits of 11; what is below 2^-26 of the row's largest magnitude loses bits).  Weights enter as fp16, for a bf16 cache
// one limb (half a step of 2^-11 beside the output's 2^-8), for an fp16 cache two (22 bits), which share one product when
// there are at most 4 rows: columns 4 to 7 repeat the queries and take the lower limbs.  In the tail of a bf16 cache the
// weights are bf16 like the values, in two limbs.
#include "block8_attn.cuh"

namespace odmkv {

namespace {

constexpr int kStepWarps = 4, kStepThreads = kStepWarps * 32;
constexpr int kStages = 3;                 // ring depth in groups
constexpr int kGroup = 16;                 // tokens
constexpr float kTailDown = 0x1p-21f;      // queries lie below 2^13
constexpr int kStageBytes = 2 * kGroup * kD;              // codes of 16 tokens, both sides
constexpr int kStepSmem = kStepWarps * kStages * kStageBytes;
constexpr int kStepCtas = 148 * 3;         // three CTAs of 49 KB and 168 registers a thread on an SM (four of 128 spill: 401 us where three took 387)
constexpr int kPad = 164;                  // floats of a joined row in shared memory, 20 per 16 coordinates: no bank conflicts
// More rows per key head than this go to the 256-row tiles of block8_tile.cu.  With cold L2 and 8 key heads, here and there: two
// sequences of 8192 tokens (33 MB: the further passes over the cache come from L2), 16 rows 31 and 41 us, 32 rows 37 to 43 and 45 us,
// 64 rows 57 and 51 us; eight of 131072 (2.1 GB, read once per 8 rows), 16 rows 680 and 1075 us, 32 rows 1290 and 1080 us.
constexpr int kMaxStepRows = 32;
// What a unit costs beside its groups, in groups: 64 ragged chats take 108 us with 0, 82 with 16 and with 80, 76 with 40 (cold L2).
constexpr int kUnitCost = 40;

__device__ __forceinline__ void cp16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint4 lds16(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
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

// State of one row tile in a warp.  Lane (g, t) has the statistics of columns 2 t and 2 t + 1 (m and D are the same in
// all lanes g, l is the lane's own part) and coordinates 16 g + 2 i, 16 g + 2 i + 1 of both (o[i][0], o[i][2]: column 2 t).
struct RowState {
    float o[8][4];
    float m[2], D[2], l[2];                // running maxima: m of the scores, m + D of scores + log2 sv; sum of 2^(score - m)
};

__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
    return y;
}

// Weights of 16 tokens and their product with the values.  s[i][e]: log2-score of token g + 8 i in column 2 t + e (masked:
// -inf); sv: the values' scale, a power of two.  o holds sum 2^(score - m - D + kLift) sv vc: D moves with the values' scale, so
// that neither large values overflow the fp16 weights nor small ones beside large ones vanish; l has a maximum of its own.
// In the tail, whose values have no scale, each token has an exponent instead: `tail` has those of tokens g and g + 8.  A maximum
// moves only when some score exceeds it by 2^kSlack, so most groups need no reduction over the lanes.
struct TailExps {
    float ev[2], low[2];                   // what D takes them for (not below what the weights' type allows), and what they are
    float reach[2];                        // running maximum of the scores + low, less m (the lane's own part)
};
template <bool BF, int LIMBS, bool TWIN, bool TAIL, class Frag>
__device__ __forceinline__ void weigh(RowState &st, float (&s)[2][2], float sv, TailExps &tail, bool upper, Frag &&frag) {
    const float es = TAIL ? 0.f : (float)((int)(__float_as_uint(sv) >> 23) - 127);
    float top[2] = {fmaxf(s[0][0], s[1][0]), fmaxf(s[0][1], s[1][1])};
    bool over = es - fminf(st.D[0], st.D[1]) > kApart;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        if constexpr (TAIL)
            over |= top[e] - st.m[e] > kSlack || fmaxf(s[0][e] - st.m[e] + tail.ev[0], s[1][e] - st.m[e] + tail.ev[1]) > st.D[e] + kSlack;
        else over |= top[e] - st.m[e] > kSlack + fminf(st.D[e] - es, 0.f);
    }
    bool apart = false;                                      // scales so far apart that the lift below would not fit fp32
    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], o));
            float2 here = make_float2(top[e], es);
            if constexpr (TAIL) {
                here.x = fmaxf(st.m[e], top[e]);
                here.y = fmaxf(s[0][e] - here.x + tail.ev[0], s[1][e] - here.x + tail.ev[1]);
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) here.y = fmaxf(here.y, __shfl_xor_sync(0xffffffffu, here.y, o));
                tail.reach[e] += st.m[e] - here.x;
            }
            const float2 now = join_tops(make_float2(st.m[e], st.D[e]), here);
            st.l[e] *= ex2(st.m[e] - now.x);
            const float f = ex2(st.m[e] - now.x + (st.D[e] - now.y));
            st.m[e] = now.x;
            st.D[e] = now.y;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                st.o[i][e] *= f;
                st.o[i][e + 2] *= f;
            }
        }
        apart = __any_sync(0xffffffffu, es - fminf(st.D[0], st.D[1]) > kApart);
    }
    if constexpr (TAIL)
#pragma unroll
        for (int e = 0; e < 2; ++e)
            tail.reach[e] = fmaxf(tail.reach[e], fmaxf(s[0][e] - st.m[e] + tail.low[0], s[1][e] - st.m[e] + tail.low[1]));
    const float lift[2] = {ex2(es + kLift - st.D[0]), ex2(es + kLift - st.D[1])};
    float w[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float p = ex2(s[i][e] - st.m[e]);
            st.l[e] += p;
            w[i][e] = p * lift[e];
        }
    if (apart)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) w[i][e] = ex2(s[i][e] - st.m[e] + (es + kLift - st.D[e]));
    uint32_t hi[2], lo[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        hi[i] = pack2<BF>(w[i][0], w[i][1]);
        if constexpr (LIMBS == 2) {
            const float2 back = unpack2<BF>(hi[i]);
            lo[i] = pack2<BF>(w[i][0] - back.x, w[i][1] - back.y);
        }
        if constexpr (TWIN) hi[i] = transpose8(upper ? lo[i] : hi[i]);
        else {
            hi[i] = transpose8(hi[i]);
            if constexpr (LIMBS == 2) lo[i] = transpose8(lo[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        uint32_t a0, a1, a2, a3;
        frag(i, a0, a1, a2, a3);
        mma<BF>(st.o[i], a0, a1, a2, a3, hi[0], hi[1]);
        if constexpr (LIMBS == 2 && !TWIN) mma<BF>(st.o[i], a0, a1, a2, a3, lo[0], lo[1]);
    }
}

// products of two chains -> log2-scores of tokens pos, pos + 8 and columns 2 t, 2 t + 1; MOD: cap and bias
template <bool MOD>
__device__ __forceinline__ void scores(const BlockAttnArgs &a, float (&s)[2][2], const float (&raw)[2][4], const float (&rs2)[2], float ks,
                                       const float (&slope2)[2], int pos, const int (&lim)[2], bool mask) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float x = (raw[0][2 * i + e] + raw[1][2 * i + e]) * (rs2[e] * ks);
            if constexpr (MOD) {
                if (a.softcap > 0.f) x = capped(x, a.cap2, a.icap2);
                x += slope2[e] * (float)(pos + 8 * i - lim[e]);
            }
            s[i][e] = mask && pos + 8 * i > lim[e] ? -INFINITY : x;
        }
}

template <int FMT, bool BF, bool MOD, bool TWIN>
__global__ void __launch_bounds__(kStepThreads, 3) block8_step_kernel(const __grid_constant__ BlockAttnArgs a) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ PieceScratch scratch;
    __shared__ float3 stat[kStepWarps][8];
    const odmkv_block_cache &c = a.c;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int Hq = c.H * a.G;

    clear_padding<kStepThreads>(a);
    const Piece piece = take_piece<kStepThreads, kGroup, kUnitCost, kStepWarps>(a, scratch);
    const int me = piece.me;
    if (me >= piece.pieces) return;
    int n = piece.n, h = piece.h, rt = piece.rt, g0 = piece.at;      // g0: first group of the unit that is this CTA's
    long long left = piece.left;
    Seq sq = seq_of(a, n);

    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * (kStages * kStageBytes);
    const int lg = c.page == 16 ? 0 : c.page == 32 ? 1 : c.page == 64 ? 2 : 3;       // groups of a page, log2
    const size_t page_bytes = (size_t)c.H * c.page * kD;

    while (left > 0) {
        const int keys = keys_of(a, sq, rt);
        const int groups = (keys + kGroup - 1) / kGroup, paged = min(groups, sq.full * (c.page / kGroup));      // those of pages
        if (g0 < groups) {
            const int g1 = (int)min((long long)groups, g0 + left);
            // pages and scales of 32 of this warp's groups, one per lane, fetched while the 32 before them are worked on; a hole
            // in the table reads page 0 and has a NaN scale, as a poisoned page
            const int first = g0 + warp;
            const int nk = first < min(g1, paged) ? (min(g1, paged) - first + kStepWarps - 1) / kStepWarps : 0;
            auto fetch_ids = [&](int k) {
                const int id = k + lane < nk ? c.table[(size_t)n * c.width + ((first + (k + lane) * kStepWarps) >> lg)] : 0;
                return id >= 0 && id < c.pages ? id : -1;
            };
            int ids = fetch_ids(0), next_ids = 0;
            // ---- queries: row g of the tile (g - 4 again, in twin columns), scaled by a power of two into fp16 ---------------
            const int row = rt * a.tile + (TWIN ? g & 3 : g), j = row / a.G, hq = h * a.G + row % a.G;
            const bool real = j < sq.more;
            uint32_t qa[16];
            float rs2[2], slope2[2];
            int lim[2];                                      // last key that the column's row sees
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
                const float rs = a.scale * pow2i(e) * kLog2e, sl = MOD && a.slopes && real ? a.slopes[hq] * kLog2e : 0.f;
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    rs2[x] = __shfl_sync(0xffffffffu, rs, 4 * (2 * t + x));
                    slope2[x] = __shfl_sync(0xffffffffu, sl, 4 * (2 * t + x));
                    lim[x] = __shfl_sync(0xffffffffu, real ? sq.have + j : 0x7fffffff, 4 * (2 * t + x));     // (unreal rows are not written)
                }
            }
            const int all_see = sq.have + rt * a.tile / a.G;  // last key that all rows see
            RowState st;
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) st.o[i][e] = 0.f;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                st.m[e] = kNone;
                st.D[e] = st.l[e] = 0.f;
            }

            // ---- the first pages are on their way ---------------------------------------------------------------------------
            const size_t head0 = (size_t)a.layer * c.pages * c.H + h;
            const unsigned char *kp = c.k_codes + head0 * ((size_t)c.page * kD), *vp = c.v_codes + head0 * ((size_t)c.page * kD);
            auto fetch_scales = [&](int id) {
                const size_t hd = head0 + (size_t)max(id, 0) * c.H;
                return id < 0 ? make_float2(__uint_as_float(0x7fc00000u), 1.f) : make_float2(c.k_scale[hd], c.v_scale[hd]);
            };
            // Stage: K rows of 128 bytes, piece p of row r at p ^ 4 (r % 2), then V rows, piece p of row r at p ^ (r & 6): both
            // products read 16 bytes a lane without bank conflicts.
            const uint32_t put_k = ring + (lane >> 3) * 128 + (((lane & 7) ^ ((lane >> 3 & 1) << 2)) * 16);
            const uint32_t put_v = ring + 2048 + (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3 & 6)) * 16);      // odd i: piece ^ 4
            auto issue = [&](int k, uint32_t stage) {
                if (k < nk) {
                    if (k && (k & 31) == 0) ids = next_ids;
                    const int id = max(__shfl_sync(0xffffffffu, ids, k & 31), 0);
                    const int in_page = (first + k * kStepWarps) & ((1 << lg) - 1);
                    const size_t off = id * page_bytes + (size_t)(in_page * kGroup * kD + lane * 16);
                    const unsigned char *ks = kp + off, *vs = vp + off;
#pragma unroll
                    for (int i = 0; i < 4; ++i) cp16(put_k + stage + i * 512, ks + i * 512);
#pragma unroll
                    for (int i = 0; i < 4; ++i) cp16(((put_v + stage) ^ ((i & 1) * 64)) + i * 512, vs + i * 512);
                }
                cp_commit();
            };
            float2 sc = fetch_scales(ids), next_sc = make_float2(0.f, 0.f);
#pragma unroll
            for (int k = 0; k < kStages - 1; ++k) issue(k, k * kStageBytes);

            // ---- tail: 16-bit rows, products in their own type ------------------------------------------------------
            const int rest = min(max(sq.have + max(c.new_lens[n], 0) - sq.full * c.page, 0), c.page);       // tokens in the tail
            const size_t tail0 = (((size_t)a.layer * c.N + n) * c.H + h) * (size_t)(c.page * kD * 2);
            TailExps tail;
            tail.reach[0] = tail.reach[1] = -INFINITY;
            for (int gi = max(g0, paged); gi < g1; ++gi) {
                if ((gi - g0) % kStepWarps != warp) continue;
                const int slot = (gi - paged) * kGroup;
                const unsigned char *kt = reinterpret_cast<const unsigned char *>(c.k_tail) + tail0, *vt = reinterpret_cast<const unsigned char *>(c.v_tail) + tail0;
                float raw[2][4] = {};
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint4 x[2][2] = {};                      // token g, token g + 8
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        if (slot + 8 * i + g < rest) {
                            const unsigned char *p = kt + (size_t)(slot + 8 * i + g) * 256 + half * 128 + 32 * t;
                            x[i][0] = *reinterpret_cast<const uint4 *>(p);
                            x[i][1] = *reinterpret_cast<const uint4 *>(p + 16);
                        }
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        uint32_t b0 = qa[half * 8 + 2 * w], b1 = qa[half * 8 + 2 * w + 1];
                        if constexpr (BF) {                  // the scaled queries, back in their own type and below 2^-8, so that no
                            const float2 p = unpack2<false>(b0), q = unpack2<false>(b1);      // sum of 128 products passes fp32
                            b0 = pack2<true>(p.x * kTailDown, p.y * kTailDown);
                            b1 = pack2<true>(q.x * kTailDown, q.y * kTailDown);
                        }
                        const uint4 &y = x[0][w >> 1], &z = x[1][w >> 1];
                        mma<BF>(raw[half], (&y.x)[2 * w & 3], (&z.x)[2 * w & 3], (&y.x)[(2 * w & 3) + 1], (&z.x)[(2 * w & 3) + 1], b0, b1);
                    }
                }
                const int key = sq.full * c.page + slot;
                float s[2][2];
                scores<MOD>(a, s, raw, rs2, BF ? 1.f / kTailDown : 1.f, slope2, key + g, lim, key + kGroup - 1 > all_see);
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
                uint32_t most[2] = {0, 0};                   // largest magnitudes of tokens 2 t, 2 t + 1 and of 2 t + 8, 2 t + 9
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t mine = 0;
#pragma unroll
                    for (int w = 0; w < 8; ++w) {
                        uint32_t &x = (&v[i][w >> 2].x)[w & 3];
                        const uint32_t top = BF ? 0x7f80u : 0x7c00u;
                        const bool l = (x & top) == top, u = (x >> 16 & top) == top;
                        if (l) x &= 0xffff0000u;
                        if (u) x &= 0xffffu;
                        odd |= l || u;
                        mine = max(mine, max(x & 0x7fffu, x >> 16 & 0x7fffu));
                    }
                    most[i >> 1] |= mine << (16 * (i & 1));
                }
                // A token counts by its largest exponent, as a page does by its scale (codes reach 2^8), so that a row is not led by
                // a larger token that it does not see.  Weights have to stay in range themselves, fp16's below 2^15 and bf16's
                // below 2^125; what that costs is given back behind the tail.
#pragma unroll
                for (int i = 0; i < 2; ++i) {
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) most[i] = __vmaxu2(most[i], __shfl_xor_sync(0xffffffffu, most[i], o));
                    const uint32_t x = __shfl_sync(0xffffffffu, most[i], g >> 1) >> (16 * (g & 1)) & 0x7fffu;
                    const int e = (BF ? (int)(x >> 7) - 127 : (int)(x >> 10) - 15) - 8;
                    tail.ev[i] = (float)max(e, BF ? -110 : 0);
                    tail.low[i] = x ? (float)max(e, -126) : -126.f;
                }
                weigh<BF, 2, TWIN, true>(st, s, 1.f, tail, t >= 2, [&](int i, uint32_t &a0, uint32_t &a1, uint32_t &a2, uint32_t &a3) {
                    const int w = i & 3, hv = i >> 2;
                    a0 = __byte_perm((&v[0][hv].x)[w], (&v[1][hv].x)[w], 0x5410);
                    a1 = __byte_perm((&v[0][hv].x)[w], (&v[1][hv].x)[w], 0x7632);
                    a2 = __byte_perm((&v[2][hv].x)[w], (&v[3][hv].x)[w], 0x5410);
                    a3 = __byte_perm((&v[2][hv].x)[w], (&v[3][hv].x)[w], 0x7632);
                });
                if (__any_sync(0xffffffffu, odd)) {
                    using T = Elem<BF ? kBF16 : kF16>;
                    for (int tok = slot; tok < min(slot + kGroup, rest); ++tok) {
                        const typename T::T *p = reinterpret_cast<const typename T::T *>(vt + (size_t)tok * 256) + 16 * g;
                        const int pos = sq.full * c.page + tok;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float x = T::to_f32(p[2 * i]), y = T::to_f32(p[2 * i + 1]);
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                if (pos > lim[e] || (TWIN && t >= 2)) continue;
                                if (!(fabsf(x) < INFINITY)) st.o[i][e] += x;
                                if (!(fabsf(y) < INFINITY)) st.o[i][e + 2] += y;
                            }
                        }
                    }
                }
            }

            if (g1 > max(g0, paged)) {                       // D as the values are, for the pages' weights
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) tail.reach[e] = fmaxf(tail.reach[e], __shfl_xor_sync(0xffffffffu, tail.reach[e], o));
                    const float down = tail.reach[e] > -INFINITY ? fmaxf(st.D[e] - fmaxf(tail.reach[e], -126.f), 0.f) : 0.f;
                    const float f = ex2(down);
                    st.D[e] -= down;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        st.o[i][e] *= f;
                        st.o[i][e + 2] *= f;
                    }
                }
            }

            // ---- pages ----------------------------------------------------------------------------------------------
            const uint32_t k_at = ring + g * 128 + ((t ^ ((g & 1) << 2)) * 16), v_at = ring + 2048 + 2 * t * 128 + ((g ^ (2 * t)) * 16);
            uint32_t at_stage = 0, to_stage = (kStages - 1) * kStageBytes;
            for (int k = 0; k < nk; ++k) {
                if ((k & 31) == 0) {
                    if (k) sc = next_sc;
                    next_ids = fetch_ids(k + 32);
                } else if ((k & 31) == 16) next_sc = fetch_scales(next_ids);
                cp_wait<kStages - 2>();
                __syncwarp();
                issue(k + kStages - 1, to_stage);            // into the stage that the last round consumed
                const uint32_t at = at_stage;
                to_stage = at;
                at_stage = at == (kStages - 1) * kStageBytes ? 0 : at + kStageBytes;
                float ks = __shfl_sync(0xffffffffu, sc.x, k & 31), vs = __shfl_sync(0xffffffffu, sc.y, k & 31);
                if (vs != vs) {                              // a poisoned page reaches the rows that see it through their scores
                    ks = vs;
                    vs = 1.f;
                }
                float raw[2][4] = {};                        // two chains
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint4 x = lds16((k_at + at) ^ (half * 64)), y = lds16(((k_at + at) ^ (half * 64)) + 1024);
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        uint32_t a0, a1, a2, a3;
                        codes_f16<FMT>((&x.x)[w], a0, a2);
                        codes_f16<FMT>((&y.x)[w], a1, a3);
                        mma<false>(raw[half], a0, a1, a2, a3, qa[half * 8 + 2 * w], qa[half * 8 + 2 * w + 1]);
                    }
                }
                const int key = (first + k * kStepWarps) * kGroup;
                float s[2][2];
                scores<MOD>(a, s, raw, rs2, ks, slope2, key + g, lim, key + kGroup - 1 > all_see);
                const uint4 v0 = lds16(v_at + at), v1 = lds16(v_at + at + 128), v2 = lds16(v_at + at + 1024), v3 = lds16(v_at + at + 1152);
                if (vs == 1.f) {
                    uint32_t some = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i) some |= (&v0.x)[i] | (&v1.x)[i] | (&v2.x)[i] | (&v3.x)[i];
                    if (!__any_sync(0xffffffffu, not_zeros<FMT>(some) != 0)) vs = 0x1p-126f;
                }
                uint32_t b[2][4];
                weigh<false, BF ? 1 : 2, TWIN, false>(st, s, vs, tail, t >= 2, [&](int i, uint32_t &a0, uint32_t &a1, uint32_t &a2, uint32_t &a3) {
                    if ((i & 1) == 0) {
                        const uint32_t w0 = (&v0.x)[i >> 1], w1 = (&v1.x)[i >> 1], w2 = (&v2.x)[i >> 1], w3 = (&v3.x)[i >> 1];
                        codes_f16<FMT>(__byte_perm(w0, w1, 0x5140), b[0][0], b[0][1]);
                        codes_f16<FMT>(__byte_perm(w0, w1, 0x7362), b[0][2], b[0][3]);
                        codes_f16<FMT>(__byte_perm(w2, w3, 0x5140), b[1][0], b[1][1]);
                        codes_f16<FMT>(__byte_perm(w2, w3, 0x7362), b[1][2], b[1][3]);
                    }
                    a0 = b[0][(i & 1) * 2];
                    a1 = b[0][(i & 1) * 2 + 1];
                    a2 = b[1][(i & 1) * 2];
                    a3 = b[1][(i & 1) * 2 + 1];
                });
            }
            cp_wait<0>();

            // ---- the warps' states, joined --------------------------------------------------------------------------
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) st.l[e] += __shfl_xor_sync(0xffffffffu, st.l[e], o);
            if constexpr (TWIN) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) st.o[i][e] += __shfl_xor_sync(0xffffffffu, st.o[i][e], 2);
            }
            __syncwarp();
            float *mine_o = reinterpret_cast<float *>(smem + warp * (kStages * kStageBytes)) + 2 * t * kPad + g * 20;
            if (!TWIN || t < 2) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *reinterpret_cast<float4 *>(mine_o + e * kPad + 4 * i) = make_float4(st.o[2 * i][e], st.o[2 * i][e + 2], st.o[2 * i + 1][e], st.o[2 * i + 1][e + 2]);
                    if (g == 0) stat[warp][2 * t + e] = make_float3(st.m[e], st.l[e], st.D[e]);
                }
            }
            __syncthreads();
            const bool begins = g0 == 0, ends = g1 == groups;
            const int slot = 2 * me + (begins ? 1 : 0);
            for (int r = warp; r < a.tile; r += kStepWarps) {
                const int row_r = rt * a.tile + r, jr = row_r / a.G;
                if (jr >= sq.more) continue;                 // (uniform in the warp)
                float2 top = make_float2(stat[0][r].x, stat[0][r].z);
#pragma unroll
                for (int w = 1; w < kStepWarps; ++w) top = join_tops(top, make_float2(stat[w][r].x, stat[w][r].z));
                const float m = top.x, D = top.y;
                float l = 0.f;
                float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kStepWarps; ++w) {
                    const float3 x = stat[w][r];
                    l += x.y * ex2(x.x - m);
                    const float f = ex2(x.x - m + (x.z - D));
                    const float4 y = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(smem + w * (kStages * kStageBytes)) + r * kPad + (lane >> 2) * 20 + (lane & 3) * 4);
                    o = make_float4(o.x + f * y.x, o.y + f * y.y, o.z + f * y.z, o.w + f * y.w);
                }
                if (begins && ends) {
                    const size_t orow = ((size_t)n * Hq + h * a.G + row_r % a.G) * a.Tq + jr;
                    finish<BF>(a.out, orow * kD + lane * 4, o, D, l);
                    if (a.lse && lane == 0) a.lse[orow] = (m + log2f(l)) * 0.69314718055994531f;
                } else {
                    *reinterpret_cast<float4 *>(a.part + ((size_t)slot * a.slot_rows + r) * kD + lane * 4) = o;
                    if (lane == 0) a.part_ml[slot * a.slot_rows + r] = make_float4(m, l, D, 0.f);
                }
            }
            if (!(begins && ends) && tid == 0) a.meta[slot] = make_int2(1, begins ? (n * c.H + h) * a.tiles + rt : (int)ends);
            __syncthreads();
        }
        if (groups > 0) left -= groups + kUnitCost - g0;
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
// A CTA takes rows blockIdx.y, + gridDim.y ...; its warps take the partials of a row in turn, and their sums are added in
// the order of the warps.
template <bool BF>
__global__ void __launch_bounds__(128) block8_join_kernel(const __grid_constant__ BlockAttnArgs a) {
    __shared__ float4 acc[4][32];
    __shared__ float2 top[4];
    __shared__ float den[4];
    const int me = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int pieces = *a.pieces;
    if (me >= pieces) return;
    const int2 head = a.meta[2 * me + 1];
    if (!head.x) return;
    const int rt = head.y % a.tiles, h = head.y / a.tiles % a.c.H, n = head.y / a.tiles / a.c.H;
    const int more = min(max(a.c.new_lens[n], 0), a.Tq);
    int count = 1;                                           // partials: slot 2 me + 1, then the even slots up to the end
    for (int base = me + 1;; base += 32) {
        const bool end = base + lane < pieces && a.meta[2 * (base + lane)].y;
        const unsigned ends = __ballot_sync(0xffffffffu, end);
        if (ends) {
            count += base - me - 1 + __ffs(ends);
            break;
        }
        if (base + 32 >= pieces) return;                     // (cannot be: the last block of all belongs to the last piece)
    }
    auto slot = [&](int i) { return i == 0 ? 2 * me + 1 : 2 * (me + i); };
    for (int r = blockIdx.y; r < a.tile; r += gridDim.y) {
        const int row = rt * a.tile + r, j = row / a.G;
        if (j >= more) break;
        float2 best = make_float2(kNone, 0.f);
        for (int i = threadIdx.x; i < count; i += 128) {
            const float4 x = a.part_ml[slot(i) * a.slot_rows + r];
            best = join_tops(best, make_float2(x.x, x.z));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            best = join_tops(best, make_float2(__shfl_xor_sync(0xffffffffu, best.x, o), __shfl_xor_sync(0xffffffffu, best.y, o)));
        if (lane == 0) top[warp] = best;
        __syncthreads();
        for (int w = 0; w < 4; ++w) best = join_tops(best, top[w]);
        const float m = best.x, D = best.y;
        float l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int i = warp; i < count; i += 4) {
            const float4 x = a.part_ml[slot(i) * a.slot_rows + r];
            const float4 y = *reinterpret_cast<const float4 *>(a.part + ((size_t)slot(i) * a.slot_rows + r) * kD + lane * 4);
            l += x.y * ex2(x.x - m);
            const float f = ex2(x.x - m + (x.z - D));
            o = make_float4(o.x + f * y.x, o.y + f * y.y, o.z + f * y.z, o.w + f * y.w);
        }
        acc[warp][lane] = o;
        if (lane == 0) den[warp] = l;
        __syncthreads();
        if (warp == 0) {
            l = den[0] + den[1] + den[2] + den[3];
            for (int w = 1; w < 4; ++w) {
                const float4 y = acc[w][lane];
                o = make_float4(o.x + y.x, o.y + y.y, o.z + y.z, o.w + y.w);
            }
            const size_t orow = ((size_t)n * a.c.H * a.G + h * a.G + row % a.G) * a.Tq + j;
            finish<BF>(a.out, orow * kD + lane * 4, o, D, l);
            if (a.lse && lane == 0) a.lse[orow] = (m + log2f(l)) * 0.69314718055994531f;
        }
        __syncthreads();
    }
}

}  // namespace

void block8_join_launch(const BlockAttnArgs &a, int ctas, cudaStream_t st) {
    const dim3 grid(ctas, min(min(a.tile, a.G * a.Tq), 32));
    if (a.c.tail_dtype == kBF16) block8_join_kernel<true><<<grid, 128, 0, st>>>(a);
    else block8_join_kernel<false><<<grid, 128, 0, st>>>(a);
}

namespace {

constexpr size_t kPartBytes = (size_t)2 * kStepCtas * 8 * kD * 4;
constexpr size_t kMlBytes = (size_t)2 * kStepCtas * 8 * 16;
constexpr size_t kMetaBytes = (size_t)2 * kStepCtas * 8;

template <int FMT, bool BF, bool MOD, bool TWIN>
int launch_step(const BlockAttnArgs &a, cudaStream_t st) {
    static_assert(kStages * kStageBytes >= 8 * kPad * 4, "a warp's joined rows lie in its ring");
    static std::atomic<unsigned long long> done{0};
    const int e = allow_smem(block8_step_kernel<FMT, BF, MOD, TWIN>, kStepSmem, done);
    if (e) return e;
    block8_step_kernel<FMT, BF, MOD, TWIN><<<kStepCtas, kStepThreads, kStepSmem, st>>>(a);
    block8_join_launch(a, kStepCtas, st);
    return launch_status();
}
template <int FMT, bool BF>
int launch_step(const BlockAttnArgs &a, cudaStream_t st) {
    const bool mod = a.softcap > 0.f || a.slopes;
    if constexpr (!BF)
        if (a.tile == 4) return mod ? launch_step<FMT, BF, true, true>(a, st) : launch_step<FMT, BF, false, true>(a, st);
    return mod ? launch_step<FMT, BF, true, false>(a, st) : launch_step<FMT, BF, false, false>(a, st);
}

}  // namespace
}  // namespace odmkv

using namespace odmkv;

extern "C" {

size_t odmkv_block8_attn_workspace_bytes(int N, int H, int G, int Tq, int width, int page) {
    if (N <= 0 || H <= 0 || G <= 0 || Tq < 0 || width <= 0 || !block_page_ok(page)) return 0;
    return (long long)G * Tq > kMaxStepRows ? block8_tile_workspace_bytes() : kPartBytes + kMlBytes + kMetaBytes + 256;
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
    const long long rows = (long long)G * Tq;
    const int tile = rows <= 4 && cache->tail_dtype == kF16 ? 4 : 8;
    const long long tiles = (rows + tile - 1) / tile;
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
    a.tile = tile;
    a.slot_rows = 8;
    a.tiles = (int)tiles;
    a.scale = scale;
    a.softcap = softcap;
    a.cap2 = fmaxf(softcap, 0x1p-100f) * kLog2e;       // (a smaller cap makes all weights equal as well, and has a reciprocal)
    a.icap2 = 1.f / a.cap2;
    if (rows > kMaxStepRows) return block8_tile_launch(a, workspace, (cudaStream_t)stream);
    unsigned char *ws = reinterpret_cast<unsigned char *>(workspace);
    a.part = reinterpret_cast<float *>(ws);
    a.part_ml = reinterpret_cast<float4 *>(ws + kPartBytes);
    a.meta = reinterpret_cast<int2 *>(ws + kPartBytes + kMlBytes);
    a.pieces = reinterpret_cast<int *>(ws + kPartBytes + kMlBytes + kMetaBytes);
    cudaStream_t st = (cudaStream_t)stream;
    if (cache->code_format == ODMKV_CODE_E4M3)
        return cache->tail_dtype == kBF16 ? launch_step<ODMKV_CODE_E4M3, true>(a, st) : launch_step<ODMKV_CODE_E4M3, false>(a, st);
    return cache->tail_dtype == kBF16 ? launch_step<ODMKV_CODE_INT8, true>(a, st) : launch_step<ODMKV_CODE_INT8, false>(a, st);
}

}  // extern "C"
