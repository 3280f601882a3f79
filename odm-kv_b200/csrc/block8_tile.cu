// Paged 8-bit cache: causal attention of many query rows per key head (a question, a chunk of a prompt) on the
// fifth-generation tensor cores (tcgen05.mma, accumulators in tensor memory).  Mathematics: block8_attn.cu.
//
// A row tile is 256 rows (row j G + g: token j, query head g), two halves A and B of 128; its keys come in blocks of 128, each
// in two steps of 64.  Per step and half: S = Q K^T (128 x 64 x 128), weights in registers, O += P V (128 x 128 x 64) with P as
// the operand in tensor memory, over the columns that held S.  A half has two such buffers: while the softmax works on one
// step, the products around it (the values of the step before, the scores of the next) run.  A CTA (one on an SM) has
// fourteen warps:
//   0-3, 4-7   softmax of half A and half B: a thread owns a row, reads it from tensor memory, writes its weights back;
//   8-11       bring K and V: 8-bit codes from global memory (copied one block ahead into a staging area), to fp16 by exact
//              conversion, into shared memory in the 128-byte swizzle (V with the same rows: token-major is the "MN-major"
//              form of the second product's B operand);
//   12, 13     issue the products of half A and of half B.  The scores of step j + 2 go where the weights of step j lie, so they
//              wait for that step's second product: only products of one accumulator follow one another by themselves.
// The softmax bounds it: one exponential per row and key, 16 a clock on an SM, is 1024 clocks per half and block (twice what its
// two products need), and with maximum, sums and synchronisation a step of 64 keys takes about 2200.  K and V are converted
// once for 256 rows.  1024 tokens over 32768, 8 key heads x 4: 615 us, 907 TFLOP/s.
//
// Blocks are taken from the newest to the oldest: a distance bias then has its largest scores first.
// Pages of one block have different scales: codes are multiplied by 2^(e - E + 7), E the largest exponent in the block, when they
// are converted, and 2^(E - 7) goes into the scores' factor and the weights' exponent.  A block whose keys' scales lie more than
// 2^21 apart, or its values' more than 2^10, is "wide": each token is converted by its own exponent, which the softmax applies to
// its score and its weight, so that a token does not disappear beside a larger one, least of all beside one that the row does not
// see.  Zeros among the values count as the smallest ones.
// Weights are fp16 in one limb for either type of cache: half a step of 2^-11 beside the output's 2^-8 or 2^-11; a second limb
// would double the second product and the room of the weights in tensor memory.  A row's running maximum may lag by 2^kSlack, so the
// accumulator is rescaled rarely.
// Work is cut into equal pieces and joined as in block8_attn.cu.  Every wait on an mbarrier is bounded; an expired one sets
// ODMKV_ATTN_EXPIRED in the cache's status and the CTA runs out without waiting again, releasing its tensor memory.
#include "block8_attn.cuh"

namespace odmkv {

namespace {

constexpr int kTileThreads = 448;
constexpr int kTileRows = 256, kHalf = 128, kBlock = 128;
constexpr int kTileCost = 3;                       // what a unit costs beside its blocks, in blocks (four questions: 150 us with 0, 141 with 3)
constexpr int kTileCtas = 148;
constexpr int kOperand = 128 * kD * 2;             // 32 KB: 128 rows x 128 coordinates in fp16
constexpr int kVOff = 0, kKOff = 2 * kOperand, kQOff = 4 * kOperand;
constexpr int kCodesOff = 6 * kOperand, kCodes = 128 * kD;      // codes of the next block: keys, values
constexpr int kTileSmem = 6 * kOperand + 2 * kCodes + 1024;
constexpr unsigned kPolls = 1u << 12;
constexpr unsigned kSuspendNs = 1000000u;

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }
__device__ __forceinline__ void mbar_init(uint64_t *bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t pred;
    asm volatile("{\n.reg .pred P1;\nelect.sync _|P1, 0xffffffff;\nselp.u32 %0, 1, 0, P1;\n}\n" : "=r"(pred));
    return pred != 0;
}
// bounded; false when it expired or another role has given up
__device__ __forceinline__ bool mbar_wait(uint64_t *bar, unsigned parity, const volatile int *abort_flag) {
    for (unsigned it = 0; it < kPolls; ++it) {
        uint32_t ok;
        asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\nselp.u32 %0, 1, 0, p;\n}\n"
                     : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity), "r"(kSuspendNs) : "memory");
        if (ok) return true;
        if (*abort_flag) return false;
    }
    return false;
}
// Shared-memory descriptors in two words: the lower one has the address in units of 16 bytes (and takes offsets by addition)
// and, from bit 16, the leading stride; the upper one is the same for all: 1024 bytes between groups of 8 rows, 128-byte
// swizzle.  K-major: no leading stride; MN-major: 16384 bytes between blocks of 64 columns.
constexpr uint32_t kDescHi = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_k(uint32_t addr) { return (addr >> 4) | 1u << 16; }
__device__ __forceinline__ uint32_t desc_mn(uint32_t addr) { return (addr >> 4) | (uint32_t)(16384 >> 4) << 16; }
// fp32 accumulator, fp16 operands, M = 128, N = 64 and 128; bit 16: B is MN-major
constexpr uint32_t kIdescS = (1u << 4) | ((uint32_t)(64 >> 3) << 17) | ((128u >> 4) << 24);
constexpr uint32_t kIdescO = (1u << 4) | (1u << 16) | ((uint32_t)(128 >> 3) << 17) | ((128u >> 4) << 24);
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t accumulate) {
    asm volatile("{\n.reg .pred p;\n.reg .b64 x, y;\nsetp.ne.b32 p, %5, 0;\nmov.b64 x, {%1, %3};\nmov.b64 y, {%2, %3};\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %4, p;\n}\n"
                 ::"r"(d), "r"(a), "r"(b), "r"(kDescHi), "r"(kIdescS), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t accumulate) {
    asm volatile("{\n.reg .pred p;\n.reg .b64 y;\nsetp.ne.b32 p, %5, 0;\nmov.b64 y, {%2, %3};\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %4, p;\n}\n"
                 ::"r"(d), "r"(a), "r"(b), "r"(kDescHi), "r"(kIdescO), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
        "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
          "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
          "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void sts16(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};\n" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ uint32_t mul_h2(uint32_t x, uint32_t f) {
    const __half2 y = __hmul2(*reinterpret_cast<__half2 *>(&x), *reinterpret_cast<__half2 *>(&f));
    return *reinterpret_cast<const uint32_t *>(&y);
}
struct TileShared {
    uint64_t k_full[2], k_free[2], v_full[2], v_free[2];     // operand stages
    uint64_t q_full[2], s_full[2][2], p_full[2][2], o_step[2][2];     // by half and buffer; o_step: the step's values are in the accumulator
    uint64_t drain[2];
    float2 exps[4];                    // log2 of a block's K and V scales (block mod 4)
    int wide[4];                       // the block's tokens have exponents of their own:
    char2 key_exps[4][kBlock];         // log2 of the scales of a token's key and value
    uint32_t some;                     // groups of a block with values other than zeros
    int top_exp[2], low_exp[2];        // largest and smallest exponents of a block that is not all in pages
    int odd_tail;                      // infinities or NaN among the tail's values
    int abort;
    uint32_t tmem;
    PieceScratch scratch;
};

// The same walk over a CTA's piece in every role.
struct Walk {
    int n, h, rt, b, b1, blocks, keys;     // block b of blocks b .. b1 - 1 that are this CTA's, of a unit of `blocks`
    long long left;
    Seq sq;
};
// the next unit with blocks of its own from (n, h, rt, at) on; false at the end of the piece
__device__ __forceinline__ bool walk_unit(const BlockAttnArgs &a, Walk &w) {
    while (w.left > 0 && w.n < a.c.N) {
        w.keys = keys_of(a, w.sq, w.rt);
        w.blocks = (w.keys + kBlock - 1) / kBlock;
        if (w.b < w.blocks) {
            w.b1 = (int)min((long long)w.blocks, w.b + w.left);
            return true;
        }
        if (w.keys) w.left -= w.blocks + kTileCost - w.b;
        w.b = 0;
        if (++w.rt == a.tiles) {
            w.rt = 0;
            if (++w.h == a.c.H) {
                w.h = 0;
                if (++w.n < a.c.N) w.sq = seq_of(a, w.n);
            }
        }
    }
    return false;
}
// behind the last block of the unit
__device__ __forceinline__ void walk_on(const BlockAttnArgs &a, Walk &w, int b0) {
    w.left -= w.blocks + kTileCost - b0;
    w.b = 0;
    if (++w.rt == a.tiles) {
        w.rt = 0;
        if (++w.h == a.c.H) {
            w.h = 0;
            if (++w.n < a.c.N) w.sq = seq_of(a, w.n);
        }
    }
}
__device__ __forceinline__ int halves_of(const BlockAttnArgs &a, const Walk &w) {
    return (w.rt * kTileRows + kHalf) / a.G < w.sq.more ? 2 : 1;
}

// ---- K and V ---------------------------------------------------------------------------------------------------------
// Thread x of 128 has 16 coordinates of one token in each of the block's eight groups of 16, which lie in one page (or in the
// tail) each: bits 0-1 of x and bit 3 choose the coordinates, bit 2 and bits 4-6 the token, so that eight neighbouring
// threads write pieces of two rows and meet no bank twice.
// The codes of the next block are on their way (cp.async) while this one is converted; a warp copies the rows that it
// converts, four of each group, and page numbers and scales lie across its lanes.
template <int FMT, bool BF>
struct Bring {
    const BlockAttnArgs &a;
    TileShared &sh;
    int lg, row, at;                   // token in a group, first coordinate
    bool first;
    uint32_t put0, put1;               // where the thread's two 16-byte pieces of fp16 go in an operand tile (group 0)
    uint32_t codes, copy_to, copy_from;    // its codes in shared memory; what it copies there, from where in a page (group 0)

    __device__ __forceinline__ Bring(const BlockAttnArgs &args, TileShared &shared, uint32_t stage, int x) : a(args), sh(shared) {
        lg = a.c.page == 16 ? 4 : a.c.page == 32 ? 5 : a.c.page == 64 ? 6 : 7;
        const int p = x & 3, half = x >> 3 & 1;
        row = (x >> 2 & 1) + 2 * (x >> 4);
        at = half * 64 + p * 16;
        first = x == 0;
        put0 = half * 16384 + row * 128 + (((2 * p) ^ (row & 7)) * 16);
        put1 = half * 16384 + row * 128 + (((2 * p + 1) ^ (row & 7)) * 16);
        // piece p of row r lies at p ^ 4 (r % 2): eight threads read two rows without bank conflicts
        codes = stage + row * 128 + (((half * 4 + p) ^ ((row & 1) << 2)) * 16);
        const int r = (x >> 5) * 4 + (x >> 3 & 3), piece = x & 7;
        copy_to = stage + r * 128 + ((piece ^ ((r & 1) << 2)) * 16);
        copy_from = r * 128 + piece * 16;
    }
    // is every group of the block in pages?
    __device__ __forceinline__ static bool plain(const Walk &w, int b, int page) {
        return (b + 1) * kBlock <= w.sq.full * page;
    }
    __device__ __forceinline__ int fetch_id(const Walk &w, int b) const {
        return a.c.table[(size_t)w.n * a.c.width + ((b * kBlock + 16 * (threadIdx.x & 7)) >> lg)];
    }
    // scales of a block: keys in lanes with bit 3 clear, values in the others
    __device__ __forceinline__ uint32_t fetch_scale(const Walk &w, int id) const {
        const odmkv_block_cache &c = a.c;
        const bool there = (uint32_t)id < (uint32_t)c.pages;
        const size_t head = ((size_t)a.layer * c.pages + (there ? id : 0)) * c.H + w.h;
        const uint32_t s = reinterpret_cast<const uint32_t *>(threadIdx.x & 8 ? c.v_scale : c.k_scale)[head];
        return there ? s : 0x7fc00000u;                      // a hole in the table, as a poisoned page
    }
    // one side of a block, group by group; nothing where id < -1
    template <bool VALUES> __device__ __forceinline__ void copy(const Walk &w, int id) const {
        const odmkv_block_cache &c = a.c;
        __syncwarp();                                        // the warp has read what lies there
        if (id >= -1) {
            const uint32_t page_bytes = c.page * kD, mask = page_bytes - 1, step = page_bytes * c.H;
            const unsigned char *src = (VALUES ? c.v_codes : c.k_codes) + ((size_t)a.layer * c.pages * c.H + w.h) * page_bytes + copy_from;
            if ((uint32_t)id >= (uint32_t)c.pages) id = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const size_t off = (size_t)(uint32_t)__shfl_sync(0xffffffffu, id, i) * step + (i * 2048 & mask);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(copy_to + (VALUES ? kCodes : 0) + i * 2048), "l"(src + off) : "memory");
            }
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
    }
    __device__ __forceinline__ static void copied() {        // all but the last group of copies
        asm volatile("cp.async.wait_group 1;\n" ::: "memory");
        __syncwarp();
    }
    __device__ __forceinline__ static int exp_of(float s) { return (int)(__float_as_uint(s) >> 23) - 127; }
    __device__ __forceinline__ void put(uint32_t tile, int i, const uint32_t (&o)[8]) const {
        const uint32_t t = tile + i * 2048;
        sts16(t + put0, o[0], o[1], o[2], o[3]);
        sts16(t + put1, o[4], o[5], o[6], o[7]);
    }
    // m: the factor 2^(e - E + 7) as fp16 bits, twice
    __device__ __forceinline__ void convert(const uint4 &u, uint32_t m, uint32_t (&o)[8]) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            uint32_t lo, hi;
            codes_f16<FMT>((&u.x)[e], lo, hi);
            o[2 * e] = mul_h2(lo, m);
            o[2 * e + 1] = mul_h2(hi, m);
        }
    }
    __device__ __forceinline__ static uint32_t factor(int e) { return (uint32_t)max(e + 15, 0) * 0x04000400u; }      // e <= 7
    // How far (powers of two) scales may lie below the largest of their block.  Keys: the factor 2^-14 is the smallest of fp16 and
    // keeps every code; a token of the tail keeps 2^-24 of its largest.  Values: as much less has a weight of the block's largest
    // page room above fp16's smallest, wherever the row's largest weight lies.
    __device__ __forceinline__ static constexpr int spread(bool values) { return values ? 10 : 21; }
    __device__ __forceinline__ static constexpr int tail_spread(bool values) { return values ? 10 : 15; }
    template <bool VALUES> __device__ __forceinline__ void store(uint32_t scale, int E, uint32_t tile) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            uint4 u;
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(codes + (VALUES ? kCodes : 0) + i * 2048));
            uint32_t o[8];
            convert(u, factor((int)(__shfl_sync(0xffffffffu, scale, VALUES ? i + 8 : i) >> 23) - 127 - E + 7), o);
            put(tile, i, o);
        }
    }
    // values' scales of 1 whose codes are all zeros become 0 (rare: the copies are waited for)
    __device__ __noinline__ uint32_t drop_zeros(uint32_t scale) const {
        asm volatile("cp.async.wait_group 0;\n" ::: "memory");
        __syncwarp();
        uint32_t some = 0;                                   // bit i: group i has a code
        for (int i = 0; i < 8; ++i) {
            uint4 u;
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(codes + kCodes + i * 2048));
            if (not_zeros<FMT>(u.x | u.y | u.z | u.w)) some |= 1u << i;
        }
        some = __reduce_or_sync(0xffffffffu, some);
        if (first) sh.some = 0;
        asm volatile("bar.sync 1, 128;\n" ::: "memory");
        if ((threadIdx.x & 31) == 0) atomicOr(&sh.some, some);
        asm volatile("bar.sync 1, 128;\n" ::: "memory");
        some = *reinterpret_cast<volatile uint32_t *>(&sh.some);
        asm volatile("bar.sync 1, 128;\n" ::: "memory");      // everybody has read
        return (threadIdx.x & 8) && scale == 0x3f800000u && !(some >> (threadIdx.x & 7) & 1) ? 0 : scale;
    }
    // the block's largest exponents; positive floats order as integers, NaN behind all of them: false where there is one, or
    // where the smallest lies too far below
    __device__ __forceinline__ static bool max_exps(uint32_t scale, int2 &e) {
        const uint32_t k = __reduce_max_sync(0xffffffffu, threadIdx.x & 8 ? 0u : scale);
        const uint32_t v = __reduce_max_sync(0xffffffffu, threadIdx.x & 8 ? scale : 0u);
        e = make_int2(max((int)(k >> 23) - 127, -119), max((int)(v >> 23) - 127, -119));
        const bool below = (threadIdx.x & 8 ? e.y : e.x) - ((int)(scale >> 23) - 127) > spread(threadIdx.x & 8);
        return max(k, v) < 0x7f800000u && !__any_sync(0xffffffffu, below);
    }

    // ---- a block that reaches into the tail, or with a poisoned page, or a wide one: everything straight from memory, a group at a time
    __device__ __forceinline__ static bool odd(uint32_t h) { return (h & (BF ? 0x7f80u : 0x7c00u)) == (BF ? 0x7f80u : 0x7c00u); }
    __device__ __forceinline__ const unsigned char *tail_row(const Walk &w, int b, int i, bool values, bool &there) const {
        const odmkv_block_cache &c = a.c;
        const int slot = b * kBlock + 16 * i + row - w.sq.full * c.page;
        there = slot >= 0 && slot < min(w.keys - w.sq.full * c.page, c.page);
        return reinterpret_cast<const unsigned char *>(values ? c.v_tail : c.k_tail) +
               ((((size_t)a.layer * c.N + w.n) * c.H + w.h) * c.page + (there ? slot : 0)) * (kD * 2) + at * 2;
    }
    __device__ __forceinline__ bool page_of(const Walk &w, int b, int i, size_t &head) const {
        const odmkv_block_cache &c = a.c;
        const int id = c.table[(size_t)w.n * c.width + ((b * kBlock + 16 * i) >> lg)];
        const bool there = id >= 0 && id < c.pages;
        head = ((size_t)a.layer * c.pages + (there ? id : 0)) * c.H + w.h;
        return there;
    }
    // the block's largest exponents, over the 128 threads, and those of its tokens (the eight threads of a token are lanes that
    // differ in bits 0, 1 and 3); wide: they are too far apart for one factor
    __device__ __noinline__ int2 mixed_exps(const Walk &w, int b, int slot, bool &wide) const {
        const odmkv_block_cache &c = a.c;
        constexpr int kNothing = -119;                        // where there is nothing but zeros; the lowest that is told apart
        if (first)
            for (int side = 0; side < 2; ++side) {
                sh.top_exp[side] = kNothing;
                sh.low_exp[side] = 1000;
            }
        asm volatile("bar.sync 1, 128;\n" ::: "memory");
        int top[2] = {kNothing, kNothing}, low[2] = {1000, 1000};
        for (int i = 0; i < 8; ++i) {
            const int pos = b * kBlock + 16 * i;
            int e[2] = {kNothing, kNothing};
            if (pos < w.keys && pos < w.sq.full * c.page) {
                size_t head;
                const bool there = page_of(w, b, i, head);
                const float ks = c.k_scale[head], vs = c.v_scale[head];
                if (there && ks == ks && vs == vs) {          // (a poisoned page is NaN at any scale)
                    const int of[2] = {exp_of(ks), exp_of(vs)};
                    uint32_t some = 1;
                    if (vs == 1.f) {
                        const size_t off = head * ((size_t)c.page * kD) + (uint32_t)(((pos & (c.page - 1)) + row) * kD + at);
                        const uint4 u = *reinterpret_cast<const uint4 *>(c.v_codes + off);
                        some = not_zeros<FMT>(u.x | u.y | u.z | u.w);
                        some |= __shfl_xor_sync(0xffffffffu, some, 1);
                        some |= __shfl_xor_sync(0xffffffffu, some, 2);
                        some |= __shfl_xor_sync(0xffffffffu, some, 8);
                    }
#pragma unroll
                    for (int side = 0; side < 2; ++side) {
                        if (side && !some) {                  // zeros: as the smallest values
                            low[side] = kNothing;
                            continue;
                        }
                        e[side] = max(of[side], kNothing);
                        top[side] = max(top[side], of[side]);
                        low[side] = min(low[side], of[side]);
                    }
                }
            } else if (pos < w.keys) {
#pragma unroll
                for (int side = 0; side < 2; ++side) {
                    bool there;
                    const uint4 *p = reinterpret_cast<const uint4 *>(tail_row(w, b, i, side, there));
                    uint32_t most = 0;
                    if (there) {
                        const uint4 u[2] = {p[0], p[1]};
#pragma unroll
                        for (int x = 0; x < 8; ++x) {
                            const uint32_t v = (&u[x >> 2].x)[x & 3], lo = v & 0x7fffu, hi = v >> 16 & 0x7fffu;
                            if (!odd(lo)) most = max(most, lo);
                            if (!odd(hi)) most = max(most, hi);
                        }
                    }
                    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
                    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
                    most = max(most, __shfl_xor_sync(0xffffffffu, most, 8));
                    if (there && side && !most) low[side] = kNothing;
                    if (most) {                               // scaled, the tail stays below 2^8 as codes do
                        e[side] = max((BF ? (int)(most >> 7) - 127 : (int)(most >> 10) - 15) - 7, kNothing);
                        top[side] = max(top[side], e[side]);
                        low[side] = min(low[side], e[side] - (spread(side) - tail_spread(side)));
                    }
                }
            }
            if ((threadIdx.x & 11) == 0) sh.key_exps[slot][16 * i + row] = make_char2((signed char)(e[0] - 7), (signed char)(e[1] - 7));
        }
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            const int t = __reduce_max_sync(0xffffffffu, top[side]), l = __reduce_min_sync(0xffffffffu, low[side]);
            if ((threadIdx.x & 31) == 0) {
                atomicMax(&sh.top_exp[side], t);
                atomicMin(&sh.low_exp[side], l);
            }
        }
        asm volatile("bar.sync 1, 128;\n" ::: "memory");
        const int2 E = make_int2(sh.top_exp[0], sh.top_exp[1]);
        wide = E.x - sh.low_exp[0] > spread(false) || E.y - sh.low_exp[1] > spread(true);
        asm volatile("bar.sync 1, 128;\n" ::: "memory");      // everybody has read
        return E;
    }
    __device__ __noinline__ void store_mixed(const Walk &w, int b, bool values, int E, int wide_slot, uint32_t tile) const {
        const odmkv_block_cache &c = a.c;
        bool found_odd = false;
        for (int i = 0; i < 8; ++i) {
            const int pos = b * kBlock + 16 * i;
            if (wide_slot >= 0) {                             // the token's own
                const char2 own = sh.key_exps[wide_slot][16 * i + row];
                E = (values ? own.y : own.x) + 7;
            }
            uint32_t o[8] = {};
            if (pos < w.keys && pos < w.sq.full * c.page) {
                size_t head;
                const bool there = page_of(w, b, i, head);
                const size_t off = head * ((size_t)c.page * kD) + (uint32_t)(((pos & (c.page - 1)) + row) * kD + at);
                const uint4 u = *reinterpret_cast<const uint4 *>((values ? c.v_codes : c.k_codes) + off);
                const float ks = c.k_scale[head], vs = c.v_scale[head];
                // poisoned: NaN keys, so that the rows that see it have NaN scores
                if (!there || ks != ks || vs != vs) convert(u, values ? 0u : 0x7e007e00u, o);
                else convert(u, factor(min(exp_of(values ? vs : ks) - E + 7, 7)), o);      // (more for a token of zeros only)
            } else if (pos < w.keys) {
                bool there;
                const uint4 *p = reinterpret_cast<const uint4 *>(tail_row(w, b, i, values, there));
                if (there) {
                    const uint4 u[2] = {p[0], p[1]};
                    const float m = pow2i(max(min(7 - E, 127), -126));
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        uint32_t v = (&u[e >> 2].x)[e & 3];
                        if (values) {                        // a weight of 0 would not hold back an infinity: see the end of a unit
                            if (odd(v)) { v &= 0xffff0000u; found_odd = true; }
                            if (odd(v >> 16)) { v &= 0xffffu; found_odd = true; }
                        }
                        const float2 y = unpack2<BF>(v);
                        o[e] = pack2<false>(y.x * m, y.y * m);
                    }
                }
            }
            put(tile, i, o);
        }
        if (found_odd) sh.odd_tail = 1;
    }
};

// ---- the softmax of a step, for what its fast form cannot do (rare): scales by token, scores beside which the lift is lost, values
// of very different sizes.  It begins anew with the products in tensor memory, 16 columns at a time in registers.
struct TileRow {
    float m, D, l;
};
struct Careful {
    const char2 *own;                  // log2 of the scales by token, or nullptr: ex for all
    float2 ex;
    float rs, slope2;
    int key0, lim;
    uint32_t t_s, t_o;
    bool carry;                        // the accumulator holds something
};
__device__ __forceinline__ void rescale(uint32_t t_o, float f) {
#pragma unroll 1
    for (int q = 0; q < 8; ++q) {
        uint32_t v[16];
        tmem_ld16(t_o + q * 16, v);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * f);
        tmem_st16(t_o + q * 16, v);
    }
}
template <bool MOD>
__device__ __noinline__ TileRow careful_step(const BlockAttnArgs &a, const Careful &s, TileRow st) {
    uint32_t v[16];
    auto ev = [&](int k) { return s.own ? (float)s.own[k].y : s.ex.y; };
    TileRow now;
    now.m = st.m;
    float reach = -INFINITY;
    // log2-scores, and their maximum
#pragma unroll 1
    for (int q = 0; q < 4; ++q) {
        tmem_ld16(s.t_s + q * 16, v);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int k = q * 16 + e;
            float x = __uint_as_float(v[e]) * (s.rs * (s.own ? pow2i(s.own[k].x) : ex2(s.ex.x)));
            if (MOD && a.softcap > 0.f) x = capped(x, a.cap2, a.icap2);
            if (MOD) x = fmaf(s.slope2, (float)(s.key0 + k - s.lim), x);
            if (s.key0 + k > s.lim) x = -INFINITY;
            now.m = fmaxf(now.m, x);
            v[e] = __float_as_uint(x);
        }
        tmem_st16(s.t_s + q * 16, v);
    }
    tmem_st_wait();
#pragma unroll 1
    for (int q = 0; q < 4; ++q) {
        tmem_ld16(s.t_s + q * 16, v);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; ++e) reach = fmaxf(reach, __uint_as_float(v[e]) - now.m + ev(q * 16 + e));
    }
    now.D = fmaxf(st.D + (st.m - now.m), reach);
    now.l = st.l * ex2(st.m - now.m);
    if (s.carry) rescale(s.t_o, ex2(st.m - now.m + (st.D - now.D)));
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {                   // (the weights lie where scores were that have been read)
        uint32_t p[16];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            tmem_ld16(s.t_s + half * 32 + q * 16, v);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                float x[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float y = __uint_as_float(v[e + i]) - now.m;
                    now.l += ex2(y);
                    x[i] = ex2(y + (ev(half * 32 + q * 16 + e + i) + kLift - now.D));
                }
                p[q * 8 + e / 2] = pack2<false>(x[0], x[1]);
            }
        }
        tmem_st16(s.t_s + half * 16, p);
    }
    return now;
}

template <int FMT, bool BF, bool MOD>
__global__ void __launch_bounds__(kTileThreads, 1) block8_tile_kernel(const __grid_constant__ BlockAttnArgs a) {
    extern __shared__ __align__(1024) unsigned char dyn[];
    __shared__ TileShared sh;
    unsigned char *smem = dyn + (1024 - (smem_u32(dyn) & 1023)) % 1024;
    const odmkv_block_cache &c = a.c;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    clear_padding<kTileThreads>(a);
    const Piece piece = take_piece<kTileThreads, kBlock, kTileCost, 2>(a, sh.scratch);
    if (piece.me >= piece.pieces) return;
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.k_full[i], 128);
            mbar_init(&sh.v_full[i], 128);
            mbar_init(&sh.k_free[i], 2);
            mbar_init(&sh.v_free[i], 2);
            mbar_init(&sh.q_full[i], 128);
            mbar_init(&sh.drain[i], 1);
            for (int t = 0; t < 2; ++t) {
                mbar_init(&sh.p_full[t][i], 128);
                mbar_init(&sh.s_full[t][i], 1);
                mbar_init(&sh.o_step[t][i], 1);
            }
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        sh.abort = 0;
        sh.odd_tail = 0;
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&sh.tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;                           // S of A, S of B, O of A, O of B: 128 columns each
    const volatile int *gave_up = &sh.abort;
    Walk w;
    w.n = piece.n;
    w.h = piece.h;
    w.rt = piece.rt;
    w.b = piece.at;
    w.left = piece.left;
    w.sq = seq_of(a, w.n);
    bool ok = true;

    if (warp >= 8 && warp < 12) {
        // ---- K and V -------------------------------------------------------------------------------------------------
        const uint32_t kv = smem_u32(smem);
        const Bring<FMT, BF> bring(a, sh, kv + kCodesOff, tid - 256);
        uint32_t it = 0;
        while (walk_unit(a, w)) {                            // (whatever happens, all 128 threads go the same way)
            const int b0 = w.b;
            // page numbers of block b: -2 where the block is not all in pages, or is not this CTA's
            auto ids_of = [&](int b) { return b >= b0 && bring.plain(w, b, c.page) ? max(bring.fetch_id(w, b), -1) : -2; };
            int id = ids_of(w.b1 - 1), next_id = ids_of(w.b1 - 2);
            uint32_t scale = id >= -1 ? bring.fetch_scale(w, id) : 0;
            bring.template copy<false>(w, id);
            bring.template copy<true>(w, id);
            for (int b = w.b1 - 1; b >= b0; --b, ++it) {
                const int st = it & 1, id_behind = ids_of(b - 2);          // (looked at in the next round)
                int2 e;
                bool plain = __all_sync(0xffffffffu, id >= -1);
                if (plain && __any_sync(0xffffffffu, (tid & 8) && scale == 0x3f800000u)) scale = bring.drop_zeros(scale);
                plain = plain && bring.max_exps(scale, e);
                bool wide = false;
                if (!plain) e = bring.mixed_exps(w, b, it & 3, wide);
                const uint32_t next_scale = next_id >= -1 ? bring.fetch_scale(w, next_id) : 0;
                if (it >= 2 && ok) ok = mbar_wait(&sh.k_free[st], (it / 2 - 1) & 1, gave_up);
                if (tid == 256) {
                    sh.exps[it & 3] = make_float2((float)(e.x - 7), wide ? 0.f : (float)(e.y - 7));
                    sh.wide[it & 3] = wide;
                }
                bring.copied();
                if (plain) bring.template store<false>(scale, e.x, kv + kKOff + st * kOperand);
                else bring.store_mixed(w, b, false, e.x, wide ? (int)(it & 3) : -1, kv + kKOff + st * kOperand);
                proxy_fence();
                mbar_arrive(&sh.k_full[st]);
                bring.template copy<false>(w, next_id);
                if (it >= 2 && ok) ok = mbar_wait(&sh.v_free[st], (it / 2 - 1) & 1, gave_up);
                bring.copied();
                if (plain) bring.template store<true>(scale, e.y, kv + kVOff + st * kOperand);
                else bring.store_mixed(w, b, true, e.y, wide ? (int)(it & 3) : -1, kv + kVOff + st * kOperand);
                proxy_fence();
                mbar_arrive(&sh.v_full[st]);
                bring.template copy<true>(w, next_id);
                id = next_id;
                scale = next_scale;
                next_id = id_behind;
            }
            walk_on(a, w, b0);
        }
    } else if (warp >= 12) {
        auto wait_all = [&](uint64_t *bar, unsigned parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, gave_up)); };
        // ---- products ------------------------------------------------------------------------------------------------
        {
            // All lanes go along and one is elected for each batch of products: descriptors then live in uniform registers (one
            // lane on its own took 200 clocks a product).
            const int t = __shfl_sync(0xffffffffu, warp, 0) - 12;
            const uint32_t base = smem_u32(smem), q_desc = desc_k(base + kQOff + t * kOperand), k_desc = desc_k(base + kKOff), v_desc = desc_mn(base + kVOff);
            const uint32_t s_at = tmem + t * 128, o_at = tmem + 256 + t * 128;
            uint32_t it = 0, use = 0, unit = 0;              // blocks of K and V; steps and units of this half
            // step j of a unit is the second half of a block (keys 64 ..) for even j, the first for odd j, in buffer j % 2 of 64 columns
            auto s_product = [&](int st, uint32_t j) {
                const uint32_t k0 = k_desc + st * (kOperand >> 4) + (1 - (j & 1)) * (8192 >> 4), d = s_at + (j & 1) * 64;
                tc_fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) {
                        const uint32_t o = ((ks >> 2) * 16384 + (ks & 3) * 32) >> 4;
                        mma_ss(d, q_desc + o, k0 + o, ks ? 1u : 0u);
                    }
                    mma_commit(&sh.s_full[t][j & 1]);
                }
            };
            while (ok && walk_unit(a, w)) {
                const int b0 = w.b, blocks = w.b1 - b0;
                if (t < halves_of(a, w)) {
                    const uint32_t steps = 2 * blocks;
                    ok = wait_all(&sh.q_full[t], unit++ & 1) && wait_all(&sh.k_full[it & 1], it / 2 & 1);
                    if (ok) {
                        s_product(it & 1, 0);
                        s_product(it & 1, 1);
                        if (elect_one()) mma_commit(&sh.k_free[it & 1]);
                    }
                    for (uint32_t j = 0; j < steps && ok; ++j) {
                        const uint32_t blk = it + j / 2;
                        if (!(j & 1) && !(ok = wait_all(&sh.v_full[blk & 1], blk / 2 & 1))) break;
                        if (!(ok = wait_all(&sh.p_full[t][j & 1], (use + j) / 2 & 1))) break;
                        tc_fence_after();
                        const uint32_t v0 = v_desc + (blk & 1) * (kOperand >> 4) + (1 - (j & 1)) * (8192 >> 4), p0 = s_at + (j & 1) * 64;
                        if (elect_one()) {
#pragma unroll
                            for (int ks = 0; ks < 4; ++ks)
                                mma_ts(o_at, p0 + ks * 8, v0 + ks * (2048 >> 4), ks || j ? 1u : 0u);
                            mma_commit(&sh.o_step[t][j & 1]);
                            if (j & 1) mma_commit(&sh.v_free[blk & 1]);
                        }
                        if (j + 2 < steps) {
                            if (!(j & 1) && !(ok = wait_all(&sh.k_full[(blk + 1) & 1], (blk + 1) / 2 & 1))) break;
                            if (!(ok = wait_all(&sh.o_step[t][j & 1], (use + j) / 2 & 1))) break;
                            s_product((blk + 1) & 1, j);
                            if ((j & 1) && elect_one()) mma_commit(&sh.k_free[(blk + 1) & 1]);
                        }
                    }
                    use += steps;
                    it += blocks;
                } else {
                    for (int i = 0; i < blocks && ok; ++i, ++it) {       // no rows in this half: the stages come back at once
                        ok = wait_all(&sh.k_full[it & 1], it / 2 & 1);
                        if (ok && lane == 0) mbar_arrive(&sh.k_free[it & 1]);
                        ok = ok && wait_all(&sh.v_full[it & 1], it / 2 & 1);
                        if (ok && lane == 0) mbar_arrive(&sh.v_free[it & 1]);
                    }
                }
                walk_on(a, w, b0);
            }
            if (!ok) {                                       // what is in flight ends before the memory is given back
                sh.abort = 1;
                if (elect_one()) mma_commit(&sh.drain[warp - 12]);
                const int never = 0;
                mbar_wait(&sh.drain[warp - 12], 0, &never);
            }
        }
        __syncwarp();
    } else {
        // ---- softmax -------------------------------------------------------------------------------------------------
        const int t = warp >> 2, r = (warp & 3) * 32 + lane;            // half, row in it
        const uint32_t t_lane = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t t_o = t_lane + 256 + t * 128;
        uint32_t it = 0, use = 0;                            // blocks; steps of this half
        while (walk_unit(a, w)) {                            // (whatever happens, a warp goes one way)
            const int b0 = w.b;
            if (t >= halves_of(a, w)) {
                it += w.b1 - b0;
                walk_on(a, w, b0);
                continue;
            }
            const int row = w.rt * kTileRows + t * kHalf + r, j = row / a.G, hq = w.h * a.G + row % a.G;
            const bool real = j < w.sq.more;
            float rs;
            {
                const unsigned char *qp = reinterpret_cast<const unsigned char *>(a.q) + 2 * (w.n * a.qs[0] + hq * a.qs[1] + j * a.qs[2]);
                float top = 0.f;
                if (real)
#pragma unroll 4
                    for (int i = 0; i < 16; ++i) {
                        const uint4 u = *reinterpret_cast<const uint4 *>(qp + 16 * i);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 x = unpack2<BF>((&u.x)[e]);
                            top = fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y)));
                        }
                    }
                const int e = top > 0.f ? max((int)(__float_as_uint(top) >> 23) - 127 - 12, -126) : 0;
                const float inv = a.scale < 0.f ? -pow2i(-e) : pow2i(-e);          // scores' factors are not negative
                rs = fabsf(a.scale) * pow2i(e) * kLog2e;
                const uint32_t q0 = smem_u32(smem) + kQOff + t * kOperand + r * 128;
#pragma unroll 4
                for (int i = 0; i < 16; ++i) {
                    uint4 u = make_uint4(0, 0, 0, 0);
                    if (real) u = *reinterpret_cast<const uint4 *>(qp + 16 * i);
                    uint32_t o[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float2 x = unpack2<BF>((&u.x)[k]);
                        o[k] = pack2<false>(x.x * inv, x.y * inv);
                    }
                    sts16(q0 + (i >> 3) * 16384 + (((i & 7) ^ (r & 7)) * 16), o[0], o[1], o[2], o[3]);
                }
            }
            proxy_fence();
            mbar_arrive(&sh.q_full[t]);
            __syncwarp();
            const int lim = real ? w.sq.have + j : 0x7fffffff;
            const int all_see = w.sq.have + (w.rt * kTileRows + t * kHalf) / a.G;
            const float slope2 = MOD && a.slopes && real ? a.slopes[hq] * kLog2e : 0.f;
            float m = kNone, D = 0.f, l = 0.f;
            float edge = kNone;                              // what a score has to exceed to move a maximum
            bool wide = false;                               // the block's tokens have scales of their own
            bool huge = false;                               // scores beside which the lift below would be lost
            // -inf where a step has to go the careful way
            auto edge_of = [&](float ey) { return huge || wide || D - ey > kApart ? -INFINITY : m + kSlack + fminf(D - ey, 0.f); };
            const int steps = 2 * (w.b1 - b0);
            float2 ex = make_float2(0.f, 0.f);
            float mult = 0.f;
            for (int jj = 0; jj < steps; ++jj, ++use) {
                const int key0 = (w.b1 - 1 - (jj >> 1)) * kBlock + (1 - (jj & 1)) * 64;
                const uint32_t t_s = t_lane + t * 128 + (jj & 1) * 64;
                if (ok) ok = mbar_wait(&sh.s_full[t][jj & 1], use / 2 & 1, gave_up);
                __syncwarp();
                tc_fence_after();
                if (!(jj & 1)) {                             // the block's scales
                    const volatile float2 *exp_at = &sh.exps[(it + (jj >> 1)) & 3];
                    ex = make_float2(exp_at->x, exp_at->y);
                    wide = *reinterpret_cast<volatile int *>(&sh.wide[(it + (jj >> 1)) & 3]);
                    // (wide: all that is asked here is whether there is a score)
                    mult = wide ? 0x1p-100f : rs * ex2(ex.x);
                    edge = edge_of(ex.y);
                }
                uint32_t u[2][32];
                tmem_ld32(t_s, u[0]);
                tmem_ld32(t_s + 32, u[1]);
                tmem_ld_wait();
                // log2-scores where there is a cap, a bias or a key to hide; otherwise the raw products, which have their order
                const bool mask = key0 + 63 > all_see;
                float top = -INFINITY, top2 = -INFINITY;
                auto each = [&](auto f) {
#pragma unroll
                    for (int e = 0; e < 64; ++e) u[e >> 5][e & 31] = __float_as_uint(f(__uint_as_float(u[e >> 5][e & 31]), e));
                };
                if (MOD || mask) {
                    if (MOD && a.softcap > 0.f)
                        each([&](float raw, int) { return capped(raw * mult, a.cap2, a.icap2); });
                    else each([&](float raw, int) { return raw * mult; });
                    if (MOD && a.slopes) {
                        const float far = slope2 * (float)(key0 - lim);
                        each([&](float s, int e) { return s + fmaf(slope2, (float)e, far); });
                    }
                    if (mask) each([&](float s, int e) { return key0 + e > lim ? -INFINITY : s; });
                }
#pragma unroll
                for (int e = 0; e < 64; e += 4) {
                    top = fmaxf(fmaxf(top, __uint_as_float(u[e >> 5][e & 31])), __uint_as_float(u[e >> 5][(e + 1) & 31]));
                    top2 = fmaxf(fmaxf(top2, __uint_as_float(u[e >> 5][(e + 2) & 31])), __uint_as_float(u[e >> 5][(e + 3) & 31]));
                }
                top = fmaxf(top, top2);
                const float unit2 = MOD || mask ? 1.f : mult;
                if (top > -INFINITY) top *= unit2;
                bool careful = false;
                if (__any_sync(0xffffffffu, top > edge)) {
                    const float2 now = join_tops(make_float2(m, D), make_float2(top, ex.y));
                    const float f = ex2(m - now.x + (D - now.y));
                    if (jj) {                                // the values of the step before are in
                        // (an o_step barrier has a phase for every second step, so the one asked for is the current or the last one)
                        if (ok) ok = mbar_wait(&sh.o_step[t][~jj & 1], (use - 1) / 2 & 1, gave_up);
                        __syncwarp();
                        tc_fence_after();
                    }
                    huge = fabsf(now.x) > 0x1p20f && now.x > kNone;
                    careful = wide || __any_sync(0xffffffffu, huge || now.y - ex.y > kApart);
                    if (!careful) {
                        l *= ex2(m - now.x);
                        m = now.x;
                        D = now.y;
                        edge = edge_of(ex.y);
                        if (jj) rescale(t_o, f);
                    }
                }
                if (careful) {
                    Careful c;
                    c.own = wide ? sh.key_exps[(it + (jj >> 1)) & 3] + (1 - (jj & 1)) * 64 : nullptr;
                    c.ex = ex;
                    c.rs = rs;
                    c.slope2 = slope2;
                    c.key0 = key0;
                    c.lim = lim;
                    c.t_s = t_s;
                    c.t_o = t_o;
                    c.carry = jj > 0;
                    const TileRow now = careful_step<MOD>(a, c, TileRow{m, D, l});
                    m = now.m;
                    D = now.D;
                    l = now.l;
                    edge = edge_of(ex.y);
                } else {
                    // weights 2^(score - m - D + log2 sv + kLift), over the columns of the scores
                    const float lift = ex.y + kLift - D, shift = lift - m;
                    float sum = 0.f, sum2 = 0.f;
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint32_t p[16];
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            float x = ex2(fmaf(__uint_as_float(u[half][e]), unit2, shift)), y = ex2(fmaf(__uint_as_float(u[half][e + 1]), unit2, shift));
                            sum += x;
                            sum2 += y;
                            p[e / 2] = pack2<false>(x, y);
                        }
                        tmem_st16(t_s + half * 16, p);
                    }
                    l += (sum + sum2) * ex2(fminf(-lift, kApart));       // (beyond it: a row that sees nothing of this)
                }
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(&sh.p_full[t][jj & 1]);
            }
            it += w.b1 - b0;
            if (ok) ok = mbar_wait(&sh.o_step[t][1], (use - 1) / 2 & 1, gave_up);      // (a unit has an even number of steps)
            __syncwarp();
            tc_fence_after();
            const bool begins = b0 == 0, ends = w.b1 == w.blocks;
            const int slot = 2 * piece.me + (begins ? 1 : 0);
            const size_t orow = ((size_t)w.n * c.H * a.G + hq) * a.Tq + j;
            const bool fix = *reinterpret_cast<volatile int *>(&sh.odd_tail);
            const int paged = w.sq.full * c.page;
#pragma unroll 1
            for (int q = 0; q < 8; ++q) {
                uint32_t u[16];
                __syncwarp();
                tmem_ld16(t_o + q * 16, u);
                tmem_ld_wait();
                if (real) {
                    if (fix) {                               // infinite values of the tail go to the rows that see their token
                        using T = Elem<BF ? kBF16 : kF16>;
                        const typename T::T *tv = reinterpret_cast<const typename T::T *>(c.v_tail) +
                                                  (((size_t)a.layer * c.N + w.n) * c.H + w.h) * ((size_t)c.page * kD) + q * 16;
                        const int last = min(min(lim, w.keys - 1), w.b1 * kBlock - 1) - paged;
                        for (int tok = max(b0 * kBlock - paged, 0); tok <= last && tok < c.page; ++tok)
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                const float x = T::to_f32(tv[(size_t)tok * kD + e]);
                                if (!(fabsf(x) < INFINITY)) u[e] = __float_as_uint(__uint_as_float(u[e]) + x);
                            }
                    }
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const float4 o = make_float4(__uint_as_float(u[e]), __uint_as_float(u[e + 1]), __uint_as_float(u[e + 2]), __uint_as_float(u[e + 3]));
                        if (begins && ends) finish<BF>(a.out, orow * kD + q * 16 + e, o, D, l);
                        else *reinterpret_cast<float4 *>(a.part + ((size_t)slot * kTileRows + t * kHalf + r) * kD + q * 16 + e) = o;
                    }
                }
            }
            __syncwarp();
            tc_fence_before();
            if (real) {
                if (begins && ends) {
                    if (a.lse) a.lse[orow] = (m + log2f(l)) * 0.69314718055994531f;
                } else a.part_ml[slot * kTileRows + t * kHalf + r] = make_float4(m, l, D, 0.f);
            }
            if (!(begins && ends) && tid == 0) a.meta[slot] = make_int2(1, begins ? (w.n * c.H + w.h) * a.tiles + w.rt : (int)ends);
            walk_on(a, w, b0);
        }
    }
    if (!ok) {
        sh.abort = 1;
        atomicOr(c.status, ODMKV_ATTN_EXPIRED);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 12) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512u) : "memory");
}

constexpr size_t kPartBytes = (size_t)2 * kTileCtas * kTileRows * kD * 4;
constexpr size_t kMlBytes = (size_t)2 * kTileCtas * kTileRows * 16;
constexpr size_t kMetaBytes = (size_t)2 * kTileCtas * 8 / 256 * 256 + 256;

template <int FMT, bool BF, bool MOD>
int launch(const BlockAttnArgs &a, cudaStream_t st) {
    static std::atomic<unsigned long long> done{0};
    const int e = allow_smem(block8_tile_kernel<FMT, BF, MOD>, kTileSmem, done);
    if (e) return e;
    block8_tile_kernel<FMT, BF, MOD><<<kTileCtas, kTileThreads, kTileSmem, st>>>(a);
    block8_join_launch(a, kTileCtas, st);
    return launch_status();
}
template <int FMT, bool BF>
int launch(const BlockAttnArgs &a, cudaStream_t st) {
    return a.softcap > 0.f || a.slopes ? launch<FMT, BF, true>(a, st) : launch<FMT, BF, false>(a, st);
}

}  // namespace

size_t block8_tile_workspace_bytes() { return kPartBytes + kMlBytes + kMetaBytes + 256; }

int block8_tile_launch(BlockAttnArgs a, void *workspace, cudaStream_t st) {
    a.tile = a.slot_rows = kTileRows;
    a.tiles = (int)(((long long)a.G * a.Tq + kTileRows - 1) / kTileRows);
    unsigned char *ws = reinterpret_cast<unsigned char *>(workspace);
    a.part = reinterpret_cast<float *>(ws);
    a.part_ml = reinterpret_cast<float4 *>(ws + kPartBytes);
    a.meta = reinterpret_cast<int2 *>(ws + kPartBytes + kMlBytes);
    a.pieces = reinterpret_cast<int *>(ws + kPartBytes + kMlBytes + kMetaBytes);
    if (a.c.code_format == ODMKV_CODE_E4M3) return a.c.tail_dtype == kBF16 ? launch<ODMKV_CODE_E4M3, true>(a, st) : launch<ODMKV_CODE_E4M3, false>(a, st);
    return a.c.tail_dtype == kBF16 ? launch<ODMKV_CODE_INT8, true>(a, st) : launch<ODMKV_CODE_INT8, false>(a, st);
}

}  // namespace odmkv
