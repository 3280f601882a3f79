// Selection step of a beam search: the K best continuations of W beams over V tokens (sm_100a).
//
//   score(w, v) = scores[w] + x[w][v] - log sum_u exp(x[w][u]),  best first, equal ones by the lower w V + v.
//
// Inside a beam the order is that of the logits, exactly: two that differ by less than fp64 resolves in the scores are not equal.
// Only candidates of different beams need the normaliser; of equal fp64 scores the lower beam's come first.  These
// can lie closer together than fp32 resolves at a score of -50 (4e-6), so the sum of exponentials is taken in fp64:
// exp(x - r) = 2^(k / 64) * exp(f), |f| <= ln 2 / 128, the first factor from a table of 64 values, the second a
// polynomial of degree 5 (remainder below 4e-17).  r is the first finite logit a lane meets, and is moved only when a later
// one exceeds it by 200 (the fp64 range holds e^700).
//
// Stage 1, a CTA per stretch of a row: reads it once, 16 bytes a lane.  The K-th largest of 64 maxima over groups of four
// threads (K > 32: of all threads' maxima) in the first pass is a bound that at least K continuations reach; what beats it is
// put into a list in shared memory, in any order (a few hundred of 14 000 for K = 16), whose best K the CTA ranks at the end.
// A list of more than 512 entries is cut down to its best K before the next pass, and the bound rises to the last of them.  Stage
// 2, one CTA per search: the normalisers, then the best K of the parts' lists, head by head.
// 16 searches of 8 beams over 128256 tokens (26 MB): 60 us, bound by instruction issue (about 75 a logit; without the
// exponentials 45 us, without the lists 41); one search of 4 beams over 32000: 14.5 us, both kernels.
#include "common.cuh"

namespace odmkv {

namespace {

constexpr int kBeamThreads = 256, kBeamWarps = kBeamThreads / 32;

struct BeamArgs {
    const void *logits;
    long long bs, ws;
    const float *scores;
    const uint8_t *done;
    int B, W, V, K, parts, part_len;
    bool staged;             // the lists of a search fit shared memory in the second stage
    long long pad;
    float *out_scores;
    int64_t *out_parents, *out_tokens;
    double2 *part_sum;       // [B * W, parts] (r, sum)
    uint64_t *part_key;      // [B * W, parts, K] (value, index) keys, best first, 0 behind the last
};

// NaN counts as -inf, +inf as the type's largest number
template <int DT> __device__ __forceinline__ float clean(float x) {
    constexpr float top = DT == kF16 ? 65504.f : DT == kBF16 ? 3.3895313892515355e38f : 3.4028234663852886e38f;
    return x != x ? -INFINITY : fminf(x, top);
}

// 2^(i / 64)
__device__ const double kRoots[64] = {
    1.0, 1.0108892860517005, 1.0218971486541166, 1.0330248790212284,
    1.0442737824274138, 1.0556451783605572, 1.0671404006768237, 1.0787607977571199,
    1.0905077326652577, 1.102382583307841, 1.1143867425958924, 1.1265216186082418,
    1.1387886347566916, 1.1511892299529827, 1.1637248587775775, 1.1763969916502812,
    1.189207115002721, 1.202156731452703, 1.215247359980469, 1.22848053610687,
    1.241857812073484, 1.255380757024691, 1.2690509571917332, 1.2828700160787783,
    1.2968395546510096, 1.3109612115247644, 1.3252366431597413, 1.339667524053303,
    1.3542555469368927, 1.3690024229745905, 1.383909881963832, 1.3989796725383112,
    1.4142135623730951, 1.42961333839197, 1.4451808069770467, 1.460917794180647,
    1.4768261459394993, 1.4929077282912648, 1.5091644275934228, 1.5255981507445384,
    1.5422108254079407, 1.559004400237837, 1.5759808451078865, 1.593142151342267,
    1.6104903319492543, 1.6280274218573478, 1.645755478153965, 1.6636765803267364,
    1.681792830507429, 1.7001063537185235, 1.718619298122478, 1.7373338352737062,
    1.7562521603732995, 1.7753764925265212, 1.7947090750031072, 1.8142521755003989,
    1.8340080864093424, 1.8539791250833855, 1.8741676341103, 1.8945759815869656,
    1.9152065613971474, 1.9360617934922943, 1.9571441241754002, 1.978456026387951,
};

// exp(y) for y in [-700, 250]; tab: kRoots in shared memory
__device__ __forceinline__ double exp64(double y, const double *tab) {
    const double magic = 6755399441055744.0;                         // 1.5 * 2^52: rounds to an integer in the low bits
    const double t = fma(y, 92.332482616893656877, magic);           // 64 / ln 2
    const int k = __double2loint(t);
    const double kd = t - magic;
    const double f = fma(kd, -0.010830424696249145459, y);           // ln 2 / 64: |kd| < 2^17, so the product's error is 1e-16
    double p = 1.0 / 120.0;
    p = fma(p, f, 1.0 / 24.0);
    p = fma(p, f, 1.0 / 6.0);
    p = fma(p, f, 0.5);
    p = fma(p, f, 1.0);
    p = fma(p, f, 1.0);
    const double s = tab[k & 63];
    return __hiloint2double(__double2hiint(s) + ((k >> 6) << 20), __double2loint(s)) * p;
}

__device__ __forceinline__ void fill_table(double *tab) {
    if (threadIdx.x < 64) tab[threadIdx.x] = kRoots[threadIdx.x];
}

// (value, index) as one key: larger is better, equal values (zeros of either sign too) by the lower index; 0 lies behind
// every key of a number
__device__ __forceinline__ uint64_t key_of(float v, int i) {
    const uint32_t u = __float_as_uint(v + 0.f), o = u & 0x80000000u ? ~u : u | 0x80000000u;
    return (uint64_t)o << 32 | (0xffffffffu - (uint32_t)i);
}
__device__ __forceinline__ float key_value(uint64_t k) {
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ int key_index(uint64_t k) { return (int)(0xffffffffu - (uint32_t)k); }

constexpr int kListHalf = 512;                                       // entries after which a list is cut down
constexpr int kListMax = kListHalf + kBeamThreads * 8;               // one more pass may add all it reads

// rank of `mine` among keys[0 .. n): how many are better
__device__ __forceinline__ int rank_of(uint64_t mine, const uint64_t *keys, int n) {
    int r = 0;
#pragma unroll 4
    for (int i = 0; i + 1 < n; i += 2) {
        const ulonglong2 k = *reinterpret_cast<const ulonglong2 *>(keys + i);
        r += (k.x > mine) + (k.y > mine);
    }
    if (n & 1) r += keys[n - 1] > mine;
    return r;
}

template <int DT>
__global__ void __launch_bounds__(kBeamThreads) beam_part_kernel(const __grid_constant__ BeamArgs a) {
    constexpr int E = DT == kF32 ? 4 : 8;                            // logits in 16 bytes
    using T = typename Elem<DT>::T;
    __shared__ __align__(16) uint64_t list[kListMax];
    __shared__ __align__(16) uint64_t best[kBeamThreads];
    // K groups of four threads reach the list's bound, each with at most kListMax / 64 entries
    __shared__ __align__(16) uint64_t shortlist[32 * kListMax / 64];
    __shared__ double tab[64];
    __shared__ double2 sums[kBeamWarps];
    __shared__ int count;
    __shared__ uint64_t bound_s;
    const int row = blockIdx.y, part = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (a.done && a.done[row]) return;                               // its only continuation needs no logits
    const T *x = reinterpret_cast<const T *>(a.logits) + (long long)(row / a.W) * a.bs + (long long)(row % a.W) * a.ws;
    const int lo = part * a.part_len, hi = min(a.V, lo + a.part_len);
    // A thread's place in the row does not depend on the row's address: equal rows have equal sums, bit for bit, and
    // their continuations tie.  (Rows off the 16-byte boundaries are read element by element.)
    const bool wide = ((uintptr_t)(x + lo) & 15) == 0;
    auto load = [&](int at, float (&v)[E]) {
        if (wide && at + E <= hi) {
            const uint4 w = *reinterpret_cast<const uint4 *>(x + at);
            const T *p = reinterpret_cast<const T *>(&w);
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = Elem<DT>::to_f32(p[e]);
            float odd = 0.f;                                         // NaN as soon as one of them is not finite
#pragma unroll
            for (int e = 0; e < E; ++e) odd = fmaf(v[e], 0.f, odd);
            if (odd != odd)
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] = clean<DT>(v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = at + e < hi ? clean<DT>(Elem<DT>::to_f32(x[at + e])) : -INFINITY;
        }
    };
    float v[E], next[E];
    load(lo + tid * E, v);
    fill_table(tab);
    if (tid == 0) count = 0;
    // ---- the first bound
    uint64_t mine = 0;
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (v[e] > -INFINITY) mine = max(mine, key_of(v[e], lo + tid * E + e));
    if (tid == 0) bound_s = 0;
    if (a.K <= 32) {
        mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, 1));
        mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, 2));
        if ((tid & 3) == 0) best[tid >> 2] = mine;
        __syncthreads();
        if (tid < 64) mine = best[tid];
        if (tid < 64 && mine && rank_of(mine, best, 64) == a.K - 1) bound_s = mine;            // (fewer than K maxima: no bound)
    } else {
        best[tid] = mine;
        __syncthreads();
        if (mine && rank_of(mine, best, kBeamThreads) == a.K - 1) bound_s = mine;
    }
    __syncthreads();
    uint64_t bound = bound_s;
    float bound_v = bound ? key_value(bound) : -INFINITY;
    float r = -INFINITY;
    double sum = 0.0;
    const int passes = (hi - lo + kBeamThreads * E - 1) / (kBeamThreads * E);
    for (int i = 0; i < passes; ++i) {
        const int at = lo + i * kBeamThreads * E + tid * E;
        if (i + 1 < passes) load(at + kBeamThreads * E, next);
        float top = v[0];
#pragma unroll
        for (int e = 1; e < E; ++e) top = fmaxf(top, v[e]);
        if (top > -INFINITY) {
            if (top > r + 200.f || r == -INFINITY) {                 // new reference
                sum = r == -INFINITY ? 0.0 : sum * exp64(fmax((double)r - (double)top, -700.0), tab);
                r = top;
            }
            const double rd = r;
            double part_sum[2] = {0.0, 0.0};
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const double y = exp64((double)v[e] - rd, tab);      // (nothing sensible below -690, and not used)
                part_sum[e & 1] += v[e] - r > -690.f ? y : 0.0;
            }
            sum += part_sum[0] + part_sum[1];
            if (top >= bound_v) {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (v[e] >= bound_v && v[e] > -INFINITY) {
                        const uint64_t k = key_of(v[e], at + e);
                        if (k >= bound) list[atomicAdd(&count, 1)] = k;
                    }
            }
        }
        __syncthreads();
        const int n = count;
        __syncthreads();                                             // (all have read it, and take the same way)
        if (n > kListHalf && i + 1 < passes) {
            // Cut down: K rounds, each takes the best entry left; a thread looks over its share of the list once and again only
            // when it has lost its best.
            uint64_t own = 0;
            int own_at = -1;
            auto scan = [&]() {
                own = 0;
                for (int j = tid; j < n; j += kBeamThreads)
                    if (list[j] > own) { own = list[j]; own_at = j; }
            };
            scan();
            uint64_t kept = 0;
            for (int k = 0; k < a.K; ++k) {
                uint64_t b = own;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, o));
                if (lane == 0) best[warp] = b;
                __syncthreads();
                b = best[0];
                for (int w = 1; w < kBeamWarps; ++w) b = max(b, best[w]);
                if (b == own && own) {
                    list[own_at] = 0;
                    scan();
                }
                if (tid == k) kept = b;
                bound = b;
                bound_v = key_value(b);
                __syncthreads();
            }
            if (tid < a.K) list[tid] = kept;
            if (tid == 0) count = a.K;
            __syncthreads();
        }
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = next[e];
    }
    // one (r, sum) per warp, then per CTA
    auto join = [&](double2 p, double2 q) {
        if (!(p.x >= q.x)) { const double2 t = p; p = q; q = t; }
        if (q.x > -INFINITY) p.y += q.y * exp64(fmax(q.x - p.x, -700.0), tab);
        return p;
    };
    double2 s = make_double2(r, sum);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        s = join(s, make_double2(__shfl_xor_sync(0xffffffffu, s.x, o), __shfl_xor_sync(0xffffffffu, s.y, o)));
    if (lane == 0) sums[warp] = s;
    // Ranking a few hundred entries against one another was half of this kernel: the bound of the first pass once more, over the
    // list, leaves a few dozen.
    int n = count;
    const uint64_t *last = list;
    if (a.K <= 32 && n > 2 * a.K) {
        __syncthreads();
        if (tid == 0) { count = 0; bound_s = 0; }
        mine = 0;
        for (int j = tid; j < n; j += kBeamThreads) mine = max(mine, list[j]);
        mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, 1));
        mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, 2));
        if ((tid & 3) == 0) best[tid >> 2] = mine;
        __syncthreads();
        if (tid < 64) mine = best[tid];
        if (tid < 64 && mine && rank_of(mine, best, 64) == a.K - 1) bound_s = mine;
        __syncthreads();
        if (bound_s) {                                               // (fewer than K groups have an entry: all are ranked)
            for (int j = tid; j < n; j += kBeamThreads)
                if (list[j] >= bound_s) shortlist[atomicAdd(&count, 1)] = list[j];
            __syncthreads();
            n = count;
            last = shortlist;
        }
    }
    const size_t slot = (size_t)row * a.parts + part;
    for (int j = tid; j < n; j += kBeamThreads) {
        const uint64_t k = last[j];
        const int at = rank_of(k, last, n);
        if (at < a.K) a.part_key[slot * a.K + at] = k;
    }
    for (int k = n + tid; k < a.K; k += kBeamThreads) a.part_key[slot * a.K + k] = 0;
    __syncthreads();
    if (tid == 0) {
        double2 t = sums[0];
        for (int w = 1; w < kBeamWarps; ++w) t = join(t, sums[w]);
        a.part_sum[slot] = t;
    }
}

// Stage 2.  A part's list is sorted, so the best candidate of a search is the best head of its lists.  All warps load the lists
// and compute the normalisers; then one warp, its lanes knowing the heads of their lists, takes the best head K times.
__device__ __forceinline__ uint64_t order64(double x) {
    const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);      // -0 and +0 are equal
    return u >> 63 ? ~u : u | 1ull << 63;
}

__global__ void __launch_bounds__(kBeamThreads) beam_join_kernel(const __grid_constant__ BeamArgs a) {
    extern __shared__ unsigned char dyn[];
    double2 *base = reinterpret_cast<double2 *>(dyn);                // [W] a beam's score, and what its logits are counted from
    uint64_t *keys = reinterpret_cast<uint64_t *>(base + a.W);       // [W * parts, K] where there is room
    // [W * parts] list's beam << 8 | its next entry (K: none; 255: the one continuation of a finished beam)
    int *head = reinterpret_cast<int *>(keys + (a.staged ? (size_t)a.W * a.parts * a.K : 0));
    __shared__ double tab[64];
    __shared__ double won_s[ODMKV_BEAM_MAX_K];
    __shared__ long long won_i[ODMKV_BEAM_MAX_K];
    const int b = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int lists = a.W * a.parts;
    fill_table(tab);
    const uint64_t *from_keys = a.part_key + (size_t)b * lists * a.K;
    if (a.staged) {
        for (int i = tid; i < lists * a.K; i += kBeamThreads) keys[i] = from_keys[i];       // (of finished beams: not looked at)
        from_keys = keys;
    }
    __syncthreads();
    for (int w = warp; w < a.W; w += kBeamWarps) {
        const int row = b * a.W + w;
        double r = -INFINITY, sum = 0.0;
        const bool done = a.done && a.done[row];
        if (!done) {
            for (int p = lane; p < a.parts; p += 32) r = fmax(r, a.part_sum[(size_t)row * a.parts + p].x);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) r = fmax(r, __shfl_xor_sync(0xffffffffu, r, o));
            for (int p = lane; p < a.parts; p += 32) {
                const double2 t = a.part_sum[(size_t)row * a.parts + p];
                if (t.x > -INFINITY) sum += t.y * exp64(fmax(t.x - r, -700.0), tab);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
        for (int p = lane; p < a.parts; p += 32) head[w * a.parts + p] = w << 8 | (done ? (p ? a.K : 255) : 0);
        if (lane == 0) base[w] = make_double2(a.scores[row], r > -INFINITY ? r + log(sum) : 0.0);     // (a row of -inf: nothing in its lists)
    }
    __syncthreads();
    if (warp) return;
    // best of the lane's heads: ordered score (0: none), beam, (logit, index), w V + v, list
    uint64_t mine, mine_k = 0;
    long long at = 0;
    int from = 0, mine_w = 0;
    auto look = [&]() {
        mine = 0;
        for (int l = lane; l < lists; l += 32) {
            const int w = head[l] >> 8, h = head[l] & 255;
            const double2 from_beam = base[w];
            double cs = from_beam.x;
            long long ci = (long long)w * a.V;
            uint64_t k = 0;
            if (h < a.K) {
                k = from_keys[(size_t)l * a.K + h];
                if (!k) continue;
                cs += (double)key_value(k) - from_beam.y;
                ci += key_index(k);
            } else if (h == 255) ci += a.pad;
            else continue;
            const uint64_t o = order64(cs);
            if (cs > -INFINITY && (o > mine || (o == mine && (w < mine_w || (w == mine_w && k > mine_k))))) {
                mine = o;
                mine_w = w;
                mine_k = k;
                at = ci;
                from = l;
            }
        }
    };
    look();
    int got = 0;
    for (; got < a.K; ++got) {
        const uint32_t hi = (uint32_t)(mine >> 32), top_hi = __reduce_max_sync(0xffffffffu, hi);
        const uint32_t lo = hi == top_hi ? (uint32_t)mine : 0u, top_lo = __reduce_max_sync(0xffffffffu, lo);
        unsigned best = __ballot_sync(0xffffffffu, hi == top_hi && (uint32_t)mine == top_lo);
        if (!(top_hi | top_lo)) break;
        while (best & (best - 1)) {                                  // equal scores: the lower beam, in it the larger (logit, index)
            const int x = __ffs(best) - 1, y = __ffs(best & (best - 1)) - 1;
            const int xw = __shfl_sync(0xffffffffu, mine_w, x), yw = __shfl_sync(0xffffffffu, mine_w, y);
            const uint64_t xk = __shfl_sync(0xffffffffu, mine_k, x), yk = __shfl_sync(0xffffffffu, mine_k, y);
            best &= ~(1u << (xw < yw || (xw == yw && xk > yk) ? y : x));
        }
        if (best >> lane & 1) {
            won_s[got] = __longlong_as_double((long long)(mine >> 63 ? mine & ~(1ull << 63) : ~mine));
            won_i[got] = at;
            head[from] = (head[from] & 255) == 255 ? (head[from] & ~255) | a.K : head[from] + 1;
            look();
        }
        __syncwarp();
    }
    // fewer than K continuations above -inf: the lowest of the others, at -inf
    if (lane == 0) {
        int k = got;
        for (long long i = 0; k < a.K; ++i) {
            bool used = false;
            for (int e = 0; e < got; ++e) used |= won_i[e] == i;
            if (used) continue;
            won_s[k] = -INFINITY;
            won_i[k++] = i;
        }
    }
    __syncwarp();
    for (int k = lane; k < a.K; k += 32) {
        a.out_scores[(size_t)b * a.K + k] = (float)won_s[k];
        a.out_parents[(size_t)b * a.K + k] = won_i[k] / a.V;
        a.out_tokens[(size_t)b * a.K + k] = won_i[k] % a.V;
    }
}

struct BeamPlan {
    int parts, part_len;
    size_t key_off, bytes;
};

// stretches of whole passes of a CTA, as many as give an SM six CTAs
BeamPlan beam_plan(int B, int W, int V, int K) {
    BeamPlan p;
    const int pass = kBeamThreads * 8;           // a multiple of both vector lengths
    const long long rows = (long long)B * W;
    const int most = (V + pass - 1) / pass;
    p.parts = (int)max(1LL, min((long long)most, (148 * 6 + rows - 1) / rows));
    p.part_len = (most + p.parts - 1) / p.parts * pass;
    p.parts = (V + p.part_len - 1) / p.part_len;
    const size_t slots = (size_t)rows * p.parts;
    p.key_off = (slots * sizeof(double2) + 255) / 256 * 256;
    p.bytes = p.key_off + (slots * K * 8 + 255) / 256 * 256;
    return p;
}

bool beam_sizes_ok(int B, int W, int V, int K) {
    return B > 0 && W > 0 && V > 0 && K > 0 && K <= ODMKV_BEAM_MAX_K && W <= 1024 && V <= (1 << 30) && (long long)K <= (long long)W * V &&
           (long long)B * W <= 65535;
}

}  // namespace
}  // namespace odmkv

using namespace odmkv;

extern "C" {

size_t odmkv_beam_select_workspace_bytes(int B, int W, int V, int K) {
    return beam_sizes_ok(B, W, V, K) ? beam_plan(B, W, V, K).bytes : 0;
}

int odmkv_beam_select(const void *logits, int dtype, const int64_t *strides, const float *scores, const uint8_t *done, int B,
                      int W, int V, int K, int64_t pad_token, float *out_scores, int64_t *out_parents, int64_t *out_tokens,
                      void *workspace, size_t workspace_bytes, void *stream) {
    if (!logits || !strides || !scores || !out_scores || !out_parents || !out_tokens) return ODMKV_ERR_ARG;
    if (dtype != kF16 && dtype != kBF16 && dtype != kF32) return ODMKV_ERR_UNSUPPORTED;
    if (B <= 0 || W <= 0 || V <= 0 || K <= 0 || (long long)K > (long long)W * V) return ODMKV_ERR_SHAPE;
    if (!beam_sizes_ok(B, W, V, K)) return ODMKV_ERR_LIMIT;
    if (pad_token < 0 || pad_token >= V) return ODMKV_ERR_ARG;
    const BeamPlan p = beam_plan(B, W, V, K);
    if (!workspace || workspace_bytes < p.bytes || ((uintptr_t)workspace & 255)) return ODMKV_ERR_WORKSPACE;
    BeamArgs a;
    a.logits = logits;
    a.bs = strides[0];
    a.ws = strides[1];
    a.scores = scores;
    a.done = done;
    a.B = B; a.W = W; a.V = V; a.K = K;
    a.parts = p.parts;
    a.part_len = p.part_len;
    const size_t heads = W * sizeof(double2) + (size_t)W * p.parts * sizeof(int), lists = (size_t)W * p.parts * K * 8;
    a.staged = heads + lists <= 40960;
    a.pad = pad_token;
    a.out_scores = out_scores;
    a.out_parents = out_parents;
    a.out_tokens = out_tokens;
    unsigned char *base = reinterpret_cast<unsigned char *>(workspace);
    a.part_sum = reinterpret_cast<double2 *>(base);
    a.part_key = reinterpret_cast<uint64_t *>(base + p.key_off);
    cudaStream_t st = (cudaStream_t)stream;
    const dim3 grid(p.parts, B * W);
    if (dtype == kF16) beam_part_kernel<kF16><<<grid, kBeamThreads, 0, st>>>(a);
    else if (dtype == kBF16) beam_part_kernel<kBF16><<<grid, kBeamThreads, 0, st>>>(a);
    else beam_part_kernel<kF32><<<grid, kBeamThreads, 0, st>>>(a);
    beam_join_kernel<<<B, kBeamThreads, heads + (a.staged ? lists : 0), st>>>(a);
    return launch_status();
}

}  // extern "C"
