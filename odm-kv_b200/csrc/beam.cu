// Selection step of a beam search: the K best continuations of W beams over V tokens (sm_100a).
//
//   score(w, v) = scores[w] + x[w][v] - log sum_u exp(x[w][u]),  best first, equal ones by the lower w V + v.
//
// Inside a beam the order is that of the logits, exactly; only candidates of different beams need the normaliser.  These
// can lie closer together than fp32 resolves at a score of -50 (4e-6), so the sum of exponentials is taken in fp64:
// exp(x - r) = 2^(k / 64) * exp(f), |f| <= ln 2 / 128, the first factor from a table of 64 values, the second a
// polynomial of degree 5 (remainder below 4e-17).  r is the first finite logit a lane meets, and is moved only when a later
// one exceeds it by 200 (the fp64 range holds e^700).
//
// Stage 1, one warp per stretch of a row: reads it once, 16 bytes a lane, and keeps the K best (value, index) in
// registers, sorted, two per lane; a vector none of whose values beats the K-th best costs one vote.  The warps of a CTA
// merge their lists in shared memory.  Stage 2, one CTA per search: the normalisers, then the best K of the lists.
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
    long long pad;
    float *out_scores;
    int64_t *out_parents, *out_tokens;
    double2 *part_sum;       // [B * W, parts] (r, sum)
    float *part_val;         // [B * W, parts, K]
    int32_t *part_idx;       // [B * W, parts, K], -1 behind the last
};

// NaN counts as -inf, +inf as the type's largest number
template <int DT> __device__ __forceinline__ float clean(float x) {
    constexpr float top = DT == kF16 ? 65504.f : DT == kBF16 ? 3.3895313892515355e38f : 3.4028234663852886e38f;
    return x != x ? -INFINITY : fminf(x, top);
}

__device__ __forceinline__ bool ahead(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

// exp(y) for y in [-700, 250]; tab[i] = 2^(i / 64)
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
    if (threadIdx.x < 64) tab[threadIdx.x] = exp2(threadIdx.x / 64.0);
}

// the running list of a warp: entry 32 i + lane, sorted best first; (-inf, INT_MAX) where there is none
struct TopList {
    float v[2];
    int i[2];
};

__device__ __forceinline__ void insert(TopList &t, float v, int i, int lane) {
    const unsigned b0 = __ballot_sync(0xffffffffu, ahead(t.v[0], t.i[0], v, i));
    const unsigned b1 = __ballot_sync(0xffffffffu, ahead(t.v[1], t.i[1], v, i));
    const int at = __popc(b0) + __popc(b1);                          // entries that stay in front
    const float last_v = __shfl_sync(0xffffffffu, t.v[0], 31);
    const int last_i = __shfl_sync(0xffffffffu, t.i[0], 31);
    const float u0 = __shfl_up_sync(0xffffffffu, t.v[0], 1), u1 = __shfl_up_sync(0xffffffffu, t.v[1], 1);
    const int j0 = __shfl_up_sync(0xffffffffu, t.i[0], 1), j1 = __shfl_up_sync(0xffffffffu, t.i[1], 1);
    if (lane + 32 >= at) {
        const bool here = lane + 32 == at;
        t.v[1] = here ? v : (lane ? u1 : last_v);
        t.i[1] = here ? i : (lane ? j1 : last_i);
    }
    if (lane >= at) {
        t.v[0] = lane == at ? v : u0;
        t.i[0] = lane == at ? i : j0;
    }
}

template <int DT>
__global__ void __launch_bounds__(kBeamThreads) beam_part_kernel(const __grid_constant__ BeamArgs a) {
    constexpr int E = DT == kF32 ? 4 : 8;                            // logits in 16 bytes
    using T = typename Elem<DT>::T;
    __shared__ double tab[64];
    __shared__ double2 sums[kBeamWarps];
    __shared__ float lv[kBeamWarps * ODMKV_BEAM_MAX_K];
    __shared__ int li[kBeamWarps * ODMKV_BEAM_MAX_K];
    const int row = blockIdx.y, part = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (a.done && a.done[row]) return;                               // its only continuation needs no logits
    fill_table(tab);
    __syncthreads();
    const T *x = reinterpret_cast<const T *>(a.logits) + (long long)(row / a.W) * a.bs + (long long)(row % a.W) * a.ws;
    const int lo = part * a.part_len, hi = min(a.V, lo + a.part_len);
    TopList top;
    top.v[0] = top.v[1] = -INFINITY;
    top.i[0] = top.i[1] = 0x7fffffff;
    float r = -INFINITY, kth = -INFINITY;
    double sum = 0.0;
    // A lane's place in the row does not depend on the row's address: equal rows have equal sums, bit for bit, and
    // their continuations tie.  (Rows off the 16-byte boundaries are read element by element.)
    const bool wide = ((uintptr_t)(x + lo) & 15) == 0;
    for (int base = lo + warp * 32 * E; base < hi; base += kBeamThreads * E) {
        const int at = base + lane * E;
        float v[E];
        if (wide && at + E <= hi) {
            const uint4 w = *reinterpret_cast<const uint4 *>(x + at);
            const T *p = reinterpret_cast<const T *>(&w);
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = clean<DT>(Elem<DT>::to_f32(p[e]));
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = at + e < hi ? clean<DT>(Elem<DT>::to_f32(x[at + e])) : -INFINITY;
        }
        float best = v[0];
#pragma unroll
        for (int e = 1; e < E; ++e) best = fmaxf(best, v[e]);
        if (best > -INFINITY) {
            if (best > r + 200.f || r == -INFINITY) {                // new reference
                sum = r == -INFINITY ? 0.0 : sum * exp64(fmax((double)r - (double)best, -700.0), tab);
                r = best;
            }
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (v[e] > -INFINITY) sum += exp64(fmax((double)v[e] - (double)r, -700.0), tab);
        }
        // (-inf never enters a list; kth is -inf until the list is full)
        unsigned hits = __ballot_sync(0xffffffffu, best > kth);
        while (hits) {
            const int src = __ffs(hits) - 1;
            hits &= hits - 1;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float c = __shfl_sync(0xffffffffu, v[e], src);
                if (c > kth) {                                       // (an equal value met later has the higher index)
                    insert(top, c, base + src * E + e, lane);
                    kth = __shfl_sync(0xffffffffu, a.K > 32 ? top.v[1] : top.v[0], (a.K - 1) & 31);
                }
            }
        }
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
    for (int i = 0; i < 2; ++i)
        if (lane + 32 * i < a.K) {
            lv[warp * a.K + lane + 32 * i] = top.v[i];
            li[warp * a.K + lane + 32 * i] = top.i[i];
        }
    __syncthreads();
    const size_t slot = (size_t)row * a.parts + part;
    if (threadIdx.x == 0) {
        double2 t = sums[0];
        for (int w = 1; w < kBeamWarps; ++w) t = join(t, sums[w]);
        a.part_sum[slot] = t;
    }
    // rank of every entry among all of them; indices differ, so ranks do (empty entries share one behind all others)
    const int count = kBeamWarps * a.K;
    int real = 0;
    for (int e = 0; e < count; ++e) real += li[e] != 0x7fffffff;
    for (int e = threadIdx.x; e < count; e += kBeamThreads) {
        const float v = lv[e];
        const int i = li[e];
        if (i == 0x7fffffff) continue;
        int rank = 0;
        for (int f = 0; f < count; ++f) rank += ahead(lv[f], li[f], v, i);
        if (rank < a.K) {
            a.part_val[slot * a.K + rank] = v;
            a.part_idx[slot * a.K + rank] = i;
        }
    }
    for (int k = real + threadIdx.x; k < a.K; k += kBeamThreads) a.part_idx[slot * a.K + k] = -1;
}

// Stage 2.  A part's list is sorted, so the best candidate of a search is the best head of its lists: K rounds in which
// the threads find the best head and its list moves on by one.
__global__ void __launch_bounds__(kBeamThreads) beam_join_kernel(const __grid_constant__ BeamArgs a) {
    extern __shared__ unsigned char dyn[];
    double *norm = reinterpret_cast<double *>(dyn);                  // [W] log of the sum of exponentials
    int *head = reinterpret_cast<int *>(norm + a.W);                 // [W * parts]
    __shared__ double tab[64];
    __shared__ double best_s[kBeamWarps];
    __shared__ long long best_i[kBeamWarps];
    __shared__ int best_l[kBeamWarps];
    __shared__ int taken;
    const int b = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int lists = a.W * a.parts;
    fill_table(tab);
    for (int l = threadIdx.x; l < lists; l += kBeamThreads) head[l] = 0;
    __syncthreads();
    for (int w = threadIdx.x; w < a.W; w += kBeamThreads) {
        const int row = b * a.W + w;
        double r = -INFINITY, sum = 0.0;
        if (!(a.done && a.done[row])) {
            for (int p = 0; p < a.parts; ++p) r = fmax(r, a.part_sum[(size_t)row * a.parts + p].x);
            for (int p = 0; p < a.parts; ++p) {
                const double2 t = a.part_sum[(size_t)row * a.parts + p];
                if (t.x > -INFINITY) sum += t.y * exp64(fmax(t.x - r, -700.0), tab);
            }
        }
        norm[w] = r > -INFINITY ? r + log(sum) : 0.0;                // a row of -inf: all its scores are -inf
    }
    __syncthreads();
    int got = 0;
    for (int k = 0; k < a.K; ++k) {
        double s = -INFINITY;
        long long at = 0x7fffffffffffffffLL;
        int from = -1;
        for (int l = threadIdx.x; l < lists; l += kBeamThreads) {
            const int w = l / a.parts, row = b * a.W + w;
            double cs;
            long long ci;
            if (a.done && a.done[row]) {
                if (l % a.parts || head[l]) continue;
                cs = a.scores[row];
                ci = (long long)w * a.V + a.pad;
            } else {
                const size_t e = ((size_t)row * a.parts + l % a.parts) * a.K + head[l];
                if (head[l] >= a.K || a.part_idx[e] < 0) continue;
                cs = (double)a.scores[row] + ((double)a.part_val[e] - norm[w]);
                ci = (long long)w * a.V + a.part_idx[e];
            }
            if (cs > -INFINITY && (cs > s || (cs == s && ci < at))) {
                s = cs;
                at = ci;
                from = l;
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const double s2 = __shfl_xor_sync(0xffffffffu, s, o);
            const long long a2 = __shfl_xor_sync(0xffffffffu, at, o);
            const int f2 = __shfl_xor_sync(0xffffffffu, from, o);
            if (s2 > s || (s2 == s && a2 < at)) { s = s2; at = a2; from = f2; }
        }
        if (lane == 0) { best_s[warp] = s; best_i[warp] = at; best_l[warp] = from; }
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < kBeamWarps; ++w)
                if (best_s[w] > s || (best_s[w] == s && best_i[w] < at)) { s = best_s[w]; at = best_i[w]; from = best_l[w]; }
            taken = from >= 0;
            if (from >= 0) {
                ++head[from];
                a.out_scores[(size_t)b * a.K + k] = (float)s;
                a.out_parents[(size_t)b * a.K + k] = at / a.V;
                a.out_tokens[(size_t)b * a.K + k] = at % a.V;
            }
        }
        __syncthreads();
        if (!taken) break;
        ++got;
    }
    // fewer than K continuations above -inf: the lowest of the others, at -inf
    if (threadIdx.x == 0 && got < a.K) {
        int k = got;
        for (long long i = 0; k < a.K; ++i) {
            bool used = false;
            for (int e = 0; e < got; ++e)
                used |= a.out_parents[(size_t)b * a.K + e] * a.V + a.out_tokens[(size_t)b * a.K + e] == i;
            if (used) continue;
            a.out_scores[(size_t)b * a.K + k] = -INFINITY;
            a.out_parents[(size_t)b * a.K + k] = i / a.V;
            a.out_tokens[(size_t)b * a.K + k] = i % a.V;
            ++k;
        }
    }
}

struct BeamPlan {
    int parts, part_len;
    size_t val_off, idx_off, bytes;
};

// stretches of whole passes of a CTA, as many as fill the device four times
BeamPlan beam_plan(int B, int W, int V, int K) {
    BeamPlan p;
    const int pass = kBeamThreads * 8;           // a multiple of both vector lengths
    const long long rows = (long long)B * W;
    const int most = (V + pass - 1) / pass;
    p.parts = (int)max(1LL, min((long long)most, (148 * 4 + rows - 1) / rows));
    p.part_len = (most + p.parts - 1) / p.parts * pass;
    p.parts = (V + p.part_len - 1) / p.part_len;
    const size_t slots = (size_t)rows * p.parts;
    p.val_off = (slots * sizeof(double2) + 255) / 256 * 256;
    p.idx_off = p.val_off + (slots * K * 4 + 255) / 256 * 256;
    p.bytes = p.idx_off + (slots * K * 4 + 255) / 256 * 256;
    return p;
}

bool beam_sizes_ok(int B, int W, int V, int K) {
    return B > 0 && W > 0 && V > 0 && K > 0 && K <= ODMKV_BEAM_MAX_K && W <= 1024 && (long long)K <= (long long)W * V &&
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
    a.pad = pad_token;
    a.out_scores = out_scores;
    a.out_parents = out_parents;
    a.out_tokens = out_tokens;
    unsigned char *base = reinterpret_cast<unsigned char *>(workspace);
    a.part_sum = reinterpret_cast<double2 *>(base);
    a.part_val = reinterpret_cast<float *>(base + p.val_off);
    a.part_idx = reinterpret_cast<int32_t *>(base + p.idx_off);
    cudaStream_t st = (cudaStream_t)stream;
    const dim3 grid(p.parts, B * W);
    if (dtype == kF16) beam_part_kernel<kF16><<<grid, kBeamThreads, 0, st>>>(a);
    else if (dtype == kBF16) beam_part_kernel<kBF16><<<grid, kBeamThreads, 0, st>>>(a);
    else beam_part_kernel<kF32><<<grid, kBeamThreads, 0, st>>>(a);
    beam_join_kernel<<<B, kBeamThreads, W * sizeof(double) + (size_t)W * p.parts * sizeof(int), st>>>(a);
    return launch_status();
}

}  // extern "C"
