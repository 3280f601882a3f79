// Paged 8-bit cache: causal attention of the running tokens over everything stored (sm_100a).
#include "block8.cuh"

namespace odmkv {

namespace {

struct BlockAttnArgs {
    odmkv_block_cache c;
    const void *q;
    long long qs[3];
    const float *slopes;
    void *out;
    float *lse;
    int layer, G, Tq;
    float scale, softcap;
};

__device__ __forceinline__ float code_f32(uint32_t byte, int fmt) {
    if (fmt == ODMKV_CODE_INT8) return (float)(int8_t)byte;
    const __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3);
    return __half2float(*reinterpret_cast<const __half *>(&h));
}

// One warp per query row: four coordinates a lane, online softmax key by key in fp32.
template <int DT>
__global__ void __launch_bounds__(128) block8_plain_kernel(const __grid_constant__ BlockAttnArgs a) {
    const odmkv_block_cache &c = a.c;
    const int lane = threadIdx.x & 31, Hq = c.H * a.G;
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= (long long)c.N * Hq * a.Tq) return;
    const int j = (int)(row % a.Tq), hq = (int)(row / a.Tq % Hq), n = (int)(row / a.Tq / Hq), h = hq / a.G;
    const int have = max(c.lens[n], 0), more = max(c.new_lens[n], 0);
    const int full = min((have + more) / c.page, c.width);
    const int qpos = have + j, keys = j < more ? qpos + 1 : 0;
    const float4 q = load4<DT>(a.q, n * a.qs[0] + hq * a.qs[1] + j * a.qs[2] + lane * 4);
    const float slope = a.slopes ? a.slopes[hq] : 0.f;
    float m = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int t = 0; t < keys; ++t) {
        float4 k, v;
        if (t / c.page < full) {
            const int p = c.table[(size_t)n * c.width + t / c.page];
            const bool there = p >= 0 && p < c.pages;
            const size_t head = ((size_t)a.layer * c.pages + (there ? p : 0)) * c.H + h;
            const size_t at = (head * c.page + t % c.page) * kD + lane * 4;
            const uint32_t kw = *reinterpret_cast<const uint32_t *>(c.k_codes + at), vw = *reinterpret_cast<const uint32_t *>(c.v_codes + at);
            const float ks = there ? c.k_scale[head] : NAN, vs = there ? c.v_scale[head] : NAN;
            k = make_float4(code_f32(kw & 255, c.code_format) * ks, code_f32(kw >> 8 & 255, c.code_format) * ks,
                            code_f32(kw >> 16 & 255, c.code_format) * ks, code_f32(kw >> 24, c.code_format) * ks);
            v = make_float4(code_f32(vw & 255, c.code_format) * vs, code_f32(vw >> 8 & 255, c.code_format) * vs,
                            code_f32(vw >> 16 & 255, c.code_format) * vs, code_f32(vw >> 24, c.code_format) * vs);
        } else {
            const size_t at = ((((size_t)a.layer * c.N + n) * c.H + h) * c.page + t % c.page) * kD + lane * 4;
            k = load4<DT>(c.k_tail, at);
            v = load4<DT>(c.v_tail, at);
        }
        float s = warp_sum(q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w) * a.scale;
        if (a.softcap > 0.f) s = a.softcap * tanhf(s / a.softcap);
        s += slope * (float)(t - qpos);
        const float mn = fmaxf(m, s), f = __expf(m - mn), p = __expf(s - mn);
        m = mn;
        l = l * f + p;
        acc = make_float4(acc.x * f + p * v.x, acc.y * f + p * v.y, acc.z * f + p * v.z, acc.w * f + p * v.w);
    }
    const float inv = keys ? 1.f / l : 0.f;
    store4<DT>(a.out, (size_t)row * kD + lane * 4, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
    if (a.lse && lane == 0) a.lse[row] = keys ? m + logf(l) : -INFINITY;
}

}  // namespace
}  // namespace odmkv

using namespace odmkv;

extern "C" {

size_t odmkv_block8_attn_workspace_bytes(int N, int H, int G, int Tq, int width, int page) {
    (void)N; (void)H; (void)G; (void)Tq; (void)width; (void)page;
    return 256;
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
    a.scale = scale;
    a.softcap = softcap;
    cudaStream_t st = (cudaStream_t)stream;
    const long long rows = (long long)cache->N * cache->H * G * Tq;
    if (rows > 0x7fffffffLL) return ODMKV_ERR_LIMIT;
    if (cache->tail_dtype == kBF16) block8_plain_kernel<kBF16><<<(int)((rows + 3) / 4), 128, 0, st>>>(a);
    else block8_plain_kernel<kF16><<<(int)((rows + 3) / 4), 128, 0, st>>>(a);
    return launch_status();
}

}  // extern "C"
