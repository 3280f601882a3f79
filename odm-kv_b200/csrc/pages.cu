// Paged 8-bit cache: taking, sharing, giving back and moving pages (sm_100a).
//
// A page is free when no table entry names it (refs = 0); there is no free list, so every result depends on the state
// alone and not on the order in which blocks ran (a quarter of 256 sequences out and in, 33 000 pages: 12 us).  Full pages never change, so a copy of a sequence is its table row
// with the references counted up, and only the tail -- the tokens behind the last full page -- is copied as data.
#include "block8.cuh"

namespace odmkv {

namespace {

constexpr int kBeginThreads = 1024;

__device__ __forceinline__ int block_excl_scan(int v, int *warp_sums, int &total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) warp_sums[w] = x;
    __syncthreads();
    if (w == 0) {
        int s = lane < (int)(blockDim.x >> 5) ? warp_sums[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += y;
        }
        warp_sums[lane] = s;
    }
    __syncthreads();
    const int before = w ? warp_sums[w - 1] : 0;
    total = warp_sums[31];
    __syncthreads();
    return before + x - v;
}

// One CTA.  need[n] = pages that sequence n completes in this step; then one pass over the references counts the free
// pages (only as far as needed), and a second one deals them out, lowest page to the first sequence that needs one.
__global__ void __launch_bounds__(kBeginThreads) begin_kernel(const __grid_constant__ odmkv_block_cache c, const int32_t *new_lens,
                                                              int new_all) {
    extern __shared__ int off[];                 // [N + 1] first page of sequence n among those dealt out; then [N]
    __shared__ int warp_sums[32];
    __shared__ int carry_s;
    int *first = off + c.N + 1;                  // pages that the sequence has
    const int tid = threadIdx.x, lg = 31 - __clz(c.page);
    int carry = 0;
    for (int base = 0; base < c.N; base += kBeginThreads) {
        const int n = base + tid;
        int need = 0;
        if (n < c.N) {
            const long long have = max((long long)c.lens[n] + c.new_lens[n], 0LL);
            long long more = max(new_lens ? new_lens[n] : new_all, 0);
            if ((have + more) >> lg > c.width) {
                atomicOr(c.status, ODMKV_PAGES_TABLE_FULL);
                more = 0;
            }
            c.lens[n] = (int)have;
            c.new_lens[n] = (int)more;
            first[n] = (int)(have >> lg);
            need = (int)((have + more) >> lg) - first[n];
        }
        int total;
        const int before = block_excl_scan(need, warp_sums, total);
        if (n < c.N) off[n] = carry + before;
        carry += total;
    }
    if (tid == 0) off[c.N] = carry;
    __syncthreads();
    if (carry == 0) return;
    auto free_mask = [&](long long p0) {         // bit i: page p0 + i is free
        if (p0 + 4 <= c.pages && ((uintptr_t)c.refs & 15) == 0) {
            const int4 x = *reinterpret_cast<const int4 *>(c.refs + p0);
            return (unsigned)((x.x == 0) | (x.y == 0) << 1 | (x.z == 0) << 2 | (x.w == 0) << 3);
        }
        unsigned m = 0;
        for (int i = 0; i < 4 && p0 + i < c.pages; ++i) m |= (unsigned)(c.refs[p0 + i] == 0) << i;
        return m;
    };
    int free_pages = 0;                          // counted 32768 at a time, eight loads in flight
    for (long long base = 0; base < c.pages && free_pages < carry; base += kBeginThreads * 32) {
        int v = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) v += __popc(free_mask(base + (i * kBeginThreads + tid) * 4));
        int total;
        block_excl_scan(v, warp_sums, total);
        free_pages += total;
    }
    if (free_pages < carry) {                    // not enough: in order, each sequence gets all of its pages or none
        if (tid == 0) {
            int left = free_pages, at = 0, next = off[0];
            for (int n = 0; n < c.N; ++n) {
                const int need = off[n + 1] - next;
                next = off[n + 1];
                off[n] = at;
                if (need > left) {
                    c.new_lens[n] = 0;
                    atomicOr(c.status, ODMKV_PAGES_EXHAUSTED);
                } else {
                    at += need;
                    left -= need;
                }
            }
            off[c.N] = at;
            carry_s = at;
        }
        __syncthreads();
        carry = carry_s;
    }
    int dealt = 0;
    unsigned m = free_mask((long long)tid * 4);
    for (long long base = 0; base < c.pages && dealt < carry; base += kBeginThreads * 4) {
        const unsigned next = free_mask(base + (kBeginThreads + tid) * 4);       // (pages that only later passes deal out)
        int total;
        int r = dealt + block_excl_scan(__popc(m), warp_sums, total);
        for (; m && r < carry; m &= m - 1, ++r) {
            const int p = (int)base + tid * 4 + __ffs(m) - 1;
            int lo = 0, hi = c.N;                // the last sequence with off[n] <= r
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (off[mid] <= r) lo = mid; else hi = mid;
            }
            c.table[(size_t)lo * c.width + first[lo] + (r - off[lo])] = p;
            c.refs[p] = 1;
        }
        m = next;
        dealt += total;
    }
}

__global__ void free_kernel(const __grid_constant__ odmkv_block_cache c, const uint8_t *leave) {
    const int n = blockIdx.x;
    if (!leave[n]) return;
    for (int i = threadIdx.x; i < c.width; i += blockDim.x) {
        int32_t *e = c.table + (size_t)n * c.width + i;
        const int p = *e;
        if (p >= 0 && p < c.pages) atomicSub(&c.refs[p], 1);
        *e = -1;
    }
    if (threadIdx.x == 0) {
        c.lens[n] = 0;
        c.new_lens[n] = 0;
    }
}

struct ForkArgs {
    odmkv_block_cache c;
    const int64_t *parents;
    int W;
};

__device__ __forceinline__ int parent_of(const ForkArgs &a, int b, int w) {
    const int64_t p = a.parents[(size_t)b * a.W + w];
    return p >= 0 && p < a.W ? (int)p : w;
}

// Table rows, references and lengths: a thread owns one column of a search, reads it for all beams and writes it back
// reordered, so no second table is needed.  An entry of a beam with m children gains m - 1 references.
__global__ void fork_table_kernel(const __grid_constant__ ForkArgs a) {
    const odmkv_block_cache &c = a.c;
    const int b = blockIdx.y, i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= c.width + 2) return;                       // two more columns: the lengths
    int32_t *col = i < c.width ? c.table + (size_t)b * a.W * c.width + i : (i == c.width ? c.lens : c.new_lens) + (size_t)b * a.W;
    const size_t step = i < c.width ? c.width : 1;
    int32_t old[ODMKV_FORK_MAX_BEAMS];
    int kids[ODMKV_FORK_MAX_BEAMS];
    for (int w = 0; w < a.W; ++w) {
        old[w] = col[w * step];
        kids[w] = 0;
    }
    for (int w = 0; w < a.W; ++w) {
        const int p = parent_of(a, b, w);
        ++kids[p];
        if (p != w) col[w * step] = old[p];
        if (i == c.width && a.parents[(size_t)b * a.W + w] != p) atomicOr(c.status, ODMKV_PAGES_BAD_PARENT);
    }
    if (i < c.width)
        for (int w = 0; w < a.W; ++w)
            if (kids[w] != 1 && old[w] >= 0 && old[w] < c.pages) atomicAdd(&c.refs[old[w]], kids[w] - 1);
}

// Tails, after the table: a thread owns 16 bytes of one slot and reads them for all beams that somebody copies before it
// writes any, so the copy works in place for every map of parents (permutations and cycles too).  A CTA stays with one
// search, whose map it keeps in shared memory, and goes over its layers; beams that stay where they are cost nothing.
// 50 MB (16 beams, 32 layers, 8 heads) in 10.4 us, both kernels.
template <int WM>
__global__ void __launch_bounds__(256) fork_tail_kernel(const __grid_constant__ ForkArgs a) {
    const odmkv_block_cache &c = a.c;
    __shared__ int parent_s[WM], used_s[WM];
    const int b = blockIdx.y;
    if (threadIdx.x < WM) {
        const int w = threadIdx.x;
        const int p = w < a.W ? parent_of(a, b, w) : w;
        const int n = b * a.W + (w < a.W ? w : 0);
        parent_s[w] = p;
        used_s[w] = p == w ? 0 : (c.lens[n] + c.new_lens[n]) % c.page;      // slots to copy; lengths are the child's already
    }
    __syncthreads();
    int parent[WM], used[WM], most = 0;
#pragma unroll
    for (int w = 0; w < WM; ++w) {
        parent[w] = parent_s[w];
        used[w] = used_s[w];
        most = max(most, used[w]);
    }
    if (most == 0) return;
    // pieces in use: 16 bytes x (most slots) x heads x sides x layers
    const int per_head = most * 16, per_layer = c.H * per_head;
    const long long total = (long long)per_layer * 2 * c.L;
    const size_t seq = (size_t)c.H * c.page * 16;            // pieces of a sequence in a layer
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const int layer2 = (int)(i / per_layer), r = (int)(i - (long long)layer2 * per_layer);
        const int h = r / per_head, piece = r - h * per_head, t = piece >> 4;
        uint4 *tail = reinterpret_cast<uint4 *>(layer2 & 1 ? c.v_tail : c.k_tail) +
                      ((size_t)(layer2 >> 1) * c.N + (size_t)b * a.W) * seq + (size_t)h * c.page * 16 + piece;
        uint4 x[WM];
#pragma unroll
        for (int w = 0; w < WM; ++w)
            if (t < used[w]) x[w] = tail[(size_t)parent[w] * seq];
#pragma unroll
        for (int w = 0; w < WM; ++w)
            if (t < used[w]) tail[(size_t)w * seq] = x[w];
    }
}

// rank of every live page among the live ones (-1 for a free page), list of the live pages, new references
__global__ void __launch_bounds__(kBeginThreads) compact_plan_kernel(const __grid_constant__ odmkv_block_cache from,
                                                                     const __grid_constant__ odmkv_block_cache to, int32_t *rank,
                                                                     int32_t *order, int32_t *count) {
    __shared__ int warp_sums[32];
    const int tid = threadIdx.x;
    int live = 0;
    for (int base = 0; base < from.pages; base += kBeginThreads * 4) {
        int v = 0, ref[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = base + tid * 4 + i;
            ref[i] = p < from.pages ? from.refs[p] : 0;
            v += ref[i] > 0;
        }
        int total;
        int r = live + block_excl_scan(v, warp_sums, total);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = base + tid * 4 + i;
            if (p >= from.pages) break;
            rank[p] = ref[i] > 0 ? r : -1;
            if (ref[i] > 0) {
                if (r < to.pages) to.refs[r] = ref[i];
                order[r++] = p;
            }
        }
        live += total;
    }
    const bool fits = live <= to.pages;
    __syncthreads();                             // a refused pool's references are zeroed behind the ones written above, by other threads
    for (int p = fits ? live : 0; p < to.pages; p += kBeginThreads)
        if (p + tid < to.pages) to.refs[p + tid] = 0;
    if (tid == 0) {
        *count = fits ? live : -1;
        if (!fits) atomicOr(to.status, ODMKV_PAGES_POOL_SMALL);
    }
}

__global__ void compact_table_kernel(const __grid_constant__ odmkv_block_cache from, const __grid_constant__ odmkv_block_cache to,
                                     const int32_t *rank, const int32_t *count) {
    const bool fits = *count >= 0;
    const size_t total = (size_t)from.N * from.width;
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (size_t)gridDim.x * blockDim.x) {
        const int p = from.table[i];
        to.table[i] = fits && p >= 0 && p < from.pages ? rank[p] : -1;
    }
    const int n = blockIdx.x * blockDim.x + threadIdx.x;
    if (n < from.N && to.lens != from.lens && to.new_lens != from.new_lens) {
        to.lens[n] = fits ? from.lens[n] : 0;
        to.new_lens[n] = fits ? from.new_lens[n] : 0;
    }
}

// one CTA per (page, side, layer) in turn: H * page * 128 contiguous bytes and the H scales (1.07 GB in and out: 183 to 196 us, 5.4 to 5.9 TB/s)
__global__ void __launch_bounds__(256) compact_copy_kernel(const __grid_constant__ odmkv_block_cache from,
                                                           const __grid_constant__ odmkv_block_cache to, const int32_t *order,
                                                           const int32_t *count) {
    const long long items = (long long)max(*count, 0) * from.L * 2;
    const int words = from.H * from.page * (kD / 16);
    for (long long it = blockIdx.x; it < items; it += gridDim.x) {
        const int side = it & 1, layer = (int)((it >> 1) % from.L), j = (int)((it >> 1) / from.L);
        const size_t s = (size_t)layer * from.pages + order[j], d = (size_t)layer * to.pages + j;
        const uint4 *src = reinterpret_cast<const uint4 *>(side ? from.v_codes : from.k_codes) + s * words;
        uint4 *dst = reinterpret_cast<uint4 *>(side ? to.v_codes : to.k_codes) + d * words;
        for (int i = threadIdx.x; i < words; i += 1024) {
            uint4 x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (i + k * 256 < words) x[k] = __ldcs(src + i + k * 256);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (i + k * 256 < words) __stcs(dst + i + k * 256, x[k]);
        }
        for (int h = threadIdx.x; h < from.H; h += 256)
            (side ? to.v_scale : to.k_scale)[d * from.H + h] = (side ? from.v_scale : from.k_scale)[s * from.H + h];
    }
}

}  // namespace
}  // namespace odmkv

using namespace odmkv;

extern "C" {

int odmkv_pages_begin(const odmkv_block_cache *cache, const int32_t *new_lens, int new_all, void *stream) {
    const int rc = block_cache_check(cache, false);
    if (rc != ODMKV_OK) return rc;
    if (!new_lens && new_all < 0) return ODMKV_ERR_SHAPE;
    begin_kernel<<<1, kBeginThreads, (2 * cache->N + 1) * sizeof(int), (cudaStream_t)stream>>>(*cache, new_lens, new_all);
    return launch_status();
}

int odmkv_pages_free(const odmkv_block_cache *cache, const uint8_t *leave, void *stream) {
    const int rc = block_cache_check(cache, false);
    if (rc != ODMKV_OK) return rc;
    if (!leave) return ODMKV_ERR_ARG;
    free_kernel<<<cache->N, 128, 0, (cudaStream_t)stream>>>(*cache, leave);
    return launch_status();
}

int odmkv_pages_fork(const odmkv_block_cache *cache, const int64_t *parents, int W, void *stream) {
    const int rc = block_cache_check(cache, true);
    if (rc != ODMKV_OK) return rc;
    if (!parents) return ODMKV_ERR_ARG;
    if (W <= 0 || cache->N % W) return ODMKV_ERR_SHAPE;
    if (W > ODMKV_FORK_MAX_BEAMS || cache->L > 32767) return ODMKV_ERR_LIMIT;
    if (((uintptr_t)cache->k_tail | (uintptr_t)cache->v_tail) & 15) return ODMKV_ERR_ARG;
    ForkArgs a{*cache, parents, W};
    cudaStream_t st = (cudaStream_t)stream;
    const int B = cache->N / W;
    fork_table_kernel<<<dim3((cache->width + 2 + 127) / 128, B), 128, 0, st>>>(a);
    // about eight CTAs an SM over all searches, none with less than a pass of its own
    const long long pieces = (long long)cache->L * 2 * cache->H * cache->page * 16;
    const dim3 grid((int)max(1LL, min((pieces + 255) / 256, (148LL * 8 + B - 1) / B)), B);
    if (W <= 4) fork_tail_kernel<4><<<grid, 256, 0, st>>>(a);
    else if (W <= 8) fork_tail_kernel<8><<<grid, 256, 0, st>>>(a);
    else if (W <= 16) fork_tail_kernel<16><<<grid, 256, 0, st>>>(a);
    else fork_tail_kernel<32><<<grid, 256, 0, st>>>(a);
    return launch_status();
}

size_t odmkv_pages_compact_workspace_bytes(int pages) { return pages <= 0 ? 0 : (size_t)pages * 8 + 256; }

int odmkv_pages_compact(const odmkv_block_cache *from, const odmkv_block_cache *to, void *workspace, size_t workspace_bytes,
                        void *stream) {
    int rc = block_cache_check(from, true);
    if (rc == ODMKV_OK) rc = block_cache_check(to, true);
    if (rc != ODMKV_OK) return rc;
    if (from->L != to->L || from->N != to->N || from->H != to->H || from->page != to->page || from->width != to->width ||
        from->code_format != to->code_format || from->tail_dtype != to->tail_dtype)
        return ODMKV_ERR_SHAPE;
    if (from->k_codes == to->k_codes || from->v_codes == to->v_codes || from->k_scale == to->k_scale || from->v_scale == to->v_scale ||
        from->table == to->table || from->refs == to->refs || (from->lens == to->lens) != (from->new_lens == to->new_lens))
        return ODMKV_ERR_ARG;
    // a refused move empties the new cache, which shared lengths would not allow: such a pool has to be large enough in any case
    if (from->lens == to->lens && to->pages < from->pages) return ODMKV_ERR_ARG;
    if (((uintptr_t)from->k_codes | (uintptr_t)from->v_codes | (uintptr_t)to->k_codes | (uintptr_t)to->v_codes) & 15) return ODMKV_ERR_ARG;
    if (!workspace || workspace_bytes < odmkv_pages_compact_workspace_bytes(from->pages) || ((uintptr_t)workspace & 255))
        return ODMKV_ERR_WORKSPACE;
    int32_t *count = (int32_t *)workspace, *rank = count + 64, *order = rank + from->pages;
    cudaStream_t st = (cudaStream_t)stream;
    compact_plan_kernel<<<1, kBeginThreads, 0, st>>>(*from, *to, rank, order, count);
    const long long cells = (long long)from->N * from->width;
    compact_table_kernel<<<(int)min((cells + 255) / 256 + from->N / 256 + 1, 1184LL), 256, 0, st>>>(*from, *to, rank, count);
    const long long items = (long long)min(from->pages, to->pages) * from->L * 2;
    compact_copy_kernel<<<(int)min(items, 148LL * 8), 256, 0, st>>>(*from, *to, order, count);
    const size_t tail = (size_t)from->L * from->N * from->H * from->page * kD * 2;
    cudaError_t e = cudaSuccess;
    if (from->k_tail != to->k_tail) e = cudaMemcpyAsync(to->k_tail, from->k_tail, tail, cudaMemcpyDeviceToDevice, st);
    if (e == cudaSuccess && from->v_tail != to->v_tail) e = cudaMemcpyAsync(to->v_tail, from->v_tail, tail, cudaMemcpyDeviceToDevice, st);
    return e != cudaSuccess ? (int)e : launch_status();
}

}  // extern "C"
