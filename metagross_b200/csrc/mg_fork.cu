// Sequences that become copies of other sequences: parallel samples of one
// prompt, beams, prompts with a common prefix.
//
// Committed pages are never written again (a page is quantized once, when it
// fills, and the tokens after it live in the sequence's own staging rows), so
// a copy shares them: the block-table entries are copied and the allocator
// counts the holders (in_use[page]; a page goes back to the free stack when its
// last holder lets go).  What is copied is the exact tail, < P rows per layer;
// a copy of a prefix that ends inside a committed page gets that page's first
// rows dequantized into its staging rows.
//
// Two launches.  fork_release_kernel checks the pairs and releases what the
// targets held (their block-table rows are still needed for the order in
// which pages go back, so nothing of them is overwritten yet);
// fork_share_kernel shares the pages and copies the tails of every layer.
// Bound while no page loses its last holder: the two launches (9 us for a few
// targets, 10 for 64 in 22 layers of 4 heads), then the latency of a CTA's one
// short copy (groups of four loads in flight): 256 prefixes that cut a page, 12
// layers of 12 heads of 64, 32 us with 102 MB moved, 3.2 TB/s.  Where targets
// hold pages of their own the last CTA of the release orders the returned ones,
// pair after pair (push_released, about 2.3 us a pair): 167 us for the 64
// targets with 743 such pages, 597 for the 256 with 1841.
#include "mg_alloc_step.cuh"
#include "mg_common.cuh"

namespace mg {

mg_status check_cache_layout(const mg_cache_layout* L);

namespace {

constexpr int kForkThreads = 256;

struct ForkParams {
    int32_t* free_stack;
    int32_t* n_free;
    int32_t* in_use;
    int64_t num_pages;
    int32_t* block_tables;
    int32_t max_blocks;
    int32_t* seq_lens;
    int32_t batch;
    const int32_t* src;
    const int32_t* dst;
    const int32_t* new_lens;  // null: whole sequences
    int32_t pairs;
    int32_t P;
    int32_t* ws;  // [0] arrivals, [1] pages released for good, [2..] 1 per accepted pair
    int32_t* status;
    // shared pages and tails
    const uint8_t* k_pool;
    const uint8_t* v_pool;
    const float* k_scales;
    const float* v_scales;
    void* staging_k;
    void* staging_v;
    int32_t layers;
    int32_t row;  // Hkv * D elements per token
    int32_t D;
    int32_t scale_th;
    int64_t pool_layer, scale_layer, staging_layer;  // bytes, floats, elements from one layer to the next
};

// Whether pair i can be done: ids in range, the source's length valid and at
// least the new length, and the target neither read by any pair nor the
// target of an earlier one.  Called by the whole CTA.
__device__ __forceinline__ bool pair_ok(const ForkParams& p, int i) {
    const int s = p.src[i], d = p.dst[i];
    bool bad = s < 0 || s >= p.batch || d < 0 || d >= p.batch || s == d;
    if (!bad) {
        const int have = p.seq_lens[s], want = p.new_lens ? p.new_lens[i] : have, old = p.seq_lens[d];
        bad = want < 0 || want > have || have / p.P > p.max_blocks || old < 0 || old / p.P > p.max_blocks;
        for (int k = threadIdx.x; k < p.pairs; k += blockDim.x)
            if (p.src[k] == d || (k < i && p.dst[k] == d)) bad = true;
    }
    return !__syncthreads_or(bad);
}

// The pages that lost their last holder go back to the free stack in the order
// in which releasing the targets one after the other would return them: by the
// last place of the flattened (pair, block-table) list that holds the page.
// One CTA; the released pages are listed, unordered, above the stack's top.
__device__ void push_released(const ForkParams& p, int released) {
    __shared__ int scratch[33];
    const int top = *p.n_free;
    for (int k = threadIdx.x; k < released; k += blockDim.x)
        p.in_use[*(volatile int32_t*)&p.free_stack[top + k]] = -1;
    __threadfence();
    __syncthreads();
    int base = 0;
    for (int i = 0; i < p.pairs; ++i) {
        if (!*(volatile int32_t*)&p.ws[2 + i]) continue;
        const int n = p.seq_lens[p.dst[i]] / p.P;
        const int32_t* bt = p.block_tables + static_cast<int64_t>(p.dst[i]) * p.max_blocks;
        for (int j = threadIdx.x; j < n; j += blockDim.x) {
            const int32_t page = bt[j];
            if (page >= 0 && page < p.num_pages && *(volatile int32_t*)&p.in_use[page] < 0)
                atomicMin(&p.in_use[page], -(base + j) - 2);
        }
        base += n;
    }
    __threadfence();
    __syncthreads();
    base = 0;
    int at = top;
    for (int i = 0; i < p.pairs; ++i) {
        if (!*(volatile int32_t*)&p.ws[2 + i]) continue;
        const int n = p.seq_lens[p.dst[i]] / p.P;
        const int32_t* bt = p.block_tables + static_cast<int64_t>(p.dst[i]) * p.max_blocks;
        for (int start = 0; start < n; start += blockDim.x) {
            const int j = start + threadIdx.x;
            int32_t page = -1;
            int last = 0;
            if (j < n) {
                page = bt[j];
                last = page >= 0 && page < p.num_pages && *(volatile int32_t*)&p.in_use[page] == -(base + j) - 2;
            }
            int cnt;
            const int excl = block_exclusive_scan(last, scratch, &cnt);
            if (last) {
                p.free_stack[at + excl] = page;
                p.in_use[page] = 0;
            }
            at += cnt;
        }
        base += n;
    }
    __syncthreads();
    if (threadIdx.x == 0) *p.n_free = at;
}

// One CTA per pair: check it, release what its target held.
__global__ void __launch_bounds__(kForkThreads) fork_release_kernel(ForkParams p) {
    __shared__ int s_last;
    grid_dependency_wait();
    grid_launch_dependents();
    const int i = blockIdx.x;
    const bool stopped = p.status && (*(volatile int32_t*)p.status & kStopBits);
    const bool ok = !stopped && pair_ok(p, i);
    if (threadIdx.x == 0) {
        p.ws[2 + i] = ok;
        if (!ok) flag(p.status, stopped ? MG_DEV_SKIPPED : MG_DEV_BAD_ARGUMENT);
    }
    if (ok) {
        const int d = p.dst[i], n = p.seq_lens[d] / p.P, top = *p.n_free;
        const int32_t* bt = p.block_tables + static_cast<int64_t>(d) * p.max_blocks;
        for (int j = threadIdx.x; j < n; j += blockDim.x) {
            const int32_t page = bt[j];
            if (page < 0 || page >= p.num_pages) {
                flag(p.status, MG_DEV_BAD_PAGE_ID);
                continue;
            }
            const int holders = atomicSub(&p.in_use[page], 1);
            if (holders <= 0) {
                atomicAdd(&p.in_use[page], 1);
                flag(p.status, MG_DEV_DOUBLE_FREE);
            } else if (holders == 1) {
                const int at = top + atomicAdd(&p.ws[1], 1);
                if (at < p.num_pages) p.free_stack[at] = page;
                else flag(p.status, MG_DEV_DOUBLE_FREE);  // more free pages than there are: the stack was not ours
            }
        }
    }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) s_last = atomicAdd(&p.ws[0], 1) == static_cast<int>(gridDim.x) - 1;
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    const int released = static_cast<int>(min(static_cast<int64_t>(*(volatile int32_t*)&p.ws[1]), p.num_pages - *p.n_free));
    if (released > 0) push_released(p, released);
    __syncthreads();
    if (threadIdx.x == 0) p.ws[0] = p.ws[1] = 0;
}

// One CTA per (pair, layer): the exact rows of K and V; layer 0's also the
// block-table entries, their counts and the length.
template <bool INT4, typename ST>
__global__ void __launch_bounds__(kForkThreads) fork_share_kernel(ForkParams p) {
    grid_dependency_wait();
    grid_launch_dependents();
    const int i = blockIdx.x, layer = blockIdx.y;
    if (!p.ws[2 + i]) return;
    const int s = p.src[i], d = p.dst[i];
    const int have = p.seq_lens[s], want = p.new_lens ? p.new_lens[i] : have;
    const int pages = want / p.P, rows = want - pages * p.P;
    const int32_t* from = p.block_tables + static_cast<int64_t>(s) * p.max_blocks;
    if (layer == 0) {
        int32_t* to = p.block_tables + static_cast<int64_t>(d) * p.max_blocks;
        for (int j = threadIdx.x; j < pages; j += blockDim.x) {
            const int32_t page = from[j];
            if (page >= 0 && page < p.num_pages) atomicAdd(&p.in_use[page], 1);
            else flag(p.status, MG_DEV_BAD_PAGE_ID);
            to[j] = page;
        }
        if (threadIdx.x == 0) p.seq_lens[d] = want;
    }
    const int64_t pe = static_cast<int64_t>(p.P) * p.row;
    const int n8 = static_cast<int>(static_cast<int64_t>(rows) * p.row / 8);
    if (pages == have / p.P) {  // the source's own tail
        constexpr int kWords = 8 * sizeof(ST) / 16;
        const int64_t off = p.staging_layer * layer;
        const uint4* ks = reinterpret_cast<const uint4*>(static_cast<const ST*>(p.staging_k) + off + s * pe);
        const uint4* vs = reinterpret_cast<const uint4*>(static_cast<const ST*>(p.staging_v) + off + s * pe);
        uint4* kd = reinterpret_cast<uint4*>(static_cast<ST*>(p.staging_k) + off + d * pe);
        uint4* vd = reinterpret_cast<uint4*>(static_cast<ST*>(p.staging_v) + off + d * pe);
        constexpr int kBatch = 4;
        for (int e0 = threadIdx.x; e0 < n8 * kWords; e0 += kForkThreads * kBatch) {
            uint4 a[kBatch], b[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int e = e0 + u * kForkThreads;
                if (e < n8 * kWords) a[u] = ks[e], b[u] = vs[e];
            }
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int e = e0 + u * kForkThreads;
                if (e < n8 * kWords) kd[e] = a[u], vd[e] = b[u];
            }
        }
        return;
    }
    // the prefix ends inside a committed page: its first rows, dequantized
    int32_t page = from[pages];
    if (page < 0 || page >= p.num_pages) {
        if (threadIdx.x == 0) flag(p.status, MG_DEV_BAD_PAGE_ID);
        page = 0;
    }
    const int64_t page_at = static_cast<int64_t>(page) * (INT4 ? pe / 2 : pe);
    const uint8_t* pool[2] = {p.k_pool + p.pool_layer * layer + page_at, p.v_pool + p.pool_layer * layer + page_at};
    const float* scales[2] = {p.k_scales + p.scale_layer * layer, p.v_scales + p.scale_layer * layer};
    ST* to[2] = {static_cast<ST*>(p.staging_k) + p.staging_layer * layer + d * pe,
                 static_cast<ST*>(p.staging_v) + p.staging_layer * layer + d * pe};
    const float page_scale[2] = {p.scale_th ? 0.0f : scales[0][page], p.scale_th ? 0.0f : scales[1][page]};
    // K and V of kBatch groups of 8 in flight before the first is stored
    constexpr int kBatch = 4;
    for (int g0 = threadIdx.x; g0 < n8; g0 += kForkThreads * kBatch) {
        uint2 w[kBatch][2];
        float sf[kBatch][2];
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                const int e = (g0 + u * kForkThreads) * 8;
                w[u][kv] = make_uint2(0u, 0u);
                sf[u][kv] = page_scale[kv];
                if (e >= n8 * 8) continue;
                if constexpr (INT4) w[u][kv].x = *reinterpret_cast<const uint32_t*>(pool[kv] + e / 2);
                else w[u][kv] = *reinterpret_cast<const uint2*>(pool[kv] + e);
                // [page][token][head]: one scale per D elements
                if (p.scale_th) sf[u][kv] = scales[kv][static_cast<int64_t>(page) * (pe / p.D) + e / p.D];
            }
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                const int e = (g0 + u * kForkThreads) * 8;
                if (e >= n8 * 8) continue;
                float v[8];
                if constexpr (INT4) {
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        v[q] = static_cast<float>(static_cast<int32_t>(w[u][kv].x << (28 - 4 * q)) >> 28) * sf[u][kv];
                } else {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        v[q] = static_cast<float>(static_cast<int8_t>(w[u][kv].x >> (8 * q))) * sf[u][kv];
                        v[4 + q] = static_cast<float>(static_cast<int8_t>(w[u][kv].y >> (8 * q))) * sf[u][kv];
                    }
                }
                if constexpr (sizeof(ST) == 2) {
                    *reinterpret_cast<uint4*>(to[kv] + e) =
                        make_uint4(pack_half2(v[0], v[1]), pack_half2(v[2], v[3]), pack_half2(v[4], v[5]),
                                   pack_half2(v[6], v[7]));
                } else {
                    *reinterpret_cast<float4*>(to[kv] + e) = make_float4(v[0], v[1], v[2], v[3]);
                    *reinterpret_cast<float4*>(to[kv] + e + 4) = make_float4(v[4], v[5], v[6], v[7]);
                }
            }
    }
}

}  // namespace
}  // namespace mg

using namespace mg;

extern "C" int64_t mg_fork_workspace_bytes(int32_t num_pairs) { return 4ll * (2 + (num_pairs < 0 ? 0 : num_pairs)); }

extern "C" mg_status mg_fork_sequences(const mg_allocator* al, const mg_cache_layout* L, const mg_layer_ptrs* lp,
                                       int32_t num_layers, int32_t* block_tables, int32_t* seq_lens, int32_t batch,
                                       const int32_t* src_ids, const int32_t* dst_ids, const int32_t* new_lens,
                                       int32_t num_pairs, void* workspace, int64_t workspace_bytes,
                                       int32_t* dev_status, mg_stream_t stream) {
    mg_status st = check_cache_layout(L);
    if (st != MG_OK) return st;
    MG_REQUIRE(al && al->free_stack && al->n_free && al->in_use, "null allocator pointer");
    MG_REQUIRE(al->num_pages == L->num_pages, "the allocator and the pools have different page counts");
    MG_REQUIRE(num_pairs >= 0 && batch >= 1, "num_pairs must be >= 0 and batch positive");
    MG_REQUIRE(num_layers >= 1 && num_layers <= 65535, "num_layers must be in [1, 65535], got %d", num_layers);
    if (num_pairs == 0) return MG_OK;
    MG_REQUIRE(lp && lp->k_pool && lp->v_pool && lp->k_scales && lp->v_scales && lp->staging_k && lp->staging_v,
               "null layer pointer");
    MG_REQUIRE(block_tables && seq_lens && src_ids && dst_ids, "null pointer");
    MG_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 3u) == 0 &&
                   workspace_bytes >= mg_fork_workspace_bytes(num_pairs),
               "the workspace needs %lld bytes (mg_fork_workspace_bytes), got %lld",
               (long long)mg_fork_workspace_bytes(num_pairs), (long long)workspace_bytes);
    const uintptr_t all = reinterpret_cast<uintptr_t>(lp->k_pool) | reinterpret_cast<uintptr_t>(lp->v_pool) |
                          reinterpret_cast<uintptr_t>(lp->staging_k) | reinterpret_cast<uintptr_t>(lp->staging_v);
    MG_REQUIRE((all & 15u) == 0, "pools and staging must be 16-byte aligned");
    const bool i4 = L->kv_dtype == MG_KV_INT4;
    const int64_t row = static_cast<int64_t>(L->num_kv_heads) * L->head_dim;
    MG_REQUIRE(row * L->page_size < (1ll << 28), "a page of more than 2^28 elements is not supported");
    ForkParams p;
    p.free_stack = al->free_stack;
    p.n_free = al->n_free;
    p.in_use = al->in_use;
    p.num_pages = al->num_pages;
    p.block_tables = block_tables;
    p.max_blocks = L->max_blocks;
    p.seq_lens = seq_lens;
    p.batch = batch;
    p.src = src_ids;
    p.dst = dst_ids;
    p.new_lens = new_lens;
    p.pairs = num_pairs;
    p.P = L->page_size;
    p.ws = static_cast<int32_t*>(workspace);
    p.status = dev_status;
    p.k_pool = static_cast<const uint8_t*>(lp->k_pool);
    p.v_pool = static_cast<const uint8_t*>(lp->v_pool);
    p.k_scales = lp->k_scales;
    p.v_scales = lp->v_scales;
    p.staging_k = lp->staging_k;
    p.staging_v = lp->staging_v;
    p.layers = num_layers;
    p.row = static_cast<int32_t>(row);
    p.D = L->head_dim;
    p.scale_th = L->scale_layout == MG_SCALE_TOKEN_HEAD;
    const int64_t page_elems = row * L->page_size;
    p.pool_layer = L->num_pages * (i4 ? page_elems / 2 : page_elems);
    p.scale_layer = p.scale_th ? L->num_pages * L->page_size * L->num_kv_heads : L->num_pages;
    p.staging_layer = batch * page_elems;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(num_pairs));
    cfg.blockDim = dim3(kForkThreads);
    cfg.stream = as_stream(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, fork_release_kernel, p);
    st = check_launch("fork_release_kernel");
    if (st != MG_OK) return st;
    cfg.gridDim = dim3(static_cast<unsigned>(num_pairs), static_cast<unsigned>(num_layers));
    const bool s16 = L->staging_dtype == MG_F16;
    if (i4 && s16) cudaLaunchKernelEx(&cfg, fork_share_kernel<true, __half>, p);
    else if (i4) cudaLaunchKernelEx(&cfg, fork_share_kernel<true, float>, p);
    else if (s16) cudaLaunchKernelEx(&cfg, fork_share_kernel<false, __half>, p);
    else cudaLaunchKernelEx(&cfg, fork_share_kernel<false, float>, p);
    return check_launch("fork_share_kernel");
}
