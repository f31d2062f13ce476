// Drafted-token attention: the step's plan, the join of split sequences, and
// the C entry points.  The attention kernels are in mg_tree_*_kernel.cuh.
#include <math.h>

#include "mg_tree.cuh"

namespace mg {

mg_status check_cache_layout(const mg_cache_layout* L);

namespace {

constexpr int kTreePlanThreads = 1024;
constexpr int kJoinThreads = 256;

struct TreePlanParams {
    const int32_t* seq_lens;
    const int32_t* n_draft;  // null: every sequence drafts T
    int32_t batch, T, P, max_blocks, Hkv, G;
    TreeGeom geo;
    TreePlanLayout lay;
    int32_t* plan;
    int32_t* status;
};

__device__ __forceinline__ int cdiv(int a, int b) { return (a + b - 1) / b; }

// Sum of one value per thread over the CTA.
__device__ __forceinline__ unsigned long long block_sum_u64(unsigned long long v, unsigned long long* acc) {
    if (threadIdx.x == 0) *acc = 0ull;
    __syncthreads();
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0 && v) atomicAdd(acc, v);
    __syncthreads();
    const unsigned long long r = *acc;
    __syncthreads();
    return r;
}

// One CTA: every (sequence, row tile) is cut along the keys into near-equal
// pieces of at most C key tiles.
//   one wave    when the uncut items fit on the GPU at once: C is the smallest
//               piece for which the pieces still do (bisection), so the
//               longest CTA is as short as it can be;
//   more waves  otherwise: C = the work over slots * waves, so that a long
//               context does not outlast the rest.
// (Two waves where one leaves a third of the slots empty were slower: 32 contexts
// of 1012 tokens, 12 heads, 29 us a layer for 25.6.)  Latency-bound: a few us for a
// step, before its first layer.
__global__ void __launch_bounds__(kTreePlanThreads) tree_plan_kernel(TreePlanParams a) {
    __shared__ unsigned long long acc;
    __shared__ int scratch[33];
    __shared__ int s_max, s_clear;
    grid_dependency_wait();
    grid_launch_dependents();
    int32_t* head = a.plan;
    int32_t* items = a.plan + a.lay.off_items;
    int32_t* seqs = a.plan + a.lay.off_seqs;
    if (threadIdx.x == 0) {
        s_max = 1;
        s_clear = 0;
        head[2] = a.geo.BM;
        head[3] = a.batch;
        head[4] = a.T;
        head[5] = a.Hkv * a.G;
    }
    __syncthreads();
    if (a.status && (*(volatile int32_t*)a.status & kStopBits)) {  // the step was refused: nothing to attend
        if (threadIdx.x == 0) head[0] = head[1] = 0;
        return;
    }
    unsigned long long work = 0, tiles0 = 0;
    for (int b = threadIdx.x; b < a.batch; b += blockDim.x) {
        int n = a.seq_lens[b], t = a.n_draft ? a.n_draft[b] : a.T;
        if (n < 0 || n / a.P > a.max_blocks || t < 0 || t > a.T) {
            flag(a.status, MG_DEV_BAD_ARGUMENT);
            n = t = 0;
        }
        const int mt = cdiv(t * a.G, a.geo.BM);
        const int U = t == 0 ? 0 : cdiv(n, a.geo.tile) + cdiv(t, a.geo.tile);
        int4* rec = reinterpret_cast<int4*>(seqs + static_cast<int64_t>(b) * 8);
        rec[0] = make_int4(t, 0, 0, n);
        rec[1] = make_int4(0, mt, U, 0);
        work += static_cast<unsigned long long>(mt) * U;
        tiles0 += mt;
        if (U > 1) atomicMax(&s_max, U);
        if (t < a.T) s_clear = 1;
    }
    work = block_sum_u64(work, &acc);
    tiles0 = block_sum_u64(tiles0, &acc);
    const unsigned long long slots = a.geo.slots;
    int C;
    if (tiles0 * a.Hkv <= slots) {
        int lo = 1, hi = s_max;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            unsigned long long cnt = 0;
            for (int b = threadIdx.x; b < a.batch; b += blockDim.x) {
                const int4 r = reinterpret_cast<const int4*>(seqs + static_cast<int64_t>(b) * 8)[1];
                cnt += static_cast<unsigned long long>(r.y) * cdiv(r.z, mid);
            }
            if (block_sum_u64(cnt, &acc) * a.Hkv <= slots) hi = mid;
            else lo = mid + 1;
        }
        C = lo;
    } else {
        const unsigned long long per = slots * a.geo.waves;
        C = static_cast<int>((work * a.Hkv + per - 1) / per);
        if (C < 1) C = 1;
    }
    // item and partial-slot prefixes, sequence by sequence
    int ibase = 0, pbase = 0;
    for (int start = 0; start < a.batch; start += blockDim.x) {
        const int b = start + threadIdx.x;
        int4* rec = reinterpret_cast<int4*>(seqs + static_cast<int64_t>(b < a.batch ? b : 0) * 8);
        int k = 0, mt = 0;
        if (b < a.batch) {
            const int4 r1 = rec[1];
            mt = r1.y;
            k = cdiv(r1.z, C);
        }
        int ti, tp;
        const int ei = block_exclusive_scan(mt * k, scratch, &ti);
        __syncthreads();
        const int ep = block_exclusive_scan(k > 1 ? mt * k : 0, scratch, &tp);
        __syncthreads();
        if (b < a.batch) {
            rec[0].y = k;
            rec[0].z = pbase + ep;
            rec[1].x = ibase + ei;
        }
        ibase += ti;
        pbase += tp;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        head[0] = ibase;
        head[1] = s_clear || pbase > 0;
    }
    // a warp per sequence writes its items: row tiles fastest, so that CTAs
    // that read the same keys run close together
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int b = warp; b < a.batch; b += kTreePlanThreads / 32) {
        const int4 r0 = reinterpret_cast<const int4*>(seqs + static_cast<int64_t>(b) * 8)[0];
        const int4 r1 = reinterpret_cast<const int4*>(seqs + static_cast<int64_t>(b) * 8)[1];
        const int k = r0.y, mt = r1.y, U = r1.z;
        for (int i = lane; i < mt * k; i += 32) {
            const int piece = i / mt, tile = i - piece * mt;
            const int u0 = static_cast<int>(static_cast<int64_t>(U) * piece / k);
            const int u1 = static_cast<int>(static_cast<int64_t>(U) * (piece + 1) / k);
            int4* it = reinterpret_cast<int4*>(items + static_cast<int64_t>(r1.x + i) * 8);
            it[0] = make_int4(b, tile, u0, u1 - u0);
            it[1] = make_int4(k > 1 ? r0.z + tile * k + piece : -1, r0.x, r0.w, 0);
        }
    }
}

// Joins the pieces of split sequences (one log-sum-exp pass per row, in piece
// order, so the result does not depend on which CTA ended first) and clears
// the rows past a sequence's drafted tokens.  One warp per row; bound by the
// launch and a chain of two loads (it overlaps the attention's last CTAs).
template <int D>
__global__ void __launch_bounds__(kJoinThreads) tree_join_kernel(TreeParams p, int BM) {
    grid_dependency_wait();
    grid_launch_dependents();
    if (p.plan[1] == 0 || !tree_plan_matches(p, BM)) return;
    constexpr int V = D / 32;
    const int lane = threadIdx.x & 31;
    const int64_t rows = static_cast<int64_t>(p.T) * p.G, total = rows * p.Hkv * p.batch;
    const int64_t nwarps = static_cast<int64_t>(gridDim.x) * (kJoinThreads / 32);
    for (int64_t i = blockIdx.x * static_cast<int64_t>(kJoinThreads / 32) + (threadIdx.x >> 5); i < total; i += nwarps) {
        const int64_t bh = i / rows;
        const int r = static_cast<int>(i - bh * rows);
        const int b = static_cast<int>(bh / p.Hkv), h = static_cast<int>(bh - static_cast<int64_t>(b) * p.Hkv);
        const int4 s = *reinterpret_cast<const int4*>(p.plan + p.lay.off_seqs + static_cast<int64_t>(b) * 8);
        const int t = r / p.G, hh = h * p.G + (r - t * p.G);
        __half* dst = p.out + ((static_cast<int64_t>(b) * p.T + t) * p.Hkv * p.G + hh) * D + lane * V;
        float a[V];
#pragma unroll
        for (int e = 0; e < V; ++e) a[e] = 0.0f;
        if (t < s.x) {
            if (s.y <= 1) continue;
            const int64_t first = s.z + static_cast<int64_t>(r / BM) * s.y;
            const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + (first * p.Hkv + h) * BM + r % BM;
            const float* po = p.part_o + ((first * p.Hkv + h) * BM + r % BM) * D + lane * V;
            const int64_t step = static_cast<int64_t>(p.Hkv) * BM;
            float mx = -INFINITY;
            for (int k = lane; k < s.y; k += 32) mx = fmaxf(mx, ml[k * step].x);
            mx = warp_max(mx);
            float ls = 0.0f;
#pragma unroll 4
            for (int k = 0; k < s.y; ++k) {
                const float2 w = ml[k * step];
                // a piece without a finite score weighs nothing, but its NaN sum goes through;
                // so does an infinity or NaN that a row saw in V, which a weight of 0 would turn
                // into NaN (as in the unsplit kernels, where it is added after the weighting)
                const float f = mx == -INFINITY ? 0.0f : ex2(w.x - mx);
                ls += f * w.y;
                float x[V];
                if constexpr (V == 4) *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(po + k * step * D);
                else *reinterpret_cast<float2*>(x) = *reinterpret_cast<const float2*>(po + k * step * D);
#pragma unroll
                for (int e = 0; e < V; ++e) a[e] += isfinite(x[e]) ? f * x[e] : x[e];
            }
            const float inv = ls > 0.0f || isnan(ls) ? 1.0f / ls : 0.0f;
#pragma unroll
            for (int e = 0; e < V; ++e) a[e] *= inv;
        }
        if constexpr (V == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(pack_half2(a[0], a[1]), pack_half2(a[2], a[3]));
        else *reinterpret_cast<uint32_t*>(dst) = pack_half2(a[0], a[1]);
    }
}

mg_status check_tree(const mg_cache_layout* L, int64_t batch, int64_t T, int64_t Hq) {
    mg_status st = check_cache_layout(L);
    if (st != MG_OK) return st;
    MG_REQUIRE(batch >= 0 && batch <= kTreeMaxBatch, "batch must be in [0, %d], got %lld", kTreeMaxBatch,
               (long long)batch);
    MG_REQUIRE(T >= 0, "max_draft must be >= 0");
    MG_REQUIRE(L->head_dim == 64 || L->head_dim == 128, "drafted-token attention supports head_dim 64 or 128, got %d",
               L->head_dim);
    MG_REQUIRE(Hq >= 1 && Hq % L->num_kv_heads == 0, "num_q_heads=%lld must be a positive multiple of num_kv_heads=%d",
               (long long)Hq, L->num_kv_heads);
    MG_REQUIRE(T * Hq < (1ll << 31), "max_draft * num_q_heads too large");
    MG_REQUIRE((L->max_blocks + 1ll) * L->page_size < (1ll << 26),
               "drafted-token attention supports contexts below 2^26 tokens, got max_blocks=%d pages of %d",
               L->max_blocks, L->page_size);
    const TreeGeom g = tree_geometry(*L, batch, T, Hq);
    MG_REQUIRE(g.max_items * L->num_kv_heads < (1ll << 31), "too many work items for one launch");
    return MG_OK;
}

int64_t part_bytes(const TreeGeom& g, const mg_cache_layout& L) {
    return g.max_parts * L.num_kv_heads * g.BM * (L.head_dim + 2) * 4;
}

bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

TreeGeom tree_geometry(const mg_cache_layout& L, int64_t batch, int64_t T, int64_t Hq) {
    TreeGeom g;
    const int64_t rows = T * (Hq / L.num_kv_heads);
    int occ;
    // Above 48 rows the tensor-core tile kernel, whose time hardly depends on the
    // rows (one B200, us per call, row kernel / tile kernel): head_dim 64, 64 sequences
    // of 1000 tokens, 4 kv heads, INT8: 32 rows 31 / 62, 40 rows 56 / 63, 64 rows 61 /
    // 68, 128 rows 85 / 86, 256 rows 162 / 93; 200 sequences of 3000, INT4: 32 rows 158 /
    // 215, 40 rows 234 / 218, 64 rows 246 / 221, 128 rows 477 / 239; head_dim 128, 12
    // sequences of 3000, 8 kv heads, INT8: 40 rows 60 / 72, 64 rows 107 / 74, 128 rows
    // 177 / 80.  The rule looks at the rows alone: between 33 and 48 it loses 7 % where
    // much work fills the GPU several times (40 rows, 200 sequences) and wins 11 to 17 %
    // on the others.
    g.tiles = rows > 48;
    if (g.tiles) {
        g.tile = kTilesKeys;
        // equal row tiles of at most 128, in whole warps
        const int64_t mt = rows > 128 ? (rows + 127) / 128 : 1;
        g.BM = static_cast<int>(((rows + mt - 1) / mt + 31) / 32 * 32);
        occ = 1;
    } else {
        g.tile = kTreeTile;
        g.BM = L.head_dim == 64 && rows > 16 ? 32 : 16;
        occ = L.head_dim == 128 ? rows_ctas_per_sm<128, 1>()
                                : (g.BM == 32 ? rows_ctas_per_sm<64, 2>() : rows_ctas_per_sm<64, 1>());
    }
    g.mt_max = static_cast<int>((rows + g.BM - 1) / g.BM);
    g.slots = sm_count() * occ;
    g.waves = 2;
    const int64_t uncut = batch * g.mt_max, hkv = L.num_kv_heads;
    if (uncut * hkv <= g.slots) {  // one wave, whatever the lengths
        g.max_items = g.max_parts = g.slots / hkv;
    } else {
        // sum of ceil(U / C) over the items <= work / C + items, and the pieces
        // of cut ones <= 2 work / C, with work * Hkv / C <= slots * waves
        g.max_items = static_cast<int64_t>(g.slots) * g.waves / hkv + 1 + uncut;
        g.max_parts = 2 * (static_cast<int64_t>(g.slots) * g.waves / hkv + 1);
    }
    return g;
}

}  // namespace mg

using namespace mg;

extern "C" int64_t mg_tree_plan_bytes(const mg_cache_layout* L, int32_t batch, int32_t max_draft,
                                      int32_t num_q_heads) {
    if (check_tree(L, batch, max_draft, num_q_heads) != MG_OK) return 0;
    return tree_plan_layout(batch, tree_geometry(*L, batch, max_draft, num_q_heads).max_items).words * 4;
}

extern "C" int64_t mg_tree_workspace_bytes(const mg_cache_layout* L, int32_t batch, int32_t max_draft,
                                           int32_t num_q_heads) {
    if (check_tree(L, batch, max_draft, num_q_heads) != MG_OK) return 0;
    return part_bytes(tree_geometry(*L, batch, max_draft, num_q_heads), *L) + 16;
}

extern "C" mg_status mg_tree_plan(const mg_cache_layout* L, const int32_t* seq_lens, const int32_t* n_draft,
                                  int32_t batch, int32_t max_draft, int32_t num_q_heads, void* plan,
                                  int64_t plan_bytes, int32_t* dev_status, mg_stream_t stream) {
    mg_status st = check_tree(L, batch, max_draft, num_q_heads);
    if (st != MG_OK) return st;
    if (batch == 0 || max_draft == 0) return MG_OK;
    MG_REQUIRE(seq_lens && plan, "null pointer");
    TreePlanParams a;
    a.geo = tree_geometry(*L, batch, max_draft, num_q_heads);
    a.lay = tree_plan_layout(batch, a.geo.max_items);
    MG_REQUIRE(aligned16(plan) && plan_bytes >= a.lay.words * 4,
               "the plan needs %lld bytes, 16-byte aligned (mg_tree_plan_bytes), got %lld", (long long)a.lay.words * 4,
               (long long)plan_bytes);
    a.seq_lens = seq_lens;
    a.n_draft = n_draft;
    a.batch = batch;
    a.T = max_draft;
    a.P = L->page_size;
    a.max_blocks = L->max_blocks;
    a.Hkv = L->num_kv_heads;
    a.G = num_q_heads / L->num_kv_heads;
    a.plan = static_cast<int32_t*>(plan);
    a.status = dev_status;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1);
    cfg.blockDim = dim3(kTreePlanThreads);
    cfg.stream = as_stream(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, tree_plan_kernel, a);
    return check_launch("tree_plan_kernel");
}

extern "C" mg_status mg_tree_attention(const mg_cache_layout* L, const mg_layer_ptrs* lp, const int32_t* block_tables,
                                       int32_t batch, const mg_tree_draft* d, const void* plan, int64_t plan_bytes,
                                       float scale, void* out, void* workspace, int64_t workspace_bytes,
                                       int32_t* dev_status, mg_stream_t stream) {
    MG_REQUIRE(lp && d, "null layer pointers or draft");
    mg_status st = check_tree(L, batch, d->max_draft, d->num_q_heads);
    if (st != MG_OK) return st;
    if (batch == 0 || d->max_draft == 0) return MG_OK;
    MG_REQUIRE(L->staging_dtype == MG_F16, "drafted-token attention reads fp16 staging");
    MG_REQUIRE(lp->k_pool && lp->v_pool && lp->k_scales && lp->v_scales && lp->staging_k && lp->staging_v,
               "null layer pointer");
    MG_REQUIRE(block_tables && plan && out && d->q && d->k && d->v, "null pointer");
    MG_REQUIRE(isfinite(scale) && scale > 0.0f, "attention scale must be positive and finite");
    const TreeGeom g = tree_geometry(*L, batch, d->max_draft, d->num_q_heads);
    const TreePlanLayout lay = tree_plan_layout(batch, g.max_items);
    MG_REQUIRE(aligned16(plan) && plan_bytes >= lay.words * 4,
               "the plan needs %lld bytes, 16-byte aligned (mg_tree_plan_bytes), got %lld", (long long)lay.words * 4,
               (long long)plan_bytes);
    const int64_t need = part_bytes(g, *L);
    MG_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= need,
               "the workspace needs %lld bytes, 16-byte aligned (mg_tree_workspace_bytes), got %lld", (long long)need,
               (long long)workspace_bytes);
    MG_REQUIRE(aligned16(lp->k_pool) && aligned16(lp->v_pool) && aligned16(lp->staging_k) && aligned16(lp->staging_v) &&
                   aligned16(out),
               "pools, staging and out must be 16-byte aligned");
    MG_REQUIRE(aligned8(d->q) && aligned8(d->k) && aligned8(d->v), "q, k and v must be 8-byte aligned");
    for (int i = 0; i < 3; ++i)
        MG_REQUIRE(d->q_stride[i] % 4 == 0 && d->k_stride[i] % 4 == 0 && d->v_stride[i] % 4 == 0,
                   "strides of q, k and v must be multiples of 4 elements");
    TreeParams p;
    p.k_pool = static_cast<const uint8_t*>(lp->k_pool);
    p.v_pool = static_cast<const uint8_t*>(lp->v_pool);
    p.k_scales = lp->k_scales;
    p.v_scales = lp->v_scales;
    p.staging_k = static_cast<const __half*>(lp->staging_k);
    p.staging_v = static_cast<const __half*>(lp->staging_v);
    p.block_tables = block_tables;
    p.max_blocks = L->max_blocks;
    p.P = L->page_size;
    p.div_p = FastDiv(static_cast<uint32_t>(L->page_size));
    p.Hkv = L->num_kv_heads;
    p.G = d->num_q_heads / L->num_kv_heads;
    p.scale_th = L->scale_layout == MG_SCALE_TOKEN_HEAD;
    p.num_pages = L->num_pages;
    p.q = static_cast<const __half*>(d->q);
    p.k = static_cast<const __half*>(d->k);
    p.v = static_cast<const __half*>(d->v);
    p.q_sb = d->q_stride[0], p.q_st = d->q_stride[1], p.q_sh = d->q_stride[2];
    p.k_sb = d->k_stride[0], p.k_st = d->k_stride[1], p.k_sh = d->k_stride[2];
    p.v_sb = d->v_stride[0], p.v_st = d->v_stride[1], p.v_sh = d->v_stride[2];
    p.mask = static_cast<const uint8_t*>(d->mask);
    p.mask_sb = d->mask_stride;
    p.T = d->max_draft;
    p.batch = batch;
    p.BM = g.BM;
    p.scale_log2 = scale * 1.4426950408889634f;
    p.out = static_cast<__half*>(out);
    p.plan = static_cast<const int32_t*>(plan);
    p.lay = lay;
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = p.part_o + g.max_parts * L->num_kv_heads * g.BM * L->head_dim;
    p.status = dev_status;
    cudaStream_t s = as_stream(stream);
    const bool i4 = L->kv_dtype == MG_KV_INT4;
    if (g.tiles) {
        if (L->head_dim == 64) i4 ? launch_tree_tiles<true, 64>(p, g, s) : launch_tree_tiles<false, 64>(p, g, s);
        else i4 ? launch_tree_tiles<true, 128>(p, g, s) : launch_tree_tiles<false, 128>(p, g, s);
    } else if (L->head_dim == 64) i4 ? launch_tree_rows<true, 64>(p, g, s) : launch_tree_rows<false, 64>(p, g, s);
    else i4 ? launch_tree_rows<true, 128>(p, g, s) : launch_tree_rows<false, 128>(p, g, s);
    st = check_launch(g.tiles ? "tree_tiles_kernel" : "tree_rows_kernel");
    if (st != MG_OK) return st;
    const int64_t tasks = static_cast<int64_t>(p.T) * d->num_q_heads * batch;
    const int64_t blocks = (tasks + kJoinThreads / 32 - 1) / (kJoinThreads / 32);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(blocks < sm_count() * 8 ? blocks : sm_count() * 8));
    cfg.blockDim = dim3(kJoinThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (L->head_dim == 64) cudaLaunchKernelEx(&cfg, tree_join_kernel<64>, p, g.BM);
    else cudaLaunchKernelEx(&cfg, tree_join_kernel<128>, p, g.BM);
    return check_launch("tree_join_kernel");
}
