// Attention of several drafted tokens per sequence over its paged, quantized
// context and over each other: parameters, work geometry and plan layout.
//
// Notation: G = Hq / Hkv query heads share a kv head; the R = t * G query rows
// of one (sequence, kv head) -- t drafted tokens, row r = token r / G, head
// r % G of the group -- all read the same keys, so they are computed together
// in row tiles of BM.  Keys are counted in tiles (64 or 128 tokens, by kernel):
// the cached context's tiles (pages, then the staged tail) first, then the
// drafted tokens'.
#pragma once

#include "mg_alloc_step.cuh"
#include "mg_common.cuh"

namespace mg {

constexpr int kTreeTile = 64;       // keys of a tile of the row kernel
constexpr int kTilesKeys = 128;     // keys of a tile of the tensor-core tile kernel
constexpr int kTreeHeader = 16;     // int32 words before the plan's records
constexpr int kTreeMaxBatch = 65535;

// What the host fixes for one (layout, batch, drafted tokens, q heads): the
// row tile, how many CTAs run at once, and the bounds on the work items.
struct TreeGeom {
    bool tiles;        // the tensor-core tile kernel, else the row kernel
    int tile;          // keys per unit of the plan
    int BM;            // query rows per work item
    int mt_max;        // row tiles of a sequence that drafts T tokens
    int slots;         // CTAs resident on the GPU at once
    int waves;         // CTAs aimed at per slot when the batch has more than one wave of items
    int64_t max_items;  // bound on work items (per kv head)
    int64_t max_parts;  // bound on partial results (per kv head)
};

// Plan words (int32): header | items [max_items][8] | sequences [batch][8].
//   header[0] items, [1] nonzero when the join has work (a split sequence, rows
//             past a sequence's drafted tokens), [2..5] BM, batch, T, q heads
//   item      {b, row tile, first key tile, key tiles, partial slot or -1, drafted, cached, 0}
//   sequence  {drafted, pieces, first partial slot, cached, first item, row tiles, key tiles, 0}
struct TreePlanLayout {
    int64_t off_items, off_seqs, words;
};
inline TreePlanLayout tree_plan_layout(int64_t batch, int64_t max_items) {
    TreePlanLayout l;
    l.off_items = kTreeHeader;
    l.off_seqs = l.off_items + max_items * 8;
    l.words = l.off_seqs + batch * 8;
    return l;
}

struct TreeParams {
    const uint8_t* k_pool;
    const uint8_t* v_pool;
    const float* k_scales;
    const float* v_scales;
    const __half* staging_k;
    const __half* staging_v;
    const int32_t* block_tables;
    int32_t max_blocks;
    int32_t P;
    FastDiv div_p;  // by P, exact below 2^26 tokens
    int32_t Hkv;
    int32_t G;
    int32_t scale_th;  // scales [N, P, Hkv] instead of [N]
    int64_t num_pages;
    const __half* q;
    const __half* k;  // drafted tokens
    const __half* v;
    int64_t q_sb, q_st, q_sh;  // strides in elements: sequence, token, head
    int64_t k_sb, k_st, k_sh;
    int64_t v_sb, v_st, v_sh;
    const uint8_t* mask;  // [T, T] or [batch, T, T]; null: token t sees u <= t
    int64_t mask_sb;
    int32_t T;
    int32_t batch;
    int32_t BM;  // query rows per work item
    float scale_log2;  // attention scale * log2(e)
    __half* out;       // [batch, T, Hq, D]
    const int32_t* plan;
    TreePlanLayout lay;
    float* part_o;   // [max_parts, Hkv, BM, D]
    float* part_ml;  // [max_parts, Hkv, BM, 2]
    int32_t* status;
};

// Whether the plan was made for this call's shape (read by one thread or all).
__device__ __forceinline__ bool tree_plan_matches(const TreeParams& p, int BM) {
    return p.plan[2] == BM && p.plan[3] == p.batch && p.plan[4] == p.T && p.plan[5] == p.Hkv * p.G;
}

// ---------------------------------------------------------------------------
// device helpers shared by the kernels
// ---------------------------------------------------------------------------

// A V scale s as s = mant * 2^e with e in [-20, 13]: the codes times 2^e are
// exact in fp16 over that whole range (|code| * 2^e never exceeds the page's
// absmax, which fp16 holds), and mant, which goes into the fp32 probabilities, is
// below 2, and at least 1 unless s is below 2^-20.  So a page of very small or
// very large values loses nothing to fp16's exponent range, which the plain
// product probability * s would.
__device__ __forceinline__ int scale_exponent(float s) {
    const int e = static_cast<int>((__float_as_uint(s) >> 23) & 255u) - 127;
    return e < -20 ? -20 : (e > 13 ? 13 : e);
}
// The part of 2^e that the conversion's one fp16 FMA can hold: its offset of
// 1152 * 2^e has to fit as well.  Scales of 64 and more need a second step.
__device__ __forceinline__ int fma_exponent(int e) { return e > 5 ? 5 : e; }
__device__ __forceinline__ float rcp(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float pow2f(int e) { return __int_as_float((e + 127) << 23); }
__device__ __forceinline__ float2 unpack_half2(uint32_t x) {
    return __half22float2(*reinterpret_cast<const __half2*>(&x));
}
__device__ __forceinline__ uint32_t half_bits(float x) {
    return static_cast<uint32_t>(__half_as_ushort(__float2half_rn(x)));
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
    return r;
}
// Any of the two halves infinite or NaN.
__device__ __forceinline__ bool nonfinite2(uint32_t x) {
    return (x & 0x7C00u) == 0x7C00u || (x & 0x7C000000u) == 0x7C000000u;
}
// The two halves with infinities and NaN replaced by zero.
__device__ __forceinline__ uint32_t finite_or_zero2(uint32_t x) {
    if ((x & 0x7C00u) == 0x7C00u) x &= 0xFFFF0000u;
    if ((x & 0x7C000000u) == 0x7C000000u) x &= 0x0000FFFFu;
    return x;
}
__device__ __forceinline__ bool tree_sees(const TreeParams& p, int b, int t, int u) {
    return p.mask ? p.mask[static_cast<int64_t>(b) * p.mask_sb + static_cast<int64_t>(t) * p.T + u] != 0 : u <= t;
}

// What the exact fp16 rows whose V holds an infinity or a NaN add to one
// output element.  Those elements are zeroed on their way into the matrix
// products, where a masked probability of zero would turn them into NaN for
// every row; a row that does see such a key gets the sum it would have: the
// infinity, or NaN.
__device__ __forceinline__ float nonfinite_sum(const TreeParams& p, int b, int h, int D, int t, int d, int tail0,
                                               int n, int u0, int u1) {
    float a = 0.0f;
    const int whole = (n / p.P) * p.P;
    for (int i = tail0; i < n; ++i) {
        const float x = __half2float(
            p.staging_v[((static_cast<int64_t>(b) * p.P + (i - whole)) * p.Hkv + h) * D + d]);
        if (!isfinite(x)) a += x;
    }
    for (int u = u0; u < u1; ++u) {
        const float x = __half2float(p.v[b * p.v_sb + u * p.v_st + h * p.v_sh + d]);
        if (!isfinite(x) && tree_sees(p, b, t, u)) a += x;
    }
    return a;
}

// CTAs per SM that the row kernel's register budget is set for; the plan counts on them.
template <int D, int RT>
__host__ __device__ constexpr int rows_ctas_per_sm() {
    return D == 128 ? 2 : (RT == 2 ? 3 : 4);
}

// host: kernel launchers (one translation unit per pool format and head_dim)
template <bool KV4, int D>
void launch_tree_rows(const TreeParams& p, const TreeGeom& g, cudaStream_t stream);

template <bool KV4, int D>
void launch_tree_tiles(const TreeParams& p, const TreeGeom& g, cudaStream_t stream);

TreeGeom tree_geometry(const mg_cache_layout& L, int64_t batch, int64_t T, int64_t Hq);

}  // namespace mg
