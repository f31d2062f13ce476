// RMS norm of every q and k head and its rotary embedding in one pass over a
// fused q | k | v projection:
//   y = x * rsqrt(mean(x^2) + eps) * w        (over one head's D values)
//   (y_d, y_{d + D/2}) -> (y_d c - y_{d+D/2} s, y_{d+D/2} c + y_d s)
// with c, s of the row's position.  Everything between the fp16 input and the
// one rounding of the output is fp32.
//
// Bound: each value is read and written once, so HBM for prompts and the
// launch for a decode step.
#include <type_traits>

#include "mg_common.cuh"

namespace mg {
namespace {

constexpr int kNormThreads = 256;

struct QkNormParams {
    const __half* qkv;
    int64_t row_stride;  // elements
    const __half* wq;
    const __half* wk;
    const int64_t* pos;
    const float* cosb;
    const float* sinb;
    int64_t table_rows;
    float eps;
    __half* q;
    __half* k;
    __half* v;  // null: v is left where it is
    int64_t rows;
    int32_t Hq, Hkv, D;
    int32_t parts;  // warps that share a row's heads
    int32_t* status;
};

__device__ __forceinline__ __half* head_out(const QkNormParams& p, int64_t r, int h) {
    if (h < p.Hq) return p.q + (r * p.Hq + h) * p.D;
    h -= p.Hq;
    return h < p.Hkv ? p.k + (r * p.Hkv + h) * p.D : p.v + (r * p.Hkv + h - p.Hkv) * p.D;
}

__device__ __forceinline__ void unpack8(const uint4& u, float (&x)[8]) {
    const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(h[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
    return make_uint4(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]), pack_half2(x[4], x[5]),
                      pack_half2(x[6], x[7]));
}

// LPH lanes per head (the power of two from D / 16 up); lane j < D / 16 holds
// values 8 j .. 8 j + 7 of both halves, so a rotation needs no exchange and the
// row's cos and sin, 8 of each per lane, serve all its heads: a warp takes a
// row (or one of `parts` shares of its heads) and keeps them in registers.
// `parts` is 1 once the rows alone fill the GPU, and splits the row below that.
// U rounds of heads are in flight.  One B200, 18423 rows of 32 + 8 + 8 heads of 128
// (453 MB): 98 / 95 / 88 / 91 us with U = 1 / 2 / 3 / 4 (5.2 TB/s, 0.79 of the
// copy rate); 1024 rows of 32 + 4 heads of 64, a round per warp: 4.5 us with U = 1,
// 5.7 with 2 (the second round's registers cost resident warps).
template <int LPH, int U>
__global__ void __launch_bounds__(kNormThreads) qk_norm_rope_kernel(QkNormParams p) {
    constexpr int HPW = 32 / LPH;  // heads a warp takes at once
    grid_dependency_wait();
    grid_launch_dependents();
    const int lane = threadIdx.x & 31, j = lane % LPH, sub = lane / LPH;
    const int D = p.D, half = D / 2;
    const bool on = j * 8 < half;
    const int64_t gw = (blockIdx.x * static_cast<int64_t>(kNormThreads) + threadIdx.x) >> 5;
    const int64_t r = gw / p.parts;
    if (r >= p.rows) return;
    const int part = static_cast<int>(gw - r * p.parts);
    const int heads = p.Hq + p.Hkv + (p.v ? p.Hkv : 0), normed = p.Hq + p.Hkv;
    const __half* src = p.qkv + r * p.row_stride + j * 8;
    const int64_t pos = p.pos[r];
    const bool inside = pos >= 0 && pos < p.table_rows;
    if (!inside && part == 0 && lane == 0) flag(p.status, MG_DEV_BAD_ARGUMENT);
    float c[8], s[8];
    uint4 wq[2] = {}, wk[2] = {};
    if (on) {
        // a position outside the tables: zeros come out
        const int64_t ti = (inside ? pos : 0) * half + j * 8;
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
            *reinterpret_cast<float4*>(c + i) = *reinterpret_cast<const float4*>(p.cosb + ti + i);
            *reinterpret_cast<float4*>(s + i) = *reinterpret_cast<const float4*>(p.sinb + ti + i);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            wq[i] = *reinterpret_cast<const uint4*>(p.wq + j * 8 + i * half);
            wk[i] = *reinterpret_cast<const uint4*>(p.wk + j * 8 + i * half);
        }
    }
    for (int h0 = part * HPW; h0 < heads; h0 += p.parts * HPW * U) {
        uint4 x[U][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = h0 + u * p.parts * HPW + sub;
            x[u][0] = x[u][1] = make_uint4(0u, 0u, 0u, 0u);
            if (h < heads && on) {
                x[u][0] = *reinterpret_cast<const uint4*>(src + static_cast<int64_t>(h) * D);
                x[u][1] = *reinterpret_cast<const uint4*>(src + static_cast<int64_t>(h) * D + half);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = h0 + u * p.parts * HPW + sub;
            float a[8], b[8], ss = 0.0f;
            unpack8(x[u][0], a);
            unpack8(x[u][1], b);
#pragma unroll
            for (int i = 0; i < 8; ++i) ss += a[i] * a[i] + b[i] * b[i];
#pragma unroll
            for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (h >= heads || !on) continue;
            if (h < normed) {
                const float inv = rsqrtf(ss / static_cast<float>(D) + p.eps);
                float wa[8], wb[8];
                unpack8(h < p.Hq ? wq[0] : wk[0], wa);
                unpack8(h < p.Hq ? wq[1] : wk[1], wb);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float ya = a[i] * inv * wa[i], yb = b[i] * inv * wb[i];
                    a[i] = inside ? ya * c[i] - yb * s[i] : 0.0f;
                    b[i] = inside ? yb * c[i] + ya * s[i] : 0.0f;
                }
                x[u][0] = pack8(a);
                x[u][1] = pack8(b);
            }
            __half* dst = head_out(p, r, h) + j * 8;
            *reinterpret_cast<uint4*>(dst) = x[u][0];
            *reinterpret_cast<uint4*>(dst + half) = x[u][1];
        }
    }
}

// Any even D and any alignment: one warp per (row, head).
__global__ void __launch_bounds__(kNormThreads) qk_norm_rope_any_kernel(QkNormParams p) {
    grid_dependency_wait();
    grid_launch_dependents();
    const int lane = threadIdx.x & 31, half = p.D / 2;
    const int heads = p.Hq + p.Hkv + (p.v ? p.Hkv : 0);
    const int64_t gw = (blockIdx.x * static_cast<int64_t>(kNormThreads) + threadIdx.x) >> 5;
    const int64_t r = gw / heads;
    if (r >= p.rows) return;
    const int h = static_cast<int>(gw - r * heads);
    const __half* src = p.qkv + r * p.row_stride + static_cast<int64_t>(h) * p.D;
    __half* dst = head_out(p, r, h);
    if (h >= p.Hq + p.Hkv) {
        for (int d = lane; d < p.D; d += 32) dst[d] = src[d];
        return;
    }
    const int64_t pos = p.pos[r];
    const bool inside = pos >= 0 && pos < p.table_rows;
    if (!inside && h == 0 && lane == 0) flag(p.status, MG_DEV_BAD_ARGUMENT);
    float ss = 0.0f;
    for (int d = lane; d < p.D; d += 32) {
        const float x = __half2float(src[d]);
        ss += x * x;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float inv = rsqrtf(ss / static_cast<float>(p.D) + p.eps);
    const __half* w = h < p.Hq ? p.wq : p.wk;
    for (int d = lane; d < half; d += 32) {
        const int64_t ti = (inside ? pos : 0) * half + d;
        const float c = p.cosb[ti], s = p.sinb[ti];
        const float a = __half2float(src[d]) * inv * __half2float(w[d]);
        const float b = __half2float(src[d + half]) * inv * __half2float(w[d + half]);
        dst[d] = __float2half_rn(inside ? a * c - b * s : 0.0f);
        dst[d + half] = __float2half_rn(inside ? b * c + a * s : 0.0f);
    }
}

}  // namespace
}  // namespace mg

using namespace mg;

extern "C" mg_status mg_qk_norm_rope_f16(const void* qkv, int64_t row_stride, const void* q_weight,
                                         const void* k_weight, const int64_t* pos, const float* cos_table,
                                         const float* sin_table, int64_t table_rows, float eps, void* q, void* k,
                                         void* v, int64_t rows, int32_t num_q_heads, int32_t num_kv_heads,
                                         int32_t head_dim, int32_t* dev_status, mg_stream_t stream) {
    MG_REQUIRE(rows >= 0 && num_q_heads >= 1 && num_kv_heads >= 1, "rows must be >= 0 and head counts positive");
    MG_REQUIRE(head_dim >= 2 && head_dim % 2 == 0, "head_dim must be positive and even, got %d", head_dim);
    MG_REQUIRE(eps >= 0.0f, "eps must be >= 0");
    const int64_t heads = static_cast<int64_t>(num_q_heads) + num_kv_heads + (v ? num_kv_heads : 0);
    const int64_t width = (num_q_heads + 2ll * num_kv_heads) * head_dim;
    MG_REQUIRE(width < (1ll << 31), "a row of more than 2^31 elements is not supported");
    if (rows == 0) return MG_OK;
    MG_REQUIRE(row_stride >= width, "the row stride must be at least %lld elements, got %lld", (long long)width,
               (long long)row_stride);
    MG_REQUIRE(table_rows >= 1, "the cos / sin tables are empty");
    MG_REQUIRE(qkv && q_weight && k_weight && pos && cos_table && sin_table && q && k, "null pointer");
    QkNormParams p;
    p.qkv = static_cast<const __half*>(qkv);
    p.row_stride = row_stride;
    p.wq = static_cast<const __half*>(q_weight);
    p.wk = static_cast<const __half*>(k_weight);
    p.pos = pos;
    p.cosb = cos_table;
    p.sinb = sin_table;
    p.table_rows = table_rows;
    p.eps = eps;
    p.q = static_cast<__half*>(q);
    p.k = static_cast<__half*>(k);
    p.v = static_cast<__half*>(v);
    p.rows = rows;
    p.Hq = num_q_heads;
    p.Hkv = num_kv_heads;
    p.D = head_dim;
    p.status = dev_status;
    const uintptr_t all = reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_weight) |
                          reinterpret_cast<uintptr_t>(k_weight) | reinterpret_cast<uintptr_t>(cos_table) |
                          reinterpret_cast<uintptr_t>(sin_table) | reinterpret_cast<uintptr_t>(q) |
                          reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v);
    const bool vec = (all & 15u) == 0 && row_stride % 8 == 0 && head_dim % 16 == 0 && head_dim <= 512;
    int lph = 1;
    while (lph * 16 < head_dim) lph *= 2;
    const int rounds = static_cast<int>((heads * lph + 31) / 32);
    // a warp per row once the rows give every SM 16 warps, else one per round of heads
    p.parts = rows >= 16ll * sm_count() ? 1 : rounds;
    const int64_t warps = vec ? rows * p.parts : rows * heads;
    const int64_t blocks = (warps + kNormThreads / 32 - 1) / (kNormThreads / 32);
    MG_REQUIRE(blocks < (1ll << 31), "too many rows for one launch");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(blocks));
    cfg.blockDim = dim3(kNormThreads);
    cfg.stream = as_stream(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    auto go = [&](auto lanes) {
        constexpr int kLanes = decltype(lanes)::value;
        if (p.parts == 1) cudaLaunchKernelEx(&cfg, qk_norm_rope_kernel<kLanes, 3>, p);
        else cudaLaunchKernelEx(&cfg, qk_norm_rope_kernel<kLanes, 1>, p);
    };
    if (!vec) cudaLaunchKernelEx(&cfg, qk_norm_rope_any_kernel, p);
    else if (lph == 1) go(std::integral_constant<int, 1>{});
    else if (lph == 2) go(std::integral_constant<int, 2>{});
    else if (lph == 4) go(std::integral_constant<int, 4>{});
    else if (lph == 8) go(std::integral_constant<int, 8>{});
    else if (lph == 16) go(std::integral_constant<int, 16>{});
    else go(std::integral_constant<int, 32>{});
    return check_launch("qk_norm_rope_kernel");
}
