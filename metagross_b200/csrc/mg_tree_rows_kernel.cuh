// Attention of a few query rows per (sequence, kv head) over the paged cache
// and the drafted tokens, on mma.sync fragments filled straight from HBM.
//
// One CTA of four warps per work item (row tile of 16 RT rows, a run of key
// tiles); warp w takes keys 16 w .. 16 w + 15 of every 64-key tile, keeps its
// own running maximum, sum and output for all rows, and the four are joined
// once at the end.  A warp's 16 keys are loaded from the pages into registers
// already in the matrix fragments' layout (no shared memory between HBM and
// the tensor cores): for S = Q K^T lane (g, c) holds the c-th quarter of key
// rows g and g + 8, for O = P V the g-th eighth of rows 2c, 2c+1, 2c+8, 2c+9;
// the order of the head dimension inside a fragment is permuted, Q's the same
// way.  Codes become fp16 by exponent insertion and one fp16 FMA.
//
// Why: with R rows a (sequence, kv head) reads 2 D bits / 8 bytes and does
// 4 R D products per key; for so few rows the conversion of a key (paid once per
// 16 RT rows here) is the largest part of the work, and a trip of the codes
// through shared memory would add to it.
// Measured (one B200, a layer): 32 INT8 contexts of ~1012 tokens, 12 heads of 64, 8
// drafted tokens: 25.6 us with its join, 2.0 TB/s; 200 log-normal INT4 contexts up to
// 32768, 5 drafted tokens for 8 heads each: 196 us.  Bound: ~330 dependent
// instructions per warp and 16 keys at 2.6 warps per scheduler (issue slots 37 %
// used, DRAM 28 %, tensor pipe 13 %).  More CTAs per SM spill; loads further ahead
// and L2 prefetch were slower.
#pragma once

#include <type_traits>

#include "mg_tree.cuh"

namespace mg {

constexpr int kRowsWarps = 4;
constexpr int kRowsThreads = kRowsWarps * 32;
// what a group of 16 keys is to the attention step
enum { kPagedGroup, kUniGroup, kTinyGroup };

template <bool KV4, int D>
struct RowsFmt {
    static constexpr int kRowBytes = KV4 ? D / 2 : D;
    static constexpr int KW = kRowBytes / 16;  // words of a key row's quarter
    static constexpr int VW = kRowBytes / 32;  // words of a value row's eighth
};

template <int N>
__device__ __forceinline__ void ldg_words(uint32_t (&w)[N], const uint8_t* ptr) {
    if constexpr (N == 1) {
        asm volatile("ld.global.cg.b32 %0, [%1];" : "=r"(w[0]) : "l"(ptr));
    } else if constexpr (N == 2) {
        asm volatile("ld.global.cg.v2.b32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(ptr));
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4)
            asm volatile("ld.global.cg.v4.b32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3])
                         : "l"(ptr + 4 * i));
    }
}
// fp16 rows: 8-byte loads (any row that starts on 8 bytes)
template <int N>
__device__ __forceinline__ void ldg_half_words(uint32_t (&w)[N], const __half* ptr) {
#pragma unroll
    for (int i = 0; i < N; i += 2)
        asm volatile("ld.global.v2.b32 {%0,%1}, [%2];" : "=r"(w[i]), "=r"(w[i + 1]) : "l"(ptr + 2 * i));
}

// Fragment pair of k-step s from a quarter row of halves, in the order the
// codes of this format come out of their words.
template <bool KV4>
__device__ __forceinline__ void half_pair(const uint32_t* x, int s, uint32_t& b0, uint32_t& b1) {
    uint32_t lo, hi;
    if constexpr (KV4) {
        const int w = s >> 1, o = s & 1;
        lo = x[4 * w + o];
        hi = x[4 * w + 2 + o];
    } else {
        lo = x[2 * s];
        hi = x[2 * s + 1];
    }
    b0 = prmt(lo, hi, 0x5410);
    b1 = prmt(lo, hi, 0x7632);
}

// fp16 multiplier and offset that turn an exponent-inserted code into code * 2^e,
// e up to 5 (see fma_exponent; groups with larger scales take the general path)
struct VScale {
    uint32_t mul, bias;       // INT8, or the low nibbles
    uint32_t mul_hi, bias_hi;  // the high nibbles (inserted as 16 * code)
};
template <bool KV4>
__device__ __forceinline__ VScale vscale_pair(int ea, int eb) {
    const float fa = pow2f(ea), fb = pow2f(eb);
    VScale s;
    s.mul = pack_half2(fa, fb);
    if constexpr (KV4) {
        s.bias = pack_half2(-1032.0f * fa, -1032.0f * fb);
        s.mul_hi = pack_half2(fa * 0.0625f, fb * 0.0625f);
        s.bias_hi = pack_half2(-72.0f * fa, -72.0f * fb);
    } else {
        s.bias = pack_half2(-1152.0f * fa, -1152.0f * fb);
        s.mul_hi = s.bias_hi = 0u;
    }
    return s;
}

template <bool KV4, int D, int RT, bool UNI>
__global__ void __launch_bounds__(kRowsThreads, rows_ctas_per_sm<D, RT>()) tree_rows_kernel(TreeParams p) {
    using F = RowsFmt<KV4, D>;
    constexpr int BM = 16 * RT, KS = D / 16, NT = D / 8;
    extern __shared__ __align__(16) float sm_o[];  // [4][BM][D] outputs, then [4][BM][2] maxima and sums
    __shared__ int s_bad;                          // an exact V row holds an infinity or a NaN
    grid_dependency_wait();
    grid_launch_dependents();
    const int item = blockIdx.x / p.Hkv, h = blockIdx.x - item * p.Hkv;
    if (!tree_plan_matches(p, BM)) {
        if (blockIdx.x == 0 && threadIdx.x == 0) flag(p.status, MG_DEV_BAD_ARGUMENT);
        return;
    }
    if (item >= p.plan[0]) return;
    if (p.status && (*(volatile int32_t*)p.status & kStopBits)) return;
    const int4 r0 = *reinterpret_cast<const int4*>(p.plan + p.lay.off_items + static_cast<int64_t>(item) * 8);
    const int4 r1 = *reinterpret_cast<const int4*>(p.plan + p.lay.off_items + static_cast<int64_t>(item) * 8 + 4);
    const int b = r0.x, row0 = r0.y * BM, j0 = r0.z, j1 = r0.z + r0.w;
    const int pslot = r1.x, nd = r1.y, n = r1.z;
    const int rows = nd * p.G;  // query rows of this (sequence, kv head)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    if (threadIdx.x == 0) s_bad = 0;
    __syncthreads();

    // Q fragments: rows g and g + 8 of each 16-row tile, quarter c of the head
    uint32_t qf[RT][KS][4];
    int tok[RT][2];  // drafted token of each row, -1 past the last
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int r = row0 + rt * 16 + g + 8 * u;
            tok[rt][u] = r < rows ? r / p.G : -1;
            uint32_t x[D / 8];
#pragma unroll
            for (int i = 0; i < D / 8; ++i) x[i] = 0u;
            if (r < rows) {
                const int t = r / p.G, hh = h * p.G + (r - t * p.G);
                ldg_half_words(x, p.q + b * p.q_sb + t * p.q_st + hh * p.q_sh + c * (D / 4));
            }
#pragma unroll
            for (int s = 0; s < KS; ++s) half_pair<KV4>(x, s, qf[rt][s][u], qf[rt][s][2 + u]);
        }

    float o[RT][NT][4], m[RT][2], l[RT][2];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int u = 0; u < 2; ++u) m[rt][u] = -INFINITY, l[rt][u] = 0.0f;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[rt][j][i] = 0.0f;
    }

    // one group of 16 keys: kfrag(nt, s) and vfrag(j) give the fragments, ks
    // the score factor and vm the probability factor of this lane's keys
    // (2c, 2c+1, 2c+8, 2c+9), ivm its reciprocal, seen(rt, u, i) whether row and key
    // meet (kUniGroup: the four are the same, ks is positive and every key is seen;
    // kTinyGroup: ivm may be 0, for a key whose factor is too small to divide out)
    auto attend = [&](auto&& kfrag, auto&& vfrag, const float (&ks)[4], const float (&vm)[4], const float (&ivm)[4],
                      auto&& seen, auto kind) {
        constexpr bool kUni = decltype(kind)::value == kUniGroup, kTiny = decltype(kind)::value == kTinyGroup;
        float s[RT][2][4];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[rt][nt][i] = 0.0f;
#pragma unroll
        for (int st = 0; st < KS; ++st)
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
                uint32_t b0, b1;
                kfrag(nt, st, b0, b1);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) mma_16816(s[rt][nt], qf[rt][st], b0, b1);
            }
        uint32_t pf[RT][4];
        const float lvm = kUni ? __log2f(vm[0]) : 0.0f;
        const float iuni = kUni ? ivm[0] : 1.0f;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = nt * 2 + (i & 1), u = i >> 1;
                    if constexpr (!kUni) s[rt][nt][i] = seen(rt, u, key) ? s[rt][nt][i] * ks[key] : -INFINITY;
                    mx[u] = fmaxf(mx[u], s[rt][nt][i]);
                }
            if constexpr (kUni) mx[0] *= ks[0], mx[1] *= ks[0];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                mx[u] = fmaxf(mx[u], __shfl_xor_sync(0xffffffffu, mx[u], 1));
                mx[u] = fmaxf(mx[u], __shfl_xor_sync(0xffffffffu, mx[u], 2));
            }
            // The reference is set 2^6 below the largest score and moves only when
            // a score passes it by 2^14: rescaling the output is rare, and skipped
            // by the whole warp; a probability times the V scale's mantissa (below
            // 2) stays inside fp16, and one of 2^-31 of the largest still counts.
            if (__any_sync(0xffffffffu, mx[0] > m[rt][0] + 14.0f || mx[1] > m[rt][1] + 14.0f)) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float mn = fmaxf(m[rt][u], mx[u] - 6.0f);
                    const float f = mn == -INFINITY ? 1.0f : ex2(m[rt][u] - mn);
                    m[rt][u] = mn;
                    l[rt][u] *= f;
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        o[rt][j][2 * u] *= f;
                        o[rt][j][2 * u + 1] *= f;
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float ref = m[rt][u] == -INFINITY ? 0.0f : m[rt][u];
                // Probabilities go to fp16 for the product with V, half a unit in
                // 2^11 each.  The sum (fp32) takes them as rounded, so that the
                // error of a row that one key dominates cancels.
                if constexpr (kUni) {
                    // the V scale's mantissa goes into the exponent, and out of the sum again
                    const float off = lvm - ref;
                    float sum = 0.0f;
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt) {
                        pf[rt][nt * 2 + u] = pack_half2(ex2(fmaf(s[rt][nt][2 * u], ks[0], off)),
                                                        ex2(fmaf(s[rt][nt][2 * u + 1], ks[0], off)));
                        const float2 pr = unpack_half2(pf[rt][nt * 2 + u]);
                        sum += pr.x + pr.y;
                    }
                    l[rt][u] = fmaf(sum, iuni, l[rt][u]);
                } else {
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt) {
                        const float p0 = ex2(s[rt][nt][2 * u] - ref), p1 = ex2(s[rt][nt][2 * u + 1] - ref);
                        pf[rt][nt * 2 + u] = pack_half2(p0 * vm[nt * 2], p1 * vm[nt * 2 + 1]);
                        const float2 pr = unpack_half2(pf[rt][nt * 2 + u]);
                        if constexpr (kTiny) {
                            const float i0 = ivm[nt * 2], i1 = ivm[nt * 2 + 1];
                            l[rt][u] = fmaf(i0 == 0.0f ? p0 : pr.x, i0 == 0.0f ? 1.0f : i0,
                                            fmaf(i1 == 0.0f ? p1 : pr.y, i1 == 0.0f ? 1.0f : i1, l[rt][u]));
                        } else {
                            l[rt][u] = fmaf(pr.x, ivm[nt * 2], fmaf(pr.y, ivm[nt * 2 + 1], l[rt][u]));
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            uint32_t b0, b1;
            vfrag(j, b0, b1);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) mma_16816(o[rt][j], pf[rt], b0, b1);
        }
    };

    const int whole = (n / p.P) * p.P;  // tokens in committed pages
    const int nct = (n + kTreeTile - 1) / kTreeTile;
    const int32_t* bt = p.block_tables + static_cast<int64_t>(b) * p.max_blocks;
    auto page_of = [&](int token) -> int32_t {
        const int32_t pg = bt[p.div_p.div(token)];
        if (pg < 0 || pg >= p.num_pages) {
            flag(p.status, MG_DEV_BAD_PAGE_ID);
            return 0;
        }
        return pg;
    };
    auto slot_of = [&](int token) { return token - static_cast<int>(p.div_p.div(token)) * p.P; };
    auto scale_at = [&](const float* scales, int32_t page, int slot) {
        return p.scale_th ? scales[(static_cast<int64_t>(page) * p.P + slot) * p.Hkv + h] : scales[page];
    };
    auto row_at = [&](const uint8_t* pool, int32_t page, int slot) {
        return pool + ((static_cast<int64_t>(page) * p.P + slot) * p.Hkv + h) * F::kRowBytes;
    };
    auto code_k = [&](const uint32_t (&w)[F::KW], int s, uint32_t& b0, uint32_t& b1) {
        if constexpr (KV4) {
            const uint32_t x = (w[s >> 1] ^ 0x88888888u) >> (8 * (s & 1));
            b0 = s4pair_lo_to_half2(x);
            b1 = s4pair_hi_to_half2(x);
        } else {
            b0 = s8pair_to_half2(w[s]);
            b1 = s8pair_to_half2(w[s] >> 8);
        }
    };
    auto code_v = [&](uint32_t wa, uint32_t wb, int j, const VScale& sc) -> uint32_t {
        if constexpr (KV4) {  // j: nibble 0..7 of the words
            const uint32_t x = (prmt(wa, wb, (j & 4) ? 0x7632 : 0x5410) ^ 0x88888888u) >> ((j & 2) ? 8 : 0);
            return (j & 1) ? hfma2_u32(lop3_and_or(x, 0x00F000F0u, 0x64006400u), sc.mul_hi, sc.bias_hi)
                           : hfma2_u32(lop3_and_or(x, 0x000F000Fu, 0x64006400u), sc.mul, sc.bias);
        } else {  // j: byte 0..3
            const uint32_t x = prmt(wa, wb, (j & 2) ? 0x7632 : 0x5410) >> ((j & 1) ? 8 : 0);
            return hfma2_u32(lop3_and_xor(x, 0x00FF00FFu, 0x64806480u), sc.mul, sc.bias);
        }
    };
    constexpr int kPerWord = KV4 ? 8 : 4;

    // ---- groups that lie in committed pages: codes only, loaded one group ahead
    struct Raw {
        uint32_t k[2][F::KW], v[4][F::VW];
        float ks[UNI ? 1 : 4], vs[UNI ? 1 : 4];
    };
    const int step = p.Hkv * F::kRowBytes;  // bytes from one token to the next
    const int64_t page_bytes = static_cast<int64_t>(p.P) * step;
    const uint8_t* k_lane = p.k_pool + static_cast<int64_t>(h) * F::kRowBytes + g * step + c * (F::KW * 4);
    const uint8_t* v_lane = p.v_pool + static_cast<int64_t>(h) * F::kRowBytes + 2 * c * step + g * (F::VW * 4);
    auto load_raw = [&](int tok0, int32_t page, Raw& r) {
        // page: of the whole group (UNI), else of key lane & 15 of the group
        if constexpr (UNI) {
            const int slot = slot_of(tok0);
            // one wide multiplication per group; everything else is this lane's own
            const int64_t at = page * page_bytes + slot * step;
            const uint8_t* kb = k_lane + at;
            const uint8_t* vb = v_lane + at;
            ldg_words(r.k[0], kb);
            ldg_words(r.k[1], kb + 8 * step);
            ldg_words(r.v[0], vb);
            ldg_words(r.v[1], vb + step);
            ldg_words(r.v[2], vb + 8 * step);
            ldg_words(r.v[3], vb + 9 * step);
            r.ks[0] = p.k_scales[page];
            r.vs[0] = p.v_scales[page];
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int key = g + 8 * i;
                const int32_t pg = __shfl_sync(0xffffffffu, page, key);
                ldg_words(r.k[i], row_at(p.k_pool, pg, slot_of(tok0 + key)) + c * (F::KW * 4));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = 2 * c + (i & 1) + 8 * (i >> 1);
                const int32_t pg = __shfl_sync(0xffffffffu, page, key);
                const int slot = slot_of(tok0 + key);
                ldg_words(r.v[i], row_at(p.v_pool, pg, slot) + g * (F::VW * 4));
                r.ks[i] = scale_at(p.k_scales, pg, slot);
                r.vs[i] = scale_at(p.v_scales, pg, slot);
            }
        }
    };
    auto group_page = [&](int tok0) { return page_of(UNI ? tok0 : tok0 + (lane & 15)); };
    const int wt = 16 * warp;
    int jp = j0;           // first tile after the paged groups of this warp
    bool some_big = false;  // a group had a V scale of 64 or more and is left for later
    // (or one below 2^-20, whose exponent does not fit either)
    auto big = [](float v) { return v >= 64.0f || v < 0x1p-20f; };
    {
        const int lim = whole - wt - 16;
        const int jend = lim < 0 ? j0 : min(j1, lim / kTreeTile + 1);
        if (jend > j0) {
            Raw cur, nxt;
            int32_t page = group_page(j0 * kTreeTile + wt);
            load_raw(j0 * kTreeTile + wt, page, nxt);
            if (j0 + 1 < jend) page = group_page((j0 + 1) * kTreeTile + wt);
            for (int j = j0; j < jend; ++j) {
                cur = nxt;
                if (j + 1 < jend) {
                    load_raw((j + 1) * kTreeTile + wt, page, nxt);
                    if (j + 2 < jend) page = group_page((j + 2) * kTreeTile + wt);
                }
                bool over = big(cur.vs[0]);
                if constexpr (!UNI) over |= big(cur.vs[1]) | big(cur.vs[2]) | big(cur.vs[3]);
                if (__any_sync(0xffffffffu, over)) {
                    some_big = true;
                    continue;
                }
                float ks[4], vm[4], ivm[4];
                VScale vsc[2];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float v = cur.vs[UNI ? 0 : i];
                    ks[i] = cur.ks[UNI ? 0 : i] * p.scale_log2;
                    vm[i] = v * pow2f(-scale_exponent(v));
                    ivm[i] = rcp(vm[i]);
                }
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    vsc[i] = vscale_pair<KV4>(scale_exponent(cur.vs[UNI ? 0 : 2 * i]),
                                              scale_exponent(cur.vs[UNI ? 0 : 2 * i + 1]));
                attend([&](int nt, int s, uint32_t& b0, uint32_t& b1) { code_k(cur.k[nt], s, b0, b1); },
                       [&](int jj, uint32_t& b0, uint32_t& b1) {
                           const int w = jj / kPerWord, e = jj % kPerWord;
                           b0 = code_v(cur.v[0][w], cur.v[1][w], e, vsc[0]);
                           b1 = code_v(cur.v[2][w], cur.v[3][w], e, vsc[1]);
                       },
                       ks, vm, ivm, [](int, int, int) { return true; },
                       std::integral_constant<int, UNI ? kUniGroup : kPagedGroup>{});
            }
            jp = jend;
        }
    }

    // ---- groups with staged rows, and the drafted tokens: fragments of halves
    bool bad = false;
    uint32_t kh[2][D / 8] = {}, vh[4][D / 16] = {};
    auto half_groups = [&](const float (&ks)[4], const float (&vm)[4], const float (&ivm)[4], auto&& seen) {
        attend([&](int nt, int s, uint32_t& b0, uint32_t& b1) { half_pair<KV4>(kh[nt], s, b0, b1); },
               [&](int jj, uint32_t& b0, uint32_t& b1) {
                   const uint32_t sel = (jj & 1) ? 0x7632 : 0x5410;
                   b0 = prmt(vh[0][jj >> 1], vh[1][jj >> 1], sel);
                   b1 = prmt(vh[2][jj >> 1], vh[3][jj >> 1], sel);
               },
               ks, vm, ivm, seen, std::integral_constant<int, kTinyGroup>{});
    };
    auto clear_half = [&]() {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) kh[0][i] = kh[1][i] = 0u;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) vh[0][i] = vh[1][i] = vh[2][i] = vh[3][i] = 0u;
    };
    auto keep_finite = [&](uint32_t (&x)[D / 16]) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
            if (nonfinite2(x[i])) {
                bad = true;
                x[i] = finite_or_zero2(x[i]);
            }
    };
    for (int j = some_big ? j0 : jp; j < min(j1, nct); ++j) {
        const int tok0 = j * kTreeTile + wt;
        if (tok0 >= n) break;
        if (j < jp) {  // of the paged groups, those left for later
            const int key = tok0 + (lane & 15);
            if (!__any_sync(0xffffffffu, big(scale_at(p.v_scales, page_of(key), slot_of(key))))) continue;
        }
        clear_half();
        float ks[4], vm[4], ivm[4];
        // a code as a half: its integer value; K's scale goes into the score,
        // V's exponent into the half and its mantissa into the probability
        auto half_code = [&](const uint32_t* w, int i) -> uint32_t {  // elements 2i, 2i + 1
            float a, bb;
            if constexpr (KV4) {
                const uint32_t x = w[i >> 2] >> (8 * (i & 3));
                a = static_cast<float>(static_cast<int32_t>(x << 28) >> 28);
                bb = static_cast<float>(static_cast<int32_t>(x << 24) >> 28);
            } else {
                const uint32_t x = w[i >> 1] >> (16 * (i & 1));
                a = static_cast<float>(static_cast<int8_t>(x & 255u));
                bb = static_cast<float>(static_cast<int8_t>((x >> 8) & 255u));
            }
            return pack_half2(a, bb);
        };
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int tk = tok0 + g + 8 * i;
            if (tk < whole) {
                uint32_t w[F::KW];
                ldg_words(w, row_at(p.k_pool, page_of(tk), slot_of(tk)) + c * (F::KW * 4));
#pragma unroll
                for (int e = 0; e < D / 8; ++e) kh[i][e] = half_code(w, e);
            } else if (tk < n) {
                ldg_half_words(kh[i], p.staging_k + ((static_cast<int64_t>(b) * p.P + (tk - whole)) * p.Hkv + h) * D +
                                          c * (D / 4));
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int tk = tok0 + 2 * c + (i & 1) + 8 * (i >> 1);
            ks[i] = p.scale_log2;
            vm[i] = ivm[i] = 1.0f;
            if (tk < whole) {
                const int32_t pg = page_of(tk);
                const float vs = scale_at(p.v_scales, pg, slot_of(tk));
                ks[i] = scale_at(p.k_scales, pg, slot_of(tk)) * p.scale_log2;
                const int e2 = scale_exponent(vs);
                // a scale below 2^-27 leaves too few bits of the rounded probability for
                // the sum, which takes the unrounded one; the key's part of the output is
                // below 127 x 2^-27, where that error is far below the smallest half
                vm[i] = vs * pow2f(-e2);
                ivm[i] = fabsf(vs) < 0x1p-27f ? 0.0f : rcp(vm[i]);
                const uint32_t f = half_bits(pow2f(e2)) * 0x10001u;
                uint32_t w[F::VW];
                ldg_words(w, row_at(p.v_pool, pg, slot_of(tk)) + g * (F::VW * 4));
#pragma unroll
                for (int e = 0; e < D / 16; ++e) vh[i][e] = hfma2_u32(half_code(w, e), f, 0u);
            } else if (tk < n) {
                ldg_half_words(vh[i], p.staging_v + ((static_cast<int64_t>(b) * p.P + (tk - whole)) * p.Hkv + h) * D +
                                          g * (D / 8));
                keep_finite(vh[i]);
            }
        }
        half_groups(ks, vm, ivm, [&](int, int, int key) { return tok0 + 2 * c + (key & 1) + 8 * (key >> 1) < n; });
    }
    // drafted tokens; without a mask none past the row tile's last token is seen
    const int tmax = min(nd, p.mask ? nd : (min(row0 + BM, rows) - 1) / p.G + 1);
    const int d0 = max(j0, nct);
    const float ones[4] = {1.0f, 1.0f, 1.0f, 1.0f};
    const float ks1[4] = {p.scale_log2, p.scale_log2, p.scale_log2, p.scale_log2};
    for (int j = d0; j < j1; ++j) {
        const int u0 = (j - nct) * kTreeTile + wt;
        if (u0 >= tmax) break;
        clear_half();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int u = u0 + g + 8 * i;
            if (u < tmax) ldg_half_words(kh[i], p.k + b * p.k_sb + u * p.k_st + h * p.k_sh + c * (D / 4));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int u = u0 + 2 * c + (i & 1) + 8 * (i >> 1);
            if (u < tmax) {
                ldg_half_words(vh[i], p.v + b * p.v_sb + u * p.v_st + h * p.v_sh + g * (D / 8));
                keep_finite(vh[i]);
            }
        }
        half_groups(ks1, ones, ones, [&](int rt, int uu, int key) {
            const int u = u0 + 2 * c + (key & 1) + 8 * (key >> 1);
            return tok[rt][uu] >= 0 && u < tmax && tree_sees(p, b, tok[rt][uu], u);
        });
    }
    if (bad) atomicOr(&s_bad, 1);

    // ---- join the four warps
    float* sm_ml = sm_o + kRowsWarps * BM * D;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            l[rt][u] += __shfl_xor_sync(0xffffffffu, l[rt][u], 1);
            l[rt][u] += __shfl_xor_sync(0xffffffffu, l[rt][u], 2);
            const int r = rt * 16 + g + 8 * u;
            if (c == 0) {
                sm_ml[(warp * BM + r) * 2] = m[rt][u];
                sm_ml[(warp * BM + r) * 2 + 1] = l[rt][u];
            }
            float* dst = sm_o + (warp * BM + r) * D + c * (D / 4);
#pragma unroll
            for (int j = 0; j < NT; j += 4) {
                *reinterpret_cast<float4*>(dst + j) = make_float4(o[rt][j][2 * u], o[rt][j + 1][2 * u],
                                                                  o[rt][j + 2][2 * u], o[rt][j + 3][2 * u]);
                *reinterpret_cast<float4*>(dst + D / 8 + j) =
                    make_float4(o[rt][j][2 * u + 1], o[rt][j + 1][2 * u + 1], o[rt][j + 2][2 * u + 1],
                                o[rt][j + 3][2 * u + 1]);
            }
        }
    __syncthreads();
    const bool fix = s_bad != 0;
    const int live = min(BM, rows - row0);
    for (int i = threadIdx.x; i < live * (D / 4); i += kRowsThreads) {
        const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
        float mw[kRowsWarps], mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < kRowsWarps; ++w) {
            mw[w] = sm_ml[(w * BM + r) * 2];
            mx = fmaxf(mx, mw[w]);
        }
        float ls = 0.0f, a[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < kRowsWarps; ++w) {
            const float f = mx == -INFINITY ? 0.0f : ex2(mw[w] - mx);
            const float4 x = *reinterpret_cast<const float4*>(sm_o + (w * BM + r) * D + d);
            ls += f * sm_ml[(w * BM + r) * 2 + 1];
            a[0] += f * x.x;
            a[1] += f * x.y;
            a[2] += f * x.z;
            a[3] += f * x.w;
        }
        const int row = row0 + r, t = row / p.G;
        if (fix)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                a[e] += nonfinite_sum(p, b, h, D, t, d + e, max(whole, j0 * kTreeTile), min(n, j1 * kTreeTile),
                                      max(0, (j0 - nct) * kTreeTile), min(tmax, (j1 - nct) * kTreeTile));
        if (pslot < 0) {
            const float inv = ls > 0.0f || isnan(ls) ? 1.0f / ls : 0.0f;
            uint2 w;
            w.x = pack_half2(a[0] * inv, a[1] * inv);
            w.y = pack_half2(a[2] * inv, a[3] * inv);
            const int hh = h * p.G + (row - t * p.G);
            *reinterpret_cast<uint2*>(p.out + ((static_cast<int64_t>(b) * p.T + t) * p.Hkv * p.G + hh) * D + d) = w;
        } else {
            const int64_t slot = (static_cast<int64_t>(pslot) * p.Hkv + h) * BM + r;
            *reinterpret_cast<float4*>(p.part_o + slot * D + d) = make_float4(a[0], a[1], a[2], a[3]);
            if (d == 0) *reinterpret_cast<float2*>(p.part_ml + slot * 2) = make_float2(mx, ls);
        }
    }
}

template <bool KV4, int D, int RT, bool UNI>
void run_tree_rows(const TreeParams& p, const TreeGeom& g, cudaStream_t stream) {
    constexpr int BM = 16 * RT;
    constexpr int smem = kRowsWarps * BM * (D + 2) * 4;
    auto kern = tree_rows_kernel<KV4, D, RT, UNI>;
    if (smem > 48 * 1024) cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(g.max_items * p.Hkv));
    cfg.blockDim = dim3(kRowsThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kern, p);
}

template <bool KV4, int D>
void launch_tree_rows(const TreeParams& p, const TreeGeom& g, cudaStream_t stream) {
    // groups of 16 keys never cross a page, and one scale serves them
    const bool uni = p.P % 16 == 0 && !p.scale_th;
    if constexpr (D == 64) {
        if (g.BM == 32) {
            uni ? run_tree_rows<KV4, D, 2, true>(p, g, stream) : run_tree_rows<KV4, D, 2, false>(p, g, stream);
            return;
        }
    }
    uni ? run_tree_rows<KV4, D, 1, true>(p, g, stream) : run_tree_rows<KV4, D, 1, false>(p, g, stream);
}

}  // namespace mg
