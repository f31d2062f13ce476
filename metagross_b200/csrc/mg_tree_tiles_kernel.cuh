// Attention of many query rows per (sequence, kv head) over the paged cache and
// the drafted tokens, on tcgen05 tensor cores.
//
// One CTA per work item: a row tile of up to 128 query rows (t-major, G heads
// each) and a run of 128-key tiles.
//   S = Q K^T    [128 rows x 128 keys]   A = Q, B = K tile, both in shared memory
//   O += P V     [128 rows x D]          A = P in tensor memory, B = V tile
// A softmax thread owns one row: its maximum and sum are registers and nothing
// is exchanged between threads.  The tiles form two streams, even and odd, each
// with its own warpgroup, references, sums and output in tensor memory, joined
// once at the end: a tile's softmax is a long chain of dependent steps, and two
// chains run side by side without ever meeting.  (With the keys in the lanes and
// four warpgroups on one tile, the common maximum took a vote per tile and P a
// trip through shared memory: 3300 clocks a tile against 1024 of exponentials.)
//
// What a row needs over all keys:
//   maximum  a reference; 32 scores at a time are compared with it, and only when
//            one passes it by a wide margin does the warp move it: sum, output and
//            the tile's probabilities so far are rescaled in place.
//   sum      fp32, of the unrounded probabilities.  The products take them rounded to
//            fp16: relative error 2.9e-4 of the output, where the row kernel, which sums
//            them as rounded at the price of unpacking every pair, has 2.2e-4.
//
// Roles (warpgroups; registers are moved to the softmax):
//   0, 1     softmax of the even / odd tiles: S from tensor memory, P over it
//   2 .. 5   a thread per key turns codes, loaded to registers ahead of time,
//            into fp16 operand tiles: K and V of the even tiles, K and V of the odd
//   6        one warp issues the products
// K, V: a slot for even and one for odd tiles; S / P: three in tensor memory
// (two for D = 128), so that S of a stream's next tile is ready before its softmax
// ends.  Only mbarriers between the roles.
//
// Bound: the exponentials (16 per clock and SM): 128 x 128 scores take 1024
// clocks, the products 512 (D = 64) or 1024; for few rows the conversion and loads.
// Measured (one B200): about 2800 clocks a tile, from the latency of a softmax warp's
// chain (issue slots 50 % used, exponentials at 35 % of their rate, tensor pipe 16 %);
// 8 chunks of 512 tokens over 3000 to 5000, 32 q / 4 kv heads of 64, INT8: 427 us a
// layer, 335 TFLOP/s, 1.7 us of an SM per tile.  Short items are dearer, since the
// registers leave room for one CTA per SM and nothing runs beside its prologue, first
// conversion and epilogue: 64 contexts U[128, 2048] with trees of 16, INT4, are 388
// items of 6.7 tiles, 79 us a layer, 4.5 us of an SM per tile.
#pragma once

#include "mg_tcgen05.cuh"
#include "mg_tree.cuh"

namespace mg {

constexpr uint32_t kTilesTries = 1u << 17;  // attempts of a bounded wait
constexpr uint32_t kTilesNap = 100;         // ns between the attempts of a role with time to spare
constexpr float kUnset = -1e30f;            // reference of a row that has seen no key
// A row's reference is set 2^kBelow (and up to twice that) below its largest score
// so far and moves when a score passes it by 2^kSlack: the probability times the V
// scale's mantissa (below 2) stays inside fp16, probabilities of 2^-18 of the largest
// keep their 11 bits and those of 2^-28 still count (the sum is fp32 and unrounded).
// Moving is slow, so when a warp does it every row that rose by 2^kRefresh over its
// reference takes part: eight chunks of 512 tokens over 3000 to 5000 tokens, two
// layers, 857 us (871 when only those past 2^kSlack do).  With the reference at the
// maximum it is 841, but then rows that one key dominates lose their tail.
constexpr float kSlack = 14.99f, kBelow = 4.0f, kRefresh = 6.0f;

template <bool KV4, int D>
struct TilesCfg {
    static constexpr int THREADS = 7 * 128;
    // registers a thread: 72 at launch, then 2 softmax + 4 conversion + 1 issue warpgroups
    static constexpr int kRegsSoftmax = 128, kRegsConvert = 56, kRegsIssue = 24;
    static_assert(2 * kRegsSoftmax + 4 * kRegsConvert + kRegsIssue == 7 * 72, "register split of the launch");
    static constexpr int RB = KV4 ? D / 2 : D;  // bytes of a code row
    static constexpr int RW = RB / 4;
    static constexpr int DB = D / 64;
    static constexpr int NB = D == 64 ? 3 : 2;  // S / P buffers in tensor memory
    static constexpr uint32_t kTileBytes = 128 * D * 2;
    static constexpr uint32_t kK = 0, kV = 2 * kTileBytes, kQ = 4 * kTileBytes, kMisc = 5 * kTileBytes;
    // misc: ks[8][128], vm[8][128], token[128], offset[128], (m, l)[2][128]
    static constexpr uint32_t kSmem = kMisc + (1024 + 1024 + 128 + 128 + 512) * 4 + 1024;
    static_assert(kSmem <= 227 * 1024, "shared memory of an SM");
    static_assert(NB * 128 + 2 * D <= 512, "tensor memory of an SM");
};

// 8 positions (16 bytes) of row r at position d0 of a swizzled operand tile
__device__ __forceinline__ void put8(uint32_t base, int block_bytes, int r, int d0, uint32_t a, uint32_t b, uint32_t c,
                                     uint32_t d) {
    const uint32_t at = base + (d0 >> 6) * block_bytes + r * 128 + ((((d0 >> 3) & 7) ^ (r & 7)) << 4);
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// Inside the head dimension the positions of K, V and Q hold the values in the
// order the codes come out of their words: 0 2 1 3 of every four (INT8), 0 4 1
// 5 2 6 3 7 of every eight (INT4).
template <bool KV4>
__device__ __forceinline__ void put_halves8(uint32_t base, int block_bytes, int r, int d0, const uint32_t (&x)[4]) {
    if constexpr (KV4)
        put8(base, block_bytes, r, d0, prmt(x[0], x[2], 0x5410), prmt(x[0], x[2], 0x7632), prmt(x[1], x[3], 0x5410),
             prmt(x[1], x[3], 0x7632));
    else
        put8(base, block_bytes, r, d0, prmt(x[0], x[1], 0x5410), prmt(x[0], x[1], 0x7632), prmt(x[2], x[3], 0x5410),
             prmt(x[2], x[3], 0x7632));
}
__device__ __forceinline__ void ldg_halves8(const __half* a, uint32_t (&x)[4]) {
    asm volatile("ld.global.v2.b32 {%0,%1}, [%2];" : "=r"(x[0]), "=r"(x[1]) : "l"(a));
    asm volatile("ld.global.v2.b32 {%0,%1}, [%2];" : "=r"(x[2]), "=r"(x[3]) : "l"(a + 4));
}
// A row of codes, times the power of two behind mul / bias, to the positions of row r.
template <bool KV4, int RW>
__device__ __forceinline__ void put_code_row(uint32_t base, int r, const uint32_t (&w)[RW], uint32_t mul, uint32_t bias,
                                             uint32_t mul_hi, uint32_t bias_hi) {
    if constexpr (KV4) {
#pragma unroll
        for (int x = 0; x < RW; ++x) {
            const uint32_t y = w[x] >> 8;
            put8(base, 16384, r, 8 * x, hfma2_u32(lop3_and_xor(w[x], 0x000F000Fu, 0x64086408u), mul, bias),
                 hfma2_u32(lop3_and_xor(w[x], 0x00F000F0u, 0x64806480u), mul_hi, bias_hi),
                 hfma2_u32(lop3_and_xor(y, 0x000F000Fu, 0x64086408u), mul, bias),
                 hfma2_u32(lop3_and_xor(y, 0x00F000F0u, 0x64806480u), mul_hi, bias_hi));
        }
    } else {
#pragma unroll
        for (int x = 0; x < RW; x += 2)
            put8(base, 16384, r, 4 * x, hfma2_u32(lop3_and_xor(w[x], 0x00FF00FFu, 0x64806480u), mul, bias),
                 hfma2_u32(lop3_and_xor(w[x] >> 8, 0x00FF00FFu, 0x64806480u), mul, bias),
                 hfma2_u32(lop3_and_xor(w[x + 1], 0x00FF00FFu, 0x64806480u), mul, bias),
                 hfma2_u32(lop3_and_xor(w[x + 1] >> 8, 0x00FF00FFu, 0x64806480u), mul, bias));
    }
}

// Which of the drafted tokens u .. u + 31 (the first cnt of them exist) token t sees.
__device__ __forceinline__ uint32_t mask_bits(const TreeParams& p, int b, int t, int u, int cnt) {
    const uint8_t* m = p.mask + static_cast<int64_t>(b) * p.mask_sb + static_cast<int64_t>(t) * p.T + u;
    uint32_t bits = 0u;
    if (cnt >= 32 && (reinterpret_cast<uintptr_t>(m) & 3u) == 0) {
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = reinterpret_cast<const uint32_t*>(m)[e];
        // four bytes of 0 or 1 to four bits: their sum weighted 1 2 4 8 lands in the top byte
#pragma unroll
        for (int e = 0; e < 8; ++e) bits |= (__vminu4(w[e], 0x01010101u) * 0x01020408u >> 24) << (4 * e);
    } else {
        // every byte asked for before the first is looked at
        uint32_t byte[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) byte[e] = e < cnt ? m[e] : 0u;
#pragma unroll
        for (int e = 0; e < 32; ++e) bits |= byte[e] ? 1u << e : 0u;
    }
    return bits;
}

// UNI: 16 keys that start on a multiple of 16 share their scales (page scales, pages
// of a multiple of 16 tokens), which then cost the softmax an eighth of the loads
// (1.42 -> 1.15 us a tile of 128 x 128 with every such load taken out).
template <bool KV4, int D, bool UNI>
__global__ void __launch_bounds__(TilesCfg<KV4, D>::THREADS, 1) tree_tiles_kernel(TreeParams p) {
    using C = TilesCfg<KV4, D>;
    constexpr int NB = C::NB;
    extern __shared__ uint8_t sm_raw[];
    // written: Q; K and V of a slot; P of a buffer.  done: S of a buffer; O += P V of a stream;
    // and every product.  A wait names a phase by its parity, so whoever waits has
    // to know that the phase before it is over; the end has a barrier of its own.
    __shared__ uint64_t bar_q, bar_k[2], bar_v[2], bar_p[3], bar_s[3], bar_o[2], bar_end;
    __shared__ uint32_t s_tmem;
    __shared__ int s_bad;
    uint8_t* sm = sm_raw + ((1024u - (smem_u32(sm_raw) & 1023u)) & 1023u);
    float* sm_ks = reinterpret_cast<float*>(sm + C::kMisc);  // a key's score factor
    float* sm_vm = sm_ks + 1024;                             // and its V scale's mantissa
    int* sm_tok = reinterpret_cast<int*>(sm_vm + 1024);      // drafted token of each row
    int* sm_off = sm_tok + 128;                              // its output row, from the sequence's first
    float2* sm_ml = reinterpret_cast<float2*>(sm_off + 128);

    grid_dependency_wait();
    grid_launch_dependents();
    const int item = blockIdx.x / p.Hkv, h = blockIdx.x - item * p.Hkv;
    if (!tree_plan_matches(p, p.BM)) {
        if (blockIdx.x == 0 && threadIdx.x == 0) flag(p.status, MG_DEV_BAD_ARGUMENT);
        return;
    }
    if (item >= p.plan[0]) return;
    if (p.status && (*(volatile int32_t*)p.status & kStopBits)) return;
    const int4 r0 = *reinterpret_cast<const int4*>(p.plan + p.lay.off_items + static_cast<int64_t>(item) * 8);
    const int4 r1 = *reinterpret_cast<const int4*>(p.plan + p.lay.off_items + static_cast<int64_t>(item) * 8 + 4);
    const int b = r0.x, row0 = r0.y * p.BM, j0 = r0.z;
    const int pslot = r1.x, nd = r1.y, n = r1.z;
    const int live = min(p.BM, nd * p.G - row0);  // query rows of this tile
    const int whole = (n / p.P) * p.P;             // tokens in committed pages
    const int nct = (n + kTilesKeys - 1) / kTilesKeys;
    // without a mask no drafted token past the row tile's last one is seen
    const int tmax = min(nd, p.mask ? nd : (row0 + live - 1) / p.G + 1);
    const int nt = max(0, min(r0.z + r0.w, nct + (tmax + kTilesKeys - 1) / kTilesKeys) - j0);
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int role = warp >> 2;

    if (warp == 0) tmem_alloc(&s_tmem, 512);
    if (tid == 0) {
        const int busy = (live + 31) / 32;  // softmax warps of a stream that hold a row
        mbar_init(&bar_q, 8);
        mbar_init(&bar_end, 1);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar_k[i], 4);
            mbar_init(&bar_v[i], 4);
            mbar_init(&bar_o[i], 1);
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            mbar_init(&bar_p[i], busy);
            mbar_init(&bar_s[i], 1);
        }
        fence_mbar_init();
        s_bad = 0;
    }
    if (tid < 128) {
        const int r = row0 + tid, t = r / p.G;
        sm_tok[tid] = t;
        sm_off[tid] = t * p.Hkv * p.G + h * p.G + (r - t * p.G);
    }
    __syncthreads();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *(volatile uint32_t*)&s_tmem, 0);
    const uint32_t tm_o = tmem + NB * 128;
    const uint32_t smb = smem_u32(sm);
    bool dead = false;  // a wait gave up: no further waits, the output is invalid
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (dead) return;
        if (!mbar_wait_bounded(bar, parity, kTilesTries)) {
            dead = true;
            flag(p.status, MG_DEV_TIMEOUT);
        }
    };
    // the same, out of the way of the warps that compute
    auto nap_wait = [&](uint64_t* bar, uint32_t parity) {
        if (dead) return;
#pragma unroll 1
        for (uint32_t i = 0; i < kTilesTries; ++i) {
            if (mbar_try_wait(bar, parity)) return;
            __nanosleep(kTilesNap);
        }
        dead = true;
        flag(p.status, MG_DEV_TIMEOUT);
    };
    auto full = [&](int i) { return (j0 + i + 1) * kTilesKeys <= whole; };  // tile of committed pages only

    if (role == 6) {
        // ------------------------------------------------ the products
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kRegsIssue));
        if (warp == 24 && nt > 0) {
            const bool leader = elect_one();
            constexpr uint32_t id_s = umma_idesc_f16(128, false, false), id_o = umma_idesc_f16(D, false, true);
            int sb = 0;  // buffer of the next S
            auto issue_s = [&](int i) {
                wait(&bar_k[i & 1], (i >> 1) & 1);
                tcgen05_fence_after();
                const uint32_t ka = smb + C::kK + (i & 1) * C::kTileBytes, qa = smb + C::kQ;
#pragma unroll
                for (int db = 0; db < C::DB; ++db)
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                        umma_f16(tmem + sb * 128, umma_desc(qa + db * 16384 + kk * 32, 16, 1024),
                                 umma_desc(ka + db * 16384 + kk * 32, 16, 1024), id_s, db + kk > 0, leader);
                umma_commit(&bar_s[sb], leader);
                sb = sb + 1 == NB ? 0 : sb + 1;
            };
            wait(&bar_q, 0);
#pragma unroll 1
            for (int i = 0; i < min(nt, NB); ++i) issue_s(i);
            int pb = 0, round = 0;  // buffer of P(i), and how often it has been used
#pragma unroll 1
            for (int i = 0; i < nt; ++i) {
                // S goes over the buffer that O(i - 1) took its P from: products with
                // different accumulators are not ordered, so that one is waited for
                if (i > 0 && i - 1 + NB < nt) {
                    wait(&bar_o[(i - 1) & 1], ((i - 1) >> 1) & 1);
                    tcgen05_fence_after();
                    issue_s(i - 1 + NB);
                }
                wait(&bar_v[i & 1], (i >> 1) & 1);
                wait(&bar_p[pb], round & 1);
                tcgen05_fence_after();
                const uint32_t va = smb + C::kV + (i & 1) * C::kTileBytes;
#pragma unroll
                for (int s = 0; s < 8; ++s)
                    umma_f16_ta(tm_o + (i & 1) * D, tmem + pb * 128 + s * 8, umma_desc(va + s * 2048, 16384, 1024), id_o,
                                i > 1 || s > 0, leader);
                umma_commit(&bar_o[i & 1], leader);
                if (++pb == NB) pb = 0, ++round;
            }
            umma_commit(&bar_end, leader);
        }
    } else if (role >= 2) {
        // ------------------------------------------------ codes to operand tiles
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kRegsConvert));
        const bool is_v = role & 1;
        const int first = (role - 2) >> 1;  // even or odd tiles
        const int r = tid & 127;            // this thread's key of every tile
        const int32_t* bt = p.block_tables + static_cast<int64_t>(b) * p.max_blocks;
        const int stride = p.Hkv * C::RB;  // bytes from one token to the next
        const int64_t page_bytes = static_cast<int64_t>(p.P) * stride;
        const uint8_t* base = (is_v ? p.v_pool : p.k_pool) + static_cast<int64_t>(h) * C::RB;
        const uint32_t dst = smb + (is_v ? C::kV : C::kK) + first * C::kTileBytes;
        bool bad = false;
        struct Place {
            int32_t page;
            int32_t slot;
        };
        auto place = [&](int32_t page, int token) -> Place {
            if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(p.num_pages)) {
                flag(p.status, MG_DEV_BAD_PAGE_ID);
                page = 0;
            }
            return Place{page, token - static_cast<int>(p.div_p.div(token)) * p.P};
        };
        auto scale_of = [&](const float* scales, const Place& q) {
            return p.scale_th ? scales[(static_cast<int64_t>(q.page) * p.P + q.slot) * p.Hkv + h] : scales[q.page];
        };
        auto load_row = [&](const Place& q, uint32_t (&w)[C::RW]) {
            const uint4* a = reinterpret_cast<const uint4*>(base + q.page * page_bytes + q.slot * stride);
#pragma unroll
            for (int x = 0; x < C::RW; x += 4) {
                const uint4 v = a[x / 4];
                w[x] = v.x, w[x + 1] = v.y, w[x + 2] = v.z, w[x + 3] = v.w;
            }
        };
        // codes to halves: K's plain, V's times the power of two of its scale
        auto put_codes = [&](const uint32_t (&w)[C::RW], float vs) {
            const int e = is_v ? scale_exponent(vs) : 0;
            const float f = pow2f(fma_exponent(e));
            const uint32_t mul = half_bits(f) * 0x10001u;
            if constexpr (KV4)
                put_code_row<true>(dst, r, w, mul, half_bits(-1032.0f * f) * 0x10001u, half_bits(f * 0.0625f) * 0x10001u,
                                   half_bits(-72.0f * f) * 0x10001u);
            else put_code_row<false>(dst, r, w, mul, half_bits(-1152.0f * f) * 0x10001u, 0u, 0u);
            if (e > 5) {  // the rest of 2^e, on the halves just written
                const uint32_t rest = half_bits(pow2f(e - 5)) * 0x10001u;
                for (int d = 0; d < D; d += 2) {
                    const uint32_t at = dst + (d >> 6) * 16384 + r * 128 + ((((d >> 3) & 7) ^ (r & 7)) << 4) + (d & 7) * 2;
                    uint32_t x;
                    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(x) : "r"(at) : "memory");
                    asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(hfma2_u32(x, rest, 0x80008000u)) : "memory");
                }
            }
        };
        // a tile with staged or drafted rows: by what this thread's key is
        auto put_mixed = [&](int i, float& ks, float& vs) {
            const int t = j0 + i, token = t * kTilesKeys + r, u = (t - nct) * kTilesKeys + r;
            const __half* src = nullptr;
            ks = vs = 1.0f;
            if (t < nct) {
                if (token < whole) {
                    const Place q = place(bt[p.div_p.div(token)], token);
                    uint32_t w[C::RW];
                    load_row(q, w);
                    ks = scale_of(p.k_scales, q);
                    vs = scale_of(p.v_scales, q);
                    put_codes(w, vs);
                    return;
                }
                if (token < n)
                    src = (is_v ? p.staging_v : p.staging_k) +
                          ((static_cast<int64_t>(b) * p.P + (token - whole)) * p.Hkv + h) * D;
            } else if (u < tmax) {
                src = is_v ? p.v + b * p.v_sb + u * p.v_st + h * p.v_sh : p.k + b * p.k_sb + u * p.k_st + h * p.k_sh;
            }
#pragma unroll 1
            for (int d0 = 0; d0 < D; d0 += 32) {  // 32 values in flight
                uint32_t y[4][4];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    y[x][0] = y[x][1] = y[x][2] = y[x][3] = 0u;
                    if (src) ldg_halves8(src + d0 + 8 * x, y[x]);
                }
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    if (is_v) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (nonfinite2(y[x][e])) {
                                bad = true;
                                y[x][e] = finite_or_zero2(y[x][e]);
                            }
                    }
                    put_halves8<KV4>(dst, 16384, r, d0 + 8 * x, y[x]);
                }
            }
        };
        // the codes of this group's next tile are loaded as soon as the registers
        // are free, the block-table entry one tile earlier (and checked only when
        // it is used).  Both scales of a tile go with its K, so that whoever has
        // its S has them.
        uint32_t w[C::RW];
        float ks = 1.0f, vs = 1.0f;
        int32_t page_next = 0;
        auto fetch_page = [&](int i) {
            if (i < nt && full(i)) page_next = bt[p.div_p.div((j0 + i) * kTilesKeys + r)];
        };
        auto fetch = [&](int i) {
            if (i >= nt || !full(i)) return;
            const Place at = place(page_next, (j0 + i) * kTilesKeys + r);
            load_row(at, w);
            vs = scale_of(p.v_scales, at);
            if (!is_v) ks = scale_of(p.k_scales, at);
        };
        fetch_page(first);
        fetch(first);
        fetch_page(first + 2);
        int sb = first == 0 ? 0 : 1, round = 0;  // buffer of S(i - 2), and how often it has been used
#pragma unroll 1
        for (int i = first; i < nt; i += 2) {
            if (i >= 2) {  // the product that read this slot last
                if (is_v) {
                    nap_wait(&bar_o[first], ((i - 2) >> 1) & 1);
                } else {
                    nap_wait(&bar_s[sb], round & 1);
                    sb += 2;
                    if (sb >= NB) sb -= NB, ++round;
                }
            }
            if (full(i)) put_codes(w, vs);
            else put_mixed(i, ks, vs);
            if (!is_v) {
                sm_ks[(i & 7) * 128 + r] = ks * p.scale_log2;
                sm_vm[(i & 7) * 128 + r] = vs * pow2f(-scale_exponent(vs));
            }
            if (bad) s_bad = 1;
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(is_v ? &bar_v[first] : &bar_k[first]);
            fetch(i + 2);
            fetch_page(i + 4);
        }
    } else {
        // ------------------------------------------------ softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kRegsSoftmax));
        const int row = tid & 127;  // this thread's row, of both streams
        const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const bool busy = (warp & 3) * 32 < live;
        const int tok = sm_tok[row];
        if (nt > 0) {
            for (int x = tid; x < 128 * (D / 8); x += 256) {
                const int r = x / (D / 8), d = (x - r * (D / 8)) * 8;
                uint32_t y[4] = {0u, 0u, 0u, 0u};
                if (r < live) {
                    const int t = sm_tok[r], hh = sm_off[r] - t * p.Hkv * p.G;
                    ldg_halves8(p.q + b * p.q_sb + t * p.q_st + hh * p.q_sh + d, y);
                }
                put_halves8<KV4>(smb + C::kQ, 16384, r, d, y);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar_q);
        }
        float nm = -kUnset, l = 0.0f;  // minus the reference, sum
        const uint32_t to = tm_o + role * D + lane_off;
        int sb = role, round = 0;
#pragma unroll 1
        for (int i = role; i < nt && busy; i += 2) {
            const uint32_t ts = tmem + sb * 128 + lane_off;
            const float* ks_at = sm_ks + (i & 7) * 128;
            const float* vm_at = sm_vm + (i & 7) * 128;
            const bool some_hidden = !full(i);
            // the keys of the tile that this row sees
            uint32_t bits[4];
            if (some_hidden) {
                const int t = j0 + i;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    int cnt;  // keys from the 32's first on
                    uint32_t b32 = 0xFFFFFFFFu;
                    if (t < nct) {
                        cnt = n - t * kTilesKeys - 32 * c;
                    } else {
                        const int u = (t - nct) * kTilesKeys + 32 * c;
                        cnt = tmax - u;
                        if (p.mask == nullptr) cnt = min(cnt, tok + 1 - u);
                        else if (cnt > 0 && row < live) b32 = mask_bits(p, b, tok, u, cnt);
                    }
                    bits[c] = cnt <= 0 ? 0u : (cnt >= 32 ? b32 : b32 & ((1u << cnt) - 1u));
                }
            }
            // the factors of keys e .. e + 3 of 32, as pairs
            auto pairs = [&](const float* at, int e) -> ulonglong2 {
                if constexpr (UNI) {
                    const float f = at[e & 16];
                    return make_ulonglong2(f2_pack(f, f), f2_pack(f, f));
                } else {
                    return *reinterpret_cast<const ulonglong2*>(at + e);
                }
            };
            // scores of 32 keys less the row's reference, and their maximum
            auto front = [&](int c, float (&x)[32], float less) -> float {
                const uint64_t nm2 = f2_pack(less, less);
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                    const ulonglong2 k2 = pairs(ks_at + 32 * c, e);
                    f2_unpack(f2_fma(f2_pack(x[e], x[e + 1]), k2.x, nm2), x[e], x[e + 1]);
                    f2_unpack(f2_fma(f2_pack(x[e + 2], x[e + 3]), k2.y, nm2), x[e + 2], x[e + 3]);
                }
                if (some_hidden) {
                    const uint32_t seen = c == 0 ? bits[0] : (c == 1 ? bits[1] : (c == 2 ? bits[2] : bits[3]));
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (!(seen >> e & 1u)) x[e] = -INFINITY;
                }
                float mx[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    mx[q] = fmaxf(x[8 * q], x[8 * q + 1]);
#pragma unroll
                    for (int e = 2; e < 8; e += 2) mx[q] = fmaxf(fmaxf(mx[q], x[8 * q + e]), x[8 * q + e + 1]);
                }
                return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
            };
            // some row's scores outgrew its reference (or it had none): the largest
            // score of the tile's keys from chunk c on becomes the reference, and
            // what is in terms of the old one is rescaled
            auto move_reference = [&](int c, float (&x)[32], float (&y)[32], float mx) {
                float top = -INFINITY;
                tmem_wait_st();  // the tile's probabilities so far are read back below
#pragma unroll 1
                for (int k = 2; k >= c; k -= 2) {  // chunks c, c + 1 last: they stay in x, y
                    tmem_ld2(ts + 32 * k, x, y);
                    top = fmaxf(top, front(k, x, 0.0f));
                    top = fmaxf(top, front(k + 1, y, 0.0f));
                }
                float f = 1.0f;
                if (mx > kRefresh) {
                    top = floorf(top - kBelow);  // whole: the factor between two is exact in fp16
                    f = ex2(-nm - top);  // 0 from an unset reference
                    nm = -top;
                }
#pragma unroll
                for (int e = 0; e < 32; ++e) x[e] += nm, y[e] += nm;
                l *= f;
                if (i >= 2) {
                    wait(&bar_o[role], ((i - 2) >> 1) & 1);
                    tcgen05_fence_after();
#pragma unroll 1
                    for (int e = 0; e < D; e += 16) {
                        float o[16];
                        tmem_ld(to + e, o);
                        uint32_t w[16];
#pragma unroll
                        for (int q = 0; q < 16; ++q) w[q] = __float_as_uint(o[q] * f);
                        tmem_st(to + e, w);
                    }
                }
                const uint32_t f2 = half_bits(f) * 0x10001u;
#pragma unroll 1
                for (int e = 0; e < 16 * c; e += 16) {
                    float o[16];
                    tmem_ld(ts + e, o);
                    uint32_t w[16];
#pragma unroll
                    for (int q = 0; q < 16; ++q) w[q] = hfma2_u32(__float_as_uint(o[q]), f2, 0x80008000u);
                    tmem_st(ts + e, w);
                }
                tmem_wait_st();
            };
            // probabilities of elements e0 .. e0 + 15: fp32 sum, fp16 (with the V
            // scale's mantissa) for the product
            uint64_t s2 = 0ull;
            auto back = [&](int c, float (&x)[32], uint32_t (&w)[16], int e0) {
#pragma unroll
                for (int e = e0; e < e0 + 16; e += 4) {
                    const ulonglong2 v2 = pairs(vm_at + 32 * c, e);
                    const uint64_t p0 = f2_pack(ex2(x[e]), ex2(x[e + 1])), p1 = f2_pack(ex2(x[e + 2]), ex2(x[e + 3]));
                    s2 = f2_add(s2, f2_add(p0, p1));
                    float a, bb;
                    f2_unpack(f2_mul(p0, v2.x), a, bb);
                    w[e / 2] = pack_half2(a, bb);
                    f2_unpack(f2_mul(p1, v2.y), a, bb);
                    w[e / 2 + 1] = pack_half2(a, bb);
                }
            };
            auto add_sum = [&]() {
                float a, bb;
                f2_unpack(s2, a, bb);
                l += a + bb;
                s2 = 0ull;
            };
            wait(&bar_s[sb], round & 1);
            tcgen05_fence_after();
            // rolled: the body is a few thousand bytes of code, and the roles share
            // the instruction cache
#pragma unroll 1
            for (int c = 0; c < 4; c += 2) {
                float x[32], y[32];
                uint32_t w[16];
                tmem_ld2(ts + 32 * c, x, y);
                const float mx = front(c, x, nm), my = front(c + 1, y, nm);
                if (__any_sync(0xffffffffu, fmaxf(mx, my) > kSlack)) move_reference(c, x, y, fmaxf(mx, my));
                back(c, x, w, 0);
                back(c, x, w, 16);
                tmem_st(ts + 16 * c, w);
                back(c + 1, y, w, 0);
                back(c + 1, y, w, 16);
                tmem_st(ts + 16 * c + 16, w);
                add_sum();
            }
            tmem_wait_st();
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar_p[sb]);
            sb += 2;
            if (sb >= NB) sb -= NB, ++round;
        }
        // ---- join the streams: each warpgroup finishes half of the head dimension of
        // all rows, and passes the other half of its output to the other one through
        // shared memory (K's slots: every product is over)
        constexpr int H = D / 2;
        if (nt > 0) {
            wait(&bar_end, 0);
            tcgen05_fence_after();
        }
        const bool has = nt > role;  // this stream had a tile
        float* sm_o = reinterpret_cast<float*>(sm + C::kK);
        // 16-byte chunks of a row in an order of its own, against bank conflicts
        auto at = [&](int half, int e) { return sm_o + (half * 128 + row) * H + (((e >> 2) ^ (row & 7)) << 2); };
        if (busy) {
#pragma unroll 1
            for (int e0 = 0; e0 < H; e0 += 32) {
                float o[32];
                if (has) tmem_ld(to + (1 - role) * H + e0, o);
#pragma unroll
                for (int e = 0; e < 32; e += 4)
                    *reinterpret_cast<float4*>(at(1 - role, e0 + e)) =
                        has ? make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
            sm_ml[role * 128 + row] = make_float2(nm == -kUnset ? -INFINITY : -nm, l);
        }
        named_barrier_sync(1, 256);
        if (busy) {
            const float2 me = sm_ml[role * 128 + row], it = sm_ml[(1 - role) * 128 + row];
            const float m = fmaxf(me.x, it.x);
            // NaN sums carry a row's NaN through; a stream that saw nothing weighs nothing
            float f0 = me.x == -INFINITY ? 0.0f : ex2(me.x - m), f1 = it.x == -INFINITY ? 0.0f : ex2(it.x - m);
            const float ls = role == 0 ? f0 * me.y + f1 * it.y : f1 * it.y + f0 * me.y;
            if (pslot < 0) {
                const float inv = ls > 0.0f || isnan(ls) ? 1.0f / ls : 0.0f;
                f0 *= inv;
                f1 *= inv;
            } else if (role == 0 && row < live) {
                const int64_t slot = (static_cast<int64_t>(pslot) * p.Hkv + h) * p.BM + row;
                *reinterpret_cast<float2*>(p.part_ml + slot * 2) = make_float2(m, ls);
            }
            const bool fix = *(volatile int*)&s_bad != 0;
            const int d0 = role * H;
            __half* out = p.out + (static_cast<int64_t>(b) * p.T * p.Hkv * p.G + sm_off[row]) * D + d0;
            float* part = p.part_o + ((static_cast<int64_t>(pslot) * p.Hkv + h) * p.BM + row) * D + d0;
#pragma unroll 1
            for (int e0 = 0; e0 < H; e0 += 32) {
                float o[32];
                if (has) tmem_ld(to + d0 + e0, o);
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                    const float4 a = *reinterpret_cast<const float4*>(at(role, e0 + e));
                    const float4 c = *reinterpret_cast<const float4*>(at(role, e0 + e + 4));
                    const float z[8] = {a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
                    float y[8];  // positions back to values
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        const int v = KV4 ? ((q & 1) << 2) | (q >> 1) : (q & 4) | ((q & 1) << 1) | ((q >> 1) & 1);
                        y[v] = (has ? f0 * o[e + q] : 0.0f) + f1 * z[q];
                    }
                    if (row >= live) continue;
                    if (fix) {
                        for (int q = 0; q < 8; ++q)
                            y[q] += nonfinite_sum(p, b, h, D, tok, d0 + e0 + e + q, max(whole, j0 * kTilesKeys),
                                                  min(n, (j0 + nt) * kTilesKeys), max(0, (j0 - nct) * kTilesKeys),
                                                  min(tmax, (j0 + nt - nct) * kTilesKeys));
                    }
                    if (pslot < 0) {
                        *reinterpret_cast<uint4*>(out + e0 + e) =
                            make_uint4(pack_half2(y[0], y[1]), pack_half2(y[2], y[3]), pack_half2(y[4], y[5]),
                                       pack_half2(y[6], y[7]));
                    } else {
                        *reinterpret_cast<float4*>(part + e0 + e) = make_float4(y[0], y[1], y[2], y[3]);
                        *reinterpret_cast<float4*>(part + e0 + e + 4) = make_float4(y[4], y[5], y[6], y[7]);
                    }
                }
            }
        }
        tcgen05_fence_before();
    }
    __syncthreads();
    if (warp == 0) {
        tcgen05_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <bool KV4, int D>
void launch_tree_tiles(const TreeParams& p, const TreeGeom& g, cudaStream_t stream) {
    using C = TilesCfg<KV4, D>;
    auto kern = p.P % 16 == 0 && !p.scale_th ? tree_tiles_kernel<KV4, D, true> : tree_tiles_kernel<KV4, D, false>;
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(g.max_items * p.Hkv));
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = C::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kern, p);
}

}  // namespace mg
