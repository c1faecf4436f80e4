// Attention over a paged cache for many query rows to a key/value head (prompt
// chunks, drafted trees): tcgen05 matrix instructions, 16-bit activations.
//
// A CTA holds one or two groups of 128 query rows and walks the keys in tiles:
// S = Q K^T into TMEM, the group's 128 threads (one row each, no shuffles)
// turn S into P = 2^(S c - m c) and write it over S as 16-bit values, and O +=
// P V takes P from TMEM.  While one group's threads work, the tensor cores
// have the other group's products: a round of both groups is 4 products of
// 128 x 128 x 128 and 32768 exponentials, about 2048 cycles of either unit.
//
//  warps 0-3, 4-7   rows: softmax, rescaling, epilogue, loading of Q
//  the next warp    issues the matrix instructions (one lane)
//  the one after    looks the pages up and copies tiles of keys and values
//                   (TMA, one box to a page) into a ring of slots
//
// The running maximum m only follows a row's true maximum when that passes it
// by 2^8, so O is rarely rescaled; P stays below 2^8 and the sums are fp32.
// P V is complete when S of the next tile is (matrix instructions complete in
// order), so whoever sees S may touch O.  P is rounded to the cache's type, at
// most half a step of each probability: the same size as the rounding of the
// 16-bit output (errors against 64 bits are up to 1.4 times that rounding's
// alone; a caller who wants them smaller passes fp32 queries, which the
// warp-level kernel takes).  fp16 has few steps below 1, so its P (and the sums
// with it) are scaled by 2^7, to at most 2^15: a probability is a normal number
// down to 2^-21 of 2^m, and below that off by at most 2^-32 of it.
//
// 4 chunks of 1025 to 2048 tokens after up to 4096, 28 heads of 128: 367 us in
// turn with other work, 0.90 PFLOP/s, and 328 replayed by itself.  What bounds it
// is each group's own chain: a tile's softmax takes its threads about 2000 cycles
// and the tensor cores 1024 for its two products, and the two groups of an SM
// cover for one another only in part; then the join of split items, 8 to 20 us.
// (Half a tile at a time, with the other half's products under way: 521 us; two
// threads to a row: slower; the groups sharing the rows and splitting the keys:
// 391.)
#pragma once
#include <algorithm>

#include "hq4_host.cuh"
#include "hq4_paged_attn.cuh"
#include "hq4_tc.cuh"
#include "hq4_tmap.cuh"

namespace hq4 {

// Of 8 pairs of exponentials, those by polynomial (4 prompt chunks of 1025
// to 2048 tokens after up to 4096: none 328 us, one 322, two 328).
constexpr int kPtSeries = 1;
constexpr uint64_t kPtWaitNs = 1000000000ull;  // 1 s: a correct kernel never waits this long

template <int kDim>
struct PtShape {
    static constexpr int kGroups = kDim <= 128 ? 2 : 1;   // of 128 rows
    static constexpr int kRows = 128 * kGroups;
    static constexpr int kKeys = kDim <= 128 ? 128 : 64;  // of a tile
    static constexpr int kBlocks = kDim / 64;             // 128-byte blocks of a row
    static constexpr int kQBytes = 128 * kDim * 2;        // of a group
    static constexpr int kSlot = kKeys * kDim * 2;        // a tile of keys or of values
    static constexpr int kSlots = kDim == 64 ? 8 : 5;
    // Two groups: whole warpgroups, which share out the registers: at launch 168 a thread, of which
    // the third keeps 88 and the two of the rows take 208 (168 x 3 = 88 + 208 x 2).
    static constexpr int kThreads = kGroups == 2 ? 384 : 192;
    static constexpr int kSmem = kGroups * kQBytes + kSlots * kSlot + 1024;
    static constexpr int kOCol = kGroups * kKeys;         // TMEM column of the first group's O
};

// D[tmem] (+)= A . B^T, 16-bit operands, fp32 accumulator; A in shared memory or
// in TMEM.
__device__ __forceinline__ void pt_mma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void pt_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Descriptor of a tile whose rows are the contraction's (values: keys x dims,
// dims contiguous): 64 dims to a 128-byte row, 8-row atoms of 1024 bytes, the
// next 64 dims `block` bytes on.
__device__ __forceinline__ uint64_t sw128_mn_desc(uint32_t smem_addr, uint32_t block) {
    const uint32_t lo = ((smem_addr & 0x3FFFFu) >> 4) | ((block >> 4) << 16);
    const uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
    return ((uint64_t)hi << 32) | lo;
}
__device__ __forceinline__ bool pt_elect() {  // one lane of the converged warp, always the same
    uint32_t on;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(on));
    return on != 0;
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* tm, int x, int y, int z, int w,
                                            uint32_t bar, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
        " [%0], [%1, {%2, %3, %4, %5}], [%6], %7;" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(tm)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar), "l"(policy)
        : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]),
                 "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
__device__ __forceinline__ float pt_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two fp32 values to an instruction.
typedef unsigned long long u64;
__device__ __forceinline__ u64 pair(float a, float b) {
    u64 d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ u64 pair(uint32_t a, uint32_t b) {
    u64 d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ float2 unpair(u64 v) {
    float2 d;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(v));
    return d;
}
__device__ __forceinline__ u64 fma2(u64 a, u64 b, u64 c) {
    u64 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ u64 add2(u64 a, u64 b) {
    u64 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ u64 mul2(u64 a, u64 b) {
    u64 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN where either is (fmaxf drops it)
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ u64 pt_ex2_both(u64 z) {
    const float2 f = unpair(z);
    return pair(pt_ex2(f.x), pt_ex2(f.y));
}
// 2^z, z <= 64, for two values on the multiply-add units: adding 1.5 * 2^23
// rounds z to an integer n and leaves it in the low bits, 2^f for the rest f in
// [-1/2, 1/2] is a polynomial (least relative error, fitted for this: 7.5e-5 for
// bf16 probabilities, whose half step is 2e-3, 2.6e-6 for fp16 ones), and the
// factor 2^n is built from its bits: 0 for n = -127, which is what -inf gives.
// NaN stays NaN (the polynomial's; a NaN or infinite key that a row sees).
template <class C>
__device__ __forceinline__ u64 pt_ex2_series(u64 z) {
    const u64 magic = pair(12582912.0f, 12582912.0f), back = pair(-12582912.0f, -12582912.0f);
    float2 v = unpair(z);
    z = pair(max_nan(v.x, -127.0f), max_nan(v.y, -127.0f));
    const u64 r = add2(z, magic);
    const u64 f = fma2(add2(r, back), pair(-1.0f, -1.0f), z);
    u64 s;
    if constexpr (Elem<C>::code == HQ4_F16) {
        s = fma2(f, pair(9.570101652e-3f, 9.570101652e-3f), pair(5.591786210e-2f, 5.591786210e-2f));
        s = fma2(s, f, pair(0.2402474485f, 0.2402474485f));
        s = fma2(s, f, pair(0.6931218145f, 0.6931218145f));
        s = fma2(s, f, pair(0.9999992614f, 0.9999992614f));
    } else {
        s = fma2(f, pair(5.517166681e-2f, 5.517166681e-2f), pair(0.2426111351f, 0.2426111351f));
        s = fma2(s, f, pair(0.6932609870f, 0.6932609870f));
        s = fma2(s, f, pair(0.9999280728f, 0.9999280728f));
    }
    v = unpair(r);
    return mul2(s, pair((__float_as_uint(v.x) << 23) + 0x3f800000u, (__float_as_uint(v.y) << 23) + 0x3f800000u));
}

// Which of the 32 entries from e0 on token tok of the item sees, a bit each.
__device__ __forceinline__ uint32_t paged_sees32(const PagedAttnParams& p, const PagedItem& it, int tok, int e0) {
    const int j0 = e0 - it.len;
    if (!p.tree_mask) {
        const int n = tok + 1 - j0;
        return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
    }
    const uint32_t* row = p.tree_mask + (size_t)(it.row0 + tok) * p.mask_words;
    auto word = [&](int w) -> uint32_t {
        if (w < 0) return 0xffffffffu;  // entries before the tree
        const int n = it.n_tok - w * 32;
        if (w >= p.mask_words || n <= 0) return 0u;
        return __ldg(row + w) & (n >= 32 ? 0xffffffffu : (1u << n) - 1u);
    };
    const int w = j0 >> 5;
    return __funnelshift_r(word(w), word(w + 1), j0 & 31);
}

template <class C, int kDim>
__global__ void __launch_bounds__(PtShape<kDim>::kThreads, 1)
    paged_tc_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                    const __grid_constant__ PagedAttnParams p) {
    using S = PtShape<kDim>;
    constexpr int kKeys = S::kKeys, kGroups = S::kGroups, kRows = S::kRows;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ PagedScan scan;
    __shared__ __align__(8) uint64_t bars[2 * S::kSlots + 4 * kGroups + 1];
    __shared__ uint32_t s_valid[8][kKeys / 32];
    __shared__ uint32_t s_tmem;
    __shared__ volatile int s_dead;
    __shared__ PagedItem s_items[4 * kGroups + 2][2];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    unsigned char* sm = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t ring = base + kGroups * S::kQBytes;
    const uint32_t bar0 = smem_u32(bars);
    auto full_bar = [&](int s) { return bar0 + 8u * s; };
    auto empty_bar = [&](int s) { return bar0 + 8u * (S::kSlots + s); };
    auto q_bar = [&](int g) { return bar0 + 8u * (2 * S::kSlots + g); };
    auto s_bar = [&](int g) { return bar0 + 8u * (2 * S::kSlots + kGroups + g); };
    auto p_bar = [&](int g) { return bar0 + 8u * (2 * S::kSlots + 2 * kGroups + g); };
    auto o_bar = [&](int g) { return bar0 + 8u * (2 * S::kSlots + 3 * kGroups + g); };
    const uint32_t end_bar = bar0 + 8u * (2 * S::kSlots + 4 * kGroups);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kSlots; s++) {
            mbar_init_nofence(full_bar(s), 1);
            mbar_init_nofence(empty_bar(s), 1);
        }
        for (int g = 0; g < kGroups; g++) {
            mbar_init_nofence(q_bar(g), 4);  // a warp each
            mbar_init_nofence(s_bar(g), 1);
            mbar_init_nofence(p_bar(g), 4);
            mbar_init_nofence(o_bar(g), 1);
        }
        mbar_init_nofence(end_bar, 1);
        mbar_init_fence();
        s_dead = 0;
    }
    if (warp == 4 * kGroups) {
        tmem_alloc(smem_u32(&s_tmem), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    pdl_wait();

    // each warp walks the part's items by itself; its item lies in shared memory, not in registers
    const PagedItem* it = &s_items[min(warp, 4 * kGroups + 1)][0];  // the item at hand; the other place takes the next one
    int left;   // units of the part that are still to do
    int from;   // the first of them within the item
    bool busy;
    const PagedWs<kRows, kDim> ws(p.ws, gridDim.x);
    {
        long long pos, end;
        const PagedStart begin = paged_part<kRows, kKeys, S::kThreads>(p, scan, pos, end);
        busy = pos < end;
        if (p.ws && threadIdx.x == 0 && (busy || blockIdx.x == 0)) ws.info[blockIdx.x] = begin;
        left = (int)(end - pos);
        from = (int)(pos - begin.first);
        if (lane == 0 && warp < 4 * kGroups + 2) s_items[warp][0] = begin.it;
        __syncwarp();
    }
    pdl_launch_dependents();
    const int D = p.head_dim, ksteps = D >> 4;
    bool fail = false;
    // A warp's wait, which ends: after so many tries (each may sleep up to a millisecond; reading a
    // timer instead costs more than most waits), or once another warp's has run out.
    auto wait = [&](uint32_t bar, uint32_t parity) -> bool {
        for (int i = 0; i < 10; i++) {
            const bool ok = mbar_wait_tries(bar, parity & 1u, 1000000u, 1000);
            if (__all_sync(0xffffffffu, ok)) return true;
            if (__any_sync(0xffffffffu, s_dead)) break;
        }
        s_dead = 1;
        fail = true;
        return false;
    };
    // The key tiles of the part's piece of the item, and the units that it takes; then the next item.
    auto piece = [&](int& t0, int& t1) -> int {
        const int units = min(left, it->weight - from);
        t0 = p.split ? paged_tiles_before(p, from) : 0;
        t1 = p.split ? paged_tiles_before(p, from + units) : it->tiles;
        return units;
    };
    auto next = [&](int units) {
        left -= units;
        from = 0;
        if (left > 0) {
            PagedItem* n = it == &s_items[warp][0] ? &s_items[warp][1] : &s_items[warp][0];
            __syncwarp();
            if (lane == 0) {
                PagedItem i = *it;
                paged_next<kRows, kKeys>(p, i);
                *n = i;
            }
            __syncwarp();
            it = n;
        }
    };
    auto groups_of = [&]() { return it->n_tok * p.group - it->rt * kRows > 128 ? kGroups : 1; };

    if (busy && warp < 4 * kGroups) {
        // ---- rows ------------------------------------------------------------------
        if constexpr (kGroups == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int g = warp >> 2;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_col = tmem + lanes + g * kKeys, o_col = tmem + lanes + S::kOCol + g * kDim;
        const int in_group = (warp & 3) * 32 + lane;
        auto load_q = [&]() {  // the group's rows of item `it`, a warp its own 32, all copies in flight at once
            const int row = it->rt * kRows + g * 128 + in_group;
            const bool there = row < it->n_tok * p.group;
            const C* src = static_cast<const C*>(p.q);
            if (there)
                src += (long long)(it->row0 + row / p.group) * p.q_stride + ((long long)it->h * p.group + row % p.group) * D;
            const uint32_t q0 = base + g * S::kQBytes;
            constexpr int kChunks = kDim / 8;  // of 16 bytes
#pragma unroll
            for (int i = 0; i < kChunks; i++) {
                const int r = (lane + 32 * i) / kChunks, c = (lane + 32 * i) % kChunks, gr = (warp & 3) * 32 + r;
                const C* from = reinterpret_cast<const C*>(__shfl_sync(0xffffffffu, (u64)src, r));
                const int ok = __shfl_sync(0xffffffffu, (int)there, r);
                if (c * 8 < D) cp_async16(q0 + (c >> 3) * (128 * 128) + sw128_off(gr, c & 7), from + c * 8, ok);
            }
            cp_async_commit();
            cp_async_wait<0>();
            if (p.scale_log2 < 0.0f) {  // a negative scale: the rows' signs instead
#pragma unroll 1
                for (int i = 0; i < kChunks; i++) {
                    const int r = (lane + 32 * i) / kChunks, c = (lane + 32 * i) % kChunks, gr = (warp & 3) * 32 + r;
                    uint4* v = reinterpret_cast<uint4*>(sm + g * S::kQBytes + (c >> 3) * (128 * 128) + sw128_off(gr, c & 7));
                    if (c * 8 < D) *v = make_uint4(v->x ^ 0x80008000u, v->y ^ 0x80008000u, v->z ^ 0x80008000u, v->w ^ 0x80008000u);
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_bar(g));
        };
        uint32_t n_s = 0, n_o = 0, tile_no = 0;  // tiles of this group, pieces of it, tiles of the CTA so far
        if (g < groups_of()) load_q();
        int pieces = 0;
        while (left > 0 && !fail) {
            int t0, t1;
            const int units = piece(t0, t1);
            if (t1 == 0) break;  // the part ends before the item's first tile
            const bool whole = t0 == 0 && t1 == it->tiles;
            const bool in = g < groups_of();
            const int row = it->rt * kRows + g * 128 + in_group, rows = it->n_tok * p.group;
            const bool on = in && row < rows;
            const bool warp_on = in && it->rt * kRows + g * 128 + (warp & 3) * 32 < rows;
            const int tok = on ? row / p.group : 0;
            float m = -INFINITY, l = 0.0f;  // of scaled scores (log2), and the row's sum
            uint32_t any = 0;               // an entry has a page
            const int t_plain = (it->len + (p.tree_mask ? 0 : it->rt * kRows / p.group + 1)) / kKeys;  // before: all seen
            const float c2 = fmaxf(fabsf(p.scale_log2), 1e-30f);  // not 0: masked scores stay -inf
            if (in) {
                for (int t = t0; t < t1; t++, n_s++) {
                    if (!wait(s_bar(g), n_s)) break;
                    __syncwarp();
                    tc_fence_after();
                    if (warp_on) {
                        constexpr int kParts = kKeys / 32;
                        uint32_t s[kParts][32];
#pragma unroll
                        for (int i = 0; i < kParts; i++) tmem_ld32(s_col + i * 32, s[i]);
                        tmem_wait_ld();
                        const uint32_t* valid = s_valid[(tile_no + (t - t0)) & 7];
                        bool plain = t < t_plain;
#pragma unroll
                        for (int i = 0; i < kParts; i++) plain = plain && valid[i] == 0xffffffffu;
                        if (__all_sync(0xffffffffu, plain)) {
                            any = 1;
                        } else {
#pragma unroll
                            for (int i = 0; i < kParts; i++) {
                                any |= valid[i];
                                const uint32_t see = on ? valid[i] & paged_sees32(p, *it, tok, t * kKeys + i * 32) : 0u;
#pragma unroll
                                for (int j = 0; j < 32; j++)
                                    if (!(see >> j & 1)) s[i][j] = 0xff800000u;  // -inf
                            }
                        }
                        float top[kParts];
#pragma unroll
                        for (int i = 0; i < kParts; i++) {
                            top[i] = fmaxf(__uint_as_float(s[i][0]), __uint_as_float(s[i][1]));
#pragma unroll
                            for (int j = 2; j < 32; j += 2)
                                top[i] = max3(top[i], __uint_as_float(s[i][j]), __uint_as_float(s[i][j + 1]));
                        }
#pragma unroll
                        for (int i = 1; i < kParts; i++) top[0] = fmaxf(top[0], top[i]);
                        const float x = top[0] * c2;
                        // m follows when it is 2^8 behind (or has seen nothing yet)
                        const bool move = x > m + 8.0f;
                        if (__any_sync(0xffffffffu, move)) {
                            const float m1 = move ? x : m;
                            const float keep = move ? pt_ex2(m - m1) : 1.0f;  // 0 from -inf
                            l *= keep;
                            m = m1;
                            if (t > t0) {
#pragma unroll 1
                                for (int c = 0; c < D; c += 8) {
                                    uint32_t o[8];
                                    tmem_ld8(o_col + c, o);
                                    tmem_wait_ld();
#pragma unroll
                                    for (int j = 0; j < 8; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * keep);
                                    tmem_st8(o_col + c, o);
                                }
                            }
                        }
                        const float mu = m == -INFINITY ? 0.0f : m;
                        constexpr float kUp = Elem<C>::code == HQ4_F16 ? 7.0f : 0.0f;
                        const u64 cc = pair(c2, c2), mm = pair(kUp - mu, kUp - mu);
                        u64 add[2] = {0, 0};
#pragma unroll
                        for (int i = 0; i < kParts; i++) {
                            uint32_t w[16];
#pragma unroll
                            for (int j = 0; j < 16; j++) {
                                const u64 z = fma2(pair(s[i][2 * j], s[i][2 * j + 1]), cc, mm);
                                const u64 e = j % 8 < kPtSeries ? pt_ex2_series<C>(z) : pt_ex2_both(z);
                                add[j & 1] = add2(add[j & 1], e);
                                const float2 f = unpair(e);
                                w[j] = pack2<C>(f.x, f.y);
                            }
                            tmem_st16(s_col + i * 16, w);  // over scores that are in registers
                        }
                        const float2 sum = unpair(add2(add[0], add[1]));
                        l += sum.x + sum.y;
                        tmem_wait_st();
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(p_bar(g));
                }
            }
            tile_no += t1 - t0;
            // ---- the next item's rows (S of the last tile is done: Q is free), then this one's output ----
            if (fail) break;
            const PagedItem* const mine = it;
            const int piece_no = 2 * blockIdx.x + (pieces++ ? 1 : 0);
            next(units);
            if (left > 0 && g < groups_of()) load_q();
            if (!in) continue;
            if (!wait(o_bar(g), n_o)) break;
            n_o++;
            __syncwarp();
            tc_fence_after();
            if (warp_on) {
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                const int r = g * 128 + in_group;
                C* out = static_cast<C*>(p.out) +
                         ((long long)(mine->row0 + tok) * p.n_heads + mine->h * p.group + row % p.group) * D;
                const size_t at = (size_t)piece_no * kRows + r;
                bool bad = on && whole && l == 0.0f && any;
                for (int c = 0; c < D; c += 32) {
                    uint32_t o[32];
                    tmem_ld32(o_col + c, o);
                    tmem_wait_ld();
                    if (on && whole) {
                        float y[32];
#pragma unroll
                        for (int j = 0; j < 32; j++) {
                            y[j] = l == 0.0f ? 0.0f : __uint_as_float(o[j]) * inv;
                            bad |= y[j] != y[j];
                        }
#pragma unroll
                        for (int j = 0; j < 4; j++) store8(out + c + 8 * j, *reinterpret_cast<float(*)[8]>(&y[8 * j]));
                    } else if (on) {
                        uint4* d = reinterpret_cast<uint4*>(ws.o + at * kDim + c);
#pragma unroll
                        for (int j = 0; j < 8; j++) d[j] = make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
                    }
                    __syncwarp();
                }
                if (on && !whole) ws.ml[at] = make_float2(m, l == 0.0f && any ? 1.0f : l);
                uint32_t again = __ballot_sync(0xffffffffu, bad);
                while (again) {
                    const int i = __ffs(again) - 1;
                    again &= again - 1;
                    paged_slow_row<C, C>(p, *mine, __shfl_sync(0xffffffffu, row, i));
                }
            }
            tc_fence_before();
        }
    } else if (busy) {
        // (one instruction for all warps of the warpgroup)
        if constexpr (kGroups == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == 4 * kGroups) {
            // ---- matrix instructions -------------------------------------------------------
            constexpr uint32_t kType = Elem<C>::code == HQ4_BF16 ? 1u : 0u;
            const uint32_t id_s = (1u << 4) | (kType << 7) | (kType << 10) | ((uint32_t)(kKeys >> 3) << 17) | (8u << 24);
            const uint32_t id_o = (1u << 4) | (kType << 7) | (kType << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | (8u << 24);
            uint32_t n_slot = 0, n_q[kGroups], n_p[kGroups];
            for (int g = 0; g < kGroups; g++) n_q[g] = n_p[g] = 0;
            auto slot_at = [&](uint32_t n) { return ring + (n % S::kSlots) * S::kSlot; };
            auto full = [&](uint32_t n) { return wait(full_bar(n % S::kSlots), n / S::kSlots); };
            auto scores = [&](int g, uint32_t slot) {
                const uint64_t a = sw128_desc(base + g * S::kQBytes), b = sw128_desc(slot);
                const uint32_t d = tmem + g * kKeys;
                if (pt_elect()) {
#pragma unroll
                    for (int k = 0; k < kDim / 16; k++) {
                        if (k >= ksteps) break;
                        // 16 dims: 32 bytes on within a 128-byte row, then the next block of 64 dims
                        pt_mma_ss(d, a + ((k >> 2) * (128 * 128 / 16) + 2 * (k & 3)),
                                  b + ((k >> 2) * (kKeys * 128 / 16) + 2 * (k & 3)), id_s, k ? 1u : 0u);
                    }
                    umma_commit(s_bar(g));
                }
                __syncwarp();
            };
            while (left > 0 && !fail) {
                int t0, t1;
                const int units = piece(t0, t1);
                if (t1 == 0) break;  // the part ends before the item's first tile
                const int ng = groups_of();
                if (!full(n_slot)) break;
                for (int g = 0; g < ng && !fail; g++) {
                    if (!wait(q_bar(g), n_q[g])) break;
                    n_q[g]++;
                    tc_fence_after();
                    scores(g, slot_at(n_slot));
                }
                if (fail) break;
                if (pt_elect()) umma_commit(empty_bar(n_slot % S::kSlots));
                __syncwarp();
                for (int t = t0; t < t1 && !fail; t++) {
                    const uint32_t nv = n_slot + 1, nk = n_slot + 2;  // this tile's values, the next one's keys
                    const bool more = t + 1 < t1;
                    if (!full(nv)) break;
                    const int past = it->keys - t * kKeys;  // values that no row sees may be anything: zeros instead
                    if (past < kKeys) {
                        for (int i = lane; i < (kKeys - max(past, 0)) * (kDim / 8); i += 32) {
                            const int r = max(past, 0) + i / (kDim / 8), c = i % (kDim / 8);
                            *reinterpret_cast<uint4*>(sm + (slot_at(nv) - base) + (c >> 3) * (kKeys * 128) +
                                                      sw128_off(r, c & 7)) = make_uint4(0, 0, 0, 0);
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                    }
                    for (int g = 0; g < ng && !fail; g++) {
                        if (!wait(p_bar(g), n_p[g])) break;
                        n_p[g]++;
                        tc_fence_after();
                        const uint64_t b = sw128_mn_desc(slot_at(nv), kKeys * 128);
                        const uint32_t d = tmem + S::kOCol + g * kDim, a = tmem + g * kKeys;
                        if (pt_elect()) {
#pragma unroll
                            for (int k = 0; k < kKeys / 16; k++)  // 16 keys: 2048 bytes on
                                pt_mma_ts(d, a + 8 * k, b + k * (2048 / 16), id_o, k || t > t0 ? 1u : 0u);
                            if (!more) umma_commit(o_bar(g));
                        }
                        __syncwarp();
                        if (more) {
                            if (g == 0 && !full(nk)) break;
                            tc_fence_after();
                            scores(g, slot_at(nk));
                        }
                    }
                    if (fail) break;
                    if (pt_elect()) {
                        umma_commit(empty_bar(nv % S::kSlots));
                        if (more) umma_commit(empty_bar(nk % S::kSlots));
                    }
                    __syncwarp();
                    n_slot += 2;
                }
                next(units);
            }
            if (pt_elect()) umma_commit(end_bar);
            __syncwarp();
            // all products are done before the memory goes (a limit of its own: the others may have failed)
            mbar_wait_ns(end_bar, 0, kPtWaitNs);
        } else if (warp == 4 * kGroups + 1) {
            // ---- keys and values -------------------------------------------------------------
            const uint64_t policy = l2_policy_evict_last();
            const int box = min(1 << p.b.page_shift, kKeys), boxes = kKeys / box;
            uint32_t n = 0, tile_no = 0;
            while (left > 0 && !fail) {
                int t0, t1;
                const int units = piece(t0, t1);
                if (t1 == 0) break;  // the part ends before the item's first tile
                if (lane == 0 && (it->len < 0 || (long long)it->len + it->n_tok > (long long)p.b.pages_per_seq << p.b.page_shift))
                    atomicOr(p.b.status, kStatusPaged);  // rows whose entries have no place
                for (int t = t0; t < t1 && !fail; t++, tile_no++) {
                    const int e = t * kKeys + lane * box;
                    int page = -1;
                    if (lane < boxes && e < it->keys) {
                        page = find_page(p.b, it->s, e);
                        if (page < 0) atomicOr(p.b.status, kStatusPaged);
                    }
                    const uint32_t ok = __ballot_sync(0xffffffffu, page >= 0);
                    if (lane < kKeys / 32) {
                        uint32_t v = 0;
                        for (int b = 0; b < 32; b += min(box, 32))
                            if (ok >> ((lane * 32 + b) / box) & 1) v |= (box >= 32 ? 0xffffffffu : (1u << box) - 1u) << b;
                        s_valid[tile_no & 7][lane] = v;
                    }
                    __syncwarp();
                    for (int kv = 0; kv < 2; kv++, n++) {
                        const int slot = n % S::kSlots;
                        if (n >= S::kSlots && !wait(empty_bar(slot), n / S::kSlots - 1)) break;
                        if (lane == 0) mbar_arrive_expect_tx(full_bar(slot), S::kSlot);
                        __syncwarp();
                        if (lane < boxes) {
                            // without a page: a place past the last page, which reads as zeros
                            const int y = e & ((1 << p.b.page_shift) - 1), w = page >= 0 ? page : p.b.n_pages;
                            for (int b = 0; b < S::kBlocks; b++)
                                tma_load_4d(ring + slot * S::kSlot + b * (kKeys * 128) + lane * box * 128,
                                            kv ? &tm_v : &tm_k, b * 64, y, it->h, w, full_bar(slot), policy);
                        }
                    }
                }
                next(units);
            }
            // no copy is left behind: each slot's last one has arrived
            for (uint32_t i = n > S::kSlots ? n - S::kSlots : 0; i < n; i++)
                mbar_wait_ns(full_bar(i % S::kSlots), (i / S::kSlots) & 1u, kPtWaitNs);
        }
    }
    if (fail && lane == 0) atomicOr(p.b.status, 1);
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 4 * kGroups) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ---- launch ------------------------------------------------------------------------

// The cache as pages x heads x entries x dims; boxes of 64 dims by min(page, tile) entries.
static inline bool pt_map(CUtensorMap* tm, const void* cache, bool bf16, int head_dim, int page_size, int n_kv,
                          int n_pages, long long page_stride, int box) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[4] = {(cuuint64_t)head_dim, (cuuint64_t)page_size, (cuuint64_t)n_kv, (cuuint64_t)n_pages};
    cuuint64_t strides[3] = {(cuuint64_t)head_dim * 2, (cuuint64_t)page_size * head_dim * 2, (cuuint64_t)page_stride * 2};
    cuuint32_t boxd[4] = {64, (cuuint32_t)box, 1, 1}, estr[4] = {1, 1, 1, 1};
    return fn(tm, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(cache),
              dims, strides, boxd, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class C, int kDim>
static int launch_pt(const PagedAttnParams& p, const PaPlan& pl, cudaStream_t st) {
    using S = PtShape<kDim>;
    auto kern = paged_tc_kernel<C, kDim>;
    static PerDeviceOnce once;
    if (smem_opt_in(once, kern, S::kSmem) != cudaSuccess) return HQ4_ERR_LAUNCH;
    CUtensorMap tk, tv;
    const bool bf16 = Elem<C>::code == HQ4_BF16;
    const int page_size = 1 << p.b.page_shift, box = std::min(page_size, S::kKeys);
    if (!pt_map(&tk, p.k, bf16, p.head_dim, page_size, p.n_kv, p.b.n_pages, p.b.page_stride, box) ||
        !pt_map(&tv, p.v, bf16, p.head_dim, page_size, p.n_kv, p.b.n_pages, p.b.page_stride, box))
        return HQ4_ERR_LAUNCH;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3(pl.ctas);
    lc.blockDim = dim3(S::kThreads);
    lc.dynamicSmemBytes = S::kSmem;
    lc.stream = st;
    lc.attrs = attr;
    lc.numAttrs = 1;
    if (cudaLaunchKernelEx(&lc, kern, tk, tv, p) != cudaSuccess) return HQ4_ERR_LAUNCH;
    if (!p.split || pl.ctas < 2) return HQ4_OK;
    lc.gridDim = dim3(pl.ctas - 1, (pl.join + pl.take - 1) / pl.take);
    lc.blockDim = dim3(kCombineWarps * 32);
    lc.dynamicSmemBytes = 0;
    return cudaLaunchKernelEx(&lc, paged_combine_kernel<C, C, S::kRows, kDim>, p, pl.ctas) == cudaSuccess
               ? HQ4_OK
               : HQ4_ERR_LAUNCH;
}

template <class C>
static int launch_pt_dim(const PagedAttnParams& p, const PaPlan& pl, cudaStream_t st) {
    return pl.dim == 64 ? launch_pt<C, 64>(p, pl, st)
         : pl.dim == 128 ? launch_pt<C, 128>(p, pl, st) : launch_pt<C, 256>(p, pl, st);
}

}  // namespace hq4
