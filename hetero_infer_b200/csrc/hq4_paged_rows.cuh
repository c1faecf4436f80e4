// Attention over a paged cache for few query rows to a key/value head (decode,
// small trees), and for fp32 queries: warp-level matrix instructions.
//
// Decode is bound by the bytes of the cache.  Each warp walks its own tiles of
// 16 keys with a running maximum and sum, from a ring of kStages tiles in
// shared memory that it fills itself with 16-byte asynchronous copies, so
// warps wait for nobody until the CTA's part of an item is done.  Scores are
// computed transposed, S^T = K Q^T: 16 keys are the M of m16n8k16 and 8 rows
// its N, so the 7 or 8 query heads of a key/value head waste nothing, and the
// fragment of S^T turns into the operand of O^T = V^T P^T by transposing 8x8
// blocks between lanes (movmatrix).
//
// fp32 queries against 16-bit entries keep fp32's precision: the entries are
// exact in the matrix instructions, and queries and probabilities are sums of
// 16-bit terms (three bf16 terms hold 24 bits; two fp16 terms of a row scaled
// by a power of two hold 22).
//
// 64 streams of 100 to 8200 entries, 28 heads of 128 over 4: 125 us, 4.9 TB/s;
// the main loop reads at 6.2 to 6.9 TB/s, the rest is starts, ends and the
// join.  One stream of 131072 with fp32 queries: 66 us, of them 45 in the main
// loop.
#pragma once
#include "hq4_host.cuh"
#include "hq4_paged_attn.cuh"

namespace hq4 {

constexpr int kPaKeys = 16;  // keys of a tile

template <int kDim>
struct PaShape {
    static constexpr int kStages = kDim == 64 ? 4 : 3;
    static constexpr int kTile = kPaKeys * kDim * 2;                  // bytes of a tile of keys or of values
    static constexpr int kRing = kStages * 2 * kTile;                 // of a warp
};
// 16-bit terms of a query.
template <class A, class C>
constexpr int pa_terms() { return sizeof(A) == 2 ? 1 : Elem<C>::code == HQ4_BF16 ? 3 : 2; }
// 16-bit terms of a probability.  Of 16-bit calls two, so that the output's own
// rounding is the only one to 16 bits (with one, errors against 64 bits are 1.13
// times as large): 64 streams of 100 to 8200 entries, 28 heads of 128: 131 us
// with one, 135 with two (flushed caches).  Wide heads keep one, which is off by
// at most half a step of each probability: two would cost 279 -> 298 us there.
template <class A, class C, int kDim>
constexpr int pa_p_terms() { return sizeof(A) == 4 ? pa_terms<A, C>() : kDim <= 128 ? 2 : 1; }
template <int kDim, int kRows, int kTerms, int W>
constexpr int pa_smem() { return W * PaShape<kDim>::kRing + kTerms * kRows * kDim * 2; }

__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
    return d;
}
template <class C>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma_f16_16816(c, a[0], a[1], a[2], a[3], b0, b1);
}
template <>
__device__ __forceinline__ void mma16<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma_bf16_16816(c, a[0], a[1], a[2], a[3], b0, b1);
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Byte of the 16-byte chunk c of row r in a tile of rows of kDim 16-bit
// values; the XOR spreads a column of 8 rows over all banks.
template <int kDim>
__device__ __forceinline__ int tile_at(int r, int c) { return r * (kDim * 2) + ((c ^ (r & 7)) << 4); }

// NT: 8-row tiles; W: warps.
template <class A, class C, int kDim, int NT, int W>
__global__ void __launch_bounds__(W * 32) paged_attn_kernel(const __grid_constant__ PagedAttnParams p) {
    constexpr int kRows = 8 * NT, kTerms = pa_terms<A, C>(), kPTerms = pa_p_terms<A, C, kDim>(), kStages = PaShape<kDim>::kStages;
    constexpr int kTile = PaShape<kDim>::kTile, kRing = PaShape<kDim>::kRing;
    constexpr int kChunks = kDim / 8, kOs = kDim + 4;
    static_assert(kRows * kOs * 4 <= kRing, "a warp's outputs fit its ring");
    // where a warp's outputs fit one stage, the next item's first tiles are under way while this one's are joined
    constexpr bool kAhead = kRows * kOs * 4 <= 2 * kTile;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ PagedScan scan;
    __shared__ float s_m[W][kRows], s_l[W][kRows], s_qs[kRows];
    __shared__ int s_os[W];  // where in shared memory each warp has left its outputs
    __shared__ uint32_t s_any[W];  // whether any of its entries had a page
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int D = p.head_dim, ksteps = D >> 4;
    long long pos, end;
    const PagedStart begin = paged_part<kRows, kPaKeys, W * 32>(p, scan, pos, end);
    const PagedWs<kRows, kDim> ws(p.ws, gridDim.x);
    if (p.ws && threadIdx.x == 0 && (pos < end || blockIdx.x == 0)) ws.info[blockIdx.x] = begin;
    if (pos >= end) {
        pdl_launch_dependents();
        return;
    }
    PagedItem it = begin.it;
    int left = (int)(end - pos), from = (int)(pos - begin.first);  // units still to do; the first of them in the item
    int pieces = 0;
    const uint32_t ring_u = smem_u32(smem + warp * kRing);
    unsigned char* qs = smem + W * kRing;
    const uint32_t qs_u = smem_u32(qs);
    const C* kc = static_cast<const C*>(p.k);
    const C* vc = static_cast<const C*>(p.v);
    const int in_page = (1 << p.b.page_shift) - 1;
    int stage = 0;                // of the ring: the next tile's
    unsigned long long oks = 0;   // 16 bits of a tile on its way, the next one lowest: which of its keys have a page

    // Lanes 0-15 (and 16-31 alike) look up where a tile's keys lie: the page, -1 for none.  A step
    // ahead of the copies, so that those do not wait for it.
    auto look_up = [&](const PagedItem& it, int t, int t1) -> int {
        const int e = t * kPaKeys + (lane & 15);
        if (t >= t1 || e >= it.keys) return -1;
        const int page = find_page(p.b, it.s, e);
        if (page < 0 && lane < 16) atomicOr(p.b.status, kStatusPaged);
        return page;
    };
    // Starts tile t of an item's piece that ends before t1 (nothing, beyond that).
    auto load_tile = [&](const PagedItem& it, int t, int t1, int page, int stage) -> uint32_t {
        const uint32_t ok = __ballot_sync(0xffffffffu, page >= 0) & 0xffffu;
        const long long at = page < 0 ? 0
                                      : (long long)page * p.b.page_stride +
                                            (((long long)it.h << p.b.page_shift) + ((t * kPaKeys + (lane & 15)) & in_page)) * D;
        if (t < t1) {
            const uint32_t kd = ring_u + stage * 2 * kTile, vd = kd + kTile;
#pragma unroll
            for (int i = 0; i < kPaKeys * kChunks / 32; i++) {
                const int idx = lane + 32 * i, r = idx / kChunks, c = idx % kChunks;
                const long long src = __shfl_sync(0xffffffffu, at, r) + c * 8;
                const bool on = ok >> r & 1;
                if (c * 8 < D) {  // without a page: zeros, so that what lies there does not reach the products
                    const int d = tile_at<kDim>(r, c);
                    cp_async16(kd + d, kc + (on ? src : 0), on);
                    cp_async16(vd + d, vc + (on ? src : 0), on);
                }
            }
        }
        cp_async_commit();
        return ok;
    };
    int page_next = -1;  // of the first tile that has not been started
    auto begin_item = [&](const PagedItem& it, int t0, int t1) {  // its first tiles
        oks = 0;
        int page[kStages];
#pragma unroll
        for (int s = 0; s < kStages; s++) page[s] = look_up(it, t0 + warp + s * W, t1);
#pragma unroll
        for (int s = 0; s < kStages - 1; s++) {
            const int at = stage + s < kStages ? stage + s : stage + s - kStages;
            oks |= (unsigned long long)load_tile(it, t0 + warp + s * W, t1, page[s], at) << (16 * s);
        }
        page_next = page[kStages - 1];
    };
    auto units_of = [&](const PagedItem& it, int from, int left) { return min(left, it.weight - from); };
    auto t_begin = [&](int from) { return p.split ? paged_tiles_before(p, from) : 0; };
    auto t_end = [&](const PagedItem& it, int from, int units) {
        return p.split ? paged_tiles_before(p, from + units) : it.tiles;
    };
    {
        const int units = units_of(it, from, left);
        begin_item(it, t_begin(from), t_end(it, from, units));
    }

    while (left > 0) {
        const int units = units_of(it, from, left);
        const int t0 = t_begin(from), t1 = t_end(it, from, units);
        if (t1 == 0) break;  // the part ends before the item's first tile
        const bool whole = t0 == 0 && t1 == it.tiles;
        const int rows = min(kRows, it.n_tok * p.group - it.rt * kRows);
        PagedItem nx = it;
        if (units < left) paged_next<kRows, kPaKeys>(p, nx);
        else pdl_launch_dependents();
        if (threadIdx.x == 0 && (it.len < 0 || (long long)it.len + it.n_tok > (long long)p.b.pages_per_seq << p.b.page_shift))
            atomicOr(p.b.status, kStatusPaged);  // rows whose entries have no place

        // ---- the queries, as 16-bit terms ----------------------------------
        for (int r = warp; r < kRows; r += W) {
            const int row = it.rt * kRows + r;
            const bool on = r < rows;
            const A* src = static_cast<const A*>(p.q) + (long long)(it.row0 + (on ? row / p.group : 0)) * p.q_stride +
                           ((long long)it.h * p.group + (on ? row % p.group : 0)) * D;
            if constexpr (kTerms == 1) {
                for (int c = lane; c < kChunks; c += 32) {
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (on && c * 8 < D) v = __ldg(reinterpret_cast<const uint4*>(src + c * 8));
                    *reinterpret_cast<uint4*>(qs + tile_at<kDim>(r, c)) = v;
                }
                if (lane == 0) s_qs[r] = 1.0f;
            } else {
                constexpr int kN = (kChunks + 31) / 32;
                float x[kN][8];
                float top = 0.0f;
#pragma unroll
                for (int n = 0; n < kN; n++) {
                    const int c = lane + 32 * n;
#pragma unroll
                    for (int i = 0; i < 8; i++) x[n][i] = 0.0f;
                    if (on && c < kChunks && c * 8 < D) load8(reinterpret_cast<const float*>(src) + c * 8, x[n]);
#pragma unroll
                    for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(x[n][i]));
                }
                // fp16 terms: the row's largest value to [2^13, 2^14), so that the second term of all
                // but the smallest values is a normal number
                float up = 1.0f;
                if constexpr (kTerms == 2) {
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                    if (top > 0.0f && top < INFINITY) {
                        const int ex = (int)(__float_as_uint(top) >> 23) - 127;
                        up = exp2i(min(max(13 - ex, -110), 110));
                    }
                }
                if (lane == 0) s_qs[r] = 1.0f / up;
#pragma unroll
                for (int n = 0; n < kN; n++) {
                    const int c = lane + 32 * n;
                    if (c >= kChunks) continue;
#pragma unroll
                    for (int term = 0; term < kTerms; term++) {
                        uint32_t w[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const float a = x[n][2 * i] * (term == 0 ? up : 1.0f), b = x[n][2 * i + 1] * (term == 0 ? up : 1.0f);
                            w[i] = pack2<C>(a, b);
                            const float2 f = unpack2<C>(w[i]);
                            x[n][2 * i] = a - f.x;
                            x[n][2 * i + 1] = b - f.y;
                        }
                        *reinterpret_cast<uint4*>(qs + term * (kRows * kDim * 2) + tile_at<kDim>(r, c)) =
                            make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
        }
        __syncthreads();

        // ---- the keys --------------------------------------------------------
        const int g = lane >> 2, t2 = (lane & 3) * 2;
        float acc[kDim / 16][NT][4], m[NT][2], l[NT][2], qf[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int d = 0; d < kDim / 16; d++)
#pragma unroll
                for (int i = 0; i < 4; i++) acc[d][n][i] = 0.0f;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                m[n][i] = -INFINITY;
                l[n][i] = 0.0f;
                qf[n][i] = s_qs[n * 8 + t2 + i] * p.scale_log2;
            }
        }
        const int first_tok = it.rt * kRows / p.group;
        uint32_t any = 0;
        for (int t = t0 + warp; t < t1; t += W) {
            int ahead = stage + kStages - 1;
            if (ahead >= kStages) ahead -= kStages;
            __syncwarp();  // the tile that is overwritten was read by all lanes
            const uint32_t more = load_tile(it, t + (kStages - 1) * W, t1, page_next, ahead);
            page_next = look_up(it, t + kStages * W, t1);
            const uint32_t ok = (uint32_t)oks & 0xffffu;
            any |= ok;
            oks = (oks >> 16) | (unsigned long long)more << (16 * (kStages - 2));
            cp_async_wait<kStages - 1>();
            __syncwarp();
            const uint32_t kd = ring_u + stage * 2 * kTile, vd = kd + kTile;
            // fp32's precision: several short sums, since the matrix unit cuts off what a sum does not hold
            constexpr int kSums = kTerms == 1 ? 1 : 4;
            float sc[NT][4], part[NT][kSums][4];
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int i = 0; i < 4 * kSums; i++) part[n][i >> 2][i & 3] = 0.0f;
#pragma unroll
            for (int k2 = 0; k2 < kDim / 32; k2++) {
                if (k2 * 2 >= ksteps) break;
                uint32_t a0[4], a1[4];
                const int r = lane & 15, c = k2 * 4 + (lane >> 4);
                ldsm4(kd + tile_at<kDim>(r, c), a0);
                ldsm4(kd + tile_at<kDim>(r, c + 2), a1);
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int term = kTerms - 1; term >= 0; term--) {
                        uint32_t b[4];
                        ldsm4(qs_u + term * (kRows * kDim * 2) + tile_at<kDim>(n * 8 + (lane & 7), k2 * 4 + (lane >> 3)), b);
                        const int s0 = kSums == 1 ? 0 : term ? 2 : k2 & 1, s1 = kSums == 1 ? 0 : term ? 3 : k2 & 1;
                        mma16<C>(part[n][s0], a0, b[0], b[1]);
                        mma16<C>(part[n][s1], a1, b[2], b[3]);
                    }
            }
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    sc[n][i] = kSums == 1 ? part[n][0][i]
                                          : (part[n][0][i] + part[n][1 % kSums][i]) + (part[n][2 % kSums][i] + part[n][3 % kSums][i]);
            const bool plain = ok == 0xffffu && (t + 1) * kPaKeys <= it.len + (p.tree_mask ? 0 : first_tok + 1);
            float keep[NT][2];
#pragma unroll
            for (int n = 0; n < NT; n++) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float z = sc[n][i] * qf[n][i & 1];
                    if (!plain) {
                        const int kr = g + (i >> 1) * 8, row = it.rt * kRows + n * 8 + t2 + (i & 1);
                        if (!(ok >> kr & 1) || n * 8 + t2 + (i & 1) >= rows ||
                            !paged_sees(p, it, row / p.group, t * kPaKeys + kr))
                            z = -INFINITY;
                    }
                    sc[n][i] = z;
                }
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    float x = fmaxf(sc[n][i], sc[n][i + 2]);
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                    const float m1 = fmaxf(m[n][i], x), mu = m1 == -INFINITY ? 0.0f : m1;
                    keep[n][i] = ex2(m[n][i] - mu);
                    m[n][i] = m1;
                    sc[n][i] = ex2(sc[n][i] - mu);
                    sc[n][i + 2] = ex2(sc[n][i + 2] - mu);
                    l[n][i] = fmaf(l[n][i], keep[n][i], sc[n][i] + sc[n][i + 2]);
                }
                if (kTerms == 1 && __any_sync(0xffffffffu, keep[n][0] != 1.0f || keep[n][1] != 1.0f)) {
#pragma unroll
                    for (int d = 0; d < kDim / 16; d++)
#pragma unroll
                        for (int i = 0; i < 4; i++) acc[d][n][i] *= keep[n][i & 1];
                }
            }
            // the probabilities as 16-bit terms, transposed (of fp16: scaled by 2^14, which the epilogue takes back,
            // so that those of 2^-28 of the largest are still normal numbers: unscaled, 10^5 entries 25 octaves
            // below one would add to the sum and nothing to the output)
            uint32_t pb[NT][kPTerms][2];
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int hh = 0; hh < 2; hh++) {
                    float a = sc[n][2 * hh], b = sc[n][2 * hh + 1];
                    if constexpr (Elem<C>::code == HQ4_F16) {
                        a *= 16384.0f;
                        b *= 16384.0f;
                    }
#pragma unroll
                    for (int term = 0; term < kPTerms; term++) {
                        const uint32_t w = pack2<C>(a, b);
                        pb[n][term][hh] = transpose8(w);
                        const float2 f = unpack2<C>(w);
                        a -= f.x;
                        b -= f.y;
                    }
                }
#pragma unroll
            for (int d = 0; d < kDim / 16; d++) {
                if (d >= ksteps) break;
                uint32_t a[4];
                ldsm4_t(vd + tile_at<kDim>((lane & 7) + (lane >> 4) * 8, d * 2 + (lane >> 3 & 1)), a);
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    if constexpr (kTerms == 1) {
#pragma unroll
                        for (int term = kPTerms - 1; term >= 0; term--) mma16<C>(acc[d][n], a, pb[n][term][0], pb[n][term][1]);
                    } else {  // fp32's precision: a tile's sum by itself, then rounded to nearest into the whole
                        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int term = kPTerms - 1; term >= 0; term--) mma16<C>(sum, a, pb[n][term][0], pb[n][term][1]);
#pragma unroll
                        for (int i = 0; i < 4; i++) acc[d][n][i] = fmaf(acc[d][n][i], keep[n][i & 1], sum[i]);
                    }
                }
            }
            if (++stage == kStages) stage = 0;
        }
        // ---- the next item's first tiles; the warps' results, joined ----------
        const float back = Elem<C>::code == HQ4_F16 ? 1.0f / 16384.0f : 1.0f;
        __syncwarp();  // the ring is the warp's own: its lanes have read their last tile
        int os_at = warp * kRing;
        if constexpr (kAhead) {
            if (units < left) begin_item(nx, t_begin(0), t_end(nx, 0, units_of(nx, 0, left - units)));
            os_at += (stage + kStages - 1) % kStages * 2 * kTile;  // the stage that those leave free
        } else {
            cp_async_wait<0>();
            __syncwarp();
        }
        float* os = reinterpret_cast<float*>(smem + os_at);
        if (lane == 0) {
            s_os[warp] = os_at;
            s_any[warp] = any;
        }
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                float x = l[n][i];
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                const int r = n * 8 + t2 + i;
                if (g == 0) {
                    s_m[warp][r] = m[n][i];
                    s_l[warp][r] = x;
                }
#pragma unroll
                for (int d = 0; d < kDim / 16; d++) {
                    if (d >= ksteps) break;
                    os[r * kOs + d * 16 + g] = acc[d][n][i] * back;
                    os[r * kOs + d * 16 + g + 8] = acc[d][n][i + 2] * back;
                }
            }
        }
        __syncthreads();
        const int piece = 2 * blockIdx.x + (pieces++ ? 1 : 0);
        for (int r = warp; r < rows; r += W) {
            float mm = -INFINITY, ll = 0.0f, w[W];
#pragma unroll
            for (int i = 0; i < W; i++) mm = fmaxf(mm, s_m[i][r]);
            const float mu = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
            for (int i = 0; i < W; i++) {
                w[i] = exp2f(s_m[i][r] - mu);
                ll = fmaf(s_l[i][r], w[i], ll);
            }
            const int row = it.rt * kRows + r;
            if (whole)
#pragma unroll
                for (int i = 0; i < W; i++) w[i] = ll == 0.0f ? 0.0f : w[i] / ll;
            A* out = static_cast<A*>(p.out) + ((long long)(it.row0 + row / p.group) * p.n_heads + it.h * p.group + row % p.group) * D;
            float* part = ws.o + ((size_t)piece * kRows + r) * kDim;
            if (ll == 0.0f) {
                any = 0;
#pragma unroll
                for (int i = 0; i < W; i++) any |= s_any[i];
                if (!whole && any) ll = 1.0f;  // (of weight 0: its maximum is -inf)
            }
            bool bad = ll == 0.0f && any;
            for (int d = lane; d < D; d += 32) {
                float y = 0.0f;
#pragma unroll
                for (int i = 0; i < W; i++)
                    y = fmaf(reinterpret_cast<const float*>(smem + s_os[i])[r * kOs + d], w[i], y);
                if (whole) {
                    if (ll == 0.0f) y = 0.0f;
                    bad |= y != y;
                    out[d] = Elem<A>::from(y);
                } else {
                    part[d] = y;
                }
            }
            if (!whole && lane == 0) ws.ml[(size_t)piece * kRows + r] = make_float2(mm, ll);
            if (whole && __any_sync(0xffffffffu, bad)) paged_slow_row<A, C>(p, it, row);
        }
        __syncthreads();  // the rings and the queries are free again
        left -= units;
        from = 0;
        it = nx;
        if (!kAhead && left > 0) begin_item(it, t_begin(0), t_end(it, 0, units_of(it, 0, left)));
    }
}

// ---- launch ------------------------------------------------------------------

static inline cudaError_t launch_pdl_kernel(const void* fn, dim3 grid, dim3 block, size_t smem, cudaStream_t st, void** args) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t lc = {};
    lc.gridDim = grid;
    lc.blockDim = block;
    lc.dynamicSmemBytes = smem;
    lc.stream = st;
    lc.attrs = attr;
    lc.numAttrs = 1;
    return cudaLaunchKernelExC(&lc, fn, args);
}

template <class A, class C, int kDim, int NT, int W>
static int launch_pa(PagedAttnParams p, const PaPlan& pl, cudaStream_t st) {
    constexpr int smem = pa_smem<kDim, 8 * NT, pa_terms<A, C>(), W>();
    auto kern = paged_attn_kernel<A, C, kDim, NT, W>;
    static PerDeviceOnce once;
    if (smem_opt_in(once, kern, smem) != cudaSuccess) return HQ4_ERR_LAUNCH;
    void* args[] = {&p};
    if (launch_pdl_kernel((const void*)kern, dim3(pl.ctas), dim3(W * 32), smem, st, args) != cudaSuccess)
        return HQ4_ERR_LAUNCH;
    if (!pl.split || pl.ctas < 2) return HQ4_OK;
    int ctas = pl.ctas;
    void* cargs[] = {&p, &ctas};
    return launch_pdl_kernel((const void*)paged_combine_kernel<A, C, 8 * NT, kDim>,
                             dim3(pl.ctas - 1, pl.join), dim3(kCombineWarps * 32), 0, st, cargs) == cudaSuccess
               ? HQ4_OK
               : HQ4_ERR_LAUNCH;
}
template <class A, class C, int kDim>
static int launch_pa_nt(const PagedAttnParams& p, const PaPlan& pl, cudaStream_t st) {
    if (pl.warps == 2) return launch_pa<A, C, kDim, 1, 2>(p, pl, st);
    // 16-bit activations of more rows have the tensor-memory kernel
    if constexpr (sizeof(A) == 4 && kDim <= 128) {
        if (pl.nt == 4) return launch_pa<A, C, kDim, 4, 4>(p, pl, st);
    }
    if constexpr (sizeof(A) == 4 || kDim == 64) {
        if (pl.nt == 2) return launch_pa<A, C, kDim, 2, 4>(p, pl, st);
    }
    return launch_pa<A, C, kDim, 1, 4>(p, pl, st);
}
template <class A, class C>
static int launch_pa_dim(const PagedAttnParams& p, const PaPlan& pl, cudaStream_t st) {
    return pl.dim == 64 ? launch_pa_nt<A, C, 64>(p, pl, st)
         : pl.dim == 128 ? launch_pa_nt<A, C, 128>(p, pl, st) : launch_pa_nt<A, C, 256>(p, pl, st);
}

}  // namespace hq4
