// What the attention kernels over a paged cache share: the parameters, the
// division of the work, the visibility rule and the row-wise slow path.
//
// The unit of work is an item: one tile of kRows query rows of one sequence
// and one key/value head.  The G = n_heads / n_kv query heads of a key/value
// head are rows of the same tile (row r of a sequence is head r % G of token
// r / G), so each entry is read once for all of them.  An item's keys are cut
// into tiles; all items' tiles, in order, are one line of `total` units, of
// which CTA c takes the c-th equal part.  A part may begin or end inside an
// item: then the CTA leaves the item's running maximum, sum and unnormalised
// output of its keys in the workspace, and the combine kernel joins them in
// key order.  A CTA has at most two such pieces (its first and its last).  An
// item counts `extra` units before its tiles, for what beginning and ending one
// costs, so that CTAs with many short items finish with the others.
#pragma once
#include "hq4_paged.cuh"

namespace hq4 {

constexpr float kLog2e = 1.4426950408889634f;

struct PagedAttnParams {
    const void* q;
    const void *k, *v;
    void* out;
    long long q_stride;
    int n_heads, n_kv, group, head_dim;
    float scale_log2;              // softmax scale times log2(e)
    const uint32_t* tree_mask;     // [n_rows][mask_words], or null: causal
    int mask_words;
    int split;                     // units are key tiles; else whole items
    int extra;                     // units of an item before its tiles
    int take;                      // rows of a joining CTA
    void* ws;
    PagedBatch b;
};

struct PagedItem {
    int s, rt, h;      // sequence, row tile, key/value head
    int row0, n_tok;   // the sequence's first row and its tokens
    int len, keys;     // entries before its rows; entries that the tile may see
    int tiles;         // key tiles
    int weight;        // units
};
// Where a CTA's part begins.
struct PagedStart {
    PagedItem it;
    int pad[3];
    long long first;  // the item's first unit
    long long total;  // units of the whole batch
};

// Rows and lengths of a sequence, clamped to what exists: entries beyond all
// pages are not there, and sums with a length stay within 32 bits.
__device__ __forceinline__ void paged_seq(const PagedAttnParams& p, int s, PagedItem& it) {
    const int a = max(__ldg(p.b.cu_rows + s), 0), e = min(__ldg(p.b.cu_rows + s + 1), p.b.n_rows);
    it.s = s;
    it.row0 = a;
    it.n_tok = max(e - a, 0);
    it.len = min(max(__ldg(p.b.lens + s), -(1 << 30)), p.b.pages_per_seq << p.b.page_shift);
}
template <int kRows>
__device__ __forceinline__ int paged_row_tiles(const PagedAttnParams& p, const PagedItem& it) {
    return (it.n_tok * p.group + kRows - 1) / kRows;
}
// Keys and weight of row tile rt.
template <int kRows, int kKeys>
__device__ __forceinline__ void paged_row_tile(const PagedAttnParams& p, int rt, PagedItem& it) {
    const int cap = p.b.pages_per_seq << p.b.page_shift;
    const int last = min((rt + 1) * kRows, it.n_tok * p.group) - 1;
    const int n = p.tree_mask ? it.n_tok : last / p.group + 1;
    it.rt = rt;
    it.keys = (int)min(max((long long)it.len + n, 0ll), (long long)cap);
    it.tiles = max((it.keys + kKeys - 1) / kKeys, 1);  // an item without keys still writes its zeros
    it.weight = p.split ? p.extra + it.tiles : 1;
}
// The tiles of an item before its unit u.
__device__ __forceinline__ int paged_tiles_before(const PagedAttnParams& p, int u) { return max(u - p.extra, 0); }
// Units of sequence s, whose lane asks for it (s < 0: none).  A sequence of
// many row tiles is added up by its whole warp.
template <int kRows, int kKeys>
__device__ __forceinline__ long long paged_seq_units(const PagedAttnParams& p, int s) {
    PagedItem it = {};
    int n = 0;
    if (s >= 0) {
        paged_seq(p, s, it);
        n = paged_row_tiles<kRows>(p, it);
    }
    if (!p.split) return (long long)n * p.n_kv;
    long long w = 0;
    if (n <= 4)
        for (int rt = 0; rt < n; rt++) {
            paged_row_tile<kRows, kKeys>(p, rt, it);
            w += it.weight;
        }
    for (uint32_t many = __ballot_sync(0xffffffffu, n > 4); many; many &= many - 1) {
        const int from = __ffs(many) - 1, tiles = __shfl_sync(0xffffffffu, n, from);
        PagedItem o = {};
        o.n_tok = __shfl_sync(0xffffffffu, it.n_tok, from);
        o.len = __shfl_sync(0xffffffffu, it.len, from);
        long long sum = 0;
        for (int rt = threadIdx.x & 31; rt < tiles; rt += 32) {
            paged_row_tile<kRows, kKeys>(p, rt, o);
            sum += o.weight;
        }
#pragma unroll
        for (int i = 16; i > 0; i >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
        if ((int)(threadIdx.x & 31) == from) w = sum;
    }
    return w * p.n_kv;
}

struct PagedScan {
    long long warp[32];
    long long before;
    int seq;
};
// Inclusive sum over the CTA's threads; *all = the CTA's sum.
template <int kThreads>
__device__ __forceinline__ long long cta_scan(PagedScan& sh, long long v, long long* all) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += y;
    }
    __syncthreads();
    if (lane == 31) sh.warp[w] = v;
    __syncthreads();
    long long t = 0;
    for (int i = 0; i < kThreads / 32; i++) {
        if (i < w) v += sh.warp[i];
        t += sh.warp[i];
    }
    *all = t;
    return v;
}

// Where the parts are cut: part c of min(ctas, total) begins at unit
// floor(c total / parts), by 32-bit divisions unless the units are very many.
struct PagedCuts {
    long long q;
    unsigned r, parts;
    __device__ __forceinline__ PagedCuts(long long total, int ctas) {
        parts = (unsigned)min((long long)ctas, total);
        const unsigned by = max(parts, 1u);
        q = total >> 32 ? total / by : (long long)((unsigned)total / by);
        r = (unsigned)(total - q * by);
    }
    __device__ __forceinline__ long long at(unsigned c) const { return c * q + c * r / parts; }  // c, r < 2^16
};

// The CTA's part [pos, end) and the item that holds its first unit; pos == end
// for a CTA without work.  Parts are cut for min(gridDim.x, total) CTAs, so that
// every one of those has some.  All threads take part and get the same.
template <int kRows, int kKeys, int kThreads>
__device__ __forceinline__ PagedStart paged_part(const PagedAttnParams& p, PagedScan& sh, long long& pos,
                                                 long long& end) {
    PagedStart st = {};
    PagedItem& it = st.it;
    const int n = p.b.n_seqs;
    long long total = 0, all;
    long long mine = paged_seq_units<kRows, kKeys>(p, (int)threadIdx.x < n ? (int)threadIdx.x : -1);
    long long upto = cta_scan<kThreads>(sh, mine, &total);
    const long long total0 = total;
    for (int base = kThreads; base < n; base += kThreads) {
        const int s = base + threadIdx.x;
        cta_scan<kThreads>(sh, paged_seq_units<kRows, kKeys>(p, s < n ? s : -1), &all);
        total += all;
    }
    const PagedCuts cuts(total, gridDim.x);
    pos = end = 0;
    st.total = total;
    if (blockIdx.x >= cuts.parts) return st;
    pos = cuts.at(blockIdx.x);
    end = cuts.at(blockIdx.x + 1);
    long long run = 0, sum = total0;
    for (int base = 0;; base += kThreads) {  // ends at the chunk that holds pos: pos < total
        if (pos < run + sum) {
            __syncthreads();
            if (run + upto - mine <= pos && pos < run + upto) {
                sh.seq = base + threadIdx.x;
                sh.before = run + upto - mine;
            }
            __syncthreads();
            break;
        }
        run += sum;
        const int s = base + kThreads + threadIdx.x;
        mine = paged_seq_units<kRows, kKeys>(p, s < n ? s : -1);
        upto = cta_scan<kThreads>(sh, mine, &sum);
    }
    paged_seq(p, sh.seq, it);
    long long first = sh.before;
    const int n_rt = paged_row_tiles<kRows>(p, it), lane = threadIdx.x & 31;
    for (int rt0 = 0;; rt0 += 32) {  // 32 row tiles at a time: a lane each (every warp alike)
        PagedItem o = it;
        long long w = 0;
        if (rt0 + lane < n_rt) {
            paged_row_tile<kRows, kKeys>(p, rt0 + lane, o);
            w = (long long)o.weight * p.n_kv;
        }
        long long upto = w;
#pragma unroll
        for (int i = 1; i < 32; i <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, upto, i);
            if (lane >= i) upto += y;
        }
        const uint32_t here = __ballot_sync(0xffffffffu, w > 0 && pos < first + upto);
        if (here || rt0 + 32 >= n_rt) {  // (pos lies in this sequence: one of its row tiles holds it)
            const int at = here ? __ffs(here) - 1 : 0;
            first += __shfl_sync(0xffffffffu, upto - w, at);
            paged_row_tile<kRows, kKeys>(p, rt0 + at, it);
            it.h = (int)((pos - first) / it.weight);
            st.first = first + (long long)it.h * it.weight;
            break;
        }
        first += __shfl_sync(0xffffffffu, upto, 31);
    }
    return st;
}
// The item after `it`, if there is one.
template <int kRows, int kKeys>
__device__ __forceinline__ void paged_next(const PagedAttnParams& p, PagedItem& it) {
    if (++it.h < p.n_kv) return;
    it.h = 0;
    int rt = it.rt + 1;
    while (rt >= paged_row_tiles<kRows>(p, it)) {
        rt = 0;
        paged_seq(p, it.s + 1, it);
    }
    paged_row_tile<kRows, kKeys>(p, rt, it);
}

// Whether token tok of the item's sequence sees entry e (0 <= e < keys).
__device__ __forceinline__ bool paged_sees(const PagedAttnParams& p, const PagedItem& it, int tok, int e) {
    const int j = e - it.len;  // its place among the new entries
    if (j < 0) return true;
    if (!p.tree_mask) return j <= tok;
    if (j >= it.n_tok || (j >> 5) >= p.mask_words) return false;
    return __ldg(p.tree_mask + (size_t)(it.row0 + tok) * p.mask_words + (j >> 5)) >> (j & 31) & 1;
}

// One output row, entry by entry (one warp).  The tiled kernels multiply
// masked probabilities of zero by values that they do not look at; where such
// a value is an infinity or a NaN, the row comes out as NaN and is computed
// here again, from the entries that it sees alone.  So is a row whose sum is 0,
// unless none of the entries has a page: one that sees nothing is zeros, one whose
// scores are all -inf is NaN (0 / 0).
template <class A, class C>
__device__ __noinline__ void paged_slow_row(const PagedAttnParams& p, const PagedItem& it, int r) {
    const int lane = threadIdx.x & 31, D = p.head_dim;
    const int tok = r / p.group, head = it.h * p.group + r % p.group;
    const A* q = static_cast<const A*>(p.q) + (long long)(it.row0 + tok) * p.q_stride + (long long)head * D;
    float qv[8], acc[8], m = -INFINITY, l = 0.0f;
    bool any = false;
    const int nd = D >> 5;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        qv[i] = i < nd ? Elem<A>::to(q[lane + 32 * i]) : 0.0f;
        acc[i] = 0.0f;
    }
    // 32 entries are looked up at once: a padded sequence that still has a length, but no pages, is passed quickly
    // (a lane's entry, and its page where the row sees it)
    int mine = -1;
    uint32_t left = 0;
    for (int e = 0; e < it.keys; e++) {
        if ((e & 31) == 0) {
            mine = e + lane < it.keys && paged_sees(p, it, tok, e + lane) ? find_page(p.b, it.s, e + lane) : -1;
            left = __ballot_sync(0xffffffffu, mine >= 0);
        }
        if (!left) {
            e |= 31;
            continue;
        }
        if (!(left >> (e & 31) & 1)) continue;
        left &= ~(1u << (e & 31));
        const int page = __shfl_sync(0xffffffffu, mine, e & 31);
        const long long at = (long long)page * p.b.page_stride +
                             (((long long)it.h << p.b.page_shift) + (e & ((1 << p.b.page_shift) - 1))) * D;
        const C* k = static_cast<const C*>(p.k) + at;
        const C* v = static_cast<const C*>(p.v) + at;
        float z = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < nd) z = fmaf(qv[i], Elem<C>::to(k[lane + 32 * i]), z);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
        z *= p.scale_log2;
        const float m1 = (z > m || z != z) ? z : m, mu = m1 == -INFINITY ? 0.0f : m1;  // (scores of -inf alone so far)
        const float keep = m == m1 ? 1.0f : exp2f(m - mu), w = exp2f(z - mu);
        m = m1;
        any = true;
        l = l * keep + w;
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < nd) acc[i] = acc[i] * keep + w * Elem<C>::to(v[lane + 32 * i]);
    }
    A* out = static_cast<A*>(p.out) + ((long long)(it.row0 + tok) * p.n_heads + head) * D;
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (i < nd) out[lane + 32 * i] = Elem<A>::from(any ? acc[i] / l : 0.0f);
}

// The pieces of split items in the workspace: CTA c's first piece is 2c, its
// last one 2c + 1.
template <int kRows, int kDim>
struct PagedWs {
    PagedStart* info;  // of each CTA's part; without any work at all, of CTA 0 alone
    float2* ml;       // [pieces][kRows]: running maximum (of log2 scores) and sum (1 for 0 where an entry had a page)
    float* o;         // [pieces][kRows][kDim], not divided
    __host__ __device__ PagedWs(void* ws, int ctas) {
        unsigned char* p = static_cast<unsigned char*>(ws);
        info = reinterpret_cast<PagedStart*>(p);
        p += (size_t)ctas * sizeof(PagedStart);
        ml = reinterpret_cast<float2*>(p);
        p += (size_t)ctas * 2 * kRows * sizeof(float2);
        o = reinterpret_cast<float*>(p);
    }
};
static_assert(sizeof(PagedStart) % 16 == 0, "the pieces behind the items keep their alignment");

// CTA (c, y): if part c begins inside an item, and c is the first part that
// does in that item, joins rows of the item's pieces.  With few rows to an item
// (decode, where a long sequence has many pieces) a CTA takes one, its warps a
// part of the pieces each; else `take`, a warp a row.  A lane has 4 consecutive
// values of each 128.  The order of the sums does not depend on timing.
constexpr int kCombineWarps = 4;
template <class A, class C, int kRows, int kDim>
__global__ void __launch_bounds__(kCombineWarps * 32) paged_combine_kernel(const __grid_constant__ PagedAttnParams p,
                                                                           int ctas) {
    constexpr int kShare = kRows <= 32 ? kCombineWarps : 1;  // warps of a row
    constexpr int kPer = (kDim + 127) / 128, kDeep = 8 / kPer;  // pieces whose values are asked for at once
    __shared__ float4 s_acc[kShare][kPer][32];
    __shared__ float s_l[kShare];
    pdl_launch_dependents();
    pdl_wait();
    const PagedWs<kRows, kDim> ws(p.ws, ctas);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, D = p.head_dim;
    const int c = blockIdx.x + 1;
    const PagedStart st = ws.info[c];
    const PagedItem& it = st.it;
    const PagedCuts cuts(ws.info[0].total, ctas);
    if (c >= (int)cuts.parts) return;
    // nothing to join where no tile lies before this cut, or one lies before the last cut
    const long long before = cuts.at(c - 1);
    if (cuts.at(c) - st.first <= p.extra || before - st.first > p.extra) return;
    const int rows = min(kRows, it.n_tok * p.group - it.rt * kRows);
    const int first_piece = 2 * (c - 1) + (st.first <= before ? 0 : 1);
    // pieces: that one, then the first ones of parts c, c + 1, ... up to the one with the item's last unit
    const long long last = st.first + it.weight - 1;
    int owner = min((int)__fdividef((float)last, (float)cuts.q + __fdividef((float)cuts.r, (float)cuts.parts)),
                    (int)cuts.parts - 1);
    while (cuts.at(owner) > last) owner--;
    while (cuts.at(owner + 1) <= last) owner++;
    const int n = owner - (c - 1) + 1;
    const int mine = kShare > 1 ? warp : 0;  // the warp's share of the pieces: each kShare-th
    const int end = kShare > 1 ? min(rows, (int)blockIdx.y + 1) : min(rows, (int)(blockIdx.y + 1) * p.take);
    for (int r = kShare > 1 ? blockIdx.y : blockIdx.y * p.take + warp; r < end; r += kCombineWarps) {
        auto at = [&](int i) { return (size_t)(i == 0 ? first_piece : 2 * (c - 1 + i)) * kRows + r; };
        float4 v[kDeep][kPer];
        auto ask = [&](int i0) {  // values of the share's next pieces, zeros behind the last
#pragma unroll
            for (int i = 0; i < kDeep; i++) {
                const float* o = ws.o + at(min(i0 + i * kShare, n - 1)) * kDim;
#pragma unroll
                for (int j = 0; j < kPer; j++)
                    v[i][j] = i0 + i * kShare < n && lane * 4 + 128 * j < D
                                  ? *reinterpret_cast<const float4*>(o + lane * 4 + 128 * j) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
        };
        ask(mine);  // (before the weights are known)
        float m = -INFINITY;
        bool any = false;  // an entry has a page
        for (int i = lane; i < n; i += 32) {
            const float2 ml = ws.ml[at(i)];
            m = fmaxf(m, ml.x);
            any |= ml.y != 0.0f;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float mu = m == -INFINITY ? 0.0f : m;
        float4 acc[kPer];
        float l = 0.0f;
#pragma unroll
        for (int j = 0; j < kPer; j++) acc[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int i0 = mine; i0 < n; i0 += 32 * kShare) {  // 32 pieces' weights, a lane each, then their values
            float w = 0.0f;
            if (i0 + lane * kShare < n) {
                const float2 ml = ws.ml[at(i0 + lane * kShare)];
                w = exp2f(ml.x - mu);
                l = fmaf(ml.y, w, l);
            }
            for (int i1 = 0; i1 < 32 && i0 + i1 * kShare < n; i1 += kDeep) {
#pragma unroll
                for (int i = 0; i < kDeep; i++) {
                    const float wi = __shfl_sync(0xffffffffu, w, i1 + i);  // 0 behind the last
#pragma unroll
                    for (int j = 0; j < kPer; j++) {
                        acc[j].x = fmaf(v[i][j].x, wi, acc[j].x);
                        acc[j].y = fmaf(v[i][j].y, wi, acc[j].y);
                        acc[j].z = fmaf(v[i][j].z, wi, acc[j].z);
                        acc[j].w = fmaf(v[i][j].w, wi, acc[j].w);
                    }
                }
                if (i0 + (i1 + kDeep) * kShare < n) ask(i0 + (i1 + kDeep) * kShare);
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        if constexpr (kShare > 1) {
#pragma unroll
            for (int j = 0; j < kPer; j++) s_acc[warp][j][lane] = acc[j];
            if (lane == 0) s_l[warp] = l;
            __syncthreads();
            if (warp != 0) return;
            for (int w = 1; w < kShare; w++) {
                l += s_l[w];
#pragma unroll
                for (int j = 0; j < kPer; j++) {
                    const float4 v = s_acc[w][j][lane];
                    acc[j].x += v.x;
                    acc[j].y += v.y;
                    acc[j].z += v.z;
                    acc[j].w += v.w;
                }
            }
        }
        const int row = it.rt * kRows + r, tok = row / p.group, head = it.h * p.group + row % p.group;
        A* out = static_cast<A*>(p.out) + ((long long)(it.row0 + tok) * p.n_heads + head) * D;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        bool bad = l == 0.0f && any;
#pragma unroll
        for (int j = 0; j < kPer; j++)
            if (lane * 4 + 128 * j < D) {
                const float4 y = l == 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                                           : make_float4(acc[j].x * inv, acc[j].y * inv, acc[j].z * inv, acc[j].w * inv);
                bad |= y.x != y.x || y.y != y.y || y.z != y.z || y.w != y.w;
                store4(out + lane * 4 + 128 * j, y);
            }
        if (__any_sync(0xffffffffu, bad)) paged_slow_row<A, C>(p, it, row);
    }
}

// How a call is run (host).
struct PaPlan {
    int tc;     // tensor-memory kernel (hq4_paged_tc.cuh), else the warp-level one (hq4_paged_rows.cuh)
    int nt;     // 8-row tiles of the latter, and its warps
    int warps;
    int dim;    // head_dim rounded up to what the kernels are built for
    int ctas, split, extra;
    int join, take;  // rows of an item at most, and those of a CTA that joins pieces
    long long ws;
};

}  // namespace hq4
