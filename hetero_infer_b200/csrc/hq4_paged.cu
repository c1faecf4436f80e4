// Appending to a paged cache: the step's keys, rotated, and its values go to
// their pages, the rotated queries come out, with an RMS norm of every query
// and key head before the rotation where the model has one.
//
//   y = x * rsqrt(mean(x^2) + eps) * w              (with norm weights)
//   (y_j, y_{j+D/2}) -> (y_j c_j - y_{j+D/2} s_j, y_{j+D/2} c_j + y_j s_j)
//
// with c, s the row of the cos/sin tables at the token's position.  All
// arithmetic is fp32; each value is rounded once, to the cache's or the
// queries' type.
//
// The work is bytes: every value is read once and written once.  8191 rows of 28
// and 4 heads of 128 take 36 us, 0.66 of the copy rate: DRAM is half idle and so
// are the issue slots; at 64 registers, which leave an SM four CTAs, a thread
// spills 52 bytes (fp32: 116).  One thread
// takes 8 consecutive values of a head's first half and the 8 they rotate with
// (16-byte loads and stores of 16-bit types), so a head is a group of D/16
// lanes, whose sum of squares is a shuffle tree, and a warp has the heads that
// fit its lanes, kAppendAhead times.  Its values are asked for first: where
// they go (sequence, length, page, cosines: four loads that wait for one
// another) is looked up meanwhile.
#include <algorithm>

#include "hq4_host.cuh"
#include "hq4_paged.cuh"

namespace hq4 {

int check_device_cap();
int* status_word();

constexpr int kAppendWarps = 8;
constexpr int kAppendAhead = 2;  // times the heads of a warp (8191 rows: 1: 36.5 us, 2: 35.6, 3: 34.6; 8 rows: 2.9, 3.2, 4.5)

struct AppendParams {
    const void *q, *k, *v;
    long long q_stride, k_stride, v_stride;
    const float *q_norm, *k_norm;
    float eps;
    const int* positions;
    const float *cos, *sin;
    int max_pos, n_heads, n_kv, head_dim, warps_per_row;
    void *k_cache, *v_cache, *q_out;
    PagedBatch b;
};

template <class A, class C>
__global__ void __launch_bounds__(kAppendWarps * 32, 4) paged_append_kernel(const __grid_constant__ AppendParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const long long w = (long long)blockIdx.x * kAppendWarps + (threadIdx.x >> 5);
    const int t = (int)(w / p.warps_per_row), part = (int)(w - (long long)t * p.warps_per_row);
    if (t >= p.b.n_rows) return;
    const int D = p.head_dim, half = D >> 1;
    const int tph = D >> 4;                                          // lanes of a head
    const int gw = tph <= 2 ? 2 : tph <= 4 ? 4 : tph <= 8 ? 8 : 16;  // those and idle ones: a power of two
    const int sub = lane & (gw - 1), per = 32 / gw;
    const int j = sub * 8, heads = p.n_heads + 2 * p.n_kv;
    const int h0 = part * kAppendAhead * per + lane / gw;  // the thread's first head; the next ones `per` on
    const bool on = sub < tph;
    Raw8<A> ra[kAppendAhead], rb[kAppendAhead];
#pragma unroll
    for (int i = 0; i < kAppendAhead; i++) {
        const int h = h0 + i * per;
        if (!on || h >= heads) continue;
        const A* src = h < p.n_heads ? static_cast<const A*>(p.q) + t * p.q_stride + (long long)h * D
                     : h < p.n_heads + p.n_kv
                         ? static_cast<const A*>(p.k) + t * p.k_stride + (long long)(h - p.n_heads) * D
                         : static_cast<const A*>(p.v) + t * p.v_stride + (long long)(h - p.n_heads - p.n_kv) * D;
        ra[i].load(src + j);
        rb[i].load(src + half + j);
    }
    const int s = find_seq(p.b.cu_rows, p.b.n_seqs, t);
    if (s < 0) return;
    const long long far = (long long)__ldg(p.b.lens + s) + (t - __ldg(p.b.cu_rows + s));
    const int e = far > 0x7fffffff ? -1 : (int)far;
    const int page = find_page(p.b, s, e), pos = p.positions ? __ldg(p.positions + t) : e;
    if (page < 0 || pos < 0 || pos >= p.max_pos) {
        if (part == 0 && lane == 0) atomicOr(p.b.status, kStatusPaged);
        return;
    }
    // the entry's place in its page's first head
    const long long at = (long long)page * p.b.page_stride + (long long)(e & ((1 << p.b.page_shift) - 1)) * D;
    float c[8], sn[8];
    if (on) {
        load8(p.cos + (size_t)pos * half + j, c);
        load8(p.sin + (size_t)pos * half + j, sn);
    }
#pragma unroll
    for (int i = 0; i < kAppendAhead; i++) {
        const int h = h0 + i * per;
        const bool is_q = h < p.n_heads, is_k = !is_q && h < p.n_heads + p.n_kv;
        float a[8], b[8];
        ra[i].get(a);
        rb[i].get(b);
        if (p.q_norm || p.k_norm) {
            float ss = 0.0f;
            if (on && h < heads)
#pragma unroll
                for (int x = 0; x < 8; x++) ss = fmaf(a[x], a[x], fmaf(b[x], b[x], ss));
            for (int o = gw >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            const float* nw = is_q ? p.q_norm : is_k ? p.k_norm : nullptr;
            if (on && nw) {
                const float inv = 1.0f / sqrtf(ss / (float)D + p.eps);
                float wa[8], wb[8];
                load8(nw + j, wa);
                load8(nw + half + j, wb);
#pragma unroll
                for (int x = 0; x < 8; x++) {
                    a[x] = a[x] * inv * wa[x];
                    b[x] = b[x] * inv * wb[x];
                }
            }
        }
        if (!on || h >= heads) continue;
        if (is_q || is_k) {
#pragma unroll
            for (int x = 0; x < 8; x++) {
                const float y = a[x], z = b[x];
                a[x] = y * c[x] - z * sn[x];
                b[x] = z * c[x] + y * sn[x];
            }
        }
        if (is_q) {
            A* dst = static_cast<A*>(p.q_out) + ((long long)t * p.n_heads + h) * D;
            store8(dst + j, a);
            store8(dst + half + j, b);
        } else {
            const int kh = h - p.n_heads - (is_k ? 0 : p.n_kv);
            C* dst = static_cast<C*>(is_k ? p.k_cache : p.v_cache) + at + ((long long)kh << p.b.page_shift) * D;
            store8(dst + j, a);
            store8(dst + half + j, b);
        }
    }
}

template <class A, class C>
static int launch_append(const AppendParams& p, cudaStream_t st) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)(((long long)p.b.n_rows * p.warps_per_row + kAppendWarps - 1) / kAppendWarps));
    lc.blockDim = dim3(kAppendWarps * 32);
    lc.stream = st;
    lc.attrs = attr;
    lc.numAttrs = 1;
    return cudaLaunchKernelEx(&lc, paged_append_kernel<A, C>, p) == cudaSuccess ? HQ4_OK : HQ4_ERR_LAUNCH;
}

// Checks of the arguments that the paged entry points share (before the device
// is looked at); fills b but for its status word.
int paged_batch(PagedBatch& b, int n_rows, int n_heads, int n_kv, int head_dim, const int* cu_rows, const int* lens,
                int n_seqs, const int* pages, int pages_per_seq, const void* k_cache, const void* v_cache,
                int cache_type, int act_type, int n_pages, int page_size, long long page_stride) {
    if (n_rows <= 0 || n_heads <= 0 || n_kv <= 0 || n_heads % n_kv || head_dim <= 0 || head_dim % 32 ||
        head_dim > 256 || n_seqs <= 0 || pages_per_seq <= 0 || n_pages <= 0)
        return HQ4_ERR_SHAPE;
    if (cache_type != HQ4_BF16 && cache_type != HQ4_F16) return HQ4_ERR_SHAPE;
    if (act_type != HQ4_F32 && act_type != cache_type) return HQ4_ERR_SHAPE;
    int shift = 0;
    while ((1 << shift) < page_size && shift < 12) shift++;
    if (page_size < 8 || (1 << shift) != page_size) return HQ4_ERR_SHAPE;
    if ((long long)pages_per_seq * page_size > 0x7fffffffll - (1 << 20)) return HQ4_ERR_SHAPE;
    if (page_stride < (long long)n_kv * page_size * head_dim) return HQ4_ERR_SHAPE;
    if (!cu_rows || !lens || !pages || !k_cache || !v_cache) return HQ4_ERR_SHAPE;
    if ((((uintptr_t)k_cache | (uintptr_t)v_cache) & 15) || (page_stride & 7) ||
        (((uintptr_t)cu_rows | (uintptr_t)lens | (uintptr_t)pages) & 3))
        return HQ4_ERR_ALIGN;
    b.cu_rows = cu_rows;
    b.lens = lens;
    b.pages = pages;
    b.n_seqs = n_seqs;
    b.n_rows = n_rows;
    b.pages_per_seq = pages_per_seq;
    b.n_pages = n_pages;
    b.page_shift = shift;
    b.page_stride = page_stride;
    return HQ4_OK;
}

}  // namespace hq4

using namespace hq4;

extern "C" int hq4_paged_append(const void* q, const void* k, const void* v, int act_type, int n_rows, int n_heads,
                                int n_kv, int head_dim, long long q_stride, long long k_stride, long long v_stride,
                                const float* q_norm, const float* k_norm, float eps, const int* cu_rows,
                                const int* lens, int n_seqs, const int* positions, const float* rope_cos,
                                const float* rope_sin, int max_pos, const int* pages, int pages_per_seq, void* k_cache,
                                void* v_cache, int cache_type, int n_pages, int page_size, long long page_stride,
                                void* q_out, void* stream) {
    AppendParams p = {};
    if (int rc = paged_batch(p.b, n_rows, n_heads, n_kv, head_dim, cu_rows, lens, n_seqs, pages, pages_per_seq,
                             k_cache, v_cache, cache_type, act_type, n_pages, page_size, page_stride))
        return rc;
    if (!q || !k || !v || !q_out || !rope_cos || !rope_sin || max_pos <= 0 || !(eps >= 0.0f)) return HQ4_ERR_SHAPE;
    if (q_stride < (long long)n_heads * head_dim || k_stride < (long long)n_kv * head_dim ||
        v_stride < (long long)n_kv * head_dim)
        return HQ4_ERR_SHAPE;
    const int per16 = act_type == HQ4_F32 ? 3 : 7;  // elements of 16 bytes, less one
    if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out | (uintptr_t)rope_cos | (uintptr_t)rope_sin |
         (uintptr_t)q_norm | (uintptr_t)k_norm) & 15 ||
        ((uintptr_t)positions & 3) || ((q_stride | k_stride | v_stride) & per16))
        return HQ4_ERR_ALIGN;
    const int elem = act_type == HQ4_F32 ? 4 : 2;
    const long long q_row = (long long)n_heads * head_dim, k_row = (long long)n_kv * head_dim, out_bytes = n_rows * q_row * elem;
    if (rows_overlap(q, n_rows, q_stride, q_row, elem, q_out, out_bytes) ||
        rows_overlap(k, n_rows, k_stride, k_row, elem, q_out, out_bytes) ||
        rows_overlap(v, n_rows, v_stride, k_row, elem, q_out, out_bytes))
        return HQ4_ERR_SHAPE;
    // what is written is not read: neither the rows nor the queries lie in the caches, nor the one cache in the other
    const long long page = (long long)n_kv * page_size * head_dim;
    const __int128 cache_bytes = ((__int128)(n_pages - 1) * page_stride + page) * 2;
    const void* const caches[2] = {k_cache, v_cache};
    for (const void* cache : caches)
        if (rows_overlap(q_out, n_rows, q_row, q_row, elem, cache, cache_bytes) ||
            rows_overlap(q, n_rows, q_stride, q_row, elem, cache, cache_bytes) ||
            rows_overlap(k, n_rows, k_stride, k_row, elem, cache, cache_bytes) ||
            rows_overlap(v, n_rows, v_stride, k_row, elem, cache, cache_bytes))
            return HQ4_ERR_SHAPE;
    if (pages_overlap(k_cache, v_cache, n_pages, page_stride, page, 2)) return HQ4_ERR_SHAPE;
    if (int rc = check_device_cap()) return rc;
    p.b.status = status_word();
    if (!p.b.status) return HQ4_ERR_LAUNCH;
    p.q = q;
    p.k = k;
    p.v = v;
    p.q_stride = q_stride;
    p.k_stride = k_stride;
    p.v_stride = v_stride;
    p.q_norm = q_norm;
    p.k_norm = k_norm;
    p.eps = eps;
    p.positions = positions;
    p.cos = rope_cos;
    p.sin = rope_sin;
    p.max_pos = max_pos;
    p.n_heads = n_heads;
    p.n_kv = n_kv;
    p.head_dim = head_dim;
    p.k_cache = k_cache;
    p.v_cache = v_cache;
    p.q_out = q_out;
    const int tph = head_dim >> 4, per = 32 / (tph <= 2 ? 2 : tph <= 4 ? 4 : tph <= 8 ? 8 : 16);
    p.warps_per_row = (n_heads + 2 * n_kv + per * kAppendAhead - 1) / (per * kAppendAhead);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (cache_type == HQ4_BF16)
        return act_type == HQ4_F32 ? launch_append<float, __nv_bfloat16>(p, st)
                                   : launch_append<__nv_bfloat16, __nv_bfloat16>(p, st);
    return act_type == HQ4_F32 ? launch_append<float, __half>(p, st) : launch_append<__half, __half>(p, st);
}
