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
// The work is bytes: every value is read once and written once.  One thread
// takes 8 consecutive values of a head's first half and the 8 they rotate
// with (16-byte loads and stores of 16-bit types), so a head is a group of
// D/16 threads, whose sum of squares is a shuffle tree.
#include <algorithm>

#include "hq4_host.cuh"
#include "hq4_paged.cuh"

namespace hq4 {

int check_device_cap();
int* status_word();

constexpr int kAppendThreads = 256;
constexpr int kAppendRows = 8;  // rows of a CTA at most

struct AppendParams {
    const void *q, *k, *v;
    long long q_stride, k_stride, v_stride;
    const float *q_norm, *k_norm;
    float eps;
    const int* positions;
    const float *cos, *sin;
    int max_pos, n_heads, n_kv, head_dim, rows_per_cta;
    void *k_cache, *v_cache, *q_out;
    PagedBatch b;
};

template <class A, class C>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const AppendParams p) {
    __shared__ int s_pos[kAppendRows];
    __shared__ long long s_at[kAppendRows];  // element of the entry in its page's first head; -1: not written
    pdl_launch_dependents();
    pdl_wait();
    const int D = p.head_dim, half = D >> 1;
    const int row0 = blockIdx.x * p.rows_per_cta;
    const int rows = min(p.rows_per_cta, p.b.n_rows - row0);
    if (threadIdx.x < rows) {
        const int t = row0 + threadIdx.x;
        const int s = find_seq(p.b.cu_rows, p.b.n_seqs, t);
        long long at = -1;
        int pos = 0;
        if (s >= 0) {
            const int e = __ldg(p.b.lens + s) + (t - __ldg(p.b.cu_rows + s));
            const int page = find_page(p.b, s, e);
            pos = p.positions ? __ldg(p.positions + t) : e;
            if (page >= 0 && pos >= 0 && pos < p.max_pos)
                at = (long long)page * p.b.page_stride + (long long)(e & ((1 << p.b.page_shift) - 1)) * D;
            else
                atomicOr(p.b.status, kStatusPaged);
        }
        s_pos[threadIdx.x] = pos;
        s_at[threadIdx.x] = at;
    }
    __syncthreads();
    const int tph = D >> 4;                            // threads of a head
    const int gw = tph <= 2 ? 2 : tph <= 4 ? 4 : tph <= 8 ? 8 : 16;  // lanes of a head: a power of two
    const int lane = threadIdx.x & (gw - 1);
    const int heads = p.n_heads + 2 * p.n_kv;
    const int items = rows * heads;
    const int step = kAppendThreads / gw;
    const int rounds = (items + step - 1) / step;  // the same for all lanes: shuffles below are warp-wide
    for (int r = 0; r < rounds; r++) {
        const int it = r * step + threadIdx.x / gw;
        const int row = it / heads, h = it - row * heads;
        const bool on = it < items && lane < tph && s_at[min(row, kAppendRows - 1)] >= 0;
        const int t = row0 + row;
        const int j = lane * 8;
        float a[8], b[8];
        const bool is_q = h < p.n_heads, is_k = !is_q && h < p.n_heads + p.n_kv;
        const int kh = h - p.n_heads - (is_k ? 0 : p.n_kv);
        if (on) {
            const A* src = is_q ? static_cast<const A*>(p.q) + t * p.q_stride + (long long)h * D
                         : is_k ? static_cast<const A*>(p.k) + t * p.k_stride + (long long)kh * D
                                : static_cast<const A*>(p.v) + t * p.v_stride + (long long)kh * D;
            load8(src + j, a);
            load8(src + half + j, b);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) a[i] = b[i] = 0.0f;
        }
        const float* nw = is_q ? p.q_norm : is_k ? p.k_norm : nullptr;
        if (p.q_norm || p.k_norm) {
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) ss = fmaf(a[i], a[i], fmaf(b[i], b[i], ss));
            for (int o = gw >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (nw && on) {
                const float inv = 1.0f / sqrtf(ss / (float)D + p.eps);
                float wa[8], wb[8];
                load8(nw + j, wa);
                load8(nw + half + j, wb);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    a[i] = a[i] * inv * wa[i];
                    b[i] = b[i] * inv * wb[i];
                }
            }
        }
        if (!on) continue;
        if (is_q || is_k) {
            float c[8], s[8];
            load8(p.cos + (size_t)s_pos[row] * half + j, c);
            load8(p.sin + (size_t)s_pos[row] * half + j, s);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float x = a[i], y = b[i];
                a[i] = x * c[i] - y * s[i];
                b[i] = y * c[i] + x * s[i];
            }
        }
        if (is_q) {
            A* dst = static_cast<A*>(p.q_out) + ((long long)t * p.n_heads + h) * D;
            store8(dst + j, a);
            store8(dst + half + j, b);
        } else {
            C* dst = static_cast<C*>(is_k ? p.k_cache : p.v_cache) + s_at[row] +
                     ((long long)kh << p.b.page_shift) * D;
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
    lc.gridDim = dim3((p.b.n_rows + p.rows_per_cta - 1) / p.rows_per_cta);
    lc.blockDim = dim3(kAppendThreads);
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
    // rows of a CTA: enough that its threads have work, few while there are few rows
    p.rows_per_cta = n_rows < 4 * 148 ? 1 : std::min(kAppendRows, std::max(1, n_rows / (4 * 148)));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (cache_type == HQ4_BF16)
        return act_type == HQ4_F32 ? launch_append<float, __nv_bfloat16>(p, st)
                                   : launch_append<__nv_bfloat16, __nv_bfloat16>(p, st);
    return act_type == HQ4_F32 ? launch_append<float, __half>(p, st) : launch_append<__half, __half>(p, st);
}
