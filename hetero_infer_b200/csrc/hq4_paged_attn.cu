// Attention over a paged cache: plans and entry points.
#include <algorithm>

#include "hq4_paged_rows.cuh"

namespace hq4 {

int check_device_cap();
int* status_word();
int paged_batch(PagedBatch& b, int n_rows, int n_heads, int n_kv, int head_dim, const int* cu_rows, const int* lens,
                int n_seqs, const int* pages, int pages_per_seq, const void* k_cache, const void* v_cache,
                int cache_type, int act_type, int n_pages, int page_size, long long page_stride);
int paged_rows_bf16(bool f32, const PagedAttnParams& p, const PaPlan& pl, cudaStream_t st);
int paged_rows_f16(bool f32, const PagedAttnParams& p, const PaPlan& pl, cudaStream_t st);
int paged_tc_bf16(const PagedAttnParams& p, const PaPlan& pl, cudaStream_t st);
int paged_tc_f16(const PagedAttnParams& p, const PaPlan& pl, cudaStream_t st);

// More than kPaTcRows rows to a sequence and key/value head on average: the
// tensor-memory kernel, whose tile of 128 rows is then worth filling (16-bit
// activations only). Else tiles of 8, 16 or 32 rows (16 at most for wide
// heads, whose outputs fill the registers). Split over keys when a sequence
// may be longer than kPaWhole entries (shorter ones are a CTA's work whole,
// and need no second kernel).
constexpr int kPaTcRows = 32;
constexpr int kPaWhole = 512;
static PaPlan pa_plan(int act_type, int n_rows, int n_heads, int n_kv, int head_dim, int n_seqs, int pages_per_seq,
                      int page_size, int sms) {
    PaPlan r;
    const long long group = n_heads / n_kv;
    const long long avg = ((long long)n_rows + n_seqs - 1) / n_seqs * group;
    r.tc = act_type != HQ4_F32 && avg > kPaTcRows;
    r.dim = head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
    r.nt = avg <= 8 ? 1 : avg <= 16 || r.dim == 256 ? 2 : 4;
    const int rows = !r.tc ? 8 * r.nt : r.dim == 256 ? 128 : 256;
    const int keys = !r.tc ? kPaKeys : r.dim == 256 ? 64 : 128;
    const int per_sm = r.tc || r.dim == 256 ? 1 : r.dim == 128 ? 2 : 3;
    const long long cap = (long long)pages_per_seq * page_size;
    const long long items = ((long long)n_rows * group / rows + n_seqs) * n_kv;  // at most
    r.split = cap > kPaWhole;
    const long long units = r.split ? items * ((cap + keys - 1) / keys) : items;
    r.ctas = (int)std::min<long long>(units, (long long)sms * per_sm);
    // what an item costs besides its tiles, in tiles, where a CTA has many: with it 64 streams of 100 to 8200
    // entries decode in 117 us, without it in 137 (16 drafted trees: 83 and 109 us)
    r.extra = units < 8ll * r.ctas ? 0 : r.tc ? 4 : 18;
    r.ws = r.split ? (long long)r.ctas * (sizeof(PagedStart) + 2ll * rows * (sizeof(float2) + r.dim * sizeof(float))) : 0;
    return r;
}

static int paged_attention(const void* q, int act_type, int n_rows, int n_heads, int n_kv, int head_dim,
                           long long q_stride, const int* cu_rows, const int* lens, int n_seqs, const int* pages,
                           int pages_per_seq, const void* k_cache, const void* v_cache, int cache_type, int n_pages,
                           int page_size, long long page_stride, const uint32_t* tree_mask, int mask_words, float scale,
                           void* out, void* workspace, long long workspace_bytes, void* stream) {
    PagedAttnParams p = {};
    if (int rc = paged_batch(p.b, n_rows, n_heads, n_kv, head_dim, cu_rows, lens, n_seqs, pages, pages_per_seq,
                             k_cache, v_cache, cache_type, act_type, n_pages, page_size, page_stride))
        return rc;
    if (!q || !out || q_stride < (long long)n_heads * head_dim || !(scale == scale)) return HQ4_ERR_SHAPE;
    if ((long long)n_rows * (n_heads / n_kv) > 0x7fffff00ll) return HQ4_ERR_SHAPE;
    if ((((uintptr_t)q | (uintptr_t)out) & 15) || (q_stride & (act_type == HQ4_F32 ? 3 : 7)) ||
        ((uintptr_t)tree_mask & 3))
        return HQ4_ERR_ALIGN;
    if (int rc = check_device_cap()) return rc;
    p.b.status = status_word();
    const int sms = device_sms();
    if (!p.b.status || sms <= 0) return HQ4_ERR_LAUNCH;
    const PaPlan pl = pa_plan(act_type, n_rows, n_heads, n_kv, head_dim, n_seqs, pages_per_seq, page_size, sms);
    if (pl.ws) {
        if (!workspace || workspace_bytes < pl.ws) return HQ4_ERR_SHAPE;
        if ((uintptr_t)workspace & 127) return HQ4_ERR_ALIGN;
    }
    p.q = q;
    p.k = k_cache;
    p.v = v_cache;
    p.out = out;
    p.q_stride = q_stride;
    p.n_heads = n_heads;
    p.n_kv = n_kv;
    p.group = n_heads / n_kv;
    p.head_dim = head_dim;
    p.scale_log2 = scale * kLog2e;
    p.tree_mask = tree_mask;
    p.mask_words = mask_words;
    p.split = pl.split;
    p.extra = pl.extra;
    p.ws = pl.ws ? workspace : nullptr;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (pl.tc) return cache_type == HQ4_BF16 ? paged_tc_bf16(p, pl, st) : paged_tc_f16(p, pl, st);
    return cache_type == HQ4_BF16 ? paged_rows_bf16(act_type == HQ4_F32, p, pl, st)
                                  : paged_rows_f16(act_type == HQ4_F32, p, pl, st);
}

}  // namespace hq4

using namespace hq4;

extern "C" long long hq4_paged_attention_workspace_bytes(int act_type, int n_rows, int n_heads, int n_kv, int head_dim,
                                                         int n_seqs, int pages_per_seq, int page_size) {
    if (n_rows <= 0 || n_heads <= 0 || n_kv <= 0 || n_heads % n_kv || head_dim <= 0 || head_dim % 32 ||
        head_dim > 256 || n_seqs <= 0 || pages_per_seq <= 0 || page_size <= 0 || act_type < HQ4_F32 ||
        act_type > HQ4_F16)
        return -1;
    const int sms = device_sms();
    if (sms <= 0) return -1;
    return pa_plan(act_type, n_rows, n_heads, n_kv, head_dim, n_seqs, pages_per_seq, page_size, sms).ws;
}

extern "C" int hq4_paged_attention(const void* q, int act_type, int n_rows, int n_heads, int n_kv, int head_dim,
                                   long long q_stride, const int* cu_rows, const int* lens, int n_seqs,
                                   const int* pages, int pages_per_seq, const void* k_cache, const void* v_cache,
                                   int cache_type, int n_pages, int page_size, long long page_stride, float scale,
                                   void* out, void* workspace, long long workspace_bytes, void* stream) {
    return paged_attention(q, act_type, n_rows, n_heads, n_kv, head_dim, q_stride, cu_rows, lens, n_seqs, pages,
                           pages_per_seq, k_cache, v_cache, cache_type, n_pages, page_size, page_stride, nullptr, 0,
                           scale, out, workspace, workspace_bytes, stream);
}

extern "C" int hq4_tree_attention(const void* q, int act_type, int n_rows, int n_heads, int n_kv, int head_dim,
                                  long long q_stride, const int* cu_rows, const int* lens, int n_seqs,
                                  const int* pages, int pages_per_seq, const void* k_cache, const void* v_cache,
                                  int cache_type, int n_pages, int page_size, long long page_stride,
                                  const uint32_t* tree_mask, int mask_words, float scale, void* out, void* workspace,
                                  long long workspace_bytes, void* stream) {
    if (!tree_mask || mask_words <= 0) return HQ4_ERR_SHAPE;
    return paged_attention(q, act_type, n_rows, n_heads, n_kv, head_dim, q_stride, cu_rows, lens, n_seqs, pages,
                           pages_per_seq, k_cache, v_cache, cache_type, n_pages, page_size, page_stride, tree_mask,
                           mask_words, scale, out, workspace, workspace_bytes, stream);
}
