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

// 16-bit activations with more than 8 rows to a sequence and key/value head on
// average (16 with heads of up to 64): the tensor-memory kernel, although that
// fills few of its 128 rows (16 sequences of 16 rows, heads of 128, 1000
// entries: 31 against 38 us, 8000 entries: 115 against 129; of 8 rows, 8000
// entries: 115 against 101.  Heads of 64, 8000 entries: 101 against 78 with 16
// rows, 102 against 121 with 24).  Else the warp-level kernel with tiles of 8,
// 16 or 32 rows (16 at most for wide heads, whose outputs fill the registers).
// The average decides for all sequences of a call: 60 decode rows beside a chunk
// of 2000 tokens, 28 heads over 4, 144 us (75 and 86 in two calls); 512 beside
// 2000, 16 heads over 16, 1164 us (532 and 68).
//
// Split over keys when a sequence may be longer than 512 entries (1024): up to
// there items are a CTA's work whole, and need no second kernel.  One stream of
// 256 entries: whole 10.4 us, split 11.6; of 1024: 26 and 13; 64 streams of 512:
// 33 and 40; 8 chunks of 32 tokens, 1024 entries: 22 and 32, 2048: 36 and 37.
static PaPlan pa_plan(int act_type, int n_rows, int n_heads, int n_kv, int head_dim, int n_seqs, int pages_per_seq,
                      int page_size, int sms) {
    PaPlan r;
    const long long group = n_heads / n_kv;
    const long long avg = ((long long)n_rows + n_seqs - 1) / n_seqs * group;
    r.dim = head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
    r.tc = act_type != HQ4_F32 && avg > (r.dim == 64 ? 16 : 8);
    r.nt = avg <= 8 ? 1 : avg <= 16 || r.dim == 256 ? 2 : 4;
    const int rows = !r.tc ? 8 * r.nt : r.dim == 256 ? 128 : 256;
    const int keys = !r.tc ? kPaKeys : r.dim == 256 ? 64 : 128;
    const long long cap = (long long)pages_per_seq * page_size;
    const long long items = ((long long)n_rows * group / rows + n_seqs) * n_kv;  // at most
    r.split = cap > (r.tc ? 1024 : 512);
    // CTAs of an SM: as many as its shared memory holds (rings, and the queries' terms); registers hold as many.
    auto per_sm_of = [&](int warps) {
        const int ring = (r.dim == 64 ? 4 : 3) * 2 * kPaKeys * r.dim * 2, terms = act_type != HQ4_F32 ? 1 : 3;
        return std::max(1, 227 * 1024 / (warps * ring + terms * rows * r.dim * 2 + 2048));
    };
    // Two warps to a CTA, and more CTAs, where a CTA's work is waiting for one short item after the other, or
    // where four warps' rings of wide heads leave an SM one CTA (58 streams of 58 to 149 entries, 8 heads of 192:
    // 32 us, with four warps 45); four where items are few, each then taking less time.
    int per_sm = r.tc ? 1 : per_sm_of(4);
    r.warps = !r.tc && r.nt == 1 && items > (long long)sms * per_sm && (!r.split || r.dim == 256) ? 2 : 4;
    if (r.warps == 2) per_sm = per_sm_of(2);
    const long long units = r.split ? items * ((cap + keys - 1) / keys) : items;
    r.ctas = (int)std::min<long long>(units, (long long)sms * per_sm);
    // what an item costs besides its tiles, in tiles, where a CTA has many: with it 64 streams of 100 to 8200
    // entries decode in 117 us, without it in 137 (16 drafted trees: 83 and 109 us)
    r.extra = units < 8ll * r.ctas ? 0 : r.tc ? 4 : 18;
    r.join = (int)std::min<long long>(rows, n_rows * group);
    // joining an item of many pieces is a long walk for a warp, and there are few such items; else fewer and larger
    // CTAs do (a tree of 26 after 1001 entries, 4 heads: 18.6 us with 4 rows to a CTA, 24.5 with 16; 16 trees of 64:
    // 86 and 77)
    r.take = !r.tc ? 1 : items * 4 <= r.ctas ? 4 : 16;
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
    const long long q_row = (long long)n_heads * head_dim;
    const int elem = act_type == HQ4_F32 ? 4 : 2;
    const long long page = (long long)n_kv * page_size * head_dim;
    auto overlaps_inputs = [&](const void* to, long long bytes) {
        return rows_overlap(q, n_rows, q_stride, q_row, elem, to, bytes) ||
               rows_overlap(k_cache, n_pages, page_stride, page, 2, to, bytes) ||
               rows_overlap(v_cache, n_pages, page_stride, page, 2, to, bytes);
    };
    if (overlaps_inputs(out, n_rows * q_row * elem)) return HQ4_ERR_SHAPE;
    if (int rc = check_device_cap()) return rc;
    p.b.status = status_word();
    const int sms = device_sms();
    if (!p.b.status || sms <= 0) return HQ4_ERR_LAUNCH;
    const PaPlan pl = pa_plan(act_type, n_rows, n_heads, n_kv, head_dim, n_seqs, pages_per_seq, page_size, sms);
    if (pl.ws) {
        if (!workspace || workspace_bytes < pl.ws) return HQ4_ERR_SHAPE;
        if ((uintptr_t)workspace & 127) return HQ4_ERR_ALIGN;
        if (overlaps_inputs(workspace, pl.ws) || rows_overlap(workspace, 1, pl.ws, pl.ws, 1, out, n_rows * q_row * elem))
            return HQ4_ERR_SHAPE;
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
    p.take = pl.take;
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
