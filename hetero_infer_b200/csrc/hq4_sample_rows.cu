// Sampling a token for each row of a batch: temperature, top-k, top-p, min-p
// and the draw for given random numbers.
//
// With the entries in descending order (equal values by index), each filter
// keeps a beginning of that order, so the kept set is what the shortest one
// keeps, and the draw walks it in index order.  Nothing is sorted: a cluster of
// CTAs holds a row in shared memory (read from memory once), and the value at
// which a filter ends is found by a radix search.  Its keys are the distances
// below the maximum in 2^12 equal steps over the 43.9 octaves that have mass -- a
// monotone function of the value whose digits, unlike the float's own, split a
// row evenly.  A first digit's sums are taken in columns of shared memory, one
// to a thread or two; the second's, of the entries that the first leaves, by
// shared-memory atomics; the entries of the last step are compared with one
// another.  Where top-k keeps few entries, those alone are compared, and all
// the rest of the work is theirs.
//
// What bounds it is neither memory (64 rows of 152064 fp32 are 6 us of it) nor
// the issue rate, but how few warps an SM has beside the slices (16, which fill
// 47% of the slots), with a cluster barrier of about 0.8 us between the steps.
// 64 such rows take 14 us greedy, 43 with top-k 50, 51 without filters, 33 with
// min-p 0.05 and 113 with top-p 0.9; one row 6, 19, 15, 10 and 23.
//
// Masses are integers of 2^-44 of the maximum's or so, and 0 below that: each is
// good to 3e-9 of itself (see mass()) and cut off to such an integer, which is
// much of a mass of a few.  Their sums are exact, so the token does not depend on
// how the work is divided, and rounding errors of fp32 sums over 1.5e5 entries,
// 1e-6 of the whole, which would move tokens, do not arise.
//
// A thread owns a run of consecutive entries, so its columns above the end that
// is found add up to what its run (or its pair's) contributes to the draw, and
// only the thread in whose run the draw falls looks at single entries again.
#include <algorithm>

#include "hq4_host.cuh"
#include "hq4_min_p.cuh"
#include "hq4_paged.cuh"

namespace hq4 {

int check_device_cap();
int* status_word();

constexpr int kSrBits = 12;              // of the search's keys
constexpr float kSrSteps = 4096.0f;
constexpr double kSrOctaves = 43.9;      // that have mass (at least 1)
constexpr int kSrList = 128;             // entries of a CTA that are compared directly
constexpr int kSrFew = 384;              // entries of a row that top-k may leave for that
constexpr int kSrMaxCluster = 8;
constexpr int kSrMaxSlice = 36864;       // entries of a CTA of the longest row
constexpr int kSrMaxRun = 192;           // entries of a thread at most: a bit each (SampleRow::Chosen)
// Entries of a thread: odd, which spreads a warp over the banks.
__host__ __device__ constexpr int sr_run(int slice, int threads) { return ((slice + threads - 1) / threads) | 1; }
// Bytes of the first digit's sums, and of the lists that take their place.
constexpr size_t sr_hist_bytes(int cols, int bits) {
    const size_t sums = (sizeof(unsigned long long) << bits) * cols;
    const size_t lists = 3 * sizeof(unsigned long long) * kSrMaxCluster * kSrList;
    return sums > lists ? sums : lists;
}
// Dynamic shared memory at most, by the bits of the first digit (the lists and sums take the rest).
constexpr size_t sr_smem_max(int bits) { return (bits == 5 ? 204 : 196) * 1024; }

struct SampleRowsParams {
    const void* x;
    long long stride;
    int n, chunk;  // chunk: entries of a CTA
    const float* temperature;
    const int* top_k;
    const float *top_p, *min_p;
    const double* u;
    int* tok;
    float* logp;
    int* status;
};

typedef unsigned long long u64;

__device__ __forceinline__ void st_cluster_u64(uint32_t addr, u64 v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
// B1: bits of the first digit.
template <int T, int B1>
struct SampleRowsShared {
    static constexpr int kBins1 = 1 << B1, kBins2 = 1 << (kSrBits - B1);
    uint32_t table[64];                  // 2^30 * 2^(1 - j / 64), and below 2^31
    u64 all1[2][kSrMaxCluster][kBins1];  // the CTAs' sums of a digit; by turns for the two searches
    u64 all2[kSrMaxCluster][kBins2];
    uint32_t part[3][kBins2];            // this CTA's of the second digit: 15 bits of the masses each, or counts
    u64 warp[T / 32];
    u64 pair[2][kSrMaxCluster];          // a number of each CTA, by turns
    uint32_t key[kSrMaxCluster][kSrList], idx[kSrMaxCluster][kSrList];  // the CTAs' lists
    uint32_t count[kSrMaxCluster];
    uint32_t n_list, best;
    u64 best_above, target, before, here;
    int bin;
};

// kCols: columns of mass sums, T or T / 2 (two threads to one then, by turns: less shared memory, so that a long
// row's slice leaves room for 512 threads).
template <class E, int T, int B1, int kCols>
struct SampleRow {
    typedef SampleRowsShared<T, B1> Shared;
    static constexpr int kBins1 = Shared::kBins1, kBins2 = Shared::kBins2, kB2 = kSrBits - B1;
    static constexpr bool kPairs = kCols < T;
    static_assert(kCols == T || kCols == T / 2, "a thread or two to a column");
    Shared& sh;
    u64* hist;         // [kBins1][kCols]; once a search is at its list, that list
    const E* xs;       // this CTA's slice
    int lo, a, b, run; // its first entry in the row; the thread's run in it, and a run's entries
    int rank, nr, turn, pturn;
    float top, steps;  // the maximum; steps of the search's keys for a unit of x
    float oct, oct_lo; // octaves for a unit of x, as a sum of two
    float shift;       // 0, or the maximum where that is far from 0
    int top_q;         // the maximum's 64ths of an octave, as mass() has them

    __device__ __forceinline__ u64* list_mass() const { return hist; }
    __device__ __forceinline__ u64* list_above() const { return hist + kSrMaxCluster * kSrList; }
    // order bits, then the index inverted: of two entries the one that comes first is the larger
    __device__ __forceinline__ u64* list_entry() const { return hist + 2 * kSrMaxCluster * kSrList; }
    __device__ __forceinline__ float at(int i) const { return Elem<E>::to(xs[i]); }

    // Sum over the cluster; every thread gets it, and the sum of lower ranks.
    __device__ u64 cluster_sum(u64 v, u64* lower = nullptr) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) sh.warp[threadIdx.x >> 5] = v;
        __syncthreads();
        if ((int)threadIdx.x < nr) {
            u64 t = 0;
            for (int w = 0; w < T / 32; w++) t += sh.warp[w];
            st_cluster_u64(map_to_rank(smem_u32(&sh.pair[pturn][rank]), threadIdx.x), t);
        }
        cluster_sync();
        u64 t = 0, low = 0;
        for (int r = 0; r < nr; r++) {
            if (r < rank) low += sh.pair[pturn][r];
            t += sh.pair[pturn][r];
        }
        pturn ^= 1;
        if (lower) *lower = low;
        return t;
    }
    // Sum over the CTA's threads before this one.
    __device__ u64 cta_before(u64 v) {
        u64 inc = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 y = __shfl_up_sync(0xffffffffu, inc, o);
            if ((threadIdx.x & 31) >= o) inc += y;
        }
        __syncthreads();
        if ((threadIdx.x & 31) == 31) sh.warp[threadIdx.x >> 5] = inc;
        __syncthreads();
        u64 before = inc - v;
        for (int w = 0; w < (int)(threadIdx.x >> 5); w++) before += sh.warp[w];
        return before;
    }
    __device__ u64 cta_sum(u64 v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) sh.warp[threadIdx.x >> 5] = v;
        __syncthreads();
        u64 t = 0;
        for (int w = 0; w < T / 32; w++) t += sh.warp[w];
        return t;
    }
    __device__ uint32_t cluster_max(uint32_t v) {  // of 32-bit numbers
        v = __reduce_max_sync(0xffffffffu, v);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) sh.warp[threadIdx.x >> 5] = v;
        __syncthreads();
        if ((int)threadIdx.x < nr) {
            u64 t = 0;
            for (int w = 0; w < T / 32; w++) t = max(t, sh.warp[w]);
            st_cluster_u64(map_to_rank(smem_u32(&sh.pair[pturn][rank]), threadIdx.x), t);
        }
        cluster_sync();
        u64 t = 0;
        for (int r = 0; r < nr; r++) t = max(t, sh.pair[pturn][r]);
        pturn ^= 1;
        return (uint32_t)t;
    }
    // The search's key of x, at least kSrSteps for an entry without mass.
    __device__ __forceinline__ float key(float x) const { return (top - x) * steps; }
    __device__ __forceinline__ bool has_mass(float x) const { return key(x) < kSrSteps; }
    // The mass of an entry that has some, in fp32 and 32-bit integer
    // arithmetic (fp64 is several times slower).  x * oct is Q / 64 + g: its
    // product as a sum of two floats (a fused multiply-add gives the rounding
    // error), Q the nearest integer (left in the low bits by adding 1.5 * 2^23),
    // |g| <= 9.3e-3 (2^-7, and of |x * oct| < 16000 what z does not hold: 5e-4,
    // and x * oct_lo: 1e-3); 2^g - 1 is three terms of its series (the fourth is
    // below 8e-11), at most 6.5e-3, as an integer of 2^-29 (9e-10; it fits the
    // 22 bits that the addition rounds to, up to 7.8e-3); 2^(Q/64) comes from a
    // table and a shift.  With their roundings a mass is good to 3e-9 (2.8e-9
    // over 8 million values).  The maximum's own g is left in all masses alike,
    // which changes no ratio: they are up to 2^(1/64) times 2^44.
    __device__ __forceinline__ u64 mass(float x) const {
        x -= shift;
        const float z = x * oct;
        const float zl = fmaf(x, oct_lo, fmaf(x, oct, -z));
        const float q = fmaf(z, 64.0f, 12582912.0f);
        const float g = fmaf(q - 12582912.0f, -0.015625f, z) + zl;
        const float m = g * fmaf(g, fmaf(g, 5.5504109e-2f, 2.4022651e-1f), 6.9314718e-1f);
        const int mi = __float_as_int(fmaf(m, 536870912.0f, 12582912.0f)) - 0x4b400000;
        const int Q = top_q - (int)__float_as_uint(q);  // 64ths of an octave below the maximum
        const uint32_t w = sh.table[Q & 63];            // 2^30 to 2^31
        return ((u64)(w + __mulhi((int)w, mi << 3)) << 32) >> ((19 + (Q >> 6)) & 63);
    }
    // use(x, w, i) of the run's entries, six at a time, so that their arithmetic
    // overlaps: first `pick` chooses, then the masses of the six are worked
    // out, then `use` gets those of the chosen ones in order.
    template <class Pick, class Use>
    __device__ __forceinline__ void masses(bool counting, Pick pick, Use use) const {
        constexpr int kW = 6;  // (4: 8% slower, 8: as 6)
        for (int i = a; i < b; i += kW) {
            float x[kW];
            bool on[kW], any = false;
            u64 w[kW];
#pragma unroll
            for (int j = 0; j < kW; j++) x[j] = i + j < b ? at(i + j) : -INFINITY;
#pragma unroll
            for (int j = 0; j < kW; j++) any |= on[j] = pick(x[j]);
            if (!any) continue;
#pragma unroll
            for (int j = 0; j < kW; j++) w[j] = counting ? 1 : mass(x[j]);
#pragma unroll
            for (int j = 0; j < kW; j++)
                if (on[j]) use(x[j], w[j], i + j);
        }
    }

    // Which entries of the run `pick` chooses, a bit each; and use(x, w, i) of
    // those, four at a time.  A warp's lanes then spend their masses on chosen
    // entries alone, where masses() works them out for all six whenever any
    // lane has chosen one.
    struct Chosen {
        u64 bits[kSrMaxRun / 64];
    };
    template <class Pick>
    __device__ __forceinline__ Chosen choose(Pick pick) const {
        Chosen c;
#pragma unroll
        for (int w = 0; w < kSrMaxRun / 32; w++) {
            uint32_t m = 0;
            const int i0 = a + 32 * w, n = min(32, b - i0);
            for (int t = 0; t < n; t += 4)
#pragma unroll
                for (int j = 0; j < 4; j++) m |= (uint32_t)pick(t + j < n ? at(i0 + t + j) : -INFINITY) << (t + j);
            if (w & 1) c.bits[w / 2] |= (u64)m << 32;
            else c.bits[w / 2] = m;
        }
        return c;
    }
    template <class Use>
    __device__ __forceinline__ void masses_of(const Chosen& c, bool counting, Use use) const {
#pragma unroll
        for (int k = 0; k < kSrMaxRun / 64; k++)
            for (u64 m = c.bits[k]; m;) {
                int i[4];
                float x[4];
                bool on[4];
                u64 w[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    on[j] = m != 0;
                    i[j] = a + 64 * k + (on[j] ? __ffsll(m) - 1 : 0);
                    m &= m - 1;  // (0 stays 0)
                    x[j] = at(i[j]);
                }
#pragma unroll
                for (int j = 0; j < 4; j++) w[j] = counting ? 1 : mass(x[j]);
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (on[j]) use(x[j], w[j], i[j]);
            }
    }

    // The bin among n (the cluster's sums in all[r][.]) that is the last to
    // begin below the target, with what lies before it and in it; `base` is
    // what lies before the first.  Thread i < n looks after bin i.
    template <int kBins>
    __device__ int find_bin(const u64 (*all)[kBins], u64 base, u64 target, u64& before, u64& here) {
        static_assert(kBins <= T, "a bin to a thread");
        u64 v = 0;
        if ((int)threadIdx.x < kBins)
            for (int r = 0; r < nr; r++) v += all[r][threadIdx.x];
        if (threadIdx.x == 0) sh.bin = 0;
        const u64 excl = base + cta_before(v);  // (has barriers)
        const bool ok = v != 0 && excl < target;
        const uint32_t any = __ballot_sync(0xffffffffu, ok);
        if (any && (threadIdx.x & 31) == 31 - __clz(any)) atomicMax(&sh.bin, (int)threadIdx.x);
        __syncthreads();
        const int bin = sh.bin;
        if ((int)threadIdx.x == bin) {
            sh.before = excl;
            sh.here = v;
        }
        __syncthreads();
        before = sh.before;
        here = sh.here;
        return bin;
    }

    // Where a filter ends.
    struct End {
        float v;        // the value, once it is known
        u64 above;      // what the entries above it weigh (each its mass, or one)
        u64 mine;       // mass above the value's step: (a pair's: of both runs)
        int step;       // that step
        int i0, i1;     // the entries of the run in that step lie in [i0, i1)
        bool listed;    // not resolved: the list holds all entries down to that step,
        int n;          // so many
    };
    // The smallest value v >= floor of an entry with mass such that the entries
    // above it weigh less than the target.  The target is `count`, or, of the
    // masses, share times `whole` (of all masses where that is 0), at least 1,
    // so that there is such a value.
    __device__ End find_end(bool counting, u64 count, double share, u64 whole, float floor) {
        End e = {};
        // first digit
        const bool odd = threadIdx.x & 1;  // (of a pair)
        uint32_t* const counts = reinterpret_cast<uint32_t*>(hist) + threadIdx.x;  // a column to every thread
        u64* const sums = hist + (kPairs ? threadIdx.x >> 1 : threadIdx.x);
        auto bin_of = [&](float x) { return (int)key(x) >> kB2; };
        auto in = [&](float x) { return has_mass(x) && x >= floor; };
        if (counting) {
#pragma unroll
            for (int i = 0; i < kBins1; i++) counts[i * T] = 0;
            masses(true, in, [&](float x, u64, int) { counts[bin_of(x) * T]++; });
        } else {
            if (!kPairs || !odd)
#pragma unroll
                for (int i = 0; i < kBins1; i++) sums[i * kCols] = 0;
            if constexpr (!kPairs) {
                masses(false, in, [&](float x, u64 w, int) { sums[bin_of(x) * kCols] += w; });
            } else {
                for (int i = 0; i < run; i += 6) {  // (all lanes alike)
                    float x[6];
                    u64 w[6];
#pragma unroll
                    for (int j = 0; j < 6; j++) {
                        x[j] = a + i + j < b ? at(a + i + j) : -INFINITY;
                        w[j] = mass(x[j]);
                    }
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        __syncwarp();
                        if (odd == (half == 1))
#pragma unroll
                            for (int j = 0; j < 6; j++)
                                if (in(x[j])) sums[bin_of(x[j]) * kCols] += w[j];
                    }
                }
            }
        }
        for (int i = threadIdx.x; i < 3 * kBins2; i += T) sh.part[0][i] = 0;
        __syncthreads();
        const int lane = threadIdx.x & 31;
        for (int i = threadIdx.x >> 5; i < kBins1; i += T / 32) {
            u64 v = 0;
            if (counting)
#pragma unroll
                for (int j = 0; j < T / 32; j++) v += reinterpret_cast<uint32_t*>(hist)[i * T + j * 32 + lane];
            else
#pragma unroll
                for (int j = 0; j < kCols / 32; j++) v += hist[i * kCols + j * 32 + lane];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
            if (lane < nr) st_cluster_u64(map_to_rank(smem_u32(&sh.all1[turn][rank][i]), lane), v);
        }
        cluster_sync();
        u64 target = count, before, here;
        if (!counting) {
            u64 all = whole;
            if (!all)
                for (int i = lane; i < kBins1 * nr; i += 32) all += sh.all1[turn][i / kBins1][i % kBins1];
            if (!whole)
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
            const double want = ceil(share * (double)all);
            target = want >= 1.0 ? (u64)want : 1;
        }
        const int bin1 = find_bin<kBins1>(sh.all1[turn], 0, target, before, here);
        turn ^= 1;
        if (!counting && (!kPairs || !odd))
            for (int i = 0; i < bin1; i++) e.mine += sums[i * kCols];
        // second digit, of the entries that have the first
        const float k_lo = (float)(bin1 << kB2), k_hi = (float)((bin1 + 1) << kB2);
        const bool all_few = counting && before + here <= kSrFew;  // all down to that digit are few: they are chosen
        const Chosen chosen = choose([&](float x) {
            const float k = key(x);
            return (all_few || k >= k_lo) && k < k_hi && x >= floor;
        });
        masses_of(chosen, counting,
               [&](float x, u64 w, int) {
                   if (all_few && key(x) < k_lo) return;
                   const int i = (int)key(x) & (kBins2 - 1);
                   atomicAdd(&sh.part[0][i], (uint32_t)w & 0x7fffu);
                   if (!counting) {
                       atomicAdd(&sh.part[1][i], (uint32_t)(w >> 15) & 0x7fffu);
                       atomicAdd(&sh.part[2][i], (uint32_t)(w >> 30));
                   }
               });
        if (threadIdx.x == 0) {
            sh.n_list = 0;
            sh.best = 0xffffffffu;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < kBins2 * nr; i += T) {
            const int k = i & (kBins2 - 1);
            st_cluster_u64(map_to_rank(smem_u32(&sh.all2[rank][k]), i >> kB2),
                           (u64)sh.part[0][k] + ((u64)sh.part[1][k] << 15) + ((u64)sh.part[2][k] << 30));
        }
        cluster_sync();
        const u64 base = before;
        const int bin2 = find_bin<kBins2>(sh.all2, base, target, before, here);
        e.step = bin1 << kB2 | bin2;
        // the entries of the last step; or, where top-k ends early, all down to it
        const bool few = counting && before + here <= kSrFew;
        e.i0 = e.i1 = 0;
        const float k_end = (float)(e.step + 1);
        auto take = [&](float x, u64 w, int i) {
            if (!(key(x) < k_end)) return;
            if (!few && (int)key(x) < e.step) {
                e.mine += w;
                return;
            }
            if (e.i1 == 0) e.i0 = i;
            e.i1 = i + 1;
            const uint32_t place = atomicAdd(&sh.n_list, 1);
            if (place < kSrList) {
                sh.key[rank][place] = order_bits(x + 0.0f);  // -0 counts as 0
                sh.idx[rank][place] = lo + i;
            }
        };
        if (few && !all_few) masses(true, [&](float x) { return key(x) < k_end && x >= floor; }, take);
        else masses_of(chosen, counting, take);
        if (counting) e.mine = 0;
        __syncthreads();
        const uint32_t n_mine = sh.n_list;
        for (int i = threadIdx.x; i < (int)min(n_mine, (uint32_t)kSrList) * nr; i += T) {
            const int k = i / nr, r = i - k * nr;
            if (r == rank) continue;
            st_cluster_u32(map_to_rank(smem_u32(&sh.key[rank][k]), r), sh.key[rank][k]);
            st_cluster_u32(map_to_rank(smem_u32(&sh.idx[rank][k]), r), sh.idx[rank][k]);
        }
        if ((int)threadIdx.x < nr) st_cluster_u32(map_to_rank(smem_u32(&sh.count[rank]), threadIdx.x), n_mine);
        cluster_sync();
        bool fits = true;
        int n_all = 0;
        for (int r = 0; r < nr; r++) {
            fits = fits && sh.count[r] <= kSrList;
            n_all += (int)sh.count[r];
        }
        if (fits) {
            // one list of all CTAs', in every CTA alike
            for (int i = threadIdx.x; i < n_all; i += T) {
                int r = 0, j = i;
                while (j >= (int)sh.count[r]) j -= (int)sh.count[r++];
                const uint32_t k = sh.key[r][j];
                list_entry()[i] = (u64)k << 32 | ~sh.idx[r][j];
                list_mass()[i] = counting && !few ? 1 : mass(order_value(k));
            }
            __syncthreads();
            e.n = n_all;
            if (few) {
                e.listed = true;
                return e;
            }
            for (int i = threadIdx.x; i < n_all; i += T) {
                const uint32_t k = (uint32_t)(list_entry()[i] >> 32);
                u64 w = before;
#pragma unroll 8
                for (int j = 0; j < n_all; j++)
                    if ((uint32_t)(list_entry()[j] >> 32) > k) w += list_mass()[j];
                list_above()[i] = w;
                if (w < target) atomicMin(&sh.best, k);
            }
            __syncthreads();
            for (int i = threadIdx.x; i < n_all; i += T)
                if ((uint32_t)(list_entry()[i] >> 32) == sh.best) sh.best_above = list_above()[i];
            __syncthreads();
            e.v = order_value(sh.best);
            e.above = sh.best_above;
            __syncthreads();
            return e;
        }
        // many entries within one step (equal ones, or a high temperature): bisection over their order
        e.i0 = a;
        e.i1 = b;
        uint32_t low = 0xffffffffu, high = 0;
        auto in_step = [&](float x) { return has_mass(x) && x >= floor && (int)key(x) == e.step; };
        for (int i = a; i < b; i++) {
            const float x = at(i);
            if (!in_step(x)) continue;
            low = min(low, order_bits(x + 0.0f));
            high = max(high, order_bits(x + 0.0f));
        }
        low = ~cluster_max(~low);
        high = cluster_max(high);  // low <= the end <= high
        e.above = before;
        while (low < high) {
            const uint32_t mid = low + ((high - low) >> 1);
            const float v = order_value(mid);
            u64 w = 0;
            masses(counting, [&](float x) { return in_step(x) && x > v; }, [&](float, u64 m, int) { w += m; });
            w = before + cluster_sum(w);
            if (w < target) {
                high = mid;
                e.above = w;
            } else {
                low = mid + 1;
            }
        }
        e.v = order_value(low);
        return e;
    }
};

// The place in [0, total) that u falls on.
__device__ __forceinline__ u64 draw_place(double u, u64 total) {
    const double want = (u > 0.0 ? u : 0.0) * (double)total;
    return want >= (double)total ? total - 1 : (u64)want;
}
// The log of 2^((x - max) oct) over the total; the maximum's mass says what the total is counted in.
template <class Row>
__device__ __forceinline__ float log_prob(float x, const Row& s, double oct, u64 total) {
    return (float)(-((double)s.top - (double)x) * oct * 0.6931471805599453094 - log((double)total / (double)s.mass(s.top)));
}

template <class E, int T, int B1, int kCols>
__global__ void __launch_bounds__(T, 512 / T) sample_rows_kernel(const SampleRowsParams p) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ SampleRowsShared<T, B1> sh;
    pdl_launch_dependents();
    if (threadIdx.x < 64) sh.table[threadIdx.x] = (uint32_t)fmin(exp2(31.0 - threadIdx.x / 64.0) + 0.5, 2147483647.0);
    pdl_wait();
    const int rank = (int)cluster_ctarank(), nr = (int)cluster_nctarank();
    const int row = blockIdx.x / nr;
    const int lo = min(p.n, rank * p.chunk), cnt = min(p.n, lo + p.chunk) - lo;
    const E* src = static_cast<const E*>(p.x) + (long long)row * p.stride + lo;
    constexpr int kV = 16 / sizeof(E);
    const int off = (int)((uintptr_t)src & 15) / (int)sizeof(E);  // the slice keeps the row's alignment
    E* xs = reinterpret_cast<E*>(smem + sr_hist_bytes(kCols, B1)) + off;

    // ---- the slice, all copies in flight at once ---------------------------------
    const int head = min(cnt, (kV - off) % kV), vecs = (cnt - head) / kV;
    for (int i = threadIdx.x; i < vecs; i += T) cp_async16(smem_u32(xs + head + i * kV), src + head + i * kV, true);
    cp_async_commit();
    for (int i = threadIdx.x; i < head; i += T) xs[i] = src[i];
    for (int i = head + vecs * kV + threadIdx.x; i < cnt; i += T) xs[i] = src[i];
    const float temp = p.temperature ? p.temperature[row] : 1.0f;
    const int top_k = p.top_k ? p.top_k[row] : 0;
    const float top_p = p.top_p ? p.top_p[row] : 1.0f;
    const float min_p = p.min_p ? p.min_p[row] : 0.0f;
    const double u = p.u[row];
    cp_async_wait<0>();
    cluster_sync();  // the slice is there, and the cluster's other CTAs run: their shared memory can be written

    // ---- its largest entry, the first of its equals; NaN ---------------------------
    const int run = sr_run(cnt, T);
    SampleRow<E, T, B1, kCols> s{sh, reinterpret_cast<u64*>(smem), xs, lo, min(cnt, (int)threadIdx.x * run), 0, run, rank, nr,
                          0, 0, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0};
    s.b = min(cnt, s.a + run);
    uint32_t best = 0, first = 0x7fffffffu;  // order bits (of a NaN: all ones), index in the row
    if (temp > 0.0f) {
        float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        bool nan = false;
        int i = s.a;
        for (; i + 4 <= s.b; i += 4)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float x = s.at(i + j);
                nan |= x != x;
                m[j] = fmaxf(m[j], x);
            }
        for (; i < s.b; i++) {
            nan |= s.at(i) != s.at(i);
            m[0] = fmaxf(m[0], s.at(i));
        }
        best = nan ? 0xffffffffu : order_bits(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])) + 0.0f);
    } else {
        for (int i = s.a; i < s.b; i++) {
            const float x = s.at(i) + 0.0f;
            const uint32_t ob = x != x ? 0xffffffffu : order_bits(x);
            if (ob > best) {
                best = ob;
                first = lo + i;
            }
        }
    }
    const uint32_t top_bits = s.cluster_max(best);
    if (!(temp > 0.0f)) {
        first = ~s.cluster_max(best == top_bits ? ~first : 0u);
        if (rank == 0 && threadIdx.x == 0) {
            p.tok[row] = (int)first;
            if (p.logp) p.logp[row] = 0.0f;
        }
        return;
    }
    const float top = top_bits == 0xffffffffu ? NAN : order_value(top_bits);
    if (!(fabsf(top) < INFINITY)) {  // NaN, +inf, or nothing above -inf
        if (rank == 0 && threadIdx.x == 0) {
            p.tok[row] = p.n - 1;
            if (p.logp) p.logp[row] = NAN;
            if (p.status) atomicOr(p.status, 8);
        }
        return;
    }
    const double oct = 1.4426950408889634074 / (double)temp;
    s.top = top;
    s.oct = (float)fmin(oct, 1e30);
    s.oct_lo = (float)(fmin(oct, 1e30) - (double)s.oct);
    // a maximum of so many octaves (mass() says why): the entries within 44 of it are so near that their distance to it
    // is exact
    s.shift = fabs((double)top * oct) < 16000.0 ? 0.0f : top;
    s.top_q = (int)__float_as_uint(fmaf((top - s.shift) * s.oct, 64.0f, 12582912.0f));
    s.steps = fminf((float)(oct * (kSrSteps / kSrOctaves)), 1e30f);

    // ---- where the filters end ---------------------------------------------------
    float floor = -INFINITY;  // entries below are out
    int ties = 0x7fffffff;    // of the entries equal to tie, how many stay
    float tie = 0.0f;
    typename SampleRow<E, T, B1, kCols>::End e = {};
    bool summed = false;      // e.mine holds the thread's mass above e.step
    const float p_end = min_p > 0.0f ? min_p_end(min_p, top, oct) : -INFINITY;
    if (top_k > 0 && top_k < p.n) {
        e = s.find_end(true, (u64)top_k, 0.0, 0, floor);
        if (e.listed) {
            // ---- few entries: all of them against one another, in every CTA alike ------
            // ranks, and what lies above each; then the draw among those that stay
            u64 *above = s.list_above(), *mass = s.list_mass(), *entry = s.list_entry();
            u64 kept = 0;
            for (int i = threadIdx.x; i < e.n; i += T) {
                const u64 me = entry[i];
                u64 w = 0;
                int before = 0;
#pragma unroll 8
                for (int j = 0; j < e.n; j++) {
                    const u64 other = entry[j];
                    if ((uint32_t)(other >> 32) > (uint32_t)(me >> 32)) w += mass[j];
                    before += other > me ? 1 : 0;
                }
                above[i] = before >= top_k ? ~0ull : w;  // (never below a target)
                if (before < top_k) kept += mass[i];
            }
            u64 target = ~0ull;
            if (top_p < 1.0f) {
                const double want = ceil((double)top_p * (double)s.cta_sum(kept));
                target = want >= 1.0 ? (u64)want : 1;
            }
            __syncthreads();
            kept = 0;
            for (int i = threadIdx.x; i < e.n; i += T) {
                const float x = order_value((uint32_t)(entry[i] >> 32));
                if (!(above[i] < target) || x < p_end) mass[i] = 0;
                kept += mass[i];
            }
            const u64 total = s.cta_sum(kept);  // (its barriers: the masses are written)
            const u64 goal = draw_place(u, total);
            if (rank == 0)
                for (int i = threadIdx.x; i < e.n; i += T) {
                    const uint32_t me = (uint32_t)entry[i];
                    u64 c = 0;
#pragma unroll 8
                    for (int j = 0; j < e.n; j++)
                        if ((uint32_t)entry[j] > me) c += mass[j];  // a lower index
                    if (mass[i] && goal >= c && goal < c + mass[i]) {
                        p.tok[row] = (int)~me;
                        if (p.logp) p.logp[row] = log_prob(order_value((uint32_t)(entry[i] >> 32)), s, oct, total);
                    }
                }
            return;
        }
        floor = tie = e.v;
        ties = top_k - (int)e.above;
    }
    if (top_p < 1.0f) {
        u64 whole = 0;
        if (ties != 0x7fffffff) {  // the mass of those top_k, with of the equal last ones those that stay
            u64 m = 0, equal = 0;
            s.masses(false, [&](float x) { return x >= tie; },
                     [&](float x, u64 w, int) {
                         if (x == tie) equal++;
                         else m += w;
                     });
            equal = s.cluster_sum(equal);
            if ((u64)ties > equal) ties = (int)equal;  // all entries with mass stay
            whole = s.cluster_sum(m) + (u64)ties * s.mass(tie);
        }
        e = s.find_end(false, 0, (double)top_p, whole, floor);
        floor = e.v;
        summed = true;
    }
    if (p_end > floor) {
        floor = p_end;
        summed = false;
    }

    // ---- the draw, in index order --------------------------------------------------
    const bool tied = ties != 0x7fffffff && floor == tie;
    int tie_before = 0;  // entries equal to the tie before this run
    if (tied) {
        u64 eq = 0, lower;
        for (int i = s.a; i < s.b; i++) eq += s.at(i) == tie ? 1 : 0;
        s.cluster_sum(eq, &lower);
        tie_before = (int)(lower + s.cta_before(eq));
    }
    int seen = tie_before;
    // whether the next entry of the run stays (it is asked once for each, in order)
    auto stays = [&](float x) {
        if (x < floor || !s.has_mass(x)) return false;
        return !(tied && x == tie && seen++ >= ties);
    };
    u64 mine = 0;
    if (!summed) {
        s.masses(false, stays, [&](float, u64 w, int) { mine += w; });
    } else {  // what lies above the search's last step has been added up
        mine = e.mine;
        for (int i = e.i0; i < e.i1; i++) {
            const float x = s.at(i);
            if (s.has_mass(x) && (int)s.key(x) == e.step && stays(x)) mine += s.mass(x);
        }
        if constexpr (kCols < T) {  // a column is two threads': the first draws for both runs
            const u64 other = __shfl_xor_sync(0xffffffffu, mine, 1);
            const int end = __shfl_xor_sync(0xffffffffu, s.b, 1);
            mine = threadIdx.x & 1 ? 0 : mine + other;
            if (!(threadIdx.x & 1)) s.b = end;
        }
    }
    u64 lower;
    const u64 total = s.cluster_sum(mine, &lower);
    u64 c = lower + s.cta_before(mine);
    const u64 goal = draw_place(u, total);
    if (goal >= c && goal < c + mine) {  // one thread of the cluster
        seen = tie_before;
        for (int i = s.a; i < s.b; i++) {
            const float x = s.at(i);
            if (stays(x)) c += s.mass(x);
            if (c > goal) {
                p.tok[row] = lo + i;
                if (p.logp) p.logp[row] = log_prob(x, s, oct, total);
                break;
            }
        }
    }
}

template <class E, int T, int B1, int kCols>
static int launch_sample_rows(const SampleRowsParams& p, int rows, int cluster, size_t smem, cudaStream_t st) {
    auto kern = sample_rows_kernel<E, T, B1, kCols>;
    static PerDeviceOnce once;
    if (smem_opt_in(once, kern, (int)sr_smem_max(B1)) != cudaSuccess) return HQ4_ERR_LAUNCH;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)rows * cluster);
    lc.blockDim = dim3(T);
    lc.dynamicSmemBytes = smem;
    lc.stream = st;
    lc.attrs = attr;
    lc.numAttrs = 2;
    return cudaLaunchKernelEx(&lc, kern, p) == cudaSuccess ? HQ4_OK : HQ4_ERR_LAUNCH;
}

// How a row is divided: CTAs, their threads, bits of the first digit, columns
// of its mass sums.  A wave of rows costs its entries, at a rate that grows
// with an SM's warps (two CTAs also fill each other's barriers), and barriers
// and fixed steps.  Measured with top-p 0.9 (top-k 50): 1 row of 152064 fp32,
// 8 CTAs of 512 threads 20.5 us (15.8), 4 of 512 39 (19), 4 of 256 59; 64 such
// rows, 4 CTAs of 512 with a column to two threads 117 (42), 4 of 256 150 (56),
// 8 of 512 with one each 117 (74); 256 rows of 32003 bf16, 2 CTAs of 256 63
// (38), 1 of 512 66 (37), 4 of 256 97.
struct SrShape {
    int cluster, threads, bits, cols;
    size_t smem;
};

template <class E>
static int sample_rows(SampleRowsParams p, int rows, int sms, cudaStream_t st) {
    SrShape best = {0, 0, 0, 0, 0};
    double best_cost = 0.0;
    for (int cluster = kSrMaxCluster; cluster >= 1; cluster >>= 1) {
        if (cluster > 1 && p.n / cluster < 2048) continue;
        static const SrShape shapes[3] = {{0, 512, 5, 512, 0}, {0, 512, 4, 256, 0}, {0, 256, 4, 256, 0}};
        for (SrShape s : shapes) {
            s.cluster = cluster;
            s.smem = (size_t)((p.n + cluster - 1) / cluster + 16) * sizeof(E) + sr_hist_bytes(s.cols, s.bits);
            // (a slice of 16-bit entries that fits can be too long for 256 threads: 289 entries each of 73728)
            if (s.smem > sr_smem_max(s.bits) || sr_run((p.n + cluster - 1) / cluster, s.threads) > kSrMaxRun) continue;
            const int per_sm = std::max(1, std::min<int>(512 / s.threads, (int)((size_t)227 * 1024 / (s.smem + 32 * 1024))));
            const int at_once = std::max(1, sms * per_sm / cluster);
            const int waves = (rows + at_once - 1) / at_once;
            const int sharing = std::min(per_sm, (rows * cluster + sms - 1) / sms);  // CTAs of an SM
            const double rate = sharing > 1 ? 1.8 : s.threads > 256 ? 1.6 : 1.0;
            const double cost = waves * ((double)p.n / cluster / 512.0 * sharing / rate + 20.0 + 2.0 * cluster);
            if (!best.cluster || cost < best_cost) {
                best_cost = cost;
                best = s;
            }
        }
    }
    if (!best.cluster) return HQ4_ERR_SHAPE;
    p.chunk = (p.n + best.cluster - 1) / best.cluster;
    return best.bits == 5      ? launch_sample_rows<E, 512, 5, 512>(p, rows, best.cluster, best.smem, st)
         : best.threads == 512 ? launch_sample_rows<E, 512, 4, 256>(p, rows, best.cluster, best.smem, st)
                               : launch_sample_rows<E, 256, 4, 256>(p, rows, best.cluster, best.smem, st);
}

}  // namespace hq4

using namespace hq4;

extern "C" int hq4_sample_rows(const void* logits, int act_type, int n_rows, int n, long long row_stride,
                               const float* temperature, const int* top_k, const float* top_p, const float* min_p,
                               const double* u, int* tok, float* logprob, void* stream) {
    if (n_rows <= 0 || n <= 0 || n > kSrMaxCluster * kSrMaxSlice || row_stride < n || !logits || !u || !tok)
        return HQ4_ERR_SHAPE;
    if (n_rows > (1 << 27)) return HQ4_ERR_SHAPE;
    if (act_type != HQ4_F32 && act_type != HQ4_BF16 && act_type != HQ4_F16) return HQ4_ERR_SHAPE;
    if (((uintptr_t)logits & (act_type == HQ4_F32 ? 3 : 1)) || ((uintptr_t)u & 7) ||
        (((uintptr_t)temperature | (uintptr_t)top_k | (uintptr_t)top_p | (uintptr_t)min_p | (uintptr_t)tok |
          (uintptr_t)logprob) & 3))
        return HQ4_ERR_ALIGN;
    // what a row's clusters write, those of other rows do not read (a row's own parameter may lie where its result goes)
    const int elem = act_type == HQ4_F32 ? 4 : 2;
    const void* const outs[2] = {tok, logprob};
    const void* const params[5] = {temperature, top_k, top_p, min_p, tok};
    for (const void* out : outs) {
        if (!out) continue;
        const long long bytes = 4ll * n_rows;
        if (rows_overlap(logits, n_rows, row_stride, n, elem, out, bytes) || rows_overlap(u, n_rows, 1, 1, 8, out, bytes))
            return HQ4_ERR_SHAPE;
        for (const void* x : params)
            if (x && (x != out || (x == tok && out == logprob)) && rows_overlap(x, n_rows, 1, 1, 4, out, bytes))
                return HQ4_ERR_SHAPE;
    }
    if (int rc = check_device_cap()) return rc;
    SampleRowsParams p = {};
    p.x = logits;
    p.stride = row_stride;
    p.n = n;
    p.temperature = temperature;
    p.top_k = top_k;
    p.top_p = top_p;
    p.min_p = min_p;
    p.u = u;
    p.tok = tok;
    p.logp = logprob;
    p.status = status_word();
    const int sms = device_sms();
    if (sms <= 0) return HQ4_ERR_LAUNCH;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return act_type == HQ4_F32 ? sample_rows<float>(p, n_rows, sms, st)
         : act_type == HQ4_BF16 ? sample_rows<__nv_bfloat16>(p, n_rows, sms, st) : sample_rows<__half>(p, n_rows, sms, st);
}
