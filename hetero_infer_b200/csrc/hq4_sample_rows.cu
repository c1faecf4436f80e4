// Sampling a token for each row of a batch: temperature, top-k, top-p, min-p
// and the draw for given random numbers.
//
// With the entries in descending order (equal values by index), each filter
// keeps a beginning of that order, so the kept set is what the shortest one
// keeps, and the draw walks it in index order.  Nothing is sorted: a cluster of
// CTAs holds a row in shared memory (read from memory once), and the value at
// which a filter ends is found by a radix search.  Its keys are the distances
// below the maximum in 2^12 equal steps over the 44 octaves that have mass --
// a monotone function of the value whose digits, unlike the float's own, split
// a row evenly -- four bits at a time; the few entries of the last step are
// compared with one another.
//
// Masses are integers: w = 2^44 * 2^((x - max) / T * log2 e) rounded, from fp64
// arithmetic, at least 1, and 0 below 2^-44 of the maximum.  Their sums are
// exact, so the token does not depend on how the work is divided, and the
// cumulative bounds are off by less than 2^-40 of the whole, where fp32 sums
// over 1.5e5 entries would be off by 1e-6 and move tokens.
//
// A digit's 16 sums are taken in columns of shared memory, one to a thread
// (no atomics: equal addresses within a warp would queue), then over the
// threads and the cluster.  A thread owns a run of consecutive entries, so its
// columns above the end that is found add up to what its run contributes to
// the draw, and only the thread in whose run the draw falls looks at single
// entries again.
#include <algorithm>

#include "hq4_host.cuh"
#include "hq4_paged.cuh"

namespace hq4 {

int check_device_cap();
int* status_word();

constexpr int kSrDigit = 4;             // bits
constexpr int kSrBins = 1 << kSrDigit;
constexpr float kSrSteps = 4096.0f;    // of the search's keys
constexpr double kSrOctaves = 44.0;    // that have mass
constexpr int kSrList = 512;            // entries of one step that are compared directly
constexpr int kSrMaxCluster = 8;
constexpr int kSrMaxSlice = 36864;     // entries of a CTA
constexpr size_t kSrSmem = 212 * 1024;

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
__device__ __forceinline__ u64 ld_cluster_u64(uint32_t addr) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t atom_add_cluster(uint32_t addr, uint32_t v) {
    uint32_t r;
    asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(r) : "r"(addr), "r"(v) : "memory");
    return r;
}
// Bits that order as the floats do, and back.
__device__ __forceinline__ uint32_t order_bits(float x) {
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float order_value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

template <int T>
struct SampleRowsShared {
    u64 all[2][kSrMaxCluster][kSrBins];  // the CTAs' sums of a digit, by turns
    u64 sums[kSrBins];
    u64 warp[T / 32];
    u64 pair[2][kSrMaxCluster];          // a number of each CTA, by turns
    uint32_t list[kSrList];              // rank 0's: keys of one step's entries, and their weights
    u64 list_w[kSrList];
    u64 target;
    uint32_t n_list, best;
    u64 best_above;
    u64 bin_before;
    int bin;
};

template <class E, int T>
struct SampleRow {
    SampleRowsShared<T>& sh;
    u64* hist;         // [kSrBins][T]
    const E* xs;       // this CTA's slice
    int a, b;          // the thread's run in it
    int rank, nr, turn, pturn;
    float top, steps;  // the maximum; steps of the search's keys for a unit of x
    double oct;        // octaves for a unit of x
    double top_wide;   // the maximum

    __device__ __forceinline__ float at(int i) const { return Elem<E>::to(xs[i]) + 0.0f; }  // -0 counts as 0
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
        u64 t = 0, lo = 0;
        for (int r = 0; r < nr; r++) {
            if (r < rank) lo += sh.pair[pturn][r];
            t += sh.pair[pturn][r];
        }
        pturn ^= 1;
        if (lower) *lower = lo;
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
    static __device__ __forceinline__ double widen(float x) {
        const uint32_t b = __float_as_uint(x);
        return __hiloint2double((int)((b & 0x80000000u) | (((b & 0x7fffffffu) >> 3) + 0x38000000u)), (int)(b << 29));
    }
    // The mass of an entry that has some: 2^-z = 2^-n 2^-f with n the nearest
    // integer (left in the low bits by adding 1.5 * 2^52) and f in [-1/2, 1/2],
    // whose power is its Taylor series (the term left out is below 2e-10); the
    // last step scales it and rounds it to an integer in the low bits of 2^52.
    // Conversions between types would be slower than all of this: the fp64
    // value of x is put together from its bits (of a subnormal's or zero's,
    // 2^-127 or less, something as small).
    __device__ __forceinline__ u64 mass(float x) const {
        const double z = (top_wide - widen(x)) * oct;
        const double r = z + 6755399441055744.0;
        const double f = z - (r - 6755399441055744.0);
        const int n = __double2loint(r);
        // (-ln 2)^k / k!
        double s = 1.3215486790144307e-6;
        s = fma(s, f, -1.5252733804059841e-5);
        s = fma(s, f, 1.5403530393381609e-4);
        s = fma(s, f, -1.3333558146428443e-3);
        s = fma(s, f, 9.6181291076284772e-3);
        s = fma(s, f, -5.5504108664821580e-2);
        s = fma(s, f, 2.4022650695910071e-1);
        s = fma(s, f, -6.9314718055994531e-1);
        s = fma(s, f, 1.0);
        const double m = fma(s, __hiloint2double((1023 + 44 - n) << 20, 0), 4503599627370496.0);
        const u64 w = (u64)__double_as_longlong(m) & 0xfffffffffffffull;
        return w ? w : 1;
    }
    // f(x, i) of the run's entries four at a time, so that their arithmetic
    // overlaps: first `pick` chooses, then the masses of the four are worked
    // out, then `use` gets those of the chosen ones in order.
    template <class Pick, class Use>
    __device__ __forceinline__ void masses(bool counting, Pick pick, Use use) const {
        for (int i = a; i < b; i += 4) {
            float x[4];
            bool on[4];
            u64 w[4];
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] = i + j < b ? at(i + j) : -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; j++) on[j] = pick(x[j]);
            if (!(on[0] || on[1] || on[2] || on[3])) continue;
#pragma unroll
            for (int j = 0; j < 4; j++) w[j] = counting ? 1 : mass(x[j]);
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (on[j]) use(x[j], w[j]);
        }
    }
    __device__ __forceinline__ u64 weight(float x, bool counting) const { return counting ? 1 : mass(x); }

    // The order bits of the smallest value v >= floor of an entry with mass such that the
    // entries above it weigh less than the target (each its mass, or one), and
    // what those weigh.  The target is `count`, or, of the masses, share times
    // `whole` (of all masses where that is 0), at least 1, so that there is
    // such a value.  `mine` gets the masses of the thread's run above v's step;
    // `step` is that step.
    __device__ uint32_t find_end(bool counting, u64 count, double share, u64 whole, float floor, u64& above,
                                 u64& mine, int& step) {
        u64 target = count;
        u64 before = 0;  // weight of the entries above the searched range
        int prefix = 0;  // the key's digits so far
        mine = 0;
        for (int shift = 2 * kSrDigit; shift >= 0; shift -= kSrDigit) {
#pragma unroll
            for (int i = 0; i < kSrBins; i++) hist[i * T + threadIdx.x] = 0;
            masses(counting,
                   [&](float x) {
                       const float k = key(x);
                       return k < kSrSteps && x >= floor && (int)k >> (shift + kSrDigit) == prefix;
                   },
                   [&](float x, u64 w) { hist[((int)key(x) >> shift & (kSrBins - 1)) * T + threadIdx.x] += w; });
            __syncthreads();
            const int lane = threadIdx.x & 31;
            for (int i = threadIdx.x >> 5; i < kSrBins; i += T / 32) {
                u64 v = 0;
#pragma unroll
                for (int j = 0; j < T / 32; j++) v += hist[i * T + j * 32 + lane];
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
                if (lane < nr) st_cluster_u64(map_to_rank(smem_u32(&sh.all[turn][rank][i]), lane), v);
            }
            cluster_sync();
            if (threadIdx.x < 32) {  // a bin to a lane
                u64 v = 0;
                if (lane < kSrBins)
                    for (int r = 0; r < nr; r++) v += sh.all[turn][r][lane];
                u64 upto = v;
#pragma unroll
                for (int o = 1; o < kSrBins; o <<= 1) {
                    const u64 y = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += y;
                }
                if (!counting && shift == 2 * kSrDigit) {
                    const u64 all = whole ? whole : __shfl_sync(0xffffffffu, upto, kSrBins - 1);
                    const double want = ceil(share * (double)all);
                    target = want >= 1.0 ? (u64)want : 1;
                    if (lane == 0) sh.target = target;
                }
                const u64 excl = before + upto - v;
                const uint32_t ok = __ballot_sync(0xffffffffu, v != 0 && excl < target);
                const int i = ok ? 31 - __clz(ok) : 0;  // the last step that begins below the target
                if (lane == i) {
                    sh.bin = i;
                    sh.bin_before = excl;
                }
            }
            __syncthreads();
            turn ^= 1;
            if (!counting) target = sh.target;
            before = sh.bin_before;
            const int bin = sh.bin;
            if (!counting)
                for (int i = 0; i < bin; i++) mine += hist[i * T + threadIdx.x];
            prefix = prefix << kSrDigit | bin;
        }
        step = prefix;
        // the entries of the last step
        if (threadIdx.x == 0) {
            sh.n_list = 0;
            sh.best = 0xffffffffu;
        }
        cluster_sync();
        const uint32_t head = map_to_rank(smem_u32(&sh.n_list), 0);
        uint32_t low = 0xffffffffu, high = 0;
        for (int i = a; i < b; i++) {
            const float x = at(i), k = key(x);
            if (!(k < kSrSteps) || (int)k != prefix || x < floor) continue;
            const uint32_t ob = order_bits(x);
            low = min(low, ob);
            high = max(high, ob);
            const uint32_t place = atom_add_cluster(head, 1);
            if (place < kSrList) st_cluster_u32(map_to_rank(smem_u32(&sh.list[place]), 0), ob);
        }
        cluster_sync();
        const uint32_t n = (uint32_t)ld_cluster_u32(head);
        if (n <= kSrList) {
            if (rank == 0) {
                for (uint32_t i = threadIdx.x; i < n; i += T) sh.list_w[i] = weight(order_value(sh.list[i]), counting);
                __syncthreads();
                for (uint32_t i = threadIdx.x; i < n; i += T) {
                    const uint32_t key_i = sh.list[i];
                    u64 w = before;
                    for (uint32_t j = 0; j < n; j++)
                        if (sh.list[j] > key_i) w += sh.list_w[j];
                    if (w < target) atomicMin(&sh.best, key_i);
                }
                __syncthreads();
                const uint32_t v = sh.best;
                u64 w = 0;
                for (uint32_t i = threadIdx.x; i < n; i += T)
                    if (sh.list[i] > v) w += sh.list_w[i];
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
                if ((threadIdx.x & 31) == 0) sh.warp[threadIdx.x >> 5] = w;
                __syncthreads();
                if (threadIdx.x == 0) {
                    w = before;
                    for (int i = 0; i < T / 32; i++) w += sh.warp[i];
                    sh.best_above = w;
                }
            }
            cluster_sync();
            const uint32_t v = ld_cluster_u32(map_to_rank(smem_u32(&sh.best), 0));
            above = ld_cluster_u64(map_to_rank(smem_u32(&sh.best_above), 0));
            cluster_sync();  // rank 0 may begin another search
            return v;
        }
        // many entries within one step (equal ones, or a high temperature): bisection over their order
        uint32_t lo = ~cluster_max(~low), hi = cluster_max(high);  // lo <= the end <= hi
        above = before;
        while (lo < hi) {
            const uint32_t mid = lo + ((hi - lo) >> 1);
            u64 w = 0;
            for (int i = a; i < b; i++) {
                const float x = at(i), k = key(x);
                if (k < kSrSteps && (int)k == prefix && order_bits(x) > mid) w += weight(x, counting);
            }
            w = before + cluster_sum(w);
            if (w < target) {
                hi = mid;
                above = w;
            } else {
                lo = mid + 1;
            }
        }
        return lo;
    }
    static __device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
        uint32_t v;
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
        return v;
    }
};

template <class E, int T>
__global__ void __launch_bounds__(T) sample_rows_kernel(const SampleRowsParams p) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ SampleRowsShared<T> sh;
    pdl_launch_dependents();
    pdl_wait();
    const int rank = (int)cluster_ctarank(), nr = (int)cluster_nctarank();
    const int row = blockIdx.x / nr;
    const int lo = min(p.n, rank * p.chunk), cnt = min(p.n, lo + p.chunk) - lo;
    const E* src = static_cast<const E*>(p.x) + (long long)row * p.stride + lo;
    constexpr int kV = 16 / sizeof(E);
    const int off = (int)((uintptr_t)src & 15) / (int)sizeof(E);  // the slice keeps the row's alignment
    E* xs = reinterpret_cast<E*>(smem + sizeof(u64) * kSrBins * T) + off;

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
    const int run = ((cnt + T - 1) / T) | 1;  // entries of a thread: odd, which spreads a warp over the banks
    SampleRow<E, T> s{sh, reinterpret_cast<u64*>(smem), xs, min(cnt, (int)threadIdx.x * run), 0, rank, nr, 0, 0, 0.0f, 0.0f, 0.0, 0.0};
    s.b = min(cnt, s.a + run);
    uint32_t best = 0, first = 0x7fffffffu;  // order bits (of a NaN: all ones), index in the row
    for (int i = s.a; i < s.b; i++) {
        const float x = s.at(i);
        const uint32_t ob = x != x ? 0xffffffffu : order_bits(x);
        if (ob > best) {
            best = ob;
            first = lo + i;
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
    s.top = top;
    s.oct = 1.4426950408889634074 / (double)temp;
    s.top_wide = s.widen(top);
    s.steps = fminf((float)(s.oct * (kSrSteps / kSrOctaves)), 1e30f);

    // ---- where the filters end ---------------------------------------------------
    float floor = -INFINITY;  // entries below are out
    int ties = 0x7fffffff;    // of the entries equal to tie, how many stay
    float tie = 0.0f;
    u64 mine = 0;             // mass that stays of the thread's run, as far as it is known:
    int step = -1;            // that above this step
    if (top_k > 0 && top_k < p.n) {
        u64 above;
        floor = tie = order_value(s.find_end(true, (u64)top_k, 0.0, 0, floor, above, mine, step));
        ties = top_k - (int)above;
        step = -1;
    }
    if (top_p < 1.0f) {
        u64 whole = 0;
        if (ties != 0x7fffffff) {  // the mass of those top_k: few, with of the equal last ones those that stay
            u64 m = 0, equal = 0;
            s.masses(false, [&](float x) { return x >= tie; },
                     [&](float x, u64 w) {
                         if (x == tie) equal++;
                         else m += w;
                     });
            equal = s.cluster_sum(equal);
            if ((u64)ties > equal) ties = (int)equal;  // all entries with mass stay
            whole = s.cluster_sum(m) + (u64)ties * s.mass(tie);
        }
        u64 above;
        floor = order_value(s.find_end(false, 0, (double)top_p, whole, floor, above, mine, step));
    }
    if (min_p > 0.0f) {  // the smallest value that it keeps
        const double most = -log2((double)fminf(min_p, 1.0f));
        auto stays = [&](float x) { return ((double)top - (double)x) * s.oct <= most; };
        const float guess = (float)((double)top - most / s.oct);
        uint32_t k = order_bits(fminf(guess == guess ? guess : top, top) + 0.0f);
        const uint32_t last = order_bits(top);
        while (k < last && !stays(order_value(k))) k++;  // a rounding or two
        while (k > 0x00800000u && stays(order_value(k - 1))) k--;
        const float end = order_value(k) + 0.0f;
        if (end > floor) {
            floor = end;
            step = -1;
        }
    }

    // ---- the draw, in index order --------------------------------------------------
    const bool few = ties != 0x7fffffff && floor == tie;
    int tie_before = 0;  // entries equal to the tie before this run
    if (few) {
        u64 eq = 0, lower;
        for (int i = s.a; i < s.b; i++) eq += s.at(i) == tie ? 1 : 0;
        s.cluster_sum(eq, &lower);
        tie_before = (int)(lower + s.cta_before(eq));
    }
    int seen = tie_before;
    // whether the next entry of the run stays (it is asked once for each, in order)
    auto stays = [&](float x) {
        if (x < floor || !s.has_mass(x)) return false;
        return !(few && x == tie && seen++ >= ties);
    };
    if (step < 0) {
        mine = 0;
        s.masses(false, stays, [&](float, u64 w) { mine += w; });
    } else {  // what lies above the last search's step has been added up
        s.masses(false, [&](float x) { return s.has_mass(x) && (int)s.key(x) == step && stays(x); },
                 [&](float, u64 w) { mine += w; });
    }
    u64 lower;
    const u64 total = s.cluster_sum(mine, &lower);
    u64 c = lower + s.cta_before(mine);
    const double want = (u > 0.0 ? u : 0.0) * (double)total;
    const u64 goal = want >= (double)total ? total - 1 : (u64)want;
    if (goal >= c && goal < c + mine) {  // one thread of the cluster
        seen = tie_before;
        for (int i = s.a; i < s.b; i++) {
            const float x = s.at(i);
            if (stays(x)) c += s.mass(x);
            if (c > goal) {
                p.tok[row] = lo + i;
                if (p.logp)
                    p.logp[row] = (float)(-((double)top - (double)x) * s.oct * 0.6931471805599453094 -
                                          log((double)total / 17592186044416.0));
                break;
            }
        }
    }
}

template <class E, int T>
static int launch_sample_rows(const SampleRowsParams& p, int rows, int cluster, size_t smem, cudaStream_t st) {
    auto kern = sample_rows_kernel<E, T>;
    static PerDeviceOnce once;
    if (smem_opt_in(once, kern, (int)kSrSmem) != cudaSuccess) return HQ4_ERR_LAUNCH;
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

// Shared memory of a CTA (without its static part).
static size_t sr_smem(int n, int cluster, int threads, size_t elem) {
    return (size_t)((n + cluster - 1) / cluster + 16) * elem + sizeof(u64) * kSrBins * threads;
}

// The largest cluster whose CTAs all fit the device at once (a row then takes
// the least time), else the one with the fewest CTAs that holds a row; 512
// threads, or 256 where that lets more CTAs share an SM or a slice fit.
template <class E>
static int sample_rows(SampleRowsParams p, int rows, int sms, cudaStream_t st) {
    int best_cluster = 0, best_threads = 0;
    double best = 0.0;
    for (int cluster = kSrMaxCluster; cluster >= 1; cluster >>= 1) {
        if (cluster > 1 && p.n / cluster < 2048) continue;
        for (int threads = 512; threads >= 256; threads >>= 1) {
            const size_t smem = sr_smem(p.n, cluster, threads, sizeof(E));
            if (smem > kSrSmem) continue;
            const int per_sm = std::min<int>(2048 / threads, (int)(kSrSmem / (smem + 8 * 1024)) < 1 ? 1 : (int)(kSrSmem / (smem + 8 * 1024)));
            const int at_once = std::max(1, sms * per_sm / cluster);  // rows
            const double waves = (rows + at_once - 1) / at_once;
            // a row's time: passes over its entries (shared by the CTAs of an SM), and the cluster's barriers
            const double each = (double)p.n / cluster / threads * std::max(1.0, (double)std::min(per_sm, (rows * cluster + sms - 1) / sms) * threads / 512.0);
            const double cost = waves * (each + 40.0 + 4.0 * cluster);
            if (!best_cluster || cost < best) {
                best = cost;
                best_cluster = cluster;
                best_threads = threads;
            }
        }
    }
    if (!best_cluster) return HQ4_ERR_SHAPE;
    p.chunk = (p.n + best_cluster - 1) / best_cluster;
    const size_t smem = sr_smem(p.n, best_cluster, best_threads, sizeof(E));
    return best_threads == 512 ? launch_sample_rows<E, 512>(p, rows, best_cluster, smem, st)
                               : launch_sample_rows<E, 256>(p, rows, best_cluster, smem, st);
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
