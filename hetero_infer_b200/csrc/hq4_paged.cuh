// Shared pieces of the paged-cache operators (append, attention, tree
// attention): element types, the batch's ragged rows and the page addressing.
//
// A batch is n_seqs sequences.  Sequence s owns the rows
// [cu_rows[s], cu_rows[s+1]) of the activations; its cache holds lens[s]
// entries before them, and its i-th row is entry lens[s] + i.  Entry e lies in
// page pages[s][e / page_size] at place e % page_size of the caches
// [n_pages][n_kv][page_size][head_dim] (page_stride elements from a page to
// the next).  All of this is device memory, so a captured step can be
// replayed while the sequences grow; what it holds is checked where it is
// used, and an entry without a page inside [0, n_pages) reads and writes
// nothing and sets kStatusPaged.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "hq4.h"
#include "hq4_common.cuh"

namespace hq4 {

constexpr int kStatusPaged = 16;  // bit 4 of the status word

struct PagedBatch {
    const int* __restrict__ cu_rows;
    const int* __restrict__ lens;
    const int* __restrict__ pages;
    int n_seqs, n_rows, pages_per_seq;
    int n_pages, page_shift;
    long long page_stride;  // elements
    int* status;
};

// The sequence of row t, or -1 for a row outside every sequence: the last s
// with cu_rows[s] <= t (an empty sequence before it shares that start).
__device__ __forceinline__ int find_seq(const int* __restrict__ cu, int n_seqs, int t) {
    int lo = 0, hi = n_seqs;  // cu[lo] <= t < cu[hi] is sought
    if (t < __ldg(cu)) return -1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(cu + mid) <= t) lo = mid;
        else hi = mid;
    }
    return t < __ldg(cu + lo + 1) ? lo : -1;
}

// Page of entry e of sequence s, or -1 where there is none.
__device__ __forceinline__ int find_page(const PagedBatch& b, int s, int e) {
    const int i = e >> b.page_shift;
    if (e < 0 || i >= b.pages_per_seq) return -1;
    const int p = __ldg(b.pages + (size_t)s * b.pages_per_seq + i);
    return (unsigned)p < (unsigned)b.n_pages ? p : -1;
}

// Whether `rows` rows of `row` elements, `stride` apart, reach into the n_bytes at b (host).
static inline bool rows_overlap(const void* a, long long rows, long long stride, long long row, int elem_bytes,
                                const void* b, __int128 n_bytes) {
    const __int128 from = (intptr_t)a, to = from + ((__int128)(rows - 1) * stride + row) * elem_bytes;
    return from < (intptr_t)b + n_bytes && (intptr_t)b < to;
}

// Whether one of n pages of `page` elements, `stride` apart, from a on reaches into one of those from b on (host).
static inline bool pages_overlap(const void* a, const void* b, long long n, long long stride, long long page, int elem_bytes) {
    const intptr_t x = (intptr_t)a, y = (intptr_t)b;
    const unsigned long long d = x < y ? (unsigned long long)y - x : (unsigned long long)x - y, step = (unsigned long long)stride * elem_bytes;
    const unsigned long long apart = d / step, rest = d % step, bytes = (unsigned long long)page * elem_bytes;
    return (apart < (unsigned long long)n && rest < bytes) || (apart + 1 < (unsigned long long)n && step - rest < bytes);
}

template <class T>
struct Elem;
template <>
struct Elem<float> {
    static constexpr int code = HQ4_F32;
    static __device__ __forceinline__ float to(float v) { return v; }
    static __device__ __forceinline__ float from(float v) { return v; }
};
template <>
struct Elem<__nv_bfloat16> {
    static constexpr int code = HQ4_BF16;
    static __device__ __forceinline__ float to(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Elem<__half> {
    static constexpr int code = HQ4_F16;
    static __device__ __forceinline__ float to(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
};

// 16 bytes to shared memory; zeros where `on` is not set (nothing is read then).
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Two fp32 values rounded to nearest and packed, the first in the low half.
template <class T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
template <class T>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
    return __half22float2(*reinterpret_cast<__half2*>(&v));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

// Eight consecutive elements (16-byte aligned) as they lie in memory.
template <class T>
struct Raw8 {
    uint4 v[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) v[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    }
    __device__ __forceinline__ void get(float (&f)[8]) const {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                f[4 * i] = __uint_as_float(v[i].x);
                f[4 * i + 1] = __uint_as_float(v[i].y);
                f[4 * i + 2] = __uint_as_float(v[i].z);
                f[4 * i + 3] = __uint_as_float(v[i].w);
            }
        } else {
            const uint32_t w[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float2 x = unpack2<T>(w[i]);
                f[2 * i] = x.x;
                f[2 * i + 1] = x.y;
            }
        }
    }
};
// Eight consecutive elements (16-byte aligned) as fp32, and back.
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <class T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = unpack2<T>(w[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]),
                                              pack2<T>(v[6], v[7]));
}

__device__ __forceinline__ void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
template <class T>
__device__ __forceinline__ void store4(T* p, float4 v) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w));
}

}  // namespace hq4
