// Paged key/value cache in 8 bits: what its kernels share.
//
// A page holds `page` tokens of every key/value head as codes (heads, tokens, channels) and one fp32 scale per (page, head) for
// the keys and one for the values: value = code * scale.  Sequence b holds start[b] tokens before a call and owns rows
// q_start[b] .. q_start[b + 1] of the call's batch; logical page j of it is physical page table[b][j].  Numbers from device
// memory are never trusted with an address: q_start is cut to the rows there are, start to the table's capacity, and a page id outside
// the pool is a page that is not there (nothing is written to it, its tokens are hidden, it reads as zeros).
//
// All of it may have been written by the launch ahead, beside which these kernels start: plain loads behind griddepcontrol.wait, and
// dependent launches are let go behind it too.
#pragma once

#include <cuda_fp8.h>

#include <cfloat>

#include "glq_common.cuh"

namespace glq {

struct PagedKv {
    unsigned char *k, *v;
    float *k_scale, *v_scale;
    const int* table;
    long long table_stride;
    int n_pages, n_kv, page, page_shift, max_pages, capacity;
};
struct PagedRows {
    const long long* start;
    const int* q_start;      // nullptr: `per` rows a sequence
    int B, N, per, start_stride;
};

__device__ __forceinline__ int rows_from(const PagedRows& r, int b) {
    return r.q_start ? min(max(r.q_start[b], 0), r.N) : b * r.per;
}
// sequence b's first row and number of rows
__device__ __forceinline__ int2 rows_of(const PagedRows& r, int b) {
    const int lo = rows_from(r, b);
    return make_int2(lo, max(rows_from(r, b + 1) - lo, 0));
}
__device__ __forceinline__ int start_of(const PagedRows& r, int b, int capacity) {
    const long long s = r.start[(long long)b * r.start_stride];
    return (int)(s < 0 ? 0 : (s > capacity ? capacity : s));
}
// The largest b whose first(b) is at most i; first grows with b (0 where first(0) is above i already).
template <class F> __device__ __forceinline__ int last_from(int B, int i, F first) {
    int lo = 0, hi = B - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first(mid) <= i) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
// physical page of sequence b's logical page j, or -1
__device__ __forceinline__ int page_of(const PagedKv& kv, int b, int j) {
    if (j >= kv.max_pages) return -1;
    const int p = kv.table[b * kv.table_stride + j];
    return p >= 0 && p < kv.n_pages ? p : -1;
}

// what all kernels here do first
__device__ __forceinline__ void after_launch_ahead() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// ---- codes --------------------------------------------------------------------------------------------------------
constexpr int kI8 = GLQ_KV_I8, kE4M3 = GLQ_KV_E4M3;
template <int DT> constexpr float kCodeMax = DT == kI8 ? 127.f : 448.f;
// Four codes -> two fp16 pairs, exact.  int8: the code + 128 in the mantissa of 1024, minus 1152.  e4m3: sign, exponent and mantissa moved
// to where fp16 has them, which is the value / 256 (kCodeUnit), subnormals included.
template <int DT> constexpr float kCodeUnit = DT == kI8 ? 1.f : 256.f;
template <int DT> __device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if (DT == kI8) {
        const uint32_t x = w ^ 0x80808080u;
        const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
        const uint32_t a = prmt(x, 0x64646464u, 0x4140u), b = prmt(x, 0x64646464u, 0x4342u);
        const __half2 l = __hsub2(*reinterpret_cast<const __half2*>(&a), off), h = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
        lo = *reinterpret_cast<const uint32_t*>(&l);
        hi = *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const uint32_t a = prmt(w, 0u, 0x1404u), b = prmt(w, 0u, 0x3424u);
        lo = ((a >> 1) & 0x3f803f80u) | (a & 0x80008000u);
        hi = ((b >> 1) & 0x3f803f80u) | (b & 0x80008000u);
    }
}
// value / scale -> code: nearest, ties to even, ends at +-kCodeMax, not-a-number as zero
template <int DT> __device__ __forceinline__ uint32_t to_code(float y) {
    y = y != y ? 0.f : fminf(fmaxf(y, -kCodeMax<DT>), kCodeMax<DT>);
    if (DT == kI8) return (uint32_t)__float2int_rn(y) & 0xffu;
    return (uint32_t)__nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
}
template <int DT> __device__ __forceinline__ float code_value(uint32_t byte) {
    if (DT == kI8) return (float)(int)(signed char)(unsigned char)byte;
    const __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3);
    return __half2float(__half(h));
}

}  // namespace glq
