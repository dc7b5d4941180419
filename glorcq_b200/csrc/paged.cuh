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

// ---- sharing out the work of an attention call -----------------------------------------------------------------------
// A segment is a block of rows of one (sequence, key/value head); its work are steps of STEP tokens.  The steps of all segments, counted in
// order (sequence, block of rows, head), are cut into equal shares, one for each CTA, whatever the lengths: the lengths are on the device, and
// a batch of 64 sequences of 800 to 8192 tokens takes as long as its sum, not as its longest.  A segment that a share's end cuts leaves
// partial results, at most two of them per CTA, which paged_join_kernel joins.
__host__ __device__ __forceinline__ long long share_begin(long long total, int cta, int n_cta) { return total * cta / n_cta; }
// the CTA in whose share step u lies
__device__ __forceinline__ int share_of(long long total, long long u, int n_cta) { return (int)(((u + 1) * n_cta + total - 1) / total) - 1; }

struct PagedSeq {
    int2 own;               // first row, rows
    int start, steps, blocks;      // tokens before the call; steps and blocks of rows of a head
};
template <int R, int STEP> __device__ __forceinline__ PagedSeq paged_seq(const PagedKv& kv, const PagedRows& r, int group, int b) {
    PagedSeq s;
    s.own = rows_of(r, b);
    s.start = start_of(r, b, kv.capacity);
    s.blocks = (s.own.y * group + R - 1) / R;
    s.steps = s.own.y > 0 ? (min(s.start + s.own.y, kv.capacity) + STEP - 1) / STEP : 0;
    return s;
}
// All threads of the block; `sm`: THREADS / 32 + 3 long longs.  Returns the total; b0, off0: the sequence, and the step of it, where
// the share of `cta` begins (nothing, where that is empty).
template <int THREADS, int R, int STEP>
__device__ __forceinline__ long long paged_plan(const PagedKv& kv, const PagedRows& r, int group, int cta, int n_cta, long long* sm, int& b0, long long& off0) {
    constexpr int W = THREADS / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (r.B + THREADS - 1) / THREADS;
    auto weight = [&](int b) {
        const PagedSeq s = paged_seq<R, STEP>(kv, r, group, b);
        return (long long)s.blocks * kv.n_kv * s.steps;
    };
    long long mine = 0;
    for (int i = 0; i < per; ++i)
        if (tid * per + i < r.B) mine += weight(tid * per + i);
    long long incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long o = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += o;
    }
    if (lane == 31) sm[warp] = incl;
    __syncthreads();
    long long before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        if (w < warp) before += sm[w];
        total += sm[w];
    }
    const long long u0 = share_begin(total, cta, n_cta);
    long long at = before + incl - mine;
    if (mine > 0 && u0 >= at && u0 < at + mine) {
        for (int i = 0;; ++i) {
            const long long w = weight(tid * per + i);
            if (u0 < at + w) {
                sm[W + 1] = tid * per + i;
                sm[W + 2] = u0 - at;
                break;
            }
            at += w;
        }
    }
    __syncthreads();
    b0 = (int)sm[W + 1];
    off0 = sm[W + 2];
    return total;
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
