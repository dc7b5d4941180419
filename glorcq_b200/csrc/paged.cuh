// Paged key/value cache in 8 bits: what its kernels share.
//
// A page holds `page` tokens of every key/value head as codes (heads, tokens, channels) and one fp32 scale per (page, head) for
// the keys and one for the values: value = code * scale.  Sequence b holds start[b] tokens before a call and owns rows
// q_start[b] .. q_start[b + 1] of the call's batch; logical page j of it is physical page table[b][j].  Numbers from device
// memory are never trusted with an address, nor with the end of a loop: q_start is cut to the rows there are, start to the table's capacity, and a page id
// outside the pool is a page that is not there (nothing is written to it, its tokens are hidden, it reads as zeros).
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
// The rows with q_start and start in shared memory, loaded together: last_from's steps take a tenth of the time that they take in global memory.  All
// threads of the block.
constexpr int kRowsShared = 512;
struct SharedRows {
    long long start[kRowsShared];
    int q_start[kRowsShared + 1];
};
__device__ __forceinline__ PagedRows rows_in_shared(const PagedRows& r, SharedRows& sm) {
    if (!r.q_start || r.B < 3 || r.B > kRowsShared) return r;
    for (int i = threadIdx.x; i <= r.B; i += blockDim.x) {
        const int q = r.q_start[i];
        const long long s = r.start[(long long)min(i, r.B - 1) * r.start_stride];
        sm.q_start[i] = q;
        if (i < r.B) sm.start[i] = s;
    }
    __syncthreads();
    PagedRows x = r;
    x.q_start = sm.q_start;
    x.start = sm.start;
    x.start_stride = 1;
    return x;
}
// physical page of sequence b's logical page j, or -1
__device__ __forceinline__ int page_of(const PagedKv& kv, int b, int j) {
    if (j >= kv.max_pages) return -1;
    const int p = kv.table[b * kv.table_stride + j];
    return p >= 0 && p < kv.n_pages ? p : -1;
}

// the same in two parts, for who looks ahead: the table's entry (-1 behind its end), and whether that is a page
__device__ __forceinline__ int page_entry(const PagedKv& kv, int b, int j) { return j < kv.max_pages ? kv.table[b * kv.table_stride + j] : -1; }
__device__ __forceinline__ bool page_there(const PagedKv& kv, int entry) { return (unsigned)entry < (unsigned)kv.n_pages; }

// what all kernels here do first
__device__ __forceinline__ void after_launch_ahead() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// ---- sharing out the work of an attention call -----------------------------------------------------------------------
// A segment is a block of R rows (token of the call, head of the group) of one (sequence, key/value head); its work are steps of STEP
// tokens, up to the last key that a row of it sees, and EXTRA steps' worth of beginning and end.  The units of all segments, counted in order
// (sequence, block of rows, head), are cut into equal shares, one for each CTA, whatever the lengths: these are on the device, and a batch of
// 64 sequences of 800 to 8192 tokens takes as long as its sum, not as its longest.  A cut that falls into a segment's EXTRA units parts nothing;
// another leaves partial results, at most two of them per CTA, which paged_join_kernel joins.
// Where shares of LEAST units do not go round, a segment's units are rounded up to a multiple of LEAST, so that no CTA has the end of one and the
// beginning of the next.
// Blocks of rows are numbered so that nobody has to count those of the sequences before: sequence b's are rows * group / R + b and on.
template <int R_, int STEP_, int EXTRA_, int LEAST_> struct ShareOf {
    static constexpr int R = R_, STEP = STEP_, EXTRA = EXTRA_;
    static constexpr int LEAST = LEAST_;      // units of a share, so long as there are fewer shares than CTAs
    // units of a segment
    static __host__ __device__ __forceinline__ int units(int steps, int grain) { return LEAST == 1 || grain == 1 ? steps + EXTRA : (steps + EXTRA + LEAST - 1) / LEAST * LEAST; }
};
// Units are counted in 32 bits (the host refuses what might not fit: 64-bit divisions took longer than the rest of a small call's planning).
__device__ __forceinline__ int share_begin(int total, int cta, int n_cta) { return total / n_cta * cta + total % n_cta * cta / n_cta; }
// the CTA in whose share unit u lies
__device__ __forceinline__ int share_of(int total, int u, int n_cta) {
    int c = min((int)((float)u / (float)total * (float)n_cta), n_cta - 1);
    while (share_begin(total, c, n_cta) > u) --c;
    while (share_begin(total, c + 1, n_cta) <= u) ++c;
    return c;
}
template <class S> __device__ __forceinline__ int share_ctas(int total, int n_cta) { return min(n_cta, max(1, total / S::LEAST)); }

struct RowBlock {
    int b, r0, n_rows;      // sequence; first row of the block, counted from the sequence's; 0 rows: there is no such block
    int2 own;               // the sequence's first row in the batch, its number of rows
    int start, steps;
};
template <class S> __device__ __forceinline__ int first_block(const PagedRows& r, int group, int b) {
    return (int)((long long)rows_from(r, b) * group / S::R) + b;
}
// block i, in sequence b (first_block(b) <= i, and b the last such)
template <class S> __device__ __forceinline__ RowBlock row_block(const PagedKv& kv, const PagedRows& r, int group, int i, int b) {
    RowBlock x;
    x.b = b;
    x.own = rows_of(r, b);
    x.r0 = (i - first_block<S>(r, group, b)) * S::R;
    x.n_rows = x.r0 < 0 ? 0 : max(0, min(x.own.y * group - x.r0, S::R));
    x.start = start_of(r, b, kv.capacity);
    x.steps = x.n_rows > 0 ? min(x.start + (x.r0 + x.n_rows - 1) / group, kv.capacity - 1) / S::STEP + 1 : 0;
    return x;
}
template <class S> __device__ __forceinline__ int block_units(const PagedKv& kv, const RowBlock& x, int grain) {
    return x.n_rows > 0 ? kv.n_kv * S::units(x.steps, grain) : 0;
}
template <class S> inline bool units_fit(int rows, int B, int group, int n_kv, int capacity) {
    return ((double)rows * group / S::R + B) * n_kv * ((double)capacity / S::STEP + 1 + S::EXTRA) < 2147483647.0;
}
template <class S> __host__ __device__ __forceinline__ int block_count(int rows, int B, int group) {
    return (int)((long long)rows * group / S::R) + B;
}

// Where a CTA's share begins: in block i, x, off units of which belong to shares before; what units are rounded to (1 or LEAST).
struct ShareStart {
    RowBlock x;
    int i, off, grain;
    int sums[32];
};
// All threads of the block; `sm` in shared memory.  Returns the units of all; what it says of the beginning holds where `cta` has a share.
template <class S, int THREADS>
__device__ __forceinline__ int paged_plan(const PagedKv& kv, const PagedRows& r, int group, int cta, int n_cta, ShareStart& sm) {
    constexpr int W = THREADS / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int blocks = block_count<S>(r.N, r.B, group), per = (blocks + THREADS - 1) / THREADS;
    const int from = tid * per, to = min(from + per, blocks);
    auto each = [&](auto&& f) {       // f(block, what it is) until it says that it is enough
        if (from >= to) return;
        int b = last_from(r.B, from, [&](int b) { return first_block<S>(r, group, b); });
        for (int i = from; i < to; ++i) {
            while (b + 1 < r.B && first_block<S>(r, group, b + 1) <= i) ++b;
            if (f(i, row_block<S>(kv, r, group, i, b))) return;
        }
    };
    int mine, before, total, grain = 1;       // units of the thread's blocks, of those before them, of all
    RowBlock x{};
    for (;; grain = S::LEAST) {
        mine = 0;
        each([&](int, const RowBlock& y) {
            x = y;
            mine += block_units<S>(kv, y, grain);
            return false;
        });
        int incl = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, incl, d);
            if (lane >= d) incl += o;
        }
        if (lane == 31) sm.sums[warp] = incl;
        __syncthreads();
        before = incl - mine;
        total = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            if (w < warp) before += sm.sums[w];
            total += sm.sums[w];
        }
        if (S::LEAST == 1 || grain > 1 || total > n_cta * S::LEAST) break;
        __syncthreads();
    }
    if (tid == 0) sm.grain = grain;
    const int n = share_ctas<S>(total, n_cta);
    const int u0 = cta < n ? share_begin(total, cta, n) : total;
    int at = before;
    if (u0 >= at && u0 < at + mine) {
        if (per == 1) {
            sm.x = x;
            sm.i = from;
            sm.off = u0 - at;
        } else {
            each([&](int i, const RowBlock& y) {
                const int w = block_units<S>(kv, y, grain);
                if (u0 < at + w) {
                    sm.x = y;
                    sm.i = i;
                    sm.off = u0 - at;
                    return true;
                }
                at += w;
                return false;
            });
        }
    }
    __syncthreads();
    return total;
}

// A segment that several CTAs share: written by the second of them, for paged_join_kernel.
struct JoinItem {
    int parts, first_cta;        // CTAs first_cta .. first_cta + parts - 1 (0 parts: nothing to join)
    int row, r0, n_rows, h;      // as in RowBlock
    int unused[2];
};

// A CTA's pieces of segments, one after another.
template <class S> struct Pieces {
    int left, off, i;
    RowBlock x;                  // block i
    int h, step0, step1;         // the piece: steps step0 .. step1 of head h of it
    int total, n_cta, grain;
    template <int THREADS> __device__ __forceinline__ void begin(const PagedKv& kv, const PagedRows& r, int group, int cta, int most_ctas, ShareStart& sm) {
        total = paged_plan<S, THREADS>(kv, r, group, cta, most_ctas, sm);
        n_cta = share_ctas<S>(total, most_ctas);
        left = cta < n_cta ? share_begin(total, cta + 1, n_cta) - share_begin(total, cta, n_cta) : 0;
        i = sm.i;
        off = sm.off;
        x = sm.x;
        grain = sm.grain;
    }
    __device__ __forceinline__ bool next(const PagedKv& kv, const PagedRows& r, int group) {
        return next(kv, r, group, [] {});
    }
    template <class F> __device__ __forceinline__ bool next(const PagedKv& kv, const PagedRows& r, int group, F&& looking) {      // looking(): at each block
        while (left > 0) {
            if (off >= block_units<S>(kv, x, grain)) {
                looking();
                // (where q_start decreases, which it must not, these blocks may not be those that were counted: the list has an end all the same)
                if (++i >= block_count<S>(r.N, r.B, group)) left = 0;
                off = 0;
                int b = x.b;
                while (b + 1 < r.B && first_block<S>(r, group, b + 1) <= i) ++b;
                x = row_block<S>(kv, r, group, i, b);
                continue;
            }
            const int units = S::units(x.steps, grain);
            h = off / units;
            const int v0 = off - h * units, v1 = min(units, v0 + left);
            off += v1 - v0;
            left -= v1 - v0;
            step0 = max(v0 - S::EXTRA, 0);
            step1 = min(max(v1 - S::EXTRA, 0), x.steps);
            if (step1 > step0) return true;
        }
        return false;
    }
    __device__ __forceinline__ bool whole() const { return step0 == 0 && step1 == x.steps; }
};
// What CTA `cta` has to say to paged_join_kernel.
template <class S> __device__ __forceinline__ JoinItem join_item(int total, int most_ctas, int cta, const ShareStart& sm) {
    JoinItem j{};
    const int n = share_ctas<S>(total, most_ctas);
    if (cta >= n || share_begin(total, cta, n) == share_begin(total, cta + 1, n)) return j;
    const int units = S::units(sm.x.steps, sm.grain), h = sm.off / units, v0 = sm.off - h * units;
    if (v0 <= S::EXTRA || v0 - S::EXTRA >= sm.x.steps) return j;
    const int u0 = share_begin(total, cta, n) - v0, c0 = share_of(total, u0 + S::EXTRA, n);
    if (c0 + 1 != cta) return j;
    j.parts = share_of(total, u0 + S::EXTRA + sm.x.steps - 1, n) - c0 + 1;
    j.first_cta = c0;
    j.row = sm.x.own.x;
    j.r0 = sm.x.r0;
    j.n_rows = sm.x.n_rows;
    j.h = h;
    return j;
}
// where CTA `cta` leaves its partial results of a piece: R rows of HD values, then (maximum, sum) of each row
template <class S, int HD> constexpr int kPartial = S::R * (HD + 2);
template <class S, int HD> __device__ __forceinline__ float* partial_of(float* partial, int cta, bool from_first_step) {
    return partial + (size_t)(2 * cta + from_first_step) * kPartial<S, HD>;
}

struct AttnParams {
    PagedKv kv;
    PagedRows r;
    const __half* q;
    __half* out;
    long long ldq, ldo;
    int group;
    float scale2;           // softmax scale * log2(e) * kCodeUnit
    JoinItem* join;         // an item for each CTA, then
    float* partial;         // two partial results for each
};
__device__ __forceinline__ float exp2_fast(float x) {      // 2 ulp; -inf -> 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float log2_fast(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Scales of values.  A block whose scale is below kLeastScale (0 above all; also what nobody has written yet) has values that are zero: what it could add
// to a result is below 448 kLeastScale, zero in fp16.  Its scores count in the sum of the softmax and must not set the maximum, relative to which
// the other blocks' weights are rounded: they count as if its scale were kLeastScale, so that it raises the maximum only above scores that weigh 2^-60 of its own,
// whose part of the result is zero in fp16 whatever the values.  (As if its scale were 1: values of 1e-4 beside a block of zeros off by 1 %.)
constexpr float kLeastScaleLog = -60.f, kLeastScale = 0x1p-60f;
__device__ __forceinline__ bool live_scale(float s) { return s >= kLeastScale && s <= FLT_MAX; }
// log2 of a block's scale, and its reciprocal, as the softmax has them
__device__ __forceinline__ float scale_log(float s) { return live_scale(s) ? log2_fast(s) : kLeastScaleLog; }
__device__ __forceinline__ float scale_inverse(float s) { return live_scale(s) ? rcp_fast(s) : 1.f / kLeastScale; }
// Blocks of rows of paged_prompt_kernel (paged_prompt.cu): many rows a head.  Two tiles of 128 rows and steps of 128 tokens; with 256 channels one tile and
// 64 tokens, which is what tensor memory and shared memory hold.  A segment's beginning and end count as two steps, the least share is four.
// Measured (us, (extra, least) = (2, 4) / (2, 6) / (2, 3) / (1, 4)): 16 heads, 512 tokens 22.5 / 22.3 / 24.7 / 24.8; 32 heads on 8, 512 tokens 24.3 / 22.9 /
// 27.8 / 25.2, 256 tokens after 1000 29.3 / 32.9 / 27.8 / 29.3, 1024 tokens 37.5 / 40.2 / 37.3 / 38.8; 32 on 4, 4096 tokens 180 / 178 / 179 / 212.
template <int HD> struct PromptShape {
    static constexpr int TILES = HD == 256 ? 1 : 2, STEP = HD == 256 ? 64 : 128;
    using Share = ShareOf<128 * TILES, STEP, 2, 4>;
};
cudaError_t launch_paged_prompt(int head_dim, int dtype, const AttnParams& p, int grid, cudaStream_t st);

// what weighted values are multiplied by; a row that saw nothing is zero, not-a-number stays
__device__ __forceinline__ float result_factor(float sum, float unit) { return sum > 0.f ? unit / sum : (sum == 0.f ? 0.f : sum); }

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
// The same for four values.  The conversions have to_code's ends and zeros but for two things: whole numbers end at -128, which the byte-wise maximum
// mends, and e4m3 keeps not-a-number (0x7f), which is rare.
template <int DT> __device__ __forceinline__ uint32_t to_codes(float a, float b, float c, float d) {
    uint32_t w;
    if (DT == kI8) {
        asm("{\n .reg .b32 t;\n cvt.pack.sat.s8.s32.b32 t, %4, %3, 0;\n cvt.pack.sat.s8.s32.b32 %0, %2, %1, t;\n}\n"
            : "=r"(w)
            : "r"(__float2int_rn(a)), "r"(__float2int_rn(b)), "r"(__float2int_rn(c)), "r"(__float2int_rn(d)));
        return __vmaxs4(w, 0x81818181u);
    }
    asm("{\n .reg .b16 l, h;\n cvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n cvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n mov.b32 %0, {l, h};\n}\n"
        : "=r"(w)
        : "f"(a), "f"(b), "f"(c), "f"(d));
    if (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) return to_code<DT>(a) | to_code<DT>(b) << 8 | to_code<DT>(c) << 16 | to_code<DT>(d) << 24;
    return w;
}
template <int DT> __device__ __forceinline__ float code_value(uint32_t byte) {
    if (DT == kI8) return (float)(int)(signed char)(unsigned char)byte;
    const __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3);
    return __half2float(__half(h));
}

}  // namespace glq
