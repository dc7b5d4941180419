// Paged key/value cache in 8 bits: writing new tokens (glq_paged_append), attention (glq_paged_attention) and reading rows
// back (glq_paged_read).  include/glorcq_b200.h has the definitions, paged.cuh what the kernels share.
#include <algorithm>
#include <utility>

#include "paged.cuh"

using namespace glq;

namespace {

// ---------------------------------------------------------------------------------------------
// Append.  A block of a page and head is one CTA's: its scale needs the largest value of all new tokens before a code can be written.  Up to four rows a
// lane stay in registers in between; of larger blocks the values are computed twice (the second time from the caches).  Two halves of a row that the
// rotation mixes belong to one lane: lane c of HD / 16 has channels 8c .. 8c+7 and HD/2 + 8c .. .  Queries: a CTA a row or two, whose lanes use a
// position's angles for all their heads.  Bound by memory: what counts is that a lane's loads are all requested before the first is used.
// ---------------------------------------------------------------------------------------------
constexpr int kAppendThreads = 128, kAppendCtas = 4;       // CTAs an SM: with five, registers spill

struct AppendParams {
    PagedKv kv;
    PagedRows r;
    const __half *q, *k, *v, *q_norm, *k_norm;
    __half* q_out;
    const float *cos, *sin;
    long long ldq, ldk, ldv, ldqo;
    int n_heads, page_items, cos_rows, query_rows, query_turns, stride;       // (rows of queries that a CTA takes at once, how often; every so many CTAs one has a block)
    float eps;
};
constexpr int kAppendHeld = 4, kQueryTurns = 2;

struct __align__(16) RowHalves {
    float a[8], b[8];      // first half's channels, second half's
};
__device__ __forceinline__ void widen8(const uint4& w, float (&f)[8]) {
    const uint32_t in[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&in[i]));
        f[2 * i] = v.x;
        f[2 * i + 1] = v.y;
    }
}
__device__ __forceinline__ uint4 narrow8(const float (&f)[8]) {
    return make_uint4(pack_half2(f[0], f[1]), pack_half2(f[2], f[3]), pack_half2(f[4], f[5]), pack_half2(f[6], f[7]));
}
// RMS norm of one row by its HD / 16 lanes, in fp32.
template <int HD> __device__ __forceinline__ void norm_row(RowHalves& x, const RowHalves& w, float eps) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += x.a[i] * x.a[i] + x.b[i] * x.b[i];
#pragma unroll
    for (int d = HD / 32; d > 0; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
    const float r = rsqrtf(ss / HD + eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x.a[i] = x.a[i] * r * w.a[i];
        x.b[i] = x.b[i] * r * w.b[i];
    }
}
// A lane's cosines (a) and sines (b) of a position.
template <int HD> __device__ __forceinline__ void load_angles(RowHalves& cs, const float* cos, const float* sin, int pos, int c) {
    const float4* cp = reinterpret_cast<const float4*>(cos + (size_t)pos * (HD / 2) + 8 * c);
    const float4* sp = reinterpret_cast<const float4*>(sin + (size_t)pos * (HD / 2) + 8 * c);
    reinterpret_cast<float4*>(cs.a)[0] = cp[0];
    reinterpret_cast<float4*>(cs.a)[1] = cp[1];
    reinterpret_cast<float4*>(cs.b)[0] = sp[0];
    reinterpret_cast<float4*>(cs.b)[1] = sp[1];
}
// Products and sums rounded one by one, so that they do not depend on what the compiler contracts.
__device__ __forceinline__ void rotate(RowHalves& x, const RowHalves& cs) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float a = __fsub_rn(__fmul_rn(x.a[i], cs.a[i]), __fmul_rn(x.b[i], cs.b[i]));
        x.b[i] = __fadd_rn(__fmul_rn(x.b[i], cs.a[i]), __fmul_rn(x.a[i], cs.b[i]));
        x.a[i] = a;
    }
}

template <int DT> __device__ __forceinline__ uint2 codes8(const float (&f)[8], float inv) {
    return make_uint2(to_codes<DT>(__fmul_rn(f[0], inv), __fmul_rn(f[1], inv), __fmul_rn(f[2], inv), __fmul_rn(f[3], inv)),
                      to_codes<DT>(__fmul_rn(f[4], inv), __fmul_rn(f[5], inv), __fmul_rn(f[6], inv), __fmul_rn(f[7], inv)));
}

template <int HD, int DT>
__global__ void __launch_bounds__(kAppendThreads, kAppendCtas) paged_append_kernel(const AppendParams p) {
    constexpr int LPR = HD / 16, RPP = kAppendThreads / LPR;       // lanes of a row, rows of a pass
    const int tid = threadIdx.x, c = tid % LPR, slot = tid / LPR;
    after_launch_ahead();
    const PagedRows& rows = p.r;
    // Blocks, whose scale waits for their last load, and queries, which stream, in turn.
    const int block_items = p.page_items * 2 * p.kv.n_kv, turn = (int)blockIdx.x / p.stride;
    const bool is_block = turn < block_items && turn * p.stride == (int)blockIdx.x;
    const int work = is_block ? turn : (int)blockIdx.x - min(turn + 1, block_items);
    RowHalves weight = {};
    auto load_weight = [&](const __half* w) {
        widen8(*reinterpret_cast<const uint4*>(w + 8 * c), weight.a);
        widen8(*reinterpret_cast<const uint4*>(w + HD / 2 + 8 * c), weight.b);
    };
    if (!is_block) {                                    // queries
        // One row, the heads of which go round the slots, or as many whole rows as there are slots for; that again for `query_turns` of them, whose loads are
        // requested together.
        const int first = p.query_rows > 1 ? slot % p.n_heads : slot;
        const int rounds = p.query_rows > 1 ? 1 : (p.n_heads + RPP - 1) / RPP;       // (alike for all threads, who stay together for the norm's shuffles)
        if (p.q_norm) load_weight(p.q_norm);
        int row[kQueryTurns];
        bool mine[kQueryTurns];
        RowHalves cs[kQueryTurns] = {};
        uint4 raw[kQueryTurns][2][2];
        auto request = [&](int t, int k) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int h = first + (k + u) * RPP;
                const bool live = mine[t] && k + u < rounds && h < p.n_heads;
                const __half* src = p.q + row[t] * p.ldq + h * HD + 8 * c;
                raw[t][u][0] = live ? *reinterpret_cast<const uint4*>(src) : make_uint4(0u, 0u, 0u, 0u);
                raw[t][u][1] = live ? *reinterpret_cast<const uint4*>(src + HD / 2) : make_uint4(0u, 0u, 0u, 0u);
            }
        };
#pragma unroll
        for (int t = 0; t < kQueryTurns; ++t) {
            if (t >= p.query_turns) break;
            row[t] = (work * p.query_turns + t) * p.query_rows + (p.query_rows > 1 ? slot / p.n_heads : 0);
            const bool there = row[t] < p.r.N && (p.query_rows == 1 || slot < p.query_rows * p.n_heads);
            // row b is usually sequence b's where a sequence has one token
            int b = min(there ? row[t] : 0, rows.B - 1);
            int2 own = rows_of(rows, b);
            if (row[t] < own.x || row[t] - own.x >= own.y) {
                b = last_from(rows.B, there ? row[t] : 0, [&](int b) { return rows_from(rows, b); });
                own = rows_of(rows, b);
            }
            // rows in front of the first sequence or behind the last are not touched
            mine[t] = there && row[t] >= own.x && row[t] - own.x < own.y;
            if (mine[t] && p.cos) {
                const long long at = (long long)start_of(rows, b, p.kv.capacity) + (row[t] - own.x);
                load_angles<HD>(cs[t], p.cos, p.sin, (int)min(at, (long long)p.cos_rows - 1), c);
            }
            request(t, 0);
        }
#pragma unroll
        for (int t = 0; t < kQueryTurns; ++t) {
            if (t >= p.query_turns) break;
            for (int k = 0; k < rounds; k += 2) {
                if (k > 0) request(t, k);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int h = first + (k + u) * RPP;
                    RowHalves x;
                    widen8(raw[t][u][0], x.a);
                    widen8(raw[t][u][1], x.b);
                    if (p.q_norm) norm_row<HD>(x, weight, p.eps);
                    if (p.cos) rotate(x, cs[t]);
                    if (mine[t] && k + u < rounds && h < p.n_heads) {
                        __half* dst = p.q_out + row[t] * p.ldqo + h * HD + 8 * c;
                        *reinterpret_cast<uint4*>(dst) = narrow8(x.a);
                        *reinterpret_cast<uint4*>(dst + HD / 2) = narrow8(x.b);
                    }
                }
            }
        }
        return;
    }
    const int hz = work % (2 * p.kv.n_kv), item = work / (2 * p.kv.n_kv);
    const int h = hz >> 1;
    const bool is_k = (hz & 1) == 0;
    // Item b is the first page of sequence b's rows; n rows lie in at most n / page + 1 more, items B + rows / page + b and on.  (Decoded tokens have
    // none of these: they come last, and nobody looks for the sequence of the others.)
    auto more = [&](int b) { return rows.B + (rows_from(rows, b) >> p.kv.page_shift) + b; };
    const int b = item < rows.B ? item : last_from(rows.B, item, more);
    const int2 own = rows_of(rows, b);
    const int start = start_of(rows, b, p.kv.capacity);
    if (item >= rows.B && item < more(b)) return;       // (rows in front of the first sequence)
    const int j = (item < rows.B ? 0 : item - more(b) + 1) + (start >> p.kv.page_shift);
    const int at = j << p.kv.page_shift;
    if (own.y == 0 || (long long)at >= (long long)start + own.y) return;
    const int s0 = max(start - at, 0), s1 = (int)min((long long)start + own.y - at, (long long)p.kv.page);
    const __half* src = (is_k ? p.k : p.v) + (long long)(own.x + at - start) * (is_k ? p.ldk : p.ldv) + h * HD + 8 * c;
    const long long ld = is_k ? p.ldk : p.ldv;
    const __half* norm = is_k ? p.k_norm : nullptr;
    const int entry = page_entry(p.kv, b, j);          // (looked at when the rows have been requested too)
    if (norm) load_weight(norm);

    // up to four rows of a lane: s + slot + u RPP.  They are held as they are; norm and rotation are done twice.
    uint4 raw[kAppendHeld][2];
    auto load_rows = [&](int s) {
#pragma unroll
        for (int u = 0; u < kAppendHeld; ++u) {
            const int r = s + slot + u * RPP;
            raw[u][0] = r < s1 ? *reinterpret_cast<const uint4*>(src + r * ld) : make_uint4(0u, 0u, 0u, 0u);
            raw[u][1] = r < s1 ? *reinterpret_cast<const uint4*>(src + r * ld + HD / 2) : make_uint4(0u, 0u, 0u, 0u);
        }
    };
    RowHalves turned = {};                             // the first row's angles
    auto values = [&](int s, int u) {
        RowHalves x;
        widen8(raw[u][0], x.a);
        widen8(raw[u][1], x.b);
        if (norm) norm_row<HD>(x, weight, p.eps);        // (whole warps: a row's lanes shuffle)
        if (is_k && p.cos && s + slot + u * RPP < s1) {
            RowHalves cs = turned;
            if (u > 0 || s != s0) load_angles<HD>(cs, p.cos, p.sin, min(at + s + slot + u * RPP, p.cos_rows - 1), c);
            rotate(x, cs);
        }
        return x;
    };
    load_rows(s0);
    if (is_k && p.cos && s0 + slot < s1) load_angles<HD>(turned, p.cos, p.sin, min(at + s0 + slot, p.cos_rows - 1), c);
    if (!page_there(p.kv, entry)) return;
    const size_t block = (size_t)entry * p.kv.n_kv + h;
    unsigned char* codes = (is_k ? p.kv.k : p.kv.v) + block * ((size_t)HD << p.kv.page_shift);
    float* scale_at = (is_k ? p.kv.k_scale : p.kv.v_scale) + block;
    const float old = *scale_at;
    const bool held = s1 - s0 <= kAppendHeld * RPP;
    __shared__ float red[kAppendThreads / 32];
    // largest magnitude of the new values; `finite`: of those that are (not-a-numbers never count)
    auto largest = [&](bool finite) {
        float big = 0.f;
        for (int s = s0; s < s1; s += kAppendHeld * RPP) {
            if (s > s0 || (finite && !held)) load_rows(s);
#pragma unroll
            for (int u = 0; u < kAppendHeld; ++u) {
                if (s + u * RPP >= s1) break;
                const RowHalves x = values(s, u);            // (rows that are not there are zero)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float v = fabsf(x.a[i]), w = fabsf(x.b[i]);
                    big = fmaxf(big, finite && v > FLT_MAX ? 0.f : v);
                    big = fmaxf(big, finite && w > FLT_MAX ? 0.f : w);
                }
            }
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, d));
        __syncthreads();
        if ((tid & 31) == 0) red[tid >> 5] = big;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kAppendThreads / 32; ++w) big = fmaxf(big, red[w]);
        return big;
    };
    float big = largest(false);
    if (big > FLT_MAX) big = largest(true);
    const float need = big / kCodeMax<DT>;
    float scale = need;
    if (s0 > 0 && old > 0.f) {
        scale = old;
        if (need > old) {
            int e0, e1;
            const float m0 = frexpf(old, &e0), m1 = frexpf(need, &e1);
            const int n = e1 - e0 + (m1 > m0 ? 1 : 0);
            scale = ldexpf(old, n);
            const float down = ldexpf(1.f, -n);
            for (int w = tid; w < s0 * (HD / 4); w += kAppendThreads) {
                const uint32_t v = reinterpret_cast<uint32_t*>(codes)[w];
                reinterpret_cast<uint32_t*>(codes)[w] = to_codes<DT>(code_value<DT>(v & 0xffu) * down, code_value<DT>(v >> 8 & 0xffu) * down,
                                                                     code_value<DT>(v >> 16 & 0xffu) * down, code_value<DT>(v >> 24) * down);
            }
        }
    }
    if (tid == 0 && scale != old) *scale_at = scale;
    const float inv = scale > 0.f ? 1.f / scale : 0.f;
    for (int s = s0; s < s1; s += kAppendHeld * RPP) {
        if (!held) load_rows(s);
#pragma unroll
        for (int u = 0; u < kAppendHeld; ++u) {
            if (s + u * RPP >= s1) break;
            const RowHalves x = values(s, u);
            if (s + slot + u * RPP < s1) {
                unsigned char* dst = codes + (size_t)(s + slot + u * RPP) * HD + 8 * c;
                *reinterpret_cast<uint2*>(dst) = codes8<DT>(x.a, inv);
                *reinterpret_cast<uint2*>(dst + HD / 2) = codes8<DT>(x.b, inv);
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------
// Read: HD / 16 lanes a (row, head), keys and values.  Bound by memory.
// ---------------------------------------------------------------------------------------------
struct ReadParams {
    PagedKv kv;
    PagedRows r;
    __half *k_out, *v_out;
};
constexpr int kReadThreads = 256;

template <int HD, int DT>
__global__ void __launch_bounds__(kReadThreads) paged_read_kernel(const ReadParams p) {
    constexpr int LPR = HD / 16, RPP = kReadThreads / LPR;
    const int c = threadIdx.x % LPR;
    const long long i = (long long)blockIdx.x * RPP + threadIdx.x / LPR;
    __shared__ SharedRows sm_q;
    after_launch_ahead();
    const PagedRows rows = rows_in_shared(p.r, sm_q);
    if (i >= (long long)p.r.N * p.kv.n_kv) return;
    const int row = (int)(i / p.kv.n_kv), h = (int)(i - (long long)row * p.kv.n_kv);
    const int b = last_from(p.r.B, row, [&](int b) { return rows_from(rows, b); });
    const int2 own = rows_of(rows, b);
    if (row < own.x || row - own.x >= own.y) return;
    const long long at = (long long)start_of(p.r, b, p.kv.capacity) + (row - own.x);
    const int phys = at < p.kv.capacity ? page_of(p.kv, b, (int)(at >> p.kv.page_shift)) : -1;
    uint4 kw = make_uint4(0u, 0u, 0u, 0u), vw = kw;
    float ks = 0.f, vs = 0.f;
    if (phys >= 0) {
        const size_t block = (size_t)phys * p.kv.n_kv + h;
        const size_t off = ((block << p.kv.page_shift) + (at & (p.kv.page - 1))) * HD + 16 * c;
        kw = *reinterpret_cast<const uint4*>(p.kv.k + off);
        vw = *reinterpret_cast<const uint4*>(p.kv.v + off);
        ks = p.kv.k_scale[block] * kCodeUnit<DT>;
        vs = p.kv.v_scale[block] * kCodeUnit<DT>;
    }
    auto put = [&](const uint4& w, float s, __half* out) {
        const uint32_t in[4] = {w.x, w.y, w.z, w.w};
        __align__(16) __half2 o[8];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            uint32_t lo, hi;
            codes_to_half<DT>(in[u], lo, hi);
            const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), d = __half22float2(*reinterpret_cast<const __half2*>(&hi));
            o[2 * u] = __floats2half2_rn(a.x * s, a.y * s);
            o[2 * u + 1] = __floats2half2_rn(d.x * s, d.y * s);
        }
        uint4* dst = reinterpret_cast<uint4*>(out + ((size_t)row * p.kv.n_kv + h) * HD + 16 * c);
        dst[0] = reinterpret_cast<const uint4*>(o)[0];
        dst[1] = reinterpret_cast<const uint4*>(o)[1];
    };
    put(kw, ks, p.k_out);
    put(vw, vs, p.v_out);
}

// ---------------------------------------------------------------------------------------------
// Attention of few rows a key/value head (a decoded token: the heads of the group).  A warp takes 16 tokens a step; scores S^T
// = K q^T and outputs O^T += V^T P^T on m16n8k16 with the tokens resp. channels as M and eight rows (token of the call, head of the group) as N, so that codes
// go from 16-byte loads through a few register instructions into fragments:
//   keys    lane (g, t) loads tokens g and g + 8, 16-byte pieces t, t + 4, ..: any assignment of channels to k positions serves, as
//           long as q's fragments have the same.
//   values  lane (g, t) loads piece g of tokens 2t, 2t+1, 2t+8, 2t+9, the k positions of its fragment; bytes of two tokens are
//           interleaved, then expanded.
//   P       movmatrix transposes the scores' fragment (tokens by g) into the second product's (tokens by t).
// Scales: c = ks * scale * log2(e) multiplies a score; vs goes into the exponent, w = 2^(c s + log2 vs - m), so that probabilities are rounded
// to fp16 (the product's operand) relative to the largest contribution, which takes the results' error from 2.1e-4, their own rounding, to 2.4e-4 .. 2.9e-4
// (w in two halves, products of both: 2.1e-4 and 2 to 5 % of the time); the sum of the softmax is that of w / vs in fp32.  The maximum m is raised only when a score
// exceeds it by 2^8 (w stays below 256 in fp16), by a vote, so that a step has no shuffles as a rule.
// ---------------------------------------------------------------------------------------------
constexpr int kRowsWarps = 8, kRowsThreads = kRowsWarps * 32;
template <int NB> using RowsShare = ShareOf<8 * NB, 16 * kRowsWarps, 1, 1>;

// weighted values / sum of the weights -> four channels of a result row; a row that saw nothing is zero, not-a-number stays
__device__ __forceinline__ void store_result(__half* dst, const float4& acc, float sum, float unit) {
    const float inv = result_factor(sum, unit);
    __half2 o[2] = {__floats2half2_rn(acc.x * inv, acc.y * inv), __floats2half2_rn(acc.z * inv, acc.w * inv)};
    *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(o);
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
    return d;
}
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// (with the constant parts of the addresses in the instructions: added up in registers they were a fifth of the kernel's whole-number operations)
template <int DST, int SRC> __device__ __forceinline__ void copy_async_16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0+%2], [%1+%3], 16;" ::"r"(dst), "l"(src), "n"(DST), "n"(SRC) : "memory");
}
__device__ __forceinline__ void copy_async_4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
template <int WORDS, int OFF> __device__ __forceinline__ void lds_words(uint32_t a, uint32_t* w) {
    if (WORDS == 4)
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4+%5];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(a), "n"(OFF) : "memory");
    else if (WORDS == 2)
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2+%3];" : "=r"(w[0]), "=r"(w[1]) : "r"(a), "n"(OFF) : "memory");
    else
        asm volatile("ld.shared.u32 %0, [%1+%2];" : "=r"(w[0]) : "r"(a), "n"(OFF) : "memory");
}
template <int... I, class F> __device__ __forceinline__ void unrolled(std::integer_sequence<int, I...>, F&& f) { (f(std::integral_constant<int, I>{}), ...); }
// f(0), f(1), .. f(N - 1), the number a constant
template <int N, class F> __device__ __forceinline__ void unrolled(F&& f) { unrolled(std::make_integer_sequence<int, N>{}, f); }

// Shared memory of paged_attention_rows_kernel.  A warp has a ring of its own: S stages of 16 tokens, keys, then values, then the two scales.  A
// row's 16-byte pieces are stored at piece ^ swizzle(row), so that the fragments' loads (8 lanes together: two rows and four pieces of the keys, four
// rows, two apart, and two pieces of the values) meet 32 banks; with 64 channels the values' meet 16.  The rings and the warps' results share the space.
template <int HD, int NB> struct RowsCfg {
    static constexpr int R = 8 * NB, PIECES = HD / 16;
    static constexpr int STAGE = 32 * HD;
    static constexpr int S = HD == 32 ? 6 : HD == 64 ? 5 : 3;
    static constexpr int RING = S * STAGE;
    static constexpr int RESULTS = kRowsWarps * R * (HD + 2) * 4;
    static constexpr int RINGS = kRowsWarps * RING > RESULTS ? kRowsWarps * RING : RESULTS;
    static constexpr size_t SMEM = RINGS + kRowsWarps * S * 8, SMEM_CLUSTER = SMEM + R * (HD + 2) * 4;
    static constexpr int CTAS = HD == 256 || NB == 2 ? 1 : 2;
    static __device__ __forceinline__ int key_swizzle(int row) { return HD >= 128 ? (row & 1) << 2 : 0; }
    static __device__ __forceinline__ int value_swizzle(int row) { return HD >= 128 ? row & 6 : HD == 64 ? (row >> 1) & 3 : 0; }
};

__device__ __forceinline__ uint32_t cluster_ctas() {
    uint32_t n;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
    return n;
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t n;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(n));
    return n;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t smem_of(uint32_t a, uint32_t rank) {       // the same place in the shared memory of another CTA of the cluster
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    return r;
}

// CLUSTER: a cluster takes one segment, its CTAs equal parts of its tokens, and joins their results through shared memory: one launch and nothing to
// plan, for calls with few segments.
template <int HD, int DT, int NB, bool CLUSTER>
__global__ void __launch_bounds__(kRowsThreads, RowsCfg<HD, NB>::CTAS) paged_attention_rows_kernel(const AttnParams p) {
    using C = RowsCfg<HD, NB>;
    using Share = RowsShare<NB>;
    constexpr int R = C::R, S = C::S;               // rows of a block, stages
    constexpr int KW = HD / 16, VW = HD / 32;       // code words of a lane: per key row, per value row
    constexpr int KC = KW < 4 ? KW : 4, VC = VW < 4 ? VW : 4;       // words of one load
    extern __shared__ __align__(128) float sm_rows[];
    float* sm_o = sm_rows;                                         // [warp][R][HD]
    float* sm_m = sm_o + kRowsWarps * R * HD;                      // [warp][R]
    float* sm_l = sm_m + kRowsWarps * R;                           // [warp][R]
    __shared__ ShareStart sm_plan;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const uint32_t ring = smem_addr(sm_rows) + warp * C::RING, scales = smem_addr(sm_rows) + (uint32_t)C::RINGS + warp * S * 8;
    __shared__ SharedRows sm_q;
    after_launch_ahead();
    const PagedRows rows = rows_in_shared(p.r, sm_q);
    Pieces<Share> piece;
    if (CLUSTER) {
        const int i = blockIdx.z;
        piece.x = row_block<Share>(p.kv, rows, p.group, i, last_from(p.r.B, i, [&](int b) { return first_block<Share>(rows, p.group, b); }));
        if (piece.x.n_rows == 0) return;        // (all of the cluster)
        piece.h = blockIdx.y;
    } else {
        piece.template begin<kRowsThreads>(p.kv, rows, p.group, blockIdx.x, gridDim.x, sm_plan);
    }

    for (bool more = true; more && (CLUSTER || piece.next(p.kv, rows, p.group)); more = !CLUSTER) {
        const int b = piece.x.b, r0 = piece.x.r0, n_rows = piece.x.n_rows, start = piece.x.start, h = piece.h, step0 = piece.step0, step1 = piece.step1;
        const int2 own = piece.x.own;
        const int limit_all = min(start + (r0 + n_rows - 1) / p.group, p.kv.capacity - 1);       // the last key that a row sees
        // this CTA's tiles of 16 tokens
        const int all = limit_all / 16 + 1, share = CLUSTER ? (all + cluster_ctas() - 1) / cluster_ctas() : 0;
        const int tile_from = CLUSTER ? cluster_rank() * share : step0 * kRowsWarps, n_tiles = min(all, CLUSTER ? tile_from + share : step1 * kRowsWarps);

        uint32_t qf[NB][KW][2];
        int limit[NB][2];
        float m[NB][2], l[NB][2], o[NB][2 * VW][4];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            const int r = r0 + 8 * n + g;
            const bool live = 8 * n + g < n_rows;
            const __half* src = p.q + (long long)(own.x + (live ? r / p.group : 0)) * p.ldq + (h * p.group + (live ? r % p.group : 0)) * HD;
#pragma unroll
            for (int w = 0; w < KW; ++w) {
                const int ch = KW < 4 ? 8 * t + 4 * w : 64 * (w / 4) + 16 * t + 4 * (w % 4);
                const uint2 v = live ? *reinterpret_cast<const uint2*>(src + ch) : make_uint2(0u, 0u);
                qf[n][w][0] = v.x;
                qf[n][w][1] = v.y;
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int rr = 8 * n + 2 * t + e;
                limit[n][e] = rr < n_rows ? min(start + (r0 + rr) / p.group, p.kv.capacity - 1) : -1;
                m[n][e] = -1e30f;
                l[n][e] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < 2 * VW; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][i][e] = 0.f;
        }
        const int limit_low = min(start + r0 / p.group, p.kv.capacity - 1);       // keys up to here are seen by every live row

        // The warp's tiles are tile0 + 8 i.  Lane k has the page table's entry of tile i + k of the current 32, asked for together.
        const int tile0 = tile_from + warp, count = tile0 < n_tiles ? (n_tiles - tile0 + kRowsWarps - 1) / kRowsWarps : 0;
        auto pages_from = [&](int i) { return i + lane < count ? page_entry(p.kv, b, (tile0 + (i + lane) * kRowsWarps) * 16 >> p.kv.page_shift) : -1; };
        int pages = pages_from(0), pages_next = pages_from(32);
        auto request = [&](int i, int stage, int phys) {
            if (page_there(p.kv, phys)) {
                const size_t block = (size_t)phys * p.kv.n_kv + h;
                const size_t from = ((block << p.kv.page_shift) + (((tile0 + i * kRowsWarps) * 16) & (p.kv.page - 1))) * HD + lane * 16;
                // Pass u of the warp: rows 32 / PIECES u + lane / PIECES.  What the swizzles take from u is a constant too.
                constexpr int RPP = 32 / C::PIECES;
                const int row = lane / C::PIECES, c = lane % C::PIECES;
                const uint32_t at = ring + stage * C::STAGE, k_at = at + row * HD + ((c ^ C::key_swizzle(row)) << 4);
                const uint32_t v_off = row * HD + ((c ^ C::value_swizzle(row)) << 4);
                unrolled<(HD + 31) / 32>([&](auto u_) {
                    constexpr int u = decltype(u_)::value;
                    copy_async_16<u * 512, u * 512>(k_at ^ (C::key_swizzle(u * RPP) << 4), p.kv.k + from);
                    copy_async_16<16 * HD + u * 512, u * 512>(at + (v_off ^ (C::value_swizzle(u * RPP) << 4)), p.kv.v + from);
                });
                if (lane < 2) copy_async_4(scales + stage * 8 + lane * 4, (lane ? p.kv.v_scale : p.kv.k_scale) + block);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int i = 0; i < S - 1; ++i) request(i, i, __shfl_sync(0xffffffffu, pages, i));
        int stage = 0;
        for (int i = 0; i < count; ++i) {
            const int tile = tile0 + i * kRowsWarps;
            asm volatile("cp.async.wait_group %0;" ::"n"(S - 2) : "memory");
            __syncwarp();
            const int phys = __shfl_sync(0xffffffffu, pages, i & 31);
            {       // the stage that the tile before this one has left
                const int j = i + S - 1;
                request(j, stage == 0 ? S - 1 : stage - 1, __shfl_sync(0xffffffffu, (j ^ i) & 32 ? pages_next : pages, j & 31));
            }
            const uint32_t at = ring + stage * C::STAGE;
            float ks, vscale;
            asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(ks), "=f"(vscale) : "r"(scales + stage * 8) : "memory");
            uint32_t kw[2][KW], vw[4][VW];
            unrolled<KW / KC>([&](auto c_) {
                constexpr int c = decltype(c_)::value;
                const uint32_t a = at + (KC == 4 ? g * HD + (((t + 4 * (c & 1)) ^ C::key_swizzle(g)) << 4) : g * HD + t * 8);
                lds_words<KC, 64 * (c & ~1)>(a, &kw[0][KC * c]);
                lds_words<KC, 8 * HD + 64 * (c & ~1)>(a, &kw[1][KC * c]);          // (row g + 8 has row g's swizzle)
            });
            unrolled<VW / VC>([&](auto c_) {
                constexpr int c = decltype(c_)::value;
                // (so have 2t and 2t + 1, and 8 more)
                const uint32_t a = at + 2 * t * HD + (VC == 4 ? (g ^ C::value_swizzle(2 * t)) << 4
                                                    : VC == 2 ? (((g >> 1) ^ C::value_swizzle(2 * t)) << 4) + (g & 1) * 8 : g * 4);
                unrolled<4>([&](auto u_) {
                    constexpr int u = decltype(u_)::value;
                    lds_words<VC, 16 * HD + ((u & 1) + 8 * (u >> 1)) * HD + 128 * c>(a, &vw[u][VC * c]);
                });
            });
            float s[NB][4];
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
            for (int w = 0; w < KW; ++w) {
                uint32_t a0, a1, a2, a3;
                codes_to_half<DT>(kw[0][w], a0, a2);
                codes_to_half<DT>(kw[1][w], a1, a3);
#pragma unroll
                for (int n = 0; n < NB; ++n) mma16816(s[n], a0, a1, a2, a3, qf[n][w][0], qf[n][w][1]);
            }
            const bool there = page_there(p.kv, phys), masked = tile * 16 + 15 > limit_low || !there, live = there && live_scale(vscale);
            const float c = ks * p.scale2, lv = scale_log(vscale), iv = scale_inverse(vscale);
            // w of token g (+ 8) and rows 2t, 2t + 1 of each block of rows
            uint32_t pf[NB][2];
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                const int tok = tile * 16 + g;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[n][e] = s[n][e] * c + lv;
                    if (masked && (!there || tok + 8 * (e >> 1) > limit[n][e & 1])) s[n][e] = -INFINITY;
                }
                const float hi0 = fmaxf(s[n][0], s[n][2]), hi1 = fmaxf(s[n][1], s[n][3]);
                if (__any_sync(0xffffffffu, hi0 > m[n][0] + 8.f || hi1 > m[n][1] + 8.f)) {
                    float x0 = fmaxf(hi0, m[n][0]), x1 = fmaxf(hi1, m[n][1]);
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) {
                        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
                        x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
                    }
                    const float f0 = exp2_fast(m[n][0] - x0), f1 = exp2_fast(m[n][1] - x1);
                    m[n][0] = x0;
                    m[n][1] = x1;
                    l[n][0] *= f0;
                    l[n][1] *= f1;
#pragma unroll
                    for (int i = 0; i < 2 * VW; ++i) {
                        o[n][i][0] *= f0;
                        o[n][i][1] *= f1;
                        o[n][i][2] *= f0;
                        o[n][i][3] *= f1;
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][e] = exp2_fast(s[n][e] - m[n][e & 1]);
                l[n][0] += (s[n][0] + s[n][2]) * iv;
                l[n][1] += (s[n][1] + s[n][3]) * iv;
                pf[n][0] = transpose8x8(live ? pack_half2(s[n][0], s[n][1]) : 0u);
                pf[n][1] = transpose8x8(live ? pack_half2(s[n][2], s[n][3]) : 0u);
            }
#pragma unroll
            for (int w = 0; w < VW; ++w) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t sel = half ? 0x7362u : 0x5140u;
                    uint32_t a0, a1, a2, a3;
                    codes_to_half<DT>(prmt(vw[0][w], vw[1][w], sel), a0, a1);
                    codes_to_half<DT>(prmt(vw[2][w], vw[3][w], sel), a2, a3);
#pragma unroll
                    for (int n = 0; n < NB; ++n) mma16816(o[n][2 * w + half], a0, a1, a2, a3, pf[n][0], pf[n][1]);
                }
            }
            if (++stage == S) stage = 0;
            if ((i & 31) == 31) {
                pages = pages_next;
                pages_next = pages_from(i + 33);
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();
        // the warps' results meet in shared memory
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], d);
                const int r = 8 * n + 2 * t + e;
                if (g == 0) {
                    sm_m[warp * R + r] = m[n][e];
                    sm_l[warp * R + r] = l[n][e];
                }
                float* dst = sm_o + (warp * R + r) * HD;
#pragma unroll
                for (int w = 0; w < VW; ++w) {
                    const int ch = VW < 4 ? 4 * VW * g + 4 * w : 128 * (w / 4) + 16 * g + 4 * (w % 4);
                    *reinterpret_cast<float4*>(dst + ch) = make_float4(o[n][2 * w][e], o[n][2 * w][e + 2], o[n][2 * w + 1][e], o[n][2 * w + 1][e + 2]);
                }
            }
        __syncthreads();
        const bool whole = !CLUSTER && piece.whole();
        // partial results: for paged_join_kernel, or for the cluster
        float* part = CLUSTER ? sm_rows + C::SMEM / 4 : partial_of<Share, HD>(p.partial, blockIdx.x, step0 == 0);
        for (int i = threadIdx.x; i < n_rows * (HD / 4); i += kRowsThreads) {
            const int r = i / (HD / 4), ch = i % (HD / 4) * 4;
            float mx = -1e30f, sum = 0.f;
#pragma unroll
            for (int w = 0; w < kRowsWarps; ++w) mx = fmaxf(mx, sm_m[w * R + r]);
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kRowsWarps; ++w) {
                const float f = exp2_fast(sm_m[w * R + r] - mx);
                const float4 v = *reinterpret_cast<const float4*>(sm_o + (w * R + r) * HD + ch);
                sum += sm_l[w * R + r] * f;
                acc.x += v.x * f;
                acc.y += v.y * f;
                acc.z += v.z * f;
                acc.w += v.w * f;
            }
            if (whole) {
                store_result(p.out + (long long)(own.x + (r0 + r) / p.group) * p.ldo + (h * p.group + (r0 + r) % p.group) * HD + ch, acc, sum, kCodeUnit<DT>);
            } else {
                *reinterpret_cast<float4*>(part + r * HD + ch) = acc;
                if (ch == 0) *reinterpret_cast<float2*>(part + R * HD + 2 * r) = make_float2(mx, sum);
            }
        }
        if (CLUSTER) {
            cluster_sync();
            const uint32_t mine = smem_addr(part), n = cluster_ctas();
            for (int i = cluster_rank() * kRowsThreads + threadIdx.x; i < n_rows * (HD / 4); i += n * kRowsThreads) {
                const int r = i / (HD / 4), ch = i % (HD / 4) * 4;
                float mx = -1e30f, sum = 0.f;
                float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
                for (uint32_t c = 0; c < n; ++c) {
                    float2 ml;
                    float4 v;
                    asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(ml.x), "=f"(ml.y) : "r"(smem_of(mine + (R * HD + 2 * r) * 4, c)) : "memory");
                    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(smem_of(mine + (r * HD + ch) * 4, c)) : "memory");
                    const float top = fmaxf(mx, ml.x), f = exp2_fast(mx - top), w = exp2_fast(ml.x - top);
                    mx = top;
                    sum = sum * f + ml.y * w;
                    acc.x = acc.x * f + v.x * w;
                    acc.y = acc.y * f + v.y * w;
                    acc.z = acc.z * f + v.z * w;
                    acc.w = acc.w * f + v.w * w;
                }
                store_result(p.out + (long long)(own.x + (r0 + r) / p.group) * p.ldo + (h * p.group + (r0 + r) % p.group) * HD + ch, acc, sum, kCodeUnit<DT>);
            }
            cluster_sync();             // nobody leaves while its results are read
        } else {
            __syncthreads();
        }
    }
    if (!CLUSTER && threadIdx.x == 0) p.join[blockIdx.x] = join_item<Share>(piece.total, gridDim.x, blockIdx.x, sm_plan);
}

// Joins the partial results of segments that several CTAs shared: 32 rows of one a CTA.  Lane c looks at the maximum and sum of the c-th part, the
// values are added in the order of the shares.  A warp takes a row, and requests eight parts together; a prompt's segment has two parts as a rule and 256
// rows, and a warp requests two parts of four rows together (four chunks of 700 rows after 2900, 38 MB of partial results: 66 us with one row at a time,
// 62 with four).
template <int HD, int DT, class S>
__global__ void __launch_bounds__(kRowsThreads) paged_join_kernel(const AttnParams p) {
    constexpr int VPL = HD / 32;                     // channels of a lane
    constexpr int ROWS = S::R >= 128 ? 4 : 1, PARTS = 8 / ROWS;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    after_launch_ahead();
    const JoinItem x = p.join[blockIdx.x];
    const int n_rows = min(x.n_rows, (int)blockIdx.y * 32 + 32), c0 = x.first_cta, c1 = c0 + x.parts - 1;
    if (x.parts == 0) return;
    auto part_of = [&](int c) { return partial_of<S, HD>(p.partial, c, c == c0); };
    for (int r0 = blockIdx.y * 32 + warp; r0 < n_rows; r0 += kRowsWarps * ROWS) {
        float mx[ROWS], sum[ROWS], acc[ROWS][VPL];
        int row[ROWS];
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
            row[k] = min(r0 + k * kRowsWarps, n_rows - 1);          // (the last row again where there are no more)
            mx[k] = -1e30f;
            sum[k] = 0.f;
#pragma unroll
            for (int i = 0; i < VPL; ++i) acc[k][i] = 0.f;
        }
        for (int base = c0; base <= c1; base += 32) {
            const int c = base + lane, n = min(32, c1 - base + 1);
            float2 ml[ROWS];
#pragma unroll
            for (int k = 0; k < ROWS; ++k) ml[k] = c <= c1 ? *reinterpret_cast<const float2*>(part_of(c) + S::R * HD + 2 * row[k]) : make_float2(-1e30f, 0.f);
            float w[ROWS];
#pragma unroll
            for (int k = 0; k < ROWS; ++k) {
                float top = fmaxf(ml[k].x, mx[k]);
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                const float f = exp2_fast(mx[k] - top);
                w[k] = exp2_fast(ml[k].x - top);
                mx[k] = top;
                sum[k] = sum[k] * f + warp_sum(ml[k].y * w[k]);
#pragma unroll
                for (int i = 0; i < VPL; ++i) acc[k][i] *= f;
            }
            for (int u0 = 0; u0 < n; u0 += PARTS) {
                float v[ROWS][PARTS][VPL];
#pragma unroll
                for (int k = 0; k < ROWS; ++k)
#pragma unroll
                    for (int u = 0; u < PARTS; ++u) {
                        const float* src = part_of(base + u0 + u) + row[k] * HD + lane * VPL;
#pragma unroll
                        for (int i = 0; i < VPL; i += VPL < 4 ? VPL : 4) {
                            float* to = v[k][u] + i;
                            const bool there = u0 + u < n;
                            if constexpr (VPL >= 4) {
                                const float4 t = there ? *reinterpret_cast<const float4*>(src + i) : make_float4(0.f, 0.f, 0.f, 0.f);
                                to[0] = t.x, to[1] = t.y, to[2] = t.z, to[3] = t.w;
                            } else if constexpr (VPL == 2) {
                                const float2 t = there ? *reinterpret_cast<const float2*>(src) : make_float2(0.f, 0.f);
                                to[0] = t.x, to[1] = t.y;
                            } else {
                                to[0] = there ? *src : 0.f;
                            }
                        }
                    }
#pragma unroll
                for (int k = 0; k < ROWS; ++k)
#pragma unroll
                    for (int u = 0; u < PARTS; ++u) {
                        const float wu = __shfl_sync(0xffffffffu, w[k], u0 + u);
#pragma unroll
                        for (int i = 0; i < VPL; ++i) acc[k][i] += v[k][u][i] * wu;
                    }
            }
        }
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
            if (r0 + k * kRowsWarps >= n_rows) break;
            const float inv = result_factor(sum[k], kCodeUnit<DT>);
            const int r = x.r0 + row[k];
            __half* dst = p.out + (long long)(x.row + r / p.group) * p.ldo + (x.h * p.group + r % p.group) * HD + lane * VPL;
            if constexpr (VPL == 1) {
                *dst = __float2half_rn(acc[k][0] * inv);
            } else {
                uint32_t o[VPL / 2];
#pragma unroll
                for (int i = 0; i < VPL / 2; ++i) o[i] = pack_half2(acc[k][2 * i] * inv, acc[k][2 * i + 1] * inv);
                if constexpr (VPL == 2) *reinterpret_cast<uint32_t*>(dst) = o[0];
                if constexpr (VPL == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(o[0], o[1]);
                if constexpr (VPL == 8) *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
int sm_count() {
    int dev = 0, n = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    return n;
}
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int check_cache(const glq_paged_kv_t* kv, const glq_paged_rows_t* r) {
    if (!kv || !r || !kv->k_pages || !kv->v_pages || !kv->k_scale || !kv->v_scale || !kv->table || !r->start) return GLQ_ERR_ARG;
    if (kv->dtype != GLQ_KV_I8 && kv->dtype != GLQ_KV_E4M3) return GLQ_ERR_UNSUPPORTED;
    if (kv->head_dim != 32 && kv->head_dim != 64 && kv->head_dim != 128 && kv->head_dim != 256) return GLQ_ERR_UNSUPPORTED;
    if (kv->page != 16 && kv->page != 32 && kv->page != 64 && kv->page != 128) return GLQ_ERR_UNSUPPORTED;
    if (kv->n_pages <= 0 || kv->n_kv <= 0 || kv->max_pages <= 0 || kv->table_stride < kv->max_pages) return GLQ_ERR_ARG;
    if ((long long)kv->max_pages * kv->page >= 1 << 30 || kv->n_kv > 1024) return GLQ_ERR_UNSUPPORTED;
    if (r->B < 0 || r->rows < 0 || r->rows >= 1 << 28 || (r->start_stride != 0 && r->start_stride != 1)) return GLQ_ERR_ARG;
    if (!r->q_start && r->B > 0 && r->rows % r->B != 0) return GLQ_ERR_ARG;
    if (!aligned16(kv->k_pages) || !aligned16(kv->v_pages)) return GLQ_ERR_ALIGN;
    return GLQ_OK;
}
PagedKv device_kv(const glq_paged_kv_t* kv) {
    int shift = 0;
    while ((1 << shift) < kv->page) ++shift;
    return {static_cast<unsigned char*>(kv->k_pages), static_cast<unsigned char*>(kv->v_pages), kv->k_scale, kv->v_scale, kv->table,
            kv->table_stride, kv->n_pages, kv->n_kv, kv->page, shift, kv->max_pages, kv->max_pages * kv->page};
}
PagedRows device_rows(const glq_paged_rows_t* r) {
    return {reinterpret_cast<const long long*>(r->start), r->q_start, r->B, r->rows, r->q_start ? 0 : r->rows / r->B, r->start_stride};
}

// f<head size, code type>()
template <class F> int by_type(const glq_paged_kv_t* kv, F&& f) {
#define GLQ_PAGED_CASE(HD)                                                                             \
    case HD:                                                                                           \
        return kv->dtype == GLQ_KV_I8 ? f(std::integral_constant<int, HD>{}, std::integral_constant<int, kI8>{}) \
                                      : f(std::integral_constant<int, HD>{}, std::integral_constant<int, kE4M3>{});
    switch (kv->head_dim) {
        GLQ_PAGED_CASE(32)
        GLQ_PAGED_CASE(64)
        GLQ_PAGED_CASE(128)
        GLQ_PAGED_CASE(256)
    }
#undef GLQ_PAGED_CASE
    return GLQ_ERR_UNSUPPORTED;
}

}  // namespace

extern "C" int glq_paged_append(const glq_paged_kv_t* kv, const glq_paged_rows_t* rows, const void* q, int64_t ldq, const void* k, int64_t ldk,
                                const void* v, int64_t ldv, void* q_out, int64_t ldqo, int n_heads, const float* cos, const float* sin,
                                int cos_rows, const void* q_norm, const void* k_norm, float eps, void* stream) {
    const int bad = check_cache(kv, rows);
    if (bad != GLQ_OK) return bad;
    if (rows->rows == 0 || rows->B == 0) return GLQ_OK;
    if (!k || !v || (q && (!q_out || n_heads <= 0)) || (!cos != !sin) || (!q_norm != !k_norm && q)) return GLQ_ERR_ARG;
    if (cos && cos_rows < kv->max_pages * kv->page) return GLQ_ERR_ARG;
    const int width = kv->n_kv * kv->head_dim;
    if (ldk < width || ldv < width || (q && (ldq < (int64_t)n_heads * kv->head_dim || ldqo < (int64_t)n_heads * kv->head_dim))) return GLQ_ERR_ARG;
    if (ldk % 8 || ldv % 8 || (q && (ldq % 8 || ldqo % 8))) return GLQ_ERR_ALIGN;
    for (const void* ptr : {k, v, q, (const void*)q_out, (const void*)cos, (const void*)sin, q_norm, k_norm})
        if (!aligned16(ptr)) return GLQ_ERR_ALIGN;
    return by_type(kv, [&](auto hd, auto dt) {
        constexpr int HD = decltype(hd)::value, DT = decltype(dt)::value;
        AppendParams p{device_kv(kv), device_rows(rows), static_cast<const __half*>(q), static_cast<const __half*>(k),
                       static_cast<const __half*>(v), static_cast<const __half*>(q_norm), static_cast<const __half*>(k_norm),
                       static_cast<__half*>(q_out), cos, sin, ldq, ldk, ldv, ldqo, n_heads, 0, cos_rows, 1, 1, 1, eps};
        if (q) p.query_rows = std::max(1, kAppendThreads / (HD / 16) / n_heads);
        // Two turns where the queries are several waves of CTAs: more loads are on their way.  Measured (graph, us, one / two): four sequences of 1024 tokens,
        // 32 heads on 4, 25.4 / 21.0; 4096 tokens, 16 heads of their own 30.7 / 27.9, 8 on 2 of 256 channels 21.9 / 19.0, 32 on 8 23.8 / 23.7; 512 tokens,
        // 16 heads 5.7 / 5.8.  With norms: four of 1024, 32 on 4, 21.6 / 19.1; 4096 tokens, 16 heads 35.6 / 28.5, 8 on 2 of 256 22.5 / 20.1, 32 on 8 26.1 / 26.2
        // and into e4m3 30.8 / 30.8; 64 of 128 tokens, 32 on 4, into e4m3 50.5 / 46.2.
        if (q && rows->rows / p.query_rows >= 2 * kAppendCtas * sm_count()) p.query_turns = kQueryTurns;
        const long long items = (long long)rows->rows / kv->page + 2ll * rows->B;
        const int query_rows = p.query_rows * p.query_turns;          // of a CTA
        const long long grid = items * 2 * kv->n_kv + (q ? (rows->rows + query_rows - 1) / query_rows : 0);
        if (items * 2 * kv->n_kv > 0x3fffffffll || grid > 0x7fffffffll) return GLQ_ERR_UNSUPPORTED;
        p.page_items = (int)items;
        p.stride = (int)std::max<long long>(1, grid / (items * 2 * kv->n_kv));
        return launch_kernel(true, paged_append_kernel<HD, DT>, dim3((unsigned)grid), dim3(kAppendThreads), 0,
                             reinterpret_cast<cudaStream_t>(stream), p) == cudaSuccess ? GLQ_OK : GLQ_ERR_CUDA;
    });
}

extern "C" int glq_paged_read(const glq_paged_kv_t* kv, const glq_paged_rows_t* rows, void* k_out, void* v_out, void* stream) {
    const int bad = check_cache(kv, rows);
    if (bad != GLQ_OK) return bad;
    if (rows->rows == 0 || rows->B == 0) return GLQ_OK;
    if (!k_out || !v_out) return GLQ_ERR_ARG;
    if (!aligned16(k_out) || !aligned16(v_out)) return GLQ_ERR_ALIGN;
    return by_type(kv, [&](auto hd, auto dt) {
        constexpr int HD = decltype(hd)::value, DT = decltype(dt)::value;
        const ReadParams p{device_kv(kv), device_rows(rows), static_cast<__half*>(k_out), static_cast<__half*>(v_out)};
        const long long grid = ((long long)rows->rows * kv->n_kv + kReadThreads / (HD / 16) - 1) / (kReadThreads / (HD / 16));
        if (grid > 0x7fffffffll) return GLQ_ERR_UNSUPPORTED;
        return launch_kernel(true, paged_read_kernel<HD, DT>, dim3((unsigned)grid), dim3(kReadThreads), 0, reinterpret_cast<cudaStream_t>(stream),
                             p) == cudaSuccess ? GLQ_OK : GLQ_ERR_CUDA;
    });
}

// How a call runs, from what the host knows: the lengths are on the device, what it has is the room of the table.
enum class AttnKernel { rows8, rows16, prompt };
struct AttnPlan {
    AttnKernel kernel;
    int grid;
    size_t partial;        // floats of a partial result
    bool fits;
    int cluster;           // CTAs of a cluster that takes a segment, 0: equal shares of all
};
// a launch beside the one ahead (launch_kernel) of clusters of `ctas` CTAs along x
template <typename K, typename A> cudaError_t launch_cluster(K* kern, dim3 grid, dim3 block, int ctas, size_t smem, cudaStream_t st, const A& arg) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_disabled() ? 1 : 2;
    return cudaLaunchKernelEx(&cfg, kern, arg);
}
AttnPlan plan_attention(const glq_paged_kv_t* kv, const glq_paged_rows_t* rows, int n_heads) {
    const long long most = (rows->q_start ? std::min(rows->max_new, rows->rows) : rows->rows / rows->B) * (long long)(n_heads / kv->n_kv);
    const int D = kv->head_dim;
    auto make = [&](AttnKernel kernel, int ctas, auto share) -> AttnPlan {
        using S = decltype(share);
        AttnPlan a{kernel, sm_count() * ctas, (size_t)S::R * (D + 2), units_fit<S>(rows->rows, rows->B, n_heads / kv->n_kv, kv->n_kv, kv->max_pages * kv->page), 0};
        // A cluster a segment, as large as leaves all resident, where the longest sequence that the table holds gives a CTA at most 2048 tokens.  Measured
        // (graph, us, equal shares / clusters): 16 heads of their own after 512 tokens 7.9 / 5.8; 16 sequences of 1000 tokens, 8 heads, 16.7 / 12.3; one of
        // 16000, 8 heads, 17.1 / 17.1; 64 of 2000, 4 heads, lengths alike 34.7 / 30.3 and ragged 28.0 / 26.3; 64 of up to 8192, ragged, 60 / 75.
        const long long segments = (most + S::R - 1) / S::R * rows->B * kv->n_kv;
        if (kernel != AttnKernel::prompt && block_count<S>(rows->rows, rows->B, n_heads / kv->n_kv) <= 65535) {
            int c = 8;
            while (c > 1 && segments * c > a.grid) c >>= 1;
            if (kv->max_pages * kv->page <= 2048 * c) a.cluster = c;
        }
        return a;
    };
    // From 64 channels on, 256 (128) rows of a head at once on the 5th-generation tensor cores, where that is much work: those tiles multiply four times
    // as fast, but a call begins and joins slower, and a tile that is not full costs as much as a full one.  Measured (graph, us, tiles of 16 / prompt
    // kernel; 128 channels, 8 heads, 4 rows of q a token): 16 tokens after 1000 8.8 / 21, 64 after 1000 14 / 27 and after 4000 39 / 30, 128 after 1000
    // 27 / 28 and after 4000 64 / 32, 256 after none 28 / 19 and after 4000 117 / 40; 16 sequences of 32 tokens, 16 heads of their own (32 rows), after
    // 1000 55 / 62 and after 4000 119 / 147, of 64 tokens 98 / 63 and 220 / 147.  256 channels, 2 heads: 64 tokens after 4000 22 / 31, 128 after 4000
    // 45 / 32; 64 channels, 4 heads: 128 after 4000 27 / 24, 256 after 4000 44 / 26 (a row there costs tiles of 16 nearly what one of 128 does).
    const long long every = most * rows->B * kv->n_kv;
    if (D >= 64 && most > 32 && (every > 4096 || every * std::max(D, 128) > (1ll << 30) / ((long long)kv->max_pages * kv->page)))
        return D == 256 ? make(AttnKernel::prompt, 1, PromptShape<256>::Share{}) : make(AttnKernel::prompt, 1, PromptShape<128>::Share{});
    if (most > 8) return make(AttnKernel::rows16, 1, RowsShare<2>{});
    return make(AttnKernel::rows8, D == 256 ? 1 : 2, RowsShare<1>{});
}
int check_attention(const glq_paged_kv_t* kv, const glq_paged_rows_t* rows, int n_heads) {
    const int bad = check_cache(kv, rows);
    if (bad != GLQ_OK) return bad;
    if (n_heads <= 0 || n_heads % kv->n_kv != 0 || (rows->q_start && rows->max_new < 0)) return GLQ_ERR_ARG;
    if ((long long)rows->rows * n_heads + rows->B > 0x7fffffffll) return GLQ_ERR_UNSUPPORTED;
    return GLQ_OK;
}

extern "C" size_t glq_paged_attention_workspace_bytes(const glq_paged_kv_t* kv, const glq_paged_rows_t* rows, int n_heads) {
    if (check_attention(kv, rows, n_heads) != GLQ_OK || rows->rows == 0 || rows->B == 0) return 0;
    const AttnPlan a = plan_attention(kv, rows, n_heads);
    return a.cluster ? 0 : (size_t)a.grid * (sizeof(JoinItem) + 2 * a.partial * sizeof(float));
}

extern "C" int glq_paged_attention(const glq_paged_kv_t* kv, const glq_paged_rows_t* rows, const void* q, int64_t ldq, void* out,
                                   int64_t ldo, int n_heads, float scale, void* workspace, size_t workspace_bytes, void* stream) {
    const int bad = check_attention(kv, rows, n_heads);
    if (bad != GLQ_OK) return bad;
    if (rows->rows == 0 || rows->B == 0) return GLQ_OK;
    if (!q || !out || !(scale >= 0.f && scale <= FLT_MAX) || ldq < (int64_t)n_heads * kv->head_dim || ldo < (int64_t)n_heads * kv->head_dim) return GLQ_ERR_ARG;
    if (ldq % 8 || ldo % 8 || !aligned16(q) || !aligned16(out)) return GLQ_ERR_ALIGN;
    const AttnPlan plan = plan_attention(kv, rows, n_heads);
    if (!plan.fits) return GLQ_ERR_UNSUPPORTED;
    const size_t bytes = glq_paged_attention_workspace_bytes(kv, rows, n_heads);
    if (bytes && (!workspace || workspace_bytes < bytes)) return GLQ_ERR_WORKSPACE;
    if (!aligned16(workspace)) return GLQ_ERR_ALIGN;
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    return by_type(kv, [&](auto hd, auto dt) {
        constexpr int HD = decltype(hd)::value, DT = decltype(dt)::value;
        const int group = n_heads / kv->n_kv;
        const AttnParams p{device_kv(kv), device_rows(rows), static_cast<const __half*>(q), static_cast<__half*>(out), ldq, ldo,
                           group, scale * 1.4426950408889634f * kCodeUnit<DT>, static_cast<JoinItem*>(workspace),
                           reinterpret_cast<float*>(static_cast<JoinItem*>(workspace) + plan.grid)};
        auto join = [&](auto share) {
            using S = decltype(share);
            const dim3 grid((unsigned)plan.grid, (S::R + 31) / 32);
            return launch_kernel(true, paged_join_kernel<HD, DT, S>, grid, dim3(kRowsThreads), 0, st, p) == cudaSuccess ? GLQ_OK : GLQ_ERR_CUDA;
        };
        auto run = [&](auto nb) {
            constexpr int NB = decltype(nb)::value;
            if (plan.cluster) {
                static SmemLimit limit;
                auto* kern = paged_attention_rows_kernel<HD, DT, NB, true>;
                constexpr size_t smem = RowsCfg<HD, NB>::SMEM_CLUSTER;
                const dim3 grid((unsigned)plan.cluster, (unsigned)kv->n_kv, (unsigned)block_count<RowsShare<NB>>(rows->rows, rows->B, group));
                return reserve_smem(reinterpret_cast<const void*>(kern), limit, smem) == cudaSuccess &&
                               launch_cluster(kern, grid, dim3(kRowsThreads), plan.cluster, smem, st, p) == cudaSuccess
                           ? GLQ_OK : GLQ_ERR_CUDA;
            }
            static SmemLimit limit;
            auto* kern = paged_attention_rows_kernel<HD, DT, NB, false>;
            if (reserve_smem(reinterpret_cast<const void*>(kern), limit, RowsCfg<HD, NB>::SMEM) != cudaSuccess ||
                launch_kernel(true, kern, dim3((unsigned)plan.grid), dim3(kRowsThreads), RowsCfg<HD, NB>::SMEM, st, p) != cudaSuccess)
                return GLQ_ERR_CUDA;
            return join(RowsShare<NB>{});
        };
        if constexpr (HD >= 64)
            if (plan.kernel == AttnKernel::prompt)
                return launch_paged_prompt(HD, DT, p, plan.grid, st) == cudaSuccess ? join(typename PromptShape<HD>::Share{}) : GLQ_ERR_CUDA;
        return plan.kernel == AttnKernel::rows8 ? run(std::integral_constant<int, 1>{}) : run(std::integral_constant<int, 2>{});
    });
}
