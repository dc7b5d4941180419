// Attention of many rows a key/value head (pieces of prompts) over the paged 8-bit cache, on tcgen05.
//
// Segment: 256 rows (token of the call, head of the group), two tiles of 128, of one (sequence, key/value head); step: 128 tokens.
// A step's products are S = Q K^T (operands in shared memory) and O += P V (P in tensor memory, over the scores that it is made of; V as it
// lies, tokens by channels, which is the MN-major form of the operand).  Tensor memory: S of both tiles, O of both tiles.
//
// Warps, which keep their roles over all segments of a CTA:
//   0..3, 4..7  softmax of tile 0 and 1: a thread has a row; reads S twice (maximum; exponentials), writes P as fp16; brings the row's Q to
//               shared memory, multiplies O where the maximum has grown, writes the result
//   8..15       codes to fp16 operands in shared memory, 16 tokens of a step each, so that one page, one pair of scales, is a warp's
//   16          issues the MMAs: P V of one tile, then the next S of it (whose columns P held until then), then the other tile's, so that
//               one tile's products run while the other's softmax does
// Scales and maximum as in paged_attention_rows_kernel: w = 2^(ks s + log2 vs - m) in fp16, the sum of w / vs in fp32, m raised only when a
// score exceeds it by 2^8.
//
// Every wait is bounded (tc_wait); a wait that runs out marks the CTA dead, all roles leave their loops and the kernel ends.
#include "paged.cuh"
#include "tc_mm.cuh"

// error word of this translation unit, merged by glq_debug_error
int glq_paged_error_words(unsigned long long* out4, int clear) {
    if (cudaMemcpyFromSymbol(out4, glq::g_glq_err, 4 * sizeof(unsigned long long)) != cudaSuccess) return GLQ_ERR_CUDA;
    if (clear) {
        const unsigned long long z[4] = {0, 0, 0, 0};
        if (cudaMemcpyToSymbol(glq::g_glq_err, z, sizeof(z)) != cudaSuccess) return GLQ_ERR_CUDA;
    }
    return GLQ_OK;
}

namespace glq {
namespace {

constexpr int kPromptSoftmax = 8, kPromptProducers = 8, kPromptMma = kPromptSoftmax + kPromptProducers;
constexpr int kPromptThreads = (kPromptMma + 1) * 32;
constexpr int kStepTokens = PromptShare::STEP, kGroups = kStepTokens / 16;

template <int HD> struct PromptCfg {
    static constexpr int TILE = 128 * HD * 2;            // an operand: [64-channel block][128 rows][128 B], 16-byte piece c of row r at c ^ (r & 7)
    static constexpr size_t SMEM = 6 * TILE + 1024;      // Q of two tiles, K and V of two stages
    static constexpr uint32_t S_COL = 0, O_COL = 256;
};

__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, volatile int* dead, int code) {
    return __all_sync(0xffffffffu, mbar_try_wait(bar, parity) || tc_wait(bar, parity, dead, code));
}
__device__ __forceinline__ void arrive_warp(uint32_t bar, int lane) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
}
__device__ __forceinline__ void commit_warp(uint32_t bar) {
    asm volatile(
        "{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
        " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(bar)
        : "memory");
}
// Four k steps, issued by one elected lane of the converged warp: both operands K-major in shared memory (32 B a step) ..
__device__ __forceinline__ void mma4_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p, o, e;\n .reg .b64 a1, a2, a3, b1, b2, b3;\n"
        " setp.ne.b32 p, %4, 0;\n setp.eq.b32 o, 0, 0;\n"
        " add.u64 a1, %1, 2;\n add.u64 a2, %1, 4;\n add.u64 a3, %1, 6;\n"
        " add.u64 b1, %2, 2;\n add.u64 b2, %2, 4;\n add.u64 b3, %2, 6;\n"
        " elect.sync _|e, 0xffffffff;\n"
        " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
        " @e tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, o;\n"
        " @e tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, o;\n"
        " @e tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, o;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
// .. the first in tensor memory (8 columns a step), the second MN-major (16 tokens, 2048 B, a step)
__device__ __forceinline__ void mma4_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p, o, e;\n .reg .b32 a1, a2, a3;\n .reg .b64 b1, b2, b3;\n"
        " setp.ne.b32 p, %4, 0;\n setp.eq.b32 o, 0, 0;\n"
        " add.u32 a1, %1, 8;\n add.u32 a2, %1, 16;\n add.u32 a3, %1, 24;\n"
        " add.u64 b1, %2, 128;\n add.u64 b2, %2, 256;\n add.u64 b3, %2, 384;\n"
        " elect.sync _|e, 0xffffffff;\n"
        " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
        " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, o;\n"
        " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, o;\n"
        " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, o;\n}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
// MN-major operand, 128-byte swizzle: 64-channel blocks 128 rows apart, groups of 8 tokens 1024 B apart
__device__ __forceinline__ uint64_t value_desc(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(16384 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
        "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
          "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
          "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr)
        : "memory");
}
template <int N> __device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t* v) {
    static_assert(N == 16, "");
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
                 "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
                 "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// What a role needs of a piece: per tile its rows, the last key that one of them sees, and the steps that it takes part in.
struct TileView {
    int rows, steps;
};
__device__ __forceinline__ TileView tile_view(const Pieces<PromptShare>& piece, const AttnParams& p, int tile) {
    TileView v;
    v.rows = max(0, min(piece.x.n_rows - 128 * tile, 128));
    const int last = min(piece.x.start + (piece.x.r0 + 128 * tile + v.rows - 1) / p.group, p.kv.capacity - 1);
    v.steps = v.rows > 0 ? max(0, min(piece.step1, last / kStepTokens + 1) - piece.step0) : 0;
    return v;
}

template <int HD, int DT>
__global__ void __launch_bounds__(kPromptThreads, 1) paged_prompt_kernel(const AttnParams p) {
    using C = PromptCfg<HD>;
    extern __shared__ unsigned char prompt_smem[];
    __shared__ __align__(8) unsigned long long bars[2 * 9];
    __shared__ float s_scale[2][3][kGroups];           // of a stage: ks, log2 vs, 1 / vs of its groups of 16 tokens
    __shared__ long long sm_plan[kPromptThreads / 32 + 3];
    __shared__ uint32_t s_tmem;
    __shared__ int s_dead;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = (smem_u32(prompt_smem) + 1023u) & ~1023u;
    const uint32_t q_smem = base, k_smem = base + 2 * C::TILE, v_smem = base + 4 * C::TILE;
    // [0], [1] of each: stages or tiles
    const uint32_t k_full = smem_u32(bars), k_empty = k_full + 16, v_full = k_full + 32, v_empty = k_full + 48, s_full = k_full + 64,
                   p_ready = k_full + 80, pv_done = k_full + 96, q_ready = k_full + 112, o_free = k_full + 128;
    volatile int* dead = &s_dead;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(k_full + 8 * i, kPromptProducers);
            mbar_init(v_full + 8 * i, kPromptProducers);
            mbar_init(k_empty + 8 * i, 1);
            mbar_init(v_empty + 8 * i, 1);
            mbar_init(s_full + 8 * i, 1);
            mbar_init(pv_done + 8 * i, 1);
            mbar_init(p_ready + 8 * i, 4);
            mbar_init(q_ready + 8 * i, 4);
            mbar_init(o_free + 8 * i, 4);
        }
        s_dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kPromptMma) tc_alloc(smem_u32(&s_tmem), 512);
    tc_fence_before();
    after_launch_ahead();
    Pieces<PromptShare> piece;
    piece.template begin<kPromptThreads>(p.kv, p.r, p.group, blockIdx.x, gridDim.x, sm_plan);
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    uint32_t gs = 0;                     // steps of the pieces before, over all roles alike
    bool ok = true;

    if (warp < kPromptSoftmax) {
        // ================= softmax: a row a thread =================
        const int tile = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t trow = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t s_tm = trow + C::S_COL + tile * 128, o_tm = trow + C::O_COL + tile * HD;
        uint32_t done = 0;               // this tile's steps of the pieces before
        while (ok && piece.next(p.kv, p.r, p.group)) {
            const TileView view = tile_view(piece, p, tile);
            const int steps = max(view.steps, tile_view(piece, p, tile ^ 1).steps);
            const bool live = row < view.rows;
            const int r = piece.x.r0 + 128 * tile + row, token = live ? r / p.group : 0, head = piece.h * p.group + (live ? r - token * p.group : 0);
            const int limit = live ? min(piece.x.start + token, p.kv.capacity - 1) : -1;
            const int limit_low = min(piece.x.start + (piece.x.r0 + 128 * tile) / p.group, p.kv.capacity - 1);       // every live row sees keys up to here
            if (view.steps > 0) {
                const __half* src = p.q + (long long)(piece.x.own.x + token) * p.ldq + head * HD;
                const uint32_t dst = q_smem + tile * C::TILE + row * 128;
#pragma unroll
                for (int c = 0; c < HD / 8; ++c) {
                    const uint4 v = live ? *reinterpret_cast<const uint4*>(src + 8 * c) : make_uint4(0u, 0u, 0u, 0u);
                    sts128(dst + (c >> 3) * 16384 + (((c & 7) ^ (row & 7)) << 4), v.x, v.y, v.z, v.w);
                }
                fence_async_smem();
                arrive_warp(q_ready + 8 * tile, lane);
            }
            float m = -1e30f, l = 0.f;
            for (int j = 0; j < view.steps && ok; ++j) {
                const uint32_t g = gs + j;
                ok = wait_warp(s_full + 8 * tile, done & 1, dead, 120) && wait_warp(v_full + 8 * (g & 1), (g >> 1) & 1, dead, 121);
                if (!ok) break;
                tc_fence_after();
                const float* scale = s_scale[g & 1][0];
                const int first = (piece.step0 + j) * kStepTokens;
                const bool masked = first + kStepTokens - 1 > limit_low;
                const int see = limit - first;                    // columns up to here are this row's
                float top = -INFINITY;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t v[32];
                    tmem_ld32(s_tm + 32 * c, v);
                    tc_ld_wait();
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const int grp = 2 * c + half;
                        float x = -INFINITY;
                        if (masked) {
#pragma unroll
                            for (int i = 0; i < 16; ++i) x = fmaxf(x, 16 * grp + i <= see ? __uint_as_float(v[16 * half + i]) : -INFINITY);
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; ++i) x = fmaxf(x, __uint_as_float(v[16 * half + i]));
                        }
                        // (nothing to see: not 0 times infinity)
                        top = fmaxf(top, x == -INFINITY ? -INFINITY : x * (scale[grp] * p.scale2) + scale[kGroups + grp]);
                    }
                }
                if (__any_sync(0xffffffffu, top > m + 8.f)) {
                    const float up = fmaxf(m, top), f = exp2_fast(m - up);
                    m = up;
                    l *= f;
                    if (j > 0) {          // (the product before this step's scores has been added)
#pragma unroll
                        for (int c = 0; c < HD / 16; ++c) {
                            uint32_t v[16];
                            tc_ld16(o_tm + 16 * c, v);
                            tc_ld_wait();
#pragma unroll
                            for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
                            tmem_st<16>(o_tm + 16 * c, v);
                        }
                    }
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t v[32], w[16];
                    tmem_ld32(s_tm + 32 * c, v);
                    tc_ld_wait();
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const int grp = 2 * c + half;
                        const float cs = scale[grp] * p.scale2, off = scale[kGroups + grp] - m, iv = scale[2 * kGroups + grp];
                        float sum = 0.f;
#pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            float a = exp2_fast(__uint_as_float(v[16 * half + i]) * cs + off), b = exp2_fast(__uint_as_float(v[16 * half + i + 1]) * cs + off);
                            if (masked) {
                                a = 16 * grp + i <= see ? a : 0.f;
                                b = 16 * grp + i + 1 <= see ? b : 0.f;
                            }
                            sum += a + b;
                            w[8 * half + i / 2] = pack_half2(a, b);
                        }
                        l += sum * iv;
                    }
                    tmem_st<16>(s_tm + 16 * c, w);
                }
                tmem_st_wait();
                tc_fence_before();
                arrive_warp(p_ready + 8 * tile, lane);
                ++done;
            }
            if (ok && view.steps > 0) ok = wait_warp(pv_done + 8 * tile, (done - 1) & 1, dead, 122);
            if (!ok) break;
            tc_fence_after();
            if (view.rows > 0) {
                const bool whole = piece.whole();
                const float f = result_factor(l, kCodeUnit<DT>);
                __half* out = p.out + (long long)(piece.x.own.x + token) * p.ldo + head * HD;
                float* part = partial_of<PromptShare, HD>(p.partial, blockIdx.x, piece.step0 == 0);
                float* mine = part + (128 * tile + row) * HD;
#pragma unroll
                for (int c = 0; c < HD / 16; ++c) {
                    uint32_t v[16];
                    if (view.steps > 0) {
                        tc_ld16(o_tm + 16 * c, v);
                        tc_ld_wait();
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] = 0u;
                    }
                    if (live && whole) {
                        uint32_t o[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) o[i] = pack_half2(__uint_as_float(v[2 * i]) * f, __uint_as_float(v[2 * i + 1]) * f);
                        *reinterpret_cast<uint4*>(out + 16 * c) = make_uint4(o[0], o[1], o[2], o[3]);
                        *reinterpret_cast<uint4*>(out + 16 * c + 8) = make_uint4(o[4], o[5], o[6], o[7]);
                    } else if (live) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) reinterpret_cast<uint4*>(mine + 16 * c)[i] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                    }
                }
                if (live && !whole) *reinterpret_cast<float2*>(part + PromptShare::R * HD + 2 * (128 * tile + row)) = make_float2(m, l);
            }
            tc_fence_before();
            if (view.steps > 0) arrive_warp(o_free + 8 * tile, lane);
            gs += steps;
        }
    } else if (warp < kPromptMma) {
        // ================= codes to operands =================
        constexpr int U = HD / 32, PIECES = HD / 16;        // 16-byte pieces: of a lane, of a row
        const int group16 = warp - kPromptSoftmax;
        // Piece u of lane: row of the group, piece of the row; its two 16-byte halves go to pieces 2 c and 2 c + 1 of their block.  With two blocks the
        // lanes of the second store the odd one first, so that eight lanes meet 32 banks.
        int row[U], off[U][2];
        bool odd_first[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = u * 32 + lane, c = i % PIECES;
            row[u] = i / PIECES;
            const int r = 16 * group16 + row[u], cc = (c & 3) * 2;
            odd_first[u] = c >= 4;
            off[u][0] = (c >> 2) * 16384 + r * 128 + ((cc ^ (r & 7)) << 4);
            off[u][1] = (c >> 2) * 16384 + r * 128 + (((cc + 1) ^ (r & 7)) << 4);
        }
        uint4 kc[U], vc[U];
        float ks = 0.f, vs = 0.f;
        auto request = [&](const unsigned char* pages, const float* scales, int step, int phys, uint4 (&c)[U], float& s) {
            s = 0.f;
            if (phys >= 0) {
                const size_t block = (size_t)phys * p.kv.n_kv + piece.h;
                s = scales[block];
                const unsigned char* src = pages + ((block << p.kv.page_shift) + ((step * kStepTokens + 16 * group16) & (p.kv.page - 1))) * HD + lane * 16;
#pragma unroll
                for (int u = 0; u < U; ++u) c[u] = *reinterpret_cast<const uint4*>(src + u * 512);
            }
        };
        auto store = [&](uint32_t tile, const uint4 (&c)[U], bool there) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                uint32_t h[8];
                if (there) {
                    codes_to_half<DT>(c[u].x, h[0], h[1]);
                    codes_to_half<DT>(c[u].y, h[2], h[3]);
                    codes_to_half<DT>(c[u].z, h[4], h[5]);
                    codes_to_half<DT>(c[u].w, h[6], h[7]);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) h[i] = 0u;
                }
                if (odd_first[u]) {
                    sts128(tile + off[u][1], h[4], h[5], h[6], h[7]);
                    sts128(tile + off[u][0], h[0], h[1], h[2], h[3]);
                } else {
                    sts128(tile + off[u][0], h[0], h[1], h[2], h[3]);
                    sts128(tile + off[u][1], h[4], h[5], h[6], h[7]);
                }
            }
        };
        while (ok && piece.next(p.kv, p.r, p.group)) {
            const int steps = max(tile_view(piece, p, 0).steps, tile_view(piece, p, 1).steps);
            auto lookup = [&](int j) { return j < steps ? page_of(p.kv, piece.x.b, ((piece.step0 + j) * kStepTokens + 16 * group16) >> p.kv.page_shift) : -1; };
            int phys = lookup(0), phys1 = lookup(1);
            request(p.kv.k, p.kv.k_scale, piece.step0, phys, kc, ks);
            request(p.kv.v, p.kv.v_scale, piece.step0, phys, vc, vs);
            for (int j = 0; j < steps; ++j) {
                const uint32_t g = gs + j, stage = g & 1, parity = ((g >> 1) & 1) ^ 1;
                const int phys2 = lookup(j + 2);
                if (!(ok = wait_warp(k_empty + 8 * stage, parity, dead, 123))) break;
                store(k_smem + stage * C::TILE, kc, phys >= 0);
                fence_async_smem();
                arrive_warp(k_full + 8 * stage, lane);
                const float ks0 = ks, vs0 = vs;
                request(p.kv.k, p.kv.k_scale, piece.step0 + j + 1, phys1, kc, ks);
                if (!(ok = wait_warp(v_empty + 8 * stage, parity, dead, 124))) break;
                store(v_smem + stage * C::TILE, vc, phys >= 0 && vs0 > 0.f);
                if (lane == 0) {
                    s_scale[stage][0][group16] = ks0;
                    s_scale[stage][1][group16] = phys < 0 ? -INFINITY : vs0 > 0.f ? log2_fast(vs0) : 0.f;
                    s_scale[stage][2][group16] = vs0 > 0.f ? rcp_fast(vs0) : 1.f;
                }
                fence_async_smem();
                arrive_warp(v_full + 8 * stage, lane);
                request(p.kv.v, p.kv.v_scale, piece.step0 + j + 1, phys1, vc, vs);
                phys = phys1;
                phys1 = phys2;
            }
            gs += steps;
        }
    } else {
        // ================= MMA issue =================
        constexpr uint32_t s_desc = tc_idesc(128), o_desc = tc_idesc(HD) | (1u << 16);       // V: MN-major
        uint32_t done[2] = {0, 0}, pieces[2] = {0, 0};       // of each tile: steps, pieces that it had steps in
        while (ok && piece.next(p.kv, p.r, p.group)) {
            const int n[2] = {tile_view(piece, p, 0).steps, tile_view(piece, p, 1).steps}, steps = max(n[0], n[1]);
            auto scores = [&](int tile, uint32_t stage) {
                const uint32_t a = q_smem + tile * C::TILE, b = k_smem + stage * C::TILE;
#pragma unroll
                for (int blk = 0; blk < HD / 64; ++blk)
                    mma4_ss(tmem + C::S_COL + tile * 128, tc_smem_desc(a + blk * 16384), tc_smem_desc(b + blk * 16384), s_desc, blk > 0);
                commit_warp(s_full + 8 * tile);
            };
            auto values = [&](int tile, uint32_t stage, bool first) {
                const uint32_t b = v_smem + stage * C::TILE;
#pragma unroll
                for (int half = 0; half < 2; ++half)
                    mma4_ts(tmem + C::O_COL + tile * HD, tmem + C::S_COL + tile * 128 + 32 * half, value_desc(b + half * 8192), o_desc, !first || half > 0);
                commit_warp(pv_done + 8 * tile);
            };
            if (steps == 0) continue;
            ok = wait_warp(k_full + 8 * (gs & 1), (gs >> 1) & 1, dead, 126);
#pragma unroll
            for (int tile = 0; tile < 2; ++tile) {
                if (!ok || n[tile] == 0 || !(ok = wait_warp(q_ready + 8 * tile, pieces[tile] & 1, dead, 125))) continue;
                tc_fence_after();
                scores(tile, gs & 1);
            }
            if (!ok) break;
            commit_warp(k_empty + 8 * (gs & 1));
            for (int j = 0; j < steps && ok; ++j) {
                const uint32_t g = gs + j, stage = g & 1;
                ok = wait_warp(v_full + 8 * stage, (g >> 1) & 1, dead, 121) &&
                     (j + 1 == steps || wait_warp(k_full + 8 * (stage ^ 1), ((g + 1) >> 1) & 1, dead, 126));
#pragma unroll
                for (int tile = 0; tile < 2; ++tile) {
                    if (!ok || j >= n[tile]) continue;
                    ok = wait_warp(p_ready + 8 * tile, done[tile] & 1, dead, 127) &&
                         (j > 0 || wait_warp(o_free + 8 * tile, (pieces[tile] & 1) ^ 1, dead, 128));
                    if (!ok) continue;
                    tc_fence_after();
                    values(tile, stage, j == 0);
                    const bool last = tile == 1 || j >= n[1];
                    if (last) commit_warp(v_empty + 8 * stage);
                    if (j + 1 < n[tile]) {
                        ok = wait_warp(pv_done + 8 * tile, done[tile] & 1, dead, 122);       // P is where the scores go
                        if (!ok) continue;
                        scores(tile, stage ^ 1);
                    }
                    ++done[tile];
                }
                if (ok && j + 1 < steps) commit_warp(k_empty + 8 * (stage ^ 1));
            }
            gs += steps;
            for (int tile = 0; tile < 2; ++tile) pieces[tile] += n[tile] > 0;
        }
    }
    __syncthreads();
    if (warp == kPromptMma) {
        tc_fence_after();
        tc_dealloc(tmem, 512);
    }
}

template <int HD, int DT> cudaError_t launch_prompt(const AttnParams& p, int grid, cudaStream_t st) {
    static SmemLimit limit;
    auto* kern = paged_prompt_kernel<HD, DT>;
    const cudaError_t e = reserve_smem(reinterpret_cast<const void*>(kern), limit, PromptCfg<HD>::SMEM);
    return e != cudaSuccess ? e : launch_kernel(true, kern, dim3((unsigned)grid), dim3(kPromptThreads), PromptCfg<HD>::SMEM, st, p);
}

}  // namespace

cudaError_t launch_paged_prompt(int head_dim, int dtype, const AttnParams& p, int grid, cudaStream_t st) {
    if (head_dim == 64) return dtype == kI8 ? launch_prompt<64, kI8>(p, grid, st) : launch_prompt<64, kE4M3>(p, grid, st);
    return dtype == kI8 ? launch_prompt<128, kI8>(p, grid, st) : launch_prompt<128, kE4M3>(p, grid, st);
}

}  // namespace glq
