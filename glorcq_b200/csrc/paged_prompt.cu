// Attention of many rows a key/value head (pieces of prompts) over the paged 8-bit cache, on tcgen05.
//
// Segment: 256 rows (token of the call, head of the group), two tiles of 128, of one (sequence, key/value head); step: 128 tokens.  (Heads of 256
// channels: one tile, 64 tokens; the warps of the other tile only give stages back.)
// A step's products are S = Q K^T (operands in shared memory) and O += P V (P in tensor memory, over the scores that it is made of; V as it
// lies, tokens by channels, which is the MN-major form of the operand), each in half steps of 64 tokens.  Tensor memory: a tile has two places
// for S, which half steps take in turn, and O.  While the softmax of one half step runs, P V of the one before and S of the one after do: the
// softmax, which takes longest, hardly ever waits (a step of 128 tokens in one piece, whose next scores had to wait for its P V: 4 heads,
// 4096 tokens, 211 us against 183).
//
// Warps, which keep their roles over all segments of a CTA:
//   0..3, 4..7  softmax of tile 0 and 1: a thread has a row; writes P as fp16, multiplies O where m has grown, writes the result
//   8..11       codes to fp16 operands in shared memory, two times 16 tokens of a step each, so that one page, one pair of scales, is a
//               warp's at a time; a segment's rows
//   12, 13      issue the MMAs of tile 0 and 1 (one warp for both needed longer for it than the MMAs themselves)
//   15          works out the CTA's pieces of segments and hands them to the others through a small queue
// Scales and m as in paged_attention_rows_kernel: w = 2^(ks s + log2 vs - m) in fp16 (the operand in tensor memory; the results' error becomes 2.5e-4 to 2.9e-4
// where their own rounding is 2.1e-4; w in two halves would double P V and what the softmax packs and stores, which is the longer of the two), the sum of w / vs in fp32, m raised only when a score exceeds it
// by 2^8 (a published idea, as is taking a part of the exponentials as polynomials).  Keys that a row does not see get a score of -inf, in the half steps that
// have such keys, and the common path has no masks.
//
// The loops around it all are rolled: every warp of a scheduler runs another role's code, and what the instruction cache does not hold costs the
// warps that issue the MMAs more than the MMAs (134 cycles an MMA with unrolled loops everywhere).
//
// Every wait is bounded; a wait that runs out marks the CTA dead, all roles leave their loops, wait (2 ms again) for copies and MMAs that they have under way,
// and the kernel ends.  What lasts a step at most has
// tc_wait's 2 ms.  Three waits last as long as a piece of a segment or several (a place in the queue of pieces; the next piece; the scores of a tile
// that had no rows in the pieces before), which behind 100000 tokens is more than that, and so may the search for a piece among thousands of sequences
// without rows: their 2 ms begin anew with every step of the CTA and every block of rows that is looked at (wait_steps).
#include "paged.cuh"
#include "tc_mm.cuh"

// error word of this translation unit, merged by glq_debug_error
extern "C" int glq_paged_error(unsigned long long* out4, int clear) {
    if (!out4) return GLQ_ERR_ARG;
    if (cudaMemcpyFromSymbol(out4, glq::g_glq_err, 4 * sizeof(unsigned long long)) != cudaSuccess) return GLQ_ERR_CUDA;
    if (clear) {
        const unsigned long long z[4] = {0, 0, 0, 0};
        if (cudaMemcpyToSymbol(glq::g_glq_err, z, sizeof(z)) != cudaSuccess) return GLQ_ERR_CUDA;
    }
    return GLQ_OK;
}

namespace glq {
namespace {

constexpr int kPromptSoftmax = 8, kPromptProducers = 4, kPromptMma = kPromptSoftmax + kPromptProducers;
constexpr int kPromptThreads = (kPromptMma + 4) * 32;
// Registers of a thread: 128 at launch.  Measured (4096 tokens, 32 heads on 4, us): this split 180.7; 136, 120, 120 180; 144, 112, 112 181.2; 152, 128, 80 and
// 152, 112, 96 and 144, 128, 96 182.7; 152, 120, 88 184.3.  (With too few the MMA warps reload what they had put away.)
constexpr int kRegsSoftmax = 144, kRegsProducer = 120, kRegsMma = 104;
static_assert((kPromptSoftmax * kRegsSoftmax + kPromptProducers * kRegsProducer + 4 * kRegsMma) * 32 <= kPromptThreads * 128, "registers");
static_assert(kRegsSoftmax >= 128 && kRegsProducer <= 128 && kRegsMma <= 128, "the softmax takes what the others give");
// every so many pairs of exponentials one is taken by exp2_poly
constexpr int kPolyEvery = 4;

// Operands: [64-channel block][rows][128 B], 16-byte piece c of row r at c ^ (r & 7).
template <int HD> struct PromptCfg {
    using Share = typename PromptShape<HD>::Share;
    static constexpr int TILES = PromptShape<HD>::TILES, STEP = Share::STEP, GROUPS = STEP / 16;
    static constexpr int Q_BLOCK = 128 * 128, KV_BLOCK = STEP * 128, BLOCKS = HD / 64;
    static constexpr int Q_TILE = BLOCKS * Q_BLOCK, KV_TILE = BLOCKS * KV_BLOCK;
    static constexpr size_t SMEM = TILES * Q_TILE + 4 * KV_TILE + 1024;       // K and V of two stages
    static constexpr uint32_t S_COL = 0, O_COL = 256;
};

__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, volatile int* dead, int code) {
    return __all_sync(0xffffffffu, mbar_try_wait(bar, parity) || tc_wait(bar, parity, dead, code));
}
// What moves while a CTA does (addresses in shared memory): the last step in either stage, the blocks of rows that warp 15 has looked at.
struct Progress {
    uint32_t step0, step1, looked;
    static __device__ __forceinline__ uint32_t word(uint32_t a) {
        uint32_t x;
        asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(x) : "r"(a) : "memory");
        return x;
    }
    __device__ __forceinline__ uint32_t now() const { return word(step0) + word(step1) + word(looked); }
};
// The same for what may last many steps.
__device__ __forceinline__ bool wait_steps(uint32_t bar, uint32_t parity, volatile int* dead, int code, const Progress& progress) {
    uint32_t seen = progress.now();
    unsigned long long t0 = global_ns();
    for (bool late = false;;) {
        if (mbar_try_wait(bar, parity)) return true;
        if (*dead) return false;
        const uint32_t now = progress.now();
        if (now != seen) {
            seen = now;
            t0 = global_ns();
            late = false;
        } else if (late) {
            glq_ok(false, code, bar, parity);
            *dead = 1;
            return false;
        } else {
            late = global_ns() - t0 > 2000000ull;
        }
    }
}
__device__ __forceinline__ bool wait_warp_steps(uint32_t bar, uint32_t parity, volatile int* dead, int code, const Progress& progress) {
    return __all_sync(0xffffffffu, mbar_try_wait(bar, parity) || wait_steps(bar, parity, dead, code, progress));
}
// At the end of a CTA that is dead: for what is under way, 2 ms at most.
__device__ __forceinline__ void wait_at_the_end(uint32_t bar) {
    for (const unsigned long long t0 = global_ns(); !mbar_try_wait(bar, 0) && global_ns() - t0 < 2000000ull;) {
    }
}
__device__ __forceinline__ void copy_async_16(uint32_t dst, const void* src, bool live) {       // not live: zeros, nothing is read
    const int bytes = live ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
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
// MN-major operand, 128-byte swizzle: 64-channel blocks `block` bytes apart, groups of 8 tokens 1024 B apart
__device__ __forceinline__ uint64_t value_desc(uint32_t saddr, int block) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(block >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
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
// tcgen05.wait::ld for values that are used behind it: they are its operands, so that no use is moved in front of it
__device__ __forceinline__ void tmem_arrived(uint32_t (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31]) :: "memory");
}
__device__ __forceinline__ void tmem_arrived(uint32_t (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]) :: "memory");
}
template <int N> __device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t* v) {
    static_assert(N == 8 || N == 16, "");
    if constexpr (N == 8)
        asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
                     "r"(v[5]), "r"(v[6]), "r"(v[7])
                     : "memory");
    else
        asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
                 "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
                 "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}
__device__ __forceinline__ unsigned long long pack2(float a, float b) {
    unsigned long long d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ void unpack2(unsigned long long v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
    unsigned long long d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// 2^x of two values on the multiply-add pipe, the special-function unit being what the exponentials are bound by: a whole number and a rest in
// [-1/2, 1/2], whose power is a polynomial (minimax by relative error, 2.6e-6), the whole number added to the exponent.  Below -126: about 2^-126,
// which fp16 has as zero.
__device__ __forceinline__ void exp2_poly(unsigned long long x, float& a, float& b) {
    unpack2(x, a, b);
    const unsigned long long y = pack2(fmaxf(a, -126.f), fmaxf(b, -126.f)), big = pack2(12582912.f, 12582912.f);
    const unsigned long long t = add2(y, big), f = fma2(add2(t, pack2(-12582912.f, -12582912.f)), pack2(-1.f, -1.f), y);
    unsigned long long r = pack2(0.0095701f, 0.0095701f);
    r = fma2(r, f, pack2(0.05591786f, 0.05591786f));
    r = fma2(r, f, pack2(0.24024745f, 0.24024745f));
    r = fma2(r, f, pack2(0.69312181f, 0.69312181f));
    r = fma2(r, f, pack2(0.99999926f, 0.99999926f));
    float ta, tb;
    unpack2(t, ta, tb);
    unpack2(r, a, b);
    a = __int_as_float(__float_as_int(a) + (__float_as_int(ta) << 23));
    b = __int_as_float(__float_as_int(b) + (__float_as_int(tb) << 23));
}
// A 4 by 4 transposition among four lanes: x[s] becomes piece lane % 4 of lane s's row, so that four lanes write one row's 64 bytes beside one another
// (each lane writing its own row: 32 lines a store, and the results of both tiles took 6500 cycles, partial ones 11500, against 3800 and 5500).
__device__ __forceinline__ void quad_transpose(uint4 (&x)[4], int lane) {
    auto swap = [&](uint4& a, uint4& b, int bit) {        // the lane without the bit keeps a
        const bool up = lane & bit;
        uint4 send = up ? a : b;
        send.x = __shfl_xor_sync(0xffffffffu, send.x, bit);
        send.y = __shfl_xor_sync(0xffffffffu, send.y, bit);
        send.z = __shfl_xor_sync(0xffffffffu, send.z, bit);
        send.w = __shfl_xor_sync(0xffffffffu, send.w, bit);
        (up ? a : b) = send;
    };
    swap(x[0], x[1], 1);
    swap(x[2], x[3], 1);
    swap(x[0], x[2], 2);
    swap(x[1], x[3], 2);
}
// has the phase ended?  (a look, no wait)
__device__ __forceinline__ bool test_warp(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return __all_sync(0xffffffffu, done != 0);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A piece as it is handed out.
struct PromptPiece {
    int b, h, row, r0, rows, start;      // sequence, head; the sequence's first row in the batch, the block's first and number of rows; tokens before the call
    int step0;
    int halves[2], most;                 // half steps that a tile takes part in; steps of both; most < 0 ends the list
    int whole;                           // the segment is this CTA's alone
};
constexpr int kPieceQueue = 4, kPieceReaders = kPromptSoftmax + kPromptProducers + 2;

template <int HD, int DT>
__global__ void __launch_bounds__(kPromptThreads, 1) paged_prompt_kernel(const AttnParams p) {
    using C = PromptCfg<HD>;
    using Share = typename C::Share;
    constexpr int kStepTokens = C::STEP, kGroups = C::GROUPS, kHalves = kStepTokens / 64;
    extern __shared__ unsigned char prompt_smem[];
    __shared__ __align__(8) unsigned long long bars[28 + 2 * kPieceQueue];
    __shared__ PromptPiece s_piece[kPieceQueue];
    __shared__ float4 s_scale[2][kGroups];             // of a stage's groups of 16 tokens: factor of the scores, log2 vs, 1 / vs, number of the step
    __shared__ ShareStart sm_plan;
    __shared__ uint32_t s_tmem;
    __shared__ int s_dead;
    __shared__ uint32_t s_looked;                      // blocks of rows that warp 15 has looked at
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = (smem_u32(prompt_smem) + 1023u) & ~1023u;
    const uint32_t q_smem = base, k_smem = base + C::TILES * C::Q_TILE, v_smem = k_smem + 2 * C::KV_TILE;
    // [0], [1] of each: stages or tiles; of s_full, p_ready and pv_done four: [tile][place of the scores]
    const uint32_t k_full = smem_u32(bars), k_empty = k_full + 16, v_full = k_full + 32, v_empty = k_full + 48, s_full = k_full + 64,
                   p_ready = k_full + 96, pv_done = k_full + 128, q_ready = k_full + 160, o_free = k_full + 176, q_free = k_full + 192,
                   piece_full = k_full + 208, piece_empty = piece_full + 8 * kPieceQueue, mma_end = piece_empty + 8 * kPieceQueue;
    volatile int* dead = &s_dead;
    const Progress progress{smem_u32(&s_scale[0][0].w), smem_u32(&s_scale[1][0].w), smem_u32(&s_looked)};
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(k_full + 8 * i, kPromptProducers);
            mbar_init(v_full + 8 * i, kPromptProducers);
            mbar_init(k_empty + 8 * i, 2);
            mbar_init(v_empty + 8 * i, 2);
            mbar_init(q_ready + 8 * i, kPromptProducers);
            mbar_init(q_free + 8 * i, 1);
            mbar_init(o_free + 8 * i, 4);
            mbar_init(mma_end + 8 * i, 1);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(s_full + 8 * i, 1);
            mbar_init(p_ready + 8 * i, 4);
            mbar_init(pv_done + 8 * i, 1);
        }
        for (int i = 0; i < kPieceQueue; ++i) {
            mbar_init(piece_full + 8 * i, 1);
            mbar_init(piece_empty + 8 * i, kPieceReaders);
        }
        s_dead = 0;
        s_scale[0][0].w = s_scale[1][0].w = 0.f;
        s_looked = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kPromptMma) tc_alloc(smem_u32(&s_tmem), 512);
    tc_fence_before();
    __shared__ SharedRows sm_q;
    after_launch_ahead();
    const PagedRows rows_q = rows_in_shared(p.r, sm_q);
    Pieces<Share> pieces;
    pieces.template begin<kPromptThreads>(p.kv, rows_q, p.group, blockIdx.x, gridDim.x, sm_plan);
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    uint32_t gs = 0;                     // steps of the pieces before, over all roles alike
    bool ok = true;
    // The pieces in order, for one role's loop: next_piece() waits for one (false: no more), done_piece() gives its place back.
    uint32_t n_piece = 0;
    const PromptPiece* piece = s_piece;
    auto next_piece = [&]() {
        piece = s_piece + n_piece % kPieceQueue;
        ok = wait_warp_steps(piece_full + 8 * (n_piece % kPieceQueue), (n_piece / kPieceQueue) & 1, dead, 131, progress);
        return ok && piece->most >= 0;
    };
    auto done_piece = [&]() {
        arrive_warp(piece_empty + 8 * (n_piece % kPieceQueue), lane);
        ++n_piece;
    };

    if (warp < kPromptSoftmax) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        // ================= softmax: a row a thread =================
        const int tile = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t trow = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t s_tm = trow + C::S_COL + tile * 128, o_tm = trow + C::O_COL + tile * HD;
        uint32_t t = 0;                  // the tile's half steps so far: half step t has its scores, and P, at place t % 2
        while (next_piece()) {
            const int halves = piece->halves[tile], first_row = piece->r0 + 128 * tile;
            const bool live = row < piece->rows - 128 * tile;
            const int limit = live ? min(piece->start + (first_row + row) / p.group, p.kv.capacity - 1) : -1;      // the last key that the row sees
            const int limit_low = min(piece->start + first_row / p.group, p.kv.capacity - 1);                      // that every row of the tile sees
            const uint32_t t0 = t;
            int first = piece->step0 * kStepTokens;
            float m = -1e30f, l = 0.f;
#pragma unroll 1
            for (; t < t0 + halves; ++t, first += 64) {
                const uint32_t half = (t - t0) % kHalves, g = gs + (t - t0) / kHalves, bar = 16 * tile + 8 * (t & 1), s_at = s_tm + 64 * (t & 1);
                // (the scores first: a tile that had no part in many steps knows by them that V's stage is not two phases behind, which looks the same)
                ok = wait_warp_steps(s_full + bar, (t >> 1) & 1, dead, 120, progress) && (half > 0 || wait_warp(v_full + 8 * (g & 1), (g >> 1) & 1, dead, 121));
                if (!ok) break;
                tc_fence_after();
                uint32_t v[2][32];
                tmem_ld32(s_at, v[0]);
                tmem_ld32(s_at + 32, v[1]);
                tmem_arrived(v[0]);
                tmem_arrived(v[1]);
                const float4* scale = s_scale[g & 1] + 4 * half;
                if (first + 63 > limit_low) {
#pragma unroll
                    for (int i = 0; i < 64; ++i)
                        if (first + i > limit) v[i / 32][i % 32] = __float_as_uint(-INFINITY);
                }
                float top = -INFINITY;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint32_t* u = v[q / 2] + 16 * (q % 2);
                    const float4 sc = scale[q];
                    float x = max3(__uint_as_float(u[0]), __uint_as_float(u[1]), __uint_as_float(u[2]));
#pragma unroll
                    for (int i = 3; i < 15; i += 2) x = max3(x, __uint_as_float(u[i]), __uint_as_float(u[i + 1]));
                    top = fmaxf(top, fmaf(fmaxf(x, __uint_as_float(u[15])), sc.x, sc.y));
                }
                if (__any_sync(0xffffffffu, top > m + 8.f)) {
                    const float up = fmaxf(m, top), f = exp2_fast(m - up);
                    if (__any_sync(0xffffffffu, fabsf(up) > 0x1p20f && up > -1e30f)) break;
                    m = up;
                    l *= f;
                    if (t > t0) {         // the products so far, the last of which may be running
                        if (!(ok = wait_warp(pv_done + 16 * tile + 8 * ((t - 1) & 1), ((t - 1) >> 1) & 1, dead, 122))) break;
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < HD / 16; ++c) {
                            uint32_t x[16];
                            tc_ld16(o_tm + 16 * c, x);
                            tmem_arrived(x);
#pragma unroll
                            for (int i = 0; i < 16; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * f);
                            tmem_st<16>(o_tm + 16 * c, x);
                        }
                    }
                }
                uint32_t w[16];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint32_t* u = v[q / 2] + 16 * (q % 2);
                    const float4 sc = scale[q];
                    const float off = sc.y - m;
                    const unsigned long long cs2 = pack2(sc.x, sc.x), off2 = pack2(off, off);
                    unsigned long long sum2 = 0ull;
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        const unsigned long long x = fma2(pack2(__uint_as_float(u[i]), __uint_as_float(u[i + 1])), cs2, off2);
                        float a, b;
                        if (i / 2 % kPolyEvery == kPolyEvery - 1) {
                            exp2_poly(x, a, b);
                        } else {
                            unpack2(x, a, b);
                            a = exp2_fast(a);
                            b = exp2_fast(b);
                        }
                        sum2 = add2(sum2, pack2(a, b));
                        w[8 * (q % 2) + i / 2] = pack_half2(a, b);
                    }
                    float a, b;
                    unpack2(sum2, a, b);
                    l += (a + b) * sc.z;
                    if (q % 2) tmem_st<16>(s_at + 16 * (q / 2), w);
                }
                tmem_st_wait();
                tc_fence_before();
                arrive_warp(p_ready + bar, lane);
            }
            // Scores that are very large.  Above, 2^(u ks + (log2 vs - m)) has u ks unrounded, and m, a rounded score, is off by up to 2^-24 of it: from
            // 2^27 on the weights overflow fp16 or nothing is left of them.  Here a score is rounded as m was before m is taken from it.  (In the loop above the
            // operations that this takes cost 6 of 180 us whether they are needed or not.)
#pragma unroll 1
            for (; ok && t < t0 + halves; ++t, first += 64) {
                const uint32_t half = (t - t0) % kHalves, g = gs + (t - t0) / kHalves, bar = 16 * tile + 8 * (t & 1), s_at = s_tm + 64 * (t & 1);
                ok = wait_warp(s_full + bar, (t >> 1) & 1, dead, 120) && (half > 0 || wait_warp(v_full + 8 * (g & 1), (g >> 1) & 1, dead, 121));
                if (!ok) break;
                tc_fence_after();
                auto scores = [&](int q, float (&y)[16]) {          // returns 1 / vs
                    uint32_t u[16];
                    tc_ld16(s_at + 16 * q, u);
                    tmem_arrived(u);
                    const float4 sc = s_scale[g & 1][4 * half + q];
#pragma unroll
                    for (int i = 0; i < 16; ++i) y[i] = first + 16 * q + i > limit ? -INFINITY : fmaf(__uint_as_float(u[i]), sc.x, sc.y);
                    return sc.z;
                };
                float y[16], top = m;
#pragma unroll 1
                for (int q = 0; q < 4; ++q) {
                    scores(q, y);
#pragma unroll
                    for (int i = 0; i < 16; ++i) top = fmaxf(top, y[i]);
                }
                const float f = exp2_fast(m - top);
                m = top;
                l *= f;
                if (t > t0 && __any_sync(0xffffffffu, f != 1.f)) {
                    if (!(ok = wait_warp(pv_done + 16 * tile + 8 * ((t - 1) & 1), ((t - 1) >> 1) & 1, dead, 122))) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < HD / 16; ++c) {
                        uint32_t x[16];
                        tc_ld16(o_tm + 16 * c, x);
                        tmem_arrived(x);
#pragma unroll
                        for (int i = 0; i < 16; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * f);
                        tmem_st<16>(o_tm + 16 * c, x);
                    }
                }
                // P of 16 tokens takes the columns of 8 scores: those of tokens that have been read
#pragma unroll 1
                for (int q = 0; q < 4; ++q) {
                    const float inverse = scores(q, y);
                    uint32_t w[8];
                    float sum = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float a = exp2_fast(y[2 * i] - m), b = exp2_fast(y[2 * i + 1] - m);
                        sum += a + b;
                        w[i] = pack_half2(a, b);
                    }
                    l += sum * inverse;
                    tmem_st<8>(s_at + 8 * q, w);
                }
                tmem_st_wait();
                tc_fence_before();
                arrive_warp(p_ready + bar, lane);
            }
            if (ok && halves > 0) ok = wait_warp(pv_done + 16 * tile + 8 * ((t - 1) & 1), ((t - 1) >> 1) & 1, dead, 122);
            if (!ok) break;
            tc_fence_after();
            if (m <= -1e30f) l = 0.f;         // nothing seen: the sum is of exp2_poly's smallest numbers
            if (tile < C::TILES && piece->rows > 128 * tile) {
                const bool whole = piece->whole;
                const float f = result_factor(l, kCodeUnit<DT>);
                const int row4 = row & ~3, n_rows = piece->rows - 128 * tile;          // the first of the four rows of a lane and its neighbours
                __half* out[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = first_row + min(row4 + i, n_rows - 1), token = r / p.group;
                    out[i] = p.out + (long long)(piece->row + token) * p.ldo + (piece->h * p.group + r - token * p.group) * HD + 8 * (lane & 3);
                }
                float* part = partial_of<Share, HD>(p.partial, blockIdx.x, piece->step0 == 0);
                float* mine = part + (128 * tile + row4) * HD + 4 * (lane & 3);
#pragma unroll 1
                for (int c = 0; c < HD / 32; ++c) {
                    uint32_t v[32];
                    if (halves > 0) {
                        tmem_ld32(o_tm + 32 * c, v);
                        tmem_arrived(v);
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = 0u;
                    }
                    uint4 x[4];
                    if (whole) {
                        uint32_t o[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = pack_half2(__uint_as_float(v[2 * i]) * f, __uint_as_float(v[2 * i + 1]) * f);
#pragma unroll
                        for (int i = 0; i < 4; ++i) x[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                        quad_transpose(x, lane);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (row4 + i < n_rows) *reinterpret_cast<uint4*>(out[i] + 32 * c) = x[i];
                    } else {
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) x[i] = make_uint4(v[16 * half + 4 * i], v[16 * half + 4 * i + 1], v[16 * half + 4 * i + 2], v[16 * half + 4 * i + 3]);
                            quad_transpose(x, lane);
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (row4 + i < n_rows) *reinterpret_cast<uint4*>(mine + i * HD + 32 * c + 16 * half) = x[i];
                        }
                    }
                }
                if (live && !whole) *reinterpret_cast<float2*>(part + Share::R * HD + 2 * (128 * tile + row)) = make_float2(m, l);
            }
            tc_fence_before();
            if (halves > 0) arrive_warp(o_free + 8 * tile, lane);
            gs += piece->most;
            done_piece();
        }
    } else if (warp < kPromptMma) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsProducer));
        // ================= codes to operands =================
        constexpr int G = kGroups / kPromptProducers, U = HD / 32, BLOCKS = C::BLOCKS;        // groups of a warp, 16-byte pieces of a lane in each
        const int group0 = G * (warp - kPromptSoftmax);
        // Piece u of lane: row lane / 4 + 8 (u / BLOCKS) of a group, piece lane % 4 of block u % BLOCKS; its halves become pieces 2c and 2c + 1 of 8 in the
        // operand's row.  Eight lanes then meet 32 banks: two rows, one even and one odd.
        const int r0 = lane >> 2, c0 = lane & 3;
        const uint32_t even = (16 * group0 + r0) * 128 + (((2 * c0) ^ (r0 & 7)) << 4), odd = (16 * group0 + r0) * 128 + (((2 * c0 + 1) ^ (r0 & 7)) << 4);
        uint4 kc[G][U], vc[G][U];
        float ks[G], vs[G];
        int phys[G], phys1[G], phys2[G], h = 0;       // entries of the page table: of this step, the next and the one behind that (looked at when used)
        uint32_t had = 0;                 // bit t: parity of the pieces that tile t had steps in
        auto request = [&](const unsigned char* pages, const float* scales, int step, const int (&phys)[G], uint4 (&c)[G][U], float (&s)[G]) {
#pragma unroll
            for (int k = 0; k < G; ++k) {
                s[k] = 0.f;
                if (!page_there(p.kv, phys[k])) {           // zeros
#pragma unroll
                    for (int u = 0; u < U; ++u) c[k][u] = make_uint4(0u, 0u, 0u, 0u);
                } else {
                    const size_t block = (size_t)phys[k] * p.kv.n_kv + h;
                    s[k] = scales[block];
                    const unsigned char* src = pages + ((block << p.kv.page_shift) + ((step * kStepTokens + 16 * (group0 + k)) & (p.kv.page - 1))) * HD + r0 * HD + c0 * 16;
#pragma unroll
                    for (int u = 0; u < U; ++u) c[k][u] = *reinterpret_cast<const uint4*>(src + (u / BLOCKS) * 8 * HD + (u % BLOCKS) * 64);
                }
            }
        };
        auto store = [&](uint32_t tile, const uint4 (&c)[G][U]) {
#pragma unroll
            for (int k = 0; k < G; ++k)
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    uint32_t h[8];
                    codes_to_half<DT>(c[k][u].x, h[0], h[1]);
                    codes_to_half<DT>(c[k][u].y, h[2], h[3]);
                    codes_to_half<DT>(c[k][u].z, h[4], h[5]);
                    codes_to_half<DT>(c[k][u].w, h[6], h[7]);
                    const uint32_t at = tile + 2048 * k + (u / BLOCKS) * 1024 + (u % BLOCKS) * C::KV_BLOCK;
                    sts128(at + even, h[0], h[1], h[2], h[3]);
                    sts128(at + odd, h[4], h[5], h[6], h[7]);
                }
        };
        while (next_piece()) {
            const int steps = piece->most, step0 = piece->step0, b = piece->b;
            h = piece->h;
            auto lookup = [&](int j, int (&to)[G]) {
#pragma unroll
                for (int k = 0; k < G; ++k) to[k] = j < steps ? page_entry(p.kv, b, ((step0 + j) * kStepTokens + 16 * (group0 + k)) >> p.kv.page_shift) : -1;
            };
            // The tiles' rows, a quarter a warp: where a place is free already, ahead of the first keys.
            constexpr int LPR = HD / 8, RPP = 32 / LPR;          // lanes of a row, rows of a pass
            const int c = lane % LPR, row0 = (warp - kPromptSoftmax) * 32 + lane / LPR;
            const int more_tokens = RPP / p.group, more_heads = RPP - more_tokens * p.group;
            const __half* from = p.q + (long long)piece->row * p.ldq + h * p.group * HD + 8 * c;
            uint32_t rows_missing = (piece->halves[0] > 0) | (piece->halves[1] > 0) << 1, rows_coming = 0;
            auto copy_rows = [&](int tile) {
                had ^= 1u << tile;
                rows_missing ^= 1u << tile;
                rows_coming |= 1u << tile;
                int token = (piece->r0 + 128 * tile + row0) / p.group, head = piece->r0 + 128 * tile + row0 - token * p.group;
                const int rows = piece->rows - 128 * tile;
#pragma unroll 2
                for (int i = 0; i < 32 / RPP; ++i) {
                    const int row = row0 + i * RPP;
                    copy_async_16(q_smem + tile * C::Q_TILE + row * 128 + (c >> 3) * C::Q_BLOCK + (((c & 7) ^ (row & 7)) << 4),
                                  from + (row < rows ? (long long)token * p.ldq + head * HD : 0ll), row < rows);
                    token += more_tokens;
                    head += more_heads;
                    if (head >= p.group) {
                        head -= p.group;
                        ++token;
                    }
                }
            };
            auto rows_there = [&]() {
                if (!rows_coming) return;
                asm volatile("cp.async.wait_all;" ::: "memory");
                fence_async_smem();
                for (int tile = 0; tile < 2; ++tile)
                    if (rows_coming >> tile & 1) arrive_warp(q_ready + 8 * tile, lane);
                rows_coming = 0;
            };
            lookup(0, phys);
            lookup(1, phys1);
#pragma unroll 1
            for (int tile = 0; tile < 2; ++tile)
                if ((rows_missing >> tile & 1) && test_warp(q_free + 8 * tile, ((had >> tile) & 1) ^ 1)) copy_rows(tile);
            request(p.kv.k, p.kv.k_scale, step0, phys, kc, ks);
            request(p.kv.v, p.kv.v_scale, step0, phys, vc, vs);
            for (int j = 0; j < steps; ++j) {
                const uint32_t g = gs + j, stage = g & 1, parity = ((g >> 1) & 1) ^ 1;
                lookup(j + 2, phys2);
                if (!(ok = wait_warp(k_empty + 8 * stage, parity, dead, 123))) break;
                store(k_smem + stage * C::KV_TILE, kc);
                fence_async_smem();
                arrive_warp(k_full + 8 * stage, lane);
                float ks0[G];
#pragma unroll
                for (int k = 0; k < G; ++k) ks0[k] = ks[k];
                request(p.kv.k, p.kv.k_scale, step0 + j + 1, phys1, kc, ks);
                if (j == 0) {
#pragma unroll 1
                    for (int tile = 0; tile < 2; ++tile) {
                        if (!(rows_missing >> tile & 1)) continue;
                        rows_there();
                        if (!(ok = wait_warp(q_free + 8 * tile, ((had >> tile) & 1) ^ 1, dead, 130))) break;
                        copy_rows(tile);
                    }
                    if (!ok) break;
                    rows_there();
                }
                if (!(ok = wait_warp(v_empty + 8 * stage, parity, dead, 124))) break;
#pragma unroll
                for (int k = 0; k < G; ++k)
                    if (!live_scale(vs[k]))       // a block without a scale: its values are zero whatever its codes
#pragma unroll
                        for (int u = 0; u < U; ++u) vc[k][u] = make_uint4(0u, 0u, 0u, 0u);
                store(v_smem + stage * C::KV_TILE, vc);
#pragma unroll
                for (int k = 0; k < G; ++k)
                    if (lane == k)         // (a factor above zero: -inf times it hides a key)
                        s_scale[stage][group0 + k] = make_float4(fmaxf(ks0[k] * p.scale2, 1e-30f), page_there(p.kv, phys[k]) ? scale_log(vs[k]) : -INFINITY,
                                                                 page_there(p.kv, phys[k]) ? scale_inverse(vs[k]) : 0.f, __uint_as_float(g));
                fence_async_smem();
                arrive_warp(v_full + 8 * stage, lane);
                request(p.kv.v, p.kv.v_scale, step0 + j + 1, phys1, vc, vs);
#pragma unroll
                for (int k = 0; k < G; ++k) {
                    phys[k] = phys1[k];
                    phys1[k] = phys2[k];
                }
            }
            gs += steps;
            if (!ok) break;
            done_piece();
        }
        if (!ok) asm volatile("cp.async.wait_all;" ::: "memory");
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsMma));
        if (warp < kPromptMma + 2) {
            // ================= MMA issue =================
            constexpr uint32_t s_desc = tc_idesc(64), o_desc = tc_idesc(HD) | (1u << 16);       // V: MN-major
            const int tile = warp - kPromptMma;
            const uint32_t s_at = tmem + C::S_COL + tile * 128, o_at = tmem + C::O_COL + tile * HD, bar = 8 * tile, bar2 = 16 * tile;
            const uint64_t q_at = tc_smem_desc(q_smem + tile * C::Q_TILE), k_at = tc_smem_desc(k_smem), v_at = value_desc(v_smem, C::KV_BLOCK);
            uint32_t t = 0, had = 0;              // half steps as in the softmax, pieces that the tile had steps in
            while (next_piece()) {
                const int n = piece->halves[tile], steps = piece->most;
                auto scores = [&](int i) {        // of the piece's half step i, t + i
                    const uint32_t g = gs + i / kHalves, place = (t + i) & 1;
                    if (i % kHalves == 0 && !wait_warp(k_full + 8 * (g & 1), (g >> 1) & 1, dead, 126)) return false;
                    tc_fence_after();
                    const uint64_t k = k_at + (g & 1) * (C::KV_TILE >> 4) + i % kHalves * (8192 >> 4);
#pragma unroll
                    for (int blk = 0; blk < C::BLOCKS; ++blk) mma4_ss(s_at + 64 * place, q_at + blk * (C::Q_BLOCK >> 4), k + blk * (C::KV_BLOCK >> 4), s_desc, blk > 0);
                    commit_warp(s_full + bar2 + 8 * place);
                    return true;
                };
                if (n > 0) ok = wait_warp(q_ready + bar, had & 1, dead, 125);
#pragma unroll 1
                for (int i = -2; i < n && ok; ++i) {
                    if (i >= 0) {
                        const uint32_t g = gs + i / kHalves, stage = g & 1, place = (t + i) & 1, parity = ((t + i) >> 1) & 1;
                        const bool last = i % kHalves == kHalves - 1 || i + 1 == n;         // of its step
                        ok = (i > 0 || wait_warp(o_free + bar, (had & 1) ^ 1, dead, 128)) && wait_warp(p_ready + bar2 + 8 * place, parity, dead, 129);
                        if (!ok) break;
                        tc_fence_after();
                        // (who has written P has waited for V)
                        mma4_ts(o_at, s_at + 64 * place, v_at + stage * (C::KV_TILE >> 4) + i % kHalves * (8192 >> 4), o_desc, i > 0);
                        commit_warp(pv_done + bar2 + 8 * place);
                        if (lane == 0) {                                      // the step's scores have all been read
                            if (last) mbar_arrive(k_empty + 8 * stage);
                            if (i + 1 == n) mbar_arrive(q_free + bar);
                        }
                        if (!(ok = wait_warp(pv_done + bar2 + 8 * place, parity, dead, 122))) break;
                        if (last && lane == 0) mbar_arrive(v_empty + 8 * stage);
                    }
                    if (i + 2 < n) ok = scores(i + 2);
                }
                t += n;
                // steps that only the other tile takes part in
                for (int j = (n + kHalves - 1) / kHalves; j < steps && ok; ++j) {
                    const uint32_t g = gs + j, stage = 8 * (g & 1);
                    ok = wait_warp(k_full + stage, (g >> 1) & 1, dead, 126) && wait_warp(v_full + stage, (g >> 1) & 1, dead, 121);
                    if (ok && lane == 0) {
                        mbar_arrive(k_empty + stage);
                        mbar_arrive(v_empty + stage);
                    }
                }
                if (!ok) break;
                gs += steps;
                had += n > 0;
                done_piece();
            }
            if (!ok) {
                commit_warp(mma_end + 8 * tile);
                wait_at_the_end(mma_end + 8 * tile);
            }
        } else if (warp == kPromptMma + 3) {
            // ================= pieces =================
            uint32_t looked = 0;
            for (bool more = true; more && ok; ++n_piece) {
                ok = wait_warp_steps(piece_empty + 8 * (n_piece % kPieceQueue), ((n_piece / kPieceQueue) & 1) ^ 1, dead, 132, progress);
                more = ok && pieces.next(p.kv, rows_q, p.group, [&] {
                    if (lane == 0) *const_cast<volatile uint32_t*>(&s_looked) = ++looked;
                });
                PromptPiece x{};
                x.most = -1;
                if (more) {
                    x.b = pieces.x.b;
                    x.h = pieces.h;
                    x.row = pieces.x.own.x;
                    x.r0 = pieces.x.r0;
                    x.rows = pieces.x.n_rows;
                    x.start = pieces.x.start;
                    x.step0 = pieces.step0;
                    x.whole = pieces.whole();
                    for (int tile = 0; tile < 2; ++tile) {
                        const int rows = tile < C::TILES ? min(x.rows - 128 * tile, 128) : 0;
                        const int last = min(x.start + (x.r0 + 128 * tile + rows - 1) / p.group, p.kv.capacity - 1);
                        x.halves[tile] = rows > 0 ? max(0, min(kHalves * pieces.step1, last / 64 + 1) - kHalves * x.step0) : 0;
                    }
                    x.most = (max(x.halves[0], x.halves[1]) + kHalves - 1) / kHalves;
                }
                if (lane == 0 && ok) s_piece[n_piece % kPieceQueue] = x;
                arrive_warp(piece_full + 8 * (n_piece % kPieceQueue), lane);
            }
            if (lane == 0) p.join[blockIdx.x] = join_item<Share>(pieces.total, gridDim.x, blockIdx.x, sm_plan);
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
    if (head_dim == 256) return dtype == kI8 ? launch_prompt<256, kI8>(p, grid, st) : launch_prompt<256, kE4M3>(p, grid, st);
    if (head_dim == 64) return dtype == kI8 ? launch_prompt<64, kI8>(p, grid, st) : launch_prompt<64, kE4M3>(p, grid, st);
    return dtype == kI8 ? launch_prompt<128, kI8>(p, grid, st) : launch_prompt<128, kE4M3>(p, grid, st);
}

}  // namespace glq
