// linear16.cu -- a linear layer in 16 bits with its epilogue (nllb_linear16,
// sm_100a):  out = act(x w^T + bias) + residual, fp32 sums, one rounding.
//
// The weights are the A operand in every form, the tokens the B operand: a
// lane then holds one output column, so that bias is one register, residual
// and output rows are read and written 32 columns at a time whatever their
// alignment, and a few tokens make a narrow tile rather than a mostly empty one.
//
// Few tokens (linear16_few): the weights' bytes bound it, or the start of a
// launch.  A warp multiplies 16 weight rows by 8 tokens at a time (warp-level
// products); the order of the summands is the same permutation for both
// operands, so that each lane's operands are 16 contiguous bytes of a row,
// straight from global memory.
//
// More (linear16_tc): tcgen05 products of 128 weight rows by a tile of up to
// 256 tokens, operands by TMA into a ring of stages (64 wide, 128-byte swizzle),
// persistent CTAs with two accumulators in tensor memory, so that one is drained
// while the other is filled.  Pairs of CTAs (cta_group::2) take 256 weight rows
// and load half of the tokens' tile each.  Where tiles are few, a cluster shares
// the sum over k of one tile and joins it through distributed shared memory.
//
// Measured (device time, short replays): one token by 4096 x 1024 3.5 to 4.1 us
// (2.4 TB/s, the start of a launch); 64 by 256206 x 1024 into fp32 93 us (6.3
// TB/s, HBM; the library's product into bf16 174); 10000 by 1024 x 4096 with a
// residual 68 us (1230 TFLOP/s, the tensor cores 75 % busy, operands from L2 in
// three rounds of tiles; 81 us in a long run of them, under the power limit).
// Under that limit 8192 by 8192 x 4096 430 us (the library's product 408).  In
// between the library's product is ahead: 128 by 1024 x 1024 6.2 us (4.1), 512 by
// 4096 x 1024 8.2 (6.2), 1000 by 8192 x 1024 17.8 (16.4); 128 by 1024 x 4096 8.2
// (8.2), 4096 by 4096 x 1024 29.0 (32.1).
#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <mutex>
#include <string>

#include "engine_kernels.h"
#include "nllb_translate.h"
#include "overlap.h"
#include "rows.cuh"

namespace nllb {
int set_error(int status, const std::string& msg);  // nllb_attn.cu

namespace {

// A bounded wait of a call without an error word of its own gave up; and what nllb_linear16_status last took from there.
__device__ int g_linear16_err, g_linear16_taken;

// (one step: what is set meanwhile stays for the next status)
__global__ void linear16_take_err() { g_linear16_taken = atomicExch(&g_linear16_err, 0); }

struct Args {
    const void *x, *w, *bias, *residual;
    void* out;
    long long ldx, ldw, ldr, ldo;
    int M, N, K, kind;
    float c1, c2;  // of the activation
    bool out_whole, res_whole;  // (there and) the rows start on 16 bytes, as TMA has it
    bool out_end;  // output rows end on 16 bytes too
    bool expire;  // test: a wait runs out
    int device;
    int* err;  // the caller's error word (null: the device's)
};

template <typename T>
__device__ __forceinline__ float as_float(T x) {
    if constexpr (std::is_same<T, float>::value) return x;
    else if constexpr (std::is_same<T, __half>::value) return __half2float(x);
    else return __bfloat162float(x);
}
template <typename T>
__device__ __forceinline__ T rounded(float x) {
    if constexpr (std::is_same<T, float>::value) return x;
    else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(x);
    else return __float2bfloat16_rn(x);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float max_nan(float a, float b) {
    float c;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
    return c;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// |y| erfc(|y| / sqrt 2) / 2, what max(y, 0) exceeds gelu(y) by, for two of them.  With z = |y| / sqrt 2 and t = 1 / (1 + z / 2),
// erfc z = t 2^(P(t) - z^2 log2 e); P of degree 9 is fitted to log2 (e^(z^2) erfc z / t) over z in [0, 10.2], where its largest
// error is 4.6e-8, and 2.1e-7 when it is evaluated in fp32.  (The library's erfcf, which branches: 471 rows of 40012 over
// k = 155 65 us.)
__device__ __forceinline__ float2 gelu_gap(float2 y) {
    auto both = [](float c) { return make_float2(c, c); };
    const float2 x = make_float2(fminf(fabsf(y.x), 30.0f), fminf(fabsf(y.y), 30.0f));  // (0 from 15 on; finite for infinities)
    const float2 d = fma2(x, both(0.35355339f), both(1.0f)), t = make_float2(rcp(d.x), rcp(d.y));
    float2 p = fma2(both(0.20728277f), t, both(-0.97266638f));
    p = fma2(p, t, both(1.6471334f));
    p = fma2(p, t, both(-0.97694308f));
    p = fma2(p, t, both(-0.13727684f));
    p = fma2(p, t, both(0.012391086f));
    p = fma2(p, t, both(0.046664748f));
    p = fma2(p, t, both(0.55840427f));
    p = fma2(p, t, both(1.4406633f));
    p = fma2(p, t, both(-2.8256532f));  // (less 1: the half)
    p = fma2(mul2(x, both(-0.72134752f)), x, p);
    return mul2(mul2(x, t), make_float2(ex2(p.x), ex2(p.y)));
}

// The activations, each in a form whose small results keep their relative accuracy, in three kinds of code:
//   kClamp  max(y, c1): none (c1 = -inf) and RELU (0); NaN stays
//   kSwish  y / (1 + 2^-(y (c1 + c2 y^2))): SILU, and GELU_TANH, since (1 + tanh u) / 2 = 1 / (1 + e^-2u).  Nothing is left
//           of y at -100, where a smaller y stops, and nothing is taken from it at 100, where the exponent's stops: infinity
//           meets neither infinity nor SILU's c2 of 0.  (Results below 2^-119 may come out as 0.)
//   kGelu
enum { kClamp = 0, kSwish = 1, kGelu = 2 };
template <int KIND>
__device__ __forceinline__ float2 activate(const Args& a, float2 y) {
    auto both = [](float c) { return make_float2(c, c); };
    if constexpr (KIND == kClamp) return make_float2(max_nan(y.x, a.c1), max_nan(y.y, a.c1));
    if constexpr (KIND == kSwish) {
        y = make_float2(max_nan(y.x, -100.f), max_nan(y.y, -100.f));
        const float2 x = make_float2(fminf(y.x, 100.f), fminf(y.y, 100.f));
        const float2 z = mul2(x, fma2(mul2(x, both(-a.c2)), x, both(-a.c1)));
        return make_float2(__fdividef(y.x, 1.0f + ex2(z.x)), __fdividef(y.y, 1.0f + ex2(z.y)));
    }
    return fma2(gelu_gap(y), both(-1.0f), make_float2(max_nan(y.x, 0.f), max_nan(y.y, 0.f)));
}
template <int KIND, int N>
__device__ __forceinline__ void activate(const Args& a, float (&v)[N]) {
#pragma unroll
    for (int j = 0; j < N; j += 2) {
        const float2 y = activate<KIND>(a, make_float2(v[j], v[j + 1]));
        v[j] = y.x, v[j + 1] = y.y;
    }
}
__device__ __forceinline__ float activate(const Args& a, float x) {
    const float2 y = make_float2(x, x);
    return (a.kind == kClamp ? activate<kClamp>(a, y) : a.kind == kSwish ? activate<kSwish>(a, y) : activate<kGelu>(a, y)).x;
}

// The tensor cores cut what they add to a sum, so that one over K comes out up to K 2^-27 of its summands' sizes short.  Sums
// that fp32 outputs are made of are taken over 1024 at most and those added in fp32 (4096 x 4096 by K = 8192: 9e-6 off as
// one, 1e-6 so); of 16-bit outputs over 16384, a quarter of fp16's half step.
constexpr int kSegment = 1024, kSegment16 = 16384;

// ---- few tokens ------------------------------------------------------------------------------------------------

constexpr int kFewWarps = 8, kFewRows = 16;  // warps of a CTA; weight rows of a warp
constexpr int kFewBlocks = 4;                // blocks of 32 k that a warp takes together

template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Elements [k, k + 8) of a row of K, zeros past its end.
template <typename T>
__device__ __forceinline__ uint4 row_chunk(const T* row, int k, int K) {
    if (k + 8 <= K) return ld_coherent(reinterpret_cast<const uint4*>(row + k));
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint16_t* p = reinterpret_cast<const uint16_t*>(row + k) + 2 * i;
        u[i] = (k + 2 * i < K ? ld_coherent(p) : 0u) | (k + 2 * i + 1 < K ? (uint32_t)ld_coherent(p + 1) : 0u) << 16;
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
}

// KG warps share k for the same 16 rows, KG = 8, or fewer where k is short; 8 / KG groups of rows to a CTA.
template <typename T, typename O, int NT, int KG>
__global__ void __launch_bounds__(kFewWarps * 32) linear16_few(const Args a, int n_split) {
    constexpr int ROWS = kFewRows * kFewWarps / KG;
    __shared__ float sums[KG][8 * NT][ROWS];
    pdl_launch_dependents();
    pdl_wait_primary();

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, lr = lane >> 2, lc = lane & 3;
    const int kg = warp % KG, rg = warp / KG * kFewRows;
    const int split = blockIdx.x % n_split;
    const long long n0 = (long long)(blockIdx.x / n_split) * ROWS;
    const T* w = static_cast<const T*>(a.w);
    // (a row past the last one: the last one's, whose sums nobody uses)
    const T* w0 = w + min(n0 + rg + lr, (long long)a.N - 1) * a.ldw + 8 * lc;
    const T* w1 = w + min(n0 + rg + lr + 8, (long long)a.N - 1) * a.ldw + 8 * lc;
    for (int m0 = blockIdx.y * 8 * NT; m0 < a.M; m0 += gridDim.y * 8 * NT) {
        const T* x[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t)
            x[t] = m0 + t * 8 + lr < a.M ? static_cast<const T*>(a.x) + (m0 + t * 8 + lr) * a.ldx + 8 * lc : nullptr;

        float c[NT][4], total[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) c[t][e] = total[t][e] = 0.f;
        constexpr int STEP = 32 * kFewBlocks;
        int steps = 0;
        for (int k = (split * KG + kg) * STEP; k < a.K; k += n_split * KG * STEP) {
            if (++steps > kSegment / STEP) {  // (the products cut what they add to a sum)
                steps = 1;
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) total[t][e] += c[t][e], c[t][e] = 0.f;
            }
            uint4 u[kFewBlocks], v[kFewBlocks], b[NT][kFewBlocks];
#pragma unroll
            for (int i = 0; i < kFewBlocks; ++i) {
                // (chunks count from this lane's own)
                u[i] = row_chunk(w0, k + 32 * i, a.K - 8 * lc);
                v[i] = row_chunk(w1, k + 32 * i, a.K - 8 * lc);
            }
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < kFewBlocks; ++i)
                    b[t][i] = x[t] ? row_chunk(x[t], k + 32 * i, a.K - 8 * lc) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int i = 0; i < kFewBlocks; ++i)
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    mma<T>(c[t], u[i].x, v[i].x, u[i].y, v[i].y, b[t][i].x, b[t][i].y);
                    mma<T>(c[t], u[i].z, v[i].z, u[i].w, v[i].w, b[t][i].z, b[t][i].w);
                }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) sums[kg][t * 8 + 2 * lc + (e & 1)][rg + lr + 8 * (e >> 1)] = total[t][e] + c[t][e];
        __syncthreads();
        // the warps' sums, then the splits', always in the same order
        if (n_split > 1) {
            for (int i = tid; i < 8 * NT * ROWS; i += kFewWarps * 32) {
                float s = 0.f;
#pragma unroll
                for (int j = 0; j < KG; ++j) s += sums[j][i / ROWS][i % ROWS];
                sums[0][i / ROWS][i % ROWS] = s;
            }
            cluster_sync_all();
        }
        constexpr int ITEMS = 8 * NT * ROWS, EACH = ITEMS / (kFewWarps * 32) < 4 ? (ITEMS + kFewWarps * 32 - 1) / (kFewWarps * 32) : 4;
        for (int i0 = split * kFewWarps * 32 + tid; i0 < ITEMS; i0 += EACH * n_split * kFewWarps * 32) {
            float bias[EACH], old[EACH];
#pragma unroll
            for (int u = 0; u < EACH; ++u) {  // (all asked for before the first is stored)
                const int i = i0 + u * n_split * kFewWarps * 32, m = m0 + i / ROWS;
                const long long n = n0 + i % ROWS;
                const bool there = i < ITEMS && m < a.M && n < a.N;
                bias[u] = there && a.bias ? as_float(ld_coherent(static_cast<const T*>(a.bias) + n)) : 0.f;
                old[u] = there && a.residual ? as_float(ld_coherent(static_cast<const O*>(a.residual) + m * a.ldr + n)) : 0.f;
            }
#pragma unroll
            for (int u = 0; u < EACH; ++u) {
                const int i = i0 + u * n_split * kFewWarps * 32, m = m0 + i / ROWS;
                const long long n = n0 + i % ROWS;
                if (i >= ITEMS || m >= a.M || n >= a.N) continue;
                float y = 0.f;
                if (n_split > 1) {
                    for (int r = 0; r < n_split; ++r) y += ld_cluster_f32(map_rank(&sums[0][i / ROWS][i % ROWS], r));
                } else {
#pragma unroll
                    for (int j = 0; j < KG; ++j) y += sums[j][i / ROWS][i % ROWS];
                }
                y = activate(a, y + bias[u]);
                static_cast<O*>(a.out)[m * a.ldo + n] = rounded<O>(a.residual ? y + old[u] : y);
            }
        }
        // the sums are free again, and no CTA leaves while another reads them
        if (n_split > 1) cluster_sync_all();
        else __syncthreads();
    }
}

// ---- tensor cores ----------------------------------------------------------------------------------------------

constexpr int kRows = 128, kChunk = 64;                 // weight rows of a CTA's tile; k of a stage
constexpr uint32_t kRowsBytes = kRows * kChunk * 2;     // 16 KB
constexpr int kDrain = 8, kThreads = (kDrain + 2) * 32; // warps that drain accumulators; 1 that fetches, 1 that multiplies
constexpr int kMaxStages = 10;
constexpr int kPiece = 16;                              // a warp drains pieces of 32 columns by 16 tokens, each through a slot
constexpr int kMaxSlots = 8;
constexpr uint32_t kBars = (2 * kMaxStages + 6 + kDrain * kMaxSlots) * 8 + 16;
constexpr uint32_t kSmem = 232448 - 1024;  // of a CTA, less what the alignment takes

enum { kSingle = 0, kPair = 1, kSplit = 2 };

struct Tiling {
    int bn;           // tokens of a tile, a multiple of 32 up to 256
    int stages;
    int slots;        // of a warp: of 16 bits 8 where residual rows come through them, or k is short and draining counts, else 4
    int segment;      // stages whose products the tensor cores add
    int acc;          // columns of an accumulator in tensor memory; behind two of them the segments' total
    int tiles_n, tiles_m;
    bool tokens_first;  // tiles of the same weights follow one another (else: of the same tokens)
};

__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
        : "memory");
}
// Into this CTA's shared memory, complete on the pair's first CTA's barrier.
__device__ __forceinline__ void tma_2d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
        "[%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
// One arrival on `bar` of each CTA of the pair.
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
}
// (relaxed: what has to be over before is a read of tensor memory, which has been waited for; a release would wait for the
// drained rows on their way to memory as well, 8000 cycles a tile of 64 rows of logits)
__device__ __forceinline__ void arrive_at(uint32_t bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void arrive_here(uint64_t* bar) {
    asm volatile("mbarrier.arrive.relaxed.cta.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, int x, int y, uint32_t src) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(x), "r"(y), "r"(src)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// All but the last N stores have read their shared memory.
template <int N>
__device__ __forceinline__ void stores_read() {
    asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void stores_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// Whether phase `parity` is over, without a wait.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

// 16 columns of this thread's lane (warp-wide), there after tmem_wait on the same registers.
__device__ __forceinline__ void tmem_ask(uint32_t taddr, float (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
          "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait(float (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]),
                   "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
                 :
                 : "memory");
}
// 16 columns of this thread's lane, written (warp-wide).
__device__ __forceinline__ void tmem_put(uint32_t taddr, const float (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]),
        "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
        : "memory");
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// Four neighbouring columns of a row, those from N on left out.  (whole: the row starts on 16 bytes)
template <typename O>
struct __align__(4 * sizeof(O)) Four {
    O v[4];
};
template <typename O>
__device__ __forceinline__ Four<O> load4(const O* row, int n, int N, bool whole) {
    using Bits = typename std::conditional<sizeof(O) == 4, uint4, uint2>::type;
    Four<O> f;
    if (whole && n + 4 <= N) {
        *reinterpret_cast<Bits*>(&f) = ld_coherent(reinterpret_cast<const Bits*>(row + n));
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) f.v[e] = n + e < N ? ld_coherent(row + n + e) : rounded<O>(0.f);
    }
    return f;
}
template <typename O>
__device__ __forceinline__ void store4(O* row, int n, int N, bool whole, const float (&v)[4]) {
    if (whole && n + 4 <= N) {
        if constexpr (sizeof(O) == 4) *reinterpret_cast<float4*>(row + n) = make_float4(v[0], v[1], v[2], v[3]);
        else *reinterpret_cast<uint2*>(row + n) = make_uint2(pack2<O>(v[0], v[1]), pack2<O>(v[2], v[3]));
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (n + e < N) row[n + e] = rounded<O>(v[e]);
}

// Joins the sums of S CTAs over one tile, [token][128 rows] in the shared memory of each: rank z finishes the tokens z, z + S,
// ..., a warp to each, 4 columns to a lane, in the order of the ranks.  The cluster's shared memory gives 14 bytes a cycle, so
// eight loads under way are enough; a kernel that runs through its code once waits for instructions, so the loop is short.
template <typename T, typename O, int KIND, int S>
__device__ __forceinline__ void join(const Args& a, const float* part, volatile int* gave_up, int rank, int warp, int lane, int n0,
                                     int m0, int bn) {
    constexpr int BATCH = 8 / S;  // tokens of a warp under way
    const int n = n0 + 4 * lane, end = min(bn, a.M - m0);
    Four<T> bias;
    if (a.bias) bias = load4(static_cast<const T*>(a.bias), n, a.N, false);
    __syncwarp();
    cluster_sync_all();
    if (warp < kDrain) {
        int given_up = 0;
        const float* mine = part + 4 * lane;
        uint32_t from[S];
#pragma unroll
        for (int r = 0; r < S; ++r) {
            given_up |= ld_cluster_s32(map_rank(const_cast<int*>(gave_up), r));
            from[r] = map_rank(mine, r);
        }
#pragma unroll 1
        for (int col = rank + S * warp; col < end; col += BATCH * S * kDrain) {
            float4 f[BATCH][S];
            Four<O> old[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                const int at = min(col + i * S * kDrain, bn - 1);
#pragma unroll
                for (int r = 0; r < S; ++r) f[i][r] = ld_cluster_f4(from[r] + at * (kRows * 4));
                if (a.residual && col + i * S * kDrain < end)
                    old[i] = load4(static_cast<const O*>(a.residual) + (long long)(m0 + at) * a.ldr, n, a.N, a.res_whole);
            }
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int r = 0; r < S; ++r) y[0] += f[i][r].x, y[1] += f[i][r].y, y[2] += f[i][r].z, y[3] += f[i][r].w;
                if (a.bias) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] += as_float(bias.v[e]);
                }
                activate<KIND>(a, y);
                if (a.residual) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] += as_float(old[i].v[e]);
                }
                const int at = col + i * S * kDrain;
                if (at < end && given_up == 0) store4(static_cast<O*>(a.out) + (long long)(m0 + at) * a.ldo, n, a.N, a.out_whole, y);
            }
        }
    }
    __syncwarp();
    // no CTA leaves while another reads its sums (relaxed: what was read has been used, and the stores need not be over)
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

template <typename T, typename O, int MODE, int KIND>
__global__ void __launch_bounds__(kThreads, 1)
    linear16_tc(const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap tx,
                const __grid_constant__ CUtensorMap to, const __grid_constant__ CUtensorMap tr, const Args a, const Tiling g,
                int n_split) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    unsigned char* sm = smem_raw + (base - raw);
    const int stages = g.stages;
    const uint32_t x_rows = MODE == kPair ? g.bn / 2 : g.bn, stage_bytes = kRowsBytes + x_rows * (kChunk * 2);
    const uint32_t ring = stages * stage_bytes;
    constexpr uint32_t kSlot = kPiece * 32 * sizeof(O);
    const uint32_t slots_at = base + ring;
    uint64_t* full = reinterpret_cast<uint64_t*>(sm + ring + g.slots * (kDrain * kSlot));
    uint64_t *empty = full + kMaxStages, *ready = empty + kMaxStages, *drained = ready + 2, *done = drained + 2, *never = done + 1;
    uint64_t* landed = never + 1;  // residual pieces, by warp and slot
    uint32_t* slot = reinterpret_cast<uint32_t*>(landed + kDrain * kMaxSlots);
    volatile int* gave_up = reinterpret_cast<volatile int*>(slot + 1);

    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int rank = MODE == kSingle ? 0 : (int)cluster_ctarank();
    const int width = MODE == kPair ? 2 * kRows : kRows;  // weight rows of a tile
    const int tiles = g.tiles_n * g.tiles_m;
    // this CTA's (pair's, cluster's) tiles: first, first + step, ...
    const int ctas = MODE == kSingle ? 1 : MODE == kPair ? 2 : n_split;
    const int first = blockIdx.x / ctas, step = gridDim.x / ctas;
    const int chunks = (a.K + kChunk - 1) / kChunk;
    const int c0 = MODE == kSplit ? (int)((long long)rank * chunks / n_split) : 0;
    const int c1 = MODE == kSplit ? (int)((long long)(rank + 1) * chunks / n_split) : chunks;
    auto rows_at = [&](int t) { return (g.tokens_first ? t / g.tiles_m : t % g.tiles_n) * width; };
    auto tokens_at = [&](int t) { return (g.tokens_first ? t % g.tiles_m : t / g.tiles_n) * g.bn; };
    constexpr uint32_t TMEM = 512;  // two accumulators of up to 256 columns, or of up to 160 and the total
    const int segments = (c1 - c0 + g.segment - 1) / g.segment;

    if (warp == kDrain + 1 && lane == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tw)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tx)) : "memory");
    }
    if (warp == kDrain) {
        if constexpr (MODE == kPair) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(TMEM)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            tmem_alloc(slot, TMEM);
        }
    }
    if (tid == 0) {
        for (int i = 0; i < stages; ++i) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(ready + i, 1);
            mbar_init(drained + i, MODE == kPair ? 2 * kDrain : kDrain);
        }
        mbar_init(done, 1);
        mbar_init(never, 1);
        for (int i = 0; i < kDrain * kMaxSlots; ++i) mbar_init(landed + i, 1);
        fence_barrier_init();
        *gave_up = 0;
    }
    tc_fence_before();
    if constexpr (MODE == kPair) cluster_sync_all();  // the partner's barriers exist
    else __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *slot;
    pdl_wait_primary();
    pdl_launch_dependents();

    auto give_up = [&] {
        *gave_up = 1;
        if constexpr (MODE == kPair)
            asm volatile("st.shared::cluster.u32 [%0], 1;" ::"r"(map_rank(const_cast<int*>(gave_up), rank ^ 1)) : "memory");
        atomicOr(a.err ? a.err : &g_linear16_err, NLLB_DEV_ERR_TIMEOUT);
    };
    // Bounded wait; false (and the CTA, or pair, gives up) once any has run out.
    auto wait_one = [&](uint64_t* bar, uint32_t parity, long long budget = kWaitBudgetCycles) -> bool {
        if (mbar_try_wait(bar, parity)) return true;
        const long long t0 = clock64();
        while (!mbar_try_wait(bar, parity)) {
            if (*gave_up) return false;
            if (clock64() - t0 > budget) {
                give_up();
                return false;
            }
        }
        return true;
    };

    if (warp == kDrain) {
        // ---- fetch (a warp's loop with one thread that asks: addresses and coordinates then lie in uniform registers; by a
        // thread alone each stage took 390 cycles to ask for)
        const uint32_t full0 = MODE == kPair ? map_rank(full, 0) : smem_u32(full);
        uint32_t s = 0, turn = 0;  // the next stage's place, and how often it has come round
        bool ok = true;
        for (int t = first; t < tiles && ok; t += step) {
            const int n0 = rows_at(t) + (MODE == kPair ? rank * kRows : 0);
            const int m0 = tokens_at(t) + (MODE == kPair ? rank * (int)x_rows : 0);
            for (int c = c0; c < c1; ++c) {
                if (turn > 0 && !(ok = __all_sync(0xffffffffu, wait_one(empty + s, (turn - 1) & 1)))) break;
                const uint32_t at = base + s * stage_bytes;
                if (elect_one()) {
                    if constexpr (MODE == kPair) {
                        if (rank == 0) mbar_arrive_expect_tx(full + s, 2 * stage_bytes);
                        tma_2d_pair(at, &tw, c * kChunk, n0, full0 + 8 * s);
                        tma_2d_pair(at + kRowsBytes, &tx, c * kChunk, m0, full0 + 8 * s);
                    } else {
                        mbar_arrive_expect_tx(full + s, stage_bytes);
                        tma_2d(at, &tw, c * kChunk, n0, full + s);
                        tma_2d(at + kRowsBytes, &tx, c * kChunk, m0, full + s);
                    }
                }
                __syncwarp();
                if (++s == (uint32_t)stages) s = 0, ++turn;
            }
        }
    } else if (warp == kDrain + 1) {
        // ---- products (of both CTAs of a pair: by the first one's)
        if (MODE != kPair || rank == 0) {
            const uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;
            const uint32_t idesc = umma_idesc_f16(width, g.bn) | fmt;
            bool ok = true;
            if (a.expire) ok = __all_sync(0xffffffffu, wait_one(never, 0, kTestWaitBudgetCycles));  // nothing arrives there
            const uint64_t da0 = umma_desc_k_sw128(base), db0 = umma_desc_k_sw128(base + kRowsBytes);
            uint32_t s = 0, turn = 0, n = 0;
            bool there = false;  // the next stage is, as a look at it showed while the last one's products were issued
            for (int t = first; t < tiles && ok; t += step)
                for (int b = c0; b < c1; b += g.segment, ++n) {
                    const uint32_t acc = n & 1;
                    if (n >= 2 && !(ok = __all_sync(0xffffffffu, wait_one(drained + acc, (n / 2 - 1) & 1)))) break;
                    tc_fence_after();
                    const uint32_t d = tmem + acc * g.acc;
                    const int e = min(c1, b + g.segment);
                    for (int c = b; c < e; ++c) {
                        if (!there && !(ok = __all_sync(0xffffffffu, wait_one(full + s, turn & 1)))) break;
                        tc_fence_after();
                        const uint64_t da = da0 + s * (stage_bytes / 16), db = db0 + s * (stage_bytes / 16);  // (addresses / 16)
                        const uint32_t next = s + 1 == (uint32_t)stages ? 0 : s + 1, next_turn = next ? turn : turn + 1;
                        const bool look = mbar_test(full + next, next_turn & 1);
                        if (elect_one()) {
#pragma unroll
                            for (int k = 0; k < kChunk / 16; ++k) {
                                if constexpr (MODE == kPair) mma_pair(d, da + 2 * k, db + 2 * k, idesc, c > b || k > 0);
                                else tc_mma_f16(d, da + 2 * k, db + 2 * k, idesc, c > b || k > 0);
                            }
                            if constexpr (MODE == kPair) commit_pair(empty + s);
                            else tc_commit(empty + s);
                        }
                        there = __all_sync(0xffffffffu, look);
                        s = next, turn = next_turn;
                    }
                    if (!ok) break;
                    if (elect_one()) {
                        if constexpr (MODE == kPair) commit_pair(ready + acc);
                        else tc_commit(ready + acc);
                    }
                    __syncwarp();
                }
            // what was issued is over before tensor memory is given back
            if (elect_one()) {
                if constexpr (MODE == kPair) commit_pair(done);
                else tc_commit(done);
                (void)mbar_wait_bounded(done, 0);
            }
            __syncwarp();
        }
    } else {
        // ---- drain: lane quarter warp % 4, a lane to a column; the tile's pieces in turns between the two halves.  Rows that
        // start on 16 bytes go out by TMA, and their residual comes by TMA into the same slot, slots - 2 pieces ahead and
        // across tiles.  (Through the lanes' registers a CTA had no more than the few KB of its L1 cache on their way: 238
        // rows of 60608 over k = 320 with a residual in fp32 46 us.)
        constexpr int PIECE = kPiece;
        const int quarter = warp & 3, half = warp >> 2;
        const uint32_t from0 = tmem + ((uint32_t)(quarter * 32) << 16), mask = g.slots - 1, shift = g.slots == 8 ? 3 : 2;
        const uint32_t slot0 = slots_at + warp * g.slots * kSlot;
        O* const mem0 = reinterpret_cast<O*>(sm + (slot0 - base)) + lane;
        uint64_t* const bars = landed + warp * kMaxSlots;
        struct Place { int t, n0, m0, count; };  // a tile; this warp's first column, its first token, its pieces with tokens
        auto place_of = [&](int t) {
            Place p = {t, 0, 0, 0};
            if (t < tiles) {
                p.n0 = rows_at(t) + (MODE == kPair ? rank * kRows : 0) + quarter * 32, p.m0 = tokens_at(t);
                p.count = p.n0 < a.N ? (min(g.bn, a.M - p.m0) + PIECE - 1) / PIECE : 0;
            }
            return p;
        };
        Place here = place_of(first), there = here;
        int next_asked = half;            // of `there`: the piece whose residual is asked for next
        uint32_t used = 0, asked = 0;     // pieces of this warp
        auto ask = [&] {
            while (there.t < tiles && next_asked >= there.count) there = place_of(there.t + step), next_asked = half;
            if (there.t >= tiles) return;
            if (lane == 0) {
                mbar_arrive_expect_tx(bars + (asked & mask), kSlot);
                tma_2d(slot0 + (asked & mask) * kSlot, &tr, there.n0, there.m0 + next_asked * PIECE, bars + (asked & mask));
            }
            ++asked, next_asked += 2;
        };
        if (MODE != kSplit && a.res_whole)
            for (int i = 0; i < g.slots - 2; ++i) ask();
        bool ok = true;
        uint32_t n = 0;  // accumulators
        const uint32_t total = from0 + 2 * g.acc;
        auto release = [&](uint32_t acc) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (MODE == kPair) arrive_at(map_rank(drained + acc, 0));
                else arrive_here(drained + acc);
            }
        };
        for (; here.t < tiles && ok; here = place_of(here.t + step), ++n) {
            // all segments but the last one are added up in tensor memory
            for (int b = 1; b < segments; ++b, ++n) {
                const uint32_t acc = n & 1, from = from0 + acc * g.acc;
                if (!(ok = __all_sync(0xffffffffu, wait_one(ready + acc, (n / 2) & 1)))) break;
                tc_fence_after();
                for (int i = half; i < here.count; i += 2) {
                    float v[PIECE], t[PIECE];
                    tmem_ask(from + i * PIECE, v);
                    if (b > 1) tmem_ask(total + i * PIECE, t);
                    tmem_wait(v);
                    if (b > 1) {
                        tmem_wait(t);
#pragma unroll
                        for (int j = 0; j < PIECE; ++j) v[j] += t[j];
                    }
                    tmem_put(total + i * PIECE, v);
                }
                release(acc);
            }
            if (!ok) break;
            const uint32_t acc = n & 1, from = from0 + acc * g.acc;
            if (!(ok = __all_sync(0xffffffffu, wait_one(ready + acc, (n / 2) & 1)))) break;
            tc_fence_after();
            if constexpr (MODE == kSplit) {
                // over the ring, which is done with and larger (a partial sum takes 64 KB at most)
                float* part = reinterpret_cast<float*>(sm) + quarter * 32 + lane;
                for (int i = half; i < here.count; i += 2) {
                    float v[PIECE], t[PIECE];
                    tmem_ask(from + i * PIECE, v);
                    if (segments > 1) tmem_ask(total + i * PIECE, t);
                    tmem_wait(v);
                    if (segments > 1) {
                        tmem_wait(t);
#pragma unroll
                        for (int j = 0; j < PIECE; ++j) v[j] += t[j];
                    }
#pragma unroll
                    for (int j = 0; j < PIECE; ++j) part[(i * PIECE + j) * kRows] = v[j];
                }
                break;  // (one tile)
            } else {
                const bool mine = here.n0 + lane < a.N;
                const float bias = a.bias && mine ? as_float(ld_coherent(static_cast<const T*>(a.bias) + here.n0 + lane)) : 0.f;
                // (a TMA store writes the 16 bytes in which a row ends as a whole, and columns of others may follow there)
                const bool by_tma = a.out_whole && (a.out_end || here.n0 + 32 <= a.N);
                if (by_tma && !a.residual && segments == 1) {
                    // (as below, and nothing that is not needed: 6318 rows of 3200 over k = 256 20 us, there 22.5)
                    float next[PIECE];
                    if (half < here.count) tmem_ask(from + half * PIECE, next);
                    for (int i = half; i < here.count; i += 2, ++used) {
                        const uint32_t at = used & mask;
                        O* mem = mem0 + at * (kSlot / sizeof(O));
                        float v[PIECE];
                        tmem_wait(next);
#pragma unroll
                        for (int j = 0; j < PIECE; ++j) v[j] = next[j] + bias;
                        if (i + 2 < here.count) tmem_ask(from + (i + 2) * PIECE, next);
                        activate<KIND>(a, v);
                        if (lane == 0) {
                            if (g.slots == 8) stores_read<7>();
                            else stores_read<3>();
                        }
                        __syncwarp();
#pragma unroll
                        for (int j = 0; j < PIECE; ++j) mem[j * 32] = rounded<O>(v[j]);
                        fence_async_smem();
                        __syncwarp();
                        if (lane == 0) tma_store_2d(&to, here.n0, here.m0 + i * PIECE, slot0 + at * kSlot);
                        __syncwarp();
                    }
                    tmem_wait(next);
                    release(acc);
                    continue;
                }
                const bool res_lanes = a.residual && !a.res_whole && mine;
                O old[PIECE];  // (asked for a piece ahead)
                auto ask_lanes = [&](int i) {
                    const int m0 = here.m0 + i * PIECE;
                    const O* p = static_cast<const O*>(a.residual) + m0 * a.ldr + here.n0 + lane;
#pragma unroll
                    for (int j = 0; j < PIECE; ++j, p += a.ldr)
                        if (m0 + j < a.M) old[j] = ld_coherent(p);
                };
                if (res_lanes && half < here.count) ask_lanes(half);
                float next[PIECE];
                if (half < here.count) tmem_ask(from + half * PIECE, next);
                if (!by_tma && lane == 0) stores_read<0>();  // (of tiles before: no piece of this one waits for a slot's store)
                for (int i = half; i < here.count; i += 2, ++used) {
                    const int m0 = here.m0 + i * PIECE, rows = min(PIECE, a.M - m0);
                    const uint32_t at = used & mask;
                    O* mem = mem0 + at * (kSlot / sizeof(O));
                    float v[PIECE];
                    tmem_wait(next);
                    if (segments > 1) {
                        float t[PIECE];
                        tmem_ask(total + i * PIECE, t);
                        tmem_wait(t);
#pragma unroll
                        for (int j = 0; j < PIECE; ++j) next[j] += t[j];
                    }
#pragma unroll
                    for (int j = 0; j < PIECE; ++j) v[j] = next[j] + bias;
                    if (i + 2 < here.count) tmem_ask(from + (i + 2) * PIECE, next);
                    activate<KIND>(a, v);
                    if (a.res_whole) {
                        if (!(ok = __all_sync(0xffffffffu, wait_one(bars + at, (used >> shift) & 1)))) break;
#pragma unroll
                        for (int j = 0; j < PIECE; ++j) v[j] += as_float(mem[j * 32]);
                    } else if (res_lanes) {
#pragma unroll
                        for (int j = 0; j < PIECE; ++j) v[j] += as_float(old[j]);  // (rows past the last one: unused)
                        if (i + 2 < here.count) ask_lanes(i + 2);
                    }
                    if (by_tma) {
                        if (!a.res_whole) {  // (else the slot's last store has been waited for)
                            if (lane == 0) stores_read<3>();
                            __syncwarp();
                        }
#pragma unroll
                        for (int j = 0; j < PIECE; ++j) mem[j * 32] = rounded<O>(v[j]);
                        fence_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            tma_store_2d(&to, here.n0, m0, slot0 + at * kSlot);
                            if (a.res_whole) stores_read<2>();
                        }
                    } else if (mine) {
                        O* p = static_cast<O*>(a.out) + m0 * a.ldo + here.n0 + lane;
#pragma unroll
                        for (int j = 0; j < PIECE; ++j, p += a.ldo)
                            if (j < rows) *p = rounded<O>(v[j]);
                    }
                    __syncwarp();
                    if (a.res_whole) ask();  // into the slot of the piece before the last
                }
                tmem_wait(next);  // (what was asked for and not used)
                release(acc);
            }
        }
        // nothing reads or writes shared memory once the CTA has ended
        if (lane == 0) stores_done();
        for (; used < asked; ++used) (void)mbar_wait_bounded(bars + (used & mask), (used >> shift) & 1, kTestWaitBudgetCycles);
    }

    tc_fence_before();
    if constexpr (MODE == kPair) cluster_sync_all();  // neither leaves while the other uses its barriers
    else if constexpr (MODE == kSingle) __syncthreads();
    if constexpr (MODE == kSplit) {
        const float* part = reinterpret_cast<const float*>(sm);
        const int n0 = rows_at(first), m0 = tokens_at(first);
        if (n_split == 2) join<T, O, KIND, 2>(a, part, gave_up, rank, warp, lane, n0, m0, g.bn);
        else if (n_split == 4) join<T, O, KIND, 4>(a, part, gave_up, rank, warp, lane, n0, m0, g.bn);
        else join<T, O, KIND, 8>(a, part, gave_up, rank, warp, lane, n0, m0, g.bn);
    }
    if (warp == kDrain) {
        // Given up: time for what is in flight to land before the CTA ends, whoever asked for it and has ended since (of a pair
        // the second CTA, whose stages complete at the first, too).  Waits on their barriers, here or behind the fetching
        // loop, would cost every launch (128 rows of 1024 over k = 1024 6.8 us instead of 6.2).
        if (lane == 0 && *gave_up) (void)mbar_wait_bounded(never, 0, kTestWaitBudgetCycles);
        __syncwarp();
        tc_fence_after();
        if constexpr (MODE == kPair)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM) : "memory");
        else
            tmem_dealloc(tmem, TMEM);
    }
}

// ---- launches --------------------------------------------------------------------------------------------------

void with_cluster(cudaLaunchConfig_t& cfg, cudaLaunchAttribute (&attr)[2], int ctas, cudaStream_t st) {
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = kPdlLaunch;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)ctas;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctas > 1 ? 2 : 1;
}

template <typename T, typename O, int NT, int KG>
cudaError_t launch_few_by(const Args& a, int num_sms, cudaStream_t st) {
    constexpr int ROWS = kFewRows * kFewWarps / KG;
    const long long rows = (a.N + ROWS - 1) / ROWS, tokens = (a.M + 8 * NT - 1) / (8 * NT);
    // CTAs that share k, while that leaves two or fewer per SM and each warp something to do
    int n_split = 1;
    while (KG == kFewWarps && n_split < 8 && rows * tokens * n_split * 2 <= 2LL * num_sms &&
           a.K > n_split * kFewWarps * 32 * kFewBlocks)
        n_split *= 2;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    cfg.gridDim = dim3((unsigned)(rows * n_split), (unsigned)std::min(tokens, 65535LL), 1);
    cfg.blockDim = dim3(kFewWarps * 32, 1, 1);
    with_cluster(cfg, attr, n_split, st);
    return cudaLaunchKernelEx(&cfg, linear16_few<T, O, NT, KG>, a, n_split);
}

template <typename T, typename O, int NT>
cudaError_t launch_few(const Args& a, int num_sms, cudaStream_t st) {
    // warps that share k where it is long enough for them (one row of 241856 over k = 64: 95 us with eight warps on k)
    constexpr int STEP = 32 * kFewBlocks;
    if (a.K <= STEP) return launch_few_by<T, O, NT, 1>(a, num_sms, st);
    if (a.K <= 4 * STEP) return launch_few_by<T, O, NT, 4>(a, num_sms, st);
    return launch_few_by<T, O, NT, 8>(a, num_sms, st);
}

template <typename T, typename O, int MODE, int KIND>
cudaError_t launch_mode(const Args& a, Tiling g, int ctas, int groups, cudaStream_t st) {
    const int width = MODE == kPair ? 2 * kRows : kRows, x_rows = MODE == kPair ? g.bn / 2 : g.bn;
    const int stage = (int)kRowsBytes + x_rows * kChunk * 2;
    constexpr uint32_t kSlot = kPiece * 32 * sizeof(O);
    g.slots = MODE == kSplit ? 0 : sizeof(O) == 2 && (a.res_whole || a.K <= 1024) ? 8 : 4;
    g.stages = std::min(kMaxStages, ((int)(kSmem - kBars) - g.slots * (int)(kDrain * kSlot)) / stage);
    g.segment = (sizeof(O) == 4 ? kSegment : kSegment16) / kChunk;
    g.acc = a.K > (MODE == kSplit ? ctas : 1) * g.segment * kChunk ? 160 : 256;
    g.tiles_n = (a.N + width - 1) / width, g.tiles_m = (a.M + g.bn - 1) / g.bn;
    g.tokens_first = (long long)a.N >= a.M;  // the larger operand is read once, while its tile is in use
    CUtensorMap tw, tx, to, tr;
    constexpr MapType type = std::is_same<T, __nv_bfloat16>::value ? MapType::bf16 : MapType::f16;
    constexpr MapType out_type = sizeof(O) == 4 ? MapType::f32 : type;
    cudaError_t e = encode_rows_map(&tw, a.w, type, a.K, a.N, a.ldw, kChunk, kRows, true);
    if (e == cudaSuccess) e = encode_rows_map(&tx, a.x, type, a.K, a.M, a.ldx, kChunk, x_rows, true);
    to = tr = tx;  // (not looked at)
    if (e == cudaSuccess && a.out_whole) e = encode_rows_map(&to, a.out, out_type, a.N, a.M, a.ldo, 32, kPiece, false);
    if (e == cudaSuccess && a.res_whole) e = encode_rows_map(&tr, a.residual, out_type, a.N, a.M, a.ldr, 32, kPiece, false);
    if (e != cudaSuccess) return e;
    // (once per device)
    static std::atomic<unsigned long long> configured{0};
    const unsigned long long bit = 1ull << (a.device & 63);
    if (!(configured.load() & bit) || a.device > 63) {
        e = cudaFuncSetAttribute(linear16_tc<T, O, MODE, KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem + 1024);
        if (e != cudaSuccess) return e;
        configured.fetch_or(bit);
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    cfg.gridDim = dim3((unsigned)(groups * ctas), 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = (size_t)g.stages * stage + g.slots * kDrain * kSlot + kBars + 1024;
    with_cluster(cfg, attr, ctas, st);
    return cudaLaunchKernelEx(&cfg, linear16_tc<T, O, MODE, KIND>, tw, tx, to, tr, a, g, ctas);
}

template <typename T, typename O, int MODE>
cudaError_t launch_kind(const Args& a, const Tiling& g, int ctas, int groups, cudaStream_t st) {
    if (a.kind == kClamp) return launch_mode<T, O, MODE, kClamp>(a, g, ctas, groups, st);
    if (a.kind == kSwish) return launch_mode<T, O, MODE, kSwish>(a, g, ctas, groups, st);
    return launch_mode<T, O, MODE, kGelu>(a, g, ctas, groups, st);
}

// How many clusters of 2, 4 or 8 CTAs a device holds at a time (asked for once; where that fails, none).
int most_clusters(int device, int ctas) {
    static std::atomic<int> known[64][3];
    const int i = ctas == 2 ? 0 : ctas == 4 ? 1 : 2;
    if (device > 63) return 0;
    int n = known[device][i].load(std::memory_order_relaxed);
    if (n == 0) {
        const auto kernel = linear16_tc<__nv_bfloat16, __nv_bfloat16, kSplit, kClamp>;
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr[2];
        cfg.gridDim = dim3(8 * ctas, 1, 1), cfg.blockDim = dim3(kThreads, 1, 1), cfg.dynamicSmemBytes = kSmem + 1024;
        with_cluster(cfg, attr, ctas, nullptr);
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem + 1024);
        if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
        if (e != cudaSuccess) (void)cudaGetLastError(), n = 0;
        known[device][i].store(n > 0 ? n : -1, std::memory_order_relaxed);
    }
    return n;
}

template <typename T, typename O>
cudaError_t launch(const Args& a, int num_sms, cudaStream_t st) {
    // Few tokens: warp-level products while the weights are few as well, for the tensor cores then take longer to start (1024 x
    // 1024 by 1, 16 and 64 tokens 2.8, 3.4 and 4.1 us against 4.8, 4.8 and 5.5 on the tensor cores; 4096 x 1024 by 16 4.1
    // against 6.1).  These keep more of the weights on their way (16384 x 1024 by 1 and 16 9.0 and 13.0 us against 8.7 and
    // 8.9), and a short k is over at once there (1024 x 128 by 16 and 64 4.1 and 6.9 us against 4.1; 2048 x 256 by 128, two
    // rounds of CTAs, 8.2 against 4.8).
    const long long weights = (long long)a.N * a.K;
    if (a.K < kChunk) return a.M <= 8 ? launch_few<T, O, 1>(a, num_sms, st) : launch_few<T, O, 2>(a, num_sms, st);
    if (a.M <= 8 && weights <= 1 << 23) return launch_few<T, O, 1>(a, num_sms, st);
    if (a.M > 8 && a.M <= 16 && a.K > 128 && a.N <= 8192 && weights <= 1 << 23) return launch_few<T, O, 2>(a, num_sms, st);
    const int few_rows = a.K > 512 ? 16 : 32;  // of a CTA (launch_few)
    if (a.M > 16 && a.K > 256 && a.K <= 1024 && (long long)((a.N + few_rows - 1) / few_rows) * ((a.M + 31) / 32) <= num_sms)
        return launch_few<T, O, 4>(a, num_sms, st);
    // The form and the tile of tokens that take the fewest cycles, as they were measured: a stage's products or its bytes from
    // L2; a drained tile beside the next one's products; for a shared k the sums' way through the cluster (14 bytes a cycle).
    const int widest = a.K > (sizeof(O) == 4 ? kSegment : kSegment16) ? 160 : 256;  // (the segments' total takes its room)
    const int chunks = (a.K + kChunk - 1) / kChunk, n_tiles = (a.N + kRows - 1) / kRows, n_pairs = (n_tiles + 1) / 2;
    Tiling g = {};
    int mode = kSingle, ctas = 1;
    double least = 1e300, groups = 1.0;
    auto take = [&](double t, int m, int c, double n, int bn) {
        if (t < least * 0.999) least = t, mode = m, ctas = c, groups = n, g.bn = bn;
    };
    const double sms = num_sms, half = num_sms / 2, per_sm = 1.0 / sms, per_half = 1.0 / half;
    for (int bn = 32; bn <= widest; bn += 32) {
        const double m_tiles = (a.M + bn - 1) / bn, tiles = n_tiles * m_tiles, pairs = n_pairs * m_tiles;
        const double drain = 880.0 / 32 * bn, stage = std::max(2.0 * bn, 256.0 + 2.0 * bn), pair_stage = std::max(2.0 * bn, 256.0 + bn);
        const double one = chunks * stage, two = chunks * pair_stage;
        auto rounds = [](double x) { return std::ceil(x - 1e-7); };
        take(rounds(tiles * per_sm) * (std::max(one, drain) + 300.0) + std::min(one, drain), kSingle, 1, std::min(tiles, sms), bn);
        take(rounds(pairs * per_half) * (std::max(two, drain) + 300.0) + std::min(two, drain), kPair, 2, std::min(pairs, half), bn);
        for (int split = 2; split <= 8 && bn <= 128 && chunks >= 2 * split && tiles * split <= sms && tiles <= most_clusters(a.device, split); split *= 2)
            take((chunks + split - 1) / split * stage + 200.0 / 32 * bn + 1500.0 + bn * 512.0 / 14.0 * (split - 1) / split, kSplit, split, tiles, bn);
        if (bn >= a.M) break;
    }
    if (mode == kSplit) return launch_kind<T, O, kSplit>(a, g, ctas, (int)groups, st);
    if (mode == kPair) return launch_kind<T, O, kPair>(a, g, ctas, (int)groups, st);
    return launch_kind<T, O, kSingle>(a, g, ctas, (int)groups, st);
}

int bad(const char* msg) { return set_error(NLLB_ATTN_EINVAL, msg); }

thread_local bool t_expire_next = false;

}  // namespace
}  // namespace nllb

extern "C" int nllb_linear16_test_expire_next_wait(void) {
    nllb::t_expire_next = true;
    return NLLB_ATTN_OK;
}

extern "C" int nllb_linear16_status(void* stream) {
    using namespace nllb;
    static std::mutex one_at_a_time;  // (g_linear16_taken)
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    int err = 0;
    cudaError_t e = cudaStreamSynchronize(st);
    if (e == cudaSuccess) {
        std::lock_guard<std::mutex> lock(one_at_a_time);
        linear16_take_err<<<1, 1, 0, st>>>();
        e = cudaGetLastError();
        if (e == cudaSuccess) e = cudaMemcpyFromSymbolAsync(&err, g_linear16_taken, sizeof(int), 0, cudaMemcpyDeviceToHost, st);
        if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    }
    if (e != cudaSuccess) return set_error(NLLB_ATTN_ECUDA, std::string("nllb_linear16_status: ") + cudaGetErrorString(e));
    if (err) return set_error(NLLB_ATTN_ETIMEOUT, "a bounded device wait of nllb_linear16 gave up");
    return NLLB_ATTN_OK;
}

namespace nllb {
namespace {

int run(const nllb_linear16_args* s, int* error, void* stream) {
    const bool expire = t_expire_next;  // (this call's, whatever becomes of it)
    t_expire_next = false;
    if (!s) return bad("args is NULL");
    if (s->dtype != NLLB_F16 && s->dtype != NLLB_BF16) return bad("dtype must be NLLB_F16 or NLLB_BF16");
    if (s->out_dtype != s->dtype && s->out_dtype != NLLB_F32) return bad("out_dtype must be dtype or NLLB_F32");
    if (s->act < NLLB_ACT_NONE || s->act > NLLB_ACT_SILU) return bad("act must be one of NLLB_ACT_*");
    if (s->M < 0 || s->N < 1 || s->K < 1) return bad("M >= 0, N >= 1 and K >= 1 required");
    if (s->M > (1 << 24) || s->N > (1 << 24) || s->K > (1 << 24)) return set_error(NLLB_ATTN_ECAPACITY, "a size above 2^24");
    if ((long long)s->M * s->N > 1LL << 40) return set_error(NLLB_ATTN_ECAPACITY, "more outputs than a call takes");
    if (s->M == 0) return NLLB_ATTN_OK;
    if (!s->x || !s->w || !s->out) return bad("x, w and out are required");
    if (s->ldx < s->K || s->ldw < s->K || s->ldo < s->N || (s->residual && s->ldr < s->N))
        return bad("ldx and ldw must be at least K, ldo and ldr at least N");
    if (((reinterpret_cast<uintptr_t>(s->x) | reinterpret_cast<uintptr_t>(s->w)) & 15u) || ((s->ldx | s->ldw) & 7))
        return bad("rows of x and w must be 16-byte aligned, ldx and ldw multiples of 8");
    if (s->ldx > (1LL << 36) || s->ldw > (1LL << 36)) return set_error(NLLB_ATTN_ECAPACITY, "ldx or ldw above 2^36");
    const uintptr_t size = s->out_dtype == NLLB_F32 ? 4 : 2;
    if ((reinterpret_cast<uintptr_t>(s->out) | reinterpret_cast<uintptr_t>(s->residual)) % size ||
        reinterpret_cast<uintptr_t>(s->bias) % 2)
        return bad("out, residual and bias must be aligned to their types");
    const MemRows out(s->out, s->M, s->ldo * (long long)size, s->N * (long long)size);
    if (meet(out, MemRows(s->x, s->M, s->ldx * 2, s->K * 2LL)) || meet(out, MemRows(s->w, s->N, s->ldw * 2, s->K * 2LL)) ||
        (s->bias && meet(out, MemRows(s->bias, 1, 0, s->N * 2LL))))
        return bad("out may not overlap x, w or bias");
    if (s->residual && !(s->residual == s->out && (s->ldr == s->ldo || s->M == 1)) &&
        meet(out, MemRows(s->residual, s->M, s->ldr * (long long)size, s->N * (long long)size)))
        return bad("residual may be out itself, with the same ldr, and may not overlap it otherwise");
    auto whole = [&](const void* base, long long ld) {
        return ((reinterpret_cast<uintptr_t>(base) | (uintptr_t)(ld * (long long)size)) & 15u) == 0 && ld <= 1LL << 36;
    };
    Args a = {s->x, s->w, s->bias, s->residual, s->out, s->ldx, s->ldw, s->ldr, s->ldo, s->M, s->N, s->K, kClamp, 0.f, 0.f,
              whole(s->out, s->ldo), s->residual && whole(s->residual, s->ldr), s->N * (long long)size % 16 == 0, expire, 0, error};
    switch (s->act) {
        case NLLB_ACT_NONE: a.c1 = -INFINITY; break;
        case NLLB_ACT_RELU: break;
        case NLLB_ACT_GELU: a.kind = kGelu; break;
        case NLLB_ACT_GELU_TANH: a.kind = kSwish, a.c1 = 2.3022082f, a.c2 = 0.10294324f; break;  // 2 sqrt(2/pi) log2 e (1, 0.044715)
        default: a.kind = kSwish, a.c1 = kLog2e;  // SILU
    }
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    int device = 0, num_sms = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&num_sms, cudaDevAttrMultiProcessorCount, device);
    a.device = device;
    if (e == cudaSuccess) {
        const bool wide = s->out_dtype == NLLB_F32;
        if (s->dtype == NLLB_F16) e = wide ? launch<__half, float>(a, num_sms, st) : launch<__half, __half>(a, num_sms, st);
        else e = wide ? launch<__nv_bfloat16, float>(a, num_sms, st) : launch<__nv_bfloat16, __nv_bfloat16>(a, num_sms, st);
    }
    if (e != cudaSuccess) return set_error(NLLB_ATTN_ECUDA, std::string("nllb_linear16: ") + cudaGetErrorString(e));
    return NLLB_ATTN_OK;
}

}  // namespace
}  // namespace nllb

extern "C" int nllb_linear16(const nllb_linear16_args* s, void* stream) { return nllb::run(s, nullptr, stream); }

extern "C" int nllb_linear16_reporting(const nllb_linear16_args* s, int* error, void* stream) {
    if (!error || reinterpret_cast<uintptr_t>(error) % 4) {
        nllb::t_expire_next = false;
        return nllb::bad("error must be an address, aligned to its type");
    }
    return nllb::run(s, error, stream);
}
