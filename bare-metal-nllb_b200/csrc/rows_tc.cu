// rows_tc.cu -- attention of many query rows over many keys on the 5th
// generation tensor cores (sm_100a).
//
//   S = Q K^T,  P = 2^(scale log2(e) S - m),  O += P V,  out = O / sum P
//
// over tiles of 128 keys, with m the running maximum of a row, held back: the
// row's sums are only rescaled when a maximum has grown by more than 2^8, so
// the accumulator in tensor memory is rarely touched between products.
//
// Roles of a CTA's warps: 4 or 8 per query tile for the softmax (one thread, or
// two, to a row = a TMEM lane), 3 that fetch, 1 that issues the products.  Key
// rows are fetched row by row (cp.async of 16 bytes, or loads and a split for
// fp32): two lanes keep a row's address in registers, so pages of any size,
// strides of any order and masks need no copy, and a hidden row becomes zeros
// without being read.  K lies K-major and V as it comes (an MN-major operand),
// both in the 128-byte swizzle; P goes back to tensor memory and is the A
// operand from there: over S, or, with two tiles of heads of 64, beside it, so
// that the next scores can be taken as soon as a row's last ones are read.
// With two query tiles per CTA the tensor cores work on one while the other's
// softmax runs, and a key tile is fetched once for 256 rows; with one tile two
// CTAs share an SM to the same end.  Few CTAs over many keys share the keys in
// a cluster and join their states through distributed shared memory.
//
// Types: 16-bit inputs are the operands as they come, the weights are rounded
// to the type (half a step each, unbiased; the sum that divides them stays
// fp32).  The tensor cores cut what they add to a sum: n keys lose up to n/16
// steps of fp32, n 2^-27 of an output (measured 6.4e-9 n).  Up to 32768 keys
// that is half of what fp16 rounds an output by, and a CTA's tiles are added
// there.  Calls of more keys move the sums of 16 tiles on to a total that the
// softmax threads add to, and fp32 ones every tile (1024 rows of 32 heads over
// 100000 keys: heads of 64 2.04 ms, 1.86 without; of 128, where two tiles leave
// no room for the total, 2.87 and 2.40).  fp32 inputs and weights are split
// into two fp16 parts, hi + lo, and a product is taken as hi hi' + hi lo' +
// lo hi' (22 bits, and an absolute 2^-25 where lo leaves fp16's normal range).
// So that this holds at any size, rows are divided by powers of two first where
// the largest size lies outside [2^-3, 65504): of 16 query or key rows, which a
// warp settles for itself, each row by its own size, and the scores undo it; of
// a tile of values, alike, which the sum over the tiles undoes.  (Ordinary
// sizes pay for the look: 64 prefixes 71 us instead of 67, 128 scored sentences
// 95 instead of 91.)  Weights are held times 2^7, so fp16 keeps them normal
// down to 2^-21 of the largest while 2^7 * 2^8 stays in its range.
//
// Measured: documents of 1500..2048 over 3500..4096 rows, heads of 128, bf16,
// a tenth of the keys hidden 306 us (687 TFLOP/s); chunks of 500..1024 tokens
// behind up to 7000, heads of 64, 340 us (496 TFLOP/s of visible pairs); 128
// sentences of fp32 95 us.  Bound by the softmax warps' instructions (without
// exponentials the chunks take 287 us, without the softmax 216); a share of
// the exponentials on the fp32 multipliers, or turns between the two tiles'
// exponentials, made it slower (a quarter of them 366 us, turns 361 us).
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "rows.cuh"

namespace nllb {
namespace {

constexpr int kTile = 128;              // query rows of a tile, keys of a tile
constexpr int kLoaders = 96;            // fetching threads: 8 or 12 warps in all, so registers divide evenly
constexpr int kLongKeys = 32768;        // of 16 bits: from there on a CTA's tiles are added outside the tensor cores
constexpr int kTilesTogether = 16;       // there: tiles that the tensor cores add
constexpr float kGrow = 8.0f;           // a maximum may lag by 2^8
constexpr float kWeightExp = 7.0f;      // weights are held times 2^7
constexpr uint32_t kBlock = 128 * 128;  // bytes of [128 rows][64 16-bit elements]

template <typename T, int D, int NQ, bool LONG>
struct Cfg {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int PARTS = F32 ? 2 : 1;
    static constexpr int KB = D / 64;                 // 64-element blocks of a row
    static constexpr uint32_t PART = kBlock * KB;     // one part of a [128][D] operand
    static constexpr uint32_t OPER = PART * PARTS;
    // key tiles in flight: what leaves room for two CTAs per SM with one query tile, or fills the SM with two
    static constexpr int ST = F32 ? 1 : (NQ == 2 ? (D == 64 ? 4 : 2) : (D == 64 || LONG ? 2 : 1));
    // Softmax warps of a query tile; with 8, two threads share a row.  Two tiles: 4 (long chunks 343 us, with 8 355);
    // one, where the time to the first result counts: 8 (64 prefixes 70 us, with 4 88).
    static constexpr int WPT = NQ == 2 ? 4 : 8, SOFT = NQ * WPT * 32;  // and softmax threads in all
    static constexpr int COLS = 128 * 4 / WPT;                      // scores of a thread
    static constexpr int WORDS = 2 * ST + 2;  // key tiles whose visible keys are kept
    static constexpr uint32_t SQ = 0, SK = NQ * OPER, SV = SK + ST * OPER, SAUX = SV + ST * OPER;
    static constexpr uint32_t VALID = SAUX, MAXS = VALID + WORDS * 16;
    // fp32: what rows of the queries and of the K tiles (the first one last), and V tiles, were divided by; a byte per
    // warp that tells of divisors other than 1; largest sizes of V: of the first tile, by softmax warp, and of others
    static constexpr uint32_t QS = MAXS + (WPT == 8 ? 2 * NQ * 2 * 128 * 4 : 0), KS = QS + (F32 ? kTile * 4 : 0);
    static constexpr uint32_t VS = KS + (F32 ? (WORDS + 1) * kTile * 4 : 0), TOPS = VS + (F32 ? (WORDS + 1) * 4 : 0);
    static constexpr uint32_t ODD = (TOPS + (F32 ? (8 + 2 * kLoaders / 32) * 4 : 0) + 7) / 8 * 8;  // queries, V's first, K tiles
    static constexpr uint32_t BARS = ODD + (F32 ? (WORDS + 3) * 8 : 0);
    // P beside S in tensor memory, where there is room: the next scores can then be taken as soon as a row is read
    static constexpr bool AHEAD = NQ == 2 && D == 64 && !LONG;
    // fp32, and 16 bits over many keys: the outputs' total.  The tensor cores cut what they accumulate, so a sum over many
    // tiles would drift; they sum one tile, or kTilesTogether, and the softmax threads add those.
    static constexpr bool TOTAL = F32 || LONG;
    static constexpr uint32_t O_COL = NQ * 128, P_COL = O_COL + NQ * D, T_COL = P_COL;
    // fp32: the softmax threads also fetch the first key tile, with all of its loads in flight at once
    static constexpr bool FIRST = F32;  // (one slot: the first tile's phase is simply not counted)
    static constexpr int N_BARS = 4 * ST + 9 * NQ + 3;
    static constexpr uint32_t SLOT = BARS + N_BARS * 8, BYTES = SLOT + 16;
    static constexpr uint32_t SMEM = BYTES + 1024;  // + alignment slack
    static constexpr int THREADS = SOFT + kLoaders + 32;
    static constexpr uint32_t TMEM = NQ == 2 || (TOTAL && D == 128) ? 512 : 256;  // S: 128 columns per tile, O: D per tile
    static constexpr int CTAS = NQ == 2 || (TOTAL && D == 128) ? 1 : 2;
    static constexpr int LD = D + 4;  // fp32 row of a split's state: D sums, then m, l
    static_assert(NQ * 128 + NQ * D + (AHEAD ? NQ * 64 : 0) + (TOTAL ? NQ * D : 0) <= (int)TMEM, "tensor memory");
    static_assert(!(F32 && LONG), "fp32 adds every tile");
    static_assert(128 * LD * 4 <= (int)SAUX || NQ == 2, "a split's state fits over the operands");
};

// byte offset of 16-byte chunk c of row r in an operand part
__device__ __forceinline__ uint32_t chunk_off(int r, int c) {
    return (uint32_t)((c >> 3) * (int)kBlock + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// Arrives on `bar` (one of its expected arrivals) once this thread's copies so far have landed.  Their writes are
// plain ones: who waits on the barrier fences before the tensor cores read them.
__device__ __forceinline__ void cp_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void cp_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

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
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}


// D[128 x N] (+)= A . B, A from tensor memory.
__device__ __forceinline__ void tc_mma_f16_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                              uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

// 16 columns of this thread's lane (warp-wide).
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// 8 columns, the load to be waited for.
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 64 or 128 columns of this thread's lane (warp-wide), under one wait.
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, float* v) {
    uint32_t r[N];
#pragma unroll
    for (int k = 0; k < N; k += 32)
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
            "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, "
            "%22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
            : "=r"(r[k]), "=r"(r[k + 1]), "=r"(r[k + 2]), "=r"(r[k + 3]), "=r"(r[k + 4]), "=r"(r[k + 5]), "=r"(r[k + 6]), "=r"(r[k + 7]),
              "=r"(r[k + 8]), "=r"(r[k + 9]), "=r"(r[k + 10]), "=r"(r[k + 11]), "=r"(r[k + 12]), "=r"(r[k + 13]), "=r"(r[k + 14]), "=r"(r[k + 15]),
              "=r"(r[k + 16]), "=r"(r[k + 17]), "=r"(r[k + 18]), "=r"(r[k + 19]), "=r"(r[k + 20]), "=r"(r[k + 21]), "=r"(r[k + 22]), "=r"(r[k + 23]),
              "=r"(r[k + 24]), "=r"(r[k + 25]), "=r"(r[k + 26]), "=r"(r[k + 27]), "=r"(r[k + 28]), "=r"(r[k + 29]), "=r"(r[k + 30]), "=r"(r[k + 31])
            : "r"(taddr + k));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ float ex2_approx(float x) {  // 2^x, -inf -> +0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float max_nan(float a, float b, float c) {  // NaN if any is
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float c;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
    return c;
}

// x rounded to 11 significant bits, exact in fp16's normal range.
__device__ __forceinline__ float round11(float x) {
    return __uint_as_float((__float_as_uint(x) + 0x1000u) & 0xFFFFE000u);
}
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
    const float ha = round11(a), hb = round11(b);
    hi = pack2<__half>(ha, hb);
    lo = pack2<__half>(a - ha, b - hb);
}

// 8 fp32 values as a 16-byte chunk of each part of an operand.
template <uint32_t PART>
__device__ __forceinline__ void split_store(unsigned char* to, const float4& a, const float4& b) {
    uint4 hi, lo;
    split2(a.x, a.y, hi.x, lo.x);
    split2(a.z, a.w, hi.y, lo.y);
    split2(b.x, b.y, hi.z, lo.z);
    split2(b.z, b.w, hi.w, lo.w);
    *reinterpret_cast<uint4*>(to) = hi;
    *reinterpret_cast<uint4*>(to + PART) = lo;
}

constexpr float kLeastSize = 0x1p-3f, kMostSize = 65504.0f;

// The larger of `top` and the sizes of 8 values (passes over NaN).
__device__ __forceinline__ float larger(float top, const float4& a, const float4& b) {
    top = fmaxf(fmaxf(top, fabsf(a.x)), fabsf(a.y));
    top = fmaxf(fmaxf(top, fabsf(a.z)), fabsf(a.w));
    top = fmaxf(fmaxf(top, fabsf(b.x)), fabsf(b.y));
    return fmaxf(fmaxf(top, fabsf(b.z)), fabsf(b.w));
}
// What values of up to `top` in size are divided by before they are split: 1 where the largest keeps 22 bits in two fp16
// parts as it is, else the power of two that takes it to 2^14 or more (values down to 2^-17 of it keep 22 bits, smaller
// ones 2^-39 of it).  Not finite: 1.
__device__ __forceinline__ float divisor(float top) {
    const uint32_t b = __float_as_uint(top);
    if ((top >= kLeastSize && top < kMostSize) || b == 0u || b >= 0x7f800000u) return 1.0f;
    return __uint_as_float((max(b >> 23, 15u) - 14u) << 23);
}
__device__ __forceinline__ float power_inverse(float x) {  // of a power of two, 2^-126 to 2^113
    return __uint_as_float((254u << 23) - __float_as_uint(x));
}
__device__ __forceinline__ float warp_top(float top) {  // the largest of a warp's sizes
    return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
}
__device__ __forceinline__ void times(float4& a, float by) { a.x *= by, a.y *= by, a.z *= by, a.w *= by; }
// A warp's rows, each divided by a power of two of its own where the largest size of all asks for a look at each (a row
// that is huge, or garbage that nobody reads, leaves its neighbours as they are).  a[i], b[i]: 8 values, LANES neighbouring
// lanes to a row for each i (ONE: for all i together); put(i, divisor) then takes row i's.  False: nothing is divided.
template <int LANES, bool ONE, int N, typename Put>
__device__ __forceinline__ bool divide(float4 (&a)[N], float4 (&b)[N], Put&& put) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) top = larger(top, a[i], b[i]);
    if (divisor(warp_top(top)) == 1.0f) return false;
    float div = 1.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (i == 0 || !ONE) {
            float t = ONE ? top : larger(0.f, a[i], b[i]);
#pragma unroll
            for (int o = 1; o < LANES; o <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
            div = divisor(t);
            put(i, div);
        }
        times(a[i], power_inverse(div)), times(b[i], power_inverse(div));
    }
    return true;
}
__device__ __forceinline__ void loaders_meet() { asm volatile("bar.sync 1, %0;" ::"n"(kLoaders) : "memory"); }

template <typename T, int D, int NQ, bool PAGED, bool LONG>
__global__ void __launch_bounds__(Cfg<T, D, NQ, LONG>::THREADS, Cfg<T, D, NQ, LONG>::CTAS)
    rows_tc_kernel(const RowsParams p, int n_split) {
    using C = Cfg<T, D, NQ, LONG>;
    constexpr int ST = C::ST;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    unsigned char* sm = smem_raw + (base - raw);
    uint64_t* k_full = reinterpret_cast<uint64_t*>(sm + C::BARS);
    uint64_t *k_empty = k_full + ST, *v_full = k_empty + ST, *v_empty = v_full + ST;
    uint64_t *s_full = v_empty + ST, *p_full = s_full + NQ, *o_full = p_full + NQ, *q_full = o_full + NQ;
    uint64_t *s_read = q_full + NQ, *pair = s_read + NQ, *done = pair + 4 * NQ, *v_first = done + 1;
    uint64_t* again = v_first + 1;  // (fp32) the first tile of V, split once more
    uint32_t* slot = reinterpret_cast<uint32_t*>(sm + C::SLOT);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + C::SLOT + 4);
    const uint32_t* valid = reinterpret_cast<const uint32_t*>(sm + C::VALID);
    // (fp32) divisors, largest sizes, and the bytes of what is divided
    float *q_div = reinterpret_cast<float*>(sm + C::QS), *k_div = reinterpret_cast<float*>(sm + C::KS);
    float *v_div = reinterpret_cast<float*>(sm + C::VS), *tops = reinterpret_cast<float*>(sm + C::TOPS);
    uint64_t *q_odd = reinterpret_cast<uint64_t*>(sm + C::ODD), *v_kinds = q_odd + 1, *k_odd = q_odd + 2;
    auto place = [](int j) { return j == 0 ? C::WORDS : j % C::WORDS; };  // of tile j among the divisors

    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // (known to be the same in all lanes)
    const int split = blockIdx.x % n_split, tiles = gridDim.x / n_split;
    // a chunk's last tokens see the most keys: they start first
    const int tile = PAGED ? tiles - 1 - blockIdx.x / n_split : blockIdx.x / n_split;
    const int g = blockIdx.y, s = blockIdx.z;
    const int row0 = tile * NQ * kTile;

    pdl_wait_primary();
    RowsSeq sq;
    if (!rows_sequence<PAGED>(p, s, sq)) return;  // (uniform over the cluster)
    const int rows = sq.qn * p.group;
    if (row0 >= rows) return;

    if (warp == C::THREADS / 32 - 1) {
        tmem_alloc(slot, C::TMEM);
        if (lane == 0) {
            for (int i = 0; i < ST; ++i) {
                mbar_init(k_full + i, kLoaders + (C::F32 ? 0 : kLoaders / 32));
                mbar_init(v_full + i, kLoaders);
                mbar_init(k_empty + i, 1);
                mbar_init(v_empty + i, 1);
            }
            for (int i = 0; i < NQ; ++i) {
                mbar_init(s_full + i, 1);
                mbar_init(p_full + i, C::WPT);
                mbar_init(q_full + i, C::WPT * 32 + (C::FIRST ? kLoaders : 0));
                mbar_init(s_read + i, C::WPT);
                for (int k = 0; k < 4; ++k) mbar_init(pair + 4 * i + k, 2);
                mbar_init(o_full + i, 1);
            }
            mbar_init(done, 1);
            mbar_init(v_first, C::SOFT);
            if constexpr (C::F32) {
                mbar_init(again, kLoaders);
                for (int i = 0; i < C::WORDS + 3; ++i) q_odd[i] = 0;
                v_div[C::WORDS] = 1.0f;
            }
            fence_barrier_init();
            *abort_flag = 0;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *slot;
    // only now: a dependent's CTA on this SM could otherwise take the tensor memory and wait for this grid with it
    pdl_launch_dependents();

    // keys of this CTA: all that its last row sees, in tiles, shared among the splits
    const int last_tok = rows_token(p, min(rows, row0 + NQ * kTile) - 1);
    const int longest = PAGED ? sq.kvn - sq.qn + last_tok + 1 : sq.kvn;
    const int all_tiles = (longest + kTile - 1) / kTile;
    const int per = (all_tiles + n_split - 1) / n_split;
    const int j0 = split * per, n = max(0, min(all_tiles, j0 + per) - j0);

    // (fp32) Whether the first tile of V has to be split again, by the softmax warps' bytes (1: a size of 2^-3, 2: too large).
    auto v_first_odd = [&]() -> bool {
        static_assert(!C::F32 || C::SOFT == 256, "a byte of each softmax warp");
        const uint64_t f = *v_kinds, bytes = 0x0101010101010101ull;
        return (f & bytes) == 0 || (f & bytes * 2) != 0;
    };

    // Bounded wait; false (and the CTA gives up) once any wait has run out.
    auto wait_one = [&](uint64_t* bar, uint32_t parity, long long budget = kWaitBudgetCycles, int pause = 0) -> bool {
        if (mbar_try_wait(bar, parity)) return true;
        const long long t0 = clock64();
        while (!mbar_try_wait(bar, parity)) {
            if (pause) __nanosleep(pause);
            if (*abort_flag) return false;
            if (clock64() - t0 > budget) {
                *abort_flag = 1;
                atomicOr(p.err, NLLB_DEV_ERR_TIMEOUT);
                return false;
            }
        }
        return true;
    };
    // One arrival for a whole warp: 32 at one address are taken one after the other.
    auto warp_arrive = [&](uint64_t* bar) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
    };
    // The same for a whole warp, with one answer.
    auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
        return __all_sync(0xffffffffu, wait_one(bar, parity));
    };

    if (warp < NQ * C::WPT) {
        // ---- softmax: a thread, or two, to a query row
        const int t = warp / C::WPT, lq = warp & 3;                     // query tile, TMEM lane quarter
        const int half = C::WPT == 8 ? (warp % C::WPT) >> 2 : 0;        // of the row's scores
        if (PAGED && p.k_new && split == 0) {
            const int t0 = rows_token(p, row0 + p.group - 1);
            const int t1 = min(sq.qn, rows_token(p, row0 + NQ * kTile + p.group - 1));
            rows_append<T, D>(p, sq, s, g, t0, t1, tid, C::SOFT);
        }
        const int row = row0 + t * kTile + lq * 32 + lane;
        const bool there = row < rows;
        const bool any = row0 + t * kTile + lq * 32 < rows;  // the warp has a row
        const int tok = rows_token(p, row);
        const int lim = there ? (PAGED ? sq.kvn - sq.qn + tok + 1 : sq.kvn) : 0;
        const uint32_t lane_off = (uint32_t)(lq * 32) << 16;
        const uint32_t tS = tmem + lane_off + (uint32_t)t * 128, tO = tmem + lane_off + C::O_COL + (uint32_t)t * D;
        const uint32_t tT = tmem + lane_off + C::T_COL + (uint32_t)t * D;  // (TOTAL) the tiles before those in O
        // the weights of 32 keys: 16 columns (and fp32's low parts in the next 16)
        auto p_at = [&](int c) { return C::AHEAD ? tmem + lane_off + C::P_COL + t * 64 + 16 * c : tS + 32 * c; };
        // x of this thread's row and y of the other thread's, whichever way round: the step'th exchange of the pair
        auto other = [&](float x, int step, float& y) -> bool {
            float* at = reinterpret_cast<float*>(sm + C::MAXS) + ((step & 1) * NQ + t) * 256 + lq * 32 + lane;
            at[half * 128] = x;
            __syncwarp();
            if (lane == 0) mbar_arrive(pair + t * 4 + lq);
            const bool ok = wait(pair + t * 4 + lq, step & 1);
            y = at[(half ^ 1) * 128];
            return ok;
        };
        const float sl = p.scale_log2;
        // this tile's queries, 16 bytes (fp32: 32) at a time
        if (n > 0) {
            constexpr int CH = D / 8, N = C::WPT * 32, TAKE = kTile * CH / N < 8 ? kTile * CH / N : 8;
            const int lt = tid - t * N;
            int entry[C::FIRST ? TAKE : 1];  // (fp32) of the first tile's keys, asked for ahead of their use
            if constexpr (C::FIRST) {
#pragma unroll
                for (int i = 0; i < TAKE; ++i) {
                    const int key = j0 * kTile + (lt + i * N) / CH;
                    entry[i] = key < longest ? rows_entry<PAGED>(p, sq, s, key) : 0;
                }
            }
#pragma unroll
            for (int i0 = 0; i0 < kTile * CH / N; i0 += TAKE) {
                const T* src[TAKE];
                float4 a[C::F32 ? TAKE : 1], b[C::F32 ? TAKE : 1];
#pragma unroll
                for (int i = 0; i < TAKE; ++i) {
                    const int x = lt + (i0 + i) * N, r = row0 + t * kTile + x / CH, tk = rows_token(p, r);
                    src[i] = r < rows ? static_cast<const T*>(p.q) + (long long)(sq.q0 + tk) * p.q_row +
                                            (long long)(g * p.group + (r - tk * p.group)) * p.q_head + (x % CH) * 8
                                      : nullptr;
                    if constexpr (C::F32) {
                        a[i] = b[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (src[i]) {
                            a[i] = ld_coherent(reinterpret_cast<const float4*>(src[i]));
                            b[i] = ld_coherent(reinterpret_cast<const float4*>(src[i]) + 1);
                        }
                    }
                }
                if constexpr (C::F32) {
                    auto put = [&](int i, float div) {
                        if ((lt + i * N) % CH == 0) q_div[(lt + i * N) / CH] = div;
                    };
#pragma unroll
                    for (int i = 0; i < TAKE; ++i) put(i, 1.0f);
                    const bool odd = divide<CH, false>(a, b, put);
                    if (lane == 0) reinterpret_cast<uint8_t*>(q_odd)[warp] = odd;
                }
#pragma unroll
                for (int i = 0; i < TAKE; ++i) {
                    const int x = lt + (i0 + i) * N;
                    const uint32_t at = C::SQ + t * C::OPER + chunk_off(x / CH, x % CH);
                    if constexpr (C::F32) split_store<C::PART>(sm + at, a[i], b[i]);
                    else cp_async16(base + at, src[i] ? src[i] : static_cast<const T*>(p.q), src[i] != nullptr);
                }
            }
            if constexpr (C::FIRST) {
                static_assert(kTile * CH == TAKE * N && NQ == 1, "a tile in registers");
                const T *k[TAKE], *v[TAKE];
#pragma unroll
                for (int i = 0; i < TAKE; ++i) {
                    const int r = (lt + i * N) / CH, key = j0 * kTile + r;
                    if (!(key < longest && rows_at<T, PAGED>(p, sq, g, key, entry[i], k[i], v[i]))) k[i] = v[i] = nullptr;
                }
#pragma unroll
                for (int kv = 0; kv < 2; ++kv) {
                    float4 a[TAKE], b[TAKE];
#pragma unroll
                    for (int i = 0; i < TAKE; ++i) {
                        const int c = (lt + i * N) % CH;
                        const float4* src = reinterpret_cast<const float4*>(kv ? v[i] : k[i]);
                        a[i] = b[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (src) a[i] = ld_coherent(src + 2 * c), b[i] = ld_coherent(src + 2 * c + 1);
                    }
                    if (kv == 0) {
                        auto put = [&](int i, float div) {
                            if ((lt + i * N) % CH == 0) k_div[C::WORDS * kTile + (lt + i * N) / CH] = div;
                        };
#pragma unroll
                        for (int i = 0; i < TAKE; ++i) put(i, 1.0f);
                        const bool odd = divide<CH, false>(a, b, put);
                        if (lane == 0) reinterpret_cast<uint8_t*>(k_odd + C::WORDS)[warp] = odd;
                    }
                    float top = 0.f;
#pragma unroll
                    for (int i = 0; i < TAKE; ++i) {
                        const int x = lt + i * N;
                        split_store<C::PART>(sm + (kv ? C::SV : C::SK) + chunk_off(x / CH, x % CH), a[i], b[i]);
                        if (kv) top = larger(top, a[i], b[i]);
                    }
                    if (kv) {  // (the fetching warps see whether the tile has to be split again)
                        top = warp_top(top);
                        if (lane == 0) {
                            reinterpret_cast<uint8_t*>(v_kinds)[warp] = (top >= kLeastSize ? 1 : 0) | (top >= kMostSize ? 2 : 0);
                            tops[warp] = top;
                        }
                    }
                    mbar_arrive(kv ? v_first : q_full + t);
                }
            } else if constexpr (C::F32) {
                mbar_arrive(q_full + t);
            } else {
                cp_arrive(q_full + t);
            }
        }
        float m = -INFINITY, l = 0.f;  // m: the maximum in use, in units of the scaled score
        bool ok = true;
        for (int j = 0; j < n && ok; ++j) {
            if (!(ok = wait(s_full + t, j & 1))) break;
            if (!C::AHEAD && j > 0 && !(ok = wait(o_full + t, (j - 1) & 1))) break;  // over: its product came first
            tc_fence_after();
            if (any) {
                const uint32_t* vw = valid + (j % C::WORDS) * 4;
                const int left = lim - (j0 + j) * kTile;  // visible keys of this tile, before the valid bits
                constexpr int NC = C::COLS / 32;
                uint32_t bits[NC], all = 0xffffffffu;
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const int x = min(max(left - 32 * (half * NC + c), 0), 32);
                    bits[c] = vw[half * NC + c] & (x == 32 ? 0xffffffffu : (1u << x) - 1u);
                    all &= bits[c];
                }
                // (one copy of the row's work for whole tiles, one for those with hidden keys)
                const bool whole = __all_sync(0xffffffffu, all == 0xffffffffu);
                const uint32_t tR = tS + half * C::COLS;
                float v[C::COLS];  // (a row's scores stay in registers between their maximum and the weights)
                auto hide = [&](float* x, uint32_t w) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) x[i] = (w >> i) & 1u ? x[i] : -INFINITY;
                };
                float y[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                tmem_ld<C::COLS>(tR, v);
                if constexpr (C::F32) {
                    if ((*q_odd | k_odd[place(j)]) != 0) {
                        const float qd = q_div[lq * 32 + lane], *kd = k_div + place(j) * kTile + half * C::COLS;
#pragma unroll
                        for (int i = 0; i < C::COLS; ++i) v[i] *= fminf(qd * kd[i], FLT_MAX);  // (no 0 times infinity)
                    }
                }
                if (!whole) {
#pragma unroll
                    for (int c = 0; c < NC; ++c) hide(v + 32 * c, bits[c]);
                }
#pragma unroll
                for (int i = 0; i < C::COLS; i += 2) y[(i >> 1) & 3] = max_nan(y[(i >> 1) & 3], v[i], v[i + 1]);
                if constexpr (C::AHEAD) {
                    tc_fence_before();
                    warp_arrive(s_read + t);
                }
                float mx = max_nan(max_nan(y[0], y[1]), max_nan(y[2], y[3]));
                if constexpr (C::WPT == 8) {
                    float his;
                    if (!(ok = other(mx, j, his))) break;
                    mx = max_nan(mx, his);
                }
                if (C::AHEAD && j > 0 && !(ok = wait(o_full + t, (j - 1) & 1))) break;  // P and O are free
                if (C::AHEAD) tc_fence_after();
                const float mn = mx * sl;
                const bool grown = !(mn <= m + kGrow);  // a NaN makes the whole row NaN
                if constexpr (LONG) {
                    const bool full = j % kTilesTogether == 0;  // the sums in O move on to the total
                    if (j > 0 && (full || __any_sync(0xffffffffu, grown))) {
                        const float to = grown ? max_nan(m, mn) : m;
                        const float corr = m == to ? 1.f : m == -INFINITY ? 0.f : ex2_approx(m - to);
                        m = to;
                        l *= corr;
#pragma unroll
                        for (int c = half * (D / 2); c < (C::WPT == 8 ? (half + 1) * (D / 2) : D); c += 8) {
                            uint32_t o[8], x[8];
                            tmem_ld8(tO + c, o);
                            if (j > kTilesTogether) tmem_ld8(tT + c, x);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const float y = __uint_as_float(o[i]), z = j > kTilesTogether ? __uint_as_float(x[i]) : 0.f;
                                o[i] = __float_as_uint(y * corr);
                                x[i] = __float_as_uint((full ? y + z : z) * corr);
                            }
                            if (!full) tmem_st8(tO + c, o);
                            if (full || j > kTilesTogether) tmem_st8(tT + c, x);
                        }
                    } else if (j == 0 && grown) {
                        m = max_nan(m, mn);
                    }
                } else if constexpr (C::TOTAL) {
                    const float to = grown ? max_nan(m, mn) : m;
                    const float corr = m == to ? 1.f : m == -INFINITY ? 0.f : ex2_approx(m - to);
                    m = to;
                    l *= corr;
                    if (j > 0) {
                        const float vd = v_div[place(j - 1)];
#pragma unroll
                        for (int c = half * (D / 2); c < (C::WPT == 8 ? (half + 1) * (D / 2) : D); c += 8) {
                            uint32_t o[8], x[8];
                            tmem_ld8(tO + c, o);
                            if (j > 1) tmem_ld8(tT + c, x);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const float y = fmaf(__uint_as_float(o[i]), vd, j > 1 ? __uint_as_float(x[i]) : 0.f);
                                o[i] = __float_as_uint(y * corr);
                            }
                            tmem_st8(tT + c, o);
                        }
                    }
                } else if (__any_sync(0xffffffffu, grown)) {
                    // (a row's own affair: what its neighbours hold changes none of its roundings)
                    const float to = grown ? max_nan(m, mn) : m;
                    const float corr = m == to ? 1.f : m == -INFINITY ? 0.f : ex2_approx(m - to);
                    m = to;
                    l *= corr;
                    if (j > 0) {
#pragma unroll
                        for (int c = half * (D / 2); c < (C::WPT == 8 ? (half + 1) * (D / 2) : D); c += 16) {
                            uint32_t o[16];
                            tmem_ld16(tO + c, o);
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
                            tmem_st16(tO + c, o);
                        }
                    }
                }
                const float off = (m == -INFINITY ? 0.f : m) - kWeightExp;
                float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    float* x = v + 32 * c;
                    uint32_t hi[16], lo[C::F32 ? 16 : 1];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float2 y = fma2(make_float2(x[2 * i], x[2 * i + 1]), make_float2(sl, sl), make_float2(-off, -off));
                        const float2 e = make_float2(ex2_approx(y.x), ex2_approx(y.y));
                        sum[i & 1] = add2(sum[i & 1], e);
                        if constexpr (C::F32) split2(e.x, e.y, hi[i], lo[i]);
                        else hi[i] = pack2<T>(e.x, e.y);
                    }
                    tmem_st16(p_at(half * NC + c), hi);
                    if constexpr (C::F32) tmem_st16(p_at(half * NC + c) + 16, lo);
                }
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                tmem_wait_st();
            } else if (C::AHEAD) {
                warp_arrive(s_read + t);
                // not a tile ahead of the other warps, whose arrivals would be taken for this one's
                if (j > 0 && !(ok = wait(o_full + t, (j - 1) & 1))) break;
            }
            tc_fence_before();
            warp_arrive(p_full + t);
        }
        if (ok && n > 0) ok = wait(o_full + t, (n - 1) & 1);
        tc_fence_after();
        if constexpr (C::WPT == 8) {  // the row's whole sum
            float his = 0.f;
            if (ok && any && n > 0) ok = other(l, n, his);
            l = half ? his + l : l + his;
        }
        auto last_output = [&](int c, float* o) {
            tmem_ld32(tO + c, o);
            if constexpr (C::TOTAL) {
                const float vd = C::F32 ? v_div[place(n - 1)] : 1.0f;
                constexpr int before = LONG ? kTilesTogether : 1;  // tiles that the total may be behind O
                if (vd != 1.0f) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] *= vd;
                }
                if (n > before) {
                    float x[32];
                    tmem_ld32(tT + c, x);
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] += x[i];
                }
            }
        };
        const int d0 = half * (D / 2), d1 = C::WPT == 8 ? d0 + D / 2 : D;  // this thread's part of the output
        if (n_split == 1) {
            if (ok && any) {
                const float inv = 1.0f / l;
                T* dst = static_cast<T*>(p.out) + (long long)(sq.q0 + tok) * p.o_row +
                         (long long)(g * p.group + (row - tok * p.group)) * p.o_head;
#pragma unroll
                for (int c = d0; c < d1; c += 32) {
                    float o[32];
                    if (n > 0) last_output(c, o);
                    constexpr int VEC = 16 / (int)sizeof(T);
                    if (there) {
#pragma unroll
                        for (int i = 0; i < 32; i += VEC) {
                            float x[VEC];
#pragma unroll
                            for (int e = 0; e < VEC; ++e) x[e] = l == 0.f ? 0.f : o[i + e] * inv;  // no visible key: zeros
                            *reinterpret_cast<uint4*>(dst + c + i) = rows_pack<T>(x);
                        }
                    }
                }
            }
        } else if constexpr (NQ == 1) {
            // the state of this split's rows goes over the operands (every product has read them)
            if (any) {
                float* st = reinterpret_cast<float*>(sm) + (lq * 32 + lane) * C::LD;
#pragma unroll
                for (int c = d0; c < d1; c += 32) {
                    float o[32];
                    if (n > 0) last_output(c, o);
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *reinterpret_cast<float4*>(st + c + i) =
                            l == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                }
                if (half == 0) *reinterpret_cast<float4*>(st + D) = make_float4(l == 0.f ? -INFINITY : m, ok ? l : -1.f, 0.f, 0.f);
            }
        }
    } else if (warp < (C::SOFT + kLoaders) / 32) {
        // ---- fetch
        // Two lanes to a row, which take its 16-byte chunks in turns (a row's 32-byte sectors are then used whole):
        // the row's address stays in a register, and a copy costs little beside it.
        const int lt = tid - C::SOFT, odd = lt & 1;
        constexpr int CH = D / 8, RP = (2 * kTile + kLoaders - 1) / kLoaders;  // chunks of 8 elements; rows of a lane
        uint16_t* seen16 = reinterpret_cast<uint16_t*>(sm + C::VALID);
        int entry[RP];
        auto look_up = [&](int j) {
#pragma unroll
            for (int i = 0; i < RP; ++i) {
                const int r = (lt >> 1) + i * (kLoaders / 2), key = (j0 + j) * kTile + r;
                entry[i] = r < kTile && key < longest ? rows_entry<PAGED>(p, sq, s, key) : 0;
            }
        };
        bool ok = true;
        if (n > 0) look_up(0);
        for (int j = 0; j < n && (ok || C::F32); ++j) {  // (fp32: the warps give up together)
            const int st = j % ST;
            const T *k[RP], *v[RP];
            // (visible keys of a tile: kept until its weights are formed, at least one tile after V of this slot)
#pragma unroll
            for (int i = 0; i < RP; ++i) {
                const int r = (lt >> 1) + i * (kLoaders / 2), key = (j0 + j) * kTile + r;
                const bool seen =
                    r < kTile && key < longest && rows_at<T, PAGED>(p, sq, g, key, entry[i], k[i], v[i]);
                if (!seen) k[i] = v[i] = nullptr;
                uint32_t w = __ballot_sync(0xffffffffu, seen) & 0x55555555u;  // a bit for two lanes
                w = (w | w >> 1) & 0x33333333u;
                w = (w | w >> 2) & 0x0f0f0f0fu;
                w = (w | w >> 4) & 0x00ff00ffu;
                w = (w | w >> 8) & 0x0000ffffu;
                if (lane == 0 && r < kTile) seen16[(j % C::WORDS) * 8 + (r >> 4)] = (uint16_t)w;
            }
            if (j + 1 < n) look_up(j + 1);
            if (C::FIRST && j == 0) mbar_arrive(q_full);  // fetched by the softmax threads
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                uint64_t *full = (kv ? v_full : k_full) + st, *empty = (kv ? v_empty : k_empty) + st;
                const uint32_t dst = (kv ? C::SV : C::SK) + st * C::OPER;
                if constexpr (!C::F32) {
                    if (j >= ST && !(ok = wait(empty, ((j / ST) - 1) & 1))) break;
                    // (an ordinary arrival, for the words of visible keys: that of the copies vouches for the copies alone)
                    if (kv == 0) warp_arrive(full);
#pragma unroll
                    for (int i = 0; i < RP; ++i) {
                        const int r = (lt >> 1) + i * (kLoaders / 2);
                        const T* src = kv ? v[i] : k[i];
                        const uint32_t to = base + dst + r * 128;
                        if (r < kTile) {
#pragma unroll
                            for (int c = 0; c < CH; c += 2)
                                cp_async16(to + (c >> 3) * kBlock + ((((c & 7) + odd) ^ (r & 7)) << 4),
                                           src ? src + (c + odd) * 8 : static_cast<const T*>(p.q), src != nullptr);
                        }
                    }
                    cp_arrive(full);
                } else {
                    // K: a row by itself.  V: the tile alike, since its sums are: split as it is (the first tile by the
                    // softmax threads) and, where the tile's largest size asks for a divisor, read and split once more.
                    if (j == 0 && kv == 0) continue;
                    float div = 1.0f;
                    if (j == 0) {
                        if (ok) ok = __all_sync(0xffffffffu, wait_one(v_first, 0, kWaitBudgetCycles, 200));
                        if (!ok || !v_first_odd()) continue;
                        float top = 0.f;
                        for (int w = 0; w < 8; ++w) top = fmaxf(top, tops[w]);
                        div = divisor(top);
                    }
                    for (int pass = j == 0; pass < 2; ++pass) {
                        const float by = power_inverse(div);
                        float top = 0.f;
                        bool odd = false;
#pragma unroll
                        for (int i = 0; i < RP; ++i) {
                            const int r = (lt >> 1) + i * (kLoaders / 2);
                            const float4* src = reinterpret_cast<const float4*>(kv ? v[i] : k[i]);
                            float4 a[CH / 2], b[CH / 2];
#pragma unroll
                            for (int c = 0; c < CH / 2; ++c) {
                                a[c] = b[c] = make_float4(0.f, 0.f, 0.f, 0.f);
                                if (src) {
                                    a[c] = ld_coherent(src + 2 * (2 * c + (lt & 1)));
                                    b[c] = ld_coherent(src + 2 * (2 * c + (lt & 1)) + 1);
                                }
                            }
                            if (kv == 0) {
                                auto put = [&](int, float d) {
                                    if ((lt & 1) == 0 && r < kTile) k_div[place(j) * kTile + r] = d;
                                };
                                put(0, 1.0f);
                                odd = divide<2, true>(a, b, put) || odd;
                            } else if (pass == 1) {
#pragma unroll
                                for (int c = 0; c < CH / 2; ++c) times(a[c], by), times(b[c], by);
                            }
                            if (i == 0 && pass == 0 && ok) ok = wait(empty, (j - 1) & 1);
                            if (ok && r < kTile) {
#pragma unroll
                                for (int c = 0; c < CH / 2; ++c) {
                                    if (kv) top = larger(top, a[c], b[c]);
                                    split_store<C::PART>(sm + dst + chunk_off(r, 2 * c + (lt & 1)), a[c], b[c]);
                                }
                            }
                        }
                        if (kv == 0 && lane == 0) reinterpret_cast<uint8_t*>(k_odd + place(j))[warp - C::SOFT / 32] = odd;
                        if (kv == 0 || pass == 1) break;
                        // A warp that gave up says so, and all leave together: nobody waits here for one that left.  (Two
                        // sets of words: the next tile's are not written where a slower warp still reads this one's.)
                        float* all = tops + 8 + (j & 1) * (kLoaders / 32);
                        top = warp_top(top);
                        if (lane == 0) all[warp - C::SOFT / 32] = ok ? top : -1.0f;
                        loaders_meet();
#pragma unroll
                        for (int w = 0; w < kLoaders / 32; ++w) {
                            ok = ok && all[w] >= 0.f;
                            top = fmaxf(top, all[w]);
                        }
                        div = divisor(top);
                        if (!ok || div == 1.0f) break;
                    }
                    if (kv && lt == 0) v_div[place(j)] = div;
                    if (ok) mbar_arrive(j == 0 ? again : full);
                }
            }
            if (!ok && (j > 0 || !C::F32)) break;  // (fp32: after the warps have met)
        }
        if constexpr (!C::F32) cp_wait_all();
    } else {
        // ---- products.  The whole warp walks the loop and one lane issues, so that descriptors and addresses are the
        // same in all lanes to the compiler and stay in uniform registers: issued from a branch of one lane, each
        // product cost about 100 cycles of moves, and the issuing thread was the kernel's bound.
        constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;
        constexpr uint32_t id_s = umma_idesc_f16(128, 128) | fmt, id_o = umma_idesc_f16(128, D) | fmt | (1u << 16);
        // V's descriptor: the leading byte offset is the distance between 64-element blocks of a row
        constexpr uint64_t lead = ((uint64_t)(kBlock >> 4) << 16) ^ ((uint64_t)1 << 16);
        const uint64_t q0 = umma_desc_k_sw128(base + C::SQ), k0 = umma_desc_k_sw128(base + C::SK);
        const uint64_t v0 = umma_desc_k_sw128(base + C::SV) ^ lead;
        const bool leader = elect_one();
        auto scores = [&](int t, int st) {
            const uint64_t q = q0 + (uint32_t)t * (C::OPER >> 4), k = k0 + (uint32_t)st * (C::OPER >> 4);
            if (leader) {
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks) {
                    const uint32_t o = ((uint32_t)(ks >> 2) * kBlock + (ks & 3) * 32) >> 4;
                    if constexpr (C::F32) {  // (the small products first, while little is cut off their sum)
                        tc_mma_f16(tmem + t * 128, q + o, k + (C::PART >> 4) + o, id_s, ks > 0);
                        tc_mma_f16(tmem + t * 128, q + (C::PART >> 4) + o, k + o, id_s, 1);
                    } else {
                        tc_mma_f16(tmem + t * 128, q + o, k + o, id_s, ks > 0);
                    }
                }
#pragma unroll
                for (int ks = 0; C::F32 && ks < D / 16; ++ks) {
                    const uint32_t o = ((uint32_t)(ks >> 2) * kBlock + (ks & 3) * 32) >> 4;
                    tc_mma_f16(tmem + t * 128, q + o, k + o, id_s, 1);
                }
                tc_commit(s_full + t);
                if (t == NQ - 1) tc_commit(k_empty + st);
            }
            __syncwarp();
        };
        auto output = [&](int t, int st, bool accumulate) {
            const uint64_t v = v0 + (uint32_t)st * (C::OPER >> 4);
            const uint32_t o = tmem + C::O_COL + t * D;
            if (leader) {
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) {
                    const uint32_t a = C::AHEAD ? tmem + C::P_COL + t * 64 + ks * 8
                                                : tmem + t * 128 + (ks >> 1) * 32 + (ks & 1) * 8;
                    const uint64_t b = v + ks * (2048 >> 4);
                    if constexpr (C::F32) {
                        tc_mma_f16_ta(o, a, b + (C::PART >> 4), id_o, ks > 0);
                        tc_mma_f16_ta(o, a + 16, b, id_o, 1);
                    } else {
                        tc_mma_f16_ta(o, a, b, id_o, accumulate || ks > 0);
                    }
                }
#pragma unroll
                for (int ks = 0; C::F32 && ks < 8; ++ks)
                    tc_mma_f16_ta(o, tmem + t * 128 + (ks >> 1) * 32 + (ks & 1) * 8, v + ks * (2048 >> 4), id_o, 1);
                tc_commit(o_full + t);
                if (t == NQ - 1) tc_commit(v_empty + st);
            }
            __syncwarp();
        };
        bool ok = true;
        if (p.expire) ok = __all_sync(0xffffffffu, wait_one(done, 0, kTestWaitBudgetCycles));  // nothing arrives there
        if (ok && n > 0 && (C::FIRST || (ok = wait(k_full, 0)))) {
            for (int t = 0; t < NQ && ok; ++t) {
                if (!(ok = wait(q_full + t, 0))) break;
                fence_async_smem();  // what the copies wrote
                tc_fence_after();
                scores(t, 0);
            }
        }
        for (int j = 0; j < n && ok; ++j) {
            const int st = j % ST, nx = (j + 1) % ST;
            // scores of the next key tile: K has come and (AHEAD) the row's last ones are read
            auto next = [&](int t) -> bool {
                if (j + 1 >= n) return true;
                if (t == 0 && !wait(k_full + nx, ((j + 1) / ST - C::FIRST) & 1)) return false;
                if (t == 0) fence_async_smem();  // what the copies wrote
                if (C::AHEAD && !wait(s_read + t, j & 1)) return false;
                tc_fence_after();
                scores(t, nx);
                return true;
            };
            if constexpr (C::AHEAD) {
                for (int t = 0; t < NQ && ok; ++t) ok = next(t);
                if (!ok) break;
            }
            for (int t = 0; t < NQ && ok; ++t) {
                if (t == 0) {
                    // (a slot's k_full and v_full do not count the first tile where the softmax threads fetched it)
                    if (!(ok = C::FIRST && j == 0 ? wait(v_first, 0) : wait(v_full + st, (j / ST - C::FIRST) & 1))) break;
                    if (C::FIRST && j == 0 && v_first_odd() && !(ok = wait(again, 0))) break;
                    fence_async_smem();
                }
                if (!(ok = wait(p_full + t, j & 1))) break;
                tc_fence_after();
                output(t, st, LONG ? j % kTilesTogether != 0 : j > 0 && !C::TOTAL);
                if constexpr (!C::AHEAD) ok = next(t);  // P lies over S
            }
        }
        // whatever was issued is over before tensor memory is given back
        if (leader) {
            tc_commit(done);
            (void)mbar_wait_bounded(done, 0);
        }
        __syncwarp();
    }

    tc_fence_before();
    __syncthreads();
    if (warp == C::THREADS / 32 - 1) {
        tc_fence_after();
        tmem_dealloc(tmem, C::TMEM);
    }
    if constexpr (NQ == 1) {
        if (n_split > 1) {
            // join the splits, rank by rank: rank z finishes the 16-byte pieces z, z + n_split, ...
            cluster_sync_all();
            constexpr int VEC = 16 / (int)sizeof(T), PIECES = D / VEC;
            const float* st = reinterpret_cast<const float*>(sm);
            const int mine = min(kTile, rows - row0);
            for (int i = split + n_split * tid; i < mine * PIECES; i += n_split * C::THREADS) {
                const int r = i / PIECES, c = i % PIECES, row = row0 + r;
                float mx = -INFINITY;
                bool good = true;
                for (int z = 0; z < n_split; ++z) mx = fmaxf(mx, ld_cluster_f32(map_rank(st + r * C::LD + D, z)));
                const float off = mx == -INFINITY ? 0.f : mx;
                float x[VEC], sum = 0.f;
#pragma unroll
                for (int e = 0; e < VEC; ++e) x[e] = 0.f;
                for (int z = 0; z < n_split; ++z) {
                    const float w = ex2_approx(ld_cluster_f32(map_rank(st + r * C::LD + D, z)) - off);
                    const float lz = ld_cluster_f32(map_rank(st + r * C::LD + D + 1, z));
                    good = good && !(lz < 0.f);  // a split that gave up says so
                    sum = fmaf(w, lz, sum);
#pragma unroll
                    for (int e = 0; e < VEC; e += 4) {
                        const float4 f = ld_cluster_f4(map_rank(st + r * C::LD + c * VEC + e, z));
                        x[e] = fmaf(w, f.x, x[e]), x[e + 1] = fmaf(w, f.y, x[e + 1]);
                        x[e + 2] = fmaf(w, f.z, x[e + 2]), x[e + 3] = fmaf(w, f.w, x[e + 3]);
                    }
                }
                const float inv = 1.f / sum;
#pragma unroll
                for (int e = 0; e < VEC; ++e) x[e] = sum == 0.f ? 0.f : x[e] * inv;
                T* dst = static_cast<T*>(p.out) + (long long)(sq.q0 + row / p.group) * p.o_row +
                         (long long)(g * p.group + row % p.group) * p.o_head;
                if (good) *reinterpret_cast<uint4*>(dst + c * VEC) = rows_pack<T>(x);
            }
            cluster_sync_all();  // no CTA leaves while another reads its state
        }
    }
}

template <typename T, int D, int NQ, bool PAGED, bool LONG>
cudaError_t launch_tc(const RowsParams& p, int n_split, cudaStream_t st) {
    using C = Cfg<T, D, NQ, LONG>;
    const long long tiles = ((long long)p.max_q * p.group + NQ * kTile - 1) / (NQ * kTile);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * n_split), (unsigned)p.kv_heads, (unsigned)p.n_seq);
    cfg.blockDim = dim3(C::THREADS, 1, 1);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = kPdlLaunch;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)n_split;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = n_split > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, rows_tc_kernel<T, D, NQ, PAGED, LONG>, p, n_split);
}

template <typename T, int D, bool PAGED>
cudaError_t launch_by_tiles(const RowsParams& p, int num_sms, cudaStream_t st) {
    const long long rows = (long long)p.max_q * p.group, heads = (long long)p.kv_heads * p.n_seq;
    const bool is_long = sizeof(T) == 2 && p.max_kv > kLongKeys;
    if constexpr (sizeof(T) == 2) {
        // two query tiles per CTA where they still give every SM one
        if (rows > kTile && (rows + 2 * kTile - 1) / (2 * kTile) * heads >= num_sms) {
            if (!is_long) return launch_tc<T, D, 2, PAGED, false>(p, 1, st);
            // (two tiles of heads of 128 fill the tensor memory)
            if constexpr (D == 64) return launch_tc<T, D, 2, PAGED, true>(p, 1, st);
        }
    }
    const long long units = (rows + kTile - 1) / kTile * heads;
    // Splits, while they leave two CTAs or fewer per SM: two from 257 keys on (one sequence of 16 heads, 21 fp32 rows
    // over 500 keys: 12.0 us instead of 17.4), more where each keeps four key tiles (128 rows over 1500 keys: 20 us
    // with four, 36 with eight), one cluster at most.
    int n_split = 1;
    while (n_split < 8 && units * n_split * 2 <= 2LL * num_sms && p.max_kv > (n_split == 1 ? 256 : 512 * n_split))
        n_split *= 2;
    if constexpr (sizeof(T) == 2) {
        if (is_long) return launch_tc<T, D, 1, PAGED, true>(p, n_split, st);
    }
    return launch_tc<T, D, 1, PAGED, false>(p, n_split, st);
}

template <typename T>
cudaError_t launch_by_dim(const RowsParams& p, int head_dim, bool paged, int num_sms, cudaStream_t st) {
    if (head_dim == 64)
        return paged ? launch_by_tiles<T, 64, true>(p, num_sms, st) : launch_by_tiles<T, 64, false>(p, num_sms, st);
    return paged ? launch_by_tiles<T, 128, true>(p, num_sms, st) : launch_by_tiles<T, 128, false>(p, num_sms, st);
}

template <typename T, int D, int NQ, bool LONG = false>
cudaError_t configure_one() {
    cudaError_t e = cudaFuncSetAttribute(rows_tc_kernel<T, D, NQ, true, LONG>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg<T, D, NQ, LONG>::SMEM);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(rows_tc_kernel<T, D, NQ, false, LONG>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (int)Cfg<T, D, NQ, LONG>::SMEM);
    return e;
}

}  // namespace

cudaError_t configure_rows_tc() {
    cudaError_t e = configure_one<float, 64, 1>();
    if (e == cudaSuccess) e = configure_one<float, 128, 1>();
    if (e == cudaSuccess) e = configure_one<__half, 64, 1>();
    if (e == cudaSuccess) e = configure_one<__half, 64, 2>();
    if (e == cudaSuccess) e = configure_one<__half, 64, 1, true>();
    if (e == cudaSuccess) e = configure_one<__half, 64, 2, true>();
    if (e == cudaSuccess) e = configure_one<__half, 128, 1>();
    if (e == cudaSuccess) e = configure_one<__half, 128, 2>();
    if (e == cudaSuccess) e = configure_one<__half, 128, 1, true>();
    if (e == cudaSuccess) e = configure_one<__nv_bfloat16, 64, 1>();
    if (e == cudaSuccess) e = configure_one<__nv_bfloat16, 64, 2>();
    if (e == cudaSuccess) e = configure_one<__nv_bfloat16, 64, 1, true>();
    if (e == cudaSuccess) e = configure_one<__nv_bfloat16, 64, 2, true>();
    if (e == cudaSuccess) e = configure_one<__nv_bfloat16, 128, 1>();
    if (e == cudaSuccess) e = configure_one<__nv_bfloat16, 128, 2>();
    if (e == cudaSuccess) e = configure_one<__nv_bfloat16, 128, 1, true>();
    return e;
}

cudaError_t launch_rows_tc(const RowsParams& p, RowType type, int head_dim, bool paged, int num_sms, cudaStream_t st) {
    switch (type) {
        case RowType::f32: return launch_by_dim<float>(p, head_dim, paged, num_sms, st);
        case RowType::f16: return launch_by_dim<__half>(p, head_dim, paged, num_sms, st);
        default: return launch_by_dim<__nv_bfloat16>(p, head_dim, paged, num_sms, st);
    }
}

}  // namespace nllb
