// rows_tc.cu -- attention of many query rows over many keys on the 5th
// generation tensor cores (sm_100a).
//
//   S = Q K^T,  P = 2^(scale log2(e) S - m),  O += P V,  out = O / sum P
//
// over tiles of 128 keys, with m the running maximum of a row, held back: the
// row's sums are only rescaled when a maximum has grown by more than 2^8, so
// the accumulator in tensor memory is rarely touched between products.
//
// Roles of a CTA's warps: 4 per query tile for the softmax (a thread owns a
// row = a TMEM lane), 3 that fetch, 1 that issues the products.  Key rows are
// fetched row by row (cp.async of 16 bytes, or loads and a split for fp32):
// each row's address is worked out once by one thread, so pages of any size,
// strides of any order and masks need no copy, and a hidden row becomes zeros
// without being read.  K lies K-major and V as it comes (an MN-major operand),
// both in the 128-byte swizzle; P goes back over S in tensor memory, 32 keys
// in the columns of the same 32 scores, and is the A operand from there.
// With two query tiles per CTA the tensor cores work on one while the other's
// softmax runs, and a key tile is fetched once for 256 rows; with one tile two
// CTAs share an SM to the same end.
//
// Types: 16-bit inputs are the operands as they come, the weights are rounded
// to the type (half a step each, unbiased; the sum that divides them stays
// fp32).  fp32 inputs and weights are split into two fp16 parts, hi + lo, and
// a product is taken as hi hi' + hi lo' + lo hi' (22 bits).  Weights are held
// times 2^7, so fp16 keeps them normal down to 2^-21 of the largest while
// 2^7 * 2^8 stays in its range.
#include <algorithm>
#include <type_traits>

#include "rows.cuh"

namespace nllb {
namespace {

constexpr int kTile = 128;              // query rows of a tile, keys of a tile
constexpr int kLoaders = 96;            // fetching threads: 8 or 12 warps in all, so registers divide evenly
constexpr float kGrow = 8.0f;           // a maximum may lag by 2^8
constexpr float kWeightExp = 7.0f;      // weights are held times 2^7
constexpr uint32_t kBlock = 128 * 128;  // bytes of [128 rows][64 16-bit elements]

template <typename T, int D, int NQ>
struct Cfg {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int PARTS = F32 ? 2 : 1;
    static constexpr int KB = D / 64;                 // 64-element blocks of a row
    static constexpr uint32_t PART = kBlock * KB;     // one part of a [128][D] operand
    static constexpr uint32_t OPER = PART * PARTS;
    // key tiles in flight: what leaves room for two CTAs per SM with one query tile, or fills the SM with two
    static constexpr int ST = F32 ? 1 : (NQ == 2 ? (D == 64 ? 4 : 2) : (D == 64 ? 2 : 1));
    // Fetch groups (K or V of a tile) in flight per thread beside the one being issued.  A group is handed over when
    // group + LAG has been issued, which waits for the buffer of group + LAG - 2 ST: for K of tile j + 1 that may be
    // K of tile j, whose products are done, but not V of tile j, which the second query tile still needs.
    static constexpr int LAG = ST == 4 ? 3 : ST;
    static constexpr uint32_t SQ = 0, SK = NQ * OPER, SV = SK + ST * OPER, SAUX = SV + ST * OPER;
    static constexpr uint32_t PTRS = SAUX, VALID = PTRS + 4 * 128 * 8, BARS = VALID + 2 * ST * 16;
    static constexpr int N_BARS = 4 * ST + 3 * NQ + 1;
    static constexpr uint32_t SLOT = BARS + N_BARS * 8, BYTES = SLOT + 16;
    static constexpr uint32_t SMEM = BYTES + 1024;  // + alignment slack
    static constexpr int THREADS = NQ * 128 + kLoaders + 32;
    static constexpr uint32_t TMEM = NQ == 2 ? 512 : 256;  // S: 128 columns per tile, O: D per tile
    static constexpr int CTAS = NQ == 2 || (F32 && D == 128) ? 1 : 2;
    static constexpr int LD = D + 4;  // fp32 row of a split's state: D sums, then m, l
    static_assert(NQ * 128 + NQ * D <= (int)TMEM, "tensor memory");
    static_assert(128 * LD * 4 <= (int)SAUX || NQ == 2, "a split's state fits over the operands");
};

// byte offset of 16-byte chunk c of row r in an operand part
__device__ __forceinline__ uint32_t chunk_off(int r, int c) {
    return (uint32_t)((c >> 3) * (int)kBlock + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
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

// 16 columns of this thread's lane (warp-wide).
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float ex2_approx(float x) {  // 2^x, -inf -> +0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
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

template <typename T, int D, int NQ, bool PAGED>
__global__ void __launch_bounds__(Cfg<T, D, NQ>::THREADS, Cfg<T, D, NQ>::CTAS)
    rows_tc_kernel(const RowsParams p, int n_split) {
    using C = Cfg<T, D, NQ>;
    constexpr int ST = C::ST;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    unsigned char* sm = smem_raw + (base - raw);
    uint64_t* k_full = reinterpret_cast<uint64_t*>(sm + C::BARS);
    uint64_t *k_empty = k_full + ST, *v_full = k_empty + ST, *v_empty = v_full + ST;
    uint64_t *s_full = v_empty + ST, *p_full = s_full + NQ, *o_full = p_full + NQ, *done = o_full + NQ;
    uint32_t* slot = reinterpret_cast<uint32_t*>(sm + C::SLOT);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + C::SLOT + 4);
    const uint32_t* valid = reinterpret_cast<const uint32_t*>(sm + C::VALID);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
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
                mbar_init(k_full + i, kLoaders);
                mbar_init(v_full + i, kLoaders);
                mbar_init(k_empty + i, 1);
                mbar_init(v_empty + i, 1);
            }
            for (int i = 0; i < NQ; ++i) {
                mbar_init(s_full + i, 1);
                mbar_init(p_full + i, kTile);
                mbar_init(o_full + i, 1);
            }
            mbar_init(done, 1);
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
    const int last_tok = (min(rows, row0 + NQ * kTile) - 1) / p.group;
    const int longest = PAGED ? sq.kvn - sq.qn + last_tok + 1 : sq.kvn;
    const int all_tiles = (longest + kTile - 1) / kTile;
    const int per = (all_tiles + n_split - 1) / n_split;
    const int j0 = split * per, n = max(0, min(all_tiles, j0 + per) - j0);

    // Bounded wait; false (and the CTA gives up) once any wait has run out.
    auto wait_one = [&](uint64_t* bar, uint32_t parity) -> bool {
        if (mbar_try_wait(bar, parity)) return true;
        const long long t0 = clock64();
        while (!mbar_try_wait(bar, parity)) {
            if (*abort_flag) return false;
            if (clock64() - t0 > kWaitBudgetCycles) {
                *abort_flag = 1;
                atomicOr(p.err, NLLB_DEV_ERR_TIMEOUT);
                return false;
            }
        }
        return true;
    };
    // The same for a whole warp, with one answer.
    auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
        return __all_sync(0xffffffffu, wait_one(bar, parity));
    };

    if (warp < NQ * 4) {
        // ---- softmax: thread = query row
        const int t = warp >> 2, lq = warp & 3;  // query tile, TMEM lane quarter
        if (PAGED && p.k_new && split == 0) {
            const int t0 = (row0 + p.group - 1) / p.group;
            const int t1 = min(sq.qn, (row0 + NQ * kTile + p.group - 1) / p.group);
            rows_append<T, D>(p, sq, s, g, t0, t1, tid, NQ * 128);
        }
        const int row = row0 + t * kTile + lq * 32 + lane;
        const bool there = row < rows;
        const bool any = row0 + t * kTile + lq * 32 < rows;  // the warp has a row
        const int tok = row / p.group;
        const int lim = there ? (PAGED ? sq.kvn - sq.qn + tok + 1 : sq.kvn) : 0;
        const uint32_t lane_off = (uint32_t)(lq * 32) << 16;
        const uint32_t tS = tmem + lane_off + (uint32_t)t * 128, tO = tmem + lane_off + NQ * 128 + (uint32_t)t * D;
        const float sl = p.scale_log2;
        float m = -INFINITY, l = 0.f;  // m: the maximum in use, in units of the scaled score
        bool ok = true;
        for (int j = 0; j < n && ok; ++j) {
            if (!(ok = wait(s_full + t, j & 1))) break;
            if (j > 0 && !(ok = wait(o_full + t, (j - 1) & 1))) break;  // long over: its product came first
            tc_fence_after();
            if (any) {
                const uint32_t* vw = valid + (j % (2 * ST)) * 4;
                const int left = lim - (j0 + j) * kTile;  // visible keys of this tile, before the valid bits
                uint32_t bits[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int x = min(max(left - 32 * c, 0), 32);
                    bits[c] = vw[c] & (x == 32 ? 0xffffffffu : (1u << x) - 1u);
                }
                float mx = -INFINITY;
#pragma unroll
                for (int c = 0; c < 4; c += 2) {
                    float v[2][32];
                    tmem_ld32x2(tS + 32 * c, tS + 32 * c + 32, v[0], v[1]);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (bits[c + h] == 0xffffffffu) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) mx = fmaxf(mx, v[h][i]);
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                mx = fmaxf(mx, (bits[c + h] >> i) & 1u ? v[h][i] : -INFINITY);
                        }
                    }
                }
                const float mn = mx * sl;
                const bool grown = mn > m + kGrow || (m == -INFINITY && mn > -INFINITY);
                if (__any_sync(0xffffffffu, grown)) {
                    const float to = fmaxf(m, mn);
                    const float corr = m == -INFINITY ? 0.f : ex2_approx(m - to);
                    m = to;
                    l *= corr;
                    if (j > 0) {
#pragma unroll
                        for (int c = 0; c < D; c += 32) {
                            float o[32];
                            tmem_ld32(tO + c, o);
                            uint32_t r[2][16];
#pragma unroll
                            for (int i = 0; i < 32; ++i) r[i >> 4][i & 15] = __float_as_uint(o[i] * corr);
                            tmem_st16(tO + c, r[0]);
                            tmem_st16(tO + c + 16, r[1]);
                        }
                    }
                }
                const float off = (m == -INFINITY ? 0.f : m) - kWeightExp;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float v[32];
                    tmem_ld32(tS + 32 * c, v);
                    if (bits[c] != 0xffffffffu) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = (bits[c] >> i) & 1u ? v[i] : -INFINITY;
                    }
                    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        v[i] = ex2_approx(fmaf(v[i], sl, -off));
                        sum[i & 3] += v[i];
                    }
                    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    uint32_t hi[16];
                    if constexpr (C::F32) {
                        uint32_t lo[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) split2(v[2 * i], v[2 * i + 1], hi[i], lo[i]);
                        tmem_st16(tS + 32 * c + 16, lo);
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) hi[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
                    }
                    tmem_st16(tS + 32 * c, hi);
                }
                tmem_wait_st();
            }
            tc_fence_before();
            mbar_arrive(p_full + t);
        }
        if (ok && n > 0) ok = wait(o_full + t, (n - 1) & 1);
        tc_fence_after();
        if (n_split == 1) {
            if (ok && any) {
                const float inv = 1.0f / l;
                T* dst = static_cast<T*>(p.out) + (long long)(sq.q0 + tok) * p.o_row +
                         (long long)(g * p.group + row % p.group) * p.o_head;
#pragma unroll
                for (int c = 0; c < D; c += 32) {
                    float o[32];
                    if (n > 0) tmem_ld32(tO + c, o);
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
                for (int c = 0; c < D; c += 32) {
                    float o[32];
                    if (n > 0) tmem_ld32(tO + c, o);
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *reinterpret_cast<float4*>(st + c + i) =
                            l == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                }
                *reinterpret_cast<float4*>(st + D) = make_float4(l == 0.f ? -INFINITY : m, ok ? l : -1.f, 0.f, 0.f);
            }
        }
    } else if (warp < NQ * 4 + kLoaders / 32) {
        // ---- fetch
        const int lt = tid - NQ * 128;
        uint64_t* ptrs = reinterpret_cast<uint64_t*>(sm + C::PTRS);
        uint32_t* vw = reinterpret_cast<uint32_t*>(sm + C::VALID);
        // barrier of the fetching threads; true if all of them are still at work
        auto loaders_sync = [](bool ok) -> bool {
            uint32_t all;
            asm volatile(
                "{\n\t.reg .pred p, q;\n\t"
                "setp.ne.b32 p, %1, 0;\n\t"
                "barrier.cta.red.and.pred q, 1, %2, p;\n\t"
                "selp.u32 %0, 1, 0, q;\n\t}"
                : "=r"(all)
                : "r"((uint32_t)ok), "n"(kLoaders)
                : "memory");
            return all != 0;
        };
        auto q_row = [&](int r) -> const T* {
            const int row = row0 + r;
            if (row >= rows) return nullptr;
            return static_cast<const T*>(p.q) + (long long)(sq.q0 + row / p.group) * p.q_row +
                   (long long)(g * p.group + row % p.group) * p.q_head;
        };
        // row addresses of key tile j, a row per thread (the first warp takes two), and which rows are visible
        auto addresses = [&](int j) {
            uint64_t* at = ptrs + (j & 1) * 256;
#pragma unroll
            for (int r = lt; r < kTile; r += kLoaders) {
                const int key = (j0 + j) * kTile + r;
                const T *k = nullptr, *v = nullptr;
                const bool seen = key < longest && rows_key<T, PAGED>(p, sq, s, g, key, k, v);
                at[r] = seen ? reinterpret_cast<uint64_t>(k) : 0;
                at[128 + r] = seen ? reinterpret_cast<uint64_t>(v) : 0;
                const uint32_t word = __ballot_sync(0xffffffffu, seen);
                if (lane == 0) vw[(j % (2 * ST)) * 4 + (r >> 5)] = word;
            }
        };
        bool ok = true;
        if constexpr (!C::F32) {
            constexpr int CH = D / 8;  // 16-byte chunks of a row
#pragma unroll 4
            // (without keys nothing is fetched: a split's state may be written at once)
            for (int i = n > 0 ? lt : NQ * kTile * CH; i < NQ * kTile * CH; i += kLoaders) {
                const int r = i / CH, c = i % CH;
                const T* src = q_row(r);
                cp_async16(base + C::SQ + (r / kTile) * C::OPER + chunk_off(r % kTile, c),
                           src ? src + c * 8 : static_cast<const T*>(p.q), src != nullptr);
            }
            // group x = 2 j fetches K of tile j (the first with Q), 2 j + 1 its V
            auto arrive = [&](int x) {
                fence_async_smem();
                mbar_arrive((x & 1 ? v_full : k_full) + (x >> 1) % ST);
            };
            for (int j = 0; j < n; ++j) {
                addresses(j);
                if (!(ok = loaders_sync(ok))) break;
                const uint64_t* at = ptrs + (j & 1) * 256;
                const int st = j % ST;
#pragma unroll
                for (int kv = 0; kv < 2; ++kv) {
                    if (j >= ST) ok = ok && wait((kv ? v_empty : k_empty) + st, ((j / ST) - 1) & 1);
                    if (!ok) continue;  // to the next barrier, which all then leave together
                    const uint32_t dst = base + (kv ? C::SV : C::SK) + st * C::OPER;
#pragma unroll
                    for (int i = 0; i < (kTile * CH + kLoaders - 1) / kLoaders; ++i) {
                        const int x = lt + i * kLoaders, r = x / CH, c = x % CH;
                        if (x >= kTile * CH) break;
                        const T* src = reinterpret_cast<const T*>(at[kv * 128 + r]);
                        cp_async16(dst + chunk_off(r, c), src ? src + c * 8 : static_cast<const T*>(p.q),
                                   src != nullptr);
                    }
                    cp_commit();
                    if (2 * j + kv >= C::LAG) {
                        cp_wait<C::LAG>();
                        arrive(2 * j + kv - C::LAG);
                    }
                }
            }
            if (ok && n > 0) {
                if constexpr (C::LAG >= 3)
                    if (n > 1) cp_wait<2>(), arrive(2 * n - 3);
                if constexpr (C::LAG >= 2) cp_wait<1>(), arrive(2 * n - 2);
                cp_wait<0>(), arrive(2 * n - 1);
            }
            cp_wait<0>();
        } else {
            // fp32: 32 bytes (8 elements) of a row per thread become a chunk of each part
            constexpr int CH = D / 8, PASSES = (kTile * CH + kLoaders - 1) / kLoaders, BATCH = 6;
            auto store = [&](uint32_t dst, int r, int c, const float4& a, const float4& b) {
                uint4 hi, lo;
                split2(a.x, a.y, hi.x, lo.x);
                split2(a.z, a.w, hi.y, lo.y);
                split2(b.x, b.y, hi.z, lo.z);
                split2(b.z, b.w, hi.w, lo.w);
                unsigned char* to = sm + dst + chunk_off(r, c);
                *reinterpret_cast<uint4*>(to) = hi;
                *reinterpret_cast<uint4*>(to + C::PART) = lo;
            };
            const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
            auto fetch = [&](uint32_t dst, auto&& row_of, uint64_t* empty, uint32_t parity, bool must_wait) {
#pragma unroll
                for (int i0 = 0; i0 < PASSES; i0 += BATCH) {
                    float4 a[BATCH], b[BATCH];
#pragma unroll
                    for (int i = 0; i < BATCH; ++i) {
                        const int x = lt + (i0 + i) * kLoaders;
                        const T* src = x < kTile * CH ? row_of(x / CH) : nullptr;
                        a[i] = b[i] = zero;
                        if (src) {
                            const float4* f = reinterpret_cast<const float4*>(src) + (x % CH) * 2;
                            a[i] = __ldg(f), b[i] = __ldg(f + 1);
                        }
                    }
                    if (i0 == 0 && must_wait && !(ok = wait(empty, parity))) return;
#pragma unroll
                    for (int i = 0; i < BATCH; ++i) {
                        const int x = lt + (i0 + i) * kLoaders;
                        if (x < kTile * CH) store(dst, x / CH, x % CH, a[i], b[i]);
                    }
                }
            };
            if (n > 0) fetch(C::SQ, q_row, nullptr, 0, false);
            for (int j = 0; j < n; ++j) {
                addresses(j);
                if (!(ok = loaders_sync(ok))) break;
                const uint64_t* at = ptrs + (j & 1) * 256;
                const int st = j % ST;
#pragma unroll
                for (int kv = 0; kv < 2; ++kv) {
                    if (!ok) continue;  // to the next barrier, which all then leave together
                    fetch((kv ? C::SV : C::SK) + st * C::OPER,
                          [&](int r) { return reinterpret_cast<const T*>(at[kv * 128 + r]); },
                          (kv ? v_empty : k_empty) + st, ((j / ST) - 1) & 1, j >= ST);
                    if (!ok) continue;
                    fence_async_smem();
                    mbar_arrive((kv ? v_full : k_full) + st);
                }
            }
        }
    } else if (lane == 0) {
        // ---- products
        constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;
        constexpr uint32_t id_s = umma_idesc_f16(128, 128) | fmt, id_o = umma_idesc_f16(128, D) | fmt | (1u << 16);
        // V's descriptor: the leading byte offset is the distance between 64-element blocks of a row
        constexpr uint64_t lead = ((uint64_t)(kBlock >> 4) << 16) ^ ((uint64_t)1 << 16);
        auto scores = [&](int t, int st) {
            const uint32_t q = base + C::SQ + t * C::OPER, k = base + C::SK + st * C::OPER;
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
                const uint32_t o = (uint32_t)(ks >> 2) * kBlock + (ks & 3) * 32;
                const uint64_t a = umma_desc_k_sw128(q + o), b = umma_desc_k_sw128(k + o);
                tc_mma_f16(tmem + t * 128, a, b, id_s, ks > 0);
                if constexpr (C::F32) {
                    tc_mma_f16(tmem + t * 128, a, umma_desc_k_sw128(k + C::PART + o), id_s, 1);
                    tc_mma_f16(tmem + t * 128, umma_desc_k_sw128(q + C::PART + o), b, id_s, 1);
                }
            }
        };
        auto output = [&](int t, int st, bool accumulate) {
            const uint32_t v = base + C::SV + st * C::OPER, o = tmem + NQ * 128 + t * D;
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
                const uint32_t a = tmem + t * 128 + (ks >> 1) * 32 + (ks & 1) * 8;
                const uint64_t b = umma_desc_k_sw128(v + ks * 2048) ^ lead;
                tc_mma_f16_ta(o, a, b, id_o, accumulate || ks > 0);
                if constexpr (C::F32) {
                    tc_mma_f16_ta(o, a, umma_desc_k_sw128(v + C::PART + ks * 2048) ^ lead, id_o, 1);
                    tc_mma_f16_ta(o, a + 16, b, id_o, 1);
                }
            }
        };
        bool ok = true;
        if (n > 0 && (ok = wait_one(k_full, 0))) {
            tc_fence_after();
            for (int t = 0; t < NQ; ++t) {
                scores(t, 0);
                tc_commit(s_full + t);
            }
            tc_commit(k_empty);
        }
        for (int j = 0; j < n && ok; ++j) {
            const int st = j % ST, nx = (j + 1) % ST;
            for (int t = 0; t < NQ && ok; ++t) {
                if (t == 0 && !(ok = wait_one(v_full + st, (j / ST) & 1))) break;
                if (!(ok = wait_one(p_full + t, j & 1))) break;
                tc_fence_after();
                output(t, st, j > 0);
                tc_commit(o_full + t);
                if (t == NQ - 1) tc_commit(v_empty + st);  // before the wait for K, which may come after the next V
                if (j + 1 < n) {
                    if (t == 0 && !(ok = wait_one(k_full + nx, ((j + 1) / ST) & 1))) break;
                    tc_fence_after();
                    scores(t, nx);
                    tc_commit(s_full + t);
                }
            }
            if (ok && j + 1 < n) tc_commit(k_empty + nx);
        }
        // whatever was issued is over before tensor memory is given back
        tc_commit(done);
        (void)mbar_wait_bounded(done, 0);
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

template <typename T, int D, int NQ, bool PAGED>
cudaError_t launch_tc(const RowsParams& p, int n_split, cudaStream_t st) {
    using C = Cfg<T, D, NQ>;
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
    return cudaLaunchKernelEx(&cfg, rows_tc_kernel<T, D, NQ, PAGED>, p, n_split);
}

template <typename T, int D, bool PAGED>
cudaError_t launch_by_tiles(const RowsParams& p, int num_sms, cudaStream_t st) {
    const long long rows = (long long)p.max_q * p.group, heads = (long long)p.kv_heads * p.n_seq;
    if constexpr (sizeof(T) == 2) {
        // two query tiles per CTA where they still give every SM one
        if (rows > kTile && (rows + 2 * kTile - 1) / (2 * kTile) * heads >= num_sms)
            return launch_tc<T, D, 2, PAGED>(p, 1, st);
    }
    const long long units = (rows + kTile - 1) / kTile * heads;
    // splits: until two CTAs per SM are at work, none below two key tiles, one cluster at most
    int n_split = 1;
    while (n_split < 8 && units * n_split * 2 <= 2LL * num_sms && p.max_kv >= 512 * n_split) n_split *= 2;
    return launch_tc<T, D, 1, PAGED>(p, n_split, st);
}

template <typename T>
cudaError_t launch_by_dim(const RowsParams& p, int head_dim, bool paged, int num_sms, cudaStream_t st) {
    if (head_dim == 64)
        return paged ? launch_by_tiles<T, 64, true>(p, num_sms, st) : launch_by_tiles<T, 64, false>(p, num_sms, st);
    return paged ? launch_by_tiles<T, 128, true>(p, num_sms, st) : launch_by_tiles<T, 128, false>(p, num_sms, st);
}

template <typename T, int D, int NQ>
cudaError_t configure_one() {
    cudaError_t e = cudaFuncSetAttribute(rows_tc_kernel<T, D, NQ, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)Cfg<T, D, NQ>::SMEM);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(rows_tc_kernel<T, D, NQ, false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (int)Cfg<T, D, NQ>::SMEM);
    return e;
}

}  // namespace

cudaError_t configure_rows_tc() {
    cudaError_t e = configure_one<float, 64, 1>();
    if (e == cudaSuccess) e = configure_one<float, 128, 1>();
    if (e == cudaSuccess) e = configure_one<__half, 64, 1>();
    if (e == cudaSuccess) e = configure_one<__half, 64, 2>();
    if (e == cudaSuccess) e = configure_one<__half, 128, 1>();
    if (e == cudaSuccess) e = configure_one<__half, 128, 2>();
    if (e == cudaSuccess) e = configure_one<__nv_bfloat16, 64, 1>();
    if (e == cudaSuccess) e = configure_one<__nv_bfloat16, 64, 2>();
    if (e == cudaSuccess) e = configure_one<__nv_bfloat16, 128, 1>();
    if (e == cudaSuccess) e = configure_one<__nv_bfloat16, 128, 2>();
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
