// sample.cu -- nllb_sample: one token per row of logits by temperature, top-k,
// top-p and min-p, from a given uniform number (sm_100a).
//
//   w_i = exp((l_i - m) / T); the kept set is a prefix of the order (logit
//   falling, index rising), cut by a count, by a share of the weight and by a
//   least weight; the token is found by inverting the running sum of the kept
//   weights in index order.
//
// The bytes of the logits are its floor.  A row is shared by the CTAs of a
// cluster, which read it once and keep their slices in shared memory for the
// later passes -- or, for many long rows, read it again in each pass, which
// leaves room for more rows at a time (launch() has both sides' times).
// Nothing is sorted but short lists.  The border of the kept set is found by
// counting steps of (m - l) / T, the counts summed over the cluster through
// distributed shared memory: top-k by 64 coarse bins whose counters never
// collide, top-p by 2048 steps, from whose counts the weights follow closely
// enough to name the few steps the border can lie in.  Where everything kept
// lies in few elements, one CTA gathers, sorts and finishes them alone (17 us
// for one row of 256206 by top-k 50 and top-p 0.95).  Otherwise the exact
// weights above those steps are summed, the elements at the border gathered
// and sorted, or told apart 11 bits of their composite (order of the logit,
// index) at a time where thousands are equal; then one more pass sums the kept
// weights chunk by chunk and the token's chunk is searched.  Bound now by the
// passes' instructions and, for few rows, by the cluster's barriers: 512 rows
// of mixed settings 575 to 600 us, 0.9 TB/s of logits; 64 rows in bf16 by top-p
// 0.9 133 us.
//
// Weights are integer multiples of 2^-44 of the largest, so their sums are
// exact and the order of the atomics changes no result.  44 bits because 2^19
// of them (NLLB_SAMPLE_MAX_VOCAB) have to stay below 2^64.
#include <climits>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <string>
#include <type_traits>

#include "device_common.cuh"
#include "nllb_translate.h"

namespace nllb {
int set_error(int status, const std::string& msg);  // nllb_attn.cu

namespace {

using u64 = unsigned long long;

constexpr int kThreads = 512, kWarpsS = kThreads / 32;
constexpr int kBins = 2048, kBinBits = 11;
constexpr int kWeightBits = 44;
constexpr int kIndexBits = 19;
static_assert(NLLB_SAMPLE_MAX_VOCAB == 1 << kIndexBits, "an index fits the composite");
// the first histogram covers (m - l) / T up to 33: exp(-33) < 2^-45 weighs 0
constexpr float kSpan = 33.0f;
constexpr int kCoarse = kBins / 64;   // steps of a coarse bin

constexpr int kList = kBins / 2;  // candidates that rank 0 finishes alone, in the place of the masses

constexpr int kMaxCluster = 16;
constexpr int kSliceBytes = 1 << 17;           // of a row that one CTA holds at most
constexpr int kMaxChunks = kSliceBytes / 512;  // records: of a chunk of 512 bytes, or of 16 of a whole row
static_assert(NLLB_SAMPLE_MAX_VOCAB * 4 / 512 / 16 <= kMaxChunks, "records of a whole row");
static_assert(NLLB_SAMPLE_MAX_VOCAB / kMaxCluster * 4 <= kSliceBytes, "every row fits a cluster");

struct Args {
    const void* logits;
    long long ld;
    int vocab, slice;  // elements of a row; of a CTA's share (a multiple of the chunk)
    const float* temperature;
    const int* top_k;
    const float* top_p;
    const float* min_p;
    const float* u;
    int* out_tok;
    float* out_logp;
    bool expire;  // test: a wait of each row's last CTA runs out
};

struct Shared {
    u64 mass[kBins];
    u64 tot_mass[kBins / 2];  // this CTA's share of the bins, summed over the cluster (two CTAs or more)
    uint32_t cnt[kBins];
    uint32_t tot_cnt[kBins / 2];
    u64 chunk[kMaxChunks];     // kept weight of each chunk of the slice
    u64 warp_sum[kWarpsS];
    u64 sum;                   // this CTA's kept weight
    u64 found_before, border;
    uint32_t found_cnt;
    int found_bin;
    float best;                // this CTA's largest logit
    uint32_t key_lo, key_hi;   // this CTA's range of keys in the border step
    float red[kWarpsS];
    u64 z[2];                  // this CTA's weight, in all and above the window
    int win_lo, win_hi;        // steps the border by weight lies between
    uint32_t coarse[64];       // this CTA's counts of the first look
    uint32_t coarse_of[kThreads / 64][64];
    uint32_t listed;           // (rank 0) candidates gathered
    uint64_t loaded;           // barrier of the copy of the slice
    uint64_t never;            // test: a barrier that nothing arrives at
    int failed;
    int first_best;            // this CTA's lowest index of the largest logit
};

__device__ __forceinline__ u64 ld_cluster_u64(uint32_t addr) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
    return r;
}

// Larger logits get smaller keys; -0 counts as +0.
__device__ __forceinline__ uint32_t order_key(float l) {
    const uint32_t b = __float_as_uint(l + 0.0f);
    return (b & 0x80000000u) ? b : 0x7fffffffu - b;
}

// exp((l - m) / T) in units of 2^-kWeightBits, by a whole warp.  y = 32 log2
// of it = (l - m) scale is split as n + f, n a whole number and |f| <= 1/2;
// 2^(y/32) = 2^(n >> 5) * 2^((n & 31) / 32) * exp(f ln2 / 32), the middle
// factor from a table of 32 that the warp's lanes hold (a shuffle reads it;
// from shared memory the look-ups' bank conflicts cost more than all the rest)
// and the last by its series to the fourth power (Tang, 1989: the remainder is
// below 1.3e-12), in fp64: a token's border may lie anywhere between its
// neighbours', and fp32 sums over 256206 tokens place it too coarsely.  There
// are eleven fp64 operations, which bound the pass over all weights.
struct Weigher {
    float floor;  // logits below it weigh nothing: it rounds to 0 itself
    double md, scale;  // widened(m); 32 log2(e) / T
    double tab;  // 2^(lane/32), with the units' exponent
};
// l as a double by whole-number operations: the conversion instruction runs at a quarter of their rate and bound the
// pass over all weights.  Zeros and subnormals come out up to 2^-126 off; the largest logit is taken the same way, so it
// weighs 1 exactly, and 2^-126 is nothing beside a temperature of 2^-100.
__device__ __forceinline__ double widened(float l) {
    const uint32_t b = __float_as_uint(l);
    return __hiloint2double((int)((b & 0x80000000u) | (((b & 0x7fffffffu) >> 3) + 0x38000000u)), (int)(b << 29));
}
__device__ __forceinline__ u64 weight(float l, const Weigher& g) {
    const double y = (widened(fmaxf(l, g.floor)) - g.md) * g.scale;  // (NaN as the floor)
    const double magic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to a whole number
    const double t = y + magic;
    const int n = __double2loint(t);
    const double f = y - (t - magic);
    constexpr double a = 0.693147180559945309417 / 32.0;
    double p = fma(f, a * a * a * a / 24.0, a * a * a / 6.0);
    p = fma(f, p, a * a / 2.0);
    p = fma(f, p, a);
    p *= f;
    const int hi = __shfl_sync(0xffffffffu, __double2hiint(g.tab), n & 31);
    const int lo = __shfl_sync(0xffffffffu, __double2loint(g.tab), n & 31);
    const double x = __hiloint2double(hi + (int)((unsigned)(n >> 5) << 20), lo);
    // w < 2^52: adding 2^52 rounds it to a whole number in the low bits
    return (u64)__double_as_longlong(fma(x, p, x) + 4503599627370496.0) & 0xfffffffffffffull;
}

template <typename T>
__device__ __forceinline__ float as_float(T v) {
    if constexpr (std::is_same<T, float>::value) return v;
    else if constexpr (std::is_same<T, __half>::value) return __half2float(v);
    else return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T minus_inf() {
    if constexpr (std::is_same<T, float>::value) return -INFINITY;
    else if constexpr (std::is_same<T, __half>::value) return __ushort_as_half((unsigned short)0xfc00u);
    else return __ushort_as_bfloat16((unsigned short)0xff80u);
}

__device__ __forceinline__ float key_logit(uint32_t k) {  // the inverse of order_key
    return __uint_as_float((k & 0x80000000u) ? k : 0x7fffffffu - k);
}
__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t add_cluster_u32(uint32_t addr, uint32_t x) {
    uint32_t v;
    asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(v) : "r"(addr), "r"(x) : "memory");
    return v;
}
__device__ __forceinline__ void st_cluster_u64(uint32_t addr, u64 x) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(x) : "memory");
}

// Sums over the cluster of the variable at p, eight remote reads in flight
// (one after the other, each would wait for the last).
__device__ __forceinline__ u64 cluster_sum_u64(const u64* p, uint32_t C) {
    u64 s = 0;
    for (uint32_t z = 0; z < C; z += 8) {
        u64 t[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) t[i] = z + i < C ? ld_cluster_u64(map_rank(p, z + i)) : 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += t[i];
    }
    return s;
}
__device__ __forceinline__ uint32_t cluster_sum_u32(const uint32_t* p, uint32_t C) {
    uint32_t s = 0;
    for (uint32_t z = 0; z < C; z += 8) {
        uint32_t t[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) t[i] = z + i < C ? ld_cluster_u32(map_rank(p, z + i)) : 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += t[i];
    }
    return s;
}

template <typename T>
struct alignas(16) Vec {
    T x[16 / sizeof(T)];
};

// The largest of this thread's elements, NaN if one is.
template <typename T>
__device__ __forceinline__ float row_max(const Vec<T>* data, int n) {
    if constexpr (sizeof(T) == 4) {
        float a = -INFINITY, b = -INFINITY;
#pragma unroll 4
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const Vec<T> v = data[i];
            asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(a) : "f"(v.x[0]), "f"(v.x[1]));
            asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(b) : "f"(v.x[2]), "f"(v.x[3]));
        }
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(b));
        return a;
    } else {
        uint32_t m[4];
        m[0] = m[1] = m[2] = m[3] = std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
#pragma unroll 4
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const uint4 v = *reinterpret_cast<const uint4*>(data + i);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (std::is_same<T, __half>::value) asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(m[e]) : "r"(w[e]));
                else asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m[e]) : "r"(w[e]));
            }
        }
        float a = -INFINITY;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            T x;
            const unsigned short h = (unsigned short)(m[e >> 1] >> (16 * (e & 1)));
            if constexpr (std::is_same<T, __half>::value) x = __ushort_as_half(h);
            else x = __ushort_as_bfloat16(h);
            asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(as_float(x)));
        }
        return a;
    }
}

__device__ __forceinline__ u64 warp_sum_u64(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ u64 warp_scan_u64(u64 v, int lane) {  // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 w = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += w;
    }
    return v;
}

// One cluster per row, its slices in shared memory or (STREAM) read from
// global memory in every pass.
template <typename T, bool STREAM>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const Args a) {
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int VEC = 16 / (int)sizeof(T);
    constexpr int CHUNK = 32 * VEC;  // one vector per lane
    Shared& sh = *reinterpret_cast<Shared*>(smem);
    Vec<T>* data = reinterpret_cast<Vec<T>*>(smem + (sizeof(Shared) + 15) / 16 * 16);
    // chunks (a vector per lane) whose kept weight is recorded together, and those loaded together
    constexpr int SUPER = STREAM ? 16 : 1, DEPTH = STREAM ? 4 : 1;

    pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) sh.z[0] = sh.z[1] = 0, sh.listed = 0, sh.first_best = INT_MAX, sh.failed = 0;
    pdl_wait_primary();

    const uint32_t C = cluster_size(), rank = cluster_ctarank();
    const int row = blockIdx.x / C;
    const int first = (int)rank * a.slice;  // the slice's first element
    const int n = min(a.slice, max(0, a.vocab - first));
    const int n_chunks = (n + CHUNK - 1) / CHUNK;
    const T* src = static_cast<const T*>(a.logits) + (long long)row * a.ld + first;

    // ---- the slice into shared memory, NaN as -inf, and its largest logit
    float best = -INFINITY;
    bool inf_row = false;  // (STREAM) only the elements equal to top count, as 0
    float top = INFINITY;
    // vector i of the row from global memory
    auto fetch = [&](int i) -> Vec<T> {
        Vec<T> v;
        if ((i + 1) * VEC <= n) {
            *reinterpret_cast<uint4*>(&v) = ld_coherent(reinterpret_cast<const uint4*>(src) + i);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v.x[e] = i * VEC + e < n ? src[i * VEC + e] : minus_inf<T>();
        }
        if (inf_row) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v.x[e] = as_float(v.x[e]) == top ? T(0.0f) : minus_inf<T>();
        }
        return v;
    };
    // f(vector index, vector) for the vectors of a chunk, all chunks of the slice; done(super chunk) after each of its
    // SUPER.  A NaN passes every test of the passes below as -inf would.
    const int n_super = (n_chunks + SUPER - 1) / SUPER;
    auto vectors = [&](auto&& f, auto&& done) {
        for (int sc = warp; sc < n_super; sc += kWarpsS) {
#pragma unroll 1
            for (int k = 0; k < SUPER; k += DEPTH) {
                Vec<T> v[DEPTH];
                const int at = (sc * SUPER + k) * 32 + lane;
#pragma unroll
                for (int d = 0; d < DEPTH; ++d) {
                    if constexpr (STREAM) v[d] = fetch(at + 32 * d);
                    else v[d] = data[at + 32 * d];
                }
#pragma unroll
                for (int d = 0; d < DEPTH; ++d) f(at + 32 * d, v[d]);
            }
            done(sc);
        }
    };
    if constexpr (STREAM) {
        vectors(
            [&](int, const Vec<T>& v) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) best = fmaxf(best, as_float(v.x[e]));  // (passes over NaN)
            },
            [](int) {});
    } else {
        const bool vec = (reinterpret_cast<uintptr_t>(src) & 15u) == 0;
        const int n_vec = vec ? n / VEC : 0;  // whole vectors come by one bulk copy
        if (n_vec > 0 && tid == 0) {
            mbar_init(&sh.loaded, 1);
            fence_barrier_init();
            mbar_arrive_expect_tx(&sh.loaded, (uint32_t)n_vec * 16u);
            bulk_g2s(data, src, (uint32_t)n_vec * 16u, &sh.loaded);
        }
        for (int i = n_vec + tid; i < n_chunks * 32; i += kThreads) {
            Vec<T> v;
#pragma unroll
            for (int e = 0; e < VEC; ++e) v.x[e] = i * VEC + e < n ? src[i * VEC + e] : minus_inf<T>();
            data[i] = v;
        }
        __syncthreads();
        if (n_vec > 0 && !mbar_wait_bounded(&sh.loaded, 0)) {
            sh.failed = 1;
            (void)mbar_wait_bounded(&sh.loaded, 0);  // the copy may still be on its way
        }
        if (a.expire && rank == C - 1) {
            if (tid == 0) {
                mbar_init(&sh.never, 1);
                fence_barrier_init();
            }
            __syncthreads();
            if (!mbar_wait_bounded(&sh.never, 0, kTestWaitBudgetCycles)) sh.failed = 1;
        }
        __syncthreads();
        best = row_max<T>(data, n_chunks * 32);
        if (best != best) {  // a NaN is among them
            best = -INFINITY;
            for (int i = tid; i < n_chunks * 32; i += kThreads) {
                Vec<T> v = data[i];
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    if (as_float(v.x[e]) != as_float(v.x[e])) v.x[e] = minus_inf<T>();
                    best = fmaxf(best, as_float(v.x[e]));
                }
                data[i] = v;
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) sh.red[warp] = best;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kWarpsS; ++w) best = fmaxf(best, sh.red[w]);
        sh.best = sh.failed ? __int_as_float(0x7fc00000) : best;  // NaN: a copy did not come
    }
    cluster_sync_all();
    float m = -INFINITY;
    bool failed = false;
    {
        const float x = ld_cluster_f32(map_rank(&sh.best, min(lane, (int)C - 1)));  // a rank's in each lane
        failed = __any_sync(0xffffffffu, x != x);
        m = x;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    }

    // ---- the row's settings
    float temp = a.temperature ? ld_coherent(a.temperature + row) : 1.0f;
    const int k = a.top_k ? ld_coherent(a.top_k + row) : 0;
    const float top_p = a.top_p ? ld_coherent(a.top_p + row) : 1.0f;
    const float min_p = a.min_p ? ld_coherent(a.min_p + row) : 0.0f;
    float u = ld_coherent(a.u + row);
    u = u > 0.0f ? fminf(u, 1.0f) : 0.0f;  // (NaN too)
    const bool usable = !failed && m > -INFINITY && temp >= 0.0f && temp < INFINITY;
    if (!usable) {  // (uniform over the cluster)
        if (rank == 0 && tid == 0) {
            a.out_tok[row] = failed ? NLLB_SAMPLE_TIMEOUT : -1;
            if (a.out_logp) a.out_logp[row] = -INFINITY;
        }
        cluster_sync_all();
        return;
    }

    // The infinite ones share all the weight: as 0 among -inf.  So do those at the lowest end of the type, 2^104 and more
    // above the next ones, which is more than 34 of the largest temperature.
    if (m == INFINITY || (m <= -3.0e38f && m > -INFINITY)) {
        top = m;
        inf_row = true;
        for (int i = tid; !STREAM && i < n_chunks * 32; i += kThreads) {
            Vec<T> v = data[i];
#pragma unroll
            for (int e = 0; e < VEC; ++e) v.x[e] = as_float(v.x[e]) == top ? T(0.0f) : minus_inf<T>();
            data[i] = v;
        }
        m = 0.0f;
        __syncthreads();
    }

    // f(l, local index) for every element of the slice, a warp's lanes together
    auto each = [&](auto&& f) {
        vectors(
            [&](int at, const Vec<T>& v) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) f(as_float(v.x[e]), at * VEC + e);
            },
            [](int) {});
    };

    if (temp == 0.0f) {  // the first of the order
        int at = INT_MAX;
        each([&](float l, int i) {
            if (l == m) at = min(at, first + i);
        });
        at = __reduce_min_sync(0xffffffffu, at);
        if (lane == 0) atomicMin(&sh.first_best, at);
        cluster_sync_all();
        if (rank == 0 && tid == 0) {
            for (uint32_t z = 0; z < C; ++z) at = min(at, (int)ld_cluster_u32(map_rank(&sh.first_best, z)));
            a.out_tok[row] = at;
            if (a.out_logp) a.out_logp[row] = 0.0f;
        }
        cluster_sync_all();
        return;
    }

    // Keeps the factors below finite, and m - 34 temp above fp32's lowest number.  Where the next smaller fp32 number is
    // more than 40 temperatures below m, it is taken as 40: that weighs nothing all the same.
    temp = fmaxf(fminf(fmaxf(temp, 0x1p-100f), 0x1p96f), (m - nextafterf(m, -INFINITY)) / 40.0f);
    const float to_bin = (float)kBins / (kSpan * temp);
    // Place of a logit on the scale of the first histogram, in steps.  Places
    // rise as logits fall, in fp32 as well as in exact arithmetic, since every
    // operation rounds monotonically; so does the step (the nearest whole
    // number, by an addition: the conversion instruction is four times slower).
    // Every pass asks this one function which step a logit belongs to, and its
    // operations are spelled out so that no pass's are contracted into others:
    // what one pass counts in a step is what the next one gathers from it.
    constexpr float kWhole = 8388608.0f;  // 2^23: adding it rounds to a whole number
    auto place = [&](float l) -> float { return __fmul_rn(__fsub_rn(m, l), to_bin); };
    auto step_of = [&](float l) -> int {
        const float d = place(l);
        return d < (float)kBins - 0.5f ? (__float_as_int(__fadd_rn(d, kWhole)) & (2 * kBins - 1)) : kBins;
    };
    Weigher weigher;
    // exp(-34) 2^44 < 1/2.  Rounded away from m: half of fp32's step at m may be many temperatures.
    weigher.floor = __fsub_rd(m, 34.0f * temp);
    weigher.scale = 32.0 * 1.4426950408889634074 / (double)temp;
    weigher.md = widened(m);
    weigher.tab = exp2((double)lane / 32.0 + (double)kWeightBits);
    auto wt = [&](float l) { return weight(l, weigher); };  // by all lanes of a warp
    auto composite = [&](float l, int i) { return ((u64)order_key(l) << kIndexBits) | (u64)(first + i); };
    u64 least = 1;  // min-p as a weight
    if (min_p > 0.0f) {
        const double t = ceil((double)fminf(min_p, 1.0f) * (double)(1ull << kWeightBits));
        least = t > 1.0 ? (u64)t : 1;
    }
    auto share_of = [&](u64 whole) -> u64 {  // the weight that top-p asks for
        const double t = ceil((double)fmaxf(top_p, 0.0f) * (double)whole);
        const u64 want = t < (double)whole ? (u64)t : whole;
        return want > 0 ? want : 1;
    };
    auto threshold = [&](u64 whole) -> u64 {  // the token is the first whose running sum is above it
        const double t = (double)u * (double)whole;
        return t < (double)whole ? min((u64)t, whole - 1) : whole - 1;
    };
    auto answer = [&](int token, float l, u64 whole) {
        a.out_tok[row] = token;
        if (a.out_logp) {
            const double x = l == m ? 0.0 : ((double)l - (double)m) / (double)temp;
            a.out_logp[row] = (float)(x - log((double)whole * (1.0 / (double)(1ull << kWeightBits))));
        }
    };

    // ---- sums over the CTA
    auto block_scan = [&](u64 mine, u64& all) -> u64 {  // sum of the threads before this one
        const u64 inc = warp_scan_u64(mine, lane);
        __syncthreads();
        if (lane == 31) sh.warp_sum[warp] = inc;
        __syncthreads();
        u64 before = inc - mine;
        all = 0;
#pragma unroll
        for (int w = 0; w < kWarpsS; ++w) {
            const u64 x = sh.warp_sum[w];
            if (w < warp) before += x;
            all += x;
        }
        return before;
    };
    auto block_scan_d = [&](double mine, double& all) -> double {  // up to and including this one
        double inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double x = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += x;
        }
        __syncthreads();
        if (lane == 31) sh.warp_sum[warp] = (u64)__double_as_longlong(inc);
        __syncthreads();
        double before = 0.0;
        all = 0.0;
#pragma unroll
        for (int w = 0; w < kWarpsS; ++w) {
            const double x = __longlong_as_double((long long)sh.warp_sum[w]);
            if (w < warp) before += x;
            all += x;
        }
        return before + inc;
    };
    // Sums over the cluster of values each thread has a part of (once per row).
    auto cluster_sums = [&](u64 x, u64 y, u64& sx, u64& sy) {
        x = warp_sum_u64(x), y = warp_sum_u64(y);
        if (lane == 0) {
            atomicAdd(&sh.z[0], x);
            atomicAdd(&sh.z[1], y);
        }
        cluster_sync_all();
        const uint32_t k = (uint32_t)min(lane, (int)C - 1);  // a rank's in each lane
        const bool in = lane < (int)C;
        const u64 a = ld_cluster_u64(map_rank(&sh.z[0], k)), b = ld_cluster_u64(map_rank(&sh.z[1], k));
        sx = warp_sum_u64(in ? a : 0), sy = warp_sum_u64(in ? b : 0);
    };

    // ---- histograms over the cluster
    constexpr int PER = kBins / kThreads;  // a thread's bins, PER tid ...
    uint32_t c[PER];                       // their counts, in the cluster
    auto clear = [&](bool by_mass) {
        for (int b = tid; b < kBins; b += kThreads) {
            sh.cnt[b] = 0;
            if (by_mass) sh.mass[b] = 0;
        }
        __syncthreads();
    };
    // Sums the CTAs' histograms: each CTA a share of the bins, then all read all.
    auto collect = [&](bool by_mass, u64 (&v)[PER]) {
        cluster_sync_all();
        const int share = kBins / (int)C;
        if (C > 1) {
            for (int b = tid; b < share; b += kThreads) {
                const uint32_t n0 = cluster_sum_u32(&sh.cnt[rank * share + b], C);
                const u64 w = by_mass ? cluster_sum_u64(&sh.mass[rank * share + b], C) : 0;
                sh.tot_cnt[b] = n0;
                if (by_mass) sh.tot_mass[b] = w;
            }
            cluster_sync_all();
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int b = tid * PER + i;
            if (C > 1) {
                const uint32_t z = (uint32_t)(b / share), at = (uint32_t)(b % share);
                c[i] = ld_cluster_u32(map_rank(&sh.tot_cnt[at], z));
                v[i] = by_mass ? ld_cluster_u64(map_rank(&sh.tot_mass[at], z)) : (u64)c[i];
            } else {
                c[i] = sh.cnt[b];
                v[i] = by_mass ? sh.mass[b] : (u64)c[i];
            }
        }
    };
    // The first bin at which the sum of the values up to and including it, from
    // `base` on, reaches `want`; found_bin -1 if none does.
    auto find = [&](const u64 (&v)[PER], u64 base, u64 want) {
        u64 mine = 0, all;
#pragma unroll
        for (int i = 0; i < PER; ++i) mine += v[i];
        u64 before = base + block_scan(mine, all);
        if (tid == 0 && !(base < want && want <= base + all)) sh.found_bin = -1, sh.found_cnt = 0, sh.found_before = base;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (before < want && want <= before + v[i]) {
                sh.found_bin = tid * PER + i;
                sh.found_cnt = c[i];
                sh.found_before = before;
            }
            before += v[i];
        }
        __syncthreads();
    };
    const bool cut_k = k > 0 && k < a.vocab, cut_p = top_p < 1.0f;
    u64 limit = ~0ull;  // the composite of the last element kept; its logit and its index in this slice
    float last_l = -INFINITY;
    int last_i = INT_MAX;
    auto set_limit = [&](u64 to) {
        if (to == ~0ull) return;  // nothing is cut
        limit = to;
        last_l = key_logit((uint32_t)(limit >> kIndexBits));
        last_i = (int)(limit & ((1ull << kIndexBits) - 1ull)) - first;
    };
    auto within = [&](float l, int i) { return l > last_l || (l == last_l && i <= last_i); };
    // Where the k-th element lies: 64 bins of kCoarse steps.  Each lane has a
    // counter of its own per bin, in its own bank of shared memory, so no two
    // of a warp's additions meet (counters by step took about two additions a
    // cycle, more than all the rest of the pass).  Every warp ends with the
    // same answers.
    struct Coarse {
        int at;            // the first bin at which the count reaches k, 64 if none does
        uint64_t before, up_to;  // elements before it, and up to it
    };
    auto look = [&]() -> Coarse {
        clear(false);
        each([&](float l, int) {
            const int b = step_of(l);
            if (b < kBins) atomicAdd(&sh.cnt[b / kCoarse * 32 + lane], 1u);
        });
        __syncthreads();
        {
            const int b = tid / (kThreads / 64), x = tid % (kThreads / 64);
            constexpr int N = 32 * 64 / kThreads;
            uint32_t sum = 0;
#pragma unroll
            for (int e = 0; e < N; ++e) sum += sh.cnt[b * 32 + x * N + e];
#pragma unroll
            for (int o = 1; o < kThreads / 64; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (x == 0) sh.coarse[b] = sum;
        }
        cluster_sync_all();
        {  // some ranks' counts of a bin per thread, then all of them
            uint32_t sum = 0;
            for (int z = tid / 64; z < (int)C; z += kThreads / 64)
                sum += ld_cluster_u32(map_rank(&sh.coarse[tid % 64], z));
            sh.coarse_of[tid / 64][tid % 64] = sum;
        }
        __syncthreads();
        uint32_t v0 = 0, v1 = 0;
#pragma unroll
        for (int z = 0; z < kThreads / 64; ++z) {
            v0 += sh.coarse_of[z][2 * lane];
            v1 += sh.coarse_of[z][2 * lane + 1];
        }
        const u64 inc = warp_scan_u64(v0 + v1, lane), c0 = inc - v1, before = c0 - v0;
        const unsigned hit = __ballot_sync(0xffffffffu, inc >= (u64)k);
        Coarse r = {64, 0, 0};
        if (hit) {
            const int f = __ffs(hit) - 1;
            const u64 a = __shfl_sync(0xffffffffu, before, f), b = __shfl_sync(0xffffffffu, c0, f);
            const u64 c = __shfl_sync(0xffffffffu, inc, f);
            r.at = 2 * f + (b < (u64)k);
            r.before = b < (u64)k ? b : a;
            r.up_to = b < (u64)k ? c : b;
        }
        return r;
    };
    // Steps fine_lo to fine_hi in fine_per bins each, at most 2048 in all: the
    // step decides, then the place within it, held inside the step.
    int fine_lo = 0, fine_hi = 0, fine_per = 0;
    auto set_fine = [&](int lo, int hi) { fine_lo = lo, fine_hi = hi, fine_per = kBins / (hi - lo + 1); };
    auto fine = [&](float l) -> int {  // -1: before them; kBins: after
        const int s = step_of(l);
        if (s < fine_lo) return -1;
        if (s > fine_hi) return kBins;
        const float d = place(l), nearest = __fsub_rn(__fadd_rn(d, kWhole), kWhole);  // s
        const float along = __fadd_rn(__fsub_rn(d, nearest), 0.5f);                   // 0 to 1
        const float x = fmaxf(__fsub_rn(__fmul_rn(along, (float)fine_per), 0.5f), 0.0f);
        return (s - fine_lo) * fine_per + min(__float_as_int(__fadd_rn(x, kWhole)) & (2 * kBins - 1), fine_per - 1);
    };
    auto count = [&](auto&& bin, u64 (&v)[PER]) {  // what `bin` puts into [0, kBins)
        __syncthreads();
        clear(false);
        each([&](float l, int i) {
            const int f = bin(l);
            if (f >= 0 && f < kBins && within(l, i)) atomicAdd(&sh.cnt[f], 1u);
        });
        collect(false, v);
    };
    // Steps between which the sum of the weights reaches top_p of the whole,
    // from the counts alone: within a step the weights differ by a factor of
    // exp(kSpan / kBins) at most.  The exact sums reach it there too: the slack
    // of 1e-5 is far above what the bounds here and the weights' units round off
    // (2^19 halves of 2^-44 of the largest weight, fp32's exponentials), and
    // steps past the last weigh nothing.
    auto window = [&] {
        double lo[PER], hi[PER], lo_mine = 0.0, hi_mine = 0.0, lo_all, hi_all;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const float x = (float)(tid * PER + i), w = kSpan / (float)kBins;
            lo[i] = (double)c[i] * (double)expf(-(x + 0.51f) * w);
            hi[i] = (double)c[i] * (double)expf(-fmaxf(x - 0.51f, 0.0f) * w);
            lo_mine += lo[i], hi_mine += hi[i];
        }
        if (tid == 0) sh.win_lo = sh.win_hi = kBins - 1;
        double lo_sum = block_scan_d(lo_mine, lo_all) - lo_mine, hi_sum = block_scan_d(hi_mine, hi_all) - hi_mine;
        const double p = (double)fmaxf(top_p, 0.0f);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            lo_sum += lo[i], hi_sum += hi[i];
            if (lo_sum >= (p + 1e-5) * (lo_sum + fmax(hi_all - hi_sum, 0.0)) && c[i] > 0)
                atomicMin(&sh.win_hi, tid * PER + i);
            if (hi_sum >= (p - 1e-5) * (hi_sum + fmax(lo_all - lo_sum, 0.0))) atomicMin(&sh.win_lo, tid * PER + i);
        }
        __syncthreads();
    };

    // ---- lists in rank 0's shared memory, in the place of the masses
    auto gather = [&](auto&& in) {  // the composites of the elements that in(l, i) picks, in any order
        vectors(
            [&](int at, const Vec<T>& v) {
                int mine = 0;
                bool is[VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    is[e] = in(as_float(v.x[e]), at * VEC + e);
                    mine += is[e];
                }
                if (mine > 0) {
                    uint32_t to = add_cluster_u32(map_rank(&sh.listed, 0), (uint32_t)mine);
#pragma unroll
                    for (int e = 0; e < VEC; ++e)
                        if (is[e]) {
                            if (to < kList)
                                st_cluster_u64(map_rank(&sh.mass[to], 0), composite(as_float(v.x[e]), at * VEC + e));
                            ++to;
                        }
                }
            },
            [](int) {});
    };
    auto sort = [&](int n) -> int {  // sh.mass[0 .. n) rising, padded to a power of two, which it returns
        int n2 = 64;
        while (n2 < n) n2 *= 2;
        for (int i = n + tid; i < n2; i += kThreads) sh.mass[i] = ~0ull;
        for (int size = 2; size <= n2; size *= 2)
            for (int stride = size / 2; stride > 0; stride /= 2) {
                __syncthreads();
                for (int t = tid; t < n2 / 2; t += kThreads) {
                    const int i = 2 * t - (t & (stride - 1)), j = i + stride;
                    const u64 x = sh.mass[i], y = sh.mass[j];
                    if ((x > y) == ((i & size) == 0)) sh.mass[i] = y, sh.mass[j] = x;
                }
            }
        __syncthreads();
        return n2;
    };

    // The composite of the element at which the sum reaches `want`, `base`
    // before the gathered ones; ~0 if none does.  Rank 0 sorts them.
    auto pick = [&](bool by_mass, u64 base, u64 want) -> u64 {
        if (rank == 0) {
            const int n = min((int)sh.listed, kList);
            (void)sort(n);
            constexpr int EACH = kList / kThreads;
            u64 w[EACH], mine = 0, all;
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                const int i = tid * EACH + e;
                const u64 weighs = by_mass ? wt(key_logit((uint32_t)(sh.mass[i] >> kIndexBits))) : 1;
                w[e] = i < n ? weighs : 0;
                mine += w[e];
            }
            u64 before = base + block_scan(mine, all);
            if (tid == 0 && !(base < want && want <= base + all)) sh.border = ~0ull;
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                if (before < want && want <= before + w[e]) sh.border = sh.mass[tid * EACH + e];
                before += w[e];
            }
            if (tid == 0) sh.listed = 0;
        }
        cluster_sync_all();
        return ld_cluster_u64(map_rank(&sh.border, 0));
    };
    // The same among any number of elements, those that in(l) picks: 11 bits of
    // their composites at a time.
    auto radix = [&](auto&& in, bool by_mass, u64 base, u64 want) -> u64 {
        bool one = false;
        uint32_t lo = 0xffffffffu, hi = 0;
        each([&](float l, int i) {
            if (in(l) && within(l, i)) {
                lo = min(lo, order_key(l));
                hi = max(hi, order_key(l));
            }
        });
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
        if (tid == 0) sh.key_lo = 0xffffffffu, sh.key_hi = 0;
        __syncthreads();
        if (lane == 0) {
            atomicMin(&sh.key_lo, lo);
            atomicMax(&sh.key_hi, hi);
        }
        cluster_sync_all();
        for (uint32_t z = 0; z < C; ++z) {
            lo = min(lo, ld_cluster_u32(map_rank(&sh.key_lo, z)));
            hi = max(hi, ld_cluster_u32(map_rank(&sh.key_hi, z)));
        }
        u64 from = (u64)lo << kIndexBits, to = ((u64)hi << kIndexBits) | ((1u << kIndexBits) - 1u);
        while (!one) {
            to = min(to, limit);
            const int bits = 64 - __clzll((long long)(to - from));
            const int shift = max(0, bits - kBinBits);
            clear(by_mass);
            each([&](float l, int i) {
                const u64 x = composite(l, i);
                const bool in = x >= from && x <= to;
                if (__any_sync(0xffffffffu, in)) {
                    const u64 w = by_mass ? wt(l) : 0;
                    if (in) {
                        const int b = (int)((x - from) >> shift);
                        atomicAdd(&sh.cnt[b], 1u);
                        if (by_mass) atomicAdd(&sh.mass[b], w);
                    }
                }
            });
            u64 v[PER];
            collect(by_mass, v);
            find(v, base, want);
            if (sh.found_bin < 0) break;  // (the sums say otherwise)
            base = sh.found_before;
            from += (u64)sh.found_bin << shift;
            to = from + ((1ull << shift) - 1ull);
            one = sh.found_cnt == 1 || shift == 0;
        }
        return min(to, limit);
    };

    if (cut_k || cut_p) {
        u64 v[PER];
        Coarse r = {64, 0, 0};
        if (cut_k) r = look();
        const bool by_k = r.at < 64;  // (fewer than k weigh anything otherwise)
        int last = by_k ? r.at * kCoarse + kCoarse - 1 : -1;  // the steps up to it hold everything kept
        u64 n_list = r.up_to;                                 // elements in them
        if (!by_k && cut_p) {
            // counts by step, and from them the steps between which the weights reach their share
            count(step_of, v);
            window();
            last = sh.win_hi;
            u64 mine = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (tid * PER + i <= last) mine += c[i];
            (void)block_scan(mine, n_list);
        }
        if (last >= 0 && n_list <= kList) {
            // ---- few candidates: rank 0 takes them all and finishes alone
            u64 whole = 0, unused = 0;
            if (!by_k) {
                u64 z = 0;
                each([&](float l, int) { z += wt(l); });
                cluster_sums(z, 0, whole, unused);
            }
            gather([&](float l, int) { return step_of(l) <= last; });
            cluster_sync_all();
            if (rank != 0) return;  // (nobody reads this CTA's shared memory any more)
            const int n = min((int)sh.listed, kList);  // (n_list: the same function counted and gathered)
            const int n2 = sort(n);
            // weights in the order, the cuts, then the kept ones in the order of their indices
            constexpr int EACH = kList / kThreads;
            u64 w[EACH], x[EACH], mine = 0, all;
            const int n_k = by_k ? min(n, k) : n;
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                const int i = tid * EACH + e;
                x[e] = i < n_k ? sh.mass[i] : ~0ull;
                const u64 weighs = wt(key_logit((uint32_t)(x[e] >> kIndexBits)));
                w[e] = i < n_k ? weighs : 0;
                mine += w[e];
            }
            u64 before = block_scan(mine, all);
            const u64 want = cut_p ? share_of(by_k ? all : whole) : ~0ull;
            mine = 0;
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                const int i = tid * EACH + e;
                const u64 weighs = w[e];
                if (!(before < want && (weighs >= least || i == 0))) w[e] = 0;
                before += weighs;
                mine += w[e];
                if (i < n2) {
                    sh.mass[i] = w[e] ? (x[e] & ((1ull << kIndexBits) - 1ull)) << 32 | (u64)i : ~0ull;
                    sh.mass[kList + i] = w[e];
                    sh.cnt[i] = (uint32_t)(x[e] >> kIndexBits);
                }
            }
            (void)block_scan(mine, all);
            (void)sort(n2);
            mine = 0;
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                const int i = tid * EACH + e;
                x[e] = i < n2 ? sh.mass[i] : ~0ull;
                w[e] = x[e] != ~0ull ? sh.mass[kList + (uint32_t)x[e]] : 0;
                mine += w[e];
            }
            u64 unused_all;
            before = block_scan(mine, unused_all);
            const u64 thr = threshold(all);
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                if (before <= thr && thr < before + w[e])
                    answer((int)(x[e] >> 32), key_logit(sh.cnt[(uint32_t)x[e]]), all);
                before += w[e];
            }
            return;
        }
        if (by_k) {
            set_fine(r.at * kCoarse, r.at * kCoarse + kCoarse - 1);
            count(fine, v);
            find(v, r.before, (u64)k);
            const int f = sh.found_bin;
            const u64 base = sh.found_before;
            const uint32_t n = sh.found_cnt;
            if (n <= kList) {
                gather([&](float l, int i) { return fine(l) == f; });
                cluster_sync_all();
                set_limit(pick(false, base, (u64)k));
            } else {
                set_limit(radix([&](float l) { return fine(l) == f; }, false, base, (u64)k));
            }
        }
        if (cut_p) {
            if (by_k) {
                count(step_of, v);
                window();
            }
            // exact weights: of everything, of what lies above the window, and in 2048 bins within it
            set_fine(sh.win_lo, sh.win_hi);
            clear(true);
            u64 z = 0, above = 0;
            each([&](float l, int i) {
                const u64 w = wt(l);
                if (!within(l, i)) return;
                z += w;
                const int f = fine(l);
                if (f < 0) above += w;
                else if (f < kBins) {
                    atomicAdd(&sh.cnt[f], 1u);
                    atomicAdd(&sh.mass[f], w);
                }
            });
            u64 all_z, all_above;
            cluster_sums(z, above, all_z, all_above);
            collect(true, v);
            const u64 want = share_of(all_z);
            find(v, all_above, want);
            const int f = sh.found_bin;
            const u64 base = sh.found_before;
            const uint32_t n = sh.found_cnt;
            if (n <= kList) {
                gather([&](float l, int i) { return fine(l) == f && within(l, i); });
                cluster_sync_all();
                set_limit(pick(true, base, want));
            } else {  // many ties
                set_limit(radix([&](float l) { return fine(l) == f; }, true, base, want));
            }
        }
    }
    // ---- the kept weight of each chunk, of this CTA, of the row
    // the weights of vector `at` of the slice that are kept, and their sum
    const bool plain = limit == ~0ull && least == 1;  // nothing is cut
    auto kept = [&](int at, const Vec<T>& v, u64 (&w)[VEC]) -> u64 {
        if (plain) {
            u64 sum = 0;
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum += w[e] = wt(as_float(v.x[e]));
            return sum;
        }
        bool in[VEC], any = false;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float l = as_float(v.x[e]);
            in[e] = within(l, at * VEC + e);
            any |= in[e];
            w[e] = 0;
        }
        u64 sum = 0;
        if (__any_sync(0xffffffffu, any)) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const u64 x = wt(as_float(v.x[e]));
                if (in[e] && x >= least) w[e] = x;
                sum += w[e];
            }
        }
        return sum;
    };
    u64 mine = 0, part = 0;
    vectors(
        [&](int at, const Vec<T>& v) {
            u64 w[VEC];
            part += kept(at, v, w);
        },
        [&](int sc) {
            if (__any_sync(0xffffffffu, part != 0)) part = warp_sum_u64(part);
            if (lane == 0) sh.chunk[sc] = part;
            mine += part;
            part = 0;
        });
    __syncthreads();
    if (lane == 0) sh.warp_sum[warp] = mine;
    __syncthreads();
    if (tid == 0) {
        u64 s = 0;
        for (int w = 0; w < kWarpsS; ++w) s += sh.warp_sum[w];
        sh.sum = s;
    }
    cluster_sync_all();
    // (a rank's sum in each lane)
    const u64 sums = warp_scan_u64(lane < (int)C ? ld_cluster_u64(map_rank(&sh.sum, lane)) : 0, lane);
    const u64 all = __shfl_sync(0xffffffffu, sums, 31), upto = __shfl_sync(0xffffffffu, sums, (int)rank);
    const u64 own = sh.sum, before = upto - own;
    const u64 thr = threshold(all);
    if (warp == 0 && before <= thr && thr < before + own) {
        // the record it lies in, 32 at a time, then the chunk, then the element
        u64 at = before;
        int sc = 0;
        for (; sc < n_super; sc += 32) {
            const u64 s = sc + lane < n_super ? sh.chunk[sc + lane] : 0;
            const u64 inc = warp_scan_u64(s, lane);
            const unsigned hit = __ballot_sync(0xffffffffu, at + inc > thr);
            if (hit) {
                const int f = __ffs(hit) - 1;
                at += __shfl_sync(0xffffffffu, inc - s, f);
                sc += f;
                break;
            }
            at += __shfl_sync(0xffffffffu, inc, 31);
        }
        for (int k = 0; k < SUPER && sc < n_super && at <= thr; ++k) {
            const int i = (sc * SUPER + k) * 32 + lane;
            Vec<T> v;
            if constexpr (STREAM) v = fetch(i);
            else v = data[i];
            u64 w[VEC];
            const u64 s = kept(i, v, w);
            const u64 inc = warp_scan_u64(s, lane);
            u64 run = at + inc - s;
            if (run <= thr && thr < run + s) {
                int found = -1;
                float l = 0.f;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    run += w[e];
                    if (found < 0 && run > thr) {
                        found = e;
                        l = as_float(v.x[e]);
                    }
                }
                answer(first + i * VEC + found, l, all);
            }
            at += __shfl_sync(0xffffffffu, inc, 31);
        }
    }
    cluster_sync_all();  // no CTA leaves while another reads its shared memory
}

template <typename T, bool STREAM>
cudaError_t launch_one(const Args& a, int rows, int C, cudaStream_t st) {
    constexpr size_t own = (sizeof(Shared) + 15) / 16 * 16;
    // (the largest slice's bytes, whatever this call's: calls of two threads do not undo each other's)
    cudaError_t e = cudaFuncSetAttribute(sample_kernel<T, STREAM>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)(own + kSliceBytes));
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(sample_kernel<T, STREAM>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)rows * (unsigned)C, 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = own + (STREAM ? 0 : (size_t)a.slice * sizeof(T));
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = kPdlLaunch;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)C;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, sample_kernel<T, STREAM>, a);
}

template <typename T>
cudaError_t launch(Args a, int rows, int num_sms, cudaStream_t st) {
    constexpr int CHUNK = 32 * 16 / (int)sizeof(T);
    int C = 1;
    auto slice = [&] { return ((a.vocab + C - 1) / C + CHUNK - 1) / CHUNK * CHUNK; };
    // Long rows, 64 MB of them and more: read from global memory in every pass, by four CTAs a row (512 rows of 256206
    // in fp32: 575 us with mixed settings, 789 from shared memory; 64 rows by top-k 58 instead of 73, greedy 22 instead
    // of 34; one CTA a row took 796, eight 669).  Below that the passes from shared memory are the faster (64 rows in
    // bf16 by top-p: 126 instead of 148; 128 rows: equal).
    const bool aligned = ((reinterpret_cast<uintptr_t>(a.logits) | (uintptr_t)(a.ld * (long long)sizeof(T))) & 15u) == 0;
    if (aligned && slice() * (int)sizeof(T) > kSliceBytes && (long long)rows * a.vocab * (int)sizeof(T) >= 1LL << 26) {
        C = 4;
        a.slice = slice();
        return launch_one<T, true>(a, rows, C, st);
    }
    // Up to eight CTAs a row while they hold more than 64 KB each, so that two share an SM (64 rows in bf16 by top-p:
    // 125 us, with four CTAs of 128 KB 144), more where they could not hold it; while there are SMs to spare, larger
    // clusters down to 4096 entries a CTA.
    while (slice() * (int)sizeof(T) > (C < 8 ? kSliceBytes / 2 : kSliceBytes) ||
           (C < kMaxCluster && (long long)rows * C * 2 <= num_sms && a.vocab > 4096 * C))
        C *= 2;
    a.slice = slice();
    return launch_one<T, false>(a, rows, C, st);
}

int bad(const char* msg) { return set_error(NLLB_ATTN_EINVAL, msg); }

thread_local bool t_expire_next = false;

}  // namespace
}  // namespace nllb

extern "C" int nllb_sample_test_expire_next_wait(void) {
    nllb::t_expire_next = true;
    return NLLB_ATTN_OK;
}

extern "C" int nllb_sample(const nllb_sample_args* s, void* stream) {
    using namespace nllb;
    if (!s) return bad("args is NULL");
    if (s->dtype != NLLB_F32 && s->dtype != NLLB_F16 && s->dtype != NLLB_BF16)
        return bad("dtype must be NLLB_F32, NLLB_F16 or NLLB_BF16");
    if (s->rows < 0 || s->vocab < 1) return bad("rows >= 0 and vocab >= 1 required");
    if (s->vocab > NLLB_SAMPLE_MAX_VOCAB) return set_error(NLLB_ATTN_ECAPACITY, "vocab above NLLB_SAMPLE_MAX_VOCAB");
    if (s->rows > (1 << 26)) return set_error(NLLB_ATTN_ECAPACITY, "more rows than a call takes");
    if (s->rows == 0) return NLLB_ATTN_OK;
    if (!s->logits || !s->u || !s->out_tok) return bad("logits, u and out_tok are required");
    if (s->ld < s->vocab) return bad("ld must be at least vocab");
    const uintptr_t size = s->dtype == NLLB_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(s->logits) % size) return bad("logits must be aligned to their type");
    Args a = {};
    a.logits = s->logits, a.ld = s->ld, a.vocab = s->vocab;
    a.temperature = s->temperature, a.top_k = s->top_k, a.top_p = s->top_p, a.min_p = s->min_p, a.u = s->u;
    a.out_tok = s->out_tok, a.out_logp = s->out_logp;
    a.expire = t_expire_next;
    t_expire_next = false;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    int device = 0, num_sms = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&num_sms, cudaDevAttrMultiProcessorCount, device);
    if (e == cudaSuccess)
        e = s->dtype == NLLB_F32   ? launch<float>(a, s->rows, num_sms, st)
            : s->dtype == NLLB_F16 ? launch<__half>(a, s->rows, num_sms, st)
                                   : launch<__nv_bfloat16>(a, s->rows, num_sms, st);
    if (e != cudaSuccess) return set_error(NLLB_ATTN_ECUDA, std::string("nllb_sample: ") + cudaGetErrorString(e));
    return NLLB_ATTN_OK;
}
