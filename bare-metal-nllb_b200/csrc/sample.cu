// sample.cu -- nllb_sample: one token per row of logits by temperature, top-k,
// top-p and min-p, from a given uniform number (sm_100a).
//
//   w_i = exp((l_i - m) / T); the kept set is a prefix of the order (logit
//   falling, index rising), cut by a count, by a share of the weight and by a
//   least weight; the token is found by inverting the running sum of the kept
//   weights in index order.
//
// The bytes of the logits bound it, so a row is read once: the CTAs of a
// cluster hold its slices in shared memory and every later pass reads those.
// Nothing is sorted.  The border of the kept set is found by counting: a
// histogram over 2048 equal steps of (m - l) / T, its totals summed over the
// cluster through distributed shared memory, names the step the border lies
// in; the elements of that step are then told apart by their composite (order
// of the logit, index), 11 bits of what is left at a time, until one is left.
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

constexpr int kMaxCluster = 16;
constexpr int kMaxSlice = NLLB_SAMPLE_MAX_VOCAB / kMaxCluster;
constexpr int kMaxChunks = kMaxSlice / 128;  // fp32's chunks are the shortest

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
};

struct Shared {
    u64 mass[kBins];
    u64 tot_mass[kBins / 2];  // this CTA's share of the bins, summed over the cluster (two CTAs or more)
    uint32_t cnt[kBins];
    uint32_t tot_cnt[kBins / 2];
    double tab[64];            // 2^(j/64)
    u64 chunk[kMaxChunks];     // kept weight of each chunk of the slice
    u64 warp_sum[kWarpsS];
    u64 total, sum;            // of a scan; of this CTA's kept weight
    u64 found_before, found_value;
    uint32_t found_cnt;
    int found_bin;
    float best;                // this CTA's largest logit
    uint32_t key_lo, key_hi;   // this CTA's range of keys in the border step
    float red[kWarpsS];
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

// exp((l - m) / T) in units of 2^-kWeightBits.  y = 64 log2 of it is split as
// n + f, n a whole number and |f| <= 1/2; 2^(y/64) = 2^(n >> 6) *
// 2^((n & 63) / 64) * exp(f ln2 / 64), the middle factor from a table and the
// last by its series to the fifth power (Tang, 1989: the remainder is below
// 4e-17), all in fp64: a token's border may lie anywhere between its
// neighbours', and fp32 sums over 256206 tokens place it too coarsely.
__device__ __forceinline__ u64 weight(float l, float m, double md, double scale, const double* tab) {
    if (l == m) return 1ull << kWeightBits;
    const double y = ((double)l - md) * scale;
    if (!(y > -64.0 * (kWeightBits + 2))) return 0;
    const double magic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to a whole number
    const double t = y + magic;
    const int n = __double2loint(t);
    const double r = (y - (t - magic)) * (0.693147180559945309417 / 64.0);
    double e = fma(r, 1.0 / 120.0, 1.0 / 24.0);
    e = fma(r, e, 1.0 / 6.0);
    e = fma(r, e, 0.5);
    e = fma(r, e, 1.0);
    e = fma(r, e, 1.0);
    const double p2 = __hiloint2double((1023 + kWeightBits + (n >> 6)) << 20, 0);
    const double w = tab[n & 63] * e * p2;
    // w < 2^52: adding 2^52 rounds it to a whole number in the low bits
    return (u64)__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull;
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

template <typename T>
struct alignas(16) Vec {
    T x[16 / sizeof(T)];
};

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

// One cluster per row.
template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const Args a) {
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int VEC = 16 / (int)sizeof(T);
    constexpr int CHUNK = 32 * VEC;  // one vector per lane
    Shared& sh = *reinterpret_cast<Shared*>(smem);
    Vec<T>* data = reinterpret_cast<Vec<T>*>(smem + (sizeof(Shared) + 15) / 16 * 16);

    pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid < 64) sh.tab[tid] = exp2((double)tid / 64.0);
    pdl_wait_primary();

    const uint32_t C = cluster_size(), rank = cluster_ctarank();
    const int row = blockIdx.x / C;
    const int first = (int)rank * a.slice;  // the slice's first element
    const int n = min(a.slice, max(0, a.vocab - first));
    const int n_chunks = (n + CHUNK - 1) / CHUNK;
    const T* src = static_cast<const T*>(a.logits) + (long long)row * a.ld + first;

    // ---- the slice into shared memory, NaN as -inf, and its largest logit
    float best = -INFINITY;
    {
        const bool vec = (reinterpret_cast<uintptr_t>(src) & 15u) == 0;
#pragma unroll 4
        for (int i = tid; i < n_chunks * 32; i += kThreads) {
            Vec<T> v;
            if (vec && (i + 1) * VEC <= n) {
                *reinterpret_cast<uint4*>(&v) = __ldcs(reinterpret_cast<const uint4*>(src) + i);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) v.x[e] = i * VEC + e < n ? src[i * VEC + e] : minus_inf<T>();
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float l = as_float(v.x[e]);
                if (l != l) v.x[e] = minus_inf<T>();
                best = fmaxf(best, l);  // (fmaxf passes over NaN)
            }
            data[i] = v;
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) sh.red[warp] = best;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kWarpsS; ++w) best = fmaxf(best, sh.red[w]);
        sh.best = best;
    }
    cluster_sync_all();
    float m = -INFINITY;
    for (uint32_t z = 0; z < C; ++z) m = fmaxf(m, ld_cluster_f32(map_rank(&sh.best, z)));

    // ---- the row's settings
    float temp = a.temperature ? __ldg(a.temperature + row) : 1.0f;
    int k = a.top_k ? __ldg(a.top_k + row) : 0;
    float top_p = a.top_p ? __ldg(a.top_p + row) : 1.0f;
    float min_p = a.min_p ? __ldg(a.min_p + row) : 0.0f;
    float u = __ldg(a.u + row);
    const bool usable = m > -INFINITY && temp >= 0.0f && temp < INFINITY;
    if (!usable) {  // (uniform over the cluster)
        if (rank == 0 && tid == 0) {
            a.out_tok[row] = -1;
            if (a.out_logp) a.out_logp[row] = -INFINITY;
        }
        cluster_sync_all();
        return;
    }
    if (temp == 0.0f) temp = 1.0f, k = 1;  // the first of the order, whatever the weights
    temp = fmaxf(temp, 0x1p-100f);         // keeps the factors below finite
    const double md = m, scale = 64.0 * 1.4426950408889634074 / (double)temp;
    const float to_bin = (float)kBins / (kSpan * temp);
    // Step of the first histogram; steps rise as logits fall, in fp32 as well
    // as in exact arithmetic, since every operation rounds monotonically.
    auto step_of = [&](float l) -> int {
        if (l == m) return 0;
        const float d = (m - l) * to_bin;
        return d < (float)kBins ? (int)d : kBins;
    };
    auto wt = [&](float l) { return weight(l, m, md, scale, sh.tab); };

    // f(l, local index) for every element of the slice
    auto each = [&](auto&& f) {
        for (int ch = warp; ch < n_chunks; ch += kWarpsS) {
            const Vec<T> v = data[ch * 32 + lane];
#pragma unroll
            for (int e = 0; e < VEC; ++e) f(as_float(v.x[e]), (ch * 32 + lane) * VEC + e);
        }
    };
    auto composite = [&](float l, int i) { return ((u64)order_key(l) << kIndexBits) | (u64)(first + i); };

    // Sums the cluster's histograms and finds the first bin at which the sum of
    // the values (counts, or masses) up to and including it, from `base` on,
    // reaches target(sum of all).  All CTAs compute the same; found_bin -1 if
    // no bin does.
    auto search = [&](bool by_mass, u64 base, auto&& target) {
        cluster_sync_all();
        const int share = kBins / (int)C;
        if (C > 1) {
            for (int b = tid; b < share; b += kThreads) {
                uint32_t c = 0;
                u64 w = 0;
                for (uint32_t z = 0; z < C; ++z) {
                    uint32_t x;
                    asm volatile("ld.shared::cluster.u32 %0, [%1];"
                                 : "=r"(x) : "r"(map_rank(&sh.cnt[rank * share + b], z)) : "memory");
                    c += x;
                    if (by_mass) w += ld_cluster_u64(map_rank(&sh.mass[rank * share + b], z));
                }
                sh.tot_cnt[b] = c;
                if (by_mass) sh.tot_mass[b] = w;
            }
            cluster_sync_all();
        }
        constexpr int PER = kBins / kThreads;
        uint32_t c[PER];
        u64 v[PER], mine = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int b = tid * PER + i;
            if (C > 1) {
                const uint32_t z = (uint32_t)(b / share), at = (uint32_t)(b % share);
                asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(c[i]) : "r"(map_rank(&sh.tot_cnt[at], z)) : "memory");
                v[i] = by_mass ? ld_cluster_u64(map_rank(&sh.tot_mass[at], z)) : (u64)c[i];
            } else {
                c[i] = sh.cnt[b];
                v[i] = by_mass ? sh.mass[b] : (u64)c[i];
            }
            mine += v[i];
        }
        const u64 inc = warp_scan_u64(mine, lane);
        if (lane == 31) sh.warp_sum[warp] = inc;
        if (tid == 0) sh.found_bin = -1;
        __syncthreads();
        u64 before = base, all = base;
#pragma unroll
        for (int w = 0; w < kWarpsS; ++w) {
            const u64 x = sh.warp_sum[w];
            if (w < warp) before += x;
            all += x;
        }
        before += inc - mine;
        const u64 want = target(all);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (before < want && want <= before + v[i]) {
                sh.found_bin = tid * PER + i;
                sh.found_cnt = c[i];
                sh.found_before = before;
            }
            before += v[i];
        }
        if (tid == 0) sh.total = all;
        __syncthreads();
        return want;
    };
    auto clear = [&](bool by_mass) {
        for (int b = tid; b < kBins; b += kThreads) {
            sh.cnt[b] = 0;
            if (by_mass) sh.mass[b] = 0;
        }
        __syncthreads();
    };

    // The composite up to which the elements (of those <= limit) are kept:
    // the first at which the count, or the weight, of the elements up to it
    // reaches target(whole).  Unchanged limit if none does.
    auto border = [&](bool by_mass, u64 limit, auto&& target) -> u64 {
        clear(by_mass);
        each([&](float l, int i) {
            const int b = step_of(l);
            if (b < kBins && composite(l, i) <= limit) {
                atomicAdd(&sh.cnt[b], 1u);
                if (by_mass) atomicAdd(&sh.mass[b], wt(l));
            }
        });
        const u64 want = search(by_mass, 0, target);
        const int b = sh.found_bin;
        if (b < 0) return limit;
        u64 base = sh.found_before;
        bool one = sh.found_cnt == 1;
        // the keys of that step
        uint32_t lo = 0xffffffffu, hi = 0;
        each([&](float l, int i) {
            if (step_of(l) == b && composite(l, i) <= limit) {
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
            uint32_t x, y;
            asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(x) : "r"(map_rank(&sh.key_lo, z)) : "memory");
            asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(y) : "r"(map_rank(&sh.key_hi, z)) : "memory");
            lo = min(lo, x);
            hi = max(hi, y);
        }
        u64 from = (u64)lo << kIndexBits, to = ((u64)hi << kIndexBits) | ((1u << kIndexBits) - 1u);
        while (!one) {
            to = to < limit ? to : limit;
            const int bits = 64 - __clzll((long long)(to - from));
            const int shift = max(0, bits - kBinBits);
            clear(by_mass);
            each([&](float l, int i) {
                const u64 c = composite(l, i);
                if (c >= from && c <= to) {
                    const int x = (int)((c - from) >> shift);
                    atomicAdd(&sh.cnt[x], 1u);
                    if (by_mass) atomicAdd(&sh.mass[x], wt(l));
                }
            });
            search(by_mass, base, [&](u64) { return want; });
            base = sh.found_before;
            from += (u64)sh.found_bin << shift;
            to = from + ((1ull << shift) - 1ull);
            one = sh.found_cnt == 1 || shift == 0;
            __syncthreads();  // the next search's writes wait for these reads
        }
        return to < limit ? to : limit;
    };

    u64 limit = ~0ull;
    if (k > 0 && k < a.vocab) limit = border(false, limit, [&](u64) { return (u64)k; });
    if (top_p < 1.0f)
        limit = border(true, limit, [&](u64 all) {
            const double t = ceil((double)fmaxf(top_p, 0.0f) * (double)all);
            const u64 want = t < (double)all ? (u64)t : all;
            return want > 0 ? want : 1;
        });
    u64 least = 1;
    if (min_p > 0.0f) {
        const double t = ceil((double)fminf(min_p, 1.0f) * (double)(1ull << kWeightBits));
        least = t > 1.0 ? (u64)t : 1;
    }
    auto kept = [&](float l, int i) -> u64 {
        if (composite(l, i) > limit) return 0;
        const u64 w = wt(l);
        return w >= least ? w : 0;
    };

    // ---- the kept weight of each chunk, of this CTA, of the row
    u64 mine = 0;
    for (int ch = warp; ch < n_chunks; ch += kWarpsS) {
        const Vec<T> v = data[ch * 32 + lane];
        u64 s = 0;
#pragma unroll
        for (int e = 0; e < VEC; ++e) s += kept(as_float(v.x[e]), (ch * 32 + lane) * VEC + e);
        s = warp_sum_u64(s);
        if (lane == 0) sh.chunk[ch] = s;
        mine += s;
    }
    __syncthreads();
    if (lane == 0) sh.warp_sum[warp] = mine;
    __syncthreads();
    if (tid == 0) {
        u64 s = 0;
        for (int w = 0; w < kWarpsS; ++w) s += sh.warp_sum[w];
        sh.sum = s;
    }
    cluster_sync_all();
    u64 all = 0, before = 0, own = 0;
    for (uint32_t z = 0; z < C; ++z) {
        const u64 s = ld_cluster_u64(map_rank(&sh.sum, z));
        if (z < rank) before += s;
        if (z == rank) own = s;
        all += s;
    }
    u = u > 0.0f ? u : 0.0f;  // (NaN too)
    const double t = fmin((double)u, 1.0) * (double)all;
    const u64 thr = t < (double)all ? min((u64)t, all - 1) : all - 1;  // the first running sum above thr
    if (warp == 0 && before <= thr && thr < before + own) {
        // the chunk, 32 at a time, then the element within it
        u64 at = before;
        int ch0 = 0;
        for (;; ch0 += 32) {
            const u64 s = ch0 + lane < n_chunks ? sh.chunk[ch0 + lane] : 0;
            const u64 inc = warp_scan_u64(s, lane);
            const unsigned hit = __ballot_sync(0xffffffffu, at + inc > thr);
            if (hit) {
                const int f = __ffs(hit) - 1;
                at += __shfl_sync(0xffffffffu, inc - s, f);
                ch0 += f;
                break;
            }
            at += __shfl_sync(0xffffffffu, inc, 31);
        }
        const Vec<T> v = data[ch0 * 32 + lane];
        u64 w[VEC], s = 0;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            w[e] = kept(as_float(v.x[e]), (ch0 * 32 + lane) * VEC + e);
            s += w[e];
        }
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
            a.out_tok[row] = first + (ch0 * 32 + lane) * VEC + found;
            if (a.out_logp) {
                const double x = l == m ? 0.0 : ((double)l - md) / (double)temp;
                a.out_logp[row] = (float)(x - log((double)all * (1.0 / (double)(1ull << kWeightBits))));
            }
        }
    }
    cluster_sync_all();  // no CTA leaves while another reads its shared memory
}

template <typename T>
size_t smem_bytes(int slice) {
    return (sizeof(Shared) + 15) / 16 * 16 + (size_t)slice * sizeof(T);
}

template <typename T>
cudaError_t launch(Args a, int rows, cudaStream_t st) {
    constexpr int CHUNK = 32 * 16 / (int)sizeof(T);
    int C = 1;
    while (C < kMaxCluster && a.vocab > 8192 * C) C *= 2;
    a.slice = ((a.vocab + C - 1) / C + CHUNK - 1) / CHUNK * CHUNK;
    const size_t smem = smem_bytes<T>(a.slice);
    // (the largest slice's bytes, whatever this call's: calls of two threads do not undo each other's)
    cudaError_t e = cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)smem_bytes<T>(kMaxSlice));
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)rows * (unsigned)C, 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = kPdlLaunch;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)C;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, sample_kernel<T>, a);
}

int bad(const char* msg) { return set_error(NLLB_ATTN_EINVAL, msg); }

}  // namespace
}  // namespace nllb

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
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const cudaError_t e = s->dtype == NLLB_F32   ? launch<float>(a, s->rows, st)
                          : s->dtype == NLLB_F16 ? launch<__half>(a, s->rows, st)
                                                 : launch<__nv_bfloat16>(a, s->rows, st);
    if (e != cudaSuccess) return set_error(NLLB_ATTN_ECUDA, std::string("nllb_sample: ") + cudaGetErrorString(e));
    return NLLB_ATTN_OK;
}
