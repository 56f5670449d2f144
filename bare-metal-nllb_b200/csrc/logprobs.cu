// logprobs.cu -- log-probabilities of given tokens, the entropy of each row of
// logits and its likeliest tokens (nllb_logprobs, sm_100a).
//
// With m the largest logit, n the number of those equal to it, and over the others
// y_i = (l_i - m) log2(e),
//   z = sum 2^y_i,   s = sum 2^y_i y_i:
//   log p_t = l_t - m - ln n - log1p(z / n),
//   H = ln n + log1p(z / n) - ln2 s / (n + z).
// The largest are counted apart from the sums: beside their weight of 1 a sum in
// fp32 would lose what is below 2^-24 of it, and the entropy of a row that one
// token dominates is of that size; as they stand no term cancels another.
//
// The bytes of the logits bound it: they are read once, each thread keeping a
// running n, z and s of its stripe of 16-byte vectors beside its warp's m; they
// are joined in a fixed order: across the warp, the CTA and the cluster that
// shares the row.
//
// For the likeliest tokens a thread notes, beside the sums, its stripe's largest
// logit, the vector that it came from and the largest of the other vectors: a few
// selections a vector, hidden behind the bytes.  Of n tokens in the
// order (falling logit, rising index) each lies in one of the n stripes whose
// maxima come first in that order -- n of them are ahead of any other stripe's
// -- so of those stripes the vectors that hold the maxima are read again, and
// the other vectors only if the largest of them is not below the n-th maximum.
// What is not behind that goes through sorted lists of 32 in registers.  A row
// with many equal or rising logits takes more batches of 32, never another way.
//
// Measured (device time, short replays; in long runs 7 to 10 % more): 1000 rows of
// 256206 in fp32 with 20 tokens 161 us (6.4 TB/s), 600 rows in bf16 without 55 us
// (5.6 TB/s; the exponentials alone would take 34); one row with 8 tokens 11 us, the
// latency of a cluster of eight (7.5 without tokens) and of two merges of lists.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <string>

#include "nllb_translate.h"
#include "rows.cuh"

namespace nllb {
int set_error(int status, const std::string& msg);  // nllb_attn.cu

namespace {

using u64 = unsigned long long;

constexpr int kThreads = 256, kWarps = kThreads / 32, kPerSm = 4;
constexpr int kUnroll = 4;         // 16-byte vectors that a thread takes together, while as many are on their way
constexpr int kMaxCluster = 2 * kWarps;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNoWeight = -200.0f;  // 2^-200 is 0 in fp32
// A largest scaled logit of this size and more: what it was rounded by could be more than an exponent holds, and different
// logits are at least 32 apart.
constexpr float kFar = 0x1.8p28f;

struct Args {
    const void* logits;
    long long ld;
    int vocab, top_n;
    const int* target;
    float *out_logp, *out_entropy;
    int* out_top_tok;
    float* out_top_logp;
};

// A set of tokens: their largest logit, how many there are of it, and the others' sums of 2^y and 2^y y, where
// y = l log2(e) - M with M = m log2(e) rounded: off by what M was rounded by, alike for all.
struct __align__(16) State {
    float m, n, z, s;
};

struct Shared {
    State warp[kWarps];
    State cta;
    u64 list[kWarps][32];
    u64 kept[kWarps][64];
    float second[kThreads];
};

// Weight 2^y, y <= 0 (or what infinities and NaN make of it): below kNoWeight, and for NaN, none.
__device__ __forceinline__ float weigh(float& y) {
    y = fmaxf(y, kNoWeight);  // (NaN: kNoWeight)
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(y));
    return e;
}

// M = m log2(e), rounded (never part of a fused operation), and what it is short by.
__device__ __forceinline__ float scaled(float m) { return __fmul_rn(m, kLog2e); }
__device__ __forceinline__ float rounded_off(float m) { return fmaf(m, kLog2e, -scaled(m)); }

// The state as others of a larger m: all in its sums.  (Nothing is left where it lies too far behind, and sums beside a
// maximum beyond kFar, which may be infinite, do not count.)
__device__ __forceinline__ void settle(State& st, float m) {
    float d = scaled(st.m) - scaled(m);
    if (!(d > kNoWeight)) {
        st.n = st.z = st.s = 0.f;
    } else {
        float r = rounded_off(st.m);
        const float w = st.n * weigh(r), f = weigh(d);
        st.z += w;
        st.s = f * fmaf(st.z, d, fmaf(w, r, st.s));
        st.z *= f;
        st.n = 0.f;
    }
    st.m = m;
}

__device__ __forceinline__ State join(State a, State b) {
    const float m = fmaxf(a.m, b.m);
    if (a.m < m) settle(a, m);
    if (b.m < m) settle(b, m);
    return {m, a.n + b.n, a.z + b.z, a.s + b.s};
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
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// The largest of a vector's logits (NaN are passed over).
template <typename T>
__device__ __forceinline__ float largest(uint4 u) {
    if constexpr (std::is_same<T, float>::value) {
        return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
    } else {
        using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
        auto as = [](uint32_t& w) { return *reinterpret_cast<T2*>(&w); };
        const T2 m = __hmax2(__hmax2(as(u.x), as(u.y)), __hmax2(as(u.z), as(u.w)));
        if constexpr (std::is_same<T, __half>::value) return fmaxf(__low2float(m), __high2float(m));
        else return fmaxf(__low2float(m), __high2float(m));
    }
}

// Bits that order like the logits (-0 as +0, NaN as -inf).
__device__ __forceinline__ uint32_t order_of(float l) {
    const uint32_t b = __float_as_uint(isnan(l) ? -INFINITY : l + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
// The order of falling logits, then rising indices.
__device__ __forceinline__ u64 order_key(float l, uint32_t index) { return (u64)order_of(l) << 32 | (~index); }
__device__ __forceinline__ uint32_t key_index(u64 key) { return ~(uint32_t)key; }
constexpr uint32_t kLeastOrder = 0x007fffffu;                           // -inf
constexpr u64 kNothing = (u64)kLeastOrder << 32 | 0xffffffffull;        // the keys up to it are not listed

// A warp's 32 keys in falling order.
__device__ __forceinline__ u64 clean(u64 x, int lane, int from, int up) {
#pragma unroll
    for (int j = from; j > 0; j >>= 1) {
        const u64 y = __shfl_xor_sync(0xffffffffu, x, j);
        const bool first = ((lane & j) == 0) == ((lane & up) == 0);
        x = (x > y) == first ? x : y;
    }
    return x;
}
__device__ __forceinline__ u64 sort32(u64 x, int lane) {
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1) x = clean(x, lane, k / 2, k);
    return x;
}
// The first 32 of two sorted lists.
__device__ __forceinline__ u64 merge32(u64 a, u64 b, int lane) {
    const u64 r = __shfl_sync(0xffffffffu, b, 31 - lane);
    return clean(a > r ? a : r, lane, 16, 32);
}
// The first 32 of the sorted lists of `n` warps (a power of two), in warp 0.
__device__ __forceinline__ u64 merge_warps(Shared& sh, u64 x, int n, int warp, int lane) {
    for (int half = n / 2; half > 0; half >>= 1) {
        __syncthreads();
        if (warp >= half && warp < 2 * half) sh.list[warp][lane] = x;
        __syncthreads();
        if (warp < half) x = merge32(x, sh.list[warp + half][lane], lane);
    }
    return x;
}

template <typename T>
__device__ __forceinline__ float to_float(T x) {
    if constexpr (std::is_same<T, float>::value) return x;
    else if constexpr (std::is_same<T, __half>::value) return __half2float(x);
    else return __bfloat162float(x);
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads, kPerSm) logprobs_kernel(const Args a, int C) {
    constexpr int VEC = 16 / (int)sizeof(T);
    __shared__ Shared sh;
    pdl_launch_dependents();
    pdl_wait_primary();

    const int rank = blockIdx.x % C, row = blockIdx.x / C;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int target = a.target ? ld_coherent(a.target + row) : 0;
    if (target < 0) {  // (the same in the whole cluster)
        if (rank == 0) {
            if (tid == 0) {
                if (a.out_logp) a.out_logp[row] = 0.f;
                if (a.out_entropy) a.out_entropy[row] = 0.f;
            }
            if (TOP && tid < a.top_n) {
                a.out_top_tok[(long long)row * a.top_n + tid] = -1;
                a.out_top_logp[(long long)row * a.top_n + tid] = -INFINITY;
            }
        }
        return;
    }
    const T* src = static_cast<const T*>(a.logits) + row * a.ld;
    // single elements up to the first 16-byte boundary and behind the last one, vectors between them
    const int head = min(a.vocab, (int)((16 - (reinterpret_cast<uintptr_t>(src) & 15)) & 15) / (int)sizeof(T));
    const int n_vec = (a.vocab - head) / VEC, tail = head + n_vec * VEC;
    const int n_single = rank == 0 ? head + a.vocab - tail : 0;  // rank 0's
    auto single = [&](int i) { return i < head ? i : tail + i - head; };
    const uint4* vec = reinterpret_cast<const uint4*>(src + head);
    const int per = (n_vec + C - 1) / C, v_end = min(n_vec, (rank + 1) * per), v_first = min(n_vec, rank * per);

    float m = -INFINITY;  // the warp's
    int n = 0;
    float2 z[2], sy[2];   // in four chains
    z[0] = z[1] = sy[0] = sy[1] = make_float2(0.f, 0.f);
    auto lane_state = [&] {
        return State{m, (float)n, (z[0].x + z[0].y) + (z[1].x + z[1].y), (sy[0].x + sy[0].y) + (sy[1].x + sy[1].y)};
    };
    // The largest logit of this batch in this lane, `t`: whether the warp has one as large as its m, or a larger one, which
    // is its m from now on.
    auto rises = [&](float t) {
        if (!__any_sync(0xffffffffu, t >= m && t > -INFINITY)) return false;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
        if (t > m) {
            State st = lane_state();
            settle(st, t);
            m = t, n = 0;
            z[0] = make_float2(st.z, 0.f), sy[0] = make_float2(st.s, 0.f), z[1] = sy[1] = make_float2(0.f, 0.f);
        }
        return true;
    };
    float best = -INFINITY;
    uint32_t best_at = 0xffffffffu;  // the stripe's first vector that holds its maximum
    float second = -INFINITY;        // the largest of its other vectors' maxima
    // (past the end: -inf in every element, no weight and no maximum)
    constexpr uint32_t none = std::is_same<T, float>::value ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
    auto load = [&](uint4 (&u)[kUnroll], int v) {
#pragma unroll
        for (int k = 0; k < kUnroll; ++k)
            u[k] = v + k * kThreads < v_end ? ld_coherent(vec + v + k * kThreads) : make_uint4(none, none, none, none);
    };
    auto batch = [&](const uint4 (&u)[kUnroll], int at) {
        float top[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            top[k] = largest<T>(u[k]);
            if constexpr (TOP) {
                second = fmaxf(second, fminf(best, top[k]));
                if (top[k] > best) best = top[k], best_at = at + k * kThreads;
            }
        }
        auto sum = [&](auto largest_among) {  // (whether the warp's m is among the batch's logits)
            const float2 off = make_float2(-scaled(m), -scaled(m)), scale = make_float2(kLog2e, kLog2e);
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) {
                float x[VEC];
                rows_unpack<T>(u[k], x);
#pragma unroll
                for (int e = 0; e < VEC; e += 2) {
                    float2 y = fma2(make_float2(x[e], x[e + 1]), scale, off), w;
                    w.x = weigh(y.x), w.y = weigh(y.y);
                    if constexpr (decltype(largest_among)::value) {
                        if (x[e] == m) w.x = 0.f, ++n;
                        if (x[e + 1] == m) w.y = 0.f, ++n;
                    }
                    z[(e >> 1) & 1] = add2(z[(e >> 1) & 1], w);
                    sy[(e >> 1) & 1] = fma2(w, y, sy[(e >> 1) & 1]);
                }
            }
        };
        if (rises(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])))) sum(std::true_type());
        else sum(std::false_type());
    };
    static_assert(kUnroll == 4, "four vectors together");
    {
        uint4 u[kUnroll], v[kUnroll];
        constexpr int STEP = kUnroll * kThreads;
        int at = v_first + tid;
        const int last = v_end - warp * 32 + tid;  // (the same turns for a whole warp)
        load(u, at);
        while (at < last) {
            load(v, at + STEP);
            batch(u, at);
            at += STEP;
            if (at >= last) break;
            load(u, at + STEP);
            batch(v, at);
            at += STEP;
        }
    }
    if (n_single > 0) {  // (fewer than 32)
        const float l = tid < n_single ? to_float(ld_coherent(src + single(tid))) : -INFINITY;
        rises(l);
        float y = fmaf(l, kLog2e, -scaled(m)), w = weigh(y);
        if (l == m) w = 0.f, n += tid < n_single;
        z[0].x += w;
        sy[0].x = fmaf(w, y, sy[0].x);
    }

    // ---- the row's state
    State st = lane_state();
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        st.n += __shfl_xor_sync(0xffffffffu, st.n, o);
        st.z += __shfl_xor_sync(0xffffffffu, st.z, o);
        st.s += __shfl_xor_sync(0xffffffffu, st.s, o);
    }
    if (lane == 0) sh.warp[warp] = st;
    u64 list = 0;
    if constexpr (TOP) {
        // the stripes whose maxima come first, by the index of the vector's first element
        sh.second[tid] = second;
        u64 key = best_at == 0xffffffffu ? 0 : order_key(best, (uint32_t)head + best_at * VEC);
        key = merge_warps(sh, sort32(key, lane), kWarps, warp, lane);
        __syncthreads();
        if (warp == 0) sh.list[0][lane] = key;
    }
    __syncthreads();
    if (warp == 0) {
        State w = lane < kWarps ? sh.warp[lane] : State{-INFINITY, 0.f, 0.f, 0.f};
#pragma unroll
        for (int o = kWarps / 2; o > 0; o >>= 1) {
            State b;
            b.m = __shfl_xor_sync(0xffffffffu, w.m, o);
            b.n = __shfl_xor_sync(0xffffffffu, w.n, o);
            b.z = __shfl_xor_sync(0xffffffffu, w.z, o);
            b.s = __shfl_xor_sync(0xffffffffu, w.s, o);
            w = join(w, b);
        }
        if (lane == 0) sh.cta = w;
    }
    if constexpr (TOP) {
        const u64 bar = sh.list[0][a.top_n - 1];  // nothing behind it is among the first (0: fewer stripes)
        const float least = logit_of((uint32_t)(bar >> 32));  // (bar 0: NaN)
        u64* const kept = sh.kept[warp];
        int n_kept = 0;
        // this lane's element, of the vector whose first element gave `key`; 32 at a time go into the list
        auto take = [&](u64 key, int further, bool there) {
            const bool in = there && key >= bar && key > kNothing;
            const unsigned who = __ballot_sync(0xffffffffu, in);
            if (who == 0) return;
            if (in) kept[n_kept + __popc(who & ((1u << lane) - 1u))] = key - further;
            n_kept += __popc(who);
            __syncwarp();
            if (n_kept >= 32) {
                n_kept -= 32;
                list = merge32(list, sort32(kept[n_kept + lane], lane), lane);
                __syncwarp();
            }
        };
        // the vectors that hold the stripes' maxima: an element to a lane
        static_assert(kWarps * 32 >= NLLB_LOGPROBS_MAX_TOP * VEC, "one round");
        if (warp * 32 < a.top_n * VEC) {
            const int i = tid / VEC, e = tid % VEC;
            const u64 stripe = i < a.top_n ? sh.list[0][i] : 0;
            const bool there = stripe > kNothing;
            const float l = there ? to_float(ld_coherent(src + key_index(stripe) + e)) : 0.f;
            take(order_key(l, key_index(stripe)), e, there);
        }
        // the others of a stripe, where one of them may be among the first too
        for (int i = warp; i < a.top_n; i += kWarps) {
            const u64 stripe = sh.list[0][i];
            if (stripe <= kNothing) break;
            const int found = (int)(key_index(stripe) - head) / VEC, t = (found - v_first) % kThreads;
            if (sh.second[t] < least) continue;
            const int first = v_first + t, n = (v_end - first + kThreads - 1) / kThreads;
            for (int k0 = 0; k0 < n; k0 += 32 * kUnroll) {
                uint4 u[kUnroll];
#pragma unroll
                for (int j = 0; j < kUnroll; ++j) {
                    const int k = k0 + 32 * j + lane;
                    u[j] = ld_coherent(vec + first + min(k, n - 1) * kThreads);
                }
#pragma unroll
                for (int j = 0; j < kUnroll; ++j) {
                    const int k = k0 + 32 * j + lane;
                    const bool there = k < n && first + k * kThreads != found;
                    const uint32_t at = (uint32_t)head + (first + k * kThreads) * VEC;
                    if (!__any_sync(0xffffffffu, there && !(largest<T>(u[j]) < least))) continue;
                    float x[VEC];
                    rows_unpack<T>(u[j], x);
                    // (an element stands behind the bar's vector, as its own vector does)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) take(order_key(x[e], at), e, there);
                }
            }
        }
        if (warp == kWarps - 1 && n_single > 0)
            take(lane < n_single ? order_key(to_float(ld_coherent(src + single(lane))), single(lane)) : 0, 0, lane < n_single);
        if (n_kept > 0) list = merge32(list, sort32(lane < n_kept ? kept[lane] : 0, lane), lane);
        list = merge_warps(sh, list, kWarps, warp, lane);
        if (C > 1) {
            __syncthreads();
            if (warp == 0) sh.list[0][lane] = list;
        }
    }
    if (C > 1) cluster_sync_all();
    else __syncthreads();
    State all = sh.cta;
    if (C > 1) {  // (the same order in every CTA)
        all = {-INFINITY, 0.f, 0.f, 0.f};
        for (int r = 0; r < C; ++r) {
            const float4 f = ld_cluster_f4(map_rank(&sh.cta, r));
            all = join(all, State{f.x, f.y, f.z, f.w});
        }
        if constexpr (TOP) {
            if (rank == 0) {
                auto of_rank = [&](int r) {
                    const uint32_t at = map_rank(&sh.list[0][lane], r);
                    return (u64)(uint32_t)ld_cluster_s32(at + 4) << 32 | (uint32_t)ld_cluster_s32(at);
                };
                list = warp < C ? of_rank(warp) : 0;
                if (C > kWarps) list = merge32(list, of_rank(warp + kWarps), lane);
                __syncthreads();
                list = merge_warps(sh, list, min(C, kWarps), warp, lane);
            }
        }
    }
    if (rank == 0 && warp == 0) {
        // A largest logit that is infinite or far out: those equal to it share all the weight.
        const bool none = all.m == -INFINITY, far = !(fabsf(scaled(all.m)) < kFar);
        float r = far ? 0.f : rounded_off(all.m), back = -r;
        const float f = weigh(back);  // (the sums without what M was rounded by)
        const float z = far ? 0.f : f * all.z, sy = far ? 0.f : f * fmaf(-r, all.z, all.s);
        const float log_z = logf(all.n) + log1pf(z / all.n);
        auto logp = [&](float l) {
            if (none || !(l > -INFINITY)) return -INFINITY;
            if (far) return (l == all.m ? 0.f : l - all.m) - log_z;
            // (a token far behind, whose scaled difference may leave fp32: what M was rounded by is nothing beside it)
            const float y = fmaf(l, kLog2e, -scaled(all.m));
            return l == all.m ? -log_z : y > -1e6f ? kLn2 * (y - r) - log_z : (l - all.m) - log_z;
        };
        if (lane == 0) {
            if (a.out_logp) a.out_logp[row] = target < a.vocab ? logp(to_float(ld_coherent(src + target))) : -INFINITY;
            if (a.out_entropy) a.out_entropy[row] = none ? 0.f : log_z - kLn2 * (sy / (all.n + z));
        }
        if (TOP && lane < a.top_n) {
            const bool there = list > kNothing;
            a.out_top_tok[(long long)row * a.top_n + lane] = there ? (int)key_index(list) : -1;
            a.out_top_logp[(long long)row * a.top_n + lane] = there ? logp(logit_of((uint32_t)(list >> 32))) : -INFINITY;
        }
    }
    if (C > 1) cluster_sync_all();  // no CTA leaves while another reads its shared memory
}

void configure(cudaLaunchConfig_t& cfg, cudaLaunchAttribute (&attr)[2], int rows, int C, cudaStream_t st) {
    cfg.gridDim = dim3((unsigned)rows * (unsigned)C, 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = kPdlLaunch;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)C;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = C > 1 ? 2 : 1;
}

// CTAs of a cluster at most on this device: kMaxCluster where one of as many, beyond the portable size, has room there (a part
// of a GPU may have none; asked for once), else 8.
template <typename T, bool TOP>
int widest(int device) {
    static std::atomic<int> known[64];
    if (device > 63) return 8;
    int c = known[device].load(std::memory_order_relaxed);
    if (c == 0) {
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr[2];
        configure(cfg, attr, 1, kMaxCluster, nullptr);
        int n = 0;
        cudaError_t e = cudaFuncSetAttribute(logprobs_kernel<T, TOP>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&n, logprobs_kernel<T, TOP>, &cfg);
        if (e != cudaSuccess) (void)cudaGetLastError(), n = 0;
        c = n > 0 ? kMaxCluster : 8;
        known[device].store(c, std::memory_order_relaxed);
    }
    return c;
}

template <typename T, bool TOP>
cudaError_t launch(const Args& a, int rows, int device, int num_sms, cudaStream_t st) {
    // CTAs of a row, by what a call takes: the stream, at 50 bytes a nanosecond of a CTA alone and 6500 of them all, and what
    // follows it, more where a cluster has to meet (1000 rows of 256206 in fp32 without tokens 154 us by one CTA each, 166 by two;
    // one row with 8 tokens 21, 16, 12, 11 and 11 us by 1, 2, 4, 8 and 16; one of 820001 in bf16 49, 29, 19, 14.4 and 13.7).
    const double bytes = (double)a.vocab * sizeof(T), slots = (double)kPerSm * num_sms;
    int C = 1;
    double least = 1e300;
    for (int c = 1; c <= kMaxCluster; c *= 2) {
        const double at_work = std::min((double)rows * c, slots);
        const double t = (double)rows * c / at_work * (bytes / c / std::min(50.0, 6500.0 / at_work) + (c == 1 ? 4000.0 : 6000.0 + 250.0 * c));
        if (t < least && (c <= 8 || c <= widest<T, TOP>(device))) least = t, C = c;
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    configure(cfg, attr, rows, C, st);
    return cudaLaunchKernelEx(&cfg, logprobs_kernel<T, TOP>, a, C);
}

int bad(const char* msg) { return set_error(NLLB_ATTN_EINVAL, msg); }

}  // namespace
}  // namespace nllb

extern "C" int nllb_logprobs(const nllb_logprobs_args* s, void* stream) {
    using namespace nllb;
    if (!s) return bad("args is NULL");
    if (s->dtype != NLLB_F32 && s->dtype != NLLB_F16 && s->dtype != NLLB_BF16)
        return bad("dtype must be NLLB_F32, NLLB_F16 or NLLB_BF16");
    if (s->rows < 0 || s->vocab < 1) return bad("rows >= 0 and vocab >= 1 required");
    if (s->vocab > (1 << 30) || s->rows > (1 << 26)) return set_error(NLLB_ATTN_ECAPACITY, "more logits than a call takes");
    if (s->top_n < 0) return bad("top_n must not be negative");
    if (s->top_n > NLLB_LOGPROBS_MAX_TOP) return set_error(NLLB_ATTN_ECAPACITY, "top_n above NLLB_LOGPROBS_MAX_TOP");
    if (s->rows == 0) return NLLB_ATTN_OK;
    if (!s->logits) return bad("logits is required");
    if (s->out_logp && !s->target) return bad("out_logp needs target");
    if (s->top_n > 0 && (!s->out_top_tok || !s->out_top_logp)) return bad("top_n needs out_top_tok and out_top_logp");
    if (!s->out_logp && !s->out_entropy && s->top_n == 0) return bad("no output is asked for");
    if (s->ld < s->vocab) return bad("ld must be at least vocab");
    const uintptr_t size = s->dtype == NLLB_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(s->logits) % size) return bad("logits must be aligned to their type");
    Args a = {};
    a.logits = s->logits, a.ld = s->ld, a.vocab = s->vocab, a.top_n = s->top_n, a.target = s->target;
    a.out_logp = s->out_logp, a.out_entropy = s->out_entropy;
    a.out_top_tok = s->out_top_tok, a.out_top_logp = s->out_top_logp;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    int device = 0, num_sms = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&num_sms, cudaDevAttrMultiProcessorCount, device);
    if (e == cudaSuccess)
        switch (s->dtype) {
            case NLLB_F32: e = s->top_n ? launch<float, true>(a, s->rows, device, num_sms, st) : launch<float, false>(a, s->rows, device, num_sms, st); break;
            case NLLB_F16: e = s->top_n ? launch<__half, true>(a, s->rows, device, num_sms, st) : launch<__half, false>(a, s->rows, device, num_sms, st); break;
            default: e = s->top_n ? launch<__nv_bfloat16, true>(a, s->rows, device, num_sms, st) : launch<__nv_bfloat16, false>(a, s->rows, device, num_sms, st);
        }
    if (e != cudaSuccess) return set_error(NLLB_ATTN_ECUDA, std::string("nllb_logprobs: ") + cudaGetErrorString(e));
    return NLLB_ATTN_OK;
}
