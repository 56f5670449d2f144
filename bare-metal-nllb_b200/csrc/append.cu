// append.cu -- new keys and values into a paged cache, queries and keys turned
// by their positions on the way (nllb_attn_append, sm_100a).
//
// Pair i of a query or key head, (x_i, x_{i + n}) or (x_{2i}, x_{2i+1}), n of
// them in the head's first 2n values, becomes
//   (a cos p f_i - b sin p f_i,  b cos p f_i + a sin p f_i),
// p the token's position, f_i a frequency.  The angle is taken as turns in 64
// bits, p f_i / 2 pi, of which the part within half a turn goes on in 32: far
// positions lose nothing (in 32 bits position 100000 would be off by 2^-8).
//
// Bytes bound it: each value is read and written once.  A CTA takes one token,
// or four, with all their heads, so that a token's angles are worked out once
// for all heads, in shared memory, and its place in the cache is looked up
// once.  A thread turns both chunks of 16 bytes that hold its pairs, one unit at
// a time: as many threads as an SM holds keep more on its way than fewer that
// are several units ahead (20000 tokens of 32/8 heads of 128 in bf16, half of
// each turned: 86 us, four ahead 108, two ahead 95).  Where lengths differ much the
// CTAs take the blocks of all sequences in turn (launch_blocks).
#include <algorithm>

#include "rows.cuh"

namespace nllb {
namespace {

constexpr int kThreads = 256;

enum { kNone = 0, kHalves = 1, kNeighbours = 2 };

// The blocks of TOK tokens of all sequences, one behind the other: which sequence's block `b` is, and its number there.  Every
// sequence has one at least, so that its lengths are looked at.
template <int TOK>
struct Blocks {
    int before;  // blocks of the sequences of the threads before this one
    int mine;    // of this thread's sequences, [first, last)
    int first, last, total;

    static __device__ __forceinline__ int of(const RowsParams& r, int s) {
        const int n = r.q_len ? ld_coherent(r.q_len + s) : r.max_q;
        return n < 1 || n > r.max_q ? 1 : (n + TOK - 1) / TOK;
    }
    __device__ __forceinline__ explicit Blocks(const RowsParams& r) {
        __shared__ int sums[kThreads / 32];
        const int per = (r.n_seq + kThreads - 1) / kThreads, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        first = min(r.n_seq, (int)threadIdx.x * per), last = min(r.n_seq, first + per), mine = 0;
        for (int s = first; s < last; ++s) mine += of(r, s);
        int x = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) sums[warp] = x;
        __syncthreads();
        before = x - mine, total = 0;
        for (int w = 0; w < kThreads / 32; ++w) {
            if (w < warp) before += sums[w];
            total += sums[w];
        }
    }
    __device__ __forceinline__ void find(const RowsParams& r, int b, int (&found)[2]) const {
        if (b < before || b >= before + mine) return;
        int at = b - before, s = first;
        for (int n; s < last - 1 && at >= (n = of(r, s)); ++s) at -= n;
        found[0] = s, found[1] = at;
    }
};

// Tokens [t0, t0 + TOK) of sequence s, by a CTA.
template <typename T, int D, int PAIRS, int TOK>
__device__ __forceinline__ void append_block(const AppendParams& p, int s, int t0) {
    constexpr int VEC = 16 / (int)sizeof(T);
    __shared__ __align__(16) float2 turn[TOK * D / 2];  // cos, sin
    // of each token: where its query, key and value heads come from and go to (null: nowhere)
    __shared__ const T* from[TOK][3];
    __shared__ T* to[TOK][3];
    const RowsParams& r = p.rows;
    const int tid = threadIdx.x;
    RowsSeq sq;
    if (!rows_sequence<true>(r, s, sq)) return;
    const int n_tok = min(TOK, sq.qn - t0);
    if (n_tok <= 0) return;
    if (tid < n_tok) {
        const int j = sq.kvn - sq.qn + t0 + tid, at = rows_page(r, j);
        const int pg = ld_coherent(r.table + (long long)s * r.table_ld + at);
        const bool ok = (unsigned)pg < (unsigned)r.n_pages;
        if (!ok) atomicOr(r.err, NLLB_DEV_ERR_BAD_PAGE);
        const long long row = sq.q0 + t0 + tid, slot = j - at * r.page;
        from[tid][0] = static_cast<const T*>(r.q) + row * r.q_row;
        from[tid][1] = static_cast<const T*>(r.k_new) + row * r.kn_row;
        from[tid][2] = static_cast<const T*>(r.v_new) + row * r.vn_row;
        to[tid][0] = static_cast<T*>(r.out) + row * r.o_row;
        to[tid][1] = ok ? static_cast<T*>(r.k_w) + pg * r.k_page + slot * r.k_row : nullptr;
        to[tid][2] = ok ? static_cast<T*>(r.v_w) + pg * r.v_page + slot * r.v_row : nullptr;
    }
    __syncthreads();

    // A head's units: chunks of 16 bytes, or, with halves, two of them half a turn's width apart.  A thread has unit `u` of
    // every lanes-th head, over all tokens.
    const int n = PAIRS == kNone ? 0 : p.half;
    const int two = PAIRS == kHalves ? n / VEC : 0, per = D / VEC - two;
    const int q_heads = r.q ? r.kv_heads * r.group : 0, k_end = q_heads + r.kv_heads, heads = k_end + r.kv_heads;
    const int lanes = kThreads / per, slot = tid / per, u = tid - slot * per;  // threads [lanes * per, kThreads) have none
    const bool pair = u < two;
    const int c = (pair ? u : u + two) * VEC;                                    // its first element
    const int angle = c >= 2 * n ? -1 : PAIRS == kHalves ? c : c / 2;            // its first pair's (-1: not turned)
    const int step_tok = lanes / heads, step_head = lanes - step_tok * heads;
    int tok = slot / heads, h = slot - tok * heads;
    if (slot >= lanes) tok = n_tok;
    auto kind = [&](int h) { return h < q_heads ? 0 : h < k_end ? 1 : 2; };
    uint4 a, b;
    auto load = [&] {
        if (tok >= n_tok) return;
        const int x = kind(h);
        const T* src = from[tok][x] + (x == 0 ? h * r.q_head : x == 1 ? (h - q_heads) * r.kn_head : (h - k_end) * r.vn_head) + c;
        a = ld_coherent(reinterpret_cast<const uint4*>(src));
        if (PAIRS == kHalves && pair) b = ld_coherent(reinterpret_cast<const uint4*>(src + n));
    };
    load();  // (under way while the angles are worked out)
    if constexpr (PAIRS != kNone) {
        for (int i = tid; i < n_tok * n; i += kThreads) {
            const int t = i / n, f = i - t * n;
            const int pos = p.position ? ld_coherent(p.position + sq.q0 + t0 + t) : sq.kvn - sq.qn + t0 + t;
            const double turns = (double)pos * (double)ld_coherent(p.inv_freq + f) * 0.15915494309189533577;
            float sin, cos;
            sincospif((float)(2.0 * (turns - rint(turns))), &sin, &cos);
            turn[i] = make_float2(cos, sin);
        }
        __syncthreads();
    }
    while (tok < n_tok) {
        const int x = kind(h);
        T* dst = to[tok][x];
        if (PAIRS != kNone && angle >= 0 && x < 2) {
            const float4* t = reinterpret_cast<const float4*>(turn + tok * n + angle);  // (two pairs)
            float v[VEC], w[VEC];
            rows_unpack<T>(a, v);
            if constexpr (PAIRS == kHalves) {
                rows_unpack<T>(b, w);
#pragma unroll
                for (int e = 0; e < VEC; e += 2) {
                    const float4 f = t[e / 2];
                    const float v0 = v[e], v1 = v[e + 1];
                    v[e] = v0 * f.x - w[e] * f.y, w[e] = w[e] * f.x + v0 * f.y;
                    v[e + 1] = v1 * f.z - w[e + 1] * f.w, w[e + 1] = w[e + 1] * f.z + v1 * f.w;
                }
                b = rows_pack<T>(w);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; e += 4) {
                    const float4 f = t[e / 4];
                    const float v0 = v[e], v2 = v[e + 2];
                    v[e] = v0 * f.x - v[e + 1] * f.y, v[e + 1] = v[e + 1] * f.x + v0 * f.y;
                    v[e + 2] = v2 * f.z - v[e + 3] * f.w, v[e + 3] = v[e + 3] * f.z + v2 * f.w;
                }
            }
            a = rows_pack<T>(v);
        }
        if (dst) {
            dst += (x == 0 ? h * r.o_head : x == 1 ? (h - q_heads) * r.k_head : (h - k_end) * r.v_head) + c;
            *reinterpret_cast<uint4*>(dst) = a;
            if (PAIRS == kHalves && pair) *reinterpret_cast<uint4*>(dst + n) = b;
        }
        tok += step_tok, h += step_head;
        if (h >= heads) h -= heads, ++tok;
        load();
    }
}

// FLAT: the CTAs take the blocks of all sequences in turn (else: one each, of a grid of the longest sequence's by sequences).
template <typename T, int D, int PAIRS, int TOK, bool FLAT>
__global__ void __launch_bounds__(kThreads, 8) append_kernel(const AppendParams p) {
    pdl_launch_dependents();
    pdl_wait_primary();
    if constexpr (FLAT) {
        __shared__ int found[2];
        const Blocks<TOK> blocks(p.rows);
        for (int b = blockIdx.x; b < blocks.total; b += gridDim.x) {
            __syncthreads();
            blocks.find(p.rows, b, found);
            __syncthreads();
            append_block<T, D, PAIRS, TOK>(p, found[0], found[1] * TOK);
        }
    } else {
        append_block<T, D, PAIRS, TOK>(p, blockIdx.y, blockIdx.x * TOK);
    }
}

template <typename T, int D, int PAIRS, int TOK>
cudaError_t launch_blocks(const AppendParams& p, cudaStream_t st) {
    const RowsParams& r = p.rows;
    const long long longest = (r.max_q + TOK - 1) / TOK, every = longest * r.n_seq, all = r.q_rows / TOK + r.n_seq;
    // Sequences of very different lengths: a grid of their longest would be empty for the most part (one chunk of 4096 tokens
    // among 255 single ones in bf16, 16/4 heads of 128: 77 us, flat 15).  Where each row is of one sequence, `all` CTAs have
    // a block each at most.  The sums of blocks stay in 32 bits, and a thread counts 64 sequences at most.
    if (every > 2 * all && every < 1ll << 31 && r.n_seq <= 64 * kThreads)
        return launch_pdl(append_kernel<T, D, PAIRS, TOK, true>, dim3((unsigned)all), dim3(kThreads), 0, st, p);
    return launch_pdl(append_kernel<T, D, PAIRS, TOK, false>, dim3((unsigned)longest, (unsigned)r.n_seq), dim3(kThreads), 0, st, p);
}

template <typename T, int D, int PAIRS>
cudaError_t launch_by_tokens(const AppendParams& p, int num_sms, cudaStream_t st) {
    // four tokens of a sequence to a CTA where that leaves every SM some
    if (p.rows.max_q > 1 && p.rows.q_rows >= 16 * num_sms) return launch_blocks<T, D, PAIRS, 4>(p, st);
    return launch_blocks<T, D, PAIRS, 1>(p, st);
}

template <typename T, int D>
cudaError_t launch_by_pairs(const AppendParams& p, int num_sms, cudaStream_t st) {
    if (p.half == 0) return launch_by_tokens<T, D, kNone>(p, num_sms, st);
    return p.neighbours ? launch_by_tokens<T, D, kNeighbours>(p, num_sms, st) : launch_by_tokens<T, D, kHalves>(p, num_sms, st);
}

}  // namespace

cudaError_t launch_append(const AppendParams& p, RowType type, int head_dim, int num_sms, cudaStream_t st) {
    const bool d64 = head_dim == 64;
    switch (type) {
        case RowType::f32: return d64 ? launch_by_pairs<float, 64>(p, num_sms, st) : launch_by_pairs<float, 128>(p, num_sms, st);
        case RowType::f16: return d64 ? launch_by_pairs<__half, 64>(p, num_sms, st) : launch_by_pairs<__half, 128>(p, num_sms, st);
        default: return d64 ? launch_by_pairs<__nv_bfloat16, 64>(p, num_sms, st) : launch_by_pairs<__nv_bfloat16, 128>(p, num_sms, st);
    }
}

}  // namespace nllb
