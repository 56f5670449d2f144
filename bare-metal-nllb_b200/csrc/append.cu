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
// once.  A thread turns both chunks of 16 bytes that hold its pairs; its first
// loads are in flight before the angles are worked out.
#include <algorithm>

#include "rows.cuh"

namespace nllb {
namespace {

constexpr int kThreads = 256;
constexpr int kAhead = 4;  // units of a thread whose loads are in flight together

enum { kNone = 0, kHalves = 1, kNeighbours = 2 };

// Chunk(s) of 16 bytes of one head of one token: source, destination, whether they are turned.
template <typename T>
struct Unit {
    const T* from;
    T* to;
    int angle;  // of its first value: into the angles of the CTA; below 0: not turned
    bool two;   // a second chunk, half a turn's width further
};

template <typename T, int D, int PAIRS, int TOK>
__global__ void __launch_bounds__(kThreads) append_kernel(const AppendParams p) {
    constexpr int VEC = 16 / (int)sizeof(T);
    __shared__ float2 turn[TOK * D / 2];  // cos, sin
    __shared__ long long k_at[TOK], v_at[TOK];  // places in the cache, below 0: none
    pdl_launch_dependents();
    pdl_wait_primary();

    const RowsParams& r = p.rows;
    const int s = blockIdx.y, t0 = blockIdx.x * TOK, tid = threadIdx.x;
    RowsSeq sq;
    if (!rows_sequence<true>(r, s, sq)) return;
    const int n_tok = min(TOK, sq.qn - t0);
    if (n_tok <= 0) return;

    const int n = PAIRS == kNone ? 0 : p.half;
    // a head's units: with halves, a unit holds chunk c and chunk c + n / VEC
    const int two = PAIRS == kHalves ? n / VEC : 0, per = D / VEC - two;
    const int q_heads = r.q ? r.kv_heads * r.group : 0, heads = q_heads + 2 * r.kv_heads;
    const int lanes = kThreads / per, slot = tid / per, u = tid - slot * per;  // threads [lanes * per, kThreads) have none
    const int c = u < two ? u : u + two, total = slot < lanes ? n_tok * heads : 0;

    auto unit = [&](int i) {
        Unit<T> x;
        const int tok = i / heads, h = i - tok * heads;
        const long long row = sq.q0 + t0 + tok;
        x.two = PAIRS == kHalves && u < two;
        x.angle = PAIRS == kNone || h >= q_heads + r.kv_heads || c * VEC >= 2 * n ? -1
                                                                                 : tok * n + (PAIRS == kHalves ? c * VEC : c * VEC / 2);
        if (h < q_heads) {
            x.from = static_cast<const T*>(r.q) + row * r.q_row + (long long)h * r.q_head + c * VEC;
            x.to = static_cast<T*>(r.out) + row * r.o_row + (long long)h * r.o_head + c * VEC;
        } else if (h < q_heads + r.kv_heads) {
            const long long g = h - q_heads;
            x.from = static_cast<const T*>(r.k_new) + row * r.kn_row + g * r.kn_head + c * VEC;
            x.to = k_at[tok] < 0 ? nullptr : static_cast<T*>(r.k_w) + k_at[tok] + g * r.k_head + c * VEC;
        } else {
            const long long g = h - q_heads - r.kv_heads;
            x.from = static_cast<const T*>(r.v_new) + row * r.vn_row + g * r.vn_head + c * VEC;
            x.to = v_at[tok] < 0 ? nullptr : static_cast<T*>(r.v_w) + v_at[tok] + g * r.v_head + c * VEC;
        }
        return x;
    };
    uint4 a[kAhead], b[kAhead];
    auto load = [&](int i0) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int i = i0 + k * lanes;
            if (i >= total) continue;
            const int tok = i / heads, h = i - tok * heads;
            const long long row = sq.q0 + t0 + tok;
            const T* from = h < q_heads ? static_cast<const T*>(r.q) + row * r.q_row + (long long)h * r.q_head
                            : h < q_heads + r.kv_heads
                                ? static_cast<const T*>(r.k_new) + row * r.kn_row + (long long)(h - q_heads) * r.kn_head
                                : static_cast<const T*>(r.v_new) + row * r.vn_row + (long long)(h - q_heads - r.kv_heads) * r.vn_head;
            a[k] = ld_coherent(reinterpret_cast<const uint4*>(from + c * VEC));
            if (PAIRS == kHalves && u < two) b[k] = ld_coherent(reinterpret_cast<const uint4*>(from + c * VEC + n));
        }
    };
    load(slot);

    if (tid < n_tok) {
        const int j = sq.kvn - sq.qn + t0 + tid, at = rows_page(r, j);
        const int pg = ld_coherent(r.table + (long long)s * r.table_ld + at);
        const bool ok = (unsigned)pg < (unsigned)r.n_pages;
        if (!ok) atomicOr(r.err, NLLB_DEV_ERR_BAD_PAGE);
        const long long in_page = j - at * r.page;
        k_at[tid] = ok ? pg * r.k_page + in_page * r.k_row : -1;
        v_at[tid] = ok ? pg * r.v_page + in_page * r.v_row : -1;
    }
    if constexpr (PAIRS != kNone) {
        for (int i = tid; i < n_tok * n; i += kThreads) {
            const int tok = i / n, f = i - tok * n;
            const int pos = p.position ? ld_coherent(p.position + sq.q0 + t0 + tok) : sq.kvn - sq.qn + t0 + tok;
            const double turns = (double)pos * (double)ld_coherent(p.inv_freq + f) * 0.15915494309189533577;
            float sin, cos;
            sincospif((float)(2.0 * (turns - rint(turns))), &sin, &cos);
            turn[i] = make_float2(cos, sin);
        }
    }
    __syncthreads();

    for (int i0 = slot; i0 < total; i0 += kAhead * lanes) {
        if (i0 > slot) load(i0);
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int i = i0 + k * lanes;
            if (i >= total) continue;
            const Unit<T> x = unit(i);
            uint4 y = a[k], z = b[k];
            if (PAIRS != kNone && x.angle >= 0) {
                float v[VEC], w[VEC];
                rows_unpack<T>(a[k], v);
                if constexpr (PAIRS == kHalves) {
                    rows_unpack<T>(b[k], w);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const float2 t = turn[x.angle + e];
                        const float f = v[e];
                        v[e] = f * t.x - w[e] * t.y;
                        w[e] = w[e] * t.x + f * t.y;
                    }
                    z = rows_pack<T>(w);
                } else {
#pragma unroll
                    for (int e = 0; e < VEC; e += 2) {
                        const float2 t = turn[x.angle + e / 2];
                        const float f = v[e];
                        v[e] = f * t.x - v[e + 1] * t.y;
                        v[e + 1] = v[e + 1] * t.x + f * t.y;
                    }
                }
                y = rows_pack<T>(v);
            }
            if (x.to) {
                *reinterpret_cast<uint4*>(x.to) = y;
                if (x.two) *reinterpret_cast<uint4*>(x.to + n) = z;
            }
        }
    }
}

template <typename T, int D, int PAIRS>
cudaError_t launch_by_tokens(const AppendParams& p, int num_sms, cudaStream_t st) {
    const RowsParams& r = p.rows;
    // four tokens of a sequence to a CTA where that leaves every SM some
    const bool many = r.max_q > 1 && r.q_rows >= 16 * num_sms;
    const dim3 grid((unsigned)((r.max_q + (many ? 3 : 0)) / (many ? 4 : 1)), (unsigned)r.n_seq);
    return many ? launch_pdl(append_kernel<T, D, PAIRS, 4>, grid, dim3(kThreads), 0, st, p)
                : launch_pdl(append_kernel<T, D, PAIRS, 1>, grid, dim3(kThreads), 0, st, p);
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
