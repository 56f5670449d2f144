// rows.cuh -- device helpers shared by the two kernels of rows.h.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "device_common.cuh"
#include "rows.h"

namespace nllb {

// A sequence's rows, checked against the buffers: the lengths come from
// device memory, so a bad one is flagged in the error word and its sequence
// left out instead of being followed out of bounds.
struct RowsSeq {
    int q0, qn;    // first query row, query rows
    int kv0, kvn;  // first key row (packed keys), keys
};

template <bool PAGED>
__device__ __forceinline__ bool rows_sequence(const RowsParams& p, int s, RowsSeq& q) {
    q.q0 = p.q_start ? ld_coherent(p.q_start + s) : s * p.max_q;
    q.qn = p.q_len ? ld_coherent(p.q_len + s) : p.max_q;
    q.kvn = ld_coherent(p.kv_len + s);
    q.kv0 = 0;
    bool ok = q.q0 >= 0 && q.qn >= 0 && q.qn <= p.max_q && q.q0 <= p.q_rows - q.qn && q.kvn >= 0 && q.kvn <= p.max_kv;
    if (PAGED) {
        ok = ok && q.kvn >= q.qn;
    } else {
        q.kv0 = p.kv_start ? ld_coherent(p.kv_start + s) : s * p.max_kv;
        ok = ok && q.kv0 >= 0 && q.kv0 <= p.kv_rows - q.kvn;
    }
    if (!ok && threadIdx.x == 0) atomicOr(p.err, NLLB_DEV_ERR_BAD_LENGTH);
    return ok;
}

// j / page by a multiplication: page_mul = ceil(2^page_shr / page), exact for
// j < 2^30 (rows_api.cu).
__device__ __forceinline__ int rows_page(const RowsParams& p, int j) {
    return (int)((unsigned long long)(uint32_t)j * p.page_mul >> p.page_shr);
}

// row / group in the same way (rows stay below 2^27).
__device__ __forceinline__ int rows_token(const RowsParams& p, int row) {
    return (int)((unsigned long long)(uint32_t)row * p.group_mul >> p.group_shr);
}

// What has to be looked up to place key `j` of the sequence (j < kvn): its
// page number, or its byte of the mask.  Apart from rows_at, so that it can be
// asked for ahead of its use.
template <bool PAGED>
__device__ __forceinline__ int rows_entry(const RowsParams& p, const RowsSeq& q, int s, int j) {
    if (PAGED) {
        if (p.k_new && j >= q.kvn - q.qn) return 0;
        return ld_coherent(p.table + (long long)s * p.table_ld + rows_page(p, j));
    }
    return p.mask ? ld_coherent(p.mask + q.kv0 + j) : 1;
}

// Where key `j` lies, for K and for V.  False: its page number is outside the
// pool (flagged), or the mask hides the key.
template <typename T, bool PAGED>
__device__ __forceinline__ bool rows_at(const RowsParams& p, const RowsSeq& q, int g, int j, int entry, const T*& k,
                                        const T*& v) {
    if (PAGED) {
        const int first_new = q.kvn - q.qn;
        if (p.k_new && j >= first_new) {  // the chunk's own rows are read where they come from
            const long long r = q.q0 + (j - first_new);
            k = static_cast<const T*>(p.k_new) + r * p.kn_row + (long long)g * p.kn_head;
            v = static_cast<const T*>(p.v_new) + r * p.vn_row + (long long)g * p.vn_head;
            return true;
        }
        if ((unsigned)entry >= (unsigned)p.n_pages) {
            atomicOr(p.err, NLLB_DEV_ERR_BAD_PAGE);
            return false;
        }
        const long long slot = j - rows_page(p, j) * p.page;
        k = static_cast<const T*>(p.k) + entry * p.k_page + slot * p.k_row + (long long)g * p.k_head;
        v = static_cast<const T*>(p.v) + entry * p.v_page + slot * p.v_row + (long long)g * p.v_head;
        return true;
    }
    const long long r = q.kv0 + j;
    k = static_cast<const T*>(p.k) + r * p.k_row + (long long)g * p.k_head;
    v = static_cast<const T*>(p.v) + r * p.v_row + (long long)g * p.v_head;
    return entry != 0;
}

template <typename T, bool PAGED>
__device__ __forceinline__ bool rows_key(const RowsParams& p, const RowsSeq& q, int s, int g, int j, const T*& k,
                                         const T*& v) {
    return rows_at<T, PAGED>(p, q, g, j, rows_entry<PAGED>(p, q, s, j), k, v);
}

// The chunk's rows of tokens [t0, t1) of key head g go into their pages.
// Nothing in the launch reads those slots: their keys come from k_new.
template <typename T, int D>
__device__ __forceinline__ void rows_append(const RowsParams& p, const RowsSeq& q, int s, int g, int t0, int t1,
                                            int tid, int n_threads) {
    constexpr int CH = D * (int)sizeof(T) / 16;
    for (int i = tid; i < (t1 - t0) * CH; i += n_threads) {
        const int t = t0 + i / CH, c = i % CH, j = q.kvn - q.qn + t;
        const int at = rows_page(p, j), pg = ld_coherent(p.table + (long long)s * p.table_ld + at);
        if ((unsigned)pg >= (unsigned)p.n_pages) {
            atomicOr(p.err, NLLB_DEV_ERR_BAD_PAGE);
            continue;
        }
        const long long r = q.q0 + t, slot = j - at * p.page;
        const uint4 kv = ld_coherent(reinterpret_cast<const uint4*>(static_cast<const T*>(p.k_new) + r * p.kn_row +
                                                               (long long)g * p.kn_head) + c);
        const uint4 vv = ld_coherent(reinterpret_cast<const uint4*>(static_cast<const T*>(p.v_new) + r * p.vn_row +
                                                               (long long)g * p.vn_head) + c);
        reinterpret_cast<uint4*>(static_cast<T*>(p.k_w) + pg * p.k_page + slot * p.k_row + (long long)g * p.k_head)[c] = kv;
        reinterpret_cast<uint4*>(static_cast<T*>(p.v_w) + pg * p.v_page + slot * p.v_row + (long long)g * p.v_head)[c] = vv;
    }
}

// 16 bytes of a row as fp32.
template <typename T>
__device__ __forceinline__ void rows_unpack(uint4 u, float (&x)[16 / sizeof(T)]) {
    if constexpr (sizeof(T) == 4) {
        x[0] = __uint_as_float(u.x), x[1] = __uint_as_float(u.y), x[2] = __uint_as_float(u.z),
        x[3] = __uint_as_float(u.w);
    } else {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same<T, __half>::value) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                x[2 * i] = f.x, x[2 * i + 1] = f.y;
            } else {
                x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    }
}

// 16 bytes into shared memory, asynchronously; zeros, without a read, if they are not `there`.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

// Two fp32 values rounded to a 16-bit type.
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

// fp32 values rounded once to the output's type.
template <typename T>
__device__ __forceinline__ uint4 rows_pack(const float (&x)[16 / sizeof(T)]) {
    uint4 u;
    if constexpr (sizeof(T) == 4) {
        u = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same<T, __half>::value) {
                const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
        u = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return u;
}

}  // namespace nllb
