// rows_stream.cu -- attention of a few query rows over many keys (sm_100a):
// the single tokens of a decoder step, and short chunks.
//
//   out_r = sum_j w_rj v_j / sum_j w_rj,   w_rj = 2^(s_rj - m_r),
//   s_rj = scale * log2(e) * q_r . k_j,    m_r the running maximum.
//
// The bytes of K and V bound it: every key row is read once for all R query
// rows of the CTA (the query heads that share a key head, and the tokens of a
// chunk).  A row is read by D * sizeof(T) / 16 lanes, 16 bytes each, straight
// into registers -- no tile in shared memory, so pages of any size, strides of
// any order and masks cost one address per row -- with U rows of K and of V in
// flight per lane.  Each group of lanes keeps the softmax state of its own
// keys; the states are joined once at the end, in the warp by shuffles, in the
// CTA through shared memory and, when few CTAs would be at work, across the
// CTAs of a cluster that share the keys of one (sequence, key head) through
// distributed shared memory: no workspace, and always in the same order.
#include <algorithm>
#include <type_traits>

#include "rows.cuh"

namespace nllb {
namespace {

constexpr int kWarps = 4;

template <typename T, int D, int R, bool PAGED>
__global__ void __launch_bounds__(kWarps * 32) rows_stream_kernel(const RowsParams p, int n_split) {
    constexpr int VEC = 16 / (int)sizeof(T);  // elements of a lane's 16 bytes
    constexpr int LPR = D / VEC;              // lanes per row
    constexpr int KPW = 32 / LPR;             // keys per warp and step
    constexpr int U = R == 1 ? 4 : 2;         // rows in flight per lane (K and V each)
    constexpr int STEP = kWarps * KPW * U;
    __shared__ float s_m[kWarps][R], s_l[kWarps][R];
    __shared__ __align__(16) float s_acc[kWarps][R][D];
    __shared__ __align__(16) float s_part[R][D + 4];  // this CTA's state: m, l, -, -, acc

    pdl_launch_dependents();
    pdl_wait_primary();

    const int split = blockIdx.x % n_split, tile = blockIdx.x / n_split;
    const int g = blockIdx.y, s = blockIdx.z;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int sub = lane / LPR, c = lane % LPR;
    RowsSeq sq;
    // (uniform over the cluster: its CTAs share tile, key head and sequence)
    if (!rows_sequence<PAGED>(p, s, sq)) return;
    const int rows = sq.qn * p.group;
    if (tile * R >= rows) return;

    if (PAGED && p.k_new && split == 0) {
        // a token belongs to the tile that holds its first row
        const int t0 = (tile * R + p.group - 1) / p.group, t1 = min(sq.qn, ((tile + 1) * R + p.group - 1) / p.group);
        rows_append<T, D>(p, sq, s, g, t0, t1, tid, kWarps * 32);
    }

    float q[R][VEC];
    int lim[R], longest = 0;  // keys a row sees
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int row = tile * R + r;
        lim[r] = 0;
#pragma unroll
        for (int i = 0; i < VEC; ++i) q[r][i] = 0.f;
        if (row < rows) {
            const int t = row / p.group, h = g * p.group + row % p.group;
            lim[r] = PAGED ? sq.kvn - sq.qn + t + 1 : sq.kvn;
            const T* src = static_cast<const T*>(p.q) + (long long)(sq.q0 + t) * p.q_row + (long long)h * p.q_head;
            rows_unpack<T>(__ldg(reinterpret_cast<const uint4*>(src) + c), q[r]);
#pragma unroll
            for (int i = 0; i < VEC; ++i) q[r][i] *= p.scale_log2;
        }
        longest = max(longest, lim[r]);
    }

    float m[R], l[R], acc[R][VEC];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[r][i] = 0.f;
    }

    // this CTA's share of the keys, in whole steps
    int per = (longest + n_split - 1) / n_split;
    per = (per + STEP - 1) / STEP * STEP;
    const int j_end = min(longest, (split + 1) * per);
    for (int j0 = split * per; j0 < j_end; j0 += STEP) {
        uint4 ku[U], vu[U];
        bool seen[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + (u * kWarps + warp) * KPW + sub;
            const T *kr, *vr;
            seen[u] = j < j_end && rows_key<T, PAGED>(p, sq, s, g, j, kr, vr);
            ku[u] = vu[u] = make_uint4(0, 0, 0, 0);  // a hidden key's rows are never read
            if (seen[u]) {
                ku[u] = __ldg(reinterpret_cast<const uint4*>(kr) + c);
                vu[u] = __ldg(reinterpret_cast<const uint4*>(vr) + c);
            }
        }
        float sc[R][U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float k[VEC];
            rows_unpack<T>(ku[u], k);
            const int j = j0 + (u * kWarps + warp) * KPW + sub;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float d = 0.f;
#pragma unroll
                for (int i = 0; i < VEC; ++i) d = fmaf(q[r][i], k[i], d);
#pragma unroll
                for (int o = LPR / 2; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
                sc[r][u] = (seen[u] && j < lim[r]) ? d : -INFINITY;
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float mn = m[r];
#pragma unroll
            for (int u = 0; u < U; ++u) mn = fmaxf(mn, sc[r][u]);
            const float base = mn == -INFINITY ? 0.f : mn;
            const float corr = exp2f(m[r] - base);  // 0 for an empty state
            m[r] = mn;
            l[r] *= corr;
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[r][i] *= corr;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                sc[r][u] = exp2f(sc[r][u] - base);
                l[r] += sc[r][u];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float v[VEC];
            rows_unpack<T>(vu[u], v);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int i = 0; i < VEC; ++i) acc[r][i] = fmaf(sc[r][u], v[i], acc[r][i]);
        }
    }

    // join the warp's lane groups
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int o = LPR; o < 32; o <<= 1) {
            const float mo = __shfl_xor_sync(0xffffffffu, m[r], o);
            const float lo = __shfl_xor_sync(0xffffffffu, l[r], o);
            const float mn = fmaxf(m[r], mo), base = mn == -INFINITY ? 0.f : mn;
            const float a = exp2f(m[r] - base), b = exp2f(mo - base);
            m[r] = mn;
            l[r] = l[r] * a + lo * b;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float x = __shfl_xor_sync(0xffffffffu, acc[r][i], o);
                acc[r][i] = acc[r][i] * a + x * b;
            }
        }
        if (sub == 0) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) s_acc[warp][r][c * VEC + i] = acc[r][i];
            if (c == 0) s_m[warp][r] = m[r], s_l[warp][r] = l[r];
        }
    }
    __syncthreads();
    // join the warps: one thread per (row, element)
    for (int i = tid; i < R * D; i += kWarps * 32) {
        const int r = i / D, d = i % D;
        float mn = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mn = fmaxf(mn, s_m[w][r]);
        const float base = mn == -INFINITY ? 0.f : mn;
        float a = 0.f, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float e = exp2f(s_m[w][r] - base);
            a = fmaf(e, s_acc[w][r][d], a);
            sum = fmaf(e, s_l[w][r], sum);
        }
        s_part[r][4 + d] = a;
        if (d == 0) s_part[r][0] = mn, s_part[r][1] = sum;
    }
    if (n_split > 1) cluster_sync_all();
    else __syncthreads();

    // join the splits (rank by rank, so the order is fixed): rank z finishes
    // the 16-byte pieces z, z + n_split, ...
    for (int i = split + n_split * tid; i < R * LPR; i += n_split * kWarps * 32) {
        const int r = i / LPR, cc = i % LPR, row = tile * R + r;
        if (row >= rows) continue;
        float x[VEC];
        if (n_split == 1) {
            const float inv = s_part[r][1] > 0.f ? 1.f / s_part[r][1] : 0.f;  // no visible key: zeros
#pragma unroll
            for (int e = 0; e < VEC; ++e) x[e] = s_part[r][4 + cc * VEC + e] * inv;
        } else {
            float mn = -INFINITY;
            for (int z = 0; z < n_split; ++z) mn = fmaxf(mn, ld_cluster_f32(map_rank(&s_part[r][0], z)));
            const float base = mn == -INFINITY ? 0.f : mn;
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) x[e] = 0.f;
            for (int z = 0; z < n_split; ++z) {
                const float w = exp2f(ld_cluster_f32(map_rank(&s_part[r][0], z)) - base);
                sum = fmaf(w, ld_cluster_f32(map_rank(&s_part[r][1], z)), sum);
#pragma unroll
                for (int e = 0; e < VEC; e += 4) {
                    const float4 f = ld_cluster_f4(map_rank(&s_part[r][4 + cc * VEC + e], z));
                    x[e] = fmaf(w, f.x, x[e]), x[e + 1] = fmaf(w, f.y, x[e + 1]);
                    x[e + 2] = fmaf(w, f.z, x[e + 2]), x[e + 3] = fmaf(w, f.w, x[e + 3]);
                }
            }
            const float inv = sum > 0.f ? 1.f / sum : 0.f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) x[e] *= inv;
        }
        const int t = row / p.group, h = g * p.group + row % p.group;
        T* dst = static_cast<T*>(p.out) + (long long)(sq.q0 + t) * p.o_row + (long long)h * p.o_head;
        reinterpret_cast<uint4*>(dst)[cc] = rows_pack<T>(x);
    }
    if (n_split > 1) cluster_sync_all();  // no CTA leaves while another reads its state
}

template <typename T, int D, int R, bool PAGED>
cudaError_t launch_one(const RowsParams& p, int num_sms, cudaStream_t st) {
    const long long tiles = ((long long)p.max_q * p.group + R - 1) / R;
    const long long units = tiles * p.kv_heads * p.n_seq;
    // as many CTAs as keep the memory busy (4 per SM), no share under 64 keys
    int n_split = 1;
    while (n_split < 16 && units * n_split < 4LL * num_sms && p.max_kv >= 128 * n_split) n_split *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * n_split), (unsigned)p.kv_heads, (unsigned)p.n_seq);
    cfg.blockDim = dim3(kWarps * 32, 1, 1);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = kPdlLaunch;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)n_split;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = n_split > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, rows_stream_kernel<T, D, R, PAGED>, p, n_split);
}

template <typename T, int D, bool PAGED>
cudaError_t launch_by_rows(const RowsParams& p, int num_sms, cudaStream_t st) {
    const long long rows = (long long)p.max_q * p.group;
    if (rows == 1) return launch_one<T, D, 1, PAGED>(p, num_sms, st);
    if (rows <= 4) return launch_one<T, D, 4, PAGED>(p, num_sms, st);
    return launch_one<T, D, 8, PAGED>(p, num_sms, st);
}

template <typename T>
cudaError_t launch_by_dim(const RowsParams& p, int head_dim, bool paged, int num_sms, cudaStream_t st) {
    if (head_dim == 64)
        return paged ? launch_by_rows<T, 64, true>(p, num_sms, st) : launch_by_rows<T, 64, false>(p, num_sms, st);
    return paged ? launch_by_rows<T, 128, true>(p, num_sms, st) : launch_by_rows<T, 128, false>(p, num_sms, st);
}

template <typename T, int D, bool PAGED>
cudaError_t configure_one() {
    // clusters of 16 CTAs are beyond the portable size
    cudaError_t e = cudaFuncSetAttribute(rows_stream_kernel<T, D, 1, PAGED>,
                                         cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(rows_stream_kernel<T, D, 4, PAGED>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(rows_stream_kernel<T, D, 8, PAGED>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    return e;
}

template <typename T>
cudaError_t configure_type() {
    cudaError_t e = configure_one<T, 64, false>();
    if (e == cudaSuccess) e = configure_one<T, 64, true>();
    if (e == cudaSuccess) e = configure_one<T, 128, false>();
    if (e == cudaSuccess) e = configure_one<T, 128, true>();
    return e;
}

}  // namespace

cudaError_t configure_rows_kernels() {
    cudaError_t e = configure_type<float>();
    if (e == cudaSuccess) e = configure_type<__half>();
    if (e == cudaSuccess) e = configure_type<__nv_bfloat16>();
    if (e == cudaSuccess) e = configure_rows_tc();
    return e;
}

cudaError_t launch_rows(const RowsParams& p, RowType type, int head_dim, bool paged, int num_sms, cudaStream_t st) {
    // more rows than one CTA of this kernel takes would read the keys again
    if ((long long)p.max_q * p.group > 8) return launch_rows_tc(p, type, head_dim, paged, num_sms, st);
    switch (type) {
        case RowType::f32: return launch_by_dim<float>(p, head_dim, paged, num_sms, st);
        case RowType::f16: return launch_by_dim<__half>(p, head_dim, paged, num_sms, st);
        default: return launch_by_dim<__nv_bfloat16>(p, head_dim, paged, num_sms, st);
    }
}

}  // namespace nllb
