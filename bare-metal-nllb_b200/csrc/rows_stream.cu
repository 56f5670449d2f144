// rows_stream.cu -- attention of a few query rows over many keys (sm_100a):
// the single tokens of a decoder step, and short chunks.
//
//   out_r = sum_j w_rj v_j / sum_j w_rj,   w_rj = 2^(s_rj - m_r),
//   s_rj = scale * log2(e) * q_r . k_j,    m_r the running maximum.
//
// The bytes of K and V bound it: every key row is read once for all R query
// rows of the CTA (the query heads that share a key head, and the tokens of a
// chunk).  Each warp works alone on blocks of 32 keys (16 of 512-byte rows):
// a lane works out the address of one row -- so pages of any size, strides of
// any order and masks cost one look-up per row -- and the warp copies the
// rows with 16-byte asynchronous copies into a ring of its own in shared
// memory, several blocks ahead of the one it computes on.
//
// One query row, and fp32: fp32 arithmetic, D * sizeof(T) / 16 lanes to a key
// row.  Several rows of 16 bits: warp-level matrix products of 16 query rows
// (half of them padding up to 8) by 8 keys; fp32 multiplies would be the bound
// there, and tcgen05's 128 rows would be padding for the most part.  There the
// weights are rounded to the type, as in rows_tc.cu, held times 2^7.
//
// The warps' softmax states are joined once at the end through shared memory
// and, when few CTAs would be at work, across a cluster of CTAs that share the
// keys of one (sequence, key head) through distributed shared memory: no
// workspace, and always in the same order.
//
// Measured: 64 sequences of one token and four query heads to a key head over
// 200..8191 keys (bf16, heads of 128) 107 us = 5.4 TB/s; 256 tokens over
// memories of 18..512 rows (bf16) 57 us = 5.0 TB/s; one fp32 token after 99
// keys 4.5 us, latency; one token over 99990 keys with two key heads 31 us,
// bound by the 32 CTAs that two clusters of 16 make.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "rows.cuh"

namespace nllb {
namespace {

constexpr int kRowsMax = 16;  // query rows of one CTA at most
constexpr int kRing = 2;      // key blocks in a warp's ring
// Warps of a CTA with several, by the bytes of a block of K and V: as many as shared memory has room for, since more
// warps of short rings beat fewer of long ones (64 sequences over 200..8191 keys, 4 rows of 128: 7 x 2 blocks of 16 KB
// 106 us, 6 x 2 113, 5 x 2 148, 4 x 3 145; one over 99990 keys, 8 rows of 64: 14 x 2 blocks of 8 KB 31.5 us, 12 x 2
// 36.2, 8 x 3 37.6, 6 x 4 48.1).
constexpr int kWarps8 = 14, kWarps16 = 7;
constexpr int kWarpKeys = 32768;
constexpr float kWeightExp = 7.0f;

__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T, int D, int R, int NW>
struct Cfg {
    static constexpr int ROW = D * (int)sizeof(T);      // bytes of a key row
    static constexpr int CH = ROW / 16;                 // its 16-byte chunks = lanes to a row
    static constexpr int KPW = 32 / CH;                 // rows a warp copies at a time
    static constexpr bool MMA = sizeof(T) == 2 && R > 1;
    // Keys of a block: 16 of 256 bytes and more, which makes room for more warps (fp32 heads of 64: 161 us instead of
    // 174; memories of 18..512 rows of 128, a warp each: 100 instead of 122 us), except for the matrix products of
    // many warps, which take 32 (106 us instead of 123 for the 64 sequences above).
    static constexpr int BLK = ROW == 512 || (ROW == 256 && (!MMA || NW == 1)) ? 16 : 32;
    static constexpr uint32_t HALF = BLK * ROW;         // K (or V) of a block
    static constexpr int MANY = 2 * HALF <= 8192 ? kWarps8 : kWarps16;
    static constexpr uint32_t RING = kRing * 2 * HALF;  // of one warp
    static constexpr int LD = D + 4;                    // a row's state: m, l, -, -, D sums
    static constexpr uint32_t STATES = (NW + 1) * R * LD * 4;  // the warps', then the CTA's; over the rings
    static constexpr uint32_t SMEM = NW * RING > STATES ? NW * RING : STATES;
};

template <typename T, int D, int R, bool PAGED, int NW>
__global__ void __launch_bounds__(NW * 32) rows_stream_kernel(const RowsParams p, int n_split) {
    using C = Cfg<T, D, R, NW>;
    constexpr int VEC = 16 / (int)sizeof(T), CH = C::CH, KPW = C::KPW, BLK = C::BLK;
    extern __shared__ __align__(128) unsigned char smem[];

    pdl_launch_dependents();
    pdl_wait_primary();

    const int split = blockIdx.x;
    const int g = blockIdx.y, s = blockIdx.z;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int sub = lane / CH, c = lane % CH;
    RowsSeq sq;
    // (uniform over the cluster: its CTAs share key head and sequence)
    if (!rows_sequence<PAGED>(p, s, sq)) return;
    const int rows = sq.qn * p.group;  // R at most
    if (rows == 0) return;
    const int past = sq.kvn - sq.qn;  // (paged) keys before the chunk

    // the keys in blocks, shared among the splits; a warp takes every NW-th
    const int blocks = (sq.kvn + BLK - 1) / BLK, per = (blocks + n_split - 1) / n_split;
    const int b_end = min(blocks, (split + 1) * per);
    int b_next = split * per + warp;  // the next block to locate

    const uint32_t ring = smem_u32(smem) + warp * C::RING;
    const T *kp = nullptr, *vp = nullptr;
    auto locate = [&] {  // this lane's row of the next block
        const int key = b_next * BLK + lane;
        if (!(lane < BLK && b_next < b_end && key < sq.kvn && rows_key<T, PAGED>(p, sq, s, g, key, kp, vp)))
            kp = vp = nullptr;
        b_next += NW;
    };
    auto fetch = [&](int buf) -> uint32_t {  // the located block into ring slot `buf`; its visible keys
        const uint32_t dst = ring + buf * 2 * C::HALF;
        if (b_next - NW < b_end) {
#pragma unroll
            for (int i = 0; i < BLK / KPW; ++i) {
                const int r = i * KPW + sub;
                const T* k = reinterpret_cast<const T*>(
                    __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(kp), r));
                const T* v = reinterpret_cast<const T*>(
                    __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(vp), r));
                const uint32_t at = dst + r * C::ROW + ((c ^ (r & 7 & (CH - 1))) << 4);
                // a hidden row becomes zeros without being read
                cp_async16(at, k ? k + c * VEC : static_cast<const T*>(p.q), k != nullptr);
                cp_async16(at + C::HALF, k ? v + c * VEC : static_cast<const T*>(p.q), k != nullptr);
            }
        }
        cp_commit();  // (an empty group where the warp has no such block)
        return __ballot_sync(0xffffffffu, kp != nullptr);
    };
    int mine = max(0, (b_end - b_next + NW - 1) / NW);  // this warp's blocks
    uint32_t vis[kRing];                                // visible keys of the blocks in the ring, oldest first
#pragma unroll
    for (int i = 0; i < kRing - 1; ++i) {
        locate();
        vis[i] = fetch(i);
    }
    locate();

    if (PAGED && p.k_new && split == 0) rows_append<T, D>(p, sq, s, g, 0, sq.qn, tid, NW * 32);

    float* state = reinterpret_cast<float*>(smem) + warp * R * C::LD;
    auto q_at = [&](int r) {  // query row r (there)
        const int t = r / p.group, h = g * p.group + r % p.group;
        return static_cast<const T*>(p.q) + (long long)(sq.q0 + t) * p.q_row + (long long)h * p.q_head;
    };
    auto sees = [&](int r) {  // keys query row r sees
        if (r >= rows) return 0;
        return PAGED ? past + r / p.group + 1 : sq.kvn;
    };
    // body(block index, its visible keys, its K in the ring) for every block of the warp
    auto run = [&](auto&& body) {
        int b = split * per + warp, buf = 0;
        for (; mine > 0; --mine, b += NW) {
            int into = buf + kRing - 1;
            vis[kRing - 1] = fetch(into >= kRing ? into - kRing : into);
            locate();
            cp_wait<kRing - 1>();
            __syncwarp();
            body(b, vis[0], ring + buf * 2 * C::HALF);
            __syncwarp();  // the slot is free
#pragma unroll
            for (int i = 0; i < kRing - 1; ++i) vis[i] = vis[i + 1];
            buf = buf + 1 == kRing ? 0 : buf + 1;
        }
        cp_wait<0>();
        __syncthreads();  // the rings are free for the states
    };

    if constexpr (C::MMA) {
        // lane: rows lr and lr + 8, columns 2 lc, 2 lc + 1 of each 8
        constexpr int HALVES = R > 8 ? 2 : 1;
        const int lr = lane >> 2, lc = lane & 3;
        uint32_t qf[D / 16][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const bool there = h < HALVES && lr + 8 * h < rows;
            const T* src = there ? q_at(lr + 8 * h) : nullptr;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                qf[k][h] = there ? ld_coherent(reinterpret_cast<const uint32_t*>(src + k * 16 + 2 * lc)) : 0u;
                qf[k][h + 2] = there ? ld_coherent(reinterpret_cast<const uint32_t*>(src + k * 16 + 8 + 2 * lc)) : 0u;
            }
        }
        const int lim[2] = {sees(lr), HALVES == 2 ? sees(lr + 8) : 0};
        float m[HALVES], l[HALVES], o[D / 8][4];
#pragma unroll
        for (int h = 0; h < HALVES; ++h) m[h] = -INFINITY, l[h] = 0.f;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        // this lane's part of the ldmatrix addresses
        const int mr = lane & 7, mm = lane >> 3;  // row of matrix mm
        run([&](int b, uint32_t seen, uint32_t kb) {
            float sc[BLK / 8][4];
#pragma unroll
            for (int n = 0; n < BLK / 8; ++n) {  // 8 keys
                sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
#pragma unroll
                for (int k = 0; k < D / 32; ++k) {
                    uint32_t f[4];  // dims 32 k + 8 mm
                    ldmatrix4(f, kb + (n * 8 + mr) * C::ROW + (((k * 4 + mm) ^ mr) << 4));
                    mma16816<T>(sc[n], qf[2 * k], f[0], f[1]);
                    mma16816<T>(sc[n], qf[2 * k + 1], f[2], f[3]);
                }
            }
            const int j0 = b * BLK;
            const bool whole = seen == (BLK == 32 ? 0xffffffffu : 0xffffu) && (!PAGED || j0 + BLK <= past);
            uint32_t pf[BLK / 16][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (h >= HALVES) {
#pragma unroll
                    for (int k = 0; k < BLK / 16; ++k) pf[k][1] = pf[k][3] = 0u;
                    continue;
                }
                float mx = -INFINITY;
#pragma unroll
                for (int n = 0; n < BLK / 8; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float& x = sc[n][2 * h + e];
                        x *= p.scale_log2;
                        const int i = n * 8 + 2 * lc + e;
                        if (!whole && !(((seen >> i) & 1u) && j0 + i < lim[h])) x = -INFINITY;
                        mx = fmaxf(mx, x);
                    }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float to = fmaxf(m[h], mx);
                const float off = (to == -INFINITY ? 0.f : to) - kWeightExp;
                const float corr = exp2f(m[h] - kWeightExp - off);  // 0 for an empty state
                m[h] = to;
                l[h] *= corr;
#pragma unroll
                for (int i = 0; i < D / 8; ++i) o[i][2 * h] *= corr, o[i][2 * h + 1] *= corr;
#pragma unroll
                for (int n = 0; n < BLK / 8; ++n) {
                    const float x = exp2f(sc[n][2 * h] - off), y = exp2f(sc[n][2 * h + 1] - off);
                    l[h] += x + y;
                    pf[n >> 1][(n & 1) * 2 + h] = pack2<T>(x, y);
                }
            }
            const uint32_t vb = kb + C::HALF;
#pragma unroll
            for (int k = 0; k < BLK / 16; ++k)  // 16 keys
#pragma unroll
                for (int n = 0; n < D / 16; ++n) {  // 16 dims: matrices (keys 0-7, 8-15) x (dims 0-7, 8-15)
                    uint32_t f[4];
                    const int r = k * 16 + (mm & 1) * 8 + mr;
                    ldmatrix4_trans(f, vb + r * C::ROW + (((n * 2 + (mm >> 1)) ^ mr) << 4));
                    mma16816<T>(o[2 * n], pf[k], f[0], f[1]);
                    mma16816<T>(o[2 * n + 1], pf[k], f[2], f[3]);
                }
        });
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            float* st = state + (lr + 8 * h) * C::LD;
            if (lc == 0) st[0] = m[h], st[1] = l[h];
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
                *reinterpret_cast<float2*>(st + 4 + i * 8 + 2 * lc) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
        }
    } else {
        constexpr int U = BLK / KPW < 4 ? BLK / KPW : 4;  // keys of a lane taken together
        float q[R][VEC], m[R], l[R], acc[R][VEC];
        int lim[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            m[r] = -INFINITY, l[r] = 0.f;
            lim[r] = sees(r);
#pragma unroll
            for (int i = 0; i < VEC; ++i) q[r][i] = acc[r][i] = 0.f;
            if (r < rows) {
                rows_unpack<T>(ld_coherent(reinterpret_cast<const uint4*>(q_at(r)) + c), q[r]);
#pragma unroll
                for (int i = 0; i < VEC; ++i) q[r][i] *= p.scale_log2;
            }
        }
        run([&](int b, uint32_t seen, uint32_t kb) {
            const unsigned char* base = smem + (kb - smem_u32(smem));
            const int j0 = b * BLK;
#pragma unroll 1
            for (int i0 = 0; i0 < BLK / KPW; i0 += U) {
                float sc[R][U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int r = (i0 + u) * KPW + sub;
                    float k[VEC];
                    rows_unpack<T>(*reinterpret_cast<const uint4*>(base + r * C::ROW + ((c ^ (r & 7 & (CH - 1))) << 4)), k);
                    const bool there = (seen >> r) & 1u;
#pragma unroll
                    for (int x = 0; x < R; ++x) {
                        float d = 0.f;
#pragma unroll
                        for (int i = 0; i < VEC; ++i) d = fmaf(q[x][i], k[i], d);
#pragma unroll
                        for (int o = CH / 2; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
                        sc[x][u] = there && j0 + r < lim[x] ? d : -INFINITY;
                    }
                }
#pragma unroll
                for (int x = 0; x < R; ++x) {
                    float to = m[x];
#pragma unroll
                    for (int u = 0; u < U; ++u) to = fmaxf(to, sc[x][u]);
                    const float off = to == -INFINITY ? 0.f : to;
                    const float corr = exp2f(m[x] - off);  // 0 for an empty state
                    m[x] = to;
                    l[x] *= corr;
#pragma unroll
                    for (int i = 0; i < VEC; ++i) acc[x][i] *= corr;
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        sc[x][u] = exp2f(sc[x][u] - off);
                        l[x] += sc[x][u];
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int r = (i0 + u) * KPW + sub;
                    float v[VEC];
                    rows_unpack<T>(*reinterpret_cast<const uint4*>(base + C::HALF + r * C::ROW +
                                                                   ((c ^ (r & 7 & (CH - 1))) << 4)), v);
#pragma unroll
                    for (int x = 0; x < R; ++x)
#pragma unroll
                        for (int i = 0; i < VEC; ++i) acc[x][i] = fmaf(sc[x][u], v[i], acc[x][i]);
                }
            }
        });
        // join the warp's lane groups
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int o = CH; o < 32; o <<= 1) {
                const float mo = __shfl_xor_sync(0xffffffffu, m[r], o);
                const float lo = __shfl_xor_sync(0xffffffffu, l[r], o);
                const float to = fmaxf(m[r], mo), off = to == -INFINITY ? 0.f : to;
                const float a = exp2f(m[r] - off), b = exp2f(mo - off);
                m[r] = to;
                l[r] = l[r] * a + lo * b;
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float x = __shfl_xor_sync(0xffffffffu, acc[r][i], o);
                    acc[r][i] = acc[r][i] * a + x * b;
                }
            }
            if (sub == 0) {
                float* st = state + r * C::LD;
#pragma unroll
                for (int i = 0; i < VEC; i += 4)
                    *reinterpret_cast<float4*>(st + 4 + c * VEC + i) =
                        make_float4(acc[r][i], acc[r][i + 1], acc[r][i + 2], acc[r][i + 3]);
                if (c == 0) st[0] = m[r], st[1] = l[r];
            }
        }
    }
    __syncthreads();

    // join the warps: one thread per (row, element), into the CTA's state
    const float* warps = reinterpret_cast<const float*>(smem);
    float* part = reinterpret_cast<float*>(smem) + NW * R * C::LD;
    for (int i = tid; i < R * D; i += NW * 32) {
        const int r = i / D, d = i % D;
        float to = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; ++w) to = fmaxf(to, warps[(w * R + r) * C::LD]);
        const float off = to == -INFINITY ? 0.f : to;
        float a = 0.f, sum = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float* st = warps + (w * R + r) * C::LD;
            const float e = exp2f(st[0] - off);
            a = fmaf(e, st[4 + d], a);
            sum = fmaf(e, st[1], sum);
        }
        part[r * C::LD + 4 + d] = a;
        if (d == 0) part[r * C::LD] = to, part[r * C::LD + 1] = sum;
    }
    if (n_split > 1) cluster_sync_all();
    else __syncthreads();

    // join the splits (rank by rank, so the order is fixed): rank z finishes
    // the 16-byte pieces z, z + n_split, ...
    for (int i = split + n_split * tid; i < R * CH; i += n_split * NW * 32) {
        const int r = i / CH, cc = i % CH;
        if (r >= rows) continue;
        const float* st = part + r * C::LD;
        float x[VEC], sum = 0.f;
        if (n_split == 1) {
            sum = st[1];
#pragma unroll
            for (int e = 0; e < VEC; ++e) x[e] = st[4 + cc * VEC + e];
        } else {
            float to = -INFINITY;
            for (int z = 0; z < n_split; ++z) to = fmaxf(to, ld_cluster_f32(map_rank(st, z)));
            const float off = to == -INFINITY ? 0.f : to;
#pragma unroll
            for (int e = 0; e < VEC; ++e) x[e] = 0.f;
            for (int z = 0; z < n_split; ++z) {
                const float w = exp2f(ld_cluster_f32(map_rank(st, z)) - off);
                sum = fmaf(w, ld_cluster_f32(map_rank(st + 1, z)), sum);
#pragma unroll
                for (int e = 0; e < VEC; e += 4) {
                    const float4 f = ld_cluster_f4(map_rank(st + 4 + cc * VEC + e, z));
                    x[e] = fmaf(w, f.x, x[e]), x[e + 1] = fmaf(w, f.y, x[e + 1]);
                    x[e + 2] = fmaf(w, f.z, x[e + 2]), x[e + 3] = fmaf(w, f.w, x[e + 3]);
                }
            }
        }
        const float inv = 1.f / sum;
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[e] = sum == 0.f ? 0.f : x[e] * inv;  // no visible key: zeros
        const int t = r / p.group, h = g * p.group + r % p.group;
        T* dst = static_cast<T*>(p.out) + (long long)(sq.q0 + t) * p.o_row + (long long)h * p.o_head;
        reinterpret_cast<uint4*>(dst)[cc] = rows_pack<T>(x);
    }
    if (n_split > 1) cluster_sync_all();  // no CTA leaves while another reads its state
}

template <typename T, int D, int R, bool PAGED, int NW>
cudaError_t launch_one(const RowsParams& p, int n_split, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)n_split, (unsigned)p.kv_heads, (unsigned)p.n_seq);
    cfg.blockDim = dim3(NW * 32, 1, 1);
    cfg.dynamicSmemBytes = Cfg<T, D, R, NW>::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = kPdlLaunch;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)n_split;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = n_split > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, rows_stream_kernel<T, D, R, PAGED, NW>, p, n_split);
}

template <typename T, int D, int R, bool PAGED>
cudaError_t launch_by_units(const RowsParams& p, int num_sms, cudaStream_t st) {
    const long long units = (long long)p.kv_heads * p.n_seq;
    // A warp alone per unit where that already fills the SMs and the keys are few (256 sequences of 16 heads over
    // 18..512 keys: 56 us, with four warps 75); else many warps, and as many splits as give every SM work (four CTAs
    // per SM instead of two cost 134 us against 113 over 200..8191 keys), none with less than a block per warp, one
    // cluster at most.
    if (units >= 8LL * num_sms && p.max_kv <= 1024) return launch_one<T, D, R, PAGED, 1>(p, 1, st);
    constexpr int MANY = Cfg<T, D, R, 0>::MANY, step = MANY * Cfg<T, D, R, 0>::BLK;
    // The matrix products' sums lose up to a step of fp32 with every 16 keys, so a warp of them takes 32768 at most.
    const int most = Cfg<T, D, R, 0>::MMA ? MANY * kWarpKeys : INT_MAX;
    int n_split = 1;
    while (n_split < 16 && ((units * n_split < 2LL * num_sms && p.max_kv > step * n_split) || p.max_kv / n_split > most))
        n_split *= 2;
    return launch_one<T, D, R, PAGED, MANY>(p, n_split, st);
}

template <typename T, int D, bool PAGED>
cudaError_t launch_by_rows(const RowsParams& p, int num_sms, cudaStream_t st) {
    const long long rows = (long long)p.max_q * p.group;
    if (rows == 1) return launch_by_units<T, D, 1, PAGED>(p, num_sms, st);
    if constexpr (sizeof(T) == 2) {
        if (rows > 8) return launch_by_units<T, D, 16, PAGED>(p, num_sms, st);
    } else {
        if (rows <= 4) return launch_by_units<T, D, 4, PAGED>(p, num_sms, st);
    }
    return launch_by_units<T, D, 8, PAGED>(p, num_sms, st);
}

template <typename T>
cudaError_t launch_by_dim(const RowsParams& p, int head_dim, bool paged, int num_sms, cudaStream_t st) {
    if (head_dim == 64)
        return paged ? launch_by_rows<T, 64, true>(p, num_sms, st) : launch_by_rows<T, 64, false>(p, num_sms, st);
    return paged ? launch_by_rows<T, 128, true>(p, num_sms, st) : launch_by_rows<T, 128, false>(p, num_sms, st);
}

template <typename T, int D, int R, bool PAGED, int NW>
cudaError_t configure_one() {
    // clusters of 16 CTAs are beyond the portable size
    cudaError_t e = cudaFuncSetAttribute(rows_stream_kernel<T, D, R, PAGED, NW>,
                                         cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    return cudaFuncSetAttribute(rows_stream_kernel<T, D, R, PAGED, NW>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)Cfg<T, D, R, NW>::SMEM);
}

template <typename T, int D, int R>
cudaError_t configure_rows() {
    cudaError_t e = configure_one<T, D, R, false, 1>();
    if (e == cudaSuccess) e = configure_one<T, D, R, true, 1>();
    if (e == cudaSuccess) e = configure_one<T, D, R, false, Cfg<T, D, R, 0>::MANY>();
    if (e == cudaSuccess) e = configure_one<T, D, R, true, Cfg<T, D, R, 0>::MANY>();
    return e;
}

template <typename T, int D>
cudaError_t configure_dim() {
    cudaError_t e = configure_rows<T, D, 1>();
    if (e == cudaSuccess) e = configure_rows<T, D, 8>();
    if constexpr (sizeof(T) == 2) {
        if (e == cudaSuccess) e = configure_rows<T, D, 16>();
    } else {
        if (e == cudaSuccess) e = configure_rows<T, D, 4>();
    }
    return e;
}

}  // namespace

cudaError_t configure_rows_kernels() {
    cudaError_t e = configure_dim<float, 64>();
    if (e == cudaSuccess) e = configure_dim<float, 128>();
    if (e == cudaSuccess) e = configure_dim<__half, 64>();
    if (e == cudaSuccess) e = configure_dim<__half, 128>();
    if (e == cudaSuccess) e = configure_dim<__nv_bfloat16, 64>();
    if (e == cudaSuccess) e = configure_dim<__nv_bfloat16, 128>();
    if (e == cudaSuccess) e = configure_rows_tc();
    return e;
}

cudaError_t launch_rows(const RowsParams& p, RowType type, int head_dim, bool paged, int num_sms, cudaStream_t st) {
    // more rows than one CTA of this kernel takes would read the keys again; and keys that a cluster of the fewest warps
    // cannot share (kWarpKeys)
    const long long rows = (long long)p.max_q * p.group;
    if (rows > (type == RowType::f32 ? 8 : kRowsMax) ||
        (type != RowType::f32 && rows > 1 && p.max_kv > 16 * kWarps16 * kWarpKeys))
        return launch_rows_tc(p, type, head_dim, paged, num_sms, st);
    switch (type) {
        case RowType::f32: return launch_by_dim<float>(p, head_dim, paged, num_sms, st);
        case RowType::f16: return launch_by_dim<__half>(p, head_dim, paged, num_sms, st);
        default: return launch_by_dim<__nv_bfloat16>(p, head_dim, paged, num_sms, st);
    }
}

}  // namespace nllb
