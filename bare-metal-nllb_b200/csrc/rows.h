// rows.h -- parameters and launchers of the attention over many query rows
// against keys of another length: a chunk of new tokens over a paged cache
// (nllb_attn_paged, and nllb_attn_window with a sliding window) and target rows
// over encoder states (nllb_attn_cross_rows).
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace nllb {

// Strides count elements of the type.  Query row r of a sequence's tile is
// (token r / group, query head kv_head * group + r % group), so all the query
// heads that share a key head read its rows together.
struct RowsParams {
    const void* q;
    const void* k;  // paged: page 0; else packed rows
    const void* v;
    const void* k_new;  // paged: rows of the chunk, written into the pages (null: already there)
    const void* v_new;
    void* k_w;  // paged: the pages again, written
    void* v_w;
    void* out;
    long long q_row, q_head, o_row, o_head;
    long long k_page, k_row, k_head, v_page, v_row, v_head;
    long long kn_row, kn_head, vn_row, vn_head;
    const int* q_start;  // null: sequence s starts at row s * max_q
    const int* q_len;    // null: max_q rows each
    const int* kv_start; // packed keys: null: s * max_kv
    const int* kv_len;
    const int* table;    // paged: [n_seq][table_ld]
    const uint8_t* mask; // packed keys: one byte per key row, 0 hides it (null: all visible)
    int n_seq, kv_heads, group;
    int q_rows, kv_rows, max_q, max_kv;
    int max_seen;  // keys that the rows of one CTA see, at most
    int window, sinks;  // paged: a token sees the last `window` positions and the first `sinks`; window 0: all
    int table_ld, n_pages, page;
    uint32_t page_mul;  // j / page = j * page_mul >> page_shr
    int page_shr;
    uint32_t group_mul;  // row / group = row * group_mul >> group_shr
    int group_shr;
    float scale_log2;  // scale * log2(e)
    int* err;
    bool expire;  // test: a wait of the tensor-core form runs out
};

enum class RowType { f32 = 0, f16 = 1, bf16 = 2 };

// nllb_attn_append: of `rows`, q, out (the turned queries), the chunk's rows, the pages, their lengths and tables.
struct AppendParams {
    RowsParams rows;
    const int* position;    // of each row of q (null: its place in the sequence)
    const float* inv_freq;  // [half]
    int half;               // pairs that are turned; 0: none
    bool neighbours;        // pairs (2i, 2i + 1), else (i, i + half)
};
cudaError_t launch_append(const AppendParams& p, RowType type, int head_dim, int num_sms, cudaStream_t st);

// Per-device kernel attributes; call once per device.
cudaError_t configure_rows_kernels();
cudaError_t configure_rows_tc();
cudaError_t launch_rows(const RowsParams& p, RowType type, int head_dim, bool paged, int num_sms, cudaStream_t st);
// the tensor-core form (rows_tc.cu), for launch_rows
cudaError_t launch_rows_tc(const RowsParams& p, RowType type, int head_dim, bool paged, int num_sms, cudaStream_t st);

}  // namespace nllb
