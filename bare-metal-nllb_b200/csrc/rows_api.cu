// rows_api.cu -- nllb_attn_paged and nllb_attn_cross_rows: argument checks and
// launch parameters.
#include <cmath>
#include <string>

#include "attn_internal.h"
#include "device_common.cuh"
#include "nllb_attn.h"
#include "rows.h"

namespace nllb {
int set_error(int status, const std::string& msg);  // nllb_attn.cu
}

using namespace nllb;

namespace {

int bad(const char* msg) { return set_error(NLLB_ATTN_EINVAL, msg); }

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int check_common(int dtype, int head_dim, int n_heads, int n_kv_heads, int n_seq, int q_rows, int max_q, int max_kv,
                 float scale) {
    if (dtype != NLLB_F32 && dtype != NLLB_F16 && dtype != NLLB_BF16) return bad("dtype must be NLLB_F32, NLLB_F16 or NLLB_BF16");
    if (head_dim != 64 && head_dim != 128) return bad("head_dim must be 64 or 128");
    if (n_heads < 1 || n_kv_heads < 1 || n_heads % n_kv_heads)
        return bad("n_heads must be a positive multiple of n_kv_heads");
    if (n_heads > 1024) return bad("at most 1024 heads");
    if (n_seq < 0 || q_rows < 0 || max_q < 0 || max_kv < 0) return bad("negative size");
    if (n_seq > 65535) return set_error(NLLB_ATTN_ECAPACITY, "at most 65535 sequences per call");
    // (n_seq * max_q and n_seq * max_kv number rows only where starts are NULL: they are held against q_rows and kv_rows)
    if ((long long)max_q * (n_heads / n_kv_heads) > (1 << 26) || max_kv > (1 << 30))
        return set_error(NLLB_ATTN_ECAPACITY, "more rows than a call takes");
    if (!(scale > 0.0f) || !std::isfinite(scale)) return bad("scale must be positive");
    return NLLB_ATTN_OK;
}

// One operand: 16-byte rows at non-negative strides.
bool rows_ok(const void* base, int dtype, int64_t a, int64_t b, int64_t c = 0) {
    const int64_t unit = dtype == NLLB_F32 ? 4 : 8;
    return aligned16(base) && a >= 0 && b >= 0 && c >= 0 && a % unit == 0 && b % unit == 0 && c % unit == 0;
}

// Rows that are written may not lie in one another: `n` of them `stride` apart.
bool apart(int64_t n, int64_t stride, int head_dim) { return n <= 1 || stride >= head_dim; }

// Division of a j < 2^30 by d: with 2^(b-1) < d <= 2^b the multiplier ceil(2^(30+b) / d) is too large by less than 1, so
// the quotient by less than 2^30 / 2^(30+b) <= 1 / d: it stays below the next whole number.
void set_division(int d, uint32_t* mul, int* shr) {
    int b = 0;
    while ((1LL << b) < d) ++b;
    *shr = 30 + b;
    *mul = (uint32_t)(((1ULL << *shr) + (uint64_t)d - 1) / (uint64_t)d);
}

int launch(nllb_attn_ctx* c, RowsParams& p, int dtype, int head_dim, bool paged) {
    if (!c) return bad("ctx is NULL");
    if (p.n_seq == 0) return NLLB_ATTN_OK;  // nothing to do
    p.err = c->err;
    set_division(p.group, &p.group_mul, &p.group_shr);
    cudaError_t e = cudaSetDevice(c->device);
    p.expire = c->expire_next_rows;
    c->expire_next_rows = false;
    if (e == cudaSuccess) e = launch_rows(p, static_cast<RowType>(dtype), head_dim, paged, c->num_sms, c->stream);
    if (e != cudaSuccess) return set_error(NLLB_ATTN_ECUDA, std::string("launch_rows: ") + cudaGetErrorString(e));
    return NLLB_ATTN_OK;
}

}  // namespace

extern "C" {

int nllb_attn_test_expire_next_rows_wait(nllb_attn_ctx* c) {
    if (!c) return bad("ctx is NULL");
    c->expire_next_rows = true;
    return NLLB_ATTN_OK;
}

int nllb_attn_paged(nllb_attn_ctx* c, const nllb_attn_paged_args* a) {
    if (!a) return bad("args is NULL");
    int rc = check_common(a->dtype, a->head_dim, a->n_heads, a->n_kv_heads, a->n_seq, a->q_rows, a->max_q, a->max_kv,
                          a->scale);
    if (rc) return rc;
    RowsParams p = {};
    if (a->n_seq == 0 || a->max_q == 0 || a->q_rows == 0) return launch(c, p, a->dtype, a->head_dim, true);
    if (!a->q || !a->k_pages || !a->v_pages || !a->out || !a->page_table || !a->kv_len)
        return bad("q, k_pages, v_pages, out, page_table and kv_len are required");
    if (!a->k_new != !a->v_new) return bad("k_new and v_new go together");
    if (a->n_pages < 1 || a->page_size < 1) return bad("n_pages and page_size must be >= 1");
    if (a->page_size > (1 << 30)) return set_error(NLLB_ATTN_ECAPACITY, "page_size above 2^30");
    if ((long long)a->page_table_stride * a->page_size < a->max_kv)
        return bad("page_table_stride * page_size must reach max_kv");
    if (!a->q_start && (long long)a->n_seq * a->max_q > a->q_rows) return bad("q_rows must reach n_seq * max_q");
    if (!rows_ok(a->q, a->dtype, a->q_stride_row, a->q_stride_head) ||
        !rows_ok(a->out, a->dtype, a->out_stride_row, a->out_stride_head) ||
        !rows_ok(a->k_pages, a->dtype, a->k_stride_page, a->k_stride_slot, a->k_stride_head) ||
        !rows_ok(a->v_pages, a->dtype, a->v_stride_page, a->v_stride_slot, a->v_stride_head) ||
        (a->k_new && (!rows_ok(a->k_new, a->dtype, a->k_new_stride_row, a->k_new_stride_head) ||
                      !rows_ok(a->v_new, a->dtype, a->v_new_stride_row, a->v_new_stride_head))))
        return bad("rows must be 16-byte aligned, strides non-negative multiples of 16 bytes");
    if (!apart(a->q_rows, a->out_stride_row, a->head_dim) || !apart(a->n_heads, a->out_stride_head, a->head_dim))
        return bad("out: strides below head_dim, its rows would overlap");
    auto pages_apart = [&](int64_t page, int64_t slot, int64_t head) {
        return apart(a->n_pages, page, a->head_dim) && apart(a->page_size, slot, a->head_dim) &&
               apart(a->n_kv_heads, head, a->head_dim);
    };
    if (a->k_new && !(pages_apart(a->k_stride_page, a->k_stride_slot, a->k_stride_head) &&
                      pages_apart(a->v_stride_page, a->v_stride_slot, a->v_stride_head)))
        return bad("k_pages, v_pages: strides below head_dim, the rows written would overlap");
    p.q = a->q, p.k = a->k_pages, p.v = a->v_pages, p.k_new = a->k_new, p.v_new = a->v_new;
    p.k_w = a->k_pages, p.v_w = a->v_pages, p.out = a->out;
    p.q_row = a->q_stride_row, p.q_head = a->q_stride_head, p.o_row = a->out_stride_row, p.o_head = a->out_stride_head;
    p.k_page = a->k_stride_page, p.k_row = a->k_stride_slot, p.k_head = a->k_stride_head;
    p.v_page = a->v_stride_page, p.v_row = a->v_stride_slot, p.v_head = a->v_stride_head;
    p.kn_row = a->k_new_stride_row, p.kn_head = a->k_new_stride_head;
    p.vn_row = a->v_new_stride_row, p.vn_head = a->v_new_stride_head;
    p.q_start = a->q_start, p.q_len = a->q_len, p.kv_len = a->kv_len, p.table = a->page_table;
    p.n_seq = a->n_seq, p.kv_heads = a->n_kv_heads, p.group = a->n_heads / a->n_kv_heads;
    p.q_rows = a->q_rows, p.max_q = a->max_q, p.max_kv = a->max_kv;
    p.table_ld = a->page_table_stride, p.n_pages = a->n_pages, p.page = a->page_size;
    set_division(a->page_size, &p.page_mul, &p.page_shr);
    p.scale_log2 = a->scale * kLog2e;
    return launch(c, p, a->dtype, a->head_dim, true);
}

int nllb_attn_cross_rows(nllb_attn_ctx* c, const nllb_attn_cross_rows_args* a) {
    if (!a) return bad("args is NULL");
    int rc = check_common(a->dtype, a->head_dim, a->n_heads, a->n_kv_heads, a->n_seq, a->q_rows, a->max_q, a->max_kv,
                          a->scale);
    if (rc) return rc;
    if (a->kv_rows < 0) return bad("negative size");
    RowsParams p = {};
    if (a->n_seq == 0 || a->max_q == 0 || a->q_rows == 0) return launch(c, p, a->dtype, a->head_dim, false);
    if (!a->q || !a->out || !a->kv_len || (a->kv_rows > 0 && (!a->k || !a->v)))
        return bad("q, k, v, out and kv_len are required");
    if (!a->q_start && (long long)a->n_seq * a->max_q > a->q_rows) return bad("q_rows must reach n_seq * max_q");
    if (!a->kv_start && (long long)a->n_seq * a->max_kv > a->kv_rows) return bad("kv_rows must reach n_seq * max_kv");
    if (!rows_ok(a->q, a->dtype, a->q_stride_row, a->q_stride_head) ||
        !rows_ok(a->out, a->dtype, a->out_stride_row, a->out_stride_head) ||
        !rows_ok(a->k, a->dtype, a->k_stride_row, a->k_stride_head) ||
        !rows_ok(a->v, a->dtype, a->v_stride_row, a->v_stride_head))
        return bad("rows must be 16-byte aligned, strides non-negative multiples of 16 bytes");
    if (!apart(a->q_rows, a->out_stride_row, a->head_dim) || !apart(a->n_heads, a->out_stride_head, a->head_dim))
        return bad("out: strides below head_dim, its rows would overlap");
    p.q = a->q, p.k = a->k, p.v = a->v, p.out = a->out;
    p.q_row = a->q_stride_row, p.q_head = a->q_stride_head, p.o_row = a->out_stride_row, p.o_head = a->out_stride_head;
    p.k_row = a->k_stride_row, p.k_head = a->k_stride_head, p.v_row = a->v_stride_row, p.v_head = a->v_stride_head;
    p.q_start = a->q_start, p.q_len = a->q_len, p.kv_start = a->kv_start, p.kv_len = a->kv_len, p.mask = a->key_mask;
    p.n_seq = a->n_seq, p.kv_heads = a->n_kv_heads, p.group = a->n_heads / a->n_kv_heads;
    p.q_rows = a->q_rows, p.kv_rows = a->kv_rows, p.max_q = a->max_q, p.max_kv = a->max_kv;
    p.page = 1;
    p.scale_log2 = a->scale * kLog2e;
    return launch(c, p, a->dtype, a->head_dim, false);
}

}  // extern "C"
