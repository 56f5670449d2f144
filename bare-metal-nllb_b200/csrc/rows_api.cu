// rows_api.cu -- nllb_attn_paged, nllb_attn_window, nllb_attn_cross_rows and
// nllb_attn_append: argument checks and launch parameters.
#include <algorithm>
#include <cmath>
#include <string>
#include <utility>

#include "attn_internal.h"
#include "device_common.cuh"
#include "nllb_attn.h"
#include "overlap.h"
#include "rows.h"

namespace nllb {
int set_error(int status, const std::string& msg);  // nllb_attn.cu
}

using namespace nllb;

namespace {

// The context's device for the time of a call, then the caller's again.
struct OnDevice {
    int before = -1;
    cudaError_t status;
    explicit OnDevice(int device) {
        status = cudaGetDevice(&before);
        if (status == cudaSuccess && before != device) status = cudaSetDevice(device);
    }
    ~OnDevice() {
        if (before >= 0) cudaSetDevice(before);
    }
};

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

int check_pages(int n_pages, int page_size, int table_stride, int max_kv) {
    if (n_pages < 1 || page_size < 1) return bad("n_pages and page_size must be >= 1");
    if (page_size > (1 << 30)) return set_error(NLLB_ATTN_ECAPACITY, "page_size above 2^30");
    if ((long long)table_stride * page_size < max_kv) return bad("page_table_stride * page_size must reach max_kv");
    return NLLB_ATTN_OK;
}

// The slots of the pages, where they are written.
template <typename Args>
bool pages_apart(const Args& a) {
    return apart(a.n_pages, a.k_stride_page, a.head_dim) && apart(a.page_size, a.k_stride_slot, a.head_dim) &&
           apart(a.n_kv_heads, a.k_stride_head, a.head_dim) && apart(a.n_pages, a.v_stride_page, a.head_dim) &&
           apart(a.page_size, a.v_stride_slot, a.head_dim) && apart(a.n_kv_heads, a.v_stride_head, a.head_dim);
}

// The memory of rows of heads, where it is rows without gaps in them (else none: not looked at).
MemRows heads_of(const void* p, int64_t rows, int64_t row, int heads, int64_t head, int64_t dim, int size) {
    constexpr int64_t far = 1LL << 36;
    if (p && (heads == 1 || head == dim) && (rows == 1 || row >= heads * dim))
        return MemRows(p, rows, std::min(row, far) * size, heads * dim * size);
    if (p && (rows == 1 || row == dim) && head >= rows * dim) return MemRows(p, heads, std::min(head, far) * size, rows * dim * size);
    return MemRows(p, 0, 0, 0);
}

// The memory of pages of slots of heads.
MemRows pages_of(const void* p, int64_t pages, int64_t page, int64_t slots, int64_t slot, int heads, int64_t head, int64_t dim, int size) {
    const bool by_slot = (heads == 1 || head == dim) && (slots == 1 || slot == heads * dim);
    const bool by_head = (slots == 1 || slot == dim) && (heads == 1 || head == slots * dim);
    const int64_t len = slots * heads * dim;
    if (!p || !(by_slot || by_head) || (pages > 1 && page < len)) return MemRows(p, 0, 0, 0);
    return MemRows(p, pages, std::min<int64_t>(page, 1LL << 36) * size, len * size);
}

// Division of a j < 2^30 by d: with 2^(b-1) < d <= 2^b the multiplier ceil(2^(30+b) / d) is too large by less than 1, so
// the quotient by less than 2^30 / 2^(30+b) <= 1 / d: it stays below the next whole number.
void set_division(int d, uint32_t* mul, int* shr) {
    int b = 0;
    while ((1LL << b) < d) ++b;
    *shr = 30 + b;
    *mul = (uint32_t)(((1ULL << *shr) + (uint64_t)d - 1) / (uint64_t)d);
}

// Whether a wait of this call is to run out: the hook is for the next call, whatever becomes of it.
bool take_expire(nllb_attn_ctx* c) { return c && std::exchange(c->expire_next_rows, false); }

int launch(nllb_attn_ctx* c, RowsParams& p, int dtype, int head_dim, bool paged) {
    if (!c) return bad("ctx is NULL");
    if (p.n_seq == 0) return NLLB_ATTN_OK;  // nothing to do
    p.err = c->err;
    set_division(p.group, &p.group_mul, &p.group_shr);
    OnDevice on(c->device);
    cudaError_t e = on.status;
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

}  // extern "C"

namespace {

// window: 0 (every position up to its own is visible to a token), or the positions that are, and the first `sinks`.
int attend_paged(nllb_attn_ctx* c, const nllb_attn_paged_args* a, int window, int sinks, bool expire) {
    int rc = check_common(a->dtype, a->head_dim, a->n_heads, a->n_kv_heads, a->n_seq, a->q_rows, a->max_q, a->max_kv,
                          a->scale);
    if (rc) return rc;
    RowsParams p = {};
    p.expire = expire;
    if (a->n_seq == 0 || a->max_q == 0 || a->q_rows == 0) return launch(c, p, a->dtype, a->head_dim, true);
    if (!a->q || !a->k_pages || !a->v_pages || !a->out || !a->page_table || !a->kv_len)
        return bad("q, k_pages, v_pages, out, page_table and kv_len are required");
    if (!a->k_new != !a->v_new) return bad("k_new and v_new go together");
    rc = check_pages(a->n_pages, a->page_size, a->page_table_stride, a->max_kv);
    if (rc) return rc;
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
    if (a->k_new && !pages_apart(*a))
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
    p.max_seen = a->max_kv;
    if (window > 0 && window < a->max_kv) {  // (a wider one hides nothing)
        p.window = window, p.sinks = std::min(sinks, a->max_kv);
        // the rows of a CTA are those of 256 tokens at most, whose windows start one after the other
        p.max_seen = (int)std::min((long long)a->max_kv, (long long)p.sinks + window + std::min(a->max_q, 256) - 1);
    }
    return launch(c, p, a->dtype, a->head_dim, true);
}

}  // namespace

extern "C" {

int nllb_attn_paged(nllb_attn_ctx* c, const nllb_attn_paged_args* a) {
    const bool expire = take_expire(c);
    if (!a) return bad("args is NULL");
    return attend_paged(c, a, 0, 0, expire);
}

int nllb_attn_window(nllb_attn_ctx* c, const nllb_attn_window_args* a) {
    const bool expire = take_expire(c);
    if (!a) return bad("args is NULL");
    if (a->window < 1) return bad("window must be >= 1");
    if (a->sinks < 0) return bad("sinks must not be negative");
    return attend_paged(c, &a->cache, a->window, a->sinks, expire);
}

int nllb_attn_cross_rows(nllb_attn_ctx* c, const nllb_attn_cross_rows_args* a) {
    const bool expire = take_expire(c);
    if (!a) return bad("args is NULL");
    int rc = check_common(a->dtype, a->head_dim, a->n_heads, a->n_kv_heads, a->n_seq, a->q_rows, a->max_q, a->max_kv,
                          a->scale);
    if (rc) return rc;
    if (a->kv_rows < 0) return bad("negative size");
    RowsParams p = {};
    p.expire = expire;
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
    p.max_seen = a->max_kv;
    p.scale_log2 = a->scale * kLog2e;
    return launch(c, p, a->dtype, a->head_dim, false);
}

int nllb_attn_append(nllb_attn_ctx* c, const nllb_attn_append_args* a) {
    if (!a) return bad("args is NULL");
    int rc = check_common(a->dtype, a->head_dim, a->n_heads, a->n_kv_heads, a->n_seq, a->q_rows, a->max_q, a->max_kv, 1.0f);
    if (rc) return rc;
    if (!c && (a->n_seq == 0 || a->max_q == 0 || a->q_rows == 0)) return bad("ctx is NULL");
    if (a->n_seq == 0 || a->max_q == 0 || a->q_rows == 0) return NLLB_ATTN_OK;
    if (!a->k_new || !a->v_new || !a->k_pages || !a->v_pages || !a->page_table || !a->kv_len)
        return bad("k_new, v_new, k_pages, v_pages, page_table and kv_len are required");
    if (!a->q != !a->q_out) return bad("q and q_out go together");
    if (a->rot_dim < 0 || a->rot_dim > a->head_dim || a->rot_dim % 16)
        return bad("rot_dim must be a multiple of 16 up to head_dim");
    if ((a->rot_dim > 0) != (a->inv_freq != nullptr)) return bad("inv_freq goes with a rot_dim above 0");
    if (a->rot_pairs != NLLB_ROT_HALVES && a->rot_pairs != NLLB_ROT_NEIGHBOURS)
        return bad("rot_pairs must be NLLB_ROT_HALVES or NLLB_ROT_NEIGHBOURS");
    rc = check_pages(a->n_pages, a->page_size, a->page_table_stride, a->max_kv);
    if (rc) return rc;
    if (!a->q_start && (long long)a->n_seq * a->max_q > a->q_rows) return bad("q_rows must reach n_seq * max_q");
    if ((a->q && (!rows_ok(a->q, a->dtype, a->q_stride_row, a->q_stride_head) ||
                  !rows_ok(a->q_out, a->dtype, a->q_out_stride_row, a->q_out_stride_head))) ||
        !rows_ok(a->k_new, a->dtype, a->k_new_stride_row, a->k_new_stride_head) ||
        !rows_ok(a->v_new, a->dtype, a->v_new_stride_row, a->v_new_stride_head) ||
        !rows_ok(a->k_pages, a->dtype, a->k_stride_page, a->k_stride_slot, a->k_stride_head) ||
        !rows_ok(a->v_pages, a->dtype, a->v_stride_page, a->v_stride_slot, a->v_stride_head))
        return bad("rows must be 16-byte aligned, strides non-negative multiples of 16 bytes");
    if (a->q && (!apart(a->q_rows, a->q_out_stride_row, a->head_dim) || !apart(a->n_heads, a->q_out_stride_head, a->head_dim)))
        return bad("q_out: strides below head_dim, its rows would overlap");
    if (a->q == a->q_out && a->q && (a->q_stride_row != a->q_out_stride_row || a->q_stride_head != a->q_out_stride_head))
        return bad("q turned in its place keeps its strides");
    if (!pages_apart(*a)) return bad("k_pages, v_pages: strides below head_dim, the rows written would overlap");
    if (!c) return bad("ctx is NULL");
    const int size = a->dtype == NLLB_F32 ? 4 : 2;
    const MemRows in[3] = {heads_of(a->k_new, a->q_rows, a->k_new_stride_row, a->n_kv_heads, a->k_new_stride_head, a->head_dim, size),
                           heads_of(a->v_new, a->q_rows, a->v_new_stride_row, a->n_kv_heads, a->v_new_stride_head, a->head_dim, size),
                           heads_of(a->q, a->q_rows, a->q_stride_row, a->n_heads, a->q_stride_head, a->head_dim, size)};
    const MemRows out[3] = {
        pages_of(a->k_pages, a->n_pages, a->k_stride_page, a->page_size, a->k_stride_slot, a->n_kv_heads, a->k_stride_head, a->head_dim, size),
        pages_of(a->v_pages, a->n_pages, a->v_stride_page, a->page_size, a->v_stride_slot, a->n_kv_heads, a->v_stride_head, a->head_dim, size),
        heads_of(a->q_out, a->q_rows, a->q_out_stride_row, a->n_heads, a->q_out_stride_head, a->head_dim, size)};
    for (int i = 0; i < 3; ++i)
        for (int j = 0; j < 3; ++j)
            if ((meet(out[i], in[j]) && !(i == 2 && j == 2 && a->q == a->q_out)) || (j < i && meet(out[i], out[j])))
                return bad("pages and q_out may not overlap q, k_new, v_new or one another (q_out may be q)");
    AppendParams p = {};
    RowsParams& r = p.rows;
    r.q = a->q, r.out = a->q_out, r.k_new = a->k_new, r.v_new = a->v_new, r.k_w = a->k_pages, r.v_w = a->v_pages;
    r.q_row = a->q_stride_row, r.q_head = a->q_stride_head, r.o_row = a->q_out_stride_row, r.o_head = a->q_out_stride_head;
    r.k_page = a->k_stride_page, r.k_row = a->k_stride_slot, r.k_head = a->k_stride_head;
    r.v_page = a->v_stride_page, r.v_row = a->v_stride_slot, r.v_head = a->v_stride_head;
    r.kn_row = a->k_new_stride_row, r.kn_head = a->k_new_stride_head;
    r.vn_row = a->v_new_stride_row, r.vn_head = a->v_new_stride_head;
    r.q_start = a->q_start, r.q_len = a->q_len, r.kv_len = a->kv_len, r.table = a->page_table;
    r.n_seq = a->n_seq, r.kv_heads = a->n_kv_heads, r.group = a->n_heads / a->n_kv_heads;
    r.q_rows = a->q_rows, r.max_q = a->max_q, r.max_kv = a->max_kv;
    r.table_ld = a->page_table_stride, r.n_pages = a->n_pages, r.page = a->page_size;
    set_division(a->page_size, &r.page_mul, &r.page_shr);
    r.err = c->err;
    p.position = a->position, p.inv_freq = a->inv_freq, p.half = a->rot_dim / 2;
    p.neighbours = a->rot_pairs == NLLB_ROT_NEIGHBOURS;
    OnDevice on(c->device);
    cudaError_t e = on.status;
    if (e == cudaSuccess) e = launch_append(p, static_cast<RowType>(a->dtype), a->head_dim, c->num_sms, c->stream);
    if (e != cudaSuccess) return set_error(NLLB_ATTN_ECUDA, std::string("launch_append: ") + cudaGetErrorString(e));
    return NLLB_ATTN_OK;
}

}  // extern "C"
