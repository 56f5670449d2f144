"""What nllb_attn_paged, nllb_attn_cross_rows and nllb_sample refuse before touching a GPU."""
import ctypes

import pytest

import nllb_attn as na

# an address that is never followed: every call here is refused, or has nothing to do
P = 1 << 20


def sample_args(**kw):
    a = dict(logits=P, ld=100, dtype=na.F32, vocab=100, rows=2, u=P, out_tok=P)
    a.update(kw)
    return na.SampleArgs(**a)


@pytest.mark.parametrize("kw,status,needle", [
    (dict(dtype=5), na.EINVAL, "dtype"),
    (dict(rows=-1), na.EINVAL, "rows"),
    (dict(vocab=0), na.EINVAL, "vocab"),
    (dict(vocab=524289, ld=524289), na.ECAPACITY, "vocab"),
    (dict(logits=None), na.EINVAL, "required"),
    (dict(u=None), na.EINVAL, "required"),
    (dict(out_tok=None), na.EINVAL, "required"),
    (dict(ld=99), na.EINVAL, "ld"),
    (dict(logits=P + 2), na.EINVAL, "aligned"),
])
def test_sample_refuses(kw, status, needle):
    lib = na.load()
    assert lib.nllb_sample(ctypes.byref(sample_args(**kw)), None) == status
    assert needle in lib.nllb_attn_last_error().decode()


def test_sample_of_no_rows_is_nothing():
    lib = na.load()
    assert lib.nllb_sample(ctypes.byref(sample_args(rows=0, logits=None, u=None, out_tok=None)), None) == na.OK
    assert lib.nllb_sample(None, None) == na.EINVAL


def test_attention_calls_refuse_null():
    lib = na.load()
    assert lib.nllb_attn_paged(None, ctypes.byref(na.PagedArgs())) == na.EINVAL
    assert lib.nllb_attn_cross_rows(None, ctypes.byref(na.CrossRowsArgs())) == na.EINVAL


def test_binding_checks_tensors():
    import torch
    q = torch.zeros(4, 2, 64)
    pages, table, lens = torch.zeros(3, 16, 2, 64), torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    make = na.Context.paged_args
    make(q, pages, pages, table, lens, q)  # nothing is followed here
    for args, kw in [
        ((q, pages, pages, table, lens, q[:3]), {}),
        ((q, pages, pages.half(), table, lens, q), {}),
        ((q, pages, pages[:, :8], table, lens, q), {}),
        ((q, pages, pages, table.long(), lens, q), {}),
        ((q, pages, pages, table[:1], lens, q), {}),
        ((q, pages, pages, table, lens.long(), q), {}),
        ((q, pages, pages, table, lens, q), dict(k_new=q)),
        ((q, pages, pages, table, lens, q), dict(max_kv=33)),
        ((q, pages, pages, table, lens, q), dict(q_len=lens[:1])),
        ((q.double(), pages, pages, table, lens, q), {}),
    ]:
        with pytest.raises(ValueError):
            make(*args, **kw)
    with pytest.raises(ValueError):
        na.Context.cross_rows_args(q, q, q, q, lens, key_mask=torch.ones(3, dtype=torch.uint8))
    with pytest.raises(ValueError):
        na.sample(torch.zeros(4, 8).t(), torch.zeros(8))


def paged_args(**kw):
    a = dict(q=P, k_pages=P, v_pages=P, out=P, page_table=P, kv_len=P, dtype=na.BF16, head_dim=64, n_heads=4,
             n_kv_heads=2, n_seq=2, q_rows=4, max_q=2, max_kv=64, n_pages=8, page_size=16, page_table_stride=4,
             scale=0.125, q_stride_row=256, q_stride_head=64, out_stride_row=256, out_stride_head=64,
             k_stride_page=2048, k_stride_slot=128, k_stride_head=64, v_stride_page=2048, v_stride_slot=128,
             v_stride_head=64)
    a.update(kw)
    return na.PagedArgs(**a)


def cross_args(**kw):
    a = dict(q=P, k=P, v=P, out=P, kv_len=P, dtype=na.F32, head_dim=128, n_heads=4, n_kv_heads=4, n_seq=2, q_rows=4,
             kv_rows=20, max_q=2, max_kv=10, scale=0.1, q_stride_row=512, q_stride_head=128, k_stride_row=512,
             k_stride_head=128, v_stride_row=512, v_stride_head=128, out_stride_row=512, out_stride_head=128)
    a.update(kw)
    return na.CrossRowsArgs(**a)


COMMON = [
    (dict(dtype=3), na.EINVAL, "dtype"),
    (dict(head_dim=32), na.EINVAL, "head_dim"),
    (dict(n_heads=3), na.EINVAL, "n_heads"),
    (dict(n_kv_heads=0), na.EINVAL, "n_heads"),
    (dict(n_seq=-1), na.EINVAL, "negative"),
    (dict(n_seq=70000), na.ECAPACITY, "sequences"),
    (dict(max_q=2 ** 30), na.ECAPACITY, "rows"),
    (dict(scale=0.0), na.EINVAL, "scale"),
    (dict(scale=float("nan")), na.EINVAL, "scale"),
    (dict(q=None), na.EINVAL, "required"),
    (dict(out=None), na.EINVAL, "required"),
    (dict(kv_len=None), na.EINVAL, "required"),
    (dict(q=P + 8), na.EINVAL, "16-byte"),
    (dict(q_stride_row=-256), na.EINVAL, "stride"),
    (dict(out_stride_head=66), na.EINVAL, "stride"),
    (dict(q_rows=3), na.EINVAL, "q_rows"),
]


@pytest.mark.parametrize("kw,status,needle", COMMON + [
    (dict(page_table=None), na.EINVAL, "required"),
    (dict(k_new=P), na.EINVAL, "together"),
    (dict(n_pages=0), na.EINVAL, "n_pages"),
    (dict(page_size=0), na.EINVAL, "page_size"),
    (dict(max_kv=65), na.EINVAL, "page_table_stride"),
    (dict(k_stride_slot=4), na.EINVAL, "stride"),
    (dict(k_new=P, v_new=P + 4), na.EINVAL, "16-byte"),
])
def test_paged_refuses(kw, status, needle):
    lib = na.load()  # (the arguments are looked at before the context)
    assert lib.nllb_attn_paged(None, ctypes.byref(paged_args(**kw))) == status
    assert needle in lib.nllb_attn_last_error().decode()


@pytest.mark.parametrize("kw,status,needle", COMMON + [
    (dict(k=None), na.EINVAL, "required"),
    (dict(kv_rows=-1), na.EINVAL, "negative"),
    (dict(kv_rows=19), na.EINVAL, "kv_rows"),
    (dict(v_stride_row=510), na.EINVAL, "stride"),
])
def test_cross_rows_refuses(kw, status, needle):
    lib = na.load()
    assert lib.nllb_attn_cross_rows(None, ctypes.byref(cross_args(**kw))) == status
    assert needle in lib.nllb_attn_last_error().decode()


def test_valid_arguments_still_need_a_context():
    lib = na.load()
    for fn, a in ((lib.nllb_attn_paged, paged_args()), (lib.nllb_attn_cross_rows, cross_args())):
        assert fn(None, ctypes.byref(a)) == na.EINVAL and "ctx" in lib.nllb_attn_last_error().decode()
        assert fn(None, None) == na.EINVAL


@pytest.mark.gpu
def test_nothing_to_do_is_ok(cuda_device):
    with na.Context(0, n_layers=0, max_sentences=0) as ctx:
        for kw in (dict(n_seq=0), dict(max_q=0), dict(q_rows=0)):
            assert ctx.lib.nllb_attn_paged(ctx.handle, ctypes.byref(paged_args(q=None, **kw))) == na.OK
            assert ctx.lib.nllb_attn_cross_rows(ctx.handle, ctypes.byref(cross_args(q=None, **kw))) == na.OK
        ctx.sync()
