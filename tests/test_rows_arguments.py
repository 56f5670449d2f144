"""Arguments of nllb_attn_paged, nllb_attn_cross_rows and nllb_sample that are taken, or refused, before touching a GPU;
beside test_rows_sample_refusals.py."""
import ctypes

import pytest

import nllb_attn as na
from test_rows_sample_refusals import P, cross_args, paged_args


def status(fn, a):
    lib = na.load()
    rc = getattr(lib, fn)(None, ctypes.byref(a))
    return rc, lib.nllb_attn_last_error().decode()


@pytest.mark.parametrize("kw", [
    dict(n_seq=4096, max_kv=1 << 20, page_table_stride=1 << 16),  # 2^32 places in the tables, of which few are used
    dict(n_seq=65535, max_q=1 << 16, q_start=P, q_len=P, q_rows=70000),  # one long chunk among single tokens
    dict(n_seq=65535, max_kv=1 << 30, page_size=1 << 20, page_table_stride=1 << 10),
])
def test_paged_takes_wide_bounds(kw):
    """Bounds of single sequences: their products number nothing where the starts are given."""
    rc, text = status("nllb_attn_paged", paged_args(**dict(dict(q_rows=65535 * 2), **kw)))
    assert rc == na.EINVAL and "ctx" in text  # all that is left to refuse


def test_cross_rows_takes_wide_bounds_with_starts():
    kw = dict(n_seq=40000, max_q=1 << 16, max_kv=1 << 18, q_start=P, q_len=P, kv_start=P, q_rows=90000, kv_rows=1 << 19)
    rc, text = status("nllb_attn_cross_rows", cross_args(**kw))
    assert rc == na.EINVAL and "ctx" in text


@pytest.mark.parametrize("fn,kw,needle", [
    ("nllb_attn_paged", dict(n_seq=65535, max_q=1 << 16, q_rows=2 ** 31 - 1), "q_rows"),
    ("nllb_attn_cross_rows", dict(n_seq=65535, max_q=1 << 16, q_rows=2 ** 31 - 1, max_kv=1), "q_rows"),
    ("nllb_attn_cross_rows", dict(n_seq=65535, max_q=1, q_rows=70000, max_kv=1 << 16, kv_rows=2 ** 31 - 1), "kv_rows"),
])
def test_rows_without_starts_have_to_exist(fn, kw, needle):
    a = paged_args(**kw) if fn.endswith("paged") else cross_args(**kw)
    rc, text = status(fn, a)
    assert rc == na.EINVAL and needle in text


@pytest.mark.parametrize("kw", [dict(out_stride_row=0), dict(out_stride_head=0), dict(out_stride_head=32)])
def test_overlapping_outputs_are_refused(kw):
    for fn, a in (("nllb_attn_paged", paged_args(**kw)), ("nllb_attn_cross_rows", cross_args(**kw))):
        rc, text = status(fn, a)
        assert rc == na.EINVAL and "overlap" in text


@pytest.mark.parametrize("kw", [dict(k_stride_page=0), dict(v_stride_slot=0), dict(k_stride_head=0), dict(v_stride_page=32)])
def test_overlapping_pages_are_refused_where_they_are_written(kw):
    new = dict(k_new=P, v_new=P, k_new_stride_row=128, k_new_stride_head=64, v_new_stride_row=128, v_new_stride_head=64)
    rc, text = status("nllb_attn_paged", paged_args(**new, **kw))
    assert rc == na.EINVAL and "overlap" in text
    for read in (paged_args(**kw), paged_args(**new)):  # read only, or apart
        rc, text = status("nllb_attn_paged", read)
        assert rc == na.EINVAL and "ctx" in text


def test_single_rows_take_any_output_stride():
    rc, text = status("nllb_attn_paged", paged_args(n_seq=1, q_rows=1, max_q=1, out_stride_row=0))
    assert rc == na.EINVAL and "ctx" in text


class FakeDevice:
    def __init__(self, type, index):
        self.type, self.index = type, index


def test_binding_refuses_tensors_of_another_device():
    """Arguments built from CPU tensors, or those of another GPU, never reach the library."""
    import torch
    q, lens = torch.zeros(4, 2, 64), torch.ones(2, dtype=torch.int32)
    pages, table = torch.zeros(3, 16, 2, 64), torch.zeros(2, 2, dtype=torch.int32)
    c = object.__new__(na.Context)  # a context without a GPU: the library refuses its handle
    c.lib, c.handle, c.device = na.load(), None, 1
    for call, args in ((c.paged, na.Context.paged_args(q, pages, pages, table, lens, q)),
                       (c.cross_rows, na.Context.cross_rows_args(q, q, q, q, lens))):
        with pytest.raises(ValueError, match="cpu"):
            call(args)
        args.tensors_on = FakeDevice("cuda", 0)
        with pytest.raises(ValueError, match="cuda:1"):
            call(args)
        args.tensors_on = FakeDevice("cuda", 1)
        with pytest.raises(na.NllbAttnError, match="ctx"):
            call(args)
    with pytest.raises(na.NllbAttnError):
        c.paged(paged_args())  # filled by hand


@pytest.mark.gpu
def test_binding_refuses_cpu_tensors_on_a_gpu(cuda_device):
    import torch
    q, lens = torch.zeros(4, 2, 64), torch.ones(2, dtype=torch.int32)
    with na.Context(0, n_layers=0, max_sentences=0) as ctx:
        with pytest.raises(ValueError, match="cpu"):
            ctx.cross_rows(na.Context.cross_rows_args(q, q, q, q, lens))
        ctx.sync()
