"""What nllb_attn_append refuses before touching a GPU."""
import ctypes

import pytest

import nllb_attn as na

P = 1 << 20  # an address that is never followed


def args(**kw):
    a = dict(q=P, q_out=P, k_new=P, v_new=P, k_pages=P, v_pages=P, page_table=P, kv_len=P, inv_freq=P, dtype=na.BF16,
             head_dim=64, n_heads=4, n_kv_heads=2, n_seq=2, q_rows=4, max_q=2, max_kv=64, n_pages=8, page_size=16,
             page_table_stride=4, rot_dim=64, rot_pairs=na.ROT_HALVES, q_stride_row=256, q_stride_head=64,
             q_out_stride_row=256, q_out_stride_head=64, k_new_stride_row=128, k_new_stride_head=64, v_new_stride_row=128,
             v_new_stride_head=64, k_stride_page=2048, k_stride_slot=128, k_stride_head=64, v_stride_page=2048,
             v_stride_slot=128, v_stride_head=64)
    a.update(kw)
    return na.AppendArgs(**a)


def status(a):
    lib = na.load()
    rc = lib.nllb_attn_append(None, ctypes.byref(a))
    return rc, lib.nllb_attn_last_error().decode()


@pytest.mark.parametrize("kw,code,needle", [
    (dict(dtype=3), na.EINVAL, "dtype"),
    (dict(head_dim=96), na.EINVAL, "head_dim"),
    (dict(n_heads=3), na.EINVAL, "n_heads"),
    (dict(n_heads=2048), na.EINVAL, "heads"),
    (dict(n_seq=-1), na.EINVAL, "negative"),
    (dict(n_seq=70000), na.ECAPACITY, "sequences"),
    (dict(max_q=2 ** 30), na.ECAPACITY, "rows"),
    (dict(k_new=None), na.EINVAL, "required"),
    (dict(v_pages=None), na.EINVAL, "required"),
    (dict(page_table=None), na.EINVAL, "required"),
    (dict(q=None), na.EINVAL, "together"),
    (dict(q_out=None), na.EINVAL, "together"),
    (dict(rot_dim=8), na.EINVAL, "rot_dim"),
    (dict(rot_dim=80), na.EINVAL, "rot_dim"),
    (dict(rot_dim=-16), na.EINVAL, "rot_dim"),
    (dict(inv_freq=None), na.EINVAL, "inv_freq"),
    (dict(rot_dim=0), na.EINVAL, "inv_freq"),
    (dict(rot_pairs=2), na.EINVAL, "rot_pairs"),
    (dict(n_pages=0), na.EINVAL, "n_pages"),
    (dict(page_size=0), na.EINVAL, "page_size"),
    (dict(max_kv=65), na.EINVAL, "page_table_stride"),
    (dict(q_rows=3), na.EINVAL, "q_rows"),
    (dict(k_new=P + 8), na.EINVAL, "16-byte"),
    (dict(q_out_stride_row=-256), na.EINVAL, "stride"),
    (dict(v_new_stride_head=4), na.EINVAL, "stride"),
    (dict(q_out=2 * P, q_out_stride_row=0), na.EINVAL, "overlap"),
    (dict(k_stride_page=0), na.EINVAL, "overlap"),
    (dict(v_stride_head=0), na.EINVAL, "overlap"),
    (dict(q_out_stride_row=512), na.EINVAL, "strides"),
])
def test_refuses(kw, code, needle):
    rc, text = status(args(**kw))
    assert rc == code and needle in text


@pytest.mark.parametrize("kw", [dict(), dict(q=None, q_out=None), dict(rot_dim=0, inv_freq=None), dict(q_out=2 * P, q_out_stride_row=512),
                                dict(n_seq=0), dict(max_q=0), dict(q_rows=0)])
def test_valid_arguments_still_need_a_context(kw):
    rc, text = status(args(**kw))
    assert rc == na.EINVAL and "ctx" in text
    assert na.load().nllb_attn_append(None, None) == na.EINVAL


def test_binding_checks_tensors():
    import torch
    k, q = torch.zeros(4, 2, 64), torch.zeros(4, 4, 64)
    pages, table, lens = torch.zeros(3, 16, 2, 64), torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    make = na.Context.append_args
    ok = (k, k, pages, pages, table, lens)
    a = make(*ok, q=q, q_out=q, inv_freq=torch.ones(32))
    assert (a.rot_dim, a.rot_pairs, a.n_heads, a.max_q, a.max_kv) == (64, na.ROT_HALVES, 4, 2, 32)
    make(*ok)
    for at, x in ((1, k[:3]), (3, pages[:, :8]), (2, pages.half()), (4, table.long()), (4, table[:1]), (5, lens.long()),
                  (0, k.double())):
        bad = list(ok)
        bad[at] = x
        with pytest.raises(ValueError):
            make(*bad)
    for kw in (dict(q=q), dict(q=q[:3], q_out=q[:3]), dict(q=q, q_out=q[:, :2]), dict(q=q.half(), q_out=q), dict(pairs="thirds"),
               dict(inv_freq=torch.ones(32).double()), dict(position=torch.ones(3, dtype=torch.int32)), dict(max_kv=33),
               dict(q_len=lens[:1])):
        with pytest.raises(ValueError):
            make(*ok, **kw)
