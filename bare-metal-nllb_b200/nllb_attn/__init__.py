"""ctypes binding of libnllb_attn.so, the C ABI declared in include/nllb_attn.h.

The product is the shared library; this module only gives Python callers
(tests, bench.py) the same calls a C host makes.  Device-pointer calls take
torch CUDA tensors (or raw integer addresses); ``*_host`` calls take numpy
arrays.  Nothing here computes attention: every call goes through the
library, and a missing library raises at import of :func:`load`.
"""
from __future__ import annotations

import ctypes
import os
from typing import Optional, Sequence

PKG_DIR = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB_PATH = os.path.join(PKG_DIR, "libnllb_attn.so")

OK, EINVAL, ECAPACITY, ECUDA, ETIMEOUT, ENODEV, ESTATE = range(7)

# Every function include/nllb_attn.h declares, with (restype, argtypes).
_c_int, _c_void_p, _c_size_t = ctypes.c_int, ctypes.c_void_p, ctypes.c_size_t
_fp = ctypes.c_void_p  # float*/const float*/int* passed as raw addresses


class Dims(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in (
        "n_layers", "n_heads", "head_dim", "max_sentences", "n_beams", "max_tgt", "max_src")]


class PrefillArgs(ctypes.Structure):
    _fields_ = [
        ("q", _fp), ("k", _fp), ("v", _fp), ("out", _fp),
        ("batch", ctypes.c_int), ("n_heads", ctypes.c_int), ("seq_len", ctypes.c_int),
        ("head_dim", ctypes.c_int),
        ("stride_batch", ctypes.c_int64), ("stride_head", ctypes.c_int64),
        ("stride_row", ctypes.c_int64),
        ("valid_len", _fp), ("mask", _fp),
        ("mask_stride_batch", ctypes.c_int64), ("mask_stride_head", ctypes.c_int64),
        ("scale", ctypes.c_float),
    ]


class TranslateOpts(ctypes.Structure):
    _fields_ = [("max_gen", ctypes.c_int), ("repetition_penalty", ctypes.c_float),
                ("no_repeat_ngram", ctypes.c_int)]


class TranslateStats(ctypes.Structure):
    _fields_ = [("encode_ms", ctypes.c_double), ("decode_ms", ctypes.c_double),
                ("steps", ctypes.c_int), ("tokens_out", ctypes.c_longlong)]


class KernelProfile(ctypes.Structure):
    _fields_ = [("name", ctypes.c_char * 32), ("launches", ctypes.c_longlong), ("ms", ctypes.c_double),
                ("flops", ctypes.c_double), ("bytes", ctypes.c_double)]


F32, F16, BF16 = range(3)
SAMPLE_TIMEOUT = -2


class PagedArgs(ctypes.Structure):
    _fields_ = ([(n, _fp) for n in ("q", "k_new", "v_new", "k_pages", "v_pages", "out", "q_start", "q_len", "kv_len",
                                    "page_table")]
                + [(n, ctypes.c_int) for n in ("dtype", "head_dim", "n_heads", "n_kv_heads", "n_seq", "q_rows",
                                               "max_q", "max_kv", "n_pages", "page_size", "page_table_stride")]
                + [("scale", ctypes.c_float)]
                + [(n, ctypes.c_int64) for n in (
                    "q_stride_row", "q_stride_head", "out_stride_row", "out_stride_head", "k_new_stride_row",
                    "k_new_stride_head", "v_new_stride_row", "v_new_stride_head", "k_stride_page", "k_stride_slot",
                    "k_stride_head", "v_stride_page", "v_stride_slot", "v_stride_head")])


class CrossRowsArgs(ctypes.Structure):
    _fields_ = ([(n, _fp) for n in ("q", "k", "v", "out", "q_start", "q_len", "kv_start", "kv_len", "key_mask")]
                + [(n, ctypes.c_int) for n in ("dtype", "head_dim", "n_heads", "n_kv_heads", "n_seq", "q_rows",
                                               "kv_rows", "max_q", "max_kv")]
                + [("scale", ctypes.c_float)]
                + [(n, ctypes.c_int64) for n in (
                    "q_stride_row", "q_stride_head", "k_stride_row", "k_stride_head", "v_stride_row",
                    "v_stride_head", "out_stride_row", "out_stride_head")])


class SampleArgs(ctypes.Structure):
    _fields_ = [("logits", _fp), ("ld", ctypes.c_longlong), ("dtype", ctypes.c_int), ("vocab", ctypes.c_int),
                ("rows", ctypes.c_int), ("temperature", _fp), ("top_k", _fp), ("top_p", _fp), ("min_p", _fp),
                ("u", _fp), ("out_tok", _fp), ("out_logp", _fp)]


PROF_CLASSES = 14

SIGNATURES = {
    "nllb_attn_create": (_c_int, [_c_int, ctypes.POINTER(Dims), ctypes.POINTER(_c_void_p)]),
    "nllb_attn_destroy": (None, [_c_void_p]),
    "nllb_attn_device_bytes": (_c_size_t, [ctypes.POINTER(Dims)]),
    "nllb_attn_set_stream": (_c_int, [_c_void_p, _c_void_p]),
    "nllb_attn_get_stream": (_c_void_p, [_c_void_p]),
    "nllb_attn_sync": (_c_int, [_c_void_p]),
    "nllb_attn_reset": (_c_int, [_c_void_p]),
    "nllb_attn_strerror": (ctypes.c_char_p, [_c_int]),
    "nllb_attn_last_error": (ctypes.c_char_p, []),
    "nllb_attn_prefill": (_c_int, [_c_void_p, ctypes.POINTER(PrefillArgs)]),
    "nllb_attn_prefill_host": (_c_int, [_c_void_p, ctypes.POINTER(PrefillArgs)]),
    "nllb_attn_decode_self": (_c_int, [_c_void_p, _c_int, _c_int, _c_int, _fp, _fp, _fp, _fp]),
    "nllb_attn_decode_self_host": (_c_int, [_c_void_p, _c_int, _c_int, _c_int, _fp, _fp, _fp, _fp]),
    "nllb_attn_reorder": (_c_int, [_c_void_p, _c_int, _fp]),
    "nllb_attn_reorder_host": (_c_int, [_c_void_p, _c_int, _fp]),
    "nllb_attn_test_expire_next_wait": (_c_int, [_c_void_p]),
    "nllb_attn_test_expire_next_cross_wait": (_c_int, [_c_void_p]),
    "nllb_attn_set_memory": (_c_int, [_c_void_p, _c_int, _c_int, _c_int, _fp, _fp,
                                      ctypes.c_int64, ctypes.c_int64]),
    "nllb_attn_set_memory_host": (_c_int, [_c_void_p, _c_int, _c_int, _c_int, _fp, _fp,
                                           ctypes.c_int64, ctypes.c_int64]),
    "nllb_attn_cross": (_c_int, [_c_void_p, _c_int, _c_int, _fp, _fp]),
    "nllb_attn_cross_host": (_c_int, [_c_void_p, _c_int, _c_int, _fp, _fp]),
    "nllb_attn_paged": (_c_int, [_c_void_p, ctypes.POINTER(PagedArgs)]),
    "nllb_attn_test_expire_next_rows_wait": (_c_int, [_c_void_p]),
    "nllb_attn_cross_rows": (_c_int, [_c_void_p, ctypes.POINTER(CrossRowsArgs)]),
    "nllb_attention_head": (None, [_fp, _fp, _fp, _fp, _fp, _fp, _c_int, _c_int]),
    "nllb_attention_head_flash": (None, [_fp, _fp, _fp, _fp, _fp, _c_int, _c_int]),
    "nllb_attn_last_status": (_c_int, []),
    # include/nllb_translate.h
    "nllb_model_load": (_c_int, [ctypes.c_char_p, _c_int, _c_int, _c_int, _c_int,
                                 ctypes.POINTER(_c_void_p)]),
    "nllb_model_free": (None, [_c_void_p]),
    "nllb_translate": (_c_int, [_c_void_p, _c_int, _fp, _fp, _c_int, ctypes.POINTER(TranslateOpts),
                                _fp, _fp, _fp, ctypes.POINTER(TranslateStats)]),
    "nllb_translate_margins": (_c_int, [_c_void_p, _c_int, _fp, _c_int]),
    "nllb_translate_profile": (_c_int, [_c_void_p, _c_int]),
    "nllb_translate_profile_read": (_c_int, [_c_void_p, ctypes.POINTER(KernelProfile), _c_int]),
    "nllb_linear_int8": (_c_int, [_fp, _c_int, _c_int, _fp, _fp, _fp, _c_int, _fp, _fp, _c_int, _c_void_p]),
    "nllb_linear_int8_status": (_c_int, []),
    "nllb_linear_int8_noalloc": (_c_int, [_fp, _c_int, _c_int, _fp, _fp, _fp, _c_int, _fp, _fp, _c_int,
                                          _c_void_p]),
    "nllb_linear_int8_noalloc_status": (_c_int, [_c_void_p]),
    "nllb_linear_prepare": (_c_int, [_fp, _fp, _fp, _c_int, _c_int, _c_void_p, ctypes.POINTER(_c_void_p)]),
    "nllb_linear_run": (_c_int, [_c_void_p, _fp, _c_int, _fp, _fp, _c_int, _c_void_p]),
    "nllb_linear_status": (_c_int, [_c_void_p]),
    "nllb_linear_test_expire_next_wait": (_c_int, [_c_void_p]),
    "nllb_linear_free": (None, [_c_void_p]),
    "nllb_apply_penalties": (_c_int, [_fp, ctypes.c_longlong, _c_int, _fp, _c_int, _fp, ctypes.c_float, _c_int,
                                      _c_void_p]),
    "nllb_logsoftmax_topk_ws_bytes": (_c_size_t, [_c_int, _c_int, _c_int]),
    "nllb_logsoftmax_topk": (_c_int, [_fp, ctypes.c_longlong, _c_int, _c_int, _c_int, _fp, _fp, _fp, _c_void_p]),
    "nllb_sample": (_c_int, [ctypes.POINTER(SampleArgs), _c_void_p]),
    "nllb_sample_test_expire_next_wait": (_c_int, []),
}

_LIB: Optional[ctypes.CDLL] = None


def load(path: str = LIB_PATH) -> ctypes.CDLL:
    """Load the library (once) and declare every signature."""
    global _LIB
    if _LIB is not None and path == LIB_PATH:
        return _LIB
    if not os.path.exists(path):
        raise FileNotFoundError(
            f"{path} is missing: build it with `make -C {PKG_DIR}` (nvcc, sm_100a)")
    lib = ctypes.CDLL(path)
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    if path == LIB_PATH:
        _LIB = lib
    return lib


class NllbAttnError(RuntimeError):
    def __init__(self, status: int, what: str, detail: str):
        super().__init__(f"{what}: status {status} ({detail})")
        self.status = status


def _check(lib, rc: int, what: str) -> None:
    if rc != OK:
        raise NllbAttnError(rc, what, lib.nllb_attn_last_error().decode())


def ptr(x) -> Optional[int]:
    """Raw address of a torch tensor, numpy array or int (None passes NULL)."""
    if x is None:
        return None
    if isinstance(x, int):
        return x
    if hasattr(x, "data_ptr"):
        if not x.is_contiguous():
            raise ValueError("tensor must be contiguous")
        return x.data_ptr()
    if hasattr(x, "ctypes"):
        if not x.flags["C_CONTIGUOUS"]:
            raise ValueError("array must be C-contiguous")
        return x.ctypes.data
    raise TypeError(f"cannot take the address of {type(x)!r}")


def _dtype_code(x) -> int:
    try:
        return {"torch.float32": F32, "torch.float16": F16, "torch.bfloat16": BF16}[str(x.dtype)]
    except KeyError:
        raise ValueError(f"dtype must be float32, float16 or bfloat16, not {x.dtype}") from None


def _rows(x, name, like, axes):
    """Address of a tensor of rows whose last axis is contiguous."""
    if x.dim() != axes or x.dtype != like.dtype or x.shape[-1] != like.shape[-1] or x.device != like.device:
        raise ValueError(f"{name} must have {axes} axes and the type, last size and device of q")
    if x.numel() and x.stride(-1) != 1:
        raise ValueError(f"the last axis of {name} must be contiguous")
    return x.data_ptr()


def _ints(x, name, n, like, dtype="torch.int32"):
    """Address of a contiguous device array of n entries (None passes NULL)."""
    if x is None:
        return None
    if str(x.dtype) != dtype or x.numel() != n or not x.is_contiguous() or x.device != like.device:
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of {n} entries on q's device")
    return x.data_ptr()


class Context:
    """One nllb_attn_ctx: caches, encoder memory and beam history on one GPU."""

    def __init__(self, device: int = 0, n_layers: int = 12, n_heads: int = 16,
                 max_sentences: int = 1, n_beams: int = 4, max_tgt: int = 256,
                 max_src: int = 512, lib: Optional[ctypes.CDLL] = None):
        self.lib = lib or load()
        self.dims = Dims(n_layers, n_heads, 64, max_sentences, n_beams, max_tgt, max_src)
        h = ctypes.c_void_p()
        _check(self.lib, self.lib.nllb_attn_create(device, ctypes.byref(self.dims), ctypes.byref(h)),
               "nllb_attn_create")
        self.handle = h
        self.device = device
        self.n_beams, self.n_heads = n_beams, n_heads

    def close(self) -> None:
        if self.handle:
            self.lib.nllb_attn_destroy(self.handle)
            self.handle = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # -- plumbing --
    def set_stream(self, stream_handle: int) -> None:
        _check(self.lib, self.lib.nllb_attn_set_stream(self.handle, stream_handle), "set_stream")

    def sync(self) -> None:
        _check(self.lib, self.lib.nllb_attn_sync(self.handle), "nllb_attn_sync")

    def reset(self) -> None:
        _check(self.lib, self.lib.nllb_attn_reset(self.handle), "nllb_attn_reset")

    # -- prefill --
    @staticmethod
    def prefill_args(q, k, v, out, batch, n_heads, seq_len, strides, valid_len=None,
                     mask=None, mask_strides=(0, 0), scale=0.125) -> PrefillArgs:
        sb, sh, sr = strides
        return PrefillArgs(ptr(q), ptr(k), ptr(v), ptr(out), batch, n_heads, seq_len, 64,
                           sb, sh, sr, ptr(valid_len), ptr(mask), mask_strides[0],
                           mask_strides[1], scale)

    def prefill(self, args: PrefillArgs) -> None:
        _check(self.lib, self.lib.nllb_attn_prefill(self.handle, ctypes.byref(args)), "prefill")

    def prefill_host(self, args: PrefillArgs) -> None:
        _check(self.lib, self.lib.nllb_attn_prefill_host(self.handle, ctypes.byref(args)),
               "prefill_host")

    # -- decoder self-attention --
    def decode_self(self, layer, step, n_sent, q, k_new, v_new, out) -> None:
        _check(self.lib, self.lib.nllb_attn_decode_self(
            self.handle, layer, step, n_sent, ptr(q), ptr(k_new), ptr(v_new), ptr(out)),
            "decode_self")

    def decode_self_host(self, layer, step, n_sent, q, k_new, v_new, out) -> None:
        _check(self.lib, self.lib.nllb_attn_decode_self_host(
            self.handle, layer, step, n_sent, ptr(q), ptr(k_new), ptr(v_new), ptr(out)),
            "decode_self_host")

    def reorder(self, n_sent, parent) -> None:
        """nllb_attn_reorder: `parent` (a device tensor) must stay unchanged
        until the next decode_self, reorder, sync or reset on this context."""
        _check(self.lib, self.lib.nllb_attn_reorder(self.handle, n_sent, ptr(parent)), "reorder")

    def test_expire_next_wait(self) -> None:
        """nllb_attn_test_expire_next_wait: the next self-attention launch's
        bounded wait runs out (a chunk that is never requested)."""
        _check(self.lib, self.lib.nllb_attn_test_expire_next_wait(self.handle), "test_expire_next_wait")

    def test_expire_next_cross_wait(self) -> None:
        """nllb_attn_test_expire_next_cross_wait: the next cross-attention
        launch's bounded wait runs out (a chunk that is never requested)."""
        _check(self.lib, self.lib.nllb_attn_test_expire_next_cross_wait(self.handle), "test_expire_next_cross_wait")

    def reorder_host(self, n_sent, parent) -> None:
        _check(self.lib, self.lib.nllb_attn_reorder_host(self.handle, n_sent, ptr(parent)),
               "reorder_host")

    # -- cross-attention --
    def set_memory(self, layer, sentence, n_src, k, v, stride_head, stride_row) -> None:
        _check(self.lib, self.lib.nllb_attn_set_memory(
            self.handle, layer, sentence, n_src, ptr(k), ptr(v), stride_head, stride_row),
            "set_memory")

    def set_memory_host(self, layer, sentence, n_src, k, v, stride_head, stride_row) -> None:
        _check(self.lib, self.lib.nllb_attn_set_memory_host(
            self.handle, layer, sentence, n_src, ptr(k), ptr(v), stride_head, stride_row),
            "set_memory_host")

    def cross(self, layer, n_sent, q, out) -> None:
        _check(self.lib, self.lib.nllb_attn_cross(self.handle, layer, n_sent, ptr(q), ptr(out)),
               "cross")

    def cross_host(self, layer, n_sent, q, out) -> None:
        _check(self.lib, self.lib.nllb_attn_cross_host(self.handle, layer, n_sent, ptr(q),
                                                       ptr(out)), "cross_host")


    # -- many query rows against keys of another length --
    @staticmethod
    def paged_args(q, k_pages, v_pages, page_table, kv_len, out, k_new=None, v_new=None, q_start=None, q_len=None,
                   max_q=None, max_kv=None, scale=None) -> PagedArgs:
        """Arguments of :meth:`paged` from torch CUDA tensors, which the caller
        keeps alive: q, out [rows][heads][dim], k_new, v_new
        [rows][kv_heads][dim], pages [n_pages][page_size][kv_heads][dim] (any
        strides, the last axis contiguous), page_table [n_seq][entries] int32.
        max_q defaults to q's rows / n_seq without q_len and to q's rows with
        it, max_kv to what the table holds, scale to dim ** -0.5."""
        n_seq, (rows, heads, dim) = kv_len.numel(), q.shape
        n_pages, page, kv_heads = k_pages.shape[:3]
        if out.shape != q.shape or v_pages.shape != k_pages.shape:
            raise ValueError("out must have q's shape, v_pages k_pages's")
        if (k_new is None) != (v_new is None):
            raise ValueError("k_new and v_new go together")
        if page_table.dim() != 2 or str(page_table.dtype) != "torch.int32" or page_table.shape[0] != n_seq \
                or (page_table.numel() and page_table.stride(1) != 1) or page_table.device != q.device:
            raise ValueError("page_table must be an int32 tensor [n_seq][entries] on q's device")
        # (a one-row table's stride may be anything: its entries bound it)
        table_ld = page_table.stride(0) if n_seq > 1 else page_table.shape[1]
        if max_q is None:
            max_q = rows if q_len is not None else rows // max(n_seq, 1)
        if max_kv is None:
            max_kv = page_table.shape[1] * page
        if max_kv > page_table.shape[1] * page:
            raise ValueError("page_table has too few entries for max_kv")
        a = PagedArgs(q=_rows(q, "q", q, 3), out=_rows(out, "out", q, 3), k_pages=_rows(k_pages, "k_pages", q, 4),
                      v_pages=_rows(v_pages, "v_pages", q, 4), q_start=_ints(q_start, "q_start", n_seq, q),
                      q_len=_ints(q_len, "q_len", n_seq, q), kv_len=_ints(kv_len, "kv_len", n_seq, q),
                      page_table=page_table.data_ptr(), dtype=_dtype_code(q), head_dim=dim, n_heads=heads,
                      n_kv_heads=kv_heads, n_seq=n_seq, q_rows=rows, max_q=max_q, max_kv=max_kv, n_pages=n_pages,
                      page_size=page, page_table_stride=table_ld, scale=dim ** -0.5 if scale is None else scale,
                      q_stride_row=q.stride(0), q_stride_head=q.stride(1),
                      out_stride_row=out.stride(0), out_stride_head=out.stride(1),
                      k_stride_page=k_pages.stride(0), k_stride_slot=k_pages.stride(1),
                      k_stride_head=k_pages.stride(2), v_stride_page=v_pages.stride(0),
                      v_stride_slot=v_pages.stride(1), v_stride_head=v_pages.stride(2))
        if k_new is not None:
            if k_new.shape != (rows, kv_heads, dim) or v_new.shape != k_new.shape:
                raise ValueError("k_new and v_new must be [q rows][kv_heads][dim]")
            a.k_new, a.v_new = _rows(k_new, "k_new", q, 3), _rows(v_new, "v_new", q, 3)
            a.k_new_stride_row, a.k_new_stride_head = k_new.stride(0), k_new.stride(1)
            a.v_new_stride_row, a.v_new_stride_head = v_new.stride(0), v_new.stride(1)
        a.tensors_on = q.device
        return a

    def _same_device(self, args) -> None:
        """The tensors the arguments were built from lie on the context's GPU
        (a structure filled by hand is the caller's to get right)."""
        on = getattr(args, "tensors_on", None)
        if on is not None and (on.type != "cuda" or on.index != self.device):
            raise ValueError(f"the tensors are on {on}, the context on cuda:{self.device}")

    def paged(self, args: PagedArgs) -> None:
        """nllb_attn_paged: a chunk of new tokens over a paged cache."""
        self._same_device(args)
        _check(self.lib, self.lib.nllb_attn_paged(self.handle, ctypes.byref(args)), "nllb_attn_paged")

    @staticmethod
    def cross_rows_args(q, k, v, out, kv_len, q_start=None, q_len=None, kv_start=None, max_q=None, max_kv=None,
                        key_mask=None, scale=None) -> CrossRowsArgs:
        """Arguments of :meth:`cross_rows` from torch CUDA tensors, which the
        caller keeps alive: q, out [rows][heads][dim], k, v
        [kv_rows][kv_heads][dim] (any strides, the last axis contiguous),
        key_mask [kv_rows] uint8.  max_q and max_kv default to rows / n_seq
        without the lengths' starts and to all rows with them."""
        n_seq, (rows, heads, dim), (kv_rows, kv_heads) = kv_len.numel(), q.shape, k.shape[:2]
        if out.shape != q.shape or v.shape != k.shape:
            raise ValueError("out must have q's shape, v k's")
        if max_q is None:
            max_q = rows if q_len is not None else rows // max(n_seq, 1)
        if max_kv is None:
            max_kv = kv_rows if kv_start is not None else kv_rows // max(n_seq, 1)
        a = CrossRowsArgs(
            q=_rows(q, "q", q, 3), k=_rows(k, "k", q, 3), v=_rows(v, "v", q, 3), out=_rows(out, "out", q, 3),
            q_start=_ints(q_start, "q_start", n_seq, q), q_len=_ints(q_len, "q_len", n_seq, q),
            kv_start=_ints(kv_start, "kv_start", n_seq, q), kv_len=_ints(kv_len, "kv_len", n_seq, q),
            key_mask=_ints(key_mask, "key_mask", kv_rows, q, "torch.uint8"), dtype=_dtype_code(q), head_dim=dim,
            n_heads=heads, n_kv_heads=kv_heads, n_seq=n_seq, q_rows=rows, kv_rows=kv_rows, max_q=max_q,
            max_kv=max_kv, scale=dim ** -0.5 if scale is None else scale,
            q_stride_row=q.stride(0), q_stride_head=q.stride(1), k_stride_row=k.stride(0), k_stride_head=k.stride(1),
            v_stride_row=v.stride(0), v_stride_head=v.stride(1), out_stride_row=out.stride(0),
            out_stride_head=out.stride(1))
        a.tensors_on = q.device
        return a

    def test_expire_next_rows_wait(self) -> None:
        """nllb_attn_test_expire_next_rows_wait: a bounded wait of the next
        call of many rows runs out."""
        _check(self.lib, self.lib.nllb_attn_test_expire_next_rows_wait(self.handle), "test_expire_next_rows_wait")

    def cross_rows(self, args: CrossRowsArgs) -> None:
        """nllb_attn_cross_rows: target rows over encoder states of another length."""
        self._same_device(args)
        _check(self.lib, self.lib.nllb_attn_cross_rows(self.handle, ctypes.byref(args)), "nllb_attn_cross_rows")


def attention_head_flash(Q, K, V, mask, out, seq_len: int, head_dim: int = 64) -> int:
    """The drop-in for attention_head_flash (tensor.c:286); returns its status."""
    lib = load()
    lib.nllb_attention_head_flash(ptr(Q), ptr(K), ptr(V), ptr(mask), ptr(out), seq_len, head_dim)
    return lib.nllb_attn_last_status()


def attention_head(Q, K, V, mask, out, scores_buf, seq_len: int, head_dim: int = 64) -> int:
    """The drop-in for attention_head (tensor.c:255); returns its status."""
    lib = load()
    lib.nllb_attention_head(ptr(Q), ptr(K), ptr(V), ptr(mask), ptr(out), ptr(scores_buf),
                            seq_len, head_dim)
    return lib.nllb_attn_last_status()


class Model:
    """A synthetic-or-real NLLB INT8 model on one GPU (include/nllb_translate.h)."""

    def __init__(self, path: str, device: int = 0, max_sentences: int = 1, max_src: int = 256,
                 max_gen: int = 36, lib: Optional[ctypes.CDLL] = None):
        self.lib = lib or load()
        h = ctypes.c_void_p()
        _check(self.lib, self.lib.nllb_model_load(path.encode(), device, max_sentences, max_src,
                                                  max_gen, ctypes.byref(h)), "nllb_model_load")
        self.handle, self.max_gen = h, max_gen

    def close(self) -> None:
        if self.handle:
            self.lib.nllb_model_free(self.handle)
            self.handle = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def translate(self, sources, tgt_lang: int, max_gen: Optional[int] = None,
                  repetition_penalty: float = 1.2, no_repeat_ngram: int = 2):
        """sources: list of token-id lists ([src_lang] ... [2]).  Returns
        (list of output token lists, normalised scores, TranslateStats)."""
        import numpy as np
        flat = np.ascontiguousarray(np.concatenate([np.asarray(x, np.int32) for x in sources]))
        offs = np.zeros(len(sources) + 1, np.int32)
        offs[1:] = np.cumsum([len(x) for x in sources])
        G = max_gen or self.max_gen
        out = np.full((len(sources), self.max_gen), -1, np.int32)
        lens = np.zeros(len(sources), np.int32)
        scores = np.zeros(len(sources), np.float32)
        opts = TranslateOpts(G, repetition_penalty, no_repeat_ngram)
        st = TranslateStats()
        _check(self.lib, self.lib.nllb_translate(self.handle, len(sources), ptr(flat), ptr(offs), tgt_lang,
                                                 ctypes.byref(opts), ptr(out), ptr(lens), ptr(scores),
                                                 ctypes.byref(st)), "nllb_translate")
        toks = [out[i, :lens[i]].tolist() for i in range(len(sources))]
        return toks, scores, st

    def profile(self, enable: bool = True) -> None:
        """nllb_translate_profile: time the following translate calls' kernel
        launches by class (clears the totals)."""
        _check(self.lib, self.lib.nllb_translate_profile(self.handle, 1 if enable else 0), "nllb_translate_profile")

    def profile_read(self):
        """Per-class totals: {name: {launches, ms, flops, bytes}}."""
        buf = (KernelProfile * PROF_CLASSES)()
        n = self.lib.nllb_translate_profile_read(self.handle, buf, PROF_CLASSES)
        return {buf[i].name.decode(): {"launches": int(buf[i].launches), "ms": float(buf[i].ms),
                                       "flops": float(buf[i].flops), "bytes": float(buf[i].bytes)}
                for i in range(n)}

    def margins(self, sentence: int, max_steps: int = 1024):
        import numpy as np
        buf = np.zeros(max_steps, np.float32)
        n = self.lib.nllb_translate_margins(self.handle, sentence, ptr(buf), max_steps)
        return buf[:n]


LINEAR_RELU = 1


def linear_int8(x, w, weight_scale, bias=None, out=None, residual=None, relu=False, stream=None):
    """nllb_linear_int8 on torch CUDA tensors: x [M][K] fp32, w [N][K] int8."""
    lib = load()
    M, K = x.shape
    N = w.shape[0]
    if out is None:
        import torch
        out = torch.empty((M, N), dtype=torch.float32, device=x.device)
    _check(lib, lib.nllb_linear_int8(ptr(x), M, K, ptr(w), ptr(weight_scale), ptr(bias), N, ptr(out),
                                     ptr(residual), LINEAR_RELU if relu else 0, stream), "nllb_linear_int8")
    return out


def linear_int8_noalloc(x, w, weight_scale, out, bias=None, residual=None, relu=False, stream=None):
    """nllb_linear_int8_noalloc on torch CUDA tensors; `out` must be given
    (the call allocates nothing, the caller owns every buffer)."""
    lib = load()
    M, K = x.shape
    N = w.shape[0]
    _check(lib, lib.nllb_linear_int8_noalloc(ptr(x), M, K, ptr(w), ptr(weight_scale), ptr(bias), N, ptr(out),
                                             ptr(residual), LINEAR_RELU if relu else 0, stream),
           "nllb_linear_int8_noalloc")
    return out


def linear_int8_status() -> int:
    """nllb_linear_int8_status: synchronises the device, reads and clears the
    error word of nllb_linear_int8 (returns the status, does not raise)."""
    return load().nllb_linear_int8_status()


def linear_int8_noalloc_status(stream=None) -> int:
    """nllb_linear_int8_noalloc_status: waits for `stream`, reads and clears
    the no-alloc entry point's error word (returns the status, does not raise)."""
    return load().nllb_linear_int8_noalloc_status(stream)


def apply_penalties(logits, tokens, n_tokens, penalty=1.2, no_repeat_ngram=2, stream=None):
    """nllb_apply_penalties on torch CUDA tensors, in place: logits [rows][ld]
    fp32, tokens [rows][tokens_ld] int32, n_tokens [rows] int32."""
    lib = load()
    rows = logits.shape[0]
    _check(lib, lib.nllb_apply_penalties(ptr(logits), logits.stride(0), rows, ptr(tokens), tokens.stride(0),
                                         ptr(n_tokens), penalty, no_repeat_ngram, stream), "nllb_apply_penalties")
    return logits


def logsoftmax_topk(logits, k=8, vocab=None, stream=None):
    """nllb_logsoftmax_topk on a torch CUDA tensor logits [rows][ld] fp32:
    returns (tokens [rows][k] int32, log-probabilities [rows][k] fp32)."""
    import torch
    lib = load()
    rows = logits.shape[0]
    V = logits.shape[1] if vocab is None else vocab
    tok = torch.empty((rows, k), dtype=torch.int32, device=logits.device)
    lp = torch.empty((rows, k), dtype=torch.float32, device=logits.device)
    ws = torch.empty(max(1, lib.nllb_logsoftmax_topk_ws_bytes(V, max(rows, 1), k)), dtype=torch.uint8,
                     device=logits.device)
    _check(lib, lib.nllb_logsoftmax_topk(ptr(logits), logits.stride(0), V, rows, k, ptr(tok), ptr(lp), ptr(ws),
                                         stream), "nllb_logsoftmax_topk")
    return tok, lp


def current_stream(device: int = 0) -> int:
    """Handle of torch's current stream of a GPU, as Context.set_stream and the
    stream arguments take it: the legacy default stream, which torch calls 0,
    is CUDA's handle 1."""
    import torch
    return torch._C._cuda_getCurrentRawStream(device) or 1


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, out_tok=None, out_logp=None,
           stream=None):
    """nllb_sample on torch CUDA tensors: logits [rows][vocab] (rows may be
    strided), u [rows] fp32; temperature, top_p, min_p [rows] fp32 and top_k
    [rows] int32 or None.  Runs on torch's current stream of the logits'
    device unless `stream` names another.  Returns (tokens [rows] int32,
    log-probabilities [rows] fp32)."""
    lib = load()
    rows, vocab = logits.shape
    if vocab > 1 and logits.stride(1) != 1:
        raise ValueError("the rows of logits must be contiguous")
    import torch
    if not logits.is_cuda:
        raise ValueError("logits must be on a GPU")
    if stream is None:
        stream = current_stream(logits.device.index)
    if out_tok is None or out_logp is None:
        out_tok = torch.empty(rows, dtype=torch.int32, device=logits.device) if out_tok is None else out_tok
        out_logp = torch.empty(rows, dtype=torch.float32, device=logits.device) if out_logp is None else out_logp
    f = "torch.float32"
    a = SampleArgs(logits.data_ptr(), logits.stride(0) if rows > 1 else vocab, _dtype_code(logits), vocab, rows,
                   _ints(temperature, "temperature", rows, logits, f), _ints(top_k, "top_k", rows, logits),
                   _ints(top_p, "top_p", rows, logits, f), _ints(min_p, "min_p", rows, logits, f),
                   _ints(u, "u", rows, logits, f), _ints(out_tok, "out_tok", rows, logits),
                   _ints(out_logp, "out_logp", rows, logits, f))
    if logits.device.index != torch.cuda.current_device():
        with torch.cuda.device(logits.device):
            _check(lib, lib.nllb_sample(ctypes.byref(a), stream), "nllb_sample")
    else:
        _check(lib, lib.nllb_sample(ctypes.byref(a), stream), "nllb_sample")
    return out_tok, out_logp


def sample_test_expire_next_wait() -> None:
    """nllb_sample_test_expire_next_wait: a bounded wait of every row of this
    thread's next sample runs out (tokens SAMPLE_TIMEOUT)."""
    lib = load()
    _check(lib, lib.nllb_sample_test_expire_next_wait(), "sample_test_expire_next_wait")


class PreparedLinear:
    """nllb_linear_prepare / nllb_linear_run: one LinearInt8 resident on the
    GPU.  Keeps references to the weight tensors, which the layer reads."""

    def __init__(self, w, weight_scale, bias=None, stream=None):
        self._lib = load()
        self._keep = (w, weight_scale, bias)
        self.N, self.K = w.shape
        h = _c_void_p()
        _check(self._lib, self._lib.nllb_linear_prepare(ptr(w), ptr(weight_scale), ptr(bias), self.N, self.K,
                                                         stream, ctypes.byref(h)), "nllb_linear_prepare")
        self._h = h

    def __call__(self, x, out=None, residual=None, relu=False, stream=None):
        M = x.shape[0]
        if out is None:
            import torch
            out = torch.empty((M, self.N), dtype=torch.float32, device=x.device)
        _check(self._lib, self._lib.nllb_linear_run(self._h, ptr(x), M, ptr(out), ptr(residual),
                                                     LINEAR_RELU if relu else 0, stream), "nllb_linear_run")
        return out

    def status(self) -> int:
        return self._lib.nllb_linear_status(self._h)

    def test_expire_next_wait(self) -> None:
        """The next run on the split-K kernel times out (tests of the bounded waits)."""
        _check(self._lib, self._lib.nllb_linear_test_expire_next_wait(self._h), "nllb_linear_test_expire_next_wait")

    def close(self) -> None:
        if getattr(self, "_h", None):
            self._lib.nllb_linear_free(self._h)
            self._h = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def exported_symbols(header_path: str) -> Sequence[str]:
    """Function names declared in the C header (for the export check)."""
    import re
    text = open(header_path).read()
    return sorted(set(re.findall(r"NLLB_ATTN_API\s+[\w\s\*]*?\b(nllb_\w+)\s*\(", text)))
