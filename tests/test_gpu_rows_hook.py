"""The hook that lets a wait of attention over many rows run out is for the context's next call and no later one."""
import ctypes

import pytest
import torch

import nllb_attn as na
from test_gpu_rows import ctx, ints  # noqa: F401 (ctx is a fixture)
from test_gpu_window import Window

pytestmark = pytest.mark.gpu


def case(lens=((140, 500),)):
    return Window(list(lens), 2, 2, 64, 16, torch.bfloat16, 100, 2)


def refused_window(ctx):  # noqa: F811
    with pytest.raises(na.NllbAttnError):
        x = case()
        x.window = 0
        x.run(ctx)


def refused_arguments(ctx):  # noqa: F811
    for name, args in (("window", na.WindowArgs(window=1)), ("paged", na.PagedArgs()), ("cross_rows", na.CrossRowsArgs())):
        ctx.test_expire_next_rows_wait()
        assert getattr(ctx.lib, "nllb_attn_" + name)(ctx.handle, ctypes.byref(args)) == na.EINVAL


def no_arguments(ctx):  # noqa: F811
    assert ctx.lib.nllb_attn_window(ctx.handle, None) == na.EINVAL


def no_rows(ctx):  # noqa: F811
    x = case()
    empty = torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    ctx.window(ctx.window_args(empty, x.k_pages, x.v_pages, x.table[:0], ints([]), empty, 100, 2))


def few_rows(ctx):  # noqa: F811
    x = case([(1, 500)])
    x.run(ctx)
    ctx.sync()
    x.verify("few rows")


@pytest.mark.parametrize("call", [refused_window, refused_arguments, no_arguments, no_rows, few_rows])
def test_used_up(ctx, call):  # noqa: F811
    ctx.test_expire_next_rows_wait()
    call(ctx)
    x = case()
    x.run(ctx)
    ctx.sync()
    x.verify("after " + call.__name__)
