"""Rows and strides whose bytes pass 64 bits: refused before anything is launched."""
import pytest
import torch

from mlx_amd import abi
from serving_util import F16, F32, Device

pytestmark = pytest.mark.gpu
ROWS, FAR = 2 ** 22 + 1, 2 ** 40  # (ROWS - 1) * FAR * 4 is 2^64


def test_append(ctx):
    with Device(ctx) as dev:
        slots = dev.up(torch.full((2 * ROWS,), -1, dtype=torch.int32))
        cache = [dev.up(torch.zeros(5, 2, 4, 8, dtype=torch.float16)) for _ in range(2)]
        for dt, rows in [(F32, ROWS), (F16, 2 * ROWS - 1), (F32, 2 * ROWS)]:
            small = dev.up(torch.zeros(64))
            near = dict(tokens=1, kv_heads=2, head_dim=8, page_size=4, num_pages=5, in_dtype=dt, cache_dtype=F16, k=small, v=small, slots=slots,
                        k_cache=cache[0], v_cache=cache[1])
            call = lambda **over: ctx.s.op_paged_append(ctx.handle, abi.PagedAppendArgs(**{**near, **over}))  # noqa: E731
            assert call(k_row_stride=FAR, v_row_stride=FAR) == abi.OK
            assert call(tokens=rows, k_row_stride=FAR, v_row_stride=FAR) == abi.ERR_INVALID_ARGUMENT
            assert call(tokens=rows, k_row_stride=FAR, v_row_stride=FAR, k_offset=1) == abi.ERR_INVALID_ARGUMENT
            assert call(k_offset=FAR) == abi.ERR_INVALID_ARGUMENT and call(k_offset=FAR + 1) == abi.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("which", ["x_row_stride", "residual_row_stride", "gate_row_stride", "residual_out_row_stride", "out_row_stride"])
def test_norm(ctx, which):
    with Device(ctx) as dev:
        small = [dev.up(torch.zeros(64)) for _ in range(5)]
        args = dict(rows=1, dim=16, post_norm=1, pre_norm=1, gate_mode=abi.GATE_FULL, x_dtype=F32, residual_dtype=F32, weight_dtype=F32,
                    residual_scale=1.0, eps=1e-5, x=small[0], residual=small[1], gate=small[2], residual_out=small[3], out=small[4])
        call = lambda **over: ctx.s.op_block_norm(ctx.handle, abi.BlockNormArgs(**{**args, **over}))  # noqa: E731
        assert call(**{which: FAR}) == abi.OK
        strides = {k: FAR for k in ("x_row_stride", "residual_row_stride", "gate_row_stride", "residual_out_row_stride", "out_row_stride")}
        assert call(rows=ROWS, **strides) == abi.ERR_INVALID_ARGUMENT
        assert call(rows=2 ** 31 - 1, **strides) == abi.ERR_INVALID_ARGUMENT
        assert call(rows=ROWS, **{which: FAR}) == abi.ERR_INVALID_ARGUMENT


def test_attention(ctx):
    with Device(ctx) as dev:
        ints = [dev.up(torch.zeros(2 * ROWS, dtype=torch.int32)) for _ in range(2)]
        cache = [dev.up(torch.zeros(5, 1, 4, 8)) for _ in range(2)]
        q, out = (dev.up(torch.zeros(64)) for _ in range(2))
        args = dict(requests=1, heads=1, kv_heads=1, head_dim=8, page_size=4, num_pages=5, max_pages=1, dtype=F32, scale=1.0, q=q,
                    k_cache=cache[0], v_cache=cache[1], block_table=ints[0], kv_lens=ints[1], out=out)
        call = lambda **over: ctx.s.op_paged_attention(ctx.handle, abi.PagedAttentionArgs(**{**args, **over}))  # noqa: E731
        assert call(q_row_stride=FAR, out_row_stride=FAR) == abi.OK
        for rows in (ROWS, 2 * ROWS):
            assert call(requests=rows, q_row_stride=FAR, out_row_stride=FAR) == abi.ERR_INVALID_ARGUMENT
            assert call(requests=rows, q_row_stride=FAR, out_row_stride=FAR, q_offset=1, out_offset=1) == abi.ERR_INVALID_ARGUMENT
