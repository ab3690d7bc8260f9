"""buffer_wrap: buffers over memory that another library allocated."""
import numpy as np
import pytest
import torch

from mlx_amd import abi, runtime

pytestmark = pytest.mark.gpu


def test_wrap_reads_writes_and_leaves_the_memory(ctx):
    t = torch.arange(1000, dtype=torch.float32, device="cuda")
    torch.cuda.synchronize()
    b = ctx.wrap(t.data_ptr() + 40, 400)
    assert np.array_equal(b.download(np.float32, (100,)), np.arange(10, 110, dtype=np.float32))
    b.upload(np.full(5, -1, np.float32))
    b.free()
    assert t[10:15].tolist() == [-1.0] * 5 and t[15].item() == 15.0
    t += 1  # still torch's
    assert t[20].item() == 21.0


def test_wrapped_buffers_in_an_operator(ctx):
    x = torch.randn(4, 64, device="cuda")
    out = torch.empty_like(x)
    torch.cuda.synchronize()
    bx, bo = ctx.wrap(x.data_ptr(), x.numel() * 4), ctx.wrap(out.data_ptr(), x.numel() * 4)
    ctx.block_norm(abi.BlockNormArgs(rows=4, dim=64, pre_norm=abi.NORM_RMS, residual_scale=1.0, residual=bx.handle, out=bo.handle))
    ctx.sync()
    want = x / x.square().mean(-1, keepdim=True).sqrt()
    assert (out - want).abs().max() < 1e-5
    bx.free()
    bo.free()


def test_wrap_refuses_what_is_not_the_device_s(ctx):
    host = np.zeros(16, np.float32)
    for address, n in [(host.ctypes.data, 64), (0, 16)]:
        with pytest.raises(runtime.LuxError):
            ctx.wrap(address, n)
    ctx.wrap(0, 0).free()
    t = torch.zeros(4, device="cuda")
    b = ctx.wrap(t.data_ptr(), 16)
    # a buffer too small for the sizes is refused, wrapped or not
    a = abi.BlockNormArgs(rows=1, dim=5, pre_norm=abi.NORM_RMS, residual=b.handle, out=b.handle)
    assert ctx.s.op_block_norm(ctx.handle, a) == abi.ERR_INVALID_ARGUMENT
    b.free()
