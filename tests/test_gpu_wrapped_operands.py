"""Wrapped memory as operands of the quantized and base ops, whose kernels read
whole vectors: taken where the bytes behind it can be read, refused where not."""
import ctypes
import os

import numpy as np
import pytest

from mlx_amd import abi

pytestmark = pytest.mark.gpu
F16, F32 = abi.FLOAT16, abi.FLOAT32
SIZE = 2 << 20


@pytest.fixture(scope="module")
def block(ctx):
    """An allocation of SIZE bytes, no more: (address, fill(offset, array))."""
    hip = ctypes.CDLL("libamdhip64.so", mode=os.RTLD_NOW | os.RTLD_GLOBAL)
    p = ctypes.c_void_p()
    assert hip.hipMalloc(ctypes.byref(p), ctypes.c_size_t(SIZE)) == 0

    def fill(at, a):
        assert hip.hipMemcpy(ctypes.c_void_p(p.value + at), a.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(a.nbytes), 1) == 0

    yield p.value, fill
    ctx.sync()
    assert hip.hipFree(p) == 0


def test_bytes_behind_a_view(ctx, block):
    """What the checks go by: the buffer record's fourth word, to the allocation's end."""
    for at, n in [(0, 1), (0, SIZE), (1 << 20, 100), (SIZE - 7, 7), (SIZE - 300, 4)]:
        b = ctx.wrap(block[0] + at, n)
        assert ctypes.c_size_t.from_address(b.handle + 24).value == SIZE - at - n, (at, n)
        b.free()


def call(ctx, op, arrays, out_bytes, make, block, wrapped, at):
    """op over uploaded arrays, operand `wrapped` in the block at `at` instead (the output is the last)."""
    address, fill = block
    bufs = []
    for i, a in enumerate(arrays):
        if i == wrapped:
            fill(at, a)
            bufs.append(ctx.wrap(address + at, a.nbytes))
        else:
            bufs.append(ctx.upload(a))
    bufs.append(ctx.wrap(address + at, out_bytes) if wrapped == len(arrays) else ctx.alloc(out_bytes))
    err = make(op, [b.handle for b in bufs])
    ctx.sync()
    got = bufs[-1].download(np.uint8, (out_bytes,))
    for b in bufs:
        b.free()
    return err, got


def sweep(ctx, block, op, arrays, out_bytes, make, needs):
    """needs: per operand, the output last, the bytes that it starts on and those behind it."""
    err, want = call(ctx, op, arrays, out_bytes, make, block, None, 0)
    assert err == abi.OK
    for i in range(len(arrays) + 1):
        n = arrays[i].nbytes if i < len(arrays) else out_bytes
        align, need = needs[i]
        end = (SIZE - n) // align * align
        for at, ok in [(0, True), (5 * align, True), ((SIZE - n - need) // align * align, True), (64 + align // 2, False),
                       (end, SIZE - n - end >= need), (end - align, SIZE - n - end + align >= need)]:
            err, got = call(ctx, op, arrays, out_bytes, make, block, i, at)
            assert err == (abi.OK if ok else abi.ERR_INVALID_ARGUMENT), (i, at, ok)
            if ok:
                assert np.array_equal(got, want), (i, at)


@pytest.mark.parametrize("M,K,N,bits", [(1, 512, 96, 4), (3, 256, 50, 3), (64, 512, 96, 8), (200, 1024, 96, 4)])
def test_quantized_matmul(ctx, oracle, block, M, K, N, bits):
    x, w, s, b, _ = oracle.make_problem(M, K, N, bits, 64, F16, F16, seed=M)
    bias = np.random.default_rng(1).standard_normal(N).astype(np.float32)
    sweep(ctx, block, ctx.q.op_quantized_matmul, [x, w, s, b], M * N * 2,
          lambda f, h: f(ctx.handle, *h, M, K, N, 64, bits, F16, F16, F16), [(16, 256)] * 4 + [(2, 0)])
    sweep(ctx, block, ctx.q.op_quantized_matmul_fused, [x, w, s, b, bias], M * N * 4,
          lambda f, h: f(ctx.handle, *h, M, K, N, 64, bits, F16, F16, F32, F32, 1), [(16, 256)] * 4 + [(4, 0)] * 2)


def test_dequantize_and_quantize(ctx, oracle, block):
    K, N = 512, 96
    _, w, s, b, _ = oracle.make_problem(1, K, N, 6, 32, F16, F32, seed=2)
    sweep(ctx, block, ctx.q.op_dequantize, [w, s, b], N * K * 2, lambda f, h: f(ctx.handle, *h, N, K, 32, 6, F32, F16), [(16, 256)] * 3 + [(16, 0)])
    full = np.random.default_rng(3).standard_normal((N, K)).astype(np.float32)
    spare = [ctx.alloc(N * K), ctx.alloc(N * K)]

    def to(which):
        def make(f, h):  # the codes, or the scales, are the last buffer
            outs = [spare[0].handle, spare[1].handle]
            outs.insert(which, h[1])
            return f(ctx.handle, h[0], *outs, N, K, 32, 4, F32, F32)
        return make

    sweep(ctx, block, ctx.q.op_quantize, [full], N * K // 2, to(0), [(16, 256), (4, 0)])
    sweep(ctx, block, ctx.q.op_quantize, [full], N * K // 32 * 4, to(1), [(16, 256), (4, 0)])
    for sp in spare:
        sp.free()


def test_base_ops(ctx, block):
    rng = np.random.default_rng(4)
    a, b = (rng.standard_normal(1003).astype(np.float32) for _ in range(2))
    for name in ("op_add_f32", "op_sub_f32", "op_mul_f32", "op_div_f32"):
        sweep(ctx, block, getattr(ctx.vt, name), [a, b], a.nbytes, lambda f, h: f(ctx.handle, *h, a.size), [(4, 0)] * 3)
    for M, K, N in [(5, 7, 9), (70, 33, 65)]:
        x, y = (rng.standard_normal(s).astype(np.float32) for s in ((M, K), (K, N)))
        sweep(ctx, block, ctx.vt.op_matmul_f32, [x, y], M * N * 4, lambda f, h: f(ctx.handle, *h, M, K, N), [(4, 12), (4, 12), (4, 0)])  # noqa: B023
    x = rng.standard_normal((33, 65)).astype(np.float32)
    sweep(ctx, block, ctx.vt.op_transpose_f32, [x], x.nbytes, lambda f, h: f(ctx.handle, *h, 33, 65), [(4, 0)] * 2)
