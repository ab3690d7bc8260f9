"""The norms around a block with gate and residual, against 64 bits: types, row
lengths from 1 to 65536, both kinds of norm, every gate, strides, in place, and
rows of large means, zeros and infinities."""
import pytest
import torch

from mlx_amd import abi
from serving_util import BF16, F16, F32, ROUND, TORCH, Device, norm_reference, randn

pytestmark = pytest.mark.gpu
NONE, CHANNEL, ROW, FULL = range(4)


def strided(gen_rows, stride, fill=3.0):
    """Storage of rows at that stride, and the rows' view of it."""
    T, D = gen_rows.shape
    store = torch.full((max(T, 1) * stride,), fill, dtype=gen_rows.dtype)
    view = torch.as_strided(store, (T, D), (stride, 1))
    view.copy_(gen_rows)
    return store, view


def run(ctx, x, r, post, pre, gate_mode, gate, rscale, eps, pw, pb, nw, nb, xd, rd, wd, pad=0, in_place=False, want=(True, True)):
    T, D = (x if x is not None else r).shape
    s = D + pad
    with Device(ctx) as dev:
        up = lambda t: None if t is None else dev.up(strided(t, s)[0])  # noqa: E731
        xh = rh = None
        if x is not None:
            xh, x_get = dev.out(strided(x, s)[0])
        if r is not None:
            rh, r_get = dev.out(strided(r, s)[0])
        if in_place:
            hh, h_get, oh, o_get = rh, r_get, xh, x_get
        else:
            hh, h_get = dev.out(strided(torch.zeros(T, D, dtype=TORCH[rd]), s)[0])
            oh, o_get = dev.out(strided(torch.zeros(T, D, dtype=TORCH[xd]), s)[0])
        g = None if gate is None else up(gate) if gate_mode == FULL else dev.up(gate)
        ctx.block_norm(abi.BlockNormArgs(
            rows=T, dim=D, post_norm=post, pre_norm=pre, gate_mode=gate_mode, x_dtype=xd, residual_dtype=rd, weight_dtype=wd,
            residual_scale=rscale, eps=eps, x_row_stride=s, residual_row_stride=s, gate_row_stride=s if gate_mode == FULL else 0,
            residual_out_row_stride=s, out_row_stride=s, x=xh, residual=rh, post_weight=dev.up(pw), post_bias=dev.up(pb), gate=g,
            pre_weight=dev.up(nw), pre_bias=dev.up(nb), residual_out=hh if want[0] else None, out=oh if want[1] else None))
        got = []
        for get in (h_get, o_get):
            store = get()
            view = torch.as_strided(store, (T, D), (s, 1)).clone()
            torch.as_strided(store, (T, D), (s, 1)).fill_(3.0)
            assert (store == 3.0).all()  # what lies between the rows stays
            got.append(view)
        return got


def compare(got, ref, off, dt, what):
    bound = off + ROUND[dt] * ref.abs() * 1.01 + (2.0 ** -25 if dt == F16 else 0)
    bad = (got.double() - ref).abs() > bound
    assert not bad.any(), f"{what}: {int(bad.sum())} off, worst {float(((got.double() - ref).abs() / bound).max()):.3g} of the bound"


def check(ctx, T, D, xd, rd, wd=None, post=1, pre=1, gate_mode=NONE, rscale=1.0, bias=False, pad=0, in_place=False, with_x=True,
          with_r=True, weights=True, seed=0, shift=0.0):
    print(f"[case] T={T} D={D} x={xd} r={rd} w={wd} post={post} pre={pre} gate={gate_mode} pad={pad} in_place={in_place}", flush=True)
    gen = torch.Generator().manual_seed(seed + D)
    wd = xd if wd is None else wd
    x = randn(gen, xd, T, D) + shift if with_x else None
    r = randn(gen, rd, T, D) if with_r else None
    w = lambda: randn(gen, wd, D) if weights else None  # noqa: E731
    pw, nw = w(), w()
    pb, nb = (randn(gen, wd, D), randn(gen, wd, D)) if bias else (None, None)
    gate = {NONE: None, CHANNEL: randn(gen, xd, D), ROW: randn(gen, xd, T), FULL: randn(gen, xd, T, D)}[gate_mode]
    h, o = run(ctx, x, r, post, pre, gate_mode, gate, rscale, 1e-5, pw, pb, nw, nb, xd, rd, wd, pad, in_place)
    rh, ro, off_h, off_o = norm_reference(x, r, post, pre, gate[:, None] if gate_mode == ROW else gate, rscale, 1e-5, pw, pb, nw, nb)
    compare(h, rh, off_h, rd, "h")
    compare(o, ro, off_o, xd, "out")


@pytest.mark.parametrize("xd,rd", [(F32, F32), (F16, F16), (BF16, BF16), (F16, F32), (BF16, F32), (F32, F16)])
@pytest.mark.parametrize("D", [1, 2, 7, 8, 9, 64, 100, 511, 512, 513, 1000, 2048, 2049, 4096, 5003, 8192, 8200, 16384, 20001, 32768, 40000,
                               65536])
def test_row_lengths(ctx, xd, rd, D):
    check(ctx, 3, D, xd, rd, gate_mode=CHANNEL, bias=True, seed=1)
    check(ctx, 2, D, xd, rd, post=2, pre=2, gate_mode=FULL, rscale=0.5, seed=2)


@pytest.mark.parametrize("post", [0, 1, 2])
@pytest.mark.parametrize("pre", [0, 1, 2])
@pytest.mark.parametrize("gate", [NONE, CHANNEL, ROW, FULL])
def test_kinds_and_gates(ctx, post, pre, gate):
    for D in (60, 1500):
        check(ctx, 9, D, F16, F16, wd=F32, post=post, pre=pre, gate_mode=gate, rscale=-1.5, bias=True, seed=5)
        check(ctx, 9, D, BF16, F32, wd=BF16, post=post, pre=pre, gate_mode=gate, weights=False, pad=3, seed=6)


@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 63, 1000])
def test_rows(ctx, T):
    check(ctx, T, 256, BF16, BF16, gate_mode=ROW, seed=7)
    check(ctx, T, 3000, F16, F32, post=2, seed=8)


@pytest.mark.parametrize("pad", [0, 1, 8])
@pytest.mark.parametrize("xd,rd", [(F16, F16), (F32, F32), (BF16, F32)])
def test_in_place(ctx, xd, rd, pad):
    for D in (300, 4096, 9001):
        check(ctx, 11, D, xd, rd, gate_mode=FULL, pad=pad, in_place=True, seed=9)


def test_without_x_or_residual(ctx):
    check(ctx, 5, 700, F16, F32, with_x=False, seed=10, rscale=2.0)
    check(ctx, 5, 700, F16, F32, with_r=False, gate_mode=CHANNEL, seed=11)


def test_one_output(ctx):
    gen = torch.Generator().manual_seed(12)
    x, r = randn(gen, F16, 4, 600), randn(gen, F16, 4, 600)
    both = run(ctx, x, r, 1, 1, NONE, None, 1.0, 1e-5, None, None, None, None, F16, F16, F16)
    h, o = run(ctx, x, r, 1, 1, NONE, None, 1.0, 1e-5, None, None, None, None, F16, F16, F16, want=(True, False))
    assert torch.equal(h, both[0]) and (o == 0).all()
    h, o = run(ctx, x, r, 1, 1, NONE, None, 1.0, 1e-5, None, None, None, None, F16, F16, F16, want=(False, True))
    assert torch.equal(o, both[1]) and (h == 0).all()


def test_large_mean_zero_rows_and_infinities(ctx):
    # a layer norm takes the mean out before it squares
    check(ctx, 4, 4096, F32, F32, post=2, pre=2, shift=1000.0, seed=13)
    z = torch.zeros(3, 512)
    h, o = run(ctx, z, z, 1, 2, NONE, None, 1.0, 1e-5, None, None, None, None, F32, F32, F32)
    assert (h == 0).all() and (o == 0).all()
    x = torch.ones(3, 600)
    x[1, 5] = float("inf")
    h, o = run(ctx, x, z[:, :1].expand(3, 600).contiguous(), 0, 1, NONE, None, 1.0, 1e-5, None, None, None, None, F32, F32, F32)
    assert torch.isnan(o[1, 5]) and (o[1, :5] == 0).all()      # inf / inf, and 1 / inf
    assert ((o[[0, 2]] - 1 / (1 + 1e-5) ** 0.5).abs() < 1e-6).all()  # the rows beside it


def test_refusals(ctx):
    I, N = abi.ERR_INVALID_ARGUMENT, abi.ERR_NOT_SUPPORTED
    with Device(ctx) as dev:
        def record(**over):
            r = dict(rows=2, dim=24, post_norm=1, pre_norm=1, x_dtype=F16, residual_dtype=F32, weight_dtype=F16, residual_scale=1.0, eps=1e-5)
            r.update({k: dev.up(torch.zeros(2, 24, dtype=t)) for k, t in [("x", torch.float16), ("residual", torch.float32),
                                                                        ("residual_out", torch.float32), ("out", torch.float16)]})
            r.update(pre_weight=dev.up(torch.zeros(24, dtype=torch.float16)))
            r.update(over)
            return abi.BlockNormArgs(**r)
        call = lambda a: ctx.s.op_block_norm(ctx.handle, a)  # noqa: E731
        assert call(record()) == abi.OK and call(record(rows=0)) == abi.OK
        for over, want in [(dict(rows=-1), I), (dict(rows=3), I), (dict(dim=0), I), (dict(dim=25), I), (dict(dim=65537), N),
                           (dict(post_norm=3), I), (dict(pre_norm=-1), I), (dict(gate_mode=4), I), (dict(gate_mode=1), I),
                           (dict(x_dtype=3), N), (dict(residual_dtype=-1), N), (dict(weight_dtype=8), N), (dict(weight_dtype=F32), I),
                           (dict(x_row_stride=23), I), (dict(x_row_stride=25), I), (dict(out_row_stride=-24), I),
                           (dict(x=None, residual=None), I), (dict(out=None, residual_out=None), I)]:
            assert call(record(**over)) == want, over
        a = record()
        a.out = a.residual
        assert call(a) == I
        a = record()
        a.residual_out, a.residual_out_row_stride = a.residual, 24
        assert call(a) == abi.OK
        b = record(x_row_stride=24, rows=1)
        b.out, b.out_row_stride = b.x, 24
        assert call(b) == abi.OK
        a = record()
        a.struct_size = 1
        assert call(a) == I
