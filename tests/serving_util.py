"""Shared helpers of the serving operators' tests: device arrays of the three
types, and the operators' definitions in 64 bits, one request, token or row at
a time.

Tolerances.  u = 2^-24, 2^-11, 2^-8 is the rounding of one value of f32, f16,
bf16.  Attention: a score is a sum of D exact products (16-bit types) or of D
fused multiply-adds in f32, so it is off by at most (D + 8) 2^-24 scale
sum |q k|, and its exp by that much relative, as is the sum of exps; 64 2^-24
covers exp2, the rescalings and the sums over a few hundred terms per lane; exp(s -
max) as the sum of two values of the type is off by u^2 of itself (and in f16 by half
of its smallest step).  All of these weigh values of at most max |v|.  Norms: a mean over a row is a tree of at most 64 serial additions
per thread and 20 more, 84 2^-24 relative to the sum of magnitudes, taken twice
in a layer norm; 2^-24 times 256 covers it with the square root and the products.
"""
import ctypes
import math

import numpy as np
import torch

F32, F16, BF16 = 0, 1, 2
TORCH = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}
ROUND = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
WEIGHT_ROUND = {F32: 0.0, F16: 2.0 ** -22 + 2.0 ** -25, BF16: 2.0 ** -16}


class Device:
    """Buffers of one test, freed together."""

    def __init__(self, ctx):
        self.ctx, self.bufs = ctx, []

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        for b in self.bufs:
            b.free()

    def up(self, t):
        """Upload a CPU tensor; the handle of its buffer."""
        if t is None:
            return None
        a = t.contiguous()
        a = a.view(torch.int16).numpy() if a.element_size() == 2 else a.numpy()
        b = self.ctx.upload(a) if a.nbytes else self.ctx.alloc(0)
        self.bufs.append(b)
        return b.handle

    def new(self, *shape, dtype=torch.int32, fill=None):
        """An output array: handle, and a function that downloads it."""
        t = torch.full(shape, fill if fill is not None else (-7 if not dtype.is_floating_point else float("nan")), dtype=dtype)
        return self.out(t)

    def out(self, t):
        h = self.up(t)
        buf = self.bufs[-1]

        def get():
            if t.numel() == 0:
                return t.clone()
            np_t = np.int16 if t.element_size() == 2 else (np.int32 if t.dtype == torch.int32 else np.float32)
            return torch.from_numpy(buf.download(np_t, tuple(t.shape))).view(t.dtype)
        return h, get


def randn(gen, dtype, *shape):
    return torch.randn(*shape, generator=gen).to(TORCH[dtype])


def wrap_all(ctx, tensors):
    return [ctx.wrap(t.data_ptr(), t.numel() * t.element_size()) for t in tensors]


def attention_reference(q, kc, vc, table, lens, H, window=0, scale=1.0, softcap=0.0):
    """(out [R, H, D], lse [R, H], tolerance before the output's rounding [R, H]) in 64 bits."""
    R, cols = table.shape
    pages, Hk, page, D = kc.shape
    G = H // Hk
    out = torch.zeros(R, H, D, dtype=torch.float64)
    lse = torch.full((R, H), -math.inf, dtype=torch.float64)
    tol = torch.zeros(R, H, dtype=torch.float64)
    for r in range(R):
        n = min(max(int(lens[r]), 0), cols * page) if pages else 0
        pos = [t for t in range(max(0, n - window) if window else 0, n) if 0 <= int(table[r, t // page]) < pages]
        if not pos:
            continue
        pg = torch.tensor([int(table[r, t // page]) for t in pos])
        at = torch.tensor([t % page for t in pos])
        for h in range(H):
            k, v = kc[pg, h // G, at].double(), vc[pg, h // G, at].double()
            qq = q[r, h * D:(h + 1) * D].double()
            s = scale * (k @ qq)
            if softcap > 0:
                s = softcap * torch.tanh(s / softcap)
            m = s.max()
            p = torch.exp(s - m)
            out[r, h] = p @ v / p.sum()
            lse[r, h] = m + torch.log(p.sum())
            ds = (D + 8) * 2.0 ** -24 * abs(scale) * float((k.abs() @ qq.abs()).max()) + 4 * 2.0 ** -24 * float(s.abs().max())
            if softcap > 0:
                ds += 8 * 2.0 ** -24 * softcap
            tol[r, h] = 2 * ds + 64 * 2.0 ** -24
    return out, lse, tol


def check_attention(got, lse, ref, v_max, dtype, what):
    out, want_lse, tol = ref
    R, H, D = out.shape
    got = got.double().view(R, H, D)
    assert torch.isfinite(got).all(), f"{what}: non-finite output"
    bound = (tol + WEIGHT_ROUND[dtype])[..., None] * v_max + ROUND[dtype] * out.abs()
    if dtype == F16:
        bound = bound + 2.0 ** -25
    bad = (got - out).abs() > bound
    assert not bad.any(), f"{what}: {int(bad.sum())} values off, worst {float(((got - out).abs() / bound).max()):.3g} of the bound"
    if lse is not None:
        empty = torch.isinf(want_lse)
        assert torch.equal(torch.isneginf(lse), empty), what
        d = (lse.double() - want_lse)[~empty].abs()
        assert (d <= (tol[~empty] + 4 * 2.0 ** -24 * want_lse[~empty].abs())).all(), f"{what}: lse off by {float(d.max()):.3g}"


def plan_reference(seq, new, free, head, table, page, pool, max_tokens):
    table = [list(map(int, row)) for row in table]
    cols = len(table[0]) if table else 0
    cap, head, F = cols * page, max(0, int(head)), len(free)
    slots, pos, req, starts, lens = [], [], [], [0], []
    taken = short = past = 0
    at = head
    for r in range(len(seq)):
        s, n = min(max(int(seq[r]), 0), cap), max(int(new[r]), 0)
        have, want = -(-s // page), min(-(-(s + n) // page), cols)
        held = have
        for i in range(have, want):
            there = at < F
            table[r][i] = int(free[at]) if there else -1
            held += there
            taken += there
            short += not there
            at += 1
        kv = min(s + n, held * page)
        lens.append(kv)
        past += s + n - kv
        for j in range(n):
            t = s + j
            p = table[r][t // page] if t < kv else -1
            slots.append(p * page + t % page if 0 <= p < pool else -1)
            pos.append(t)
            req.append(r)
        starts.append(len(slots))
    total = len(slots)
    fill = lambda v, x: (v + [x] * max_tokens)[:max_tokens]  # noqa: E731
    as_t = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return {"block_table": as_t(table).reshape(len(seq), cols), "slots": as_t(fill(slots, -1)), "positions": as_t(fill(pos, 0)),
            "token_request": as_t(fill(req, -1)), "token_starts": as_t(starts), "kv_lens": as_t(lens),
            "counts": as_t([head + taken, total, short, past])}


def norm_reference(x, r, post, pre, gate, rscale, eps, pw, pb, nw, nb):
    """(h, out) in 64 bits, and the sizes that their tolerances go by; post / pre: 0 none, 1 rms, 2 layer."""
    d = lambda t: None if t is None else t.double()  # noqa: E731
    x, r, gate, pw, pb, nw, nb = map(d, (x, r, gate, pw, pb, nw, nb))

    def norm(v, kind, w, b, off):
        if kind == 0:
            return v, off
        c = v - v.mean(-1, keepdim=True) if kind == 2 else v
        rs = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
        f = w if w is not None else torch.ones(v.shape[-1], dtype=torch.float64)
        y = c * rs * f
        # v off by `off` moves y by that times its factor, and the row's scale by as much
        far = (off + 256 * 2.0 ** -24 * v.abs().amax(-1, keepdim=True)) * rs * f.abs() * 2 + y.abs() * (
            256 * 2.0 ** -24 + 2 * off.amax(-1, keepdim=True) * rs)
        return (y + b if b is not None else y), far + (2.0 ** -23 * (y + b).abs() if b is not None else 0)

    h, off = 0.0, torch.zeros(1, 1, dtype=torch.float64)
    if x is not None:
        a, off = norm(x, post, pw, pb, off.expand(x.shape))
        if gate is not None:
            a, off = a * gate, off * gate.abs()
        h = a
    if r is not None:
        h = h + rscale * r
        off = (off + 2.0 ** -23 * ((rscale * r).abs() + h.abs())).expand(h.shape)
    out, out_off = norm(h, pre, nw, nb, off)
    return h, out, off, out_off


def c_address(buffer):
    """Device address of a plugin buffer (its record's first word)."""
    return ctypes.c_void_p.from_address(buffer.handle).value
