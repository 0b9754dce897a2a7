"""Inputs, 64-bit results and error bounds for the tests of the gated feed-forward
block and of the block-scaled FP8 product.

Bounds, element by element, each from the roundings made.  u is half a step of the
16-bit type relative to the value (bf16 2^-8, fp16 2^-11), `tiny` its smallest step.
  sums      an fp32 sum of n products is off by at most n 2^-23 of their magnitudes'
            sum, whatever its order and also if each addition truncates
  silu      z s(z) in fp32 by an exponential of the hardware (|z| 2^-23 and one step),
            a reciprocal (one step) and a few roundings: (8 + 2 |z|) 2^-23 relative, and
            2^-118 where the sigmoid is subnormal and counts as 0 (below |z| = 128); for the
            error of z itself |silu'| <= 1.1, |silu''| <= 0.5
  h, dgu    rounded once to 16 bits
  results   rounded once to 16 bits; the router's weights' gradient is fp32
Errors of the factors go through the products that follow by their magnitudes.
"""
from __future__ import annotations

import torch

from grouped_cases import HALF, TINY

STEP = 2.0 ** -23


def make(T, k, E, H, I, dtype, seed=0, drop=0.0, skew=False, device="cuda"):
    """x, w13, w2, ids, topk weights and dy; dense with E = 0: ids and topk weights are None."""
    g = torch.Generator().manual_seed(1000 * seed + 7 * T + 3 * H + I + E)
    x = torch.randn((T, H), generator=g).to(dtype).to(device)
    dy = torch.randn((T, H), generator=g).to(dtype).to(device)
    lead = (E,) if E else ()
    scale = min(1.0, 2.0 * H ** -0.5)  # projections of a few units: both ends of the activation
    w13 = (torch.randn((*lead, 2 * I, H), generator=g) * scale).to(dtype).to(device)
    w2 = (torch.randn((*lead, H, I), generator=g) * 0.1).to(dtype).to(device)
    if not E:
        return x, w13, w2, None, None, dy
    scores = torch.rand((T, E), generator=g)
    if skew:  # most slots go to one expert, most experts have none
        scores[:, E // 2] += 2.0
        scores[:, : E // 3] -= 2.0
    ids = torch.topk(scores, k, dim=1).indices if T else torch.empty((0, k), dtype=torch.int64)
    if drop:
        ids = torch.where(torch.rand((T, k), generator=g) < drop, torch.tensor(-1), ids)
        ids = torch.where(torch.rand((T, k), generator=g) < drop / 2, torch.tensor(E), ids)
    weight = torch.rand((T, k), generator=g)
    return x, w13, w2, ids.to(torch.int32).to(device), weight.to(device), dy


def exact(x, w13, w2, ids, weight, dy):
    """[(result in 64 bits, bound of its error)] for y, dx, dw13, dw2 and the router's weights' gradient (None: dense)."""
    dense = ids is None
    u, tiny = HALF[x.dtype], TINY[x.dtype]
    T, H = x.shape
    I = w2.shape[-1]  # noqa: E741
    k = 1 if dense else ids.shape[1]
    flat = torch.zeros(T, dtype=torch.int64, device=x.device) if dense else ids.reshape(-1).long()
    wt = torch.ones(T * k, dtype=torch.float64, device=x.device)
    if weight is not None:
        wt = weight.reshape(-1).double()
    w13s, w2s = (w13[None], w2[None]) if dense else (w13, w2)
    z = lambda *s: torch.zeros(s, dtype=torch.float64, device=x.device)  # noqa: E731
    y, ey, dx, edx, dw, edw = z(T, H), z(T, H), z(T, H), z(T, H), z(T * k), z(T * k)
    d13, e13, d2, e2 = z(*w13s.shape), z(*w13s.shape), z(*w2s.shape), z(*w2s.shape)
    for e in range(w13s.shape[0]):
        at = (flat == e).nonzero().view(-1)
        if not at.numel():
            continue
        n, t = at.numel(), at // k
        xe, dye, w = x[t].double(), dy[t].double(), wt[at][:, None]
        wgu, wd = w13s[e].double(), w2s[e].double()
        gu, egu = xe @ wgu.t(), H * STEP * (xe.abs() @ wgu.abs().t())
        g, up, eg, eu = gu[:, :I], gu[:, I:], egu[:, :I], egu[:, I:]
        s = torch.sigmoid(g)
        a = g * s
        ev = (8 + 2 * g.abs()) * STEP
        ea = 1.1 * eg + ev * a.abs() + 2.0 ** -118
        h = w * a * up
        eh = w.abs() * (up.abs() * ea + (a.abs() + ea) * eu) + 4 * STEP * h.abs()
        eh = eh + u * (h.abs() + eh) + tiny
        y.index_add_(0, t, h @ wd.t())
        ey.index_add_(0, t, eh @ wd.abs().t() + (I + k) * STEP * ((h.abs() + eh) @ wd.abs().t()))
        D, eD = dye @ wd, H * STEP * (dye.abs() @ wd.abs())
        f = s + a * (1 - s)
        ef = 0.5 * eg + ev * (1 + 2 * a.abs()) + 2.0 ** -118
        du, dg = w * D * a, w * D * up * f
        edu = w.abs() * ((D.abs() + eD) * ea + eD * a.abs())
        edg = w.abs() * ((D.abs() + eD) * (up.abs() + eu) * ef + ((D.abs() + eD) * eu + eD * up.abs()) * f.abs())
        d = torch.cat((dg, du), 1)
        ed = torch.cat((edg, edu), 1) + 5 * STEP * d.abs()
        ed = ed + u * (d.abs() + ed) + tiny
        dx.index_add_(0, t, d @ wgu)
        edx.index_add_(0, t, ed @ wgu.abs() + (2 * I + k) * STEP * ((d.abs() + ed) @ wgu.abs()))
        d13[e], e13[e] = d.t() @ xe, ed.t() @ xe.abs() + n * STEP * ((d.abs() + ed).t() @ xe.abs())
        d2[e], e2[e] = dye.t() @ h, dye.abs().t() @ eh + n * STEP * (dye.abs().t() @ (h.abs() + eh))
        dw[at] = (D * a * up).sum(1)
        each = (D.abs() + eD) * ((a.abs() + ea) * eu + up.abs() * ea) + eD * (a * up).abs()
        edw[at] = (each + (I + 64 + 5) * STEP * ((D * a * up).abs() + each)).sum(1)
    rounded = lambda v, err: (v, err + u * (v.abs() + err) + tiny)  # noqa: E731
    out = [rounded(y, ey), rounded(dx, edx), rounded(d13, e13), rounded(d2, e2)]
    if dense:
        return [out[0], out[1], tuple(v[0] for v in out[2]), tuple(v[0] for v in out[3]), None]
    return [*out, (dw.view(T, k), edw.view(T, k) + 2.0 ** -140)]


def over(got, want):
    """How far over its bound the worst element is (<= 0: within); NaN counts as infinitely far."""
    value, bound = want
    assert got.shape == value.shape, (got.shape, value.shape)
    if not got.numel():
        return 0.0
    d = (got.double() - value).abs() - bound
    return float(torch.where(torch.isnan(d), torch.inf, d).max())


def apart(got, want):
    """The norm of the error over the result's."""
    return float((got.double() - want).norm() / want.norm().clamp(min=1e-300))


# ---------------------------------------------------------------- the block-scaled FP8 product

def make_fp8(M, N, K, seed=0, device="cuda"):
    """a, b [e4m3fn], their scales; every code that is a number comes up."""
    g = torch.Generator().manual_seed(1000 * seed + 7 * M + 3 * N + K)
    kb, nb = -(-K // 128), -(-N // 128)
    a = (torch.randn((M, K), generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    b = (torch.randn((N, K), generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    sa = torch.exp(torch.randn((M, kb), generator=g)) * 1e-2
    sb = torch.exp(torch.randn((nb, kb), generator=g)) * 1e-3
    return a.to(device), b.to(device), sa.to(device), sb.to(device)


def exact_fp8(a, b, sa, sb, bias, dtype):
    """(result in 64 bits, bound).  In a block each group of 8 products is cut 13 bits below the exponent of its
    largest: 8 * 2^-13 of that one's magnitude at most, so 2^-10 of the products' magnitudes; their fp32 sum, the
    scales' product, the blocks' fused additions and the bias' addition round as above."""
    K, N = a.shape[1], b.shape[0]
    kb = sa.shape[1]
    ad = a.double() * sa.double().repeat_interleave(128, 1)[:, :K]
    bd = b.double() * sb.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    y, mags = ad @ bd.t(), ad.abs() @ bd.abs().t()
    err = (2.0 ** -10 + (128 + kb + 4) * STEP) * mags
    if bias is not None:
        y = y + bias.double()
        err = err + STEP * (y.abs() + err)
    u, tiny = HALF[dtype], TINY[dtype]
    return y, err + u * (y.abs() + err) + tiny
