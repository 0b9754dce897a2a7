"""Inputs, 64-bit results and error bounds for the tests of the grouped 16-bit
and 8-bit products.

Bounds, element by element.  u is half a step of the output type relative to the
value (bf16 2^-8, fp16 2^-11), and its smallest step is `tiny`.  An fp32 sum of n
products whose products are exact (16-bit factors) is off by at most
n * 2^-23 * sum |products|, whatever the order and also if each addition
truncates.  So |y - exact| <= u |exact| + (1 + u) n 2^-23 sum|products| + tiny.
"""
from __future__ import annotations

import torch

HALF = {torch.bfloat16: torch.finfo(torch.bfloat16).eps / 2, torch.float16: torch.finfo(torch.float16).eps / 2}
TINY = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}


def make(T, k, E, K, N, dtype, seed=0, by_slot=False, drop=0.0, skew=False, device="cuda"):
    g = torch.Generator().manual_seed(1000 * seed + 7 * T + 3 * K + N + E)
    S = T * k
    x = torch.randn((S if by_slot else T, K), generator=g).to(dtype).to(device)
    w = (torch.randn((E, N, K), generator=g) * 0.1).to(dtype).to(device)
    scores = torch.rand((T, E), generator=g)
    if skew:  # most slots go to one expert, most experts have none
        scores[:, E // 2] += 2.0
        scores[:, : E // 3] -= 2.0
    ids = torch.topk(scores, k, dim=1).indices if T else torch.empty((0, k), dtype=torch.int64)
    if drop:
        ids = torch.where(torch.rand((T, k), generator=g) < drop, torch.tensor(-1), ids)
        ids = torch.where(torch.rand((T, k), generator=g) < drop / 2, torch.tensor(E), ids)
    dy = torch.randn((S, N), generator=g).to(dtype).to(device)
    return x, w, ids.to(device), dy


def rows_of(ids, x, k):
    """For each slot its row of x."""
    S = ids.numel()
    s = torch.arange(S, device=x.device)
    return s if x.shape[0] == S else s // k


def products64(x, w, ids, dy):
    """(y, dxs, dw) in 64 bits and the sums of their products' magnitudes."""
    S, k = ids.numel(), ids.shape[1]
    E, N, K = w.shape
    row = rows_of(ids, x, k)
    flat = ids.reshape(-1)
    out = []
    for f in (lambda t: t.double(), lambda t: t.double().abs()):
        xd, wd, dyd = f(x)[row], f(w), f(dy)
        y = torch.zeros((S, N), dtype=torch.float64, device=x.device)
        dx = torch.zeros((S, K), dtype=torch.float64, device=x.device)
        dw = torch.zeros((E, N, K), dtype=torch.float64, device=x.device)
        for e in range(E):
            at = (flat == e).nonzero().view(-1)
            if at.numel():
                y[at] = xd[at] @ wd[e].t()
                dx[at] = dyd[at] @ wd[e]
                dw[e] = dyd[at].t() @ xd[at]
        out.append((y, dx, dw))
    return out


def off(got, exact, mags, n):
    """How far over its bound the worst element is (<= 0: within)."""
    if not got.numel():
        return 0.0
    u, tiny = HALF[got.dtype], TINY[got.dtype]
    bound = u * exact.abs() + (1 + u) * n * 2.0 ** -23 * mags + tiny
    return float(((got.double() - exact).abs() - bound).max())


def by_token(t, k):
    return t.view(-1, k, t.shape[-1]).sum(1)


def off_by_token(got, dxs, mags, n, k):
    """The same for the gradient by the tokens: each slot's row is rounded to the
    type (u of its value and of its sum's error), the fp32 sum of k of them is off
    by k 2^-23 of their magnitudes, and is rounded again."""
    if not got.numel():
        return 0.0
    u, tiny = HALF[got.dtype], TINY[got.dtype]
    slot = u * dxs.abs() + (1 + u) * n * 2.0 ** -23 * mags + tiny
    exact = by_token(dxs, k)
    err = by_token(slot, k) + k * 2.0 ** -23 * by_token(dxs.abs() + slot, k)
    bound = u * exact.abs() + (1 + u) * err + tiny
    return float(((got.double() - exact).abs() - bound).max())


def quant64(x):
    """Codes and scales as the format defines them: fp32 true divisions, ties to even."""
    import numpy as np
    v = x.detach().float().cpu().numpy()
    amax = np.abs(v).max(axis=1) if v.shape[1] else np.zeros(v.shape[0], np.float32)
    s = np.maximum(amax / np.float32(127.0), np.float32(1e-12)).astype(np.float32)
    q = np.clip(np.rint((v / s[:, None]).astype(np.float32)), -127, 127).astype(np.int8)
    return torch.from_numpy(q).to(x.device), torch.from_numpy(s).to(x.device)


def off_int8(got, exact, bias_mag=0.0, tiny_scale=1.0):
    """The integer sum is exact; its conversion, the two scales, the bias and the
    routed weight each round once in fp32 (2^-24 of the value, or of the larger
    addend), then the output type's half step."""
    if not got.numel():
        return 0.0
    u, tiny = HALF[got.dtype], TINY[got.dtype]
    bound = (u + 6 * 2.0 ** -24) * (exact.abs() + 2 * bias_mag * 2.0 ** -23) + 4 * 2.0 ** -24 * bias_mag + tiny
    return float(((got.double() - exact).abs() - bound).max())
