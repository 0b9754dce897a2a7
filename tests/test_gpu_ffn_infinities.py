"""GPU: infinities at widths that are padded to whole chunks: the padding counts for
nothing, so that a row that the formula makes infinite is infinite and not NaN."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from ffn_cases import make  # noqa: E402

BF16, FP16 = torch.bfloat16, torch.float16


def same(got, want, name):
    """Alike where the formula gives no number: infinities of the same sign, NaN; numbers elsewhere."""
    assert torch.equal(torch.isnan(got), torch.isnan(want)), name
    hit = torch.isinf(want)
    assert torch.equal(torch.isinf(got), hit) and torch.equal(got[hit].double(), want[hit].double()), name


@pytest.mark.parametrize("I", [1, 7, 8, 33, 40, 61, 129])
@pytest.mark.parametrize("H,T,E,k,block_m", [(24, 5, 0, 1, None), (33, 70, 0, 1, None), (1096, 5, 0, 1, None), (1096, 9, 3, 2, 16),
                                             (40, 300, 3, 2, 256), (64, 90, 3, 1, 64)])
def test_an_infinite_row(H, I, T, E, k, block_m):
    """All operands positive: with an infinity in a token its projections, h and y are infinite; with one in dy its D and
    with it the gradients that it reaches."""
    from td_benchmark_amd import ops
    dtype = FP16 if I % 2 else BF16
    print(f"case: H={H} I={I} T={T} E={E} k={k} BM={block_m} {dtype}", flush=True)
    x, w13, w2, ids, weight, dy = (None if t is None else t if i == 3 else t.abs() * 0.1 + 0.01
                                   for i, t in enumerate(make(T, k, E, H, I, dtype)))
    inf = float("inf")
    for where in ("x", "dy"):
        xs, dys = x.clone(), dy.clone()
        (xs if where == "x" else dys)[2, H // 2] = inf
        leaves = [t.detach().requires_grad_() for t in (xs, w13, w2) + ((weight,) if E else ())]
        y = ops.experts_ffn(*leaves[:3], ops.ExpertSlots(ids, E, block_m), leaves[3]) if E else ops.gated_ffn(*leaves)
        got = [y.detach(), *torch.autograd.grad(y, leaves, dys)]
        # the formulas in 64 bits, slot by slot, with the activation as it is defined for an infinity: z s(z)
        flat = ids.reshape(-1).long() if E else torch.zeros(T, dtype=torch.int64, device="cuda")
        tok = torch.arange(T * k, device="cuda") // k
        w13d, w2d = (t.double() if E else t.double()[None] for t in (w13, w2))
        w = weight.double().view(-1, 1) if E else torch.ones((T, 1), dtype=torch.float64, device="cuda")
        want = [torch.zeros((T, H), dtype=torch.float64, device="cuda") for _ in range(2)]
        dw = torch.zeros(T * k, dtype=torch.float64, device="cuda")
        for s in range(T * k) if T * k <= 20 else [s for s in range(T * k) if int(tok[s]) in (0, 2, T - 1)]:
            e, t = int(flat[s]), int(tok[s])
            wgu, wd = w13d[e], w2d[e]
            gu = (xs[t].double()[None] * wgu).sum(1)
            g, u = gu[:I], gu[I:]
            sg = 1 / (1 + torch.exp(-g))
            h = w[s] * g * sg * u
            D = (dys[t].double()[:, None] * wd).sum(0)
            dG, dU = w[s] * D * u * (sg + g * sg * (1 - sg)), w[s] * D * g * sg
            want[0][t] += (h[None] * wd).sum(1)
            want[1][t] += (torch.cat((dG, dU))[:, None] * wgu).sum(0)
            dw[s] = (D * g * sg * u).sum()
        rows = torch.tensor([0, 2, T - 1], device="cuda")
        assert bool(torch.isinf(want[0][2]).all()) == (where == "x")
        same(got[0][rows], want[0][rows], "y")
        same(got[1][rows], want[1][rows], "dx")
        if E:
            same(got[4][rows], dw.view(T, k)[rows].to(got[4].dtype), "dweights")
