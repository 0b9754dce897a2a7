"""GPU: the feed-forward block in every tile of its products, forward and backward,
against 64-bit results element by element, on rows that are random throughout."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from ffn_cases import apart, exact, over  # noqa: E402
from ffn_tile_cases import ALL_TILES, CASES, tiles_of  # noqa: E402
from grouped_cases import HALF  # noqa: E402

BF16, FP16 = torch.bfloat16, torch.float16
# slots over whole tiles of 256 rows: none, tiles of one row and just up to 64, which are short, and longer ones
RESTS = (1, 40, 64, 65, 0, 200)


def routed(T, k, E, gen):
    """Each slot's expert: the experts' counts leave the rests above, the slots that are left over have no expert, and a
    token may have an expert twice."""
    S = T * k
    each = S // E
    counts = [each // 256 * 256 + RESTS[e % 6] if each >= 256 else max(0, each - e % 7) for e in range(E)]
    flat, at = torch.full((S,), -1, dtype=torch.int32), 0
    for e, n in enumerate(counts):
        flat[at:at + n] = e
        at += n
    if at < S:
        flat[at::2] = E
    return flat[torch.randperm(S, generator=gen)].view(T, k)


def make(T, k, E, H, I, dtype):  # noqa: E741
    host = torch.Generator().manual_seed(T + 3 * H + 7 * I + E)
    gen = torch.Generator(device="cuda").manual_seed(T + 3 * H + 7 * I + E)
    rand = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    lead = (E,) if E else ()
    x, dy = rand(T, H).to(dtype), rand(T, H).to(dtype)
    w13 = (rand(*lead, 2 * I, H) * min(1.0, 2.0 * H ** -0.5)).to(dtype)
    w2 = (rand(*lead, H, I) * 0.1).to(dtype)
    if not E:
        return x, w13, w2, None, None, dy
    return x, w13, w2, routed(T, k, E, host).cuda(), torch.rand((T, k), generator=gen, device="cuda"), dy


@pytest.mark.parametrize("at", range(len(CASES)))
def test_tiles(at):
    from td_benchmark_amd import ops
    T, k, E, H, I, block_m = CASES[at]  # noqa: E741
    dtype = FP16 if at % 3 == 0 else BF16
    print(f"case: {CASES[at]} {dtype} {sorted(tiles_of(*CASES[at]))}", flush=True)
    assert tiles_of(*CASES[at]) <= ALL_TILES
    x, w13, w2, ids, weight, dy = make(T, k, E, H, I, dtype)
    leaves = [t.detach().requires_grad_() for t in (x, w13, w2) + ((weight,) if E else ())]
    if E:
        y = ops.experts_ffn(*leaves[:3], ops.ExpertSlots(ids, E, block_m), leaves[3])
    else:
        y = ops.gated_ffn(*leaves)
    got = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    want = exact(x, w13, w2, ids, weight, dy)
    for name, a, b in zip(("y", "dx", "dw13", "dw2", "dweights"), got, want):
        assert over(a, b) <= 0, name
    # a rounding to 16 bits is off by half a step at most, two follow one another: their errors are independent, so
    # that the norm of the whole is below that of two half steps of one sign
    if min(T, H, I) >= 32:
        for name, a, b in zip(("y", "dx", "dw13", "dw2"), got, want):
            if bool(b[0].any()):
                assert apart(a, b[0]) <= 2 * HALF[dtype], name
