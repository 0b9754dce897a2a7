"""GPU: the feed-forward block at counts of slots that one launch of a wave a slot
does not have the threads for."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from ffn_cases import exact, over  # noqa: E402

BF16 = torch.bfloat16


def test_more_slots_than_waves_of_one_launch():
    """2^26 slots and a few (2^32 threads with a wave a slot): y and the gradients by the tokens and the router's
    weights, all rows in parts."""
    from td_benchmark_amd import ops
    T, E, H, I = (1 << 26) + 5, 64, 8, 8
    print(f"case: T={T} E={E} H={H} I={I}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(9)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda", dtype=BF16)  # noqa: E731
    x, dy, w13, w2 = rand(T, H), rand(T, H), rand(E, 2 * I, H), rand(E, H, I)
    ids = torch.randint(0, E, (T, 1), generator=g, device="cuda", dtype=torch.int32)
    weight = torch.rand((T, 1), generator=g, device="cuda")
    slots = ops.ExpertSlots(ids, E)
    leaves = [x.requires_grad_(), weight.requires_grad_()]
    y = ops.experts_ffn(x, w13, w2, slots, weight)
    dx, dweight = torch.autograd.grad(y, leaves, dy)
    torch.cuda.synchronize()
    print("computed", flush=True)
    step = 1 << 22
    for at in range(0, T, step):
        part = slice(at, min(at + step, T))
        want = exact(x[part].detach(), w13, w2, ids[part], weight[part].detach(), dy[part])
        for name, a, b in zip(("y", "dx", "dweights"), (y[part].detach(), dx[part], dweight[part]), (want[0], want[1], want[4])):
            assert over(a, b) <= 0, (name, at)
        del want
