"""GPU: the feed-forward block's workspaces at the C entries and what a call allocates."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from ffn_cases import exact, make, over  # noqa: E402

BF16 = torch.bfloat16


@pytest.mark.parametrize("k", [1, 2])
@pytest.mark.parametrize("H", [136, 133])
@pytest.mark.parametrize("shifts", [(0, 0, 0), (1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 1)])
def test_c_calls_in_workspaces_of_their_size(k, H, shifts):
    """y, dx and dy aligned or an element off, each pass in a workspace of just the bytes asked for, behind which and
    around y and dx nothing is written."""
    from td_benchmark_amd import _lib, ops
    T, E, I = 50, 3, 72
    print(f"case: k={k} H={H} shifts={shifts}", flush=True)
    x, w13, w2, ids, weight, dy = make(T, k, E, H, I, BF16)
    slots = ops.ExpertSlots(ids, E)
    want = exact(x, w13, w2, ids, weight, dy)
    f = ops._ffn(x, w13, w2, slots, weight)
    gu, h = (torch.empty(n, dtype=torch.uint8, device="cuda") for n in ops._ffn_saved_bytes(f))
    f.gu, f.h = gu.data_ptr(), h.data_ptr()
    n = T * H

    def place(shift):  # n values at an element's shift, and the whole they lie in
        whole = torch.full((n + 16,), 7.0, dtype=BF16, device="cuda")
        return whole[8 + shift:8 + shift + n].view(T, H), whole, shift

    def untouched(whole, shift):
        return bool((whole[:8 + shift] == 7.0).all()) and bool((whole[8 + shift + n:] == 7.0).all())

    def work(which):
        size = _lib.lib().moe_ffn_workspace_bytes(f, which)
        assert size >= 0
        return torch.full((size + 512,), 0x5A, dtype=torch.uint8, device="cuda"), size
    y, dx, dyv = (place(s) for s in shifts)
    dyv[0].copy_(dy)
    dw13, dw2, dweight = torch.empty_like(w13), torch.empty_like(w2), torch.empty_like(weight)
    ws, size = work(0 if shifts[0] else 256)
    f.workspace = ws.data_ptr() if size else None
    _lib.check(_lib.lib().moe_ffn_forward(f, y[0].data_ptr(), ops._stream_handle()), "moe_ffn_forward")
    assert bool((ws[size:] == 0x5A).all())
    ws, size = work(1 if shifts[1] or shifts[2] else 257)
    f.workspace = ws.data_ptr() if size else None
    _lib.check(_lib.lib().moe_ffn_backward(f, dyv[0].data_ptr(), dx[0].data_ptr(), dw13.data_ptr(), dw2.data_ptr(),
                                           dweight.data_ptr(), ops._stream_handle()), "moe_ffn_backward")
    assert bool((ws[size:] == 0x5A).all()) and untouched(*y[1:]) and untouched(*dx[1:])
    for name, a, b in zip(("y", "dx", "dw13", "dw2", "dweights"), (y[0], dx[0], dw13, dw2, dweight), want):
        assert over(a, b) <= 0, name


def test_no_room_for_copies_that_no_pass_makes():
    """Whole rows of long tokens: serving takes y and h, a training step the operands' gradients, what is kept and the
    gradient of the projections, and no copy of x's size beside them."""
    from td_benchmark_amd import ops
    T, H, I = 4096, 4096, 64
    x, w13, w2, _, _, dy = make(T, 1, 0, H, I, BF16)
    row, slack = 2 * T * H, 4 << 20

    def peak(call):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        out = call()
        torch.cuda.synchronize()
        assert out is not None
        return torch.cuda.max_memory_allocated() - before
    with torch.no_grad():
        assert peak(lambda: ops.gated_ffn(x, w13, w2)) <= row + 2 * T * I + slack
    leaves = [t.detach().requires_grad_() for t in (x, w13, w2)]

    def step():
        y = ops.gated_ffn(*leaves)
        return y, torch.autograd.grad(y, leaves, dy)
    # y and dx; gu, h and the gradient of the projections 14 bytes an element of [T, I]; the weights' gradients
    assert peak(step) <= 2 * row + 14 * T * I + 2 * (w13.numel() + w2.numel()) + slack


def test_only_w2_requires_a_gradient():
    """Without the projections kept: the same gradient, by experts and dense, and in C with gu NULL."""
    from td_benchmark_amd import ops
    for E in (0, 3):
        x, w13, w2, ids, weight, dy = make(70, 2, E, 136, 72, BF16)
        slots = ops.ExpertSlots(ids, E) if E else None
        leaf = w2.detach().requires_grad_()
        y = ops.gated_ffn(x, w13, leaf) if slots is None else ops.experts_ffn(x, w13, leaf, slots, weight)
        got = torch.autograd.grad(y, leaf, dy)[0]
        want = exact(x, w13, w2, ids, weight, dy)
        assert over(y.detach(), want[0]) <= 0 and over(got, want[3]) <= 0
