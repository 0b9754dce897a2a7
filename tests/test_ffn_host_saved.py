"""CPU: what the feed-forward block keeps for its backward pass."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from td_benchmark_amd import ops  # noqa: E402

BF16 = torch.bfloat16
T, H, I = 8, 16, 24


@pytest.mark.parametrize("need", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 1, 1)])
def test_the_projections_are_kept_where_their_gradient_is_needed(monkeypatch, need):
    """gu is kept for the gradients by x and w13; w2's reads h alone.  Both passes have h behind it."""
    seen = {}

    class Stub:
        def __getattr__(self, name):
            def call(*args):
                f = args[0]
                seen[name] = (f.gu, f.h)
                return 0
            return call

    monkeypatch.setattr(ops, "lib", Stub)
    monkeypatch.setattr(ops, "_need_here", lambda *args: None)
    monkeypatch.setattr(ops, "_stream_handle", lambda: 0)
    leaves = [torch.zeros(s, dtype=BF16).requires_grad_(bool(n)) for s, n in zip(((T, H), (2 * I, H), (H, I)), need)]
    y = ops.gated_ffn(*leaves)
    saved = y.grad_fn.saved_tensors[-1]
    gu = 8 * T * I if need[0] or need[1] else 0
    assert saved.numel() == gu + 2 * T * I
    torch.autograd.grad(y, [t for t in leaves if t.requires_grad], torch.ones_like(y))
    at = saved.data_ptr()
    assert seen["moe_ffn_forward"] == seen["moe_ffn_backward"] == (at if gu else None, at + gu)
