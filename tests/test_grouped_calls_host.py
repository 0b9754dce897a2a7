"""CPU: calls of the grouped products that no refusal of shapes or types covers,
with the native library replaced by a stub: inputs with a forward-mode tangent."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import torch.autograd.forward_ad as fwd  # noqa: E402

from td_benchmark_amd import ops  # noqa: E402

BF16 = torch.bfloat16


class Slots:
    """The slots of 4 tokens of 2 on 3 experts, without a GPU."""
    T, top_k, S, E, block_size_m, max_padded = 4, 2, 8, 3, 16, 64
    _buf = torch.zeros(64, dtype=torch.int32)
    _at = (0, 0, 0, 0)


@pytest.fixture
def calls(monkeypatch):
    """The native entries called, none of which runs."""
    seen = []

    class Stub:
        def __getattr__(self, name):
            return lambda *args: seen.append(name) or 0

    monkeypatch.setattr(ops, "lib", Stub)
    monkeypatch.setattr(ops, "_need_here", lambda *args: None)
    monkeypatch.setattr(ops, "_stream_handle", lambda: 0)
    return seen


def _operands(by_slot=False):
    return torch.randn((8 if by_slot else 4, 16), dtype=BF16), torch.randn((3, 24, 16), dtype=BF16), torch.randn((8, 24), dtype=BF16)


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("entry", ["grouped_mm", "grouped_mm_dgrad", "grouped_mm_wgrad"])
def test_a_tangent_is_refused(calls, entry, grad, which):
    """A result without a tangent would count as a derivative of zero."""
    x, w, dy = _operands()
    args = {"grouped_mm": [x, w], "grouped_mm_dgrad": [dy, w], "grouped_mm_wgrad": [dy, x]}[entry]
    with fwd.dual_level():
        args[which] = fwd.make_dual(args[which].requires_grad_(grad), torch.randn_like(args[which]))
        with pytest.raises(NotImplementedError):
            getattr(ops, entry)(*args, Slots())
    assert not calls


def test_a_tangent_that_reaches_the_backward_is_refused(calls):
    x, w, dy = _operands()
    y = ops.grouped_mm(x.requires_grad_(), w, Slots())
    with fwd.dual_level():
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(y, x, fwd.make_dual(dy, torch.randn_like(dy)))
    assert calls == ["moe_grouped_mm"]


def test_plain_inputs_inside_a_dual_level(calls):
    x, w, dy = _operands()
    with fwd.dual_level():
        assert ops.grouped_mm(x, w, Slots()).shape == (8, 24)
        assert ops.grouped_mm_dgrad(dy, w, Slots()).shape == (8, 16)
        assert ops.grouped_mm_wgrad(dy, x, Slots()).shape == (3, 24, 16)
    assert calls == ["moe_grouped_mm", "moe_grouped_mm_dgrad", "moe_grouped_mm_wgrad"]
