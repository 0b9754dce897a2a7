"""CPU: the block-scaled FP8 product has no derivatives, and says so."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import torch.autograd.forward_ad as fwd  # noqa: E402

from td_benchmark_amd import ops  # noqa: E402

BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn


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


def operands():
    return dict(a=torch.zeros((4, 160)).to(FP8), b=torch.zeros((24, 160)).to(FP8), a_scale=torch.ones((4, 2)),
                b_scale=torch.ones((1, 2)), bias=torch.zeros(24, dtype=BF16), out=torch.zeros((4, 24), dtype=BF16))


@pytest.mark.parametrize("name", ["a", "b", "a_scale", "b_scale", "bias", "out"])
def test_an_operand_that_requires_a_gradient_is_refused(calls, name):
    """A result without a graph would leave the operand's gradient out in silence."""
    args = operands()
    args[name].requires_grad_()
    with pytest.raises(NotImplementedError, match="no gradient"):
        ops.fp8_scaled_mm(**args)
    assert not calls
    with torch.no_grad():
        assert not ops.fp8_scaled_mm(**{**args, "out": None}).requires_grad
    ops.fp8_scaled_mm(**{n: t.detach() for n, t in args.items()})
    assert calls.count("moe_fp8_scaled_mm") == 2


@pytest.mark.parametrize("name", ["a_scale", "b_scale", "bias"])
def test_a_tangent_is_refused(calls, name):
    args = operands()
    with fwd.dual_level():
        args[name] = fwd.make_dual(args[name], torch.ones_like(args[name]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ops.fp8_scaled_mm(**args)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            ops.fp8_scaled_mm(**args)
    assert not calls


def test_the_int8_product_takes_what_it_took(calls):
    """Its scales and bias may require gradients, as ever; the result has none."""
    bias = torch.zeros(24, dtype=BF16, requires_grad=True)
    scales = torch.ones(4, requires_grad=True), torch.ones(24)
    y = ops.int8_scaled_mm(torch.zeros((4, 160), dtype=torch.int8), torch.zeros((24, 160), dtype=torch.int8), *scales, bias)
    assert not y.requires_grad and calls == ["moe_int8_scaled_mm"]
