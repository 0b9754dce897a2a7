"""CPU: calls of the grouped products that no refusal of shapes or types covers:
inputs with a forward-mode tangent and copies of the slots, with the native calls
replaced by a stub, and sizes past the threads of one launch."""
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


# ---------------------------------------------------------------- copies of the slots

@pytest.fixture
def native(monkeypatch):
    """The arguments of the native calls that launch, none of which runs; sizes come from the library."""
    from td_benchmark_amd import _lib
    if not _lib.LIB_PATH.exists():
        pytest.skip("native library not built")
    real, seen = _lib.lib(), []

    class Stub:
        def __getattr__(self, name):
            if name.endswith(("_bytes", "_table", "_max_padded")):
                return getattr(real, name)
            return lambda *args: seen.append((name, args)) or 0

    monkeypatch.setattr(ops, "lib", Stub)
    monkeypatch.setattr(ops, "_need_here", lambda *args: None)
    monkeypatch.setattr(ops, "_stream_handle", lambda: 0)
    return seen


@pytest.mark.parametrize("how", ["deepcopy", "pickle", "copy"])
def test_a_copy_reads_its_own_memory(native, how):
    """Sorted ids, block experts, their count and the table come from the copy's buffer."""
    import copy
    import pickle
    slots = ops.ExpertSlots(torch.tensor([[0, 2], [1, 0], [2, -1], [1, 2]], dtype=torch.int32), 3)
    x, w, dy = _operands()
    ops.grouped_mm(x, w, slots)
    first = native[-1][1][3:7]
    start = slots._buf.data_ptr()
    new = {"deepcopy": copy.deepcopy, "pickle": lambda s: pickle.loads(pickle.dumps(s)), "copy": copy.copy}[how](slots)
    assert (new._buf.data_ptr() == start) == (how == "copy")
    assert (new.T, new.S, new.E, new.device) == (slots.T, slots.S, slots.E, slots.device)
    del slots
    for call, args, at in ((ops.grouped_mm, (x, w), 3), (ops.grouped_mm_dgrad, (dy, w), 2), (ops.grouped_mm_wgrad, (dy, x), 3)):
        call(*args, new)
        assert [p - new._buf.data_ptr() for p in native[-1][1][at:at + 4]] == [p - start for p in first], native[-1][0]
    inside = range(new._buf.data_ptr(), new._buf.data_ptr() + 4 * new._buf.numel())
    assert all(p in inside for p in native[-1][1][3:7])
    assert new.sorted_ids.data_ptr() == native[-1][1][3] and new.expert_ids.data_ptr() == native[-1][1][4]
    assert new.ntpp.data_ptr() == native[-1][1][5]


# ---------------------------------------------------------------- more workgroups than a launch has

def test_grouped_products_past_one_launch():
    """A launch has fewer than 2^32 threads: a grouped product that needs more is a bad shape, found before the launch."""
    import ctypes
    from td_benchmark_amd import _lib
    if not _lib.LIB_PATH.exists():
        pytest.skip("native library not built")
    L = _lib.lib()
    bad = next(code for code, name in _lib.STATUS.items() if name == "MOE_ERR_BAD_SHAPE")
    if torch.cuda.is_available():
        pytest.skip("a call that is not rejected would launch on host memory")
    buf = (ctypes.c_int32 * 64)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    # (S, N, K, BM, max_padded): the kernel of any widths, of few rows, of rows of whole chunks
    for S, N, K, BM, mp in ((1 << 28, 1, 1, 16, 1 << 28), (8, 8, 1024, 16, 1 << 27), (1 << 28, 8, 8, 16, 1 << 29),
                            (1 << 30, 256, 8, 32, 1 << 30)):
        for dtype in (0, 1):
            assert L.moe_grouped_mm(p, K, p, p, p, p, None, S, 1, N, K, 3, BM, mp, dtype, p, None) == bad
            if N != 8 or K != 1024:
                assert L.moe_grouped_mm_dgrad(p, p, p, p, p, None, S, K, N, 3, BM, mp, dtype, 0, p, None) == bad
        assert L.moe_grouped_gemm_int8(p, p, p, p, p, p, p, None, S, 1, 0, N, 2 * K, 3, BM, mp, 0, p, None) == bad
    for E, N, K in ((1 << 24, 1, 1), (1 << 24, 8, 8), (1 << 23, 8, 520), (1 << 24, 8, 9)):
        assert L.moe_grouped_mm_wgrad(p, p, K, p, p, p, None, 8, 1, N, K, E, 16, 64, 0, p, None) == bad
