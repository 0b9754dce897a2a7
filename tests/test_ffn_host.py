"""CPU: what the gated feed-forward block and the block-scaled FP8 product refuse, in
Python by its own errors and in the C ABI by status codes, before any device work;
inputs with a tangent; what a backward pass asks for."""
from __future__ import annotations

import ctypes

import pytest

torch = pytest.importorskip("torch")

import torch.autograd.forward_ad as fwd  # noqa: E402

from td_benchmark_amd import _lib, ops  # noqa: E402

BF16, FP16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def L():
    if not _lib.LIB_PATH.exists():
        pytest.skip("native library not built")
    return _lib.lib()


class Slots:
    """The slots of 4 tokens of 2 on 3 experts, without a GPU."""
    T, top_k, S, E, block_size_m, max_padded = 4, 2, 8, 3, 16, 48
    _buf = torch.zeros(48, dtype=torch.int32)
    _at = (0, 0, 0, 0)


X, W13, W2 = torch.zeros((4, 16), dtype=BF16), torch.zeros((3, 24, 16), dtype=BF16), torch.zeros((3, 16, 12), dtype=BF16)
TW = torch.ones((4, 2))


@pytest.mark.parametrize("exc,args", [
    (ValueError, (X[0], W13, W2)), (TypeError, (X.float(), W13.float(), W2.float())), (TypeError, (X, W13.to(FP16), W2)),
    (TypeError, (X, W13, W2.to(FP16))), (ValueError, (X, W13[0], W2)), (ValueError, (X, W13, W2[0])), (ValueError, (X, W13[:2], W2)),
    (ValueError, (X, W13[:, :23].contiguous(), W2)), (ValueError, (X, W13[:, :22].contiguous(), W2)),
    (ValueError, (X[:, :8], W13, W2)), (ValueError, (X, W13, W2[:, :8].contiguous())), (ValueError, (X[:3], W13, W2)),
    (ValueError, (X, W13.transpose(1, 2).contiguous().transpose(1, 2), W2)), (ValueError, (X, W13, W2[:, :, :12:1].transpose(1, 2).contiguous().transpose(1, 2))),
    (ValueError, (X[:, :0], W13[:, :, :0].contiguous(), W2[:, :0].contiguous())), (ValueError, (X, W13[:, :0].contiguous(), W2[:, :, :0].contiguous())),
    (ValueError, (X[:1].expand(4, 16), W13, W2)), (ValueError, (X.t().contiguous().t(), W13, W2)),
    (TypeError, (X, W13, W2, TW.double())), (ValueError, (X, W13, W2, TW[:, :1])), (ValueError, (X, W13, W2, TW.view(-1))),
    (ValueError, (X, W13, W2, TW.t().contiguous().t())),
    (ValueError, (X, W13, W2, TW))])  # the last: CPU tensors
def test_experts_ffn_refuses(exc, args):
    with pytest.raises(exc):
        ops.experts_ffn(*args[:3], Slots(), *args[3:])


@pytest.mark.parametrize("exc,args", [
    (ValueError, (X[0], W13[0], W2[0])), (ValueError, (X, W13, W2[0])), (ValueError, (X, W13[0], W2)), (TypeError, (X.double(), W13[0], W2[0])),
    (TypeError, (X.to(FP16), W13[0], W2[0])), (ValueError, (X[:, :8], W13[0], W2[0])), (ValueError, (X, W13[0][:23], W2[0])),
    (ValueError, (X, W13[0], W2[0][:8])), (ValueError, (X, W13[0], W2[0]))])
def test_gated_ffn_refuses(exc, args):
    with pytest.raises(exc):
        ops.gated_ffn(*args)


def test_fp8_refuses():
    a, b = torch.zeros((4, 200)).to(FP8), torch.zeros((300, 200)).to(FP8)
    sa, sb = torch.ones((4, 2)), torch.ones((3, 2))
    wide = torch.zeros((1, 1 << 23), dtype=torch.uint8).view(FP8)
    for exc, args, kw in (
            (ValueError, (a[0], b, sa, sb), {}), (ValueError, (a, b[:, :100], sa, sb), {}), (TypeError, (a.view(torch.uint8), b, sa, sb), {}),
            (TypeError, (a, b.float(), sa, sb), {}), (TypeError, (a, b, sa, sb), dict(out_dtype=torch.float32)),
            (TypeError, (a, b, sa.double(), sb), {}), (ValueError, (a, b, sa[:, :1], sb), {}), (ValueError, (a, b, sa, sb[:2]), {}),
            (ValueError, (a, b, sa.t().contiguous().t(), sb), {}), (ValueError, (a[:, :0], b[:, :0], sa[:, :0], sb[:, :0]), {}),
            (ValueError, (wide, wide, torch.ones((1, 65536)), torch.ones((1, 65536))), {}),
            (TypeError, (a, b, sa, sb), dict(bias=torch.zeros(300))), (ValueError, (a, b, sa, sb), dict(bias=torch.zeros(299, dtype=BF16))),
            (ValueError, (a, b, sa, sb), dict(out=torch.zeros((4, 299), dtype=BF16))),
            (TypeError, (a, b, sa, sb), dict(out=torch.zeros((4, 300)))),
            (ValueError, (a, b.t().contiguous().t(), sa, sb), {}), (ValueError, (a, b, sa, sb), {})):
        with pytest.raises(exc):
            ops.fp8_scaled_mm(*args, **kw)


@pytest.fixture
def calls(monkeypatch):
    """The native entries called, none of which runs, with their arguments."""
    seen = []

    class Stub:
        def __getattr__(self, name):
            return lambda *args: seen.append((name, args)) or 0

    monkeypatch.setattr(ops, "lib", Stub)
    monkeypatch.setattr(ops, "_need_here", lambda *args: None)
    monkeypatch.setattr(ops, "_stream_handle", lambda: 0)
    return seen


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("grad", [False, True])
def test_a_tangent_is_refused(calls, grad, which):
    """A result without a tangent would count as a derivative of zero."""
    args = [t.clone() for t in (X, W13, W2, TW)]
    with fwd.dual_level():
        args[which] = fwd.make_dual(args[which].requires_grad_(grad), torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError):
            ops.experts_ffn(*args[:3], Slots(), args[3])
        if which < 3:
            dense = [args[0], args[1][0], args[2][0]]
            with pytest.raises(NotImplementedError):
                ops.gated_ffn(*dense)
    assert not calls


def test_a_tangent_that_reaches_the_backward_is_refused(calls):
    y = ops.gated_ffn(X.clone().requires_grad_(), W13[0], W2[0])
    with fwd.dual_level():
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(y, y.grad_fn.next_functions[0][0].variable, fwd.make_dual(torch.ones_like(y), torch.ones_like(y)))
    assert "moe_ffn_backward" not in [name for name, _ in calls]


@pytest.mark.parametrize("need", [(1, 1, 1, 1), (1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1)])
def test_the_backward_asks_for_what_is_needed(calls, need):
    leaves = [t.clone().requires_grad_(bool(n)) for t, n in zip((X, W13, W2, TW), need)]
    y = ops.experts_ffn(*leaves[:3], Slots(), leaves[3])
    torch.autograd.grad(y, [t for t in leaves if t.requires_grad], torch.ones_like(y))
    name, args = calls[-1]
    assert name == "moe_ffn_backward" and [p is not None for p in args[2:6]] == [bool(n) for n in need]


def test_no_products_are_saved_without_gradients(calls):
    """gu is what only a backward pass reads."""
    ops.gated_ffn(X, W13[0], W2[0])
    assert calls[-1][0] == "moe_ffn_forward" and not calls[-1][1][0].gu
    ops.gated_ffn(X.clone().requires_grad_(), W13[0], W2[0])
    assert calls[-1][1][0].gu
    with torch.no_grad():
        ops.gated_ffn(X.clone().requires_grad_(), W13[0], W2[0])
    assert not calls[-1][1][0].gu


# ---------------------------------------------------------------- the C ABI

def _codes(*names):
    by_name = {name: code for code, name in _lib.STATUS.items()}
    return [by_name["MOE_" + n] for n in names]


def test_c_ffn_refuses(L):
    ok, bad, null, block, topk, experts = _codes("OK", "ERR_BAD_SHAPE", "ERR_NULL_POINTER", "ERR_BAD_BLOCK_SIZE", "ERR_BAD_TOPK",
                                                 "ERR_BAD_EXPERTS")
    buf = (ctypes.c_int32 * 256)()  # host memory: only ever passed to a rejected call
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    base = dict(T=4, H=16, I=12, ldx=16, max_padded=48, top_k=2, E=3, block_size_m=16, dtype=0, x=p, w13=p, w2=p, topk_weights=p,
                sorted_ids=p, expert_ids=p, ntpp=p, expert_table=p, h=p, gu=p, workspace=p)
    common = ((bad, dict(T=-1)), (bad, dict(H=0)), (bad, dict(I=0)), (bad, dict(ldx=15)), (bad, dict(dtype=2)), (bad, dict(max_padded=-1)),
              (bad, dict(max_padded=0)), (bad, dict(max_padded=15)),
              (bad, dict(H=(1 << 29) + 1, ldx=(1 << 29) + 1)), (bad, dict(I=(1 << 28) + 1)), (bad, dict(T=1 << 30)),
              (topk, dict(top_k=0)), (experts, dict(E=0)), (block, dict(block_size_m=48)), (null, dict(ntpp=None)),
              (null, dict(sorted_ids=None)), (null, dict(expert_ids=None)),
              (experts, dict(sorted_ids=None, expert_ids=None, ntpp=None)))
    only = ((null, dict(x=None)), (null, dict(w13=None)), (null, dict(w2=None)), (null, dict(h=None)), (null, dict(workspace=None)),
            (bad, dict(x=p + 1)), (bad, dict(w13=p + 1)), (bad, dict(w2=p + 1)), (bad, dict(h=p + 8)), (bad, dict(gu=p + 8)),
            (bad, dict(workspace=p + 8)), (bad, dict(topk_weights=p + 2)))
    for want, kw in common:
        f = _lib.MoeFfn(**{**base, **kw})
        assert L.moe_ffn_workspace_bytes(f, 0) == want and L.moe_ffn_workspace_bytes(f, 1) == want, kw
    for want, kw in common + only:
        f = _lib.MoeFfn(**{**base, **kw})
        assert L.moe_ffn_forward(f, p, None) == want, kw
        assert L.moe_ffn_backward(f, p, p, p, p, p, None) == want, kw
    f = _lib.MoeFfn(**base)
    assert L.moe_ffn_workspace_bytes(None, 0) == L.moe_ffn_forward(None, p, None) == L.moe_ffn_backward(None, p, p, p, p, p, None) == null
    assert L.moe_ffn_forward(f, None, None) == null and L.moe_ffn_forward(f, p + 1, None) == bad
    assert L.moe_ffn_backward(f, None, p, p, p, p, None) == null
    for at in range(1, 6):
        args = [p] * 6
        args[at - 1] += 1
        assert L.moe_ffn_backward(f, *args[:5], None) == bad, at
    assert L.moe_ffn_backward(_lib.MoeFfn(**{**base, "gu": None}), p, p, p, p, p, None) == null
    assert L.moe_ffn_backward(_lib.MoeFfn(**{**base, "topk_weights": None}), p, p, p, p, p, None) == null
    assert L.moe_ffn_forward(_lib.MoeFfn(**{**base, "T": 0}), p, None) == ok
    assert L.moe_ffn_backward(f, p, None, None, None, None, None) == ok  # no gradient is asked for


def test_c_fp8_refuses(L):
    ok, bad, null = _codes("OK", "ERR_BAD_SHAPE", "ERR_NULL_POINTER")
    buf = (ctypes.c_int32 * 256)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    mm = lambda a=p, lda=160, sa=p, b=p, ldb=160, sb=p, bias=p, M=4, N=24, K=160, dt=0, y=p, ldy=24, ws=p: L.moe_fp8_scaled_mm(  # noqa: E731
        a, lda, sa, b, ldb, sb, bias, M, N, K, dt, y, ldy, ws, None)
    for want, kw in ((null, dict(a=None)), (null, dict(b=None)), (null, dict(sa=None)), (null, dict(sb=None)), (null, dict(y=None)),
                     (bad, dict(M=-1)), (bad, dict(N=-1)), (bad, dict(K=0)), (bad, dict(K=1 << 23, lda=1 << 23, ldb=1 << 23)),
                     (bad, dict(lda=159)), (bad, dict(ldb=159)), (bad, dict(ldy=23)), (bad, dict(dt=2)), (bad, dict(M=1 << 31)),
                     (bad, dict(y=p + 1)), (bad, dict(bias=p + 1)), (bad, dict(sa=p + 2)), (bad, dict(sb=p + 2)), (bad, dict(ws=p + 8)),
                     (null, dict(a=p + 1, ws=None)), (null, dict(ldb=161, ws=None)), (ok, dict(M=0)), (ok, dict(N=0))):
        assert mm(**kw) == want, kw
    size = L.moe_fp8_scaled_mm_workspace_bytes
    assert size(p, 160, p, 160, 4, 24, 160) == 0
    assert size(p + 1, 160, p, 160, 4, 24, 160) == 768 and size(p, 160, p, 161, 4, 24, 160) == 3840
    assert size(p, 161, p, 161, 4, 24, 161) == 768 + 4352
    for args in ((p, 15, p, 16, 4, 24, 16), (p, 16, p, 15, 4, 24, 16), (p, 16, p, 16, -1, 24, 16), (p, 16, p, 16, 4, -1, 16)):
        assert size(*args) == bad
