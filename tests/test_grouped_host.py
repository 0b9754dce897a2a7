"""CPU: what the 16-bit grouped and the int8 products refuse, in Python by its
own errors and in the C ABI by status codes, before any device work."""
from __future__ import annotations

import ctypes

import pytest

torch = pytest.importorskip("torch")

from td_benchmark_amd import _lib, ops  # noqa: E402

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def L():
    if not _lib.LIB_PATH.exists():
        pytest.skip("native library not built")
    return _lib.lib()


class FakeSlots:
    """What the checks read of ExpertSlots, without a GPU."""
    T, top_k, S, E, block_size_m, max_padded = 4, 2, 8, 3, 16, 48
    sorted_ids = _buf = torch.zeros(48, dtype=torch.int32)


def test_slots_refuse():
    ids = torch.zeros((4, 2), dtype=torch.int32)
    for exc, args in ((ValueError, (ids.view(-1), 3)), (TypeError, (ids.float(), 3)), (ValueError, (ids, 0)),
                      (ValueError, (ids, 1024)), (ValueError, (ids[:, :0], 3)), (ValueError, (ids, 3, 48)),
                      (ValueError, (ids, 3))):  # the last: a CPU tensor
        with pytest.raises(exc):
            ops.ExpertSlots(*args)


def test_grouped_mm_refuses():
    x, w, dy = torch.zeros((4, 16), dtype=BF16), torch.zeros((3, 24, 16), dtype=BF16), torch.zeros((8, 24), dtype=BF16)
    s = FakeSlots()
    for exc, a, b in ((ValueError, x, w[0]), (TypeError, x.float(), w.float()), (TypeError, x, w.to(FP16)),
                      (ValueError, x, w[:2]), (ValueError, x[:, :8], w), (ValueError, x[0], w), (ValueError, x[:3], w),
                      (ValueError, x, w.transpose(1, 2).contiguous().transpose(1, 2)), (ValueError, x, w)):
        with pytest.raises(exc):
            ops.grouped_mm(a, b, s)
    for exc, a, b in ((ValueError, dy[0], w), (TypeError, dy.float(), w), (ValueError, dy[:4], w), (TypeError, dy, w.to(FP16)),
                      (ValueError, dy, w[:2]), (ValueError, dy[:, :8], w), (ValueError, dy, w)):
        with pytest.raises(exc):
            ops.grouped_mm_dgrad(a, b, s)
    for exc, a, b in ((ValueError, dy[0], x), (TypeError, dy.float(), x), (TypeError, dy, x.to(FP16)), (ValueError, dy[:4], x),
                      (ValueError, dy, x[:3]), (ValueError, dy, x)):
        with pytest.raises(exc):
            ops.grouped_mm_wgrad(a, b, s)


def test_int8_refuses():
    a, b = torch.zeros((4, 16), dtype=torch.int8), torch.zeros((6, 16), dtype=torch.int8)
    sa, sb = torch.ones(4), torch.ones(6)
    for exc, args, kw in (
            (ValueError, (a[0], b, sa, sb), {}), (ValueError, (a, b[:, :8], sa, sb), {}), (TypeError, (a.to(torch.uint8), b, sa, sb), {}),
            (TypeError, (a, b.float(), sa, sb), {}), (TypeError, (a, b, sa, sb), dict(out_dtype=torch.float32)),
            (TypeError, (a, b, sa.double(), sb), {}), (ValueError, (a, b, sa[:1], sb), {}), (ValueError, (a, b, sa, sa), {}),
            (TypeError, (a, b, sa, sb), dict(bias=torch.zeros(6))), (ValueError, (a, b, sa, sb), dict(bias=torch.zeros(5, dtype=BF16))),
            (ValueError, (a, b, sa, sb), dict(out=torch.zeros((4, 5), dtype=BF16))), (ValueError, (a, b, sa, sb), {}),
            (ValueError, (torch.zeros((1, 131072), dtype=torch.int8), torch.zeros((6, 131072), dtype=torch.int8), sa[:1], sb), {})):
        with pytest.raises(exc):
            ops.int8_scaled_mm(*args, **kw)
    for exc, x in ((ValueError, torch.zeros(4, dtype=BF16)), (TypeError, torch.zeros((4, 4))), (ValueError, torch.zeros((4, 4), dtype=BF16))):
        with pytest.raises(exc):
            ops.per_token_quant_int8(x)
    with pytest.raises(NotImplementedError):
        ops.moe_kernel_quantize_input(torch.zeros((4, 4), dtype=BF16), None, torch.int8, False)
    with pytest.raises(NotImplementedError):
        ops.moe_kernel_quantize_input(torch.zeros((4, 4), dtype=BF16), None, torch.int8, True, [128, 128])


def test_int8_dispatch_refuses():
    A, B = torch.zeros((4, 16), dtype=torch.int8), torch.zeros((3, 8, 16), dtype=torch.int8)
    C, sa, sb = torch.zeros((4, 2, 8), dtype=BF16), torch.ones((4, 1)), torch.ones((3, 8))
    srt, eids, n = torch.zeros(48, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    base = dict(A=A, B=B, C=C, A_scale=sa, B_scale=sb, B_zp=None, topk_weights=None, sorted_token_ids=srt, expert_ids=eids,
                num_tokens_post_padded=n, mul_routed_weight=False, top_k=2, config={"BLOCK_SIZE_M": 16}, use_fp8_w8a8=False,
                use_int8_w8a8=True, per_channel_quant=True)
    for exc, change in (
            (NotImplementedError, dict(per_channel_quant=False)), (NotImplementedError, dict(use_fp8_w8a8=True)),
            (NotImplementedError, dict(use_int8_w8a16=True)), (NotImplementedError, dict(block_shape=[128, 128])),
            (NotImplementedError, dict(B_zp=1)), (NotImplementedError, dict(B_bias=1)), (NotImplementedError, dict(tile_m=64)),
            (NotImplementedError, dict(tile_order=1)), (TypeError, dict(A=A.float())), (TypeError, dict(B=B.float())),
            (TypeError, dict(C=C.float())), (ValueError, dict(A=A[:, :8])), (ValueError, dict(B=B[0])),
            (ValueError, dict(C=torch.zeros((4, 2, 7), dtype=BF16))), (ValueError, dict(A=A[:3], A_scale=sa[:3])),
            (ValueError, dict(A_scale=sa[:3])), (ValueError, dict(B_scale=sb[:2])), (ValueError, dict(top_k=0)),
            (ValueError, dict(config={"BLOCK_SIZE_M": 24})), (ValueError, dict(mul_routed_weight=True)),
            (ValueError, dict(mul_routed_weight=True, topk_weights=torch.ones(7))), (ValueError, dict(expert_ids=eids[:2])),
            (ValueError, dict(a_by_pos=True)), (ValueError, {})):
        with pytest.raises(exc):
            ops.dispatch_fused_moe_kernel(**{**base, **change})


def test_c_entries_refuse(L):
    E = {name: code for code, name in _lib.STATUS.items()}
    buf = (ctypes.c_int32 * 256)()  # host memory: only ever passed to a rejected call
    p = ctypes.cast(buf, ctypes.c_void_p)
    odd = ctypes.c_void_p(ctypes.addressof(buf) + 1)
    bad, null, block, topk, experts = (E[n] for n in ("MOE_ERR_BAD_SHAPE", "MOE_ERR_NULL_POINTER", "MOE_ERR_BAD_BLOCK_SIZE",
                                                      "MOE_ERR_BAD_TOPK", "MOE_ERR_BAD_EXPERTS"))
    ok = E["MOE_OK"]
    mm = lambda x=p, ldx=16, w=p, srt=p, S=8, k=2, N=24, K=16, e=3, bm=16, mp=48, dt=0, y=p: L.moe_grouped_mm(  # noqa: E731
        x, ldx, w, srt, p, p, None, S, k, N, K, e, bm, mp, dt, y, None)
    for want, kw in ((null, dict(x=None)), (null, dict(w=None)), (null, dict(srt=None)), (null, dict(y=None)), (bad, dict(ldx=15)),
                     (bad, dict(S=-1)), (bad, dict(N=-1)), (bad, dict(K=-1)), (bad, dict(dt=2)), (bad, dict(mp=-1)), (bad, dict(x=odd)),
                     (topk, dict(k=0)), (experts, dict(e=0)), (block, dict(bm=48)), (ok, dict(S=0)), (ok, dict(N=0))):
        assert mm(**kw) == want, kw
    dg = lambda dy=p, w=p, S=8, N=24, K=16, e=3, bm=16, mp=48, dt=0, dx=p: L.moe_grouped_mm_dgrad(  # noqa: E731
        dy, w, p, p, p, None, S, N, K, e, bm, mp, dt, 0, dx, None)
    for want, kw in ((null, dict(dy=None)), (null, dict(w=None)), (null, dict(dx=None)), (bad, dict(N=-1)), (bad, dict(dt=7)),
                     (bad, dict(dx=odd)), (experts, dict(e=-1)), (block, dict(bm=0)), (ok, dict(S=0)), (ok, dict(K=0))):
        assert dg(**kw) == want, kw
    wg = lambda dy=p, x=p, ldx=16, S=8, k=2, N=24, K=16, e=3, bm=16, mp=48, dt=0, dw=p: L.moe_grouped_mm_wgrad(  # noqa: E731
        dy, x, ldx, p, p, p, None, S, k, N, K, e, bm, mp, dt, dw, None)
    for want, kw in ((null, dict(dy=None)), (null, dict(x=None)), (null, dict(dw=None)), (bad, dict(ldx=8)), (bad, dict(dt=-1)),
                     (bad, dict(dw=odd)), (topk, dict(k=-1)), (experts, dict(e=0)), (block, dict(bm=512)), (ok, dict(N=0))):
        assert wg(**kw) == want, kw
    sl = lambda ids=p, nb=4, S=8, e=3, bm=16, out=p, mp=4096, ws=p: L.moe_expert_slots(  # noqa: E731
        ids, nb, S, e, bm, out, p, p, p, mp, ws, None)
    for want, kw in ((null, dict(ids=None)), (null, dict(out=None)), (null, dict(ws=None)), (bad, dict(nb=2)), (bad, dict(S=-1)),
                     (experts, dict(e=0)), (experts, dict(e=1024)), (block, dict(bm=8)), (E["MOE_ERR_CAPACITY"], dict(mp=4))):
        assert sl(**kw) == want, kw
    qn = lambda x=p, ldx=16, T=4, H=16, dt=0, q=p, s=p: L.moe_quant_int8(x, ldx, T, H, dt, q, s, None)  # noqa: E731
    for want, kw in ((null, dict(x=None)), (null, dict(q=None)), (null, dict(s=None)), (bad, dict(ldx=8)), (bad, dict(T=-1)),
                     (bad, dict(H=-1)), (bad, dict(dt=3)), (bad, dict(x=odd)), (ok, dict(T=0))):
        assert qn(**kw) == want, kw
    im = lambda a=p, lda=16, sa=p, b=p, ldb=16, sb=p, M=4, N=8, K=16, dt=0, y=p, ldy=8: L.moe_int8_scaled_mm(  # noqa: E731
        a, lda, sa, b, ldb, sb, None, M, N, K, dt, y, ldy, None)
    for want, kw in ((null, dict(a=None)), (null, dict(b=None)), (null, dict(sa=None)), (null, dict(sb=None)), (null, dict(y=None)),
                     (bad, dict(lda=8)), (bad, dict(ldb=8)), (bad, dict(ldy=4)), (bad, dict(M=-1)), (bad, dict(K=131072, lda=131072, ldb=131072)),
                     (bad, dict(dt=9)), (bad, dict(y=odd)), (ok, dict(M=0)), (ok, dict(N=0))):
        assert im(**kw) == want, kw
    ig = lambda a=p, sa=p, b=p, sb=p, S=8, k=2, N=8, K=16, e=3, bm=16, mp=48, dt=0, y=p: L.moe_grouped_gemm_int8(  # noqa: E731
        a, sa, b, sb, p, p, p, None, S, k, 0, N, K, e, bm, mp, dt, y, None)
    for want, kw in ((null, dict(a=None)), (null, dict(b=None)), (null, dict(sa=None)), (null, dict(sb=None)), (null, dict(y=None)),
                     (bad, dict(K=131072)), (bad, dict(dt=2)), (bad, dict(S=-1)), (topk, dict(k=0)), (experts, dict(e=0)),
                     (block, dict(bm=20)), (ok, dict(S=0))):
        assert ig(**kw) == want, kw
    ss = lambda d=p, T=4, k=2, H=8, dt=0, y=p: L.moe_slot_sum(d, T, k, H, dt, y, None)  # noqa: E731
    for want, kw in ((null, dict(d=None)), (null, dict(y=None)), (bad, dict(T=-1)), (bad, dict(dt=2)), (bad, dict(d=odd)),
                     (topk, dict(k=0)), (ok, dict(T=0)), (ok, dict(H=0))):
        assert ss(**kw) == want, kw


def test_bounds_find_a_planted_mistake():
    """The element-wise bounds of the GPU tests let a correctly rounded result
    through and stop one that misses a single product, a slot or a half step."""
    from grouped_cases import make, off, products64
    x, w, ids, dy = make(20, 2, 3, 64, 48, BF16, device="cpu")
    (y, dx, dw), (my, mx, mw) = products64(x, w, ids, dy)
    for exact, mags, n in ((y, my, 64), (dx, mx, 48), (dw, mw, 40)):
        good = exact.to(BF16)
        assert off(good, exact, mags, n) <= 0
        assert off(good * (1 + 2.0 ** -6), exact, mags, n) > 0
    x2 = x.clone()
    x2[:, 63] = 0
    assert off(products64(x2, w, ids, dy)[0][0].to(BF16), y, my, 64) > 0
