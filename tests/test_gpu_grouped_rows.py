"""GPU: rows and sizes of the grouped and int8 products: slots behind padding, more
workgroups than a launch has, both tiles of the gradient by weights, and the one
rounding of the gradient by tokens."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

BF16 = torch.bfloat16


def _holes(BM, slots, S):
    """Sorted positions of one block: the given slots at its first, some inner and its last places, else padding."""
    places = [0, BM - 1, 1, BM // 2 + 1, BM // 2 - 1][:len(slots)]
    ids = torch.full((BM,), S, dtype=torch.int32)
    ids[torch.tensor(places)] = torch.tensor(slots, dtype=torch.int32)
    return ids


@pytest.mark.parametrize("a_by_pos", [False, True])
@pytest.mark.parametrize("BM,K,N", [(16, 2048, 64), (32, 4096, 64), (16, 160, 200), (32, 160, 200), (64, 160, 200), (128, 160, 264),
                                    (256, 160, 264), (64, 33, 50), (256, 33, 50)])
def test_int8_slots_behind_padding(BM, K, N, a_by_pos):
    """Every listed slot gets its row wherever it stands in its block, as in the FP8 form of the same call."""
    from td_benchmark_amd import ops
    S = 13
    g = torch.Generator(device="cuda").manual_seed(BM + K)
    blocks = [_holes(BM, [2], S), _holes(BM, [7, 0, 3, 9, 11], S), _holes(BM, [1, 4], S), torch.full((BM,), S, dtype=torch.int32),
              _holes(BM, [5, 12, 8], S).flip(0)]
    experts = [0, 1, 1, 0, -1]  # the last one's rows are zeros
    ids = torch.cat(blocks).cuda()
    a = torch.randint(-127, 128, (ids.numel() if a_by_pos else S, K), generator=g, device="cuda").to(torch.int8)
    b = torch.randint(-127, 128, (2, N, K), generator=g, device="cuda").to(torch.int8)
    sa, sb = torch.ones(a.shape[0], device="cuda"), torch.ones((2, N), device="cuda")
    y = torch.full((S, 1, N), 7.0, dtype=BF16, device="cuda")
    ops.dispatch_fused_moe_kernel(a, b, y, sa, sb, None, None, ids, torch.tensor(experts, dtype=torch.int32, device="cuda"),
                                  torch.tensor([ids.numel()], dtype=torch.int32, device="cuda"), False, 1, {"BLOCK_SIZE_M": BM},
                                  use_fp8_w8a8=False, use_int8_w8a8=True, per_channel_quant=True, a_by_pos=a_by_pos)
    want = torch.full((S, N), 7.0, dtype=BF16, device="cuda")
    for p, s in enumerate(ids.tolist()):
        if s < S:  # whole sums below 2^24 are exact in fp32, then rounded once
            e = experts[p // BM]
            want[s] = (a[p if a_by_pos else s].double() @ b[e].double().t()).float().to(BF16) if e >= 0 else 0.0
    assert (y.view(S, N) == want).all(1).tolist() == [True] * S


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("BM,K,N", [(16, 2048, 64), (32, 160, 200), (64, 160, 200), (128, 160, 264), (256, 160, 264), (256, 33, 50)])
def test_16_bit_slots_behind_padding(BM, K, N, dtype):
    """The same of the C entries of the 16-bit product and its gradient by rows, in both types of its rows."""
    from td_benchmark_amd import _lib
    S, E = 9, 2
    code = {torch.bfloat16: 0, torch.float16: 1}[dtype]
    g = torch.Generator(device="cuda").manual_seed(BM + K)
    ids = torch.cat([_holes(BM, [2, 8, 0], S), _holes(BM, [7, 3], S).flip(0), _holes(BM, [6, 1, 4, 5], S)]).cuda()
    experts = [0, 1, -1]
    eids = torch.tensor(experts, dtype=torch.int32, device="cuda")
    ntpp = torch.tensor([ids.numel()], dtype=torch.int32, device="cuda")
    # small whole numbers: every sum is exact in fp32
    x, dy = (torch.randint(-3, 4, (S, n), generator=g, device="cuda").to(dtype) for n in (K, N))
    w = torch.randint(-3, 4, (E, N, K), generator=g, device="cuda").to(dtype)
    y, dx = (torch.full((S, n), 7.5, dtype=dtype, device="cuda") for n in (N, K))
    dx32 = torch.full((S, K), 7.5, dtype=torch.float32, device="cuda")
    L, st = _lib.lib(), torch.cuda.current_stream().cuda_stream
    at = (ids.data_ptr(), eids.data_ptr(), ntpp.data_ptr(), None)
    assert L.moe_grouped_mm(x.data_ptr(), K, w.data_ptr(), *at, S, 1, N, K, E, BM, ids.numel(), code, y.data_ptr(), st) == 0
    for f32, out in ((0, dx), (1, dx32)):
        assert L.moe_grouped_mm_dgrad(dy.data_ptr(), w.data_ptr(), *at, S, N, K, E, BM, ids.numel(), code, f32, out.data_ptr(), st) == 0
    for p, s in enumerate(ids.tolist()):
        if s >= S:
            continue
        e = experts[p // BM]
        wy, wx = (x[s].double() @ w[e].double().t(), dy[s].double() @ w[e].double()) if e >= 0 else (y.new_zeros(N), y.new_zeros(K))
        assert torch.equal(y[s], wy.to(dtype)) and torch.equal(dx[s], wx.to(dtype)), (p, s)
        assert torch.equal(dx32[s], wx.float()), (p, s)


@pytest.mark.parametrize("M,N", [((1 << 30) + 5, 1), (3, (1 << 30) // 3 + 71), (1, (1 << 26) + 64 * 9 + 8)])
def test_int8_product_past_one_launch(M, N):
    """More rows or columns than one launch's threads take: parts, each with its own scales and bias."""
    from td_benchmark_amd import ops
    K = 16 if N == (1 << 26) + 64 * 9 + 8 else 1  # the last: whole chunks
    a = torch.randint(-9, 10, (M, K), device="cuda", dtype=torch.int8)
    b = torch.randint(-9, 10, (N, K), device="cuda", dtype=torch.int8)
    # scales of 1 and 2 and a bias of whole numbers: every step is exact in fp32, and rounded once
    sa, sb = (1.0 + torch.arange(n, device="cuda").remainder(5).eq(0).float() for n in (M, N))
    a, b = (a.remainder(3), b.remainder(3)) if K > 1 else (a.remainder(8), b.remainder(8))
    bias = torch.arange(N, device="cuda").remainder(7).to(BF16)
    y = ops.int8_scaled_mm(a, b, sa, sb, bias=bias)
    step = 1 << 26
    for m in range(0, M, step):
        for n in range(0, N, step):
            am, bn = a[m:m + step], b[n:n + step]
            want = sum(am[:, k:k + 1].float() * bn[:, k] for k in range(K)) * sa[m:m + step, None] * sb[n:n + step] + bias[n:n + step].float()
            assert torch.equal(y[m:m + step, n:n + step], want.to(BF16)), (m, n)


@pytest.mark.parametrize("rows", [0, 1, 31, 32, 33, 64, 97, 128, 129, 160, 225, 257, 300])
@pytest.mark.parametrize("over", [0, 1])
def test_weights_gradient_of_long_runs_in_two_rounds(over, rows):
    """64 experts of 224 slots on average and of one more in all, in two rounds of tiles of either kind; one expert
    around the lengths of a step and of the ring, and one with no slot."""
    from grouped_cases import make, off, products64
    from td_benchmark_amd import ops
    E, K, N = 64, 520, 504
    S = 224 * E + over
    x, w, _, dy = make(S, 1, E, K, N, BF16 if rows % 2 else torch.float16)
    g = torch.Generator().manual_seed(rows)
    ids = torch.randint(2, E, (S,), generator=g)
    ids[ids == 7] = 9
    ids[torch.randperm(S, generator=g)[:rows]] = 7
    ids = ids.view(-1, 1).cuda()
    (_, _, dw), (_, _, mw) = products64(x, w, ids, dy)
    for block_m in (16, 256):
        got = ops.grouped_mm_wgrad(dy, x, ops.ExpertSlots(ids, E, block_m))
        assert off(got, dw, mw, S) <= 0
        assert not got[:2].any() and (rows > 0 or not got[7].any())


@pytest.mark.parametrize("K,N", [(1, 1), (8, 8), (7, 5), (33, 47), (64, 64), (72, 136), (128, 256), (200, 264), (256, 128), (136, 520),
                                 (520, 72), (1000, 24), (130, 258)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_autograd_by_tokens_rounds_once(K, N, dtype):
    """The gradient by the tokens is one fp32 sum of k N products, rounded once, at every width and block size."""
    from grouped_cases import by_token, make, off, products64
    from td_benchmark_amd import ops
    for T, k, E, block_m, how in ((37, 2, 5, None, {}), (129, 4, 6, 16, dict(skew=True, drop=0.05)), (129, 4, 6, 64, dict(drop=0.05)),
                                  (515, 3, 6, 256, dict(skew=True))):
        x, w, ids, dy = make(T, k, E, K, N, dtype, **how)
        (_, dx, _), (_, mx, _) = products64(x, w, ids, dy)
        x.requires_grad_()
        got = torch.autograd.grad(ops.grouped_mm(x, w, ops.ExpertSlots(ids, E, block_m)), x, dy)[0]
        assert off(got, by_token(dx, k), by_token(mx, k), N + k) <= 0
