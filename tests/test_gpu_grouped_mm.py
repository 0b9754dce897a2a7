"""GPU: the experts' product in 16-bit floats and its gradients against 64-bit
results, element by element, at the sizes, strides and routings where tiles,
chunks and runs end."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from grouped_cases import (by_token, make, off, off_by_token, products64)  # noqa: E402

BF16, FP16 = torch.bfloat16, torch.float16


def check_all(T, k, E, K, N, dtype, block_m=None, **how):
    from td_benchmark_amd import ops
    print(f"case: T={T} k={k} E={E} K={K} N={N} {dtype} BM={block_m} {how}", flush=True)
    x, w, ids, dy = make(T, k, E, K, N, dtype, **how)
    slots = ops.ExpertSlots(ids, E, block_m)
    (y, dx, dw), (my, mx, mw) = products64(x, w, ids, dy)
    assert off(ops.grouped_mm(x, w, slots), y, my, K) <= 0
    assert off(ops.grouped_mm_dgrad(dy, w, slots), dx, mx, N) <= 0
    n = ids.numel()
    assert off(ops.grouped_mm_wgrad(dy, x, slots), dw, mw, n) <= 0
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    out = ops.grouped_mm(xg, wg, slots)
    gx, gw = torch.autograd.grad(out, (xg, wg), dy)
    assert gx.shape == x.shape and gw.shape == w.shape and gx.dtype == gw.dtype == dtype
    if how.get("by_slot") or k == 1:
        assert off(gx, dx, mx, N) <= 0
    else:
        assert off_by_token(gx, dx, mx, N, k) <= 0
    assert off(gw, dw, mw, n) <= 0


SIZES = [  # K, N: one, below and over a chunk, a step, a tile; odd; ragged multiples of 8
    (1, 1), (8, 8), (7, 5), (33, 47), (64, 64), (72, 136), (128, 256), (200, 264), (256, 128), (136, 520), (520, 72),
    (1000, 24), (130, 258),
]


@pytest.mark.parametrize("K,N", SIZES)
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_sizes(K, N, dtype):
    check_all(37, 2, 5, K, N, dtype)
    check_all(150, 3, 4, K, N, dtype, by_slot=True, drop=0.1)


@pytest.mark.parametrize("block_m", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("T", [1, 2, 31, 64, 129, 515])
def test_blocks(T, block_m):
    check_all(T, 2, 6, 136, 200, BF16, block_m)
    check_all(T, 4, 6, 192, 328, FP16, block_m, skew=True, drop=0.05)


@pytest.mark.parametrize("T,k,E", [(1, 1, 1), (1, 8, 128), (3, 6, 60), (700, 1, 3), (9, 8, 1023), (260, 4, 256)])
def test_routing(T, k, E):
    check_all(T, k, E, 64, 72, BF16)
    check_all(T, k, E, 72, 64, FP16, by_slot=True, skew=True)


def test_long_contractions_and_wide_outputs():
    check_all(70, 2, 2, 6144, 88, BF16)
    check_all(70, 2, 2, 88, 6152, FP16)
    check_all(3000, 2, 2, 72, 80, BF16)  # many slots an expert: the weights' gradient is the long sum


def test_no_tokens_no_slots_no_columns():
    from td_benchmark_amd import ops
    x, w, ids, dy = make(0, 2, 3, 16, 24, BF16)
    slots = ops.ExpertSlots(ids, 3)
    assert ops.grouped_mm(x, w, slots).shape == (0, 24)
    assert ops.grouped_mm_dgrad(dy, w, slots).shape == (0, 16)
    assert torch.equal(ops.grouped_mm_wgrad(dy, x, slots), torch.zeros_like(w))
    # every slot dropped: zero rows, zero gradients, also where the operands hold NaN
    x, w, ids, dy = make(9, 2, 3, 16, 24, BF16)
    slots = ops.ExpertSlots(torch.full_like(ids, 3), 3)
    nan_x, nan_dy = torch.full_like(x, float("nan")), torch.full_like(dy, float("nan"))
    assert torch.equal(ops.grouped_mm(nan_x, w, slots), torch.zeros_like(dy))
    assert torch.equal(ops.grouped_mm_dgrad(nan_dy, w, slots), torch.zeros((18, 16), dtype=BF16, device="cuda"))
    assert torch.equal(ops.grouped_mm_wgrad(nan_dy, nan_x, slots), torch.zeros_like(w))
    # no columns of the contraction, or of the output
    x, w, ids, dy = make(9, 2, 3, 0, 24, BF16)
    slots = ops.ExpertSlots(ids, 3)
    assert torch.equal(ops.grouped_mm(x, w, slots), torch.zeros_like(dy))
    assert ops.grouped_mm_wgrad(dy, x, slots).shape == (3, 24, 0)
    x, w, ids, dy = make(9, 2, 3, 16, 0, BF16)
    slots = ops.ExpertSlots(ids, 3)
    assert ops.grouped_mm(x, w, slots).shape == (18, 0)
    assert torch.equal(ops.grouped_mm_dgrad(dy, w, slots), torch.zeros((18, 16), dtype=BF16, device="cuda"))


@pytest.mark.parametrize("K,N", [(128, 256), (136, 200), (2056, 264)])
def test_bad_values_stay_in_their_rows(K, N):
    """An infinity or a NaN in one slot's row, in a dropped slot's row or in an
    unused expert's weights reaches only what the formula lets it reach."""
    from td_benchmark_amd import ops
    T, k, E = 90, 2, 4
    x, w, ids, dy = make(T, k, E, K, N, BF16)
    ids[ids == 3] = -1  # expert 3 has no slots
    w[3] = float("nan")
    (y, dx, dw), (my, mx, mw) = products64(x, w, ids, dy)
    x[5] = float("nan")
    dy[11] = float("inf")
    dropped = (ids.view(-1) < 0).nonzero().view(-1)
    assert dropped.numel()
    dy[dropped] = float("nan")
    slots = ops.ExpertSlots(ids, E)
    got = ops.grouped_mm(x, w, slots)
    bad = torch.zeros(T * k, dtype=torch.bool, device="cuda")
    bad[10:12] = ids.view(-1)[10:12] >= 0
    assert torch.isnan(got[bad]).all()
    assert off(got[~bad], y[~bad], my[~bad], K) <= 0
    got = ops.grouped_mm_dgrad(dy, w, slots)
    bad = torch.zeros(T * k, dtype=torch.bool, device="cuda")
    bad[11] = ids.view(-1)[11] >= 0
    assert not torch.isfinite(got[bad]).any()
    assert off(got[~bad], dx[~bad], mx[~bad], N) <= 0
    got = ops.grouped_mm_wgrad(dy, x, slots)
    hit = {int(e) for e in ids.view(-1)[10:12] if e >= 0}
    for e in range(E):
        if e in hit:
            assert not torch.isfinite(got[e]).any()
        else:
            assert off(got[e], dw[e], mw[e], T * k) <= 0


def test_strided_rows():
    from td_benchmark_amd import ops
    for pad, shift in ((8, 0), (16, 8), (3, 0), (8, 1)):  # whole chunks, and rows that start inside one
        x, w, ids, dy = make(50, 2, 3, 136, 72, BF16)
        wide = torch.full((50, 136 + pad + shift), float("nan"), dtype=BF16, device="cuda")
        view = wide[:, shift:shift + 136]
        view.copy_(x)
        slots = ops.ExpertSlots(ids, 3)
        assert torch.equal(ops.grouped_mm(view, w, slots), ops.grouped_mm(x, w, slots)) or shift or pad % 8
        (y, dx, dw), (my, mx, mw) = products64(x, w, ids, dy)
        assert off(ops.grouped_mm(view, w, slots), y, my, 136) <= 0
        assert off(ops.grouped_mm_wgrad(dy, view, slots), dw, mw, 100) <= 0


def test_unaligned_bases():
    from td_benchmark_amd import ops
    x, w, ids, dy = make(40, 2, 3, 64, 72, FP16)
    slots = ops.ExpertSlots(ids, 3)
    (y, dx, dw), (my, mx, mw) = products64(x, w, ids, dy)

    def shifted(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        v = flat[1:].view(t.shape)
        v.copy_(t)
        return v
    assert off(ops.grouped_mm(shifted(x), shifted(w), slots), y, my, 64) <= 0
    assert off(ops.grouped_mm_dgrad(shifted(dy), shifted(w), slots), dx, mx, 72) <= 0
    assert off(ops.grouped_mm_wgrad(shifted(dy), shifted(x), slots), dw, mw, 80) <= 0


def test_equal_bits_and_id_types():
    from td_benchmark_amd import ops
    x, w, ids, dy = make(333, 4, 16, 264, 392, BF16)
    a = ops.ExpertSlots(ids.to(torch.int64), 16)
    b = ops.ExpertSlots(ids.to(torch.int32), 16)
    strided = torch.stack((ids, ids + 1), dim=2)[:, :, 0]
    c = ops.ExpertSlots(strided, 16)
    for f in (lambda s: ops.grouped_mm(x, w, s), lambda s: ops.grouped_mm_dgrad(dy, w, s, by_token=True),
              lambda s: ops.grouped_mm_wgrad(dy, x, s)):
        r = f(a)
        assert torch.equal(r, f(a)) and torch.equal(r, f(b)) and torch.equal(r, f(c))


def test_the_ids_may_change_afterwards():
    from td_benchmark_amd import ops
    x, w, ids, dy = make(65, 2, 4, 64, 72, BF16)
    slots = ops.ExpertSlots(ids, 4)
    want = ops.grouped_mm(x, w, slots), ops.grouped_mm_wgrad(dy, x, slots)
    ids.fill_(-1)
    assert torch.equal(ops.grouped_mm(x, w, slots), want[0])
    assert torch.equal(ops.grouped_mm_wgrad(dy, x, slots), want[1])


def test_gradients_against_differences():
    """The directional derivative of sum(y * c) by x and by w against a central
    difference of the product in 64 bits."""
    from td_benchmark_amd import ops
    x, w, ids, c = make(40, 2, 3, 64, 48, FP16)
    slots = ops.ExpertSlots(ids, 3)
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    (ops.grouped_mm(xg, wg, slots) * c).sum().backward()
    flat = ids.reshape(-1)
    g = torch.Generator().manual_seed(1)

    def value(xd, wd):
        y = torch.einsum("sk,snk->sn", xd[torch.arange(80, device="cuda") // 2], wd[flat])
        return float((y * c.double()).sum())
    for leaf, grad, at in ((x, xg.grad, 0), (w, wg.grad, 1)):
        d = torch.randn(leaf.shape, generator=g).to("cuda").double()
        args = [x.double(), w.double()]
        h = 1e-3
        up, down = list(args), list(args)
        up[at], down[at] = args[at] + h * d, args[at] - h * d
        diff = (value(*up) - value(*down)) / (2 * h)  # the product is linear in each: exact but for 64-bit rounding
        got = float((grad.double() * d).sum())
        # each gradient element is off by two roundings of 2^-11 of the slots' magnitudes, all of one sign at worst
        mags = float((grad.double().abs() * d.abs()).sum())
        assert abs(got - diff) <= 4 * 2.0 ** -11 * mags


def test_expanded_gradient_and_partial_needs():
    from td_benchmark_amd import ops
    x, w, ids, _ = make(33, 2, 3, 64, 72, BF16)
    slots = ops.ExpertSlots(ids, 3)
    ones = torch.ones((66, 72), dtype=BF16, device="cuda")
    xg = x.clone().requires_grad_()
    ops.grouped_mm(xg, w, slots).sum().backward()  # a gradient of stride 0
    assert torch.equal(xg.grad, ops.grouped_mm_dgrad(ones, w, slots, by_token=True))
    wg = w.clone().requires_grad_()
    ops.grouped_mm(x, wg, slots).sum().backward()
    assert torch.equal(wg.grad, ops.grouped_mm_wgrad(ones, x, slots))
    with torch.no_grad():
        assert not ops.grouped_mm(xg, wg, slots).requires_grad
    dy = ones.clone().requires_grad_()
    g = torch.autograd.grad(ops.grouped_mm(xg, wg, slots), xg, dy, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once_differentiable|differentiate"):
        g.sum().backward()


def test_a_training_layer():
    """Both products with SiLU*up between and the router's weights after, as a
    layer uses them, against the layer in 64 bits."""
    from td_benchmark_amd import ops
    T, k, E, H, I = 203, 2, 5, 128, 96
    g = torch.Generator().manual_seed(5)
    x = torch.randn((T, H), generator=g).cuda().to(BF16)
    w13 = (torch.randn((E, 2 * I, H), generator=g) * 0.1).cuda().to(BF16)
    w2 = (torch.randn((E, H, I), generator=g) * 0.1).cuda().to(BF16)
    p = torch.softmax(torch.randn((T, E), generator=g), -1).cuda()
    tw, ids = torch.topk(p, k, dim=1)
    up = torch.randn((T, H), generator=g).cuda()

    def layer(x, w13, w2, tw, product):
        c = product(x, w13)
        h = torch.nn.functional.silu(c[:, :I]) * c[:, I:]
        return (product(h, w2).view(T, k, H) * tw[..., None]).sum(1)

    leaves = [t.clone().requires_grad_() for t in (x, w13, w2, tw)]
    slots = ops.ExpertSlots(ids, E)
    y = layer(*leaves, lambda a, b: ops.grouped_mm(a, b, slots))
    y.float().backward(up)
    exact = [t.double().requires_grad_() for t in (x, w13, w2, tw)]
    flat = ids.reshape(-1)

    def product64(a, b):
        rows = a if a.shape[0] == T * k else a.repeat_interleave(k, 0)
        return torch.einsum("sk,snk->sn", rows, b[flat])
    y64 = layer(*exact, product64)
    y64.backward(up.double())
    # the chain rounds to bf16 about ten times (2^-8 each) on the way to a leaf; rounding errors of one sign in
    # all of them would give ten half steps of the result's norm
    for got, want in ((y.detach(), y64.detach()), *((a.grad, b.grad) for a, b in zip(leaves, exact))):
        assert float((got.double() - want).norm() / want.norm()) <= 10 * 2.0 ** -8


def test_captured_step_replays():
    """Slots, product and gradients in one graph, replayed on changed inputs between other work."""
    from td_benchmark_amd import ops
    T, k, E, K, N = 130, 2, 6, 136, 264
    x, w, ids, dy = make(T, k, E, K, N, BF16)

    def step():
        slots = ops.ExpertSlots(ids, E)
        return (ops.grouped_mm(x, w, slots), ops.grouped_mm_dgrad(dy, w, slots, by_token=True),
                ops.grouped_mm_wgrad(dy, x, slots))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(1, 4):
        x2, w2, ids2, dy2 = make(T, k, E, K, N, BF16, seed=seed, drop=0.1 * (seed - 1))
        for a, b in ((x, x2), (w, w2), (ids, ids2), (dy, dy2)):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


def test_two_streams_at_once():
    from td_benchmark_amd import ops
    cases = [make(300, 4, 8, 264, 520, BF16, seed=s) for s in range(2)]
    want = []
    for x, w, ids, dy in cases:
        slots = ops.ExpertSlots(ids, 8)
        want.append((ops.grouped_mm(x, w, slots), ops.grouped_mm_wgrad(dy, x, slots)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for (x, w, ids, dy), st in zip(cases, streams):
        with torch.cuda.stream(st):
            slots = ops.ExpertSlots(ids, 8)
            got.append((ops.grouped_mm(x, w, slots), ops.grouped_mm_wgrad(dy, x, slots)))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_tensors_past_32_bits():
    """Weights, rows and outputs whose byte offsets pass 2^32."""
    from td_benchmark_amd import ops
    E, N, K = 5, 16384, 32768  # 1 GiB of weights an expert
    T = 132000                 # rows of 64 KiB in x (8.6e9 bytes) and of 32 KiB in y
    w = torch.zeros((E, N, K), dtype=BF16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    w[4] = torch.randn((N, K), generator=g, device="cuda") * 0.02
    x = torch.zeros((T, K), dtype=BF16, device="cuda")
    x[-40:] = torch.randn((40, K), generator=g, device="cuda")
    ids = torch.full((T, 1), -1, dtype=torch.int32, device="cuda")
    ids[-40:] = 4
    slots = ops.ExpertSlots(ids, E)
    y = ops.grouped_mm(x, w, slots)
    xd, wd = x[-40:].double(), w[4].double()
    assert off(y[-40:], xd @ wd.t(), xd.abs() @ wd.abs().t(), K) <= 0
    assert not y[:-40].any()
    dy = y
    dy[-40:] = torch.randn((40, N), generator=g, device="cuda")
    dyd = dy[-40:].double()
    dw = ops.grouped_mm_wgrad(dy, x, slots)
    assert off(dw[4], dyd.t() @ xd, dyd.abs().t() @ xd.abs(), 40) <= 0
    assert not dw[:4].any()
    del dw
    dx = ops.grouped_mm_dgrad(dy, w, slots)
    assert off(dx[-40:], dyd @ wd, dyd.abs() @ wd.abs(), N) <= 0
    assert not dx[:-40].any()
