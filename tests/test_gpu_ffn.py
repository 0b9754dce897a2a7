"""GPU: the gated feed-forward block, dense and by experts, and its gradients against
64-bit results, element by element, at the sizes, strides and routings where tiles,
chunks and runs end; gradients against differences; graphs, streams, long offsets."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from ffn_cases import apart, exact, make, over  # noqa: E402
from grouped_cases import HALF  # noqa: E402

BF16, FP16 = torch.bfloat16, torch.float16


def train(x, w13, w2, slots, weight, dy):
    """y and the gradients by all of the block's operands."""
    from td_benchmark_amd import ops
    leaves = [t.detach().requires_grad_() for t in (x, w13, w2) + (() if weight is None else (weight,))]
    y = ops.gated_ffn(*leaves) if slots is None else ops.experts_ffn(*leaves[:3], slots, *leaves[3:])
    return [y.detach(), *torch.autograd.grad(y, leaves, dy)]


def serve(x, w13, w2, slots, weight):
    from td_benchmark_amd import ops
    return ops.gated_ffn(x, w13, w2) if slots is None else ops.experts_ffn(x, w13, w2, slots, weight)


def check(T, k, E, H, I, dtype, block_m=None, weighted=True, **how):
    from td_benchmark_amd import ops
    print(f"case: T={T} k={k} E={E} H={H} I={I} {dtype} BM={block_m} {how}", flush=True)
    x, w13, w2, ids, weight, dy = make(T, k, E, H, I, dtype, **how)
    if not weighted:
        weight = None
    slots = ops.ExpertSlots(ids, E, block_m) if E else None
    want = exact(x, w13, w2, ids, weight, dy)
    got = train(x, w13, w2, slots, weight, dy)
    for name, a, b in zip(("y", "dx", "dw13", "dw2", "dweights"), got, want):
        assert over(a, b) <= 0, name
    # a rounding to 16 bits is off by half a step at most, two follow one another: their errors are independent, so
    # that the norm of the whole is below that of two half steps of one sign
    if min(T, H, I) >= 32:
        for name, a, b in zip(("y", "dx", "dw13", "dw2"), got, want):
            assert apart(a, b[0]) <= 2 * HALF[dtype], name
    with torch.no_grad():
        assert torch.equal(serve(x, w13, w2, slots, weight), got[0])


SIZES = [(1, 1), (8, 8), (7, 5), (5, 16), (33, 47), (64, 72), (136, 200), (200, 136), (256, 512), (520, 264), (1032, 40),
         (1001, 65), (24, 1000)]


@pytest.mark.parametrize("H,I", SIZES)
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_sizes(H, I, dtype):
    check(37, 1, 0, H, I, dtype)
    check(70, 2, 5, H, I, dtype, drop=0.1)


@pytest.mark.parametrize("T", [1, 2, 16, 17, 32, 33, 64, 65, 128, 129, 256, 257, 600])
def test_dense_rows(T):
    check(T, 1, 0, 264, 328, BF16)
    check(T, 1, 0, 1040, 72, FP16)


@pytest.mark.parametrize("block_m", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("T", [1, 31, 129, 515])
def test_blocks(T, block_m):
    check(T, 2, 6, 136, 200, BF16, block_m)
    check(T, 4, 6, 192, 328, FP16, block_m, skew=True, drop=0.05)


@pytest.mark.parametrize("T,k,E", [(1, 1, 1), (1, 8, 128), (3, 6, 60), (700, 1, 3), (9, 8, 1023), (260, 4, 256), (90, 12, 16)])
def test_routing(T, k, E):
    check(T, k, E, 64, 72, BF16)
    check(T, k, E, 72, 64, FP16, skew=True)
    check(T, k, E, 40, 24, BF16, weighted=False)


def test_an_expert_chosen_twice():
    """A token whose slots go to the same expert, and operands that are one tensor."""
    from td_benchmark_amd import ops
    x, w13, w2, ids, weight, _ = make(90, 4, 5, 136, 72, BF16)
    ids[::2, 1] = ids[::2, 0]
    ids[::3] = 2
    got = train(x, w13, w2, ops.ExpertSlots(ids, 5), weight, x)
    for name, a, b in zip(("y", "dx", "dw13", "dw2", "dweights"), got, exact(x, w13, w2, ids, weight, x)):
        assert over(a, b) <= 0, name


def test_weights_streams():
    """Few rows on long rows of weights, in each of the two kernels for them."""
    for T, k, E, H, I in ((1, 1, 0, 2048, 1536), (19, 1, 0, 1536, 1032), (1, 4, 8, 1024, 1160), (5, 4, 64, 1032, 520),
                          (40, 2, 4, 1024, 1032)):
        check(T, k, E, H, I, BF16 if H % 16 else FP16)


def test_long_runs():
    """Tiles of 256 rows by the experts' counts with short last tiles, alone and shared, and both tiles of the
    gradient by weights."""
    check(4000, 2, 4, 264, 296, BF16, skew=True)
    check(1621, 2, 4, 4104, 4104, FP16)          # long contractions: a short tile is shared by four workgroups
    check(600, 2, 2, 4096, 2056, BF16)           # square tiles by weights
    check(1030, 1, 0, 2048, 1544, FP16)


def test_large_activations():
    """Projections of tens and hundreds, where the sigmoid is 0 or 1 and exp(-z) overflows fp32."""
    from td_benchmark_amd import ops
    x, w13, w2, ids, weight, dy = make(66, 2, 3, 128, 96, BF16)
    w13 *= 60.0
    slots = ops.ExpertSlots(ids, 3)
    got = train(x, w13, w2, slots, weight, dy)
    for name, a, b in zip(("y", "dx", "dw13", "dw2", "dweights"), got, exact(x, w13, w2, ids, weight, dy)):
        assert over(a, b) <= 0, name


def test_nothing_to_do():
    """No tokens, and no slot with an expert, also where the operands hold NaN."""
    from td_benchmark_amd import ops
    for E in (0, 3):
        x, w13, w2, ids, weight, dy = make(0, 2, E, 16, 24, BF16)
        got = train(x, w13, w2, ops.ExpertSlots(ids, 3) if E else None, weight, dy)
        assert got[0].shape == got[1].shape == (0, 16)
        assert not got[2].any() and not got[3].any() and got[2].shape == w13.shape
    x, w13, w2, ids, weight, dy = make(9, 2, 3, 16, 24, BF16)
    nan = [torch.full_like(t, float("nan")) for t in (x, w13, w2)]
    for fill in (-1, 3):
        slots = ops.ExpertSlots(torch.full_like(ids, fill), 3)
        for t in train(*nan, slots, weight, torch.full_like(dy, float("nan"))):
            assert torch.equal(t, torch.zeros_like(t))


@pytest.mark.parametrize("H,I", [(128, 256), (136, 200), (2056, 264), (33, 47)])
def test_bad_values_stay_in_their_rows(H, I):
    """A NaN in one token, in an unused expert's weights or in a dropped slot's router's weight reaches only what
    the formula lets it reach."""
    from td_benchmark_amd import ops
    T, k, E = 90, 2, 4
    x, w13, w2, ids, weight, dy = make(T, k, E, H, I, BF16)
    ids[ids == 3] = -1  # expert 3 has no slots
    want = exact(x, w13, w2, ids, weight, dy)
    w13[3] = w2[3] = float("nan")
    weight[ids < 0] = float("nan")
    x[5] = float("nan")
    got = train(x, w13, w2, ops.ExpertSlots(ids, E), weight, dy)
    hit = sorted({int(e) for e in ids[5] if e >= 0})
    assert hit
    rest = torch.arange(T, device="cuda") != 5
    for i in (0, 1):
        assert torch.isnan(got[i][5]).all()
        assert over(got[i][rest], tuple(v[rest] for v in want[i])) <= 0
    assert over(got[4][rest], tuple(v[rest] for v in want[4])) <= 0
    assert not got[4][ids < 0].any()
    for e in range(E):
        for i in (2, 3):
            if e in hit:
                assert torch.isnan(got[i][e]).any()
            else:
                assert over(got[i][e], tuple(v[e] for v in want[i])) <= 0


def test_strided_and_unaligned_operands():
    from td_benchmark_amd import ops

    def shifted(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        v = flat[1:].view(t.shape)
        v.copy_(t)
        return v
    for E in (0, 3):
        x, w13, w2, ids, weight, dy = make(50, 2, E, 136, 72, BF16)
        slots = ops.ExpertSlots(ids, 3) if E else None
        want = exact(x, w13, w2, ids, weight, dy)
        for pad, shift in ((8, 0), (16, 8), (3, 0), (8, 1)):
            wide = torch.full((50, 136 + pad + shift), float("nan"), dtype=BF16, device="cuda")
            view = wide[:, shift:shift + 136]
            view.copy_(x)
            for name, a, b in zip(("y", "dx", "dw13", "dw2", "dweights"), train(view, w13, w2, slots, weight, dy), want):
                assert over(a, b) <= 0, (name, pad, shift)
        for args in ((shifted(x), w13, w2, dy), (x, shifted(w13), w2, dy), (x, w13, shifted(w2), dy), (x, w13, w2, shifted(dy))):
            for a, b in zip(train(*args[:3], slots, weight, args[3]), want):
                assert over(a, b) <= 0


def test_expanded_gradient_and_partial_needs():
    from td_benchmark_amd import ops
    x, w13, w2, ids, weight, _ = make(33, 2, 3, 64, 72, BF16)
    slots = ops.ExpertSlots(ids, 3)
    ones = torch.ones_like(x)
    want = train(x, w13, w2, slots, weight, ones)
    operands = [x, w13, w2, weight]
    for only in range(4):
        leaves = [t.detach().clone().requires_grad_(i == only) for i, t in enumerate(operands)]
        y = ops.experts_ffn(leaves[0], leaves[1], leaves[2], slots, leaves[3])
        y.sum().backward()  # a gradient of stride 0
        assert torch.equal(leaves[only].grad, want[1 + only])
        assert all(t.grad is None for i, t in enumerate(leaves) if i != only)
    leaves = [t.detach().requires_grad_() for t in operands]
    with torch.no_grad():
        assert not ops.experts_ffn(leaves[0], leaves[1], leaves[2], slots, leaves[3]).requires_grad
    y = ops.gated_ffn(leaves[0], w13[0], w2[0])
    dy = ones.clone().requires_grad_()
    g = torch.autograd.grad(y, leaves[0], dy, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once_differentiable|differentiate"):
        g.sum().backward()


def test_a_graph_kept_and_a_changed_operand():
    """A second backward pass over a kept graph gives the same; an operand changed in between is found out."""
    from td_benchmark_amd import ops
    x, w13, w2, _, _, dy = make(40, 1, 0, 64, 72, BF16)
    leaves = [t.detach().clone().requires_grad_() for t in (x, w13, w2)]
    y = ops.gated_ffn(*leaves)
    first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    for a, b in zip(first, torch.autograd.grad(y, leaves, dy, retain_graph=True)):
        assert torch.equal(a, b)
    with torch.no_grad():
        leaves[1].mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, leaves, dy)


def test_gradients_against_differences():
    """Directional derivatives of sum(y c) against a central difference of the block in 64 bits."""
    from td_benchmark_amd import ops
    x, w13, w2, ids, weight, c = make(40, 2, 3, 64, 48, FP16)
    slots = ops.ExpertSlots(ids, 3)
    grads = train(x, w13, w2, slots, weight, c)[1:]
    want = exact(x, w13, w2, ids, weight, c)[1:]
    flat, tok = ids.reshape(-1).long(), torch.arange(80, device="cuda") // 2

    def value(x, w13, w2, weight):
        gu = (x[tok][:, None, :] * w13[flat]).sum(-1)
        h = weight.view(-1, 1) * torch.nn.functional.silu(gu[:, :48]) * gu[:, 48:]
        return float(((h[:, None, :] * w2[flat]).sum(-1) * c.double()[tok]).sum())
    g = torch.Generator().manual_seed(1)
    args = [t.double() for t in (x, w13, w2, weight)]
    for i, (grad, (_, bound)) in enumerate(zip(grads, want)):
        d = torch.randn(grad.shape, generator=g).to("cuda").double()
        h = 1e-5
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + h * d, args[i] - h * d
        diff = (value(*up) - value(*down)) / (2 * h)
        got = float((grad.double() * d).sum())
        # the elements' bounds in one direction; the difference: h^2 of the third derivative, some 1e-10 of the
        # value's scale, and 64-bit rounding over 2 h, 1e-16 / 1e-5 of it: both below 1e-9 of the magnitudes
        mags = float((grad.double().abs() * d.abs()).sum())
        assert abs(got - diff) <= float((bound * d.abs()).sum()) + 1e-7 * mags, i


def test_equal_bits():
    from td_benchmark_amd import ops
    x, w13, w2, ids, weight, dy = make(333, 4, 16, 264, 200, BF16)
    a = train(x, w13, w2, ops.ExpertSlots(ids, 16), weight, dy)
    for s in (ops.ExpertSlots(ids, 16), ops.ExpertSlots(ids.long(), 16)):
        for p, q in zip(a, train(x.clone(), w13.clone(), w2.clone(), s, weight.clone(), dy.clone())):
            assert torch.equal(p, q)


def test_a_dense_block_is_one_expert():
    """One expert that every token goes to, without weights: the dense block's result."""
    from td_benchmark_amd import ops
    x, w13, w2, _, _, dy = make(130, 1, 0, 136, 200, FP16)
    want = exact(x, w13, w2, None, None, dy)
    slots = ops.ExpertSlots(torch.zeros((130, 1), dtype=torch.int32, device="cuda"), 1)
    got = train(x, w13[None], w2[None], slots, None, dy)
    for a, b in zip(got, want):
        assert over(a if a.dim() == 2 else a[0], b) <= 0


@pytest.mark.parametrize("E", [0, 6])
def test_captured_step_replays(E):
    """Slots, block and gradients in one graph, replayed on changed inputs between other work."""
    from td_benchmark_amd import ops
    T, k, H, I = 130, 2, 136, 264
    ins = make(T, k, E, H, I, BF16)

    def step():
        x, w13, w2, ids, weight, dy = ins
        return train(x, w13, w2, ops.ExpertSlots(ids, E) if E else None, weight, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(1, 5):
        new = make(T, k, E, H, I, BF16, seed=seed, drop=0.1 * (seed - 1) if E else 0.0)
        for a, b in zip(ins, new):
            if a is not None:
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


def test_two_streams_at_once():
    from td_benchmark_amd import ops
    cases = [make(300, 4, 8, 264, 200, BF16, seed=s) for s in range(2)]
    go = lambda c: train(*c[:3], ops.ExpertSlots(c[3], 8), c[4], c[5])  # noqa: E731
    want = [go(c) for c in cases]
    torch.cuda.synchronize()
    got = []
    for c, st in zip(cases, [torch.cuda.Stream() for _ in cases]):
        with torch.cuda.stream(st):
            got.append(go(c))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_weights_past_32_bits():
    """An expert's weights whose byte offsets pass 2^32, of which the last expert's are used."""
    from td_benchmark_amd import ops
    E, H, I = 4, 12288, 24576
    w13, w2 = torch.zeros((E, 2 * I, H), dtype=BF16, device="cuda"), torch.zeros((E, H, I), dtype=BF16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    w13[3] = torch.randn((2 * I, H), generator=g, device="cuda") * 0.02
    w2[3] = torch.randn((H, I), generator=g, device="cuda") * 0.02
    x = torch.randn((20, H), generator=g, device="cuda").to(BF16)
    dy = torch.randn((20, H), generator=g, device="cuda").to(BF16)
    ids = torch.full((20, 1), 3, dtype=torch.int32, device="cuda")
    got = train(x, w13, w2, ops.ExpertSlots(ids, E), None, dy)
    want = exact(x, w13[3], w2[3], None, None, dy)
    for a, b in zip(got, want):
        assert over(a if a.shape[0] == 20 else a[3], b) <= 0
    assert not got[2][:3].any() and not got[3][:3].any()


def test_rows_past_32_bits():
    """Rows whose byte offsets pass 2^32, in x, y, dy, dx and the saved products; the last ones are checked."""
    from td_benchmark_amd import ops
    T, H, I = 270000, 8192, 2048
    g = torch.Generator(device="cuda").manual_seed(4)
    x, dy = (torch.zeros((T, H), dtype=BF16, device="cuda") for _ in range(2))
    x[-40:], dy[-40:] = (torch.randn((40, H), generator=g, device="cuda") for _ in range(2))
    w13 = (torch.randn((2 * I, H), generator=g, device="cuda") * 0.02).to(BF16)
    w2 = (torch.randn((H, I), generator=g, device="cuda") * 0.1).to(BF16)
    y, dx, dw13, dw2 = train(x, w13, w2, None, None, dy)
    want = exact(x[-40:], w13, w2, None, None, dy[-40:])
    # rows of zeros add nothing to the weights' sums
    for a, b in zip((y[-40:], dx[-40:], dw13, dw2), want):
        assert over(a, b) <= 0
    assert not y[:-40].any() and not dx[:-40].any()
    del y, dx
    with torch.no_grad():
        assert over(ops.gated_ffn(x, w13, w2)[-40:], want[0]) <= 0


def test_train_then_serve_in_fp8():
    """The shared expert's life: steps of gradient descent in 16 bits, its weights quantised by blocks, and the two
    products served in 8 bits, against the same in 64 bits from the same codes."""
    from td_benchmark_amd import ops
    T, H, I = 70, 264, 200
    x, w13, w2, _, _, target = make(T, 1, 0, H, I, BF16)
    for _ in range(3):
        w13, w2 = w13.detach().requires_grad_(), w2.detach().requires_grad_()
        y = ops.gated_ffn(x, w13, w2)
        g13, g2 = torch.autograd.grad(y, (w13, w2), ((y - target) / T).detach())
        want = exact(x, w13.detach(), w2.detach(), None, None, ((y - target) / T).detach())
        assert over(g13, want[2]) <= 0 and over(g2, want[3]) <= 0
        # a hundredth of each weight's norm a step: the block is cubic in them, and a fixed rate runs away
        w13, w2 = ((w - 0.01 * w.float().norm() / g.float().norm() * g).detach().to(BF16) for w, g in ((w13, g13), (w2, g2)))
    (q13, s13), (q2, s2) = ([t[0] for t in ops.quantize_block128(w.float()[None])] for w in (w13, w2))

    def dense(q, s, n, m):
        return q.double()[:n, :m] * s.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :m]
    xq, xs = ops.per_token_group_quant_fp8(x)
    c = ops.fp8_scaled_mm(xq, q13, xs, s13)
    x64 = xq.double()[:, :H] * xs.double().repeat_interleave(128, 1)[:, :H]
    c64 = x64 @ dense(q13, s13, 2 * I, H).t()
    # a rounding to bf16, and the 8-bit product's own cuts, 2^-10 of magnitudes that cancel in the sum: a norm
    assert apart(c, c64) <= 2 * 2.0 ** -8
    h = torch.empty((T, I), dtype=BF16, device="cuda")
    ops.silu_and_mul(h, c)
    hq, hs = ops.per_token_group_quant_fp8(h)
    y = ops.fp8_scaled_mm(hq, q2, hs, s2)
    h64 = hq.double()[:, :I] * hs.double().repeat_interleave(128, 1)[:, :I]
    assert apart(y, h64 @ dense(q2, s2, H, I).t()) <= 2 * 2.0 ** -8
