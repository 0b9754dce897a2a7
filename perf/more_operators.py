"""The gated feed-forward block and the block-scaled FP8 linear layer, as performance cases.

Five operators, each called as a program calls it:

  "ffn"           ops.gated_ffn: gate and up projection, SiLU, product and down projection in 16-bit floats
                  (a shared expert or a dense layer), without gradients
  "ffn_train"     the same with the gradients by the tokens and both weights: one training step's share of it
  "experts"       ops.experts_ffn: the block by experts with the router's weights, serving; the slots' grouping
                  (ops.ExpertSlots) is made from the router's choice within the pass
  "experts_train" the same with the gradients by the tokens, both weights and the router's weights
  "fp8"           a linear layer in 8-bit floating point: ops.per_token_group_quant_fp8 of the activations (a scale
                  for each row and 128 columns), then ops.fp8_scaled_mm with a scale for each 128 x 128 block of
                  the weights

A case's fields:
  op       one of the five
  T        tokens
  H, I     hidden and intermediate size; "fp8": columns of the activations and of the product
  E, k     experts and the slots of a token (dense operators: 1 and 1)
  routing  softmax (top-k of N(0,1) logits) | zipf (k distinct experts drawn per token, Zipf 1.2)
  drop     the share of slots that the router dropped (capacity): they have no expert and add nothing
  type     bf16 | fp16: activations, weights and outputs; "fp8": the outputs
  bias     "fp8": with a bias

Sizes are those of the benchmark configurations of ``td_benchmark_amd/workloads.py`` (tiny, mixtral, dsv3, qwen3)
and of the microbench sweep's GroupGEMM shape, or generic.
"""
import math

import torch

own = False

ZIPF_ALPHA = 1.2
WEIGHT_STD = 0.02
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
FP8 = torch.float8_e4m3fn


def _case(name, op, T, H, I, E=1, k=1, routing="softmax", drop=0.0, type="bf16", bias=False):
    return dict(name=name, op=op, T=T, H=H, I=I, E=E, k=k, routing=routing, drop=drop, type=type, bias=bias)


def listed():
    return [
        # one user's token through the shared expert: the weights' stream
        _case("token", "ffn", 1, 7168, 2048),
        # a training step of the shared expert: the matrix cores
        _case("shared_train", "ffn_train", 4096, 7168, 2048),
        # widths whose rows are not whole 16-byte runs, few odd tokens, fp16
        _case("ragged_train", "ffn_train", 333, 1001, 1365, type="fp16"),
        # one user's token through a layer of many small experts: launches and eight experts' weights
        _case("experts_token", "experts", 1, 2048, 768, 128, 8),
        # a decode batch on few large experts, fp16: the weights' stream
        _case("experts_decode", "experts", 37, 4096, 14336, 8, 2, type="fp16"),
        # a prompt through the microbench sweep's GroupGEMM shape, skewed routing, an odd token count
        _case("experts_prompt", "experts", 4093, 4096, 768, 64, 8, routing="zipf"),
        # the benchmark's tiny layer in training: launches
        _case("tiny_train", "experts_train", 64, 256, 512, 8, 2),
        # many small experts in training, a router that drops slots over the experts' capacity
        _case("small_experts_train", "experts_train", 4096, 2048, 768, 128, 8, drop=0.06),
        # few large experts in training: the matrix cores
        _case("large_experts_train", "experts_train", 4096, 4096, 14336, 8, 2),
        # one token through the shared expert's W13: the weights' stream
        _case("fp8_token", "fp8", 1, 7168, 4096),
        # a decode batch with a bias, fp16 outputs, a width that is no multiple of 128
        _case("fp8_decode", "fp8", 45, 4096, 14344, type="fp16", bias=True),
        # a prompt through the shared expert's W13: the matrix cores
        _case("fp8_prompt", "fp8", 8192, 7168, 4096),
    ]


_SHAPES = ((256, 512, 8, 2), (4096, 14336, 8, 2), (2048, 768, 128, 8), (4096, 768, 64, 8), (7168, 2048, 16, 4))
_MAX_FLOP = 8.6e12
_MAX_WEIGHTS = 1.5e9


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("ffn", "ffn_train", "experts", "experts_train", "fp8"))
    E = k = 1
    while True:
        # most widths are whole 16-byte runs, some whole blocks of 128, a few anything
        H, I = _log_int(rng, 128, 14336), _log_int(rng, 128, 14336)
        step = rng.choice((16, 16, 128, 128, 128, 1))
        H, I = -(-H // step) * step, -(-I // step) * step
        if op.startswith("experts"):
            if rng.random() < 0.5:
                H, I, E, k = rng.choice(_SHAPES)
            else:
                E, k = rng.choice((4, 8, 16, 32, 60, 64, 72, 128)), rng.choice((1, 2, 4, 6, 8))
        if k <= E and 3 * E * H * I <= _MAX_WEIGHTS:
            break
    routing = "zipf" if op.startswith("experts") and rng.random() < 0.3 else "softmax"
    # rows that the most chosen expert makes every expert's share have room for
    rows = k if routing == "softmax" else E
    passes = 3 if op.endswith("train") else 1
    most = _MAX_FLOP / (6.0 * passes * rows * H * I)
    if step == 1 and E == 1:
        most /= 32
    T = max(1, min(_log_int(rng, 1, 8192), int(most)))
    c = _case("", op, T, H, I, E, k, routing=routing,
              drop=0.05 if op.startswith("experts") and rng.random() < 0.3 else 0.0,
              type=rng.choice(("bf16", "bf16", "fp16")), bias=op == "fp8" and rng.random() < 0.5)
    del c["name"]
    return c


# ---------------------------------------------------------------- inputs

def _true_div(a, b):
    """a / b by a true division (torch multiplies by the reciprocal of a number)."""
    return a / torch.full_like(a, b)


def _route(c, gen):
    T, E, k = c["T"], c["E"], c["k"]
    if c["routing"] == "zipf":
        p = torch.empty(E, device="cuda")
        p[torch.randperm(E, generator=gen, device="cuda")] = \
            torch.arange(1, E + 1, dtype=torch.float32, device="cuda").pow(-ZIPF_ALPHA)
        ids = torch.multinomial(p.expand(T, E).contiguous(), k, replacement=False, generator=gen)
        w = torch.softmax(torch.randn((T, k), generator=gen, device="cuda"), -1)
    else:
        scores = torch.softmax(torch.randn((T, E), generator=gen, device="cuda"), -1)
        w, ids = torch.topk(scores, k, dim=-1)
        w = w / w.sum(-1, keepdim=True)
    if c["drop"]:
        ids = torch.where(torch.rand((T, k), generator=gen, device="cuda") < c["drop"], -1, ids)
    return ids.to(torch.int32).contiguous(), w.float().contiguous()


def _block_weights(N, K, gen):
    """e4m3 codes [N, K] and a scale for each 128 x 128 block: max(amax / 448, 1e-12)."""
    w = torch.randn((N, K), generator=gen, device="cuda") * WEIGHT_STD
    nb, kb = -(-N // 128), -(-K // 128)
    pad = torch.zeros((nb * 128, kb * 128), device="cuda")
    pad[:N, :K] = w
    s = _true_div(pad.view(nb, 128, kb, 128).abs().amax((1, 3)), 448.0).clamp(min=1e-12)
    q = (w / s.repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]).clamp_(-448.0, 448.0)
    return q.to(FP8).contiguous(), s.contiguous()


def _weights(shape, dt, gen):
    w = torch.empty(shape, dtype=dt, device="cuda")
    step = max(1, int(2.5e8 // (shape[1] * shape[2])))
    for e in range(0, shape[0], step):
        n = min(step, shape[0] - e)
        w[e:e + n] = torch.randn((n, *shape[1:]), generator=gen, device="cuda") * WEIGHT_STD
    return w


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    T, H, I, E = (case[n] for n in ("T", "H", "I", "E"))
    dt = DTYPES[case["type"]]
    d = {"case": case}
    if case["op"] == "fp8":
        d["x"] = torch.randn((T, H), generator=gen, device="cuda").to(torch.bfloat16)
        d["w"], d["w_scale"] = _block_weights(I, H, gen)
        d["bias"] = torch.randn(I, generator=gen, device="cuda").to(dt) if case["bias"] else None
        return d
    d["x"] = torch.randn((T, H), generator=gen, device="cuda").to(dt)
    if case["op"].endswith("train"):
        d["dy"] = torch.randn((T, H), generator=gen, device="cuda").to(dt)
    if case["op"].startswith("ffn"):
        d["w13"], d["w2"] = _weights((1, 2 * I, H), dt, gen)[0], _weights((1, H, I), dt, gen)[0]
        return d
    d["w13"], d["w2"] = _weights((E, 2 * I, H), dt, gen), _weights((E, H, I), dt, gen)
    d["ids"], d["topk_w"] = _route(case, gen)
    # the most slots of one expert, which the plain form makes room for in each of them
    used = d["ids"][d["ids"] >= 0].long()
    d["room"] = int(torch.bincount(used, minlength=E).max()) if used.numel() else 0
    return d


# ---------------------------------------------------------------- the plain forms

def _places(ids, E, room):
    """For each slot its row among E * room rows, `room` of them for each expert, and one last for the slots without."""
    e = ids.reshape(-1).long()
    e = torch.where((e >= 0) & (e < E), e, E)
    order = torch.argsort(e, stable=True)
    count = torch.zeros(E + 1, dtype=torch.int64, device=e.device).scatter_add_(0, e, torch.ones_like(e))
    first = torch.cumsum(count, 0) - count
    rank = torch.empty_like(e)
    rank[order] = torch.arange(e.numel(), device=e.device) - first[e[order]]
    return torch.where(e < E, e * room + rank, E * room)


def _spread(rows, place, E, room):
    """fp32 [S, n] -> [E, room, n], zeros where an expert has no slot."""
    out = torch.zeros((E * room + 1, rows.shape[1]), dtype=torch.float32, device=rows.device)
    out.index_copy_(0, place, rows)
    return out[:-1].view(E, room, -1)


def _gather(rows, place):
    """fp32 [E, room, n] -> [S, n], zeros for the slots without an expert."""
    n = rows.shape[0] * rows.shape[1]
    got = rows.reshape(n, -1)[place.clamp(max=n - 1)]
    return torch.where((place < n)[:, None], got, 0.0)


def _plain_fp8(d):
    x, K = d["x"].float(), d["case"]["H"]
    T, kb = x.shape[0], -(-K // 128)
    pad = torch.zeros((T, kb * 128), device=x.device)
    pad[:, :K] = x
    s = _true_div(pad.view(T, kb, 128).abs().amax(-1), 448.0).clamp(min=1e-12)
    q = (pad.view(T, kb, 128) / s[:, :, None]).clamp_(-448.0, 448.0).to(FP8).float()
    a = (q * s[:, :, None]).view(T, -1)[:, :K]
    N = d["w"].shape[0]
    w = d["w"].float() * d["w_scale"].repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    y = a @ w.t()
    return (y if d["bias"] is None else y + d["bias"].float()).to(DTYPES[d["case"]["type"]])


def _plain(d):
    c = d["case"]
    if c["op"] == "fp8":
        return _plain_fp8(d)
    T, E, k, I, dt = c["T"], c["E"], c["k"], c["I"], DTYPES[c["type"]]
    train = c["op"].endswith("train")
    dense = c["op"].startswith("ffn")
    x, w13, w2 = d["x"].float(), d["w13"].float(), d["w2"].float()
    if dense:
        xs, w13, w2, weight = x[None], w13[None], w2[None], 1.0
    else:
        room = max(1, d["room"])
        place = _places(d["ids"], E, room)
        xs = _spread(x.repeat_interleave(k, 0), place, E, room)
        weight = _spread(d["topk_w"].view(-1, 1), place, E, room)
    gu = torch.bmm(xs, w13.transpose(1, 2))
    g, u = gu[..., :I], gu[..., I:]
    sig = torch.sigmoid(g)
    act = g * sig
    h = act * u * weight
    y = torch.bmm(h, w2.transpose(1, 2))
    y = y[0] if dense else _gather(y, place).view(T, k, -1).sum(1)
    if not train:
        return y.to(dt)
    dy = d["dy"].float()
    dys = dy[None] if dense else _spread(dy.repeat_interleave(k, 0), place, E, room)
    dh = torch.bmm(dys, w2)
    dgu = torch.cat((dh * weight * u * (sig + act * (1.0 - sig)), dh * weight * act), -1)
    dx = torch.bmm(dgu, w13)
    dx = dx[0] if dense else _gather(dx, place).view(T, k, -1).sum(1)
    dw13 = torch.bmm(dgu.transpose(1, 2), xs).to(dt)
    dw2 = torch.bmm(dys.transpose(1, 2), h).to(dt)
    if dense:
        return y.to(dt), dx.to(dt), dw13[0], dw2[0]
    dweight = _gather((dh * act * u).sum(-1, keepdim=True), place).view(T, k)
    return y.to(dt), dx.to(dt), dw13, dw2, dweight


def run(state):
    c = state["case"]
    if not own:
        return _plain(state)
    from td_benchmark_amd import ops
    if c["op"] == "fp8":
        q, s = ops.per_token_group_quant_fp8(state["x"])
        return ops.fp8_scaled_mm(q, state["w"], s, state["w_scale"], bias=state["bias"], out_dtype=DTYPES[c["type"]])
    x, w13, w2 = state["x"], state["w13"], state["w2"]
    if c["op"] == "ffn":
        return ops.gated_ffn(x, w13, w2)
    if c["op"] == "experts":
        return ops.experts_ffn(x, w13, w2, ops.ExpertSlots(state["ids"], c["E"]), state["topk_w"])
    x, w13, w2 = (t.detach().requires_grad_() for t in (x, w13, w2))
    if c["op"] == "ffn_train":
        y = ops.gated_ffn(x, w13, w2)
        return (y.detach(), *torch.autograd.grad(y, (x, w13, w2), state["dy"]))
    weight = state["topk_w"].detach().requires_grad_()
    y = ops.experts_ffn(x, w13, w2, ops.ExpertSlots(state["ids"], c["E"]), weight)
    return (y.detach(), *torch.autograd.grad(y, (x, w13, w2, weight), state["dy"]))


# ---------------------------------------------------------------- what a pass needs

def work(case):
    T, H, I, E, k = (case[n] for n in ("T", "H", "I", "E", "k"))
    if case["op"] == "fp8":
        return {"bytes": 2 * T * H + I * H + 4 * -(-I // 128) * -(-H // 128) + 2 * T * I + (2 * I if case["bias"] else 0),
                "flops": 2 * T * H * I}
    if case["routing"] == "zipf":
        p = [(e + 1) ** -ZIPF_ALPHA for e in range(E)]
        active = sum(1.0 - (1.0 - min(1.0, k * v / sum(p))) ** T for v in p)
    else:
        active = E * (1.0 - (1.0 - k / E) ** T)
    S = T * k
    kept = S * (1.0 - case["drop"])
    routed = 8 * S if case["op"].startswith("experts") else 0  # the ids and the weights
    fwd = 4 * T * H + routed + 6 * active * H * I
    if not case["op"].endswith("train"):
        return {"bytes": fwd, "flops": 6 * kept * H * I}
    # the gradient of the outputs is read, those of the tokens, both weights and the router's weights are written
    return {"bytes": fwd + 4 * T * H + 6 * E * H * I + routed / 2, "flops": 18 * kept * H * I}


# ---------------------------------------------------------------- in 64 bits

def _exact_fp8(d):
    # the codes and the scales are fp32's, as the format defines them; the rest in 64 bits
    c, v = d["case"], d["x"].float()
    K, N = c["H"], c["I"]
    y = torch.zeros((c["T"], N), dtype=torch.float64, device="cuda")
    for b in range(0, K, 128):
        part = v[:, b:b + 128]
        s = _true_div(part.abs().amax(1), 448.0).clamp(min=1e-12)
        q = (part / s[:, None]).clamp(-448.0, 448.0).to(FP8)
        sb = d["w_scale"][:, b // 128].double().repeat_interleave(128)[:N]
        y += (q.double() @ d["w"][:, b:b + 128].double().t()) * s.double()[:, None] * sb
    return y if d["bias"] is None else y + d["bias"].double()


def exact(case, seed):
    d = prepare(case, seed)
    if case["op"] == "fp8":
        return _exact_fp8(d)
    T, H, I, E, k = (case[n] for n in ("T", "H", "I", "E", "k"))
    dense, train = case["op"].startswith("ffn"), case["op"].endswith("train")
    w13, w2 = (d["w13"][None], d["w2"][None]) if dense else (d["w13"], d["w2"])
    ids = torch.zeros(T, dtype=torch.int64, device="cuda") if dense else d["ids"].view(-1).long()
    weight = torch.ones(T, dtype=torch.float64, device="cuda") if dense else d["topk_w"].view(-1).double()
    x = d["x"].double()
    y = torch.zeros_like(x)
    if train:
        dy = d["dy"].double()
        dx, dweight = torch.zeros_like(x), torch.zeros_like(weight)
        dw13, dw2 = (torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in (w13, w2))
    for e in range(E):
        at = (ids == e).nonzero().view(-1)
        if not at.numel():
            continue
        src = torch.div(at, k, rounding_mode="floor")
        wg, wu, wd = w13[e, :I].double(), w13[e, I:].double(), w2[e].double()
        xe, we = x[src], weight[at][:, None]
        g, u = xe @ wg.t(), xe @ wu.t()
        sig = 1.0 / (1.0 + torch.exp(-g))
        y.index_add_(0, src, (g * sig * u * we) @ wd.t())
        if not train:
            continue
        dye = dy[src]
        dh = dye @ wd
        dweight[at] = (dh * g * sig * u).sum(1)
        dh *= we
        du, dg = dh * g * sig, dh * u * sig * (1.0 + g * (1.0 - sig))
        dx.index_add_(0, src, dg @ wg + du @ wu)
        dw13[e, :I], dw13[e, I:] = dg.t() @ xe, du.t() @ xe
        dw2[e] = dye.t() @ (g * sig * u * we)
    if not train:
        return y
    if dense:
        return y, dx, dw13[0], dw2[0]
    return y, dx, dw13, dw2, dweight.view(T, k)
