"""The expert layers' further matrix products, as performance cases.

Four operators, each called as a program calls it:

  "grouped"       ops.grouped_mm: token slots times their own expert's weights, 16-bit floats; serving, so
                  the slots' grouping (ops.ExpertSlots) is made from the router's choice within the pass
  "grouped_train" the same product with its gradients by the tokens and by the weights: one training step's
                  share of it
  "int8"          a linear layer in 8-bit integers: ops.per_token_quant_int8 of the activations, then
                  ops.int8_scaled_mm with a scale for each token and each output channel, and a bias
  "int8_experts"  the experts' product in 8-bit integers: quant, align and
                  ops.dispatch_fused_moe_kernel(use_int8_w8a8=True, per_channel_quant=True), with or
                  without the router's weights

A case's fields:
  op       one of the four
  T, K, N  tokens, columns of the activations, columns of the product
  E, k     experts and the slots of a token ("int8": 1 and 1)
  slots    the activations have a row for each slot (the second product of a layer), not for each token
  routing  softmax (top-k of N(0,1) logits) | zipf (k distinct experts drawn per token, Zipf 1.2)
  drop     the share of slots that the router dropped (capacity): they have no expert and a zero row
  type     bf16 | fp16: the activations, the outputs and, but for int8, the weights
  weighted "int8_experts": rows times the router's weights; "int8": with a bias

K and N are those of the benchmark configurations of ``td_benchmark_amd/workloads.py`` (tiny, mixtral,
dsv3, qwen3) and of the microbench sweep's GroupGEMM shape, or generic.
"""
import math

import torch

own = False

ZIPF_ALPHA = 1.2
WEIGHT_STD = 0.02
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _case(name, op, T, K, N, E=1, k=1, slots=False, routing="softmax", drop=0.0, type="bf16", weighted=False):
    return dict(name=name, op=op, T=T, K=K, N=N, E=E, k=k, slots=slots, routing=routing, drop=drop, type=type,
                weighted=weighted)


def listed():
    return [
        # one user's token through W13 of a layer of many small experts: launches and eight experts' weights
        _case("token", "grouped", 1, 2048, 1536, 128, 8),
        # a decode batch through W2 of few large experts, fp16: the weights' stream
        _case("decode_w2", "grouped", 37, 14336, 4096, 8, 2, slots=True, type="fp16"),
        # a prompt through W13 of the microbench sweep's GroupGEMM shape, skewed routing, an odd token count
        _case("prompt", "grouped", 4093, 4096, 1536, 64, 8, routing="zipf"),
        # the benchmark's tiny layer in training: launches
        _case("tiny_train", "grouped_train", 64, 256, 1024, 8, 2),
        # widths that are no multiples of 128, fp16, a router that drops slots over the experts' capacity
        _case("ragged_train", "grouped_train", 777, 2200, 1160, 32, 4, drop=0.06, type="fp16"),
        # many small experts in training: the weights' gradients are most of the bytes
        _case("small_experts_train", "grouped_train", 4096, 2048, 1536, 128, 8),
        # few large experts in training: the matrix cores
        _case("large_experts_train", "grouped_train", 4096, 4096, 28672, 8, 2),
        # one token through the shared expert's W13: the weights' stream
        _case("int8_token", "int8", 1, 7168, 4096),
        # a decode batch, fp16 activations, with a bias, a width that is no multiple of 128
        _case("int8_decode", "int8", 45, 4096, 14344, type="fp16", weighted=True),
        # a prompt through the shared expert's W13: the matrix cores
        _case("int8_prompt", "int8", 8192, 7168, 4096),
        # a decode batch through W2 of many small experts with the router's weights
        _case("int8_experts_decode", "int8_experts", 61, 768, 2048, 128, 8, slots=True, weighted=True),
        # a prompt through W13 of many small experts
        _case("int8_experts_prompt", "int8_experts", 16384, 2048, 1536, 128, 8),
    ]


_SHAPES = ((256, 1024, 8, 2), (512, 256, 8, 2), (4096, 28672, 8, 2), (14336, 4096, 8, 2), (2048, 1536, 128, 8),
           (768, 2048, 128, 8), (4096, 1536, 64, 8), (768, 4096, 64, 8))  # K, N, E, k
_MAX_FLOP = 5.7e12
_MAX_WEIGHTS = 1.0e9


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("grouped", "grouped_train", "int8", "int8_experts"))
    step = 16 if op.startswith("int8") else 8
    E = k = 1
    while True:
        K, N = step * _log_int(rng, 128 // step, 14336 // step), 8 * _log_int(rng, 16, 2048)
        if rng.random() < 0.5:
            K, N = -(-K // 128) * 128, -(-N // 128) * 128
        if op != "int8":
            if rng.random() < 0.4:
                K, N, E, k = rng.choice(_SHAPES)
            else:
                E, k = rng.choice((4, 8, 16, 32, 60, 64, 72, 128)), rng.choice((1, 2, 4, 6, 8))
        if k <= E and E * K * N <= _MAX_WEIGHTS:
            break
    routing = "zipf" if rng.random() < 0.3 else "softmax"
    # rows that the most chosen expert makes every expert's share have room for
    rows = k if routing == "softmax" else E
    passes = 3 if op == "grouped_train" else 1
    most = _MAX_FLOP / (2.0 * passes * rows * K * N)
    T = max(1, min(_log_int(rng, 1, 16384), int(most)))
    train = op == "grouped_train"
    c = _case("", op, T, K, N, E, k, slots=op != "int8" and rng.random() < 0.5, routing=routing,
              drop=0.05 if train and rng.random() < 0.3 else 0.0, type=rng.choice(("bf16", "bf16", "fp16")),
              weighted=op.startswith("int8") and rng.random() < 0.5)
    del c["name"]
    return c


# ---------------------------------------------------------------- inputs

def _row_scale(amax):
    """max(amax / 127, 1e-12) by a true division (torch multiplies by the reciprocal of a number)."""
    return (amax / torch.full_like(amax, 127.0)).clamp(min=1e-12)


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


def _int8_weights(E, N, K, gen):
    q = torch.empty((E, N, K), dtype=torch.int8, device="cuda")
    s = torch.empty((E, N), dtype=torch.float32, device="cuda")
    step = max(1, int(2.5e8 // (N * K)))
    for e in range(0, E, step):
        n = min(step, E - e)
        w = torch.randn((n, N, K), generator=gen, device="cuda") * WEIGHT_STD
        s[e:e + n] = _row_scale(w.abs().amax(-1))
        q[e:e + n] = torch.round(w / s[e:e + n, :, None]).clamp_(-127, 127).to(torch.int8)
    return q, s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    T, K, N, E, k = (case[n] for n in ("T", "K", "N", "E", "k"))
    dt = DTYPES[case["type"]]
    rows = T * k if case["slots"] else T
    d = {"case": case, "x": torch.randn((rows, K), generator=gen, device="cuda").to(dt)}
    if case["op"] == "int8":
        q, s = _int8_weights(1, N, K, gen)
        d["w"], d["w_scale"] = q[0], s[0]
        d["bias"] = torch.randn(N, generator=gen, device="cuda").to(dt) if case["weighted"] else None
        return d
    d["ids"], d["topk_w"] = _route(case, gen)
    # the most slots of one expert, which the plain form makes room for in each of them
    used = d["ids"][d["ids"] >= 0].long()
    d["room"] = int(torch.bincount(used, minlength=E).max()) if used.numel() else 0
    if case["op"] == "int8_experts":
        d["w"], d["w_scale"] = _int8_weights(E, N, K, gen)
        # the align block size, from the average rows of an expert
        rows = T * k / E
        d["block_m"] = 32 if rows <= 28 else 64 if rows <= 44 else 128 if rows <= 100 else 256
        return d
    d["w"] = torch.empty((E, N, K), dtype=dt, device="cuda")
    step = max(1, int(2.5e8 // (N * K)))
    for e in range(0, E, step):
        n = min(step, E - e)
        d["w"][e:e + n] = torch.randn((n, N, K), generator=gen, device="cuda") * WEIGHT_STD
    if case["op"] == "grouped_train":
        d["dy"] = torch.randn((T * k, N), generator=gen, device="cuda").to(dt)
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


def _plain_quant(x):
    x = x.float()
    s = _row_scale(x.abs().amax(-1, keepdim=True))
    return torch.round(x / s).clamp_(-127.0, 127.0), s


def _plain(d):
    c = d["case"]
    T, E, k, dt = c["T"], c["E"], c["k"], DTYPES[c["type"]]
    if c["op"] == "int8":
        q, s = _plain_quant(d["x"])
        y = (q @ d["w"].float().t()) * s * d["w_scale"]
        return (y if d["bias"] is None else y + d["bias"].float()).to(dt)
    room = max(1, d["room"])
    place = _places(d["ids"], E, room)
    if c["op"] == "int8_experts":
        q, s = _plain_quant(d["x"])
        if not c["slots"]:
            q, s = q.repeat_interleave(k, 0), s.repeat_interleave(k, 0)
        y = torch.bmm(_spread(q, place, E, room), d["w"].float().transpose(1, 2)) * d["w_scale"][:, None, :]
        y = _gather(y, place) * s
        if c["weighted"]:
            y = y * d["topk_w"].view(-1, 1)
        return y.to(dt).view(T, k, -1)
    x = d["x"].float()
    xs = _spread(x if c["slots"] else x.repeat_interleave(k, 0), place, E, room)
    w = d["w"].float()
    y = _gather(torch.bmm(xs, w.transpose(1, 2)), place).to(dt)
    if c["op"] == "grouped":
        return y
    dys = _spread(d["dy"].float(), place, E, room)
    dx = _gather(torch.bmm(dys, w), place)
    if not c["slots"]:
        dx = dx.view(T, k, -1).sum(1)
    return y, dx.to(dt), torch.bmm(dys.transpose(1, 2), xs).to(dt)


def run(state):
    c = state["case"]
    if not own:
        return _plain(state)
    from td_benchmark_amd import ops
    x, w = state["x"], state["w"]
    if c["op"] == "int8":
        q, s = ops.per_token_quant_int8(x)
        return ops.int8_scaled_mm(q, w, s, state["w_scale"], bias=state["bias"], out_dtype=x.dtype)
    if c["op"] == "int8_experts":
        q, s = ops.per_token_quant_int8(x)
        sorted_ids, expert_ids, ntpp = ops.moe_align_block_size(state["ids"], state["block_m"], c["E"])
        y = torch.empty((c["T"], c["k"], c["N"]), dtype=x.dtype, device=x.device)
        ops.dispatch_fused_moe_kernel(q, w, y, s, state["w_scale"], None, state["topk_w"], sorted_ids, expert_ids,
                                      ntpp, c["weighted"], 1 if c["slots"] else c["k"],
                                      {"BLOCK_SIZE_M": state["block_m"]}, use_fp8_w8a8=False, use_int8_w8a8=True,
                                      per_channel_quant=True)
        return y
    slots = ops.ExpertSlots(state["ids"], c["E"])
    if c["op"] == "grouped":
        return ops.grouped_mm(x, w, slots)
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    y = ops.grouped_mm(x, w, slots)
    dx, dw = torch.autograd.grad(y, (x, w), state["dy"])
    return y.detach(), dx, dw


# ---------------------------------------------------------------- what a pass needs

def work(case):
    T, K, N, E, k = (case[n] for n in ("T", "K", "N", "E", "k"))
    S = T * k
    rows = S if case["slots"] else T
    if case["op"] == "int8":
        return {"bytes": 2 * T * K + N * K + 4 * N + 2 * T * N, "flops": 2 * T * N * K}
    if case["routing"] == "zipf":
        p = [(e + 1) ** -ZIPF_ALPHA for e in range(E)]
        active = sum(1.0 - (1.0 - min(1.0, k * v / sum(p))) ** T for v in p)
    else:
        active = E * (1.0 - (1.0 - k / E) ** T)
    kept = S * (1.0 - case["drop"])
    if case["op"] == "int8_experts":
        return {"bytes": 2 * rows * K + 8 * S + active * N * (K + 4) + 2 * S * N, "flops": 2 * kept * N * K}
    fwd = 2 * rows * K + 4 * S + 2 * active * N * K + 2 * S * N
    if case["op"] == "grouped":
        return {"bytes": fwd, "flops": 2 * kept * N * K}
    # the gradient of the rows is read, those of the activations and of every expert's weights are written
    return {"bytes": fwd + 2 * S * N + 2 * rows * K + 2 * E * N * K, "flops": 6 * kept * N * K}


# ---------------------------------------------------------------- in 64 bits

def exact(case, seed):
    d = prepare(case, seed)
    k = case["k"]
    x = d["x"].double()
    if case["op"].startswith("int8"):
        # the codes and the scales are fp32's, as the format defines them; the rest in 64 bits
        v = d["x"].float()
        s = _row_scale(v.abs().amax(1))
        x = torch.round(v / s[:, None]).clamp(-127, 127).double() * s.double()[:, None]
    if case["op"] == "int8":
        y = x @ d["w"].double().t() * d["w_scale"].double()
        return y if d["bias"] is None else y + d["bias"].double()
    ids = d["ids"].view(-1)
    S, N, K = ids.numel(), case["N"], case["K"]
    train = case["op"] == "grouped_train"
    y = torch.zeros((S, N), dtype=torch.float64, device="cuda")
    dx = torch.zeros_like(x) if train else None
    dw = torch.zeros((case["E"], N, K), dtype=torch.float64, device="cuda") if train else None
    for e in range(case["E"]):
        at = (ids == e).nonzero().view(-1)
        if not at.numel():
            continue
        src = at if case["slots"] else torch.div(at, k, rounding_mode="floor")
        w = d["w"][e].double()
        if case["op"] == "int8_experts":
            w = w * d["w_scale"][e].double()[:, None]
        y[at] = x[src] @ w.t()
        if train:
            dy = d["dy"][at].double()
            dx.index_add_(0, src, dy @ w)
            dw[e] = dy.t() @ x[src]
    if case["op"] == "int8_experts":
        if case["weighted"]:
            y *= d["topk_w"].double().view(-1, 1)
        return y.view(case["T"], k, N)
    return (y, dx, dw) if train else y
