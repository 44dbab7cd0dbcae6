"""Measured cases of the 8-bit operators: the W8A8 linear layer, the mixture-of-experts feed-forward block built on
its grouped form, and the ordering of tokens by expert with its gradient.

`run` computes each case in plain torch operations, or -- where `own` is set -- through this package's operators on
the same inputs.  `exact` restates the definitions in 64 bits.

Definitions
    quantise     s = amax(|row|) / 127,  q = rint(127 * x / amax(|row|)) with ties to even; an all-zero row has s = 0, q = 0
    linear       y[m, n] = sx[m] * sw[n] * sum_k qx[m, k] * qw[n, k] + bias[n]
    experts      for the entries (t, j) of each expert e = ids[t, j] (ids outside [0, E) name no expert):
                     h = silu(g) * u with (g, u) = the two halves of linear(x[t]; w13[e]),  o = linear(h; w2[e]),
                     y[t] = sum_j weights[t, j] * o(t, j)
    order        entries (t, j) sorted by expert, stable in t * k + j: pos[t, j] is the row of the entry (-1: no expert),
                     offsets[e] the first row of expert e; rows[pos[t, j]] = x[t], the rows behind the last entry are zero;
                     y[t] = sum_j w[t, j] * ys[pos[t, j]]
    order back   d_ys[pos[t, j]] = w[t, j] * dy[t],  d_w[t, j] = <dy[t], ys[pos[t, j]]>,  dx[t] = sum_j d_rows[pos[t, j]]
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 128          # rows of one block of the plain grouped product


def listed():
    return [
        # the gate + up projection of a 70B decoder layer, one new token
        {"name": "linear decode 1 row", "op": "linear", "M": 1, "K": 8192, "N": 57344, "type": "bf16", "bias": False},
        # gate + up of an 8B layer under a batch of 23 sequences, with sizes that fit no tile
        {"name": "linear decode 23 rows odd sizes", "op": "linear", "M": 23, "K": 4112, "N": 24571, "type": "fp16", "bias": True},
        # a down projection, the layer kept in 8 bits most often, on a ragged prompt chunk
        {"name": "linear 333 rows down", "op": "linear", "M": 333, "K": 28672, "N": 8192, "type": "bf16", "bias": False},
        # a prompt of 4096 tokens through the gate + up projection
        {"name": "linear prefill 4096 rows", "op": "linear", "M": 4096, "K": 8192, "N": 57344, "type": "bf16", "bias": False},
        # one new token of a model with many small experts
        {"name": "experts decode 1 token", "op": "experts", "T": 1, "H": 2048, "I": 1024, "E": 64, "k": 8, "drop": 0.0, "type": "bf16"},
        # a decode batch that reaches nearly every expert
        {"name": "experts decode 48 tokens", "op": "experts", "T": 48, "H": 4096, "I": 1408, "E": 32, "k": 4, "drop": 0.0, "type": "fp16"},
        # a prompt chunk with padding tokens and few large experts
        {"name": "experts 777 tokens padded", "op": "experts", "T": 777, "H": 4096, "I": 7168, "E": 8, "k": 2, "drop": 0.1, "type": "fp16"},
        # a prompt batch over many small experts
        {"name": "experts prefill 4096 tokens", "op": "experts", "T": 4096, "H": 2048, "I": 1024, "E": 64, "k": 8, "drop": 0.0, "type": "bf16"},
        # decode: few tokens, many experts
        {"name": "order 64 tokens", "op": "order", "T": 64, "H": 2048, "E": 128, "k": 8, "drop": 0.0, "type": "bf16"},
        # the largest prompt batch
        {"name": "order 16384 tokens", "op": "order", "T": 16384, "H": 4096, "E": 256, "k": 8, "drop": 0.02, "type": "bf16"},
        # training in 32 bits with sizes that fit no vector, and a training batch in 16
        {"name": "order back 2500 tokens odd", "op": "back", "T": 2500, "H": 1001, "E": 60, "k": 5, "drop": 0.1, "type": "fp32"},
        {"name": "order back 8192 tokens", "op": "back", "T": 8192, "H": 4096, "E": 64, "k": 4, "drop": 0.0, "type": "fp16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "experts", "order", "back"])
    if op == "linear":
        while True:
            c = {"op": op, "M": _log(rng, 1, 4096), "K": 16 * _log(rng, 16, 1792), "N": _log(rng, 256, 57344),
                 "type": rng.choice(["bf16", "fp16"]), "bias": rng.random() < 0.3}
            if c["N"] * c["K"] <= 57344 * 8192:
                return c
    if op == "experts":
        while True:
            c = {"op": op, "T": _log(rng, 1, 4096), "H": 16 * _log(rng, 32, 256), "I": 16 * _log(rng, 16, 448),
                 "E": _log(rng, 4, 128), "drop": rng.choice([0.0, 0.0, 0.1]), "type": rng.choice(["bf16", "fp16"])}
            c["k"] = rng.randint(1, min(8, c["E"]))
            blocks = c["T"] * c["k"] / BLOCK + c["E"]
            if blocks * c["H"] * c["I"] <= 8 * 2.0e9 and c["E"] * c["H"] * c["I"] <= 4.0e8 and c["T"] * c["k"] <= 32768:
                return c
    while True:
        c = {"op": op, "T": _log(rng, 1, 16384), "H": _log(rng, 64, 4096), "E": _log(rng, 2, 256),
             "drop": rng.choice([0.0, 0.02, 0.3]), "type": rng.choice(["bf16", "fp16", "fp32"])}
        c["k"] = rng.randint(1, min(8, c["E"]))
        if rng.random() < 0.6:
            c["H"] = -(-c["H"] // 64) * 64
        if c["T"] * c["k"] * c["H"] * (2 if c["type"] == "fp32" else 1) <= 16384 * 8 * 4096:
            return c


def _activations(rows, width, dtype, gen):
    """N(0, 1) with one channel in two hundred twenty times as large."""
    x = torch.randn(rows, width, generator=gen, device="cuda")
    wide = torch.rand(width, generator=gen, device="cuda") < 0.005
    return (x * torch.where(wide, 20.0, 1.0)).to(dtype)


def _codes(shape, gen):
    """Codes of Gaussian weights whose largest value of a row is about four deviations."""
    q = torch.empty(shape, dtype=torch.int8, device="cuda")
    flat = q.view(-1, shape[-1])
    step = max(1, (1 << 28) // shape[-1])
    for i in range(0, flat.shape[0], step):
        part = flat[i:i + step]
        part.copy_(torch.randn(part.shape, generator=gen, device="cuda").mul_(32).round_().clamp_(-127, 127))
    return q


def _scales(shape, width, gen):
    return (torch.rand(shape, generator=gen, device="cuda") + 0.5) * (4.0 / 127 / math.sqrt(width))


def _route(T, E, k, drop, gen):
    """Experts of each token by a router with favourites, all k of a token different; `drop` of the tokens are padding."""
    logits = torch.randn(T, E, generator=gen, device="cuda") + torch.randn(E, generator=gen, device="cuda") * 0.5
    top, ids = logits.topk(k, dim=-1)
    w = torch.softmax(top, dim=-1)
    if drop > 0:
        ids = torch.where(torch.rand(T, 1, generator=gen, device="cuda") < drop, -1, ids)
    return ids, w


def _sorted(ids, E):
    """pos and offsets of the definition, in torch operations."""
    flat = ids.reshape(-1)
    known = (flat >= 0) & (flat < E)
    key = torch.where(known, flat, E)
    order = torch.argsort(key, stable=True)
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device=ids.device)
    pos = torch.where(known, place, -1).to(torch.int32).view(ids.shape)
    counts = torch.zeros(E + 1, dtype=torch.int64, device=ids.device).index_add_(0, key, torch.ones_like(key))
    offsets = torch.cat((counts.new_zeros(1), counts[:E].cumsum(0))).to(torch.int32)
    return pos, offsets


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["type"]]
    s = {"case": dict(case)}
    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        s["x"] = _activations(M, K, dtype, gen)
        s["wq"], s["ws"] = _codes((N, K), gen), _scales((N,), K, gen)
        s["bias"] = torch.randn(N, generator=gen, device="cuda") * 0.5 if case["bias"] else None
        return s
    T, H, E, k = case["T"], case["H"], case["E"], case["k"]
    s["ids"], s["w"] = _route(T, E, k, case["drop"], gen)
    if case["op"] == "experts":
        inner = case["I"]
        s["x"] = _activations(T, H, dtype, gen)
        s["w13q"], s["w13s"] = _codes((E, 2 * inner, H), gen), _scales((E, 2 * inner), H, gen)
        s["w2q"], s["w2s"] = _codes((E, H, inner), gen), _scales((E, H), inner, gen)
        return s
    s["ys"] = torch.randn(T * k, H, generator=gen, device="cuda").to(dtype)
    if case["op"] == "order":
        s["x"] = torch.randn(T, H, generator=gen, device="cuda").to(dtype)
        return s
    s["dy"] = torch.randn(T, H, generator=gen, device="cuda").to(dtype)
    s["d_rows"] = torch.randn(T * k, H, generator=gen, device="cuda").to(dtype)
    s["pos"], s["offsets"] = _sorted(s["ids"], E)           # kept from the forward pass
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------

def _quantise(x):
    x = x.float()
    amax = x.abs().amax(-1, keepdim=True)
    q = torch.where(amax > 0, torch.round(x * 127.0 / amax), 0.0)
    return q, amax / 127.0


def _plain_linear(s):
    q, sx = _quantise(s["x"])
    y = (q @ s["wq"].float().t()) * sx * s["ws"]
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["x"].dtype)


def _plain_experts(s):
    c, x = s["case"], s["x"]
    T, H, inner, E, k = c["T"], c["H"], c["I"], c["E"], c["k"]
    pos, offsets = _sorted(s["ids"], E)
    counts = (offsets[1:] - offsets[:-1]).long()
    # every expert's rows start a new block; the number of blocks has a bound that the shapes give
    n_blocks = T * k // BLOCK + min(E, T * k)
    first = torch.cat((counts.new_zeros(1), ((counts + BLOCK - 1) // BLOCK).cumsum(0)))
    owner = torch.searchsorted(first[1:], torch.arange(n_blocks, device=x.device), right=True).clamp(max=E - 1)
    known = pos.reshape(-1) >= 0
    expert = torch.where(known, s["ids"].reshape(-1), 0)
    slot = first[expert] * BLOCK + pos.reshape(-1).long() - offsets.long()[expert]
    slot = torch.where(known, slot, n_blocks * BLOCK)           # entries without an expert: one row behind the last block
    q, sx = _quantise(x)
    xb = q.new_zeros(n_blocks * BLOCK + 1, H).index_copy_(0, slot, q.repeat_interleave(k, 0))[:-1]
    sb = q.new_zeros(n_blocks * BLOCK + 1, 1).index_copy_(0, slot, sx.repeat_interleave(k, 0))[:-1]
    gu = torch.bmm(xb.view(n_blocks, BLOCK, H), s["w13q"][owner].float().transpose(1, 2))
    gu = gu * sb.view(n_blocks, BLOCK, 1) * s["w13s"][owner].unsqueeze(1)
    h = gu[..., :inner] / (1 + torch.exp(-gu[..., :inner])) * gu[..., inner:]
    hq, hs = _quantise(h)
    o = torch.bmm(hq, s["w2q"][owner].float().transpose(1, 2)) * hs * s["w2s"][owner].unsqueeze(1)
    o = torch.cat((o.view(n_blocks * BLOCK, H), o.new_zeros(1, H)))[slot].view(T, k, H)
    return (o * torch.where(pos >= 0, s["w"], 0.0).unsqueeze(-1)).sum(1).to(x.dtype)


def _plain_order(s):
    x, E = s["x"], s["case"]["E"]
    T, k = s["ids"].shape
    pos, offsets = _sorted(s["ids"], E)
    flat = torch.where(pos >= 0, pos, T * k).long().reshape(-1)
    rows = x.new_zeros(T * k + 1, x.shape[1]).index_copy_(0, flat, x.repeat_interleave(k, 0))[:-1]
    picked = s["ys"].float()[pos.clamp(min=0).long()]
    y = (picked * torch.where(pos >= 0, s["w"], 0.0).unsqueeze(-1)).sum(1).to(x.dtype)
    return {"pos": pos, "offsets": offsets, "rows": rows, "y": y}


def _plain_back(s):
    pos, dy = s["pos"], s["dy"].float()
    T, k = pos.shape
    here = (pos >= 0).unsqueeze(-1)
    flat = torch.where(pos >= 0, pos, T * k).long().reshape(-1)
    at = pos.clamp(min=0).long()
    d_ys = dy.new_zeros(T * k + 1, dy.shape[1]).index_copy_(0, flat, (s["w"].unsqueeze(-1) * dy.unsqueeze(1)).view(T * k, -1))[:-1]
    d_w = torch.where(here, s["ys"].float()[at] * dy.unsqueeze(1), 0.0).sum(-1)
    dx = torch.where(here, s["d_rows"].float()[at], 0.0).sum(1)
    return {"d_ys": d_ys.to(s["ys"].dtype), "d_w": d_w, "dx": dx.to(s["dy"].dtype)}


def run(state):
    op = state["case"]["op"]
    if own:
        from my_int4 import _C

        if op == "linear":
            return _C.w8a8_linear(state["x"], state["wq"], state["ws"], state["bias"])
        if op == "experts":
            return _C.w8a8_expert_ffn(state["x"], state["ids"], state["w"], state["w13q"], state["w13s"], state["w2q"],
                                      state["w2s"])
        if op == "order":
            pos, offsets = _C.expert_sort(state["ids"], state["case"]["E"])
            rows = _C.expert_gather(state["x"], pos, offsets)
            y = _C.expert_combine(state["ys"], pos, state["w"])
            return {"pos": pos, "offsets": offsets, "rows": rows, "y": y}
        d_ys, d_w = _C.expert_combine_grad(state["dy"], state["ys"], state["pos"], state["offsets"], state["w"])
        dx = _C.expert_combine(state["d_rows"], state["pos"])
        return {"d_ys": d_ys, "d_w": d_w, "dx": dx}
    return {"linear": _plain_linear, "experts": _plain_experts, "order": _plain_order, "back": _plain_back}[op](state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    size = TYPES[case["type"]].itemsize
    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": M * K * size + N * K + 4 * N * (2 if case["bias"] else 1) + M * N * size, "flops": 2 * M * N * K}
    T, H, E, k = case["T"], case["H"], case["E"], case["k"]
    R = T * k * (1 - case["drop"])
    if case["op"] == "experts":
        inner = case["I"]
        reached = E * (1 - (1 - k / E) ** (T * (1 - case["drop"])))       # by a router without favourites
        return {"bytes": reached * (3 * inner * H + 4 * (2 * inner + H)) + 2 * T * H * size + T * k * 12, "flops": 6 * R * inner * H}
    rows = T * k * H * size
    if case["op"] == "order":       # x and ys read, rows and y written; ids, pos, offsets, weights
        return {"bytes": 2 * T * H * size + rows + R * H * size + T * k * 16 + 4 * (E + 1), "flops": 2 * R * H}
    # dy, ys, d_rows, pos and weights read; d_ys, d_w and dx written
    return {"bytes": 2 * T * H * size + rows + 2 * R * H * size + T * k * 12, "flops": 4 * R * H}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------

def _codes64(x):
    x = x.double()
    top = x.abs().max(dim=-1, keepdim=True).values
    return torch.where(top == 0, 0.0, (127 * x / top).round()), top / 127


def _entries(ids, E):
    """Flat entry numbers of each expert in order, from the definition: one list after another."""
    flat = ids.reshape(-1)
    return [torch.nonzero(flat == e).reshape(-1) for e in range(E)]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        q, sx = _codes64(s["x"])
        y = torch.empty(case["M"], case["N"], dtype=torch.float64, device="cuda")
        for n in range(0, case["N"], 8192):
            y[:, n:n + 8192] = (q @ s["wq"][n:n + 8192].double().T) * (sx * s["ws"][n:n + 8192].double())
        return y if s["bias"] is None else y + s["bias"].double()
    T, H, E, k = case["T"], case["H"], case["E"], case["k"]
    w = s["w"].double().reshape(-1)
    if case["op"] == "experts":
        q, sx = _codes64(s["x"])
        y = torch.zeros(T, H, dtype=torch.float64, device="cuda")
        for e, entry in enumerate(_entries(s["ids"], E)):
            if entry.numel():
                t = entry // k
                gu = (q[t] @ s["w13q"][e].double().T) * sx[t] * s["w13s"][e].double()
                g, u = gu.chunk(2, dim=-1)
                hq, hs = _codes64(g * torch.sigmoid(g) * u)
                y.index_add_(0, t, (hq @ s["w2q"][e].double().T) * hs * s["w2s"][e].double() * w[entry].unsqueeze(-1))
        return y
    lists = _entries(s["ids"], E)
    entry = torch.cat(lists)
    pos = torch.full((T * k,), -1, dtype=torch.int32, device="cuda")
    pos[entry] = torch.arange(entry.numel(), dtype=torch.int32, device="cuda")
    n = entry.numel()
    if case["op"] == "order":
        y = torch.zeros(T, H, dtype=torch.float64, device="cuda")
        rows = torch.zeros(T * k, H, dtype=torch.float64, device="cuda")
        rows[:n] = s["x"][entry // k].double()
        for j in range(k):
            mine = entry % k == j                                          # at most one row of each token
            at = torch.nonzero(mine).reshape(-1)
            y[entry[at] // k] += w[entry[at]].unsqueeze(-1) * s["ys"][at].double()
        sizes = torch.tensor([0] + [v.numel() for v in lists], device="cuda")
        return {"pos": pos.view(T, k), "offsets": sizes.cumsum(0).to(torch.int32), "rows": rows, "y": y}
    d_ys = torch.zeros(T * k, H, dtype=torch.float64, device="cuda")
    d_w = torch.zeros(T * k, dtype=torch.float64, device="cuda")
    dx = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    dy = s["dy"][entry // k].double()
    d_ys[:n] = w[entry].unsqueeze(-1) * dy
    d_w[entry] = (dy * s["ys"][:n].double()).sum(-1)
    dx.index_add_(0, entry // k, s["d_rows"][:n].double())
    return {"d_ys": d_ys, "d_w": d_w.view(T, k), "dx": dx}
