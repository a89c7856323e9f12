"""The operators between and around an MoE layer's GEMMs in training, as cases that can be timed and compared.

One case = one pass through one operator.  With `own` false it is computed from elementary torch operations in 32 bits
(64 where differences of weights cancel), with `own` true by the calls of `justgoal_b200`.  A case is a dict:

  op      sort             expert-sorted tables from the tokens' expert ids
          permute          part "forward": token rows into expert order; "backward": their gradient;
                           "restore": token rows kept in 8 bits, read back into expert order
          combine          part "forward": weighted sum of a token's expert rows; "backward": gradients of rows and weights
          swiglu           part "save": activation and the 8-bit copy of its inputs; "backward": gradients from that copy
          route            gradient of the routing weights down to the logits
  tokens, hidden, experts (global), local (held here), rank (whose share), top_k, type of the rows
  rows, inner   swiglu: rows that hold something, of `room` rows, and columns of the activation
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MODES = {"deepseek": 0, "renorm_naive": 1, "default": 2, "renormalize": 3, "llama4": 4, "topk": 5}
ALIGN = 16           # rows that an expert's segment is padded to
FACTOR = 2.5         # routed scaling factor
LARGEST = 8192 * 8 * 7168      # row elements of the largest listed case


def _moe(name, op, part, tokens, hidden, experts, local, rank=0, top_k=8, type="bf16"):
    return {"name": name, "op": op, "part": part, "tokens": tokens, "hidden": hidden, "experts": experts, "local": local,
            "rank": rank, "top_k": top_k, "type": type}


def _swiglu(name, part, rows, room, inner, type="bf16"):
    return {"name": name, "op": "swiglu", "part": part, "rows": rows, "room": room, "inner": inner, "type": type}


def _route(name, mode, tokens, experts, top_k):
    return {"name": name, "op": "route", "mode": mode, "tokens": tokens, "experts": experts, "top_k": top_k}


def listed():
    return [
        # a few tokens of a decode step, one rank's share of the experts: latency alone
        _moe("sort_7", "sort", "", 7, 0, 256, 32, rank=3),
        # several long prompts in one ragged batch, every expert on this GPU
        _moe("sort_14107", "sort", "", 14107, 0, 256, 256),
        # a training batch into expert order, the whole layer on one GPU
        _moe("permute_8192", "permute", "forward", 8192, 7168, 256, 256),
        # the gradient of a ragged micro-batch on one rank of eight, half precision
        _moe("permute_grad_901", "permute", "backward", 901, 4096, 128, 16, rank=5, type="fp16"),
        # the backward pass rebuilds GEMM1's input rows from the 8-bit copy of the tokens
        _moe("restore_4096", "permute", "restore", 4096, 7168, 256, 256),
        # rows back to their tokens, kept in fp32, on one rank's share
        _moe("combine_2048", "combine", "forward", 2048, 4096, 128, 64, rank=1, type="fp32"),
        # the gradient of the combine: rows and routing weights, the whole layer on one GPU
        _moe("combine_grad_4096", "combine", "backward", 4096, 7168, 256, 256),
        # activation of one rank's rows, a buffer sized for more than came
        _swiglu("swiglu_save_32768", "save", 32768 + 1877, 40000, 2048),
        # the same rows in the backward pass
        _swiglu("swiglu_grad_32768", "backward", 32768 + 1877, 40000, 2048),
        # a handful of rows of a small expert
        _swiglu("swiglu_save_77", "save", 77, 77, 256, type="fp16"),
        # the router of a training batch
        _route("route_grad_8192", "deepseek", 8192, 256, 8),
        # a softmax router, odd batch
        _route("route_grad_261", "default", 261, 128, 8),
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["sort", "permute", "permute", "combine", "combine", "swiglu", "swiglu", "route"])
    if op == "route":
        # (uniform weights have no gradient, and one pick that is normalised by itself has none either)
        mode = rng.choice(["deepseek", "deepseek", "renorm_naive", "default", "renormalize", "llama4"])
        return {"op": op, "mode": mode, "tokens": _spread(rng, 1, 8192), "experts": 32 * rng.randint(1, 8),
                "top_k": 1 if mode == "llama4" else rng.randint(2, 8)}
    kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "swiglu":
        inner = 128 * _spread(rng, 1, 16)
        most = 40000 * 2048 // inner // (2 if kind == "fp32" else 1)
        room = _spread(rng, 1, min(most, 40000))
        rows = room if rng.random() < 0.4 else rng.randint(1, room)
        return {"op": op, "part": rng.choice(["save", "backward"]), "rows": rows, "room": room, "inner": inner, "type": kind}
    experts, top_k = 32 * rng.randint(1, 8), rng.randint(1, 8)
    part, hidden, tokens = "", 0, _spread(rng, 1, 14107)
    if op != "sort":
        part = rng.choice(["forward", "backward", "restore"] if op == "permute" else ["forward", "backward"])
        hidden = 128 * _spread(rng, 1, 56)
        tokens = _spread(rng, 1, min(8192, LARGEST // 2 // (2 if kind == "fp32" else 1) // (8 * hidden)))
    # a rank's share only of batches that leave it some pairs
    local = experts // rng.choice([1, 1, 2, 4, 8] if tokens * top_k >= 256 else [1])
    return {"op": op, "part": part, "tokens": tokens, "hidden": hidden, "experts": experts, "local": local,
            "rank": rng.randrange(experts // local), "top_k": top_k, "type": kind}


# ------------------------------------------------------------------ inputs

def _gen(seed, k):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 64 + k) % (1 << 62))
    return g


def _randn(seed, k, *shape):
    return torch.randn(*shape, generator=_gen(seed, k), device="cuda")


def _room(case):
    return case["tokens"] * case["top_k"] + (ALIGN - 1) * case["local"]


def _picks(case, seed):
    """Expert ids of a router with liked and disliked experts, and normalised weights."""
    logits = _randn(seed, 1, case["tokens"], case["experts"]) + 0.4 * _randn(seed, 2, case["experts"])
    top = torch.sigmoid(logits).topk(case["top_k"], dim=1)
    return top.indices.to(torch.int32), (top.values / top.values.sum(dim=1, keepdim=True) * FACTOR)


def _tables(idx, offset, local, room):
    """Expert-sorted tables by a stable sort: (first row of each expert, pair of each row, row of each pair), -1 for none."""
    flat = idx.long().flatten() - offset
    key = torch.where((flat >= 0) & (flat < local), flat, local)
    count = (key[:, None] == torch.arange(local + 1, device=idx.device)).sum(dim=0)
    padded = (count + ALIGN - 1) // ALIGN * ALIGN
    row0 = padded.cumsum(0) - padded
    order = key.argsort(stable=True)
    k = key[order]
    rank = torch.arange(k.numel(), device=idx.device) - (count.cumsum(0) - count)[k]
    rows = torch.where(k < local, row0[k] + rank, room)
    row_pair = torch.full((room + 1,), -1, dtype=torch.int32, device=idx.device)
    row_pair[rows] = order.to(torch.int32)
    pair_row = torch.empty_like(rows)
    pair_row[order] = torch.where(k < local, rows, -1)
    row_pair = torch.where(torch.arange(room, device=idx.device) < row0[local], row_pair[:room], -1)
    return row0.to(torch.int32), row_pair, pair_row.to(torch.int32).view(idx.shape)


def _activations(seed, k, rows, cols, kind):
    """Values of a hidden state: a few channels are much larger than the others."""
    x = _randn(seed, k, rows, cols)
    x *= torch.exp(0.5 * _randn(seed, k + 20, cols))
    return x.to(TYPES[kind])


def _eight_bits(x):
    """e4m3 codes and scales [groups, rows] of 1x128 groups, scale = largest magnitude / 448."""
    g = x.float().view(x.shape[0], -1, 128)
    amax = g.abs().amax(dim=2)
    scale = torch.where(amax > 0, amax / 448.0, torch.ones_like(amax))
    return (g / scale[:, :, None]).view(x.shape).to(torch.float8_e4m3fn), scale.t().contiguous()


def _eight_bits_exponent(x):
    """The same with the smallest power of two not below largest magnitude / 448 as the scale."""
    g = x.float().view(x.shape[0], -1, 128)
    amax = g.abs().amax(dim=2)
    mantissa, exponent = torch.frexp(amax)                # amax = mantissa * 2^exponent, mantissa in [0.5, 1); 448 = 0.875 * 2^9
    exponent = (exponent - 9 + (mantissa > 0.875).to(exponent.dtype)).clamp(min=-126)
    scale = torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), exponent), torch.ones_like(amax))
    return (g / scale[:, :, None]).view(x.shape).to(torch.float8_e4m3fn), scale.t().contiguous()


def prepare(case, seed):
    op = case["op"]
    if op == "route":
        mode, T, E, K = case["mode"], case["tokens"], case["experts"], case["top_k"]
        logits = _randn(seed, 1, T, E)
        bias = None if seed % 2 else (0.1 * _randn(seed, 2, E)).to(torch.bfloat16)
        by = torch.sigmoid(logits) if mode == "deepseek" else logits
        idx = (by if bias is None else by + bias.float()).topk(K, dim=1).indices.to(torch.int32)
        return {"case": case, "logits": logits, "bias": bias, "idx": idx, "grad_w": 1e-2 * _randn(seed, 3, T, K)}
    if op == "swiglu":
        n, room, inner, kind = case["rows"], case["room"], case["inner"], case["type"]
        x = torch.zeros(room, 2 * inner, dtype=TYPES[kind], device="cuda")
        x[:n] = _activations(seed, 1, n, 2 * inner, kind)
        state = {"case": case, "row0": torch.tensor([0, n // 3, n], dtype=torch.int32, device="cuda"),
                 "act": torch.zeros(room, inner, dtype=TYPES[kind], device="cuda")}
        if case["part"] == "save":
            state |= {"x": x, "q": torch.zeros(room, 2 * inner, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn),
                      "scale": torch.zeros(2 * inner // 128, room, device="cuda")}
        else:
            q, scale = _eight_bits_exponent(x)
            state |= {"q": q, "scale": scale, "grad": (1e-2 * _randn(seed, 3, room, inner)).to(TYPES[kind]),
                      "grad_x": torch.zeros(room, 2 * inner, dtype=TYPES[kind], device="cuda")}
        return state
    T, H, kind = case["tokens"], case["hidden"], case["type"]
    idx, w = _picks(case, seed)
    offset, room = case["rank"] * case["local"], _room(case)
    if op == "sort":
        return {"case": case, "idx": idx, "offset": offset}
    row0, row_pair, pair_row = _tables(idx, offset, case["local"], room)
    state = {"case": case, "row0": row0, "row_pair": row_pair, "pair_row": pair_row, "w": w}
    if op == "permute" and case["part"] == "forward":
        return {**state, "x": _activations(seed, 4, T, H, kind), "rows": torch.zeros(room, H, dtype=TYPES[kind], device="cuda")}
    if op == "permute" and case["part"] == "restore":
        q, scale = _eight_bits(_activations(seed, 4, T, H, "bf16"))
        return {**state, "q": q, "scale": scale, "rows": torch.zeros(room, H, dtype=TYPES[kind], device="cuda")}
    rows = torch.zeros(room, H, dtype=TYPES[kind], device="cuda")
    live = (row_pair >= 0).nonzero().flatten()
    rows[live] = _activations(seed, 5, live.numel(), H, kind)
    if op == "combine" and case["part"] == "backward":
        state |= {"grad": (1e-2 * _randn(seed, 6, T, H)).to(TYPES[kind]), "grad_rows": torch.zeros(room, H, dtype=TYPES[kind], device="cuda")}
    return {**state, "rows": rows}


# ------------------------------------------------------------------ one pass

def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    return {"sort": _sort, "permute": _permute, "combine": _combine, "swiglu": _swiglu_pass, "route": _route_pass}[case["op"]](case, state)


def _sort(case, s):
    row0, row_pair, pair_row = _tables(s["idx"], s["offset"], case["local"], _room(case))
    return {"row0": row0, "row_pair": row_pair, "pair_row": pair_row}


def _into_rows(s, x, kind):
    pair = s["row_pair"].long()
    token = pair.clamp(min=0) // s["pair_row"].shape[1]
    return torch.where((pair >= 0)[:, None], x[token], 0.0).to(kind)


def _of_tokens(s, rows):
    """Rows of every (token, pick), zeros where the pick has none: [tokens, picks, columns] in 32 bits."""
    at = s["pair_row"].long()
    return torch.where((at >= 0)[:, :, None], rows[at.clamp(min=0)].float(), 0.0)


def _permute(case, s):
    kind = TYPES[case["type"]]
    if case["part"] == "forward":
        return {"rows": _into_rows(s, s["x"].float(), kind)}
    if case["part"] == "restore":
        T, H = s["q"].shape
        x = s["q"].float().view(T, H // 128, 128) * s["scale"].t()[:, :, None]
        return {"rows": _into_rows(s, x.view(T, H), kind)}
    return {"grad_x": _of_tokens(s, s["rows"]).sum(dim=1).to(kind)}


def _combine(case, s):
    kind = TYPES[case["type"]]
    if case["part"] == "forward":
        return {"out": (_of_tokens(s, s["rows"]) * s["w"][:, :, None]).sum(dim=1).to(kind)}
    grad = s["grad"].float()
    grad_w = (_of_tokens(s, s["rows"]) * grad[:, None, :]).sum(dim=2)
    pair = s["row_pair"].long()
    weight = torch.where(pair >= 0, s["w"].flatten()[pair.clamp(min=0)], 0.0)
    grad_rows = grad[pair.clamp(min=0) // s["w"].shape[1]] * weight[:, None]
    return {"grad_rows": grad_rows.to(kind), "grad_w": grad_w}


def _swiglu_pass(case, s):
    kind, inner = TYPES[case["type"]], case["inner"]
    live = (torch.arange(case["room"], device="cuda") < s["row0"][-1])[:, None]
    if case["part"] == "save":
        x = s["x"].float()
        up, gate = x[:, :inner], x[:, inner:]
        act = up * (gate / (1.0 + torch.exp(-gate)))
        q, scale = _eight_bits_exponent(s["x"])
        return {"act": torch.where(live, act, 0.0).to(kind), "q": q, "scale": torch.where(live.t(), scale, 0.0)}
    rows = case["room"]
    x = (s["q"].float().view(rows, -1, 128) * s["scale"].t()[:, :, None]).view(rows, 2 * inner)
    up, gate, grad = x[:, :inner], x[:, inner:], s["grad"].float()
    sig = 1.0 / (1.0 + torch.exp(-gate))
    grad_x = torch.cat([grad * gate * sig, grad * up * sig * (1.0 + gate * (1.0 - sig))], dim=1)
    return {"grad_x": torch.where(live, grad_x, 0.0).to(kind), "act": torch.where(live, up * gate * sig, 0.0).to(kind)}


def _route_pass(case, s):
    mode, at = case["mode"], s["idx"].long()
    logits, grad = s["logits"].double(), s["grad_w"].double()
    if s["bias"] is not None and mode != "deepseek":
        logits = logits + s["bias"].double()
    picked = logits.gather(1, at)
    if mode == "deepseek":
        sig = 1.0 / (1.0 + torch.exp(-picked))
        total = sig.sum(dim=1, keepdim=True) + 1e-20
        g = FACTOR * (grad - (grad * sig).sum(dim=1, keepdim=True) / total) / total * sig * (1.0 - sig)
    elif mode in ("renorm_naive", "renormalize"):
        p = torch.exp(picked - picked.amax(dim=1, keepdim=True))
        p = p / p.sum(dim=1, keepdim=True)
        g = FACTOR * p * (grad - (p * grad).sum(dim=1, keepdim=True))
    elif mode == "default":
        p = torch.exp(logits - logits.amax(dim=1, keepdim=True))
        p = p / p.sum(dim=1, keepdim=True)
        d = torch.zeros_like(p).scatter(1, at, grad)
        return {"grad_logits": (FACTOR * p * (d - (p * d).sum(dim=1, keepdim=True))).float()}
    elif mode == "llama4":
        sig = 1.0 / (1.0 + torch.exp(-picked))
        g = FACTOR * grad * sig * (1.0 - sig)
    else:
        g = torch.zeros_like(grad)
    return {"grad_logits": torch.zeros_like(logits).scatter(1, at, g).float()}


def _run_own(case, s):
    import justgoal_b200 as jg
    op, part = case["op"], case.get("part")
    if op == "route":
        return {"grad_logits": jg.route_backward(s["logits"], s["bias"], s["idx"], s["grad_w"], FACTOR, MODES[case["mode"]])}
    if op == "swiglu":
        if part == "save":
            act, q, scale = jg.swiglu_save(s["x"], s["row0"], out=(s["act"], s["q"], s["scale"]))
            return {"act": act, "q": q, "scale": scale}
        grad_x, act = jg.swiglu_backward(s["q"], s["scale"], s["grad"], s["row0"], out=(s["grad_x"], s["act"]))
        return {"grad_x": grad_x, "act": act}
    if op == "sort":
        order = jg.sort_tokens(s["idx"], case["local"], s["offset"])
        return {"row0": order.expert_row0, "row_pair": order.row_pair, "pair_row": order.pair_row}
    order = jg.TokenOrder(s["row0"], s["row_pair"], s["pair_row"])
    if op == "permute" and part == "forward":
        return {"rows": jg.permute(s["x"], order, out=s["rows"])}
    if op == "permute" and part == "restore":
        return {"rows": jg.restore_1x128(s["q"], s["scale"], order, out=s["rows"])}
    if op == "permute":
        return {"grad_x": jg.permute_backward(s["rows"], order)}
    if part == "forward":
        return {"out": jg.combine(s["rows"], s["w"], order)}
    grad_rows, grad_w = jg.combine_backward(s["grad"], s["rows"], s["w"], order, out=s["grad_rows"])
    return {"grad_rows": grad_rows, "grad_w": grad_w}


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    op, part = case["op"], case.get("part")
    if op == "route":
        T, E, K = case["tokens"], case["experts"], case["top_k"]
        reads = 4 * T * E if case["mode"] == "default" else 0 if case["mode"] == "topk" else 4 * T * K
        return {"bytes": reads + 8 * T * K + 4 * T * E, "flops": 20 * T * K + (10 * T * E if case["mode"] == "default" else 0)}
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["type"]]
    if op == "swiglu":
        n, inner = case["rows"], case["inner"]
        copy = 2 * inner + 4 * 2 * inner // 128
        if part == "save":
            return {"bytes": n * (3 * inner * size + copy) + 4, "flops": 12 * n * inner}
        return {"bytes": n * (4 * inner * size + copy) + 4, "flops": 18 * n * inner}
    T, H, K, E, local = case["tokens"], case["hidden"], case["top_k"], case["experts"], case["local"]
    if op == "sort":
        return {"bytes": 8 * T * K + 4 * _room(case) + 4 * (local + 1), "flops": 4 * T * K}
    pairs = T * K * local / E                              # expected, with even experts
    each = T * K / E
    padded = local * (each + ((ALIGN - 1) / 2 if each >= 1 else each * (ALIGN - 1)))
    table = 4 * T * K
    if op == "permute" and part == "restore":
        return {"bytes": T * (H + 4 * H // 128) + padded * H * size + table, "flops": pairs * H}
    if op == "permute" and part == "forward":
        return {"bytes": T * H * size + padded * H * size + table, "flops": 0}
    if op == "permute":
        return {"bytes": pairs * H * size + T * H * size + table, "flops": pairs * H}
    if part == "forward":
        return {"bytes": pairs * H * size + T * H * size + 2 * table, "flops": 2 * pairs * H}
    return {"bytes": pairs * H * size + padded * H * size + T * H * size + 3 * table, "flops": 3 * pairs * H}


# ------------------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    op, part = case["op"], case.get("part")
    if op == "sort":
        return None
    if op == "route":
        return {"grad_logits": _exact_route(case, s)}
    if op == "swiglu":
        return _exact_swiglu(case, s)
    T, K = s["pair_row"].shape
    live = (s["row_pair"] >= 0).nonzero().flatten()
    pair = s["row_pair"][live].long()
    token = torch.div(pair, K, rounding_mode="floor")
    H = case["hidden"]
    if op == "permute" and part in ("forward", "restore"):
        rows = torch.zeros(s["row_pair"].numel(), H, dtype=torch.float64, device="cuda")
        if part == "forward":
            rows.index_copy_(0, live, s["x"].double().index_select(0, token))
        else:
            x = s["q"].double() * s["scale"].t().double().repeat_interleave(128, dim=1)
            rows.index_copy_(0, live, x.index_select(0, token))
        return {"rows": rows}
    if part == "forward" or op == "permute":
        y = s["rows"].double().index_select(0, live)
        if op == "combine":
            y *= s["w"].double().view(-1).index_select(0, pair).unsqueeze(1)
        out = torch.zeros(T, H, dtype=torch.float64, device="cuda").index_add_(0, token, y)
        return {"out" if op == "combine" else "grad_x": out}
    grad_rows = torch.zeros(s["rows"].shape, dtype=torch.float64, device="cuda")
    grad_w = torch.zeros(T * K, dtype=torch.float64, device="cuda")
    for a in range(0, live.numel(), 8192):
        r, p, t = live[a:a + 8192], pair[a:a + 8192], token[a:a + 8192]
        d = s["grad"].index_select(0, t).double()
        grad_w.index_copy_(0, p, torch.einsum("rh,rh->r", d, s["rows"].index_select(0, r).double()))
        grad_rows.index_copy_(0, r, torch.einsum("rh,r->rh", d, s["w"].view(-1).index_select(0, p).double()))
    return {"grad_rows": grad_rows, "grad_w": grad_w.view(T, K)}


def _exact_swiglu(case, s):
    n, inner, room = case["rows"], case["inner"], case["room"]
    act = torch.zeros(room, inner, dtype=torch.float64, device="cuda")
    if case["part"] == "save":
        x = s["x"][:n].double()
        act[:n] = x[:, :inner] * x[:, inner:] * torch.sigmoid(x[:, inner:])
        group = x.view(n, 2 * inner // 128, 128)
        most = group.abs().amax(dim=2)
        two = torch.exp2(torch.ceil(torch.log2((most / 448.0).clamp(min=2.0 ** -126))))
        two = torch.where((two > 2.0 ** -126) & (224.0 * two >= most), two / 2, two)       # (the quotient and its logarithm are rounded)
        two = torch.where(448.0 * two < most, two * 2, two)
        two = torch.where(most > 0, two, 1.0)
        scale = torch.zeros(2 * inner // 128, room, dtype=torch.float64, device="cuda")
        scale[:, :n] = two.t()
        q = torch.zeros(room, 2 * inner, dtype=torch.float64, device="cuda")
        q[:n] = (group / two[:, :, None]).reshape(n, 2 * inner)
        return {"act": act, "q": q, "scale": scale}
    x = s["q"][:n].double() * s["scale"][:, :n].t().double().repeat_interleave(128, dim=1)
    up, gate, grad = x[:, :inner], x[:, inner:], s["grad"][:n].double()
    grad_x = torch.zeros(room, 2 * inner, dtype=torch.float64, device="cuda")
    sig = torch.sigmoid(gate)
    grad_x[:n, :inner] = grad * gate * sig
    grad_x[:n, inner:] = grad * up * (sig + gate * sig * torch.sigmoid(-gate))
    act[:n] = up * gate * sig
    return {"grad_x": grad_x, "act": act}


def _exact_route(case, s):
    """Reverse mode over the forward's definition in 64 bits."""
    mode, at = case["mode"], s["idx"].long()
    logits = s["logits"].double().requires_grad_(True)
    x = logits if s["bias"] is None or mode == "deepseek" else logits + s["bias"].double()
    if mode == "deepseek":
        p = torch.sigmoid(x).gather(1, at)
        w = p / (p.sum(dim=1, keepdim=True) + 1e-20)
    elif mode in ("renorm_naive", "renormalize"):
        w = torch.softmax(x.gather(1, at), dim=1)
    elif mode == "default":
        w = torch.softmax(x, dim=1).gather(1, at)
    elif mode == "llama4":
        w = torch.sigmoid(x.gather(1, at))
    else:
        return torch.zeros_like(s["logits"], dtype=torch.float64)
    (w * FACTOR * s["grad_w"].double()).sum().backward()
    return logits.grad
