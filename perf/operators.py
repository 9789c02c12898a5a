"""Timing cases of the operators around a layer whose tokens go to several experts each, and of per-request adapters.

A case is one call of one operator on what the program already holds on the device.  The operators:

  "select"    the k best experts of every token from its gating logits, and their weights (TopKRouter.select)
  "scatter"   token rows copied into expert order, once per chosen expert (scatter_topk)
  "combine"   weighted sum of every token's k expert results (combine_topk)
  "adapters"  low-rank adapters, one per request, added to the output of a shared projection (Adapters.apply)

With `own` false each is computed in plain torch operations, with `own` true by the library.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def _select(name, T, E, k, dtype, score="softmax", bias=False, groups=1, top_groups=1, group_best=1, renormalise=True,
            scale=1.0, masked=0.0):
    return {"name": name, "op": "select", "tokens": T, "experts": E, "top_k": k, "dtype": dtype, "score": score, "bias": bias,
            "groups": groups, "top_groups": top_groups, "group_best": group_best, "renormalise": renormalise, "scale": scale,
            "masked": masked}


def _rows(name, op, T, E, k, D, dtype, residual=False, dropped=0.0):
    return {"name": name, "op": op, "tokens": T, "experts": E, "top_k": k, "d_model": D, "dtype": dtype,
            "residual": residual, "dropped": dropped}


def _adapters(name, T, n, rank, d_in, d_out, dtype, requests, without=0.0, ragged=False):
    return {"name": name, "op": "adapters", "tokens": T, "adapters": n, "rank": rank, "d_in": d_in, "d_out": d_out,
            "dtype": dtype, "requests": requests, "without": without, "ragged": ragged}


def listed():
    return [
        # one sequence generating: the router of one token, sigmoid scores with a balance bias, four of eight groups
        _select("select_decode", 1, 128, 8, "f32", "sigmoid", True, 8, 4, 2, True, 2.5),
        # a batch of 8 x 512 tokens, two of 64 experts, logits as a 16-bit gate leaves them
        _select("select_batch", 4096, 64, 2, "bf16"),
        # expert and token counts that fill nothing evenly, padding tokens and disabled experts masked out
        _select("select_ragged", 777, 60, 6, "f16", "softmax", False, 5, 3, 1, False, 1.0, 0.1),
        # the largest batches: 128 x 512 tokens over many experts in groups
        _select("select_large", 65536, 256, 8, "f32", "sigmoid", True, 8, 4, 2, True, 2.5),
        # eight sequences generating, rows of the layer's own type
        _rows("scatter_decode", "scatter", 8, 64, 8, 4096, "f32"),
        # a batch in 16 bits, padding tokens have no expert
        _rows("scatter_batch", "scatter", 4096, 128, 8, 4096, "bf16", dropped=0.05),
        # eight sequences generating
        _rows("combine_decode", "combine", 8, 64, 8, 4096, "bf16"),
        # the layer's batch in FP32, weights that do not sum to one and the token's own row for the rest
        _rows("combine_batch", "combine", 4096, 32, 4, 4096, "f32", residual=True, dropped=0.05),
        # 64 sequences generating, every one with an adapter of its own choice
        _adapters("adapters_decode", 64, 64, 16, 4096, 4096, "bf16", 64),
        # eight prompts of about 512 tokens, some without an adapter
        _adapters("adapters_prompts", 4096, 8, 16, 4096, 4096, "bf16", 8, without=0.1),
        # FP32 rows of a small layer, widths and prompt lengths that fill no tile, adapters of several ranks
        _adapters("adapters_odd", 777, 6, 24, 1000, 2724, "f32", 13, without=0.1, ragged=True),
        # the largest batch: long prompts, wide adapters, onto a wider projection
        _adapters("adapters_large", 16384, 16, 64, 4096, 10240, "f16", 32),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A row width: mostly a multiple of eight, sometimes any number."""
    d = _log_int(rng, lo, hi)
    return d if rng.random() < 0.25 else max(8, d // 8 * 8)


def draw(rng):
    op = rng.choice(["select", "scatter", "combine", "adapters", "adapters"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    T = _log_int(rng, 1, 65536 if op == "select" else 16384)
    if op == "select":
        groups = rng.choice([1, 1, 2, 4, 5, 8, 16])
        E = groups * max(2, _log_int(rng, 8, 256) // groups)
        top_groups = rng.randint(max(1, groups // 4), groups)
        k = rng.randint(1, min(8, top_groups * (E // groups)))
        return _select("", T, E, k, dtype, rng.choice(["softmax", "sigmoid"]), rng.random() < 0.5, groups, top_groups,
                       rng.choice([1, 2]), rng.random() < 0.7, rng.choice([1.0, 2.5]), rng.choice([0.0, 0.1]))
    if op != "adapters":
        k, D = rng.randint(1, 8), _width(rng, 64, 4096)
        while T * k * D * BYTES[dtype] > 268e6:
            T = max(1, T // 2)
        return _rows("", op, T, rng.choice([8, 32, 60, 128]), k, D, dtype, op == "combine" and rng.random() < 0.5,
                     rng.choice([0.0, 0.05]))
    n, rank = _log_int(rng, 1, 64), _log_int(rng, 4, 64)
    d_in, d_out = _width(rng, 64, 4096), _width(rng, 64, 10240)
    while T * (d_in + 2 * d_out) * BYTES[dtype] > 800e6 or (T * n * rank * (d_in + d_out) > 1.5e11 and T > 64):
        T = max(1, T // 2)
    return _adapters("", T, n, rank, d_in, d_out, dtype, rng.randint(1, min(T, 64)), rng.choice([0.0, 0.1]),
                     rng.random() < 0.3)


def _choices(case, g, dev):
    """Experts of every token, k different ones, -1 in the slots of tokens that have none; their weights; and the rows that
    expert order gives them: pos (slot of row j), offset (first row of every expert), row_of (row of a slot)."""
    T, E, k = case["tokens"], case["experts"], case["top_k"]
    gate = torch.rand(T, E, generator=g, device=dev).argsort(1)[:, :k].to(torch.int32)
    weight = torch.rand(T, k, generator=g, device=dev) / k
    gone = torch.rand(T, generator=g, device=dev) < case["dropped"]
    gate[gone] = -1
    weight[gone] = 0
    flat = gate.flatten().long()
    bucket = torch.where(flat < 0, E, flat)
    pos = bucket.sort(stable=True).indices
    count = torch.bincount(bucket, minlength=E + 1)[:E]
    offset = torch.zeros(E + 1, dtype=torch.int32, device=dev)
    offset[1:] = count.cumsum(0)
    row_of = torch.empty(T * k, dtype=torch.int32, device=dev)
    row_of[pos] = torch.arange(T * k, dtype=torch.int32, device=dev)
    row_of[flat < 0] = -1
    return gate, weight.contiguous(), pos.to(torch.int32), offset, row_of.view(T, k)


def _adapter_of_token(case, g, dev):
    """Requests of different lengths, each with an adapter or (-1) none."""
    T, R = case["tokens"], case["requests"]
    if R == T:
        request = torch.arange(T, device=dev)
    else:
        ends = (torch.rand(R - 1, generator=g, device=dev) * T).long().sort().values
        request = torch.searchsorted(ends, torch.arange(T, device=dev), right=True)
    adapter = (torch.rand(R, generator=g, device=dev) * case["adapters"]).to(torch.int32)
    adapter[torch.rand(R, generator=g, device=dev) < case["without"]] = -1
    return adapter[request].contiguous()


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    s = {"case": case}
    T = case["tokens"]
    if case["op"] == "select":
        E = case["experts"]
        logits = 1.5 * torch.randn(T, E, generator=g, device=dev)
        masked = torch.rand(E, generator=g, device=dev) < case["masked"]
        masked[torch.arange(E, device=dev) % max(1, E // case["groups"]) == 0] = False
        logits[:, masked] = -math.inf                                  # disabled experts
        if T > 1:
            logits[torch.rand(T, generator=g, device=dev) < case["masked"] / 2] = -math.inf   # padding tokens
        s["logits"] = logits.to(dtype)
        s["bias"] = 0.1 * torch.randn(E, generator=g, device=dev) if case["bias"] else None
        if own:
            from infmoe_b200 import TopKRouter
            s["router"] = TopKRouter(E, case["top_k"], score=case["score"], bias=s["bias"], groups=case["groups"],
                                     top_groups=case["top_groups"], group_best=case["group_best"],
                                     renormalise=case["renormalise"], scale=case["scale"])
    elif case["op"] in ("scatter", "combine"):
        D, k = case["d_model"], case["top_k"]
        s["gate"], s["weight"], s["pos"], s["offset"], s["row_of"] = _choices(case, g, dev)
        s["x"] = torch.randn(T, D, generator=g, device=dev).to(dtype)
        if case["op"] == "scatter":
            s["routed"] = torch.zeros(T * k, D, dtype=dtype, device=dev)   # rows of no expert stay as they are
        else:
            s["y"] = torch.randn(T * k, D, generator=g, device=dev).to(dtype)
    else:
        n, r, d_in, d_out = case["adapters"], case["rank"], case["d_in"], case["d_out"]
        s["a"] = (torch.randn(n, r, d_in, generator=g, device=dev) / math.sqrt(d_in)).to(dtype)
        s["b"] = (torch.randn(n, d_out, r, generator=g, device=dev) / math.sqrt(r)).to(dtype)
        s["scale"] = 0.25 + torch.rand(n, generator=g, device=dev)
        s["rank"] = (1 + torch.rand(n, generator=g, device=dev) * r).to(torch.int32).clamp(max=r) if case["ragged"] else None
        s["x"] = torch.randn(T, d_in, generator=g, device=dev).to(dtype)
        s["y"] = torch.randn(T, d_out, generator=g, device=dev).to(dtype)
        s["adapter_of_token"] = _adapter_of_token(case, g, dev)
        if own:
            from infmoe_b200 import Adapters
            s["adapters"] = Adapters(s["a"], s["b"], scale=s["scale"], rank=s["rank"])
            s["plan"] = s["adapters"].plan(s["adapter_of_token"])
    return s


def _plain_select(s):
    case, l = s["case"], s["logits"]
    T, E, k, G = case["tokens"], case["experts"], case["top_k"], case["groups"]
    ok = l > torch.finfo(l.dtype).min
    # the order of the choice scores is decided in 64 bits: neighbours lie closer than 32 bits tell apart
    wide = l.double().masked_fill(~ok, -math.inf)
    if case["score"] == "softmax":
        p = (wide - wide.amax(1, keepdim=True).clamp(min=-1e300)).exp()
        p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
    else:
        p = 1 / (1 + (-wide).exp())
    c = p + s["bias"].double() if s["bias"] is not None else p
    c = c.masked_fill(~ok, -math.inf)
    if G > 1:
        best = c.view(T, G, E // G).sort(2, descending=True).values
        score = best[:, :, 0]
        if case["group_best"] == 2:
            score = score + best[:, :, 1].masked_fill(best[:, :, 1] == -math.inf, 0)
        stay = score.sort(dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        keep = torch.zeros(T, G, dtype=torch.bool, device=l.device).scatter(1, stay, True)
        c = c.view(T, G, E // G).masked_fill(~keep[:, :, None], -math.inf).view(T, E)
    order = c.sort(dim=1, descending=True, stable=True)
    gate, found = order.indices[:, :k], order.values[:, :k] > -math.inf
    w = p.float().gather(1, gate).masked_fill(~found, 0)
    if case["renormalise"]:
        w = w / w.sum(1, keepdim=True).clamp(min=1e-30)
    return gate.masked_fill(~found, -1).to(torch.int32), w * case["scale"]


def _plain_scatter(s):
    k, n = s["case"]["top_k"], s["offset"][-1]
    live = torch.arange(s["pos"].numel(), device=s["pos"].device) < n
    slot = s["pos"].long()
    routed = torch.where(live[:, None], s["x"].float()[slot // k], s["routed"].float()).to(s["x"].dtype)
    row_of = torch.empty_like(s["pos"])
    row_of[slot] = torch.where(live, torch.arange(slot.numel(), device=slot.device), -1).to(torch.int32)
    return routed, row_of.view(-1, k)


def _plain_combine(s):
    row = s["row_of"].long()
    w = s["weight"].masked_fill(row < 0, 0)
    out = (s["y"].float()[row.clamp(min=0)] * w[:, :, None]).sum(1)
    if s["case"]["residual"]:
        out = out + (1 - w.sum(1, keepdim=True)) * s["x"].float()
    return out.to(s["y"].dtype)


def _plain_adapters(s):
    n, r, T = s["case"]["adapters"], s["case"]["rank"], s["case"]["tokens"]
    at = s["adapter_of_token"].long()
    # the products with all adapters at once; what is not a token's own is multiplied by zero in between
    v = (s["x"].float() @ s["a"].float().view(n * r, -1).T).view(T, n, r)
    mine = at[:, None] == torch.arange(n, device=at.device)
    v = v * (mine * s["scale"])[:, :, None]
    if s["rank"] is not None:
        v = v * (torch.arange(r, device=at.device) < s["rank"][:, None])
    return (s["y"].float() + v.view(T, n * r) @ s["b"].float().transpose(1, 2).reshape(n * r, -1)).to(s["y"].dtype)


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"select": _plain_select, "scatter": _plain_scatter, "combine": _plain_combine,
                "adapters": _plain_adapters}[op](s)
    import infmoe_b200 as m
    if op == "select":
        return s["router"].select(s["logits"])
    if op == "scatter":
        return m.scatter_topk(s["x"], s["pos"], s["offset"], s["case"]["top_k"], out=s["routed"])
    if op == "combine":
        return m.combine_topk(s["y"], s["weight"], row_of=s["row_of"], residual=s["x"] if s["case"]["residual"] else None)
    return s["adapters"].apply(s["x"], s["y"], s["plan"])


def work(case):
    T, size = case["tokens"], BYTES[case["dtype"]]
    if case["op"] == "select":
        E, k = case["experts"], case["top_k"]
        return {"bytes": T * E * size + (4 * E if case["bias"] else 0) + 8 * T * k, "flops": 10 * T * E}
    if case["op"] != "adapters":
        k, D = case["top_k"], case["d_model"]
        live = T * k * (1 - case["dropped"])
        if case["op"] == "scatter":
            return {"bytes": T * (1 - case["dropped"]) * D * size + live * D * size + 8 * T * k, "flops": 0}
        return {"bytes": (live + T + (T if case["residual"] else 0)) * D * size + 8 * T * k, "flops": 2 * live * D}
    n, r, d_in, d_out = case["adapters"], case["rank"], case["d_in"], case["d_out"]
    R, share = case["requests"], 1 - case["without"]
    used = n * (1 - (1 - 1 / n) ** (R * share)) * (0.5 if case["ragged"] else 1)   # adapters that some request asks for
    return {"bytes": (T * share * d_in + 2 * T * d_out + used * r * (d_in + d_out)) * size + 4 * T,
            "flops": 2 * T * share * r * (d_in + d_out) * (0.5 if case["ragged"] else 1)}


def _exact_select(s):
    case = s["case"]
    T, E, k, G = case["tokens"], case["experts"], case["top_k"], case["groups"]
    l = s["logits"].to(torch.float64)
    out = l <= torch.finfo(s["logits"].dtype).min
    if case["score"] == "softmax":
        score = torch.exp(l - torch.logsumexp(l.masked_fill(out, -math.inf), 1, keepdim=True))
    else:
        score = torch.exp(-torch.logaddexp(torch.zeros_like(l), -l))
    score = torch.where(out, 0.0, score)
    choice = score.clone()
    if s["bias"] is not None:
        choice += s["bias"].to(torch.float64)
    choice[out] = -math.inf
    size = E // G
    if G > 1:
        parts = choice.reshape(T, G, size)
        top = parts.amax(2)
        if case["group_best"] == 2 and size > 1:
            second = parts.scatter(2, parts.argmax(2, keepdim=True), -math.inf).amax(2)
            top = torch.where(second == -math.inf, top, top + second)
        gone = torch.ones(T, G, dtype=torch.bool, device=l.device)
        for _ in range(case["top_groups"]):
            at = top.argmax(1, keepdim=True)
            gone.scatter_(1, at, False)
            top.scatter_(1, at, -math.inf)
        choice[gone.repeat_interleave(size, 1)] = -math.inf
    gates, weights = [], []
    for _ in range(k):
        value, at = choice.max(1, keepdim=True)
        none = value == -math.inf
        at = torch.where(choice == value, torch.arange(E, device=l.device), E).amin(1, keepdim=True)   # the lowest index
        choice.scatter_(1, at.clamp(max=E - 1), -math.inf)
        gates.append(torch.where(none, -1, at))
        weights.append(torch.where(none, 0.0, score.gather(1, at)))
    weight = torch.cat(weights, 1)
    if case["renormalise"]:
        total = weight.sum(1, keepdim=True)
        weight = torch.where(total > 0, weight / total, 0.0)
    return torch.cat(gates, 1).to(torch.int32), weight * case["scale"]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "select":
        return _exact_select(s)
    if case["op"] == "scatter":
        k, n = case["top_k"], int(s["offset"][-1])
        routed = s["routed"].double()
        row_of = torch.full((case["tokens"] * k,), -1, dtype=torch.int32, device=routed.device)
        for e in range(case["experts"]):
            for_e = (s["gate"].flatten() == e).nonzero().flatten()
            at = int(s["offset"][e])
            routed[at:at + len(for_e)] = s["x"][for_e // k].double()
            row_of[for_e] = torch.arange(at, at + len(for_e), dtype=torch.int32, device=routed.device)
        assert int((row_of >= 0).sum()) == n
        return routed, row_of.view(-1, k)
    if case["op"] == "combine":
        k = case["top_k"]
        out = torch.zeros_like(s["x"], dtype=torch.float64)
        rest = torch.ones(case["tokens"], 1, dtype=torch.float64, device=out.device)
        for i in range(k):
            row = s["row_of"][:, i].long()
            w = torch.where(row < 0, 0.0, s["weight"][:, i].double())[:, None]
            out += w * s["y"][row.clamp(min=0)].double()
            rest -= w
        return out + rest * s["x"].double() if case["residual"] else out
    out = s["y"].double()
    for a in range(case["adapters"]):
        rows = (s["adapter_of_token"] == a).nonzero().flatten()
        r = int(s["rank"][a]) if s["rank"] is not None else case["rank"]
        inner = s["x"][rows].double() @ s["a"][a, :r].double().T
        out[rows] += s["scale"][a].double() * (inner @ s["b"][a, :, :r].double().T)
    return out
