"""Operators around the ternary projections and the MoE layer of a model that serves many requests at once: routing to
experts in groups, the plan that sorts a batch's rows by the adapter of their request, low-rank adapters beside a shared
projection, and low-rank adapters of the routed experts.

`run` computes them by elementary torch operations, or through the framework where `own` is true. Activations and
projection outputs are ~ N(0, 1); an adapter's A keeps that variance, its B gives about a third of it, as trained
adapters do. One request in eight has no adapter.
"""

import torch

own = False
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------------------------------------- the cases
def route(name, tokens, experts, groups, kept, top_k, score, group_score, bias, dtype, renorm=True):
    return {"name": name, "kind": "route", "tokens": tokens, "experts": experts, "groups": groups, "kept": kept, "top_k": top_k,
            "score": score, "group_score": group_score, "bias": bias, "dtype": dtype, "renorm": renorm}


def plan(name, rows, requests, adapters):
    return {"name": name, "kind": "plan", "rows": rows, "requests": requests, "adapters": adapters}


def linear(name, rows, requests, adapters, rank, K, N, dtype="bf16", base="f32", out="bf16"):
    return {"name": name, "kind": "linear", "rows": rows, "requests": requests, "adapters": adapters, "rank": rank, "K": K, "N": N,
            "dtype": dtype, "base": base, "out": out}


def experts(name, tokens, requests, adapters, rank, experts, top_k, K, N, parts):
    return {"name": name, "kind": "experts", "tokens": tokens, "requests": requests, "adapters": adapters, "rank": rank,
            "experts": experts, "top_k": top_k, "K": K, "N": N, "parts": parts}


def listed():
    return [
        # one decoding sequence through the router of a large MoE layer
        route("route_1tok", 1, 256, 8, 4, 8, "sigmoid", "top2", True, "f32"),
        # a ragged prompt, a gate that writes bf16 logits, groups by their best expert
        route("route_777tok_bf16", 777, 384, 8, 3, 6, "softmax", "max", False, "bf16"),
        # the benchmark's own step
        route("route_16384tok", 16384, 384, 8, 4, 6, "sqrtsoftplus", "top2", True, "f32"),
        # a decode batch: one row per request
        plan("plan_64rows", 64, 64, 32),
        # a mixed batch: long and short prompts beside decoding requests
        plan("plan_16384rows", 16384, 96, 64),
        # one decoding sequence beside one dense projection: the smallest call
        linear("linear_1row", 1, 1, 8, 16, 4096, 4096),
        # a decode batch of as many requests, most with an adapter of their own, a wide projection
        linear("linear_64rows", 64, 64, 48, 32, 4096, 11008),
        # a short ragged prompt batch in fp16, added to a projection's fp16 rows
        linear("linear_333rows_f16", 333, 5, 4, 8, 4096, 4096, dtype="f16", base="f16", out="f16"),
        # prompts of a few requests, larger adapters, float32 rows kept
        linear("linear_4000rows_r64", 4000, 9, 16, 64, 2048, 4096, out="f32"),
        # the benchmark's token count through one projection
        linear("linear_16384rows", 16384, 24, 16, 16, 4096, 4096),
        # a small decode batch: the gate and up matrices of the experts, mostly one row per expert and adapter
        experts("experts_8tok", 8, 8, 2, 16, 384, 6, 4096, 4096, 2),
        # prefill through a smaller MoE layer's down projection, the rows of each expert from four adapters
        experts("experts_2048tok", 2048, 6, 4, 16, 64, 8, 1024, 2048, 1),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["route"] * 2 + ["plan"] + ["linear"] * 4 + ["experts"] * 2)
    if kind == "route":
        groups = rng.choice([2, 4, 8, 16])
        size = rng.randint(8, 48)
        kept, top_k = rng.randint(1, groups), rng.randint(1, 8)
        return {"kind": "route", "tokens": _log(rng, 1, 16384 * 384 // (groups * max(size, 24))), "experts": groups * size, "groups": groups,
                "kept": kept, "top_k": top_k, "score": rng.choice(["softmax", "sigmoid", "sqrtsoftplus"]), "group_score": rng.choice(["max", "top2"]),
                "bias": rng.random() < 0.5, "dtype": rng.choice(["f32", "f32", "bf16", "f16"]), "renorm": rng.random() < 0.8}
    if kind == "plan":
        rows = _log(rng, 1, 16384)
        return {"kind": "plan", "rows": rows, "requests": _log(rng, 1, min(rows, 256)), "adapters": _log(rng, 1, 128)}
    if kind == "linear":
        dtype = rng.choice(["bf16", "bf16", "f16"])
        base, out = rng.choice([("f32", dtype), ("f32", dtype), (dtype, dtype), ("f32", "f32")])
        step = rng.choice([128, 8, 1])  # whole scale groups, whole vectors, anything
        K, N = step * _log(rng, 512 // step, 8192 // step), step * _log(rng, 512 // step, 8192 // step)
        rows = _log(rng, 1, min(16384, 16384 * 4096 * 8 // (2 * K + 6 * N)))
        requests = _log(rng, 1, min(rows, 64))
        return {"kind": "linear", "rows": rows, "requests": requests, "adapters": _log(rng, 1, 48), "rank": rng.choice([4, 8, 16, 16, 32, 64, 100, 128]),
                "K": K, "N": N, "dtype": dtype, "base": base, "out": out}
    E, top_k, hidden, inter = rng.choice([(64, 8, 2048, 1024), (128, 8, 2048, 768), (96, 6, 4096, 2048)])
    tokens = _log(rng, 1, 2048 * 2048 // hidden)
    rank = rng.choice([4, 8, 16])
    up = rng.random() < 0.5
    return {"kind": "experts", "tokens": tokens, "requests": _log(rng, 1, min(tokens, 64)), "adapters": rng.randint(1, 4), "rank": rank,
            "experts": E, "top_k": top_k, "K": hidden if up else inter, "N": 2 * inter if up else hidden, "parts": 2 if up else 1}


# ------------------------------------------------------------------------------------------------- inputs
def _requests(gen, rows, requests, adapters):
    """(offsets [R + 1], adapter of each request [R], adapter of each row [rows]) as int32; -1: no adapter."""
    cuts = torch.randperm(rows - 1, generator=gen, device=DEV)[:requests - 1].sort().values + 1 if requests > 1 else None
    ends = [torch.full((1,), rows, device=DEV)]
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV)] + ([cuts] if cuts is not None else []) + ends)
    slots = torch.randint(0, adapters, (requests,), generator=gen, device=DEV)
    slots = torch.where(torch.rand(requests, generator=gen, device=DEV) < 0.125, -1, slots).to(torch.int32)
    return offsets.to(torch.int32), slots, slots.repeat_interleave(offsets.diff(), output_size=rows)


def _adapter_values(c, gen, dtype, *lead, parts=1):
    """A [*lead, parts * r, K], B [*lead, N, r] and the scales [adapters] of a case's adapters."""
    r, K, N = c["rank"], c["K"], c["N"]
    A = torch.empty(*lead, parts * r, K, dtype=dtype, device=DEV)
    B = torch.empty(*lead, N, r, dtype=dtype, device=DEV)
    for i in range(lead[0]):  # one adapter at a time: the float32 values in between stay small
        A[i] = torch.randn(A[i].shape, generator=gen, device=DEV) / K ** 0.5
        B[i] = torch.randn(B[i].shape, generator=gen, device=DEV) * (0.3 / r ** 0.5)
    return A, B, 0.5 + torch.rand(lead[0], generator=gen, device=DEV)


def _inputs(case, seed):
    c, gen = case, torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": c}
    if c["kind"] == "route":
        s["logits"] = torch.randn(c["tokens"], c["experts"], generator=gen, device=DEV).to(TYPES[c["dtype"]])
        s["bias"] = torch.randn(c["experts"], generator=gen, device=DEV) * 0.05 if c["bias"] else None
        return s
    s["offsets"], s["slots"], s["row_slots"] = _requests(gen, c["tokens"] if c["kind"] == "experts" else c["rows"], c["requests"], c["adapters"])
    if c["kind"] == "linear":
        dtype = TYPES[c["dtype"]]
        s["A"], s["B"], s["scale"] = _adapter_values(c, gen, dtype, c["adapters"])
        s["x"] = torch.randn(c["rows"], c["K"], generator=gen, device=DEV).to(dtype)
        s["base"] = torch.randn(c["rows"], c["N"], generator=gen, device=DEV).to(TYPES[c["base"]])
    if c["kind"] == "experts":
        s["A"], s["B"], s["scale"] = _adapter_values(c, gen, torch.bfloat16, c["adapters"], c["experts"], parts=c["parts"])
        P = c["tokens"] * c["top_k"]
        s["ids"] = torch.rand(c["tokens"], c["experts"], generator=gen, device=DEV).topk(c["top_k"], -1).indices.to(torch.int32)
        # the first products read the tokens' rows, the second ones the pairs' own rows, in the experts' order
        s["x"] = torch.randn(c["tokens"] if c["parts"] == 2 else P, c["K"], generator=gen, device=DEV).bfloat16()
        s["base"] = torch.randn(P, c["N"], generator=gen, device=DEV)
    return s


def prepare(case, seed):
    """A serving program has its adapters laid out when it takes them up, and the plan of a step serves every projection of
    the step's layers."""
    s, c = _inputs(case, seed), case
    if own and c["kind"] == "route":
        from deepseekternarized_b200.moe import B200Ops

        s["ops"] = B200Ops()
    if own and c["kind"] in ("linear", "experts"):
        from deepseekternarized_b200.ternary.adapters import AdapterPlan, LowRankAdapters

        rows = c["tokens"] if c["kind"] == "experts" else c["rows"]
        s["plan"] = AdapterPlan.from_requests(s["offsets"], s["slots"], rows, c["adapters"])
        s["adapters"] = LowRankAdapters(c["adapters"], c["K"], c["N"], c["rank"], dtype=s["A"].dtype, experts=c.get("experts"), parts=c.get("parts", 1))
        for i, scale in enumerate(s["scale"].tolist()):
            s["adapters"].load(i, s["A"][i], s["B"][i], scale)
    return s


# ------------------------------------------------------------------------------------------------- one pass
def run(state):
    s, c = state, state["case"]
    if own:
        return _run_own(s, c)
    if c["kind"] == "route":
        return _route(s["logits"], s["bias"], c)
    if c["kind"] == "plan":
        return _plan(s["offsets"], s["slots"], c["rows"], c["adapters"])
    if c["kind"] == "linear":
        return _linear(s["x"], s["base"], s["row_slots"].long(), s["A"], s["B"], s["scale"], TYPES[c["out"]])
    return _experts(s, c)


def _run_own(s, c):
    if c["kind"] == "route":
        return s["ops"].route(s["logits"], c["top_k"], 2.5, renorm=c["renorm"], score_func=c["score"], bias=s["bias"], n_groups=c["groups"],
                              topk_groups=c["kept"], group_score=c["group_score"])
    from deepseekternarized_b200.ternary.adapters import AdapterPlan

    if c["kind"] == "plan":
        p = AdapterPlan.from_requests(s["offsets"], s["slots"], c["rows"], c["adapters"])
        return p.rows, p.offsets
    if c["kind"] == "linear":
        return s["adapters"](s["x"], s["plan"], base=s["base"], out_dtype=TYPES[c["out"]])
    p = s["plan"].for_experts(s["ids"], c["experts"])
    return s["adapters"](s["x"], p, base=s["base"], out_dtype=torch.bfloat16, pair_rows=c["parts"] == 1), p.order


# ------------------------------------------------------------------------------------------------- the plain forms
def _route(logits, bias, c):
    """Scores in 64 bits: two experts or groups next to the border are told apart as their exact scores are."""
    T, E, g = c["tokens"], c["experts"], c["groups"]
    v = logits.double()
    if c["score"] == "softmax":
        s = (v - v.amax(-1, keepdim=True)).exp()
        s = s / s.sum(-1, keepdim=True)
    elif c["score"] == "sigmoid":
        s = 1 / (1 + (-v).exp())
    else:
        s = (v.clamp(min=0) + (-v.abs()).exp().log1p()).sqrt()
    key = s if bias is None else s + bias.double()
    best = key.view(T, g, E // g).sort(-1, descending=True).values
    group = best[..., 0] if c["group_score"] == "max" else best[..., :2].sum(-1)
    kept = group.sort(dim=-1, descending=True, stable=True).indices[:, :c["kept"]]
    open_ = torch.zeros(T, g, dtype=torch.bool, device=v.device).scatter_(1, kept, True)
    key = key.masked_fill(~open_.repeat_interleave(E // g, 1), -torch.inf)
    ids = key.sort(dim=-1, descending=True, stable=True).indices[:, :c["top_k"]]
    w = s.gather(1, ids)
    if c["renorm"] and c["top_k"] > 1:
        w = w / (w.sum(-1, keepdim=True) + 1e-20)
    return (w * 2.5).float(), ids.to(torch.int32)


def _plan(offsets, slots, rows, n):
    """Rows in the order of their adapters (those without one last), and where each adapter's rows start."""
    row = torch.arange(rows, device=offsets.device)
    of = slots.long()[(row[:, None] >= offsets[None, 1:]).sum(1)]
    bin_ = torch.where(of < 0, n, of)
    start = (bin_[:, None] < torch.arange(n + 2, device=of.device)).sum(0)
    return bin_.sort(stable=True).indices.to(torch.int32), start.to(torch.int32)


def _linear(x, base, of, A, B, scale, out):
    """Few rows: the products of each row with its own adapter's matrices. Many: with all adapters' at once, and only the
    row's own kept."""
    n, r, K = A.shape
    N, T = B.size(1), x.size(0)
    f = torch.where(of >= 0, scale[of.clamp(min=0)], 0.0)[:, None]
    if T * r * (K + N) <= 1 << 29:
        at = of.clamp(min=0)
        h = torch.bmm(A[at].float(), x.float()[:, :, None])
        d = torch.bmm(B[at].float(), h)[:, :, 0]
    else:
        mine = (of[:, None] == torch.arange(n, device=of.device)).float()
        h = (x.float() @ A.float().view(n * r, K).T).view(T, n, r) * mine[:, :, None]
        d = h.view(T, n * r) @ B.float().transpose(1, 2).reshape(n * r, N)
    return (base.float() + f * d).to(out)


def _experts(s, c):
    """Pairs (token, expert) in the order of experts, inside an expert of adapters (those without one last)."""
    n, E, parts, r = c["adapters"], c["experts"], c["parts"], c["rank"]
    of = s["row_slots"].long().repeat_interleave(c["top_k"])
    bin_ = torch.where(of < 0, n, of)
    order = (s["ids"].view(-1).long() * (n + 1) + bin_).sort(stable=True).indices
    of, e = of[order], s["ids"].view(-1).long()[order]
    at = of.clamp(min=0) * E + e
    x = s["x"][order // c["top_k"]] if parts == 2 else s["x"]
    h = torch.bmm(s["A"].view(n * E, parts * r, c["K"])[at].float(), x.float()[:, :, None])
    d = torch.matmul(s["B"].view(n * E, parts, c["N"] // parts, r)[at].float(), h.view(-1, parts, r, 1)).reshape(-1, c["N"])
    f = torch.where(of >= 0, s["scale"][of.clamp(min=0)], 0.0)[:, None]
    return (s["base"] + f * d).bfloat16(), order


# ------------------------------------------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    """What run() returns, from the definitions, one adapter (of one expert) at a time; None for whole numbers but those of
    the router, which the weights go with."""
    c, s = case, _inputs(case, seed)
    if c["kind"] == "plan":
        return None
    if c["kind"] == "route":
        v = s["logits"].double()
        score = {"softmax": lambda: v.softmax(-1), "sigmoid": lambda: torch.sigmoid(v),
                 "sqrtsoftplus": lambda: torch.logaddexp(v, torch.zeros_like(v)).sqrt()}[c["score"]]()
        key = score if s["bias"] is None else score + s["bias"].double()
        rows = []
        size = c["experts"] // c["groups"]
        two = min(2, size) if c["group_score"] == "top2" else 1
        group = key.unfold(1, size, size).topk(two, -1).values.sum(-1)
        rank = (group[:, None, :] > group[:, :, None]).sum(-1)  # groups above this one, and equal ones before it
        rank += ((group[:, None, :] == group[:, :, None]).tril(-1)).sum(-1)
        allowed = (rank < c["kept"])[:, torch.arange(c["experts"], device=v.device) // size]
        key = torch.where(allowed, key, -torch.inf)
        for _ in range(c["top_k"]):  # arg-max, the lowest id among equals
            best = (key == key.amax(-1, keepdim=True)).to(torch.int8).argmax(-1, keepdim=True)
            rows.append(best)
            key = key.scatter(1, best, -torch.inf)
        ids = torch.cat(rows, 1)
        w = score.gather(1, ids)
        w = w / (w.sum(-1, keepdim=True) + 1e-20) if c["renorm"] and c["top_k"] > 1 else w
        return 2.5 * w, None
    y = s["base"].double()
    if c["kind"] == "linear":
        for a in range(c["adapters"]):
            at = (s["row_slots"] == a).nonzero()[:, 0]
            if at.numel():
                y[at] += s["scale"][a].double() * (s["x"][at].double() @ s["A"][a].double().T @ s["B"][a].double().T)
        return y
    ids, k, r, N = s["ids"].reshape(-1).cpu().tolist(), c["top_k"], c["rank"], c["N"] // c["parts"]
    of = s["row_slots"].cpu().tolist()
    pairs = sorted(range(len(ids)), key=lambda p: (ids[p], of[p // k] if of[p // k] >= 0 else c["adapters"], p))
    members = {}
    for at, p in enumerate(pairs):
        if of[p // k] >= 0:
            members.setdefault((of[p // k], ids[p]), []).append((at, p // k if c["parts"] == 2 else at))
    for (a, e), both in members.items():
        at, rows = torch.tensor(both, device=DEV).T
        for part in range(c["parts"]):
            h = s["x"][rows].double() @ s["A"][a, e, part * r:(part + 1) * r].double().T
            y[at, part * N:(part + 1) * N] += s["scale"][a].double() * (h @ s["B"][a, e, part * N:(part + 1) * N].double().T)
    return y, None


# ------------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if c["kind"] == "route":
        T, E = c["tokens"], c["experts"]
        return {"bytes": T * E * size[c["dtype"]] + (4 * E if c["bias"] else 0) + 8 * T * c["top_k"], "flops": 8 * T * E}
    if c["kind"] == "plan":
        return {"bytes": 4 * c["rows"] + 8 * c["requests"] + 4 * (c["adapters"] + 2), "flops": c["rows"]}
    if c["kind"] == "linear":
        T, n, r, K, N = c["rows"], c["adapters"], c["rank"], c["K"], c["N"]
        seen = n * (1 - (1 - 7 / (8 * n)) ** c["requests"])  # adapters that the requests name, expected
        return {"bytes": int(2 * T * K + T * N * (size[c["base"]] + size[c["out"]]) + 2 * seen * r * (K + N)), "flops": int(1.75 * T * r * (K + N))}
    T, n, r, K, N, E = c["tokens"], c["adapters"], c["rank"], c["K"], c["N"], c["experts"]
    P = T * c["top_k"]
    used = n * (1 - (1 - 7 / (8 * n)) ** c["requests"])  # adapters, and of those the experts that their pairs reach
    seen = used * E * (1 - (1 - 1 / E) ** (0.875 * P / max(used, 1e-9)))
    return {"bytes": int(2 * (T if c["parts"] == 2 else P) * K + 6 * P * N + 2 * seen * r * (c["parts"] * K + N) + 12 * P),
            "flops": int(1.75 * P * r * (c["parts"] * K + N))}
