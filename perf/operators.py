"""Products in which every row of states picks its own weights, and what picks them: routing to experts, the experts'
feed-forward on packed weights, and the low-rank adapters of many requests beside a shared projection.

A case is a dict:

  op      "route"     logits [tokens, experts] to the ``k`` experts of each token and their weights
          "experts"   a gated feed-forward (features -> width -> features) of the experts that each token was given
          "adapters"  the low-rank terms of each request's adapter, added onto the output of a projection

Sizes are those of the test-suite and of the benchmark (5120, 20480, 11008, 8192, 4096) or powers of two and odd multiples
of 64 beside them.  ``own`` chooses between the framework's kernels and elementary torch operations.
"""
import math

import torch

own = False
DEV = "cuda"
LARGEST = 2 * 4096 * 8 * 3 * 2048 * 1024          # flops of the largest listed experts' case


def _route(name, tokens, experts, k, scoring="softmax", bias=False, groups=1, of_groups=1, group_score="max", renormalize=True,
           scale=1.0, half=True, masked=0.0):
    case = dict(op="route", tokens=tokens, experts=experts, k=k, scoring=scoring, bias=bias, groups=groups, of_groups=of_groups,
                group_score=group_score, renormalize=renormalize, scale=scale, half=half, masked=masked)
    return dict(name=name, **case) if name else case


def _experts(name, tokens, experts, k, features, width, bits=4, group=128, sparse=False, expo=0.0, idle=0.0):
    case = dict(op="experts", tokens=tokens, experts=experts, k=k, features=features, width=width, bits=bits, group=group,
                sparse=sparse, expo=expo, idle=idle)
    return dict(name=name, **case) if name else case


def _adapters(name, batch, rows, adapters, rank, features, out, per_token=False, idle=0.0):
    case = dict(op="adapters", batch=batch, rows=rows, adapters=adapters, rank=rank, features=features, out=out,
                per_token=per_token, idle=idle)
    return dict(name=name, **case) if name else case


def listed():
    return [
        # one generated token: a launch and little else
        _route("route_token", 1, 64, 8),
        # a batch of prompts, scores of their own with a bias that balances the experts, groups, logits in 32 bits
        _route("route_prompts", 4096, 256, 8, "sigmoid", True, 8, 4, "top2", True, 2.5, half=False),
        # a ragged number of tokens and of experts, some of which a token may not use
        _route("route_ragged", 777, 60, 4, masked=0.2, renormalize=False),
        # one generated token through eight of 64 small experts: bound by the launches and the latency of memory
        _experts("experts_token", 1, 64, 8, 2048, 1024),
        # 64 sequences that generate a token each, through two of eight large experts: bound by reading the weights
        _experts("experts_tokens_64", 64, 8, 2, 4096, 11008),
        # a short prompt of odd length through 16:32 experts of an odd width
        _experts("experts_prompt_45_sparse", 45, 16, 4, 2048, 1408, group=64, sparse=True),
        # a prompt of ragged length, three bits with one group, some rows padding that goes to no expert
        _experts("experts_prompt_777_int3", 777, 32, 4, 2048, 768, bits=3, group=-1, idle=0.1),
        # a batch of prompts: bound by the matrix cores
        _experts("experts_prompts_4096", 4096, 64, 8, 2048, 1024),
        # one generated token with an adapter
        _adapters("adapters_token", 1, 1, 8, 16, 5120, 5120),
        # 64 requests that generate a token each, every one with an adapter of its own choice of 128
        _adapters("adapters_tokens_64", 64, 1, 128, 64, 5120, 20480),
        # eight prompts, an adapter each, some without one
        _adapters("adapters_prompts", 8, 512, 4, 16, 5120, 20480, idle=0.2),
        # a packed batch of ragged requests: the adapter changes from token to token, odd rank
        _adapters("adapters_ragged", 1, 777, 24, 20, 2048, 1408, per_token=True, idle=0.1),
    ]


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def draw(rng):
    op = rng.choice(["route", "experts", "experts", "adapters", "adapters"])
    if op == "route":
        groups = rng.choice([1, 1, 4, 8])
        experts = max(1, int(_log(rng, 8, 512)) // groups) * groups
        if groups > 1:
            experts = max(experts, 4 * groups)
        of_groups = rng.randint(1, groups)
        k = rng.randint(1, min(10, experts // groups * of_groups))
        return _route(None, int(_log(rng, 1, 8193)), experts, k, rng.choice(["softmax", "sigmoid"]), rng.random() < 0.5, groups, of_groups,
                      rng.choice(["max", "top2"]), rng.random() < 0.7, rng.choice([1.0, 2.5]), rng.random() < 0.5, rng.choice([0.0, 0.0, 0.3]))
    if op == "experts":
        bits, sparse = rng.choice([(4, False), (4, False), (4, False), (3, False), (2, False), (4, True)])
        group = rng.choice([64, 128, 128, -1] if not sparse else [64, 128])
        experts = int(_log(rng, 4, 129))
        k = rng.randint(1, min(8, experts))
        while True:
            features, width = (max(512, int(_log(rng, 512, 8192)) // 64 * 64) for _ in range(2))
            if 3 * experts * features * width <= 1.0e9:
                break
        tokens = int(_log(rng, 1, 4097))
        while 2 * tokens * k * 3 * features * width > LARGEST:
            tokens = max(1, tokens // 2)
        return _experts(None, tokens, experts, k, features, width, bits, group, sparse, rng.choice([0.0, 0.0, 0.0, 0.025]), rng.choice([0.0, 0.1]))
    rank = rng.choice([4, 8, 16, 16, 32, 64, int(_log(rng, 1, 129))])
    features, out = (max(512, int(_log(rng, 512, 20481)) // 64 * 64) for _ in range(2))
    adapters = max(1, min(int(_log(rng, 1, 129)), int(3e8 / (rank * (features + out)))))
    if rng.random() < 0.5:
        return _adapters(None, int(_log(rng, 1, 257)), 1, adapters, rank, features, out, idle=rng.choice([0.0, 0.2]))
    batch = rng.choice([1, 1, 2, 4])
    rows = max(2, int(_log(rng, 2, 4096)) // batch)
    while batch * rows * adapters * rank * (features + out) > 4e11:
        rows = max(1, rows // 2)
    return _adapters(None, batch, rows, adapters, rank, features, out, rng.random() < 0.5, rng.choice([0.0, 0.2]))


# ---------------------------------------------------------------------------------------------------------- inputs
def _masks(n, s, gen):
    """int32 [n, s]: words with exactly 16 bits set"""
    kept = torch.rand((4096, 32), generator=gen, device=DEV).argsort(dim=1) < 16
    words = (kept.to(torch.int64) << torch.arange(32, device=DEV)).sum(dim=1).to(torch.int32)
    return words[torch.randint(0, 4096, (n, s), generator=gen, device=DEV)]


def _packed(case, k, s, gen):
    """packed matrices, scales, zeros and masks of all experts: uniform codes are uniform words in every dense format"""
    n, bits = case["experts"], case["bits"]
    groups = 1 if case["group"] < 0 else (k + case["group"] - 1) // case["group"]
    matrix = torch.randint(-2 ** 31, 2 ** 31, (n, k // 16 if case["sparse"] else k * bits // 32, s), dtype=torch.int32, generator=gen, device=DEV)
    lo, hi = (0.001, 0.02) if bits == 4 else (0.004, 0.08)
    scales = torch.empty((n, groups, s), device=DEV).uniform_(lo, hi, generator=gen)
    if bits == 4:
        zeros = torch.empty((n, groups, s), device=DEV).uniform_(5.0, 10.0, generator=gen).half()
    else:
        zeros = torch.full((n, groups, s), (2 ** bits - 1) / 2, device=DEV).half()
    if case["expo"] > 0:
        # (a weight of a group in exponent mode is z -+ s 2^e)
        chosen = torch.rand((n, groups, s), generator=gen, device=DEV) < case["expo"]
        scales = torch.where(chosen, -scales / 2 ** (2 ** (bits - 1) - bits + 1), scales)
        zeros = torch.where(chosen, torch.zeros_like(zeros), zeros)
    mask = _masks(n * k // 32, s, gen).reshape(n, k // 32, s) if case["sparse"] else None
    return matrix, scales.half(), zeros, mask


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEV)

    state = dict(case=case)
    if case["op"] == "route":
        # some experts are liked better than others
        logits = 1.5 * normal(case["tokens"], case["experts"]) + 0.5 * normal(case["experts"])
        if case["masked"] > 0:
            barred = torch.rand((case["tokens"], case["experts"]), generator=gen, device=DEV) < case["masked"]
            logits = logits.masked_fill(barred, -math.inf)
        state["logits"] = logits.half() if case["half"] else logits
        state["bias"] = 0.1 * normal(case["experts"]) if case["bias"] else None
    elif case["op"] == "experts":
        t, n, k = case["tokens"], case["experts"], case["k"]
        state["x"] = normal(t, case["features"]).half()
        liking = normal(t, n) + 0.5 * normal(n)
        ids = liking.argsort(dim=1, descending=True)[:, :k]
        state["weights"] = liking.gather(1, ids).softmax(dim=1)
        if case["idle"] > 0:
            ids = torch.where(torch.rand((t, 1), generator=gen, device=DEV) < case["idle"], -1, ids)
        state["ids"] = ids.to(torch.int32).contiguous()
        state["up"] = _packed(case, case["features"], 2 * case["width"], gen)
        state["down"] = _packed(case, case["width"], case["features"], gen)
    else:
        shape = case["batch"], case["rows"]
        state["x"] = normal(*shape, case["features"]).half()
        state["base"] = normal(*shape, case["out"]).half()
        state["a"] = (normal(case["adapters"], case["rank"], case["features"]) / math.sqrt(case["features"])).half()
        state["b"] = (0.2 * normal(case["adapters"], case["rank"], case["out"])).half()
        state["scales"] = torch.empty(case["adapters"], device=DEV).uniform_(0.25, 2.0, generator=gen)
        of = shape if case["per_token"] else shape[:1]
        ids = torch.randint(0, case["adapters"], of, generator=gen, device=DEV)
        if case["idle"] > 0:
            ids = torch.where(torch.rand(of, generator=gen, device=DEV) < case["idle"], -1, ids)
        state["ids"] = ids.to(torch.int32)
    return state


# ------------------------------------------------------------------------------------------------------- plain forms
def _plain_route(state):
    """in 64 bits: which expert comes last may hang on a difference that 32 bits lose"""
    case = state["case"]
    logits = state["logits"].double()
    tokens, experts = logits.shape
    logits = torch.where(logits.isnan(), -math.inf, logits)
    top = logits.max(dim=1, keepdim=True).values
    if case["scoring"] == "softmax":
        p = torch.where(logits == -math.inf, 0.0, torch.exp(logits - top))
        p = p / p.sum(dim=1, keepdim=True)
    else:
        p = 1.0 / (1.0 + torch.exp(-logits))
    shown = p if state["bias"] is None else p + state["bias"].double()
    key = logits if state["bias"] is None else torch.where(logits == -math.inf, -math.inf, shown)
    if case["groups"] > 1:
        size = experts // case["groups"]
        parts = key.reshape(tokens, case["groups"], size)
        best = parts.max(dim=2).values
        if case["group_score"] == "top2":
            out = torch.where(key == -math.inf, -math.inf, shown).reshape(parts.shape).sort(dim=2, descending=True).values
            two = out[:, :, 0] + torch.where(out[:, :, 1] == -math.inf, 0.0, out[:, :, 1]) if size > 1 else out[:, :, 0]
            best = torch.where(best == -math.inf, -math.inf, two)
        rank = best.sort(dim=1, descending=True, stable=True).indices
        kept = torch.zeros_like(best, dtype=torch.bool).scatter_(1, rank[:, :case["of_groups"]], True)
        key = torch.where(kept[:, :, None], parts, -math.inf).reshape(tokens, experts)
    found, ids = key.sort(dim=1, descending=True, stable=True)
    found, ids = found[:, :case["k"]], ids[:, :case["k"]]
    none = found == -math.inf
    weights = torch.where(none, 0.0, p.gather(1, ids))
    if case["renormalize"]:
        total = weights.sum(dim=1, keepdim=True)
        weights = torch.where(total > 0, weights / total, weights)
    return (weights * case["scale"]).float(), torch.where(none, -1, ids).to(torch.int32)


def _plain_weights(case, packed, active):
    """the weights of the experts ``active`` in 32 bits, [experts, k, s]"""
    matrix, scales, zeros, mask = (None if part is None else part[active] for part in packed)
    n, rows, s = matrix.shape
    bits = case["bits"]
    if mask is not None:
        kept = (mask[:, :, None] >> torch.arange(32, dtype=torch.int32, device=DEV)[:, None]) & 1
        rank = (kept.cumsum(dim=2, dtype=torch.int32) - kept).clamp(max=15)
        word = torch.where(rank < 8, matrix[:, 0::2, None], matrix[:, 1::2, None])
        q = (word >> (4 * (rank & 7))) & 15
        q, kept = q.reshape(n, -1, s), kept.reshape(n, -1, s)
    elif bits == 3:
        words = matrix.reshape(n, rows // 3, 3, s)
        at = 3 * torch.arange(32, device=DEV)
        low = words[:, :, at // 32] >> (at % 32).to(torch.int32)[:, None]
        # (the bits that an arithmetic shift brings in from above are the sign's: they are cut off first)
        left = torch.clamp(32 - at % 32, max=3).to(torch.int32)
        low = low & ((1 << left) - 1)[:, None]
        high = words[:, :, torch.clamp(at // 32 + 1, max=2)] & ((1 << (3 - left)) - 1)[:, None]
        q = (low | (high << left[:, None])).reshape(n, -1, s)
    else:
        q = ((matrix[:, :, None] >> torch.arange(0, 32, bits, dtype=torch.int32, device=DEV)[:, None]) & (2 ** bits - 1)).reshape(n, -1, s)
    k = q.shape[1]
    group = k if case["group"] < 0 else case["group"]
    scales, zeros = (part.float().repeat_interleave(group, dim=1)[:, :k] for part in (scales, zeros))
    w = (q.float() - zeros) * scales
    if case["expo"] > 0:
        half = 2 ** (bits - 1)
        power = torch.where(q >= half, -1.0, 1.0) * torch.exp2((q % half).float())
        w = torch.where(scales >= 0, w, zeros - scales * power)
    return w if mask is None else w * kept


def _plain_experts(state):
    """the rows of each expert side by side, padded to the most that one has"""
    case, x, ids = state["case"], state["x"].float(), state["ids"].long()
    tokens, k = ids.shape
    order = ids.reshape(-1).sort(stable=True).indices
    chosen = ids.reshape(-1)[order]
    order, chosen = order[chosen >= 0], chosen[chosen >= 0]
    y = torch.zeros((tokens, case["features"]), device=DEV)
    if order.numel() == 0:
        return y.half()
    active, expert, counts = chosen.unique_consecutive(return_inverse=True, return_counts=True)
    first = counts.cumsum(0) - counts
    slot = torch.arange(order.numel(), device=DEV) - first[expert]
    rows = torch.zeros((active.numel(), int(counts.max()), case["features"]), device=DEV)
    rows[expert, slot] = x[order // k]
    both = torch.bmm(rows, _plain_weights(case, state["up"], active))
    gate, up = both[:, :, :case["width"]], both[:, :, case["width"]:]
    h = gate / (1.0 + torch.exp(-gate)) * up
    out = torch.bmm(h, _plain_weights(case, state["down"], active))
    term = out[expert, slot] * state["weights"].reshape(-1)[order, None]
    by_slot = torch.zeros((tokens * k, case["features"]), device=DEV)
    by_slot[order] = term
    return by_slot.reshape(tokens, k, -1).sum(dim=1).half()


def _plain_adapters(state):
    """every row through every adapter in use, the others' terms left out"""
    x, base, ids = state["x"].float(), state["base"].float(), state["ids"].long()
    batch, rows, features = x.shape
    each = (ids if ids.dim() == 2 else ids[:, None].expand(batch, rows)).reshape(-1)
    active, which = each.unique(return_inverse=True)
    a, b = (state[name][active.clamp(min=0)].float() for name in ("a", "b"))
    down = (x.reshape(-1, features) @ a.reshape(-1, features).t()).reshape(batch * rows, active.numel(), -1)
    mine = torch.zeros((batch * rows, active.numel()), device=DEV)
    scale = torch.where(each >= 0, state["scales"][each.clamp(min=0)], 0.0)
    mine.scatter_(1, which[:, None], scale[:, None])
    term = (down * mine[:, :, None]).reshape(batch * rows, -1) @ b.reshape(-1, b.shape[-1])
    return (base + term.reshape(base.shape)).half()


def run(state):
    case = state["case"]
    if not own:
        return {"route": _plain_route, "experts": _plain_experts, "adapters": _plain_adapters}[case["op"]](state)
    import int4matmul_kernels_amd as pkg
    ext = pkg.load_extension()
    if case["op"] == "route":
        return ext.route_experts(state["logits"], case["k"], case["scoring"], state["bias"], case["groups"], case["of_groups"],
                                 case["group_score"], case["renormalize"], case["scale"])
    if case["op"] == "experts":
        (up, up_scales, up_zeros, up_mask), (down, down_scales, down_zeros, down_mask) = state["up"], state["down"]
        return ext.experts_forward(case["bits"], state["x"], state["weights"], state["ids"], up, up_scales, up_zeros,
                                   down, down_scales, down_zeros, case["group"], up_mask, down_mask)
    return ext.low_rank_add(state["base"], state["x"], state["a"], state["b"], state["scales"], state["ids"])


# --------------------------------------------------------------------------------------------------- what it costs
def work(case):
    if case["op"] == "route":
        t, n = case["tokens"], case["experts"]
        return {"bytes": t * n * (2 if case["half"] else 4) + 4 * n * case["bias"] + 8 * t * case["k"], "flops": 4 * t * n}
    if case["op"] == "experts":
        t, n, k, features, width = (case[name] for name in ("tokens", "experts", "k", "features", "width"))
        used = n * (1 - (1 - k / n) ** t)
        bits = 3 if case["sparse"] else case["bits"]
        up, down = (1 if case["group"] < 0 else -(-rows // case["group"]) for rows in (features, width))
        one = 3 * features * width * bits / 8 + 4 * (up * 2 * width + down * features)
        return {"bytes": used * one + 4 * t * features + 8 * t * k, "flops": 2 * t * k * 3 * features * width}
    rows, features, out, rank, n = case["batch"] * case["rows"], case["features"], case["out"], case["rank"], case["adapters"]
    picks = rows if case["per_token"] else case["batch"]
    used = n * (1 - (1 - 1 / n) ** picks)
    return {"bytes": 2 * rows * (features + 2 * out) + 2 * used * rank * (features + out), "flops": 2 * rows * rank * (features + out)}


# ----------------------------------------------------------------------------------------------- in 64 bits, by the letter
def _exact_route(state):
    import numpy as np
    case = state["case"]
    logits = state["logits"].double().cpu().numpy()
    bias = None if state["bias"] is None else state["bias"].double().cpu().numpy()
    tokens, experts = logits.shape
    weights, ids = np.zeros((tokens, case["k"])), np.full((tokens, case["k"]), -1, dtype=np.int32)
    size = experts // case["groups"]
    for t in range(tokens):
        row = logits[t]
        allowed = row > -math.inf                                   # (False for NaN as well)
        if not allowed.any():
            continue
        if case["scoring"] == "softmax":
            p = np.exp(np.where(allowed, row, -math.inf) - row[allowed].max())
            p /= p.sum()
        else:
            p = np.where(allowed, 1 / (1 + np.exp(-np.where(allowed, row, 0.0))), 0.0)
        value = p if bias is None else p + bias
        order_by = row if bias is None else value
        live = np.flatnonzero(allowed)
        if case["groups"] > 1:
            scores = []
            for g in range(case["groups"]):
                members = live[live // size == g]
                if members.size == 0:
                    continue
                if case["group_score"] == "max":
                    scores.append((-order_by[members].max(), g))
                else:
                    scores.append((-np.sort(value[members])[-2:].sum(), g))
            chosen = {g for _, g in sorted(scores)[:case["of_groups"]]}
            live = live[np.isin(live // size, list(chosen))]
        best = live[np.argsort(-order_by[live], kind="stable")][:case["k"]]
        w = p[best]
        if case["renormalize"] and w.sum() > 0:
            w = w / w.sum()
        ids[t, :best.size], weights[t, :best.size] = best, w * case["scale"]
    return torch.from_numpy(weights), torch.from_numpy(ids)


def _exact_weights(case, packed, e):
    matrix, scales, zeros, mask = (None if part is None else part[e] for part in packed)
    words = matrix.long() & 0xFFFFFFFF
    s, bits = words.shape[1], case["bits"]
    if mask is not None:
        bit = (mask.long()[:, None] >> torch.arange(32, device=DEV)[None, :, None]) & 1
        codes = torch.zeros((mask.shape[0], 32, s), dtype=torch.long, device=DEV)
        left = words[0::2] | (words[1::2] << 32)                     # sixteen codes, the next one lowest
        for row in range(32):
            codes[:, row] = left & 15
            left = torch.where(bit[:, row] == 1, (left >> 4) & (2 ** 60 - 1), left)
        codes, bit = codes.reshape(-1, s), bit.reshape(-1, s)
    else:
        # the column's bits in a row, ``bits`` of them to a code (three bits: 96 to a block; the others never straddle a word)
        stream = ((words[:, None] >> torch.arange(32, device=DEV)[None, :, None]) & 1).reshape(-1, bits, s)
        codes = (stream << torch.arange(bits, device=DEV)[None, :, None]).sum(dim=1)
    k = codes.shape[0]
    group = torch.arange(k, device=DEV) // (k if case["group"] < 0 else case["group"])
    q, scale, zero = codes.double(), scales.double()[group], zeros.double()[group]
    half = 2 ** (bits - 1)
    power = 2.0 ** (codes % half).double() * torch.where(codes < half, 1.0, -1.0).double()
    w = torch.where(scale >= 0, (q - zero) * scale, zero - scale * power)
    return w if mask is None else torch.where(bit == 1, w, torch.zeros_like(w))


def _exact_experts(state):
    case, x, ids = state["case"], state["x"].double(), state["ids"].long()
    y = torch.zeros((case["tokens"], case["features"]), dtype=torch.float64, device=DEV)
    for e in range(case["experts"]):
        token, slot = (ids == e).nonzero(as_tuple=True)
        if token.numel() == 0:
            continue
        gate, up = (x[token] @ _exact_weights(case, state["up"], e)).split(case["width"], dim=1)
        h = gate * torch.sigmoid(gate) * up
        y.index_add_(0, token, state["weights"].double()[token, slot][:, None] * (h @ _exact_weights(case, state["down"], e)))
    return y


def _exact_adapters(state):
    y, x, ids = state["base"].double(), state["x"].double(), state["ids"].long()
    for e in range(state["case"]["adapters"]):
        rows = ids == e
        if bool(rows.any()):
            a, b = state["a"][e].double(), state["b"][e].double()
            y[rows] += state["scales"][e].double() * (x[rows] @ a.t() @ b)
    return y


def exact(case, seed):
    return {"route": _exact_route, "experts": _exact_experts, "adapters": _exact_adapters}[case["op"]](prepare(case, seed))
