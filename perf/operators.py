"""Operators of a mixture of experts, as cases that can be measured: routing of tokens to experts, the
expert order of the chosen rows, products in 8-bit integers with a scale for each row of both operands
(dense or by expert), and the weighted sum of the experts' rows that brings them back to the tokens.

``own = False`` computes every operator from elementary torch operations; ``own = True`` makes the
calls that a user makes of `sklearn_numba_dpex_b200.common`.
"""
import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decoding step of a small batch: scores by sigmoid, a bias for balance, groups of experts
        _route("route_decode", 4, 256, 8, "bf16", "sigmoid", bias=True, groups=8, topk_groups=4,
               group_best=2, renorm=True, scale=2.5),
        # a packed prompt with padding rows at its end
        _route("route_prompt", 16384, 128, 8, "fp32", "softmax", renorm=True, padded=True),
        # a training step: forward and backward, weights that are not renormalised
        _route("route_train", 65521, 64, 6, "bf16", "softmax", renorm=False, backward=True),
        # expert order of a decoding step, and of a long packed prompt
        _slots("slots_decode", 64, 8, 256),
        _slots("slots_prompt", 131071, 8, 256, dropped=True),
        # a linear layer in 8 bits: one token, and a long prompt
        _linear("linear_decode", 1, 4096, 4096, "bf16", "bf16"),
        _linear("linear_prompt", 8192, 8192, 4096, "bf16", "bf16", bias=True),
        # the experts' layer: a decoding batch that touches every expert a little, and a ragged prompt
        _experts("experts_decode", 48, 8, 64, 2048, 1024, "bf16", "bf16"),
        _experts("experts_prompt", 4099, 4, 32, 1408, 2056, "fp16", "fp32", dropped=True),
        # the way back to the tokens: a decoding step, a prompt of odd width, a training step
        _combine("combine_decode", 8, 8, 4096, "bf16"),
        _combine("combine_prompt", 8191, 6, 1031, "fp32", dropped=True),
        _combine("combine_train", 8192, 8, 2048, "bf16", backward=True),
    ]


def _route(name, n, experts, k, dtype, scoring, bias=False, groups=1, topk_groups=1, group_best=1,
           renorm=True, scale=1.0, padded=False, backward=False):
    return {"name": name, "op": "route", "n": n, "experts": experts, "k": k, "dtype": dtype,
            "scoring": scoring, "bias": bias, "groups": groups, "topk_groups": topk_groups,
            "group_best": group_best, "renorm": renorm, "scale": scale, "padded": padded,
            "backward": backward}


def _slots(name, n, k, experts, dropped=False):
    return {"name": name, "op": "slots", "n": n, "k": k, "experts": experts, "dropped": dropped}


def _linear(name, m, n, d, dtype, out, bias=False):
    return {"name": name, "op": "linear", "m": m, "n": n, "d": d, "dtype": dtype, "out": out, "bias": bias}


def _experts(name, tokens, k, experts, n, d, dtype, out, bias=False, dropped=False):
    return {"name": name, "op": "experts", "tokens": tokens, "k": k, "experts": experts, "n": n, "d": d,
            "dtype": dtype, "out": out, "bias": bias, "dropped": dropped}


def _combine(name, n, k, d, dtype, dropped=False, backward=False):
    return {"name": name, "op": "combine", "n": n, "k": k, "d": d, "dtype": dtype, "dropped": dropped,
            "backward": backward}


def _spread(rng, low, high):
    """A whole number in [low, high], even over its logarithm."""
    return min(high, max(low, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    op = rng.choice(["route", "slots", "linear", "experts", "combine"])
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    flag = lambda p: rng.random() < p  # noqa: E731
    if op == "route":
        n, backward = _spread(rng, 1, 65521), flag(0.4)
        scoring, renorm = rng.choice(["softmax", "sigmoid"]), flag(0.6)
        if flag(0.4):
            groups = rng.choice([2, 4, 8, 16])
            experts = groups * rng.randint(2, 32)
            topk_groups = rng.randint(1, groups)
            k = rng.randint(1, min(16, topk_groups * (experts // groups)))
            best = rng.choice([1, 2])
        else:
            groups, topk_groups, best = 1, 1, 1
            experts = _spread(rng, 2, 512)
            k = rng.randint(1, min(16, experts))
        c = _route("", n, experts, k, dtype, scoring, flag(0.5), groups, topk_groups, best, renorm,
                   rng.choice([1.0, 2.5]), flag(0.3), backward)
    elif op == "slots":
        experts = _spread(rng, 2, 512)
        c = _slots("", _spread(rng, 1, 131071), rng.randint(1, min(12, experts)), experts, flag(0.5))
    elif op == "linear":
        c = _linear("", _spread(rng, 1, 8192), _spread(rng, 64, 8192), _spread(rng, 64, 4096), dtype,
                    rng.choice(["bf16", "fp16", "fp32"]), flag(0.4))
    elif op == "experts":
        experts = _spread(rng, 2, 128)
        c = _experts("", _spread(rng, 1, 4099), rng.randint(1, min(8, experts)), experts,
                     _spread(rng, 64, 2048), _spread(rng, 64, 2056), dtype,
                     rng.choice(["bf16", "fp16", "fp32"]), flag(0.4), flag(0.4))
    else:
        c = _combine("", _spread(rng, 1, 8192), rng.randint(1, 8), _spread(rng, 16, 4096), dtype,
                     flag(0.4), flag(0.5))
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------ inputs
def _chosen(n, experts, k, gen):
    """k distinct experts for each of n tokens, some experts more popular than others."""
    popular = torch.randn(experts, device="cuda", generator=gen)
    noise = -torch.log(torch.rand((n, experts), device="cuda", generator=gen).clamp_min(1e-20))
    score = popular - noise.clamp_min(1e-20).log()
    return score.topk(k, dim=1).indices.to(torch.int32)


def _drop(experts, gen):
    """A twentieth of the choices, and the last tokens (padding), go to no expert."""
    gone = torch.rand(experts.shape, device="cuda", generator=gen) < 0.05
    gone[experts.shape[0] - experts.shape[0] // 16:] = True
    return torch.where(gone, torch.full_like(experts, -1), experts)


def _weights(shape, gen):
    """8-bit weights with their scales, rows at a pitch of a multiple of 16 bytes."""
    *lead, d = shape
    pitch = -(-d // 16) * 16
    q = torch.randint(-127, 128, (*lead, pitch), device="cuda", generator=gen, dtype=torch.int8)
    scales = (0.5 + torch.rand(lead, device="cuda", generator=gen)) * (1.7 / 127 / d ** 0.5)
    return q[..., :d], scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    randn = lambda *s: torch.randn(s, device="cuda", generator=gen)  # noqa: E731
    s = {"case": dict(case)}
    op = case["op"]
    if op == "route":
        n, e = case["n"], case["experts"]
        logits = (randn(n, e) * 1.5 + randn(e) * 0.5).to(_TYPES[case["dtype"]])
        if case["padded"]:
            logits[n - n // 16:] = float("-inf")    # padding tokens
            logits[: n // 2, e - e // 8:] = float("-inf")  # experts that these tokens may not use
        s["logits"] = logits
        s["bias"] = randn(e) * 0.05 if case["bias"] else None
        s["grad"] = randn(n, case["k"]) if case["backward"] else None
    elif op == "slots":
        experts = _chosen(case["n"], case["experts"], case["k"], gen)
        s["experts"] = _drop(experts, gen) if case["dropped"] else experts
    elif op == "linear":
        s["x"] = (randn(case["m"], case["d"]) * (1 + 3 * randn(case["d"]).abs())).to(_TYPES[case["dtype"]])
        s["w"], s["w_scales"] = _weights((case["n"], case["d"]), gen)
        s["bias"] = randn(case["n"]) if case["bias"] else None
    elif op == "experts":
        g = case["experts"]
        chosen = _chosen(case["tokens"], g, case["k"], gen)
        if case["dropped"]:
            chosen = _drop(chosen, gen)
        _, s["rows"], s["offsets"] = _slots_plain(chosen, g)
        s["most"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())
        s["x"] = (randn(case["tokens"], case["d"]) * (1 + 3 * randn(case["d"]).abs())).to(_TYPES[case["dtype"]])
        s["w"], s["w_scales"] = _weights((g, case["n"], case["d"]), gen)
        s["bias"] = randn(g, case["n"]) if case["bias"] else None
    else:
        n, k = case["n"], case["k"]
        s["values"] = randn(n * k, case["d"]).to(_TYPES[case["dtype"]])
        slots = torch.randperm(n * k, device="cuda", generator=gen).to(torch.int32).view(n, k)
        s["slots"] = _drop(slots, gen) if case["dropped"] else slots
        s["weights"] = torch.softmax(randn(n, k), dim=1)
        s["grad"] = randn(n, case["d"]).to(_TYPES[case["dtype"]]) if case["backward"] else None
    return s


# ------------------------------------------------------------------------------------------ plain forms
def _scores_plain(logits, scoring):
    """Scores in 64 bits: the choice of experts hangs on values that lie next to each other."""
    x = logits.double()
    if scoring == "sigmoid":
        return 1 / (1 + torch.exp(-x))
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = e.sum(1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def _route_plain(c, logits, bias, grad):
    n, e = logits.shape
    k = c["k"]
    scores = _scores_plain(logits, c["scoring"])
    # without a bias the order of the scores is the logits' own, unless two of them are added
    key = logits.double() if bias is None and c["group_best"] == 1 else scores
    key = key if bias is None else key + bias.double()
    key = torch.where(logits == float("-inf"), torch.full_like(key, float("-inf")), key)
    if c["groups"] > 1:
        by_group = key.view(n, c["groups"], -1)
        best = by_group.sort(dim=2, descending=True, stable=True).values[:, :, : c["group_best"]].sum(2)
        order = best.sort(dim=1, descending=True, stable=True).indices[:, : c["topk_groups"]]
        kept = torch.zeros_like(best, dtype=torch.bool).scatter_(1, order, True)
        key = torch.where(kept[:, :, None], by_group, torch.full_like(by_group, float("-inf"))).view(n, e)
    top = key.sort(dim=1, descending=True, stable=True)
    chosen, there = top.indices[:, :k], top.values[:, :k] != float("-inf")
    experts = torch.where(there, chosen, torch.full_like(chosen, -1)).to(torch.int32)
    picked = torch.where(there, scores.gather(1, chosen), torch.zeros_like(scores[:, :1]))
    total = picked.sum(1, keepdim=True)
    total = torch.where(total == 0, torch.ones_like(total), total)
    share = picked / total if c["renorm"] else picked
    weights = (share * c["scale"]).float()
    if grad is None:
        return weights, experts
    g = torch.where(there, grad.double() * c["scale"], torch.zeros_like(share))
    if c["renorm"]:
        inner = share * (g - (share * g).sum(1, keepdim=True))
        inner = inner * (1 - picked) if c["scoring"] == "sigmoid" else inner
        grads = torch.zeros_like(scores).scatter_add_(1, chosen, inner)
    elif c["scoring"] == "sigmoid":
        grads = torch.zeros_like(scores).scatter_add_(1, chosen, g * picked * (1 - picked))
    else:
        dense = torch.zeros_like(scores).scatter_add_(1, chosen, g)
        grads = scores * (dense - (g * picked).sum(1, keepdim=True))
    return weights, experts, grads.to(logits.dtype)


def _slots_plain(experts, n_experts):
    n, k = experts.shape
    flat = experts.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < n_experts), flat, torch.full_like(flat, n_experts))
    ordered, order = key.sort(stable=True)
    place = torch.empty_like(flat)
    place[order] = torch.arange(n * k, device=flat.device)
    slots = torch.where(key < n_experts, place, torch.full_like(place, -1)).view(n, k)
    rows = torch.where(ordered < n_experts, order // k, torch.full_like(order, -1))
    offsets = torch.searchsorted(ordered, torch.arange(n_experts + 1, device=flat.device))
    return slots.to(torch.int32), rows.to(torch.int32), offsets.to(torch.int32)


def _quantize_plain(x):
    """Rows in 8 bits, as whole numbers in 32-bit floats; in 64 bits where the border of a rounding counts."""
    top = x.abs().amax(1, keepdim=True).double()
    q = torch.round(x.double() * 127 / torch.where(top == 0, torch.ones_like(top), top))
    return q.float(), (top / 127).float()


def _linear_plain(c, x, w, w_scales, bias):
    q, scales = _quantize_plain(x)
    out = (q @ w.float().t()) * scales * w_scales
    return (out if bias is None else out + bias).to(_TYPES[c["out"]])


def _experts_plain(c, s):
    rows, offsets, most, g = s["rows"].long(), s["offsets"].long(), s["most"], c["experts"]
    x = s["x"][rows.clamp_min(0)]
    q, scales = _quantize_plain(x)
    at = torch.arange(rows.numel(), device=rows.device)
    group = torch.searchsorted(offsets[1:].contiguous(), at, right=True)
    there = (group < g)[:, None]
    group = group.clamp_max(g - 1)
    place = torch.where(there[:, 0], group * most + at - offsets[group], torch.full_like(at, g * most))
    padded = torch.zeros((g * most + 1, c["d"]), device=x.device).index_copy_(
        0, place, torch.where(there, q, torch.zeros_like(q)))[: g * most].view(g, most, c["d"])
    out = torch.bmm(padded, s["w"].float().transpose(1, 2)).view(g * most, c["n"])[place.clamp_max(g * most - 1)]
    out = out * scales * s["w_scales"][group]
    if s["bias"] is not None:
        out = out + s["bias"][group]
    return torch.where(there, out, torch.zeros_like(out)).to(_TYPES[c["out"]])


def _combine_plain(values, slots, weights, grad):
    there = (slots >= 0)[:, :, None]
    at = slots.long().clamp_min(0)
    picked = torch.where(there, values.float()[at], torch.zeros((), device=values.device))
    share = torch.where(there, weights[:, :, None], torch.zeros((), device=values.device))
    out = (picked * share).sum(1).to(values.dtype)
    if grad is None:
        return out
    g = grad.float()[:, None, :]
    grad_weights = (picked * g).sum(2)
    grad_values = torch.zeros(values.shape, device=values.device).index_add_(
        0, at.reshape(-1), (share * g).reshape(-1, values.shape[1]))
    return out, grad_values.to(values.dtype), grad_weights


def _run_plain(s):
    c = s["case"]
    if c["op"] == "route":
        return _route_plain(c, s["logits"], s["bias"], s["grad"])
    if c["op"] == "slots":
        return _slots_plain(s["experts"], c["experts"])
    if c["op"] == "linear":
        return _linear_plain(c, s["x"], s["w"], s["w_scales"], s["bias"])
    if c["op"] == "experts":
        return _experts_plain(c, s)
    return _combine_plain(s["values"], s["slots"], s["weights"], s["grad"])


# ------------------------------------------------------------------------------------------ the framework's calls
def _run_own(s):
    from sklearn_numba_dpex_b200 import common

    c = s["case"]
    if c["op"] == "route":
        weights, experts = common.route_topk(
            s["logits"], c["k"], bias=s["bias"], scoring=c["scoring"], n_groups=c["groups"],
            topk_groups=c["topk_groups"], group_best=c["group_best"], renormalize=c["renorm"],
            scale=c["scale"])
        if s["grad"] is None:
            return weights, experts
        return weights, experts, common.route_topk_grad(
            s["logits"], experts, s["grad"], scoring=c["scoring"], renormalize=c["renorm"], scale=c["scale"])
    if c["op"] == "slots":
        return common.expert_slots(s["experts"], c["experts"])
    if c["op"] == "linear":
        q, scales = common.quantize_rows(s["x"])
        return common.int8_matmul(q, scales, s["w"], s["w_scales"], bias=s["bias"], out_dtype=_TYPES[c["out"]])
    if c["op"] == "experts":
        q, scales = common.quantize_rows(s["x"], rows=s["rows"])
        return common.int8_matmul(q, scales, s["w"], s["w_scales"], bias=s["bias"], offsets=s["offsets"],
                                  out_dtype=_TYPES[c["out"]])
    out = common.combine_experts(s["values"], s["slots"], s["weights"])
    if s["grad"] is None:
        return out
    return (out, *common.combine_experts_grad(s["values"], s["slots"], s["weights"], s["grad"]))


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    op = case["op"]
    if op == "route":
        n, e, k, size = case["n"], case["experts"], case["k"], _SIZE[case["dtype"]]
        there = n * e * size + n * k * 8 + (4 * e if case["bias"] else 0)
        back = n * e * size + n * k * 4 if case["backward"] else 0
        return {"bytes": there + back, "flops": 4 * n * e * (2 if case["backward"] else 1)}
    if op == "slots":
        return {"bytes": 12 * case["n"] * case["k"] + 4 * (case["experts"] + 1), "flops": 0}
    if op == "linear":
        m, n, d = case["m"], case["n"], case["d"]
        return {"bytes": m * d * _SIZE[case["dtype"]] + n * d + 4 * n * (2 if case["bias"] else 1)
                + m * n * _SIZE[case["out"]], "flops": 2 * m * n * d}
    if op == "experts":
        t, n, d, g = case["tokens"], case["n"], case["d"], case["experts"]
        r = t * case["k"]
        used = min(g, r)    # an expert without rows needs none of its weights
        return {"bytes": t * d * _SIZE[case["dtype"]] + 4 * r + used * n * (d + 4 * (2 if case["bias"] else 1))
                + r * n * _SIZE[case["out"]], "flops": 2 * r * n * d}
    n, k, d, size = case["n"], case["k"], case["d"], _SIZE[case["dtype"]]
    there = n * k * d * size + n * d * size + 8 * n * k
    back = n * k * d * size + n * d * size + 4 * n * k if case["backward"] else 0
    return {"bytes": there + back, "flops": 2 * n * k * d * (3 if case["backward"] else 1)}


# ------------------------------------------------------------------------------------------ 64 bits
def _exact_quantize(x):
    x = x.to(torch.float64)
    top = x.abs().max(1).values
    ratio = x * 127 / top.clamp_min(1e-300)[:, None]
    low = ratio.floor()
    rest = ratio - low
    up = (rest > 0.5) | ((rest == 0.5) & (low.remainder(2) == 1))
    return low + up, top / 127


def _exact_route(c, logits, bias, grad):
    x = logits.to(torch.float64).cpu().numpy()
    n, e = x.shape
    closed = np.isneginf(x)
    with np.errstate(all="ignore"):
        if c["scoring"] == "sigmoid":
            s = np.exp(-np.logaddexp(0, -x))
        else:
            top = np.where(closed.all(1), 0, x.max(1, where=~closed, initial=-np.inf))
            s = np.exp(x - top[:, None])
            s /= np.maximum(s.sum(1), 1e-300)[:, None]
    key = s if bias is None else s + bias.double().cpu().numpy()
    key = x if bias is None and c["group_best"] == 1 else key
    key = np.where(closed, -np.inf, key)
    if c["groups"] > 1:
        parts = key.reshape(n, c["groups"], -1)
        best = -np.sort(-parts, axis=2)[:, :, : c["group_best"]].sum(2)
        rank = np.argsort(np.argsort(-best, axis=1, kind="stable"), axis=1, kind="stable")
        key = np.where((rank < c["topk_groups"])[:, :, None], parts, -np.inf).reshape(n, e)
    key = key.copy()
    experts, picked = np.full((n, c["k"]), -1, np.int64), np.zeros((n, c["k"]))
    row = np.arange(n)
    for j in range(c["k"]):
        at = key.argmax(1)
        there = key[row, at] > -np.inf
        experts[there, j] = at[there]
        picked[there, j] = s[row, at][there]
        key[row, at] = -np.inf
    total = np.where(picked.sum(1) > 0, picked.sum(1), 1)[:, None]
    p = picked / total if c["renorm"] else picked
    out = [torch.from_numpy(p * c["scale"]), torch.from_numpy(experts.astype(np.int32))]
    if grad is not None:
        g = np.where(experts >= 0, grad.double().cpu().numpy() * c["scale"], 0)
        # d p_j / d s_i, then d s / d logits
        ds = (g - (g * p).sum(1, keepdims=True)) / total if c["renorm"] else g
        ds = np.where(experts >= 0, ds, 0)
        full = np.zeros((n, e + 1))
        full[row[:, None], experts] = ds
        full = full[:, :e]
        if c["scoring"] == "sigmoid":
            full = full * s * (1 - s)
        else:
            full = s * (full - (s * full).sum(1, keepdims=True))
        out.append(torch.from_numpy(full))
    return tuple(out)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "route":
        return _exact_route(case, s["logits"], s["bias"], s["grad"])
    if op == "slots":
        e, k = s["experts"].cpu().numpy().reshape(-1), case["k"]
        key = np.where(e < 0, case["experts"], e)
        order = np.argsort(key, kind="stable")
        valid = int((e >= 0).sum())
        slots = np.full(e.size, -1, np.int32)
        slots[order[:valid]] = np.arange(valid, dtype=np.int32)
        rows = np.full(e.size, -1, np.int32)
        rows[:valid] = order[:valid] // k
        offsets = np.concatenate([[0], np.cumsum(np.bincount(key, minlength=case["experts"] + 1)[: case["experts"]])])
        return (torch.from_numpy(slots.reshape(-1, k)), torch.from_numpy(rows),
                torch.from_numpy(offsets.astype(np.int32)))
    if op == "linear":
        q, step = _exact_quantize(s["x"])
        out = torch.einsum("md,nd->mn", q, s["w"].to(torch.float64))
        out = out * (step[:, None] * s["w_scales"].double())
        return out if s["bias"] is None else out + s["bias"].double()
    if op == "experts":
        rows = s["rows"].long()
        q, step = _exact_quantize(s["x"])
        out = torch.zeros((rows.numel(), case["n"]), dtype=torch.float64, device="cuda")
        ends = s["offsets"].tolist()
        for g in range(case["experts"]):
            r = rows[ends[g]: ends[g + 1]]
            y = q[r] @ s["w"][g].double().t() * step[r][:, None] * s["w_scales"][g].double()
            out[ends[g]: ends[g + 1]] = y if s["bias"] is None else y + s["bias"][g].double()
        return out
    slots, there = s["slots"].long(), s["slots"] >= 0
    share = torch.where(there, s["weights"].double(), torch.zeros((), dtype=torch.float64, device="cuda"))
    out = torch.zeros((case["n"], case["d"]), dtype=torch.float64, device="cuda")
    grad_values = torch.zeros(s["values"].shape, dtype=torch.float64, device="cuda")
    grad_weights = torch.zeros(slots.shape, dtype=torch.float64, device="cuda")
    for j in range(case["k"]):
        ok = there[:, j]
        at = slots[:, j][ok]
        out[ok] += share[ok, j][:, None] * s["values"][at].double()
        if s["grad"] is not None:
            grad_values[at] += share[ok, j][:, None] * s["grad"][ok].double()
            grad_weights[ok, j] = (s["values"][at].double() * s["grad"][ok].double()).sum(1)
    return out if s["grad"] is None else (out, grad_values, grad_weights)
