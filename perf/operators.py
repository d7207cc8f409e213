"""The token routing operators as a user calls them, with their plain forms and sizes to time them at.

T tokens choose k of E experts each (`select`), the T * k slots are ordered by expert (`order`), rows of H
elements go to expert order (`dispatch`) and come back weighted (`combine`); `*_grad` are the
backward passes.  `own` switches `run` from the plain torch form to the library's calls.
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "u8": torch.uint8}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2, "u8": 1}
_DEVICE = "cuda"


# ---- the cases ------------------------------------------------------------------------------
def _gate(name, op, tokens, experts, topk, dtype, gate, normalize, scale=1.0, bias=False, masked=0.0):
    return dict(name=name, op=op, tokens=tokens, experts=experts, topk=topk, dtype=dtype, gate=gate,
                normalize=normalize, scale=scale, bias=bias, masked=masked)


def _move(name, op, tokens, experts, topk, hidden, dtype, align=1, drop=0.0, capacity=0, pad=0):
    return dict(name=name, op=op, tokens=tokens, experts=experts, topk=topk, hidden=hidden, dtype=dtype,
                align=align, drop=drop, capacity=capacity, pad=pad)


def listed():
    return [
        # one decoding step of a few sequences: nothing but latency
        _gate("select_decode", "select", 8, 256, 8, "bf16", "softmax", True),
        # a long prompt, some experts masked off for some tokens, weights from the softmax over all experts
        _gate("select_prompt", "select", 16384, 128, 8, "f32", "softmax", False, masked=0.05),
        # a training step: choice steered by a balancing bias, weights from sigmoids, and the scores' gradient
        _gate("select_train", "select_grad", 65536, 256, 8, "f32", "sigmoid", True, scale=2.5, bias=True),
        # the slots of one decoding step, segments aligned to a small tile of a grouped product
        _move("order_decode", "order", 64, 256, 8, 0, "f32", align=16),
        # 2^20 slots of a training step, aligned to a large tile, at most 1.25 times the even share per expert
        _move("order_train", "order", 131072, 256, 8, 0, "f32", align=128, capacity=5120),
        # rows of one decoding step
        _move("dispatch_decode", "dispatch", 32, 64, 8, 4096, "bf16", align=16),
        # rows of a long prompt
        _move("dispatch_prompt", "dispatch", 16384, 128, 8, 4096, "bf16", align=128),
        # the tokens' gradient of a training step, some slots dropped
        _move("dispatch_grad_train", "dispatch_grad", 16384, 64, 4, 2048, "bf16", align=128, drop=0.02),
        # one token comes back from its experts
        _move("combine_decode", "combine", 1, 256, 8, 4096, "f16", align=16),
        # a long prompt comes back
        _move("combine_prompt", "combine", 16384, 128, 8, 4096, "bf16", align=128),
        # the backward pass of the way back, whole
        _move("combine_grad_train", "combine_grad", 16384, 128, 8, 4096, "bf16", align=128),
        # odd everything: 3000 tokens, three slots, a prime row length inside a wider buffer, a third of the slots dropped
        _move("combine_grad_odd", "combine_grad", 3000, 60, 3, 1109, "f32", drop=0.3, pad=5),
    ]


def _log_int(rng, lo, hi):
    """An integer spread evenly over its logarithm, odd ones among them."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["select", "select_grad", "order", "dispatch", "dispatch", "dispatch_grad", "combine", "combine",
                     "combine_grad", "combine_grad"])
    topk = rng.choice([1, 2, 3, 4, 6, 8, 8, 10, 16])
    experts = max(topk, rng.choice([8, 16, 60, 64, 128, 160, 256, 257, 384, 512]))
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op in ("select", "select_grad"):
        tokens = _log_int(rng, 1, min(65536, (1 << 24) // experts))
        return dict(op=op, tokens=tokens, experts=experts, topk=topk, dtype=dtype,
                    gate=rng.choice(["softmax", "sigmoid"]), normalize=rng.random() < 0.5,
                    scale=rng.choice([1.0, 2.5]), bias=rng.random() < 0.5, masked=rng.choice([0.0, 0.0, 0.1]))
    align = rng.choice([1, 1, 8, 16, 64, 128])
    drop = rng.choice([0.0, 0.0, 0.02, 0.5])
    if op == "order":
        tokens = _log_int(rng, 1, (1 << 20) // topk)
        capacity = rng.choice([0, 0, max(1, tokens * topk // experts)])
        return dict(op=op, tokens=tokens, experts=experts, topk=topk, hidden=0, dtype="f32", align=align, drop=drop,
                    capacity=capacity, pad=0)
    if op == "dispatch" and rng.random() < 0.2:
        dtype = "u8"  # rows quantised before they are moved
    hidden = _log_int(rng, 16, 8192)
    if rng.random() < 0.6:
        hidden = max(16, hidden // 16 * 16)
    most = min(32768, (256 << 20) // (topk * hidden * _BYTES[dtype]))
    tokens = _log_int(rng, 1, max(1, most))
    if tokens * topk < experts:
        align = min(align, 16)  # hardly any user aligns a few rows to a large tile
    return dict(op=op, tokens=tokens, experts=experts, topk=topk, hidden=hidden, dtype=dtype, align=align, drop=drop,
                capacity=0, pad=rng.choice([0, 0, 0, 3, 16]))


def work(case):
    t, e, k, es = case["tokens"], case["experts"], case["topk"], _BYTES[case["dtype"]]
    n, op = t * k, case["op"]
    if op in ("select", "select_grad"):
        if op == "select":
            return {"bytes": t * e * es + 8 * n, "flops": 4 * t * e}
        return {"bytes": 2 * t * e * es + 12 * n, "flops": 8 * t * e}
    if op == "order":
        return {"bytes": 8 * n + 4 * _max_rows(case) + 8 * e, "flops": n}
    kept = n * (1.0 - case["drop"])
    row = case["hidden"] * es
    # padding rows: half a tile for every expert that has a row
    padded = min(kept, e) * (case["align"] - 1) / 2
    if op == "dispatch":
        return {"bytes": int(t * row + (kept + padded) * row + 4 * n), "flops": 0}
    if op == "dispatch_grad":
        return {"bytes": int(t * row + kept * row + 4 * n), "flops": int(kept * case["hidden"])}
    if op == "combine":
        return {"bytes": int(t * row + kept * row + 8 * n), "flops": int(2 * kept * case["hidden"])}
    return {"bytes": int(t * row + (2 * kept + padded) * row + 12 * n), "flops": int(3 * kept * case["hidden"])}


# ---- what a program has in hand before the call ---------------------------------------------
def _max_rows(case):
    n, e, a, c = case["tokens"] * case["topk"], case["experts"], case["align"], case["capacity"]
    rows = n + min(n, e) * (a - 1)
    return min(rows, e * (-(-c // a) * a)) if c else rows


def _generator(seed):
    g = torch.Generator(device=_DEVICE)
    g.manual_seed(seed)
    return g


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=_DEVICE, dtype=dtype)


def _choose(case, g):
    """Expert ids of every slot: some experts are asked for more often than others, some slots go nowhere."""
    t, e, k = case["tokens"], case["experts"], case["topk"]
    popularity = _normal(g, e)
    ids = torch.empty(t, k, dtype=torch.int32, device=_DEVICE)
    for lo in range(0, t, 16384):
        hi = min(t, lo + 16384)
        ids[lo:hi] = torch.topk(_normal(g, hi - lo, e) * 2.0 + popularity, k, dim=1).indices.to(torch.int32)
    if case["drop"]:
        lost = torch.rand(t, k, generator=g, device=_DEVICE) < case["drop"]
        ids = torch.where(lost, torch.full_like(ids, -1), ids)
    return ids


def _rows(g, rows, hidden, case):
    """A [rows, hidden] tensor, inside wider rows where the case has `pad`."""
    dtype = _DTYPES[case["dtype"]]
    width = hidden + case["pad"]
    if dtype == torch.uint8:
        full = torch.randint(0, 256, (rows, width), generator=g, device=_DEVICE, dtype=torch.uint8)
    else:
        full = torch.empty(rows, width, dtype=dtype, device=_DEVICE)
        for lo in range(0, rows, 32768):
            hi = min(rows, lo + 32768)
            full[lo:hi] = _normal(g, hi - lo, width)
    return full[:, :hidden]


_context = None


def _plan(case):
    """The handle a program keeps: one plan for the shapes of a layer."""
    global _context
    import wgpu_morton_code_radix_sort_test_amd as mrs

    if _context is None:
        _context = mrs.Context(0)
    gates = {"softmax": mrs.GATE_SOFTMAX, "sigmoid": mrs.GATE_SIGMOID}
    return mrs, mrs.RoutePlan(_context, case["tokens"], case["experts"], case["topk"], align=case.get("align", 1),
                              capacity=case.get("capacity", 0), gate=gates[case.get("gate", "softmax")],
                              normalize=case.get("normalize", True), scale=case.get("scale", 1.0))


def prepare(case, seed):
    g = _generator(seed)
    t, e, k = case["tokens"], case["experts"], case["topk"]
    state = {"case": case}
    if own:
        mrs, state["plan"] = _plan(case)
    if case["op"] in ("select", "select_grad"):
        scores = _normal(g, t, e) * 1.5 + _normal(g, e)
        if case["masked"]:
            scores = scores.masked_fill(torch.rand(t, e, generator=g, device=_DEVICE) < case["masked"], -math.inf)
            if t > 8:
                scores[t // 3] = -math.inf  # a padding token: nothing to choose from
        state["scores"] = scores.to(_DTYPES[case["dtype"]])
        state["bias"] = _normal(g, e) * 0.25 if case["bias"] else None
        state["dweights"] = _normal(g, t, k)
        return state
    ids = _choose(case, g)
    if case["op"] == "order":
        state["ids"] = ids
        if own:
            state["map"] = state["plan"].new_map()
        return state
    h = case["hidden"]
    parts = _order(ids, e, case["align"], case["capacity"], _max_rows(case))
    state["row_of_slot"] = parts[0]
    if own:
        state["map"] = mrs.RouteMap(*parts)
    rows = _max_rows(case)
    if case["op"] == "dispatch":
        state["x"] = _rows(g, t, h, case)
        state["out"] = torch.zeros(rows, h, dtype=_DTYPES[case["dtype"]], device=_DEVICE)
    elif case["op"] == "dispatch_grad":
        state["drows"] = _rows(g, rows, h, case)
    else:
        state["rows"] = _rows(g, rows, h, case)
        state["weights"] = torch.softmax(_normal(g, t, k), dim=1)
        if case["op"] == "combine_grad":
            state["dout"] = _rows(g, t, h, case)
            state["out"] = torch.zeros(rows, h, dtype=_DTYPES[case["dtype"]], device=_DEVICE)
    return state


# ---- the plain forms ------------------------------------------------------------------------
def _order(ids, experts, align, capacity, rows):
    """row_of_slot [T, k], slot_of_row [rows], counts [E], offsets [E + 1]."""
    flat = ids.reshape(-1).to(torch.int64)
    n = flat.numel()
    key = torch.where((flat >= 0) & (flat < experts), flat, torch.full_like(flat, experts))
    sorted_key, slot = torch.sort(key, stable=True)
    asked = torch.zeros(experts + 1, dtype=torch.int64, device=ids.device).scatter_add_(0, key, torch.ones_like(key))
    first = torch.cumsum(asked, 0) - asked
    rank = torch.arange(n, device=ids.device) - first[sorted_key]
    counts = asked[:experts].clamp(max=capacity) if capacity else asked[:experts]
    offsets = torch.zeros(experts + 1, dtype=torch.int64, device=ids.device)
    offsets[1:] = torch.cumsum((counts + align - 1) // align * align, 0)
    row = offsets[sorted_key] + rank
    kept = sorted_key < experts
    if capacity:
        kept = kept & (rank < capacity)
    row_of_slot = torch.empty(n, dtype=torch.int64, device=ids.device)
    row_of_slot[slot] = torch.where(kept, row, torch.full_like(row, -1))
    # one entry more than there are rows takes the slots without one
    slot_of_row = torch.full((rows + 1,), -1, dtype=torch.int64, device=ids.device)
    slot_of_row[torch.where(kept, row, torch.full_like(row, rows))] = slot
    return (row_of_slot.to(torch.int32).reshape(ids.shape), slot_of_row[:rows].to(torch.int32), counts.to(torch.int32),
            offsets.to(torch.int32))


def _select(scores, bias, case):
    s = scores.to(torch.float32)
    key = s + bias if bias is not None else s + 0.0
    part = key > -math.inf
    order_key = torch.where(part, key, torch.full_like(key, -math.inf))
    ids = torch.sort(order_key, dim=1, descending=True, stable=True).indices[:, : case["topk"]]
    chosen = torch.gather(part, 1, ids)
    p = _probabilities(s, part, case)
    q = torch.where(chosen, torch.gather(p, 1, ids), torch.zeros((), device=s.device))
    if case["normalize"]:
        q = q / q.sum(dim=1, keepdim=True).clamp(min=1e-37)
    return torch.where(chosen, ids, torch.full_like(ids, -1)).to(torch.int32), q * case["scale"]


def _probabilities(s, part, case):
    zero = torch.zeros((), device=s.device)
    if case["gate"] == "sigmoid":
        return torch.where(part, 1.0 / (1.0 + torch.exp(-s)), zero)
    m = torch.where(part, s, torch.full_like(s, -3e38)).amax(dim=1, keepdim=True)
    x = torch.where(part, torch.exp(s - m), zero)
    return x / x.sum(dim=1, keepdim=True).clamp(min=1e-37)


def _select_grad(scores, bias, ids, dweights, case):
    s = scores.to(torch.float32)
    part = (s + bias if bias is not None else s) > -math.inf
    p = _probabilities(s, part, case)
    chosen = ids >= 0
    at = ids.clamp(min=0).to(torch.int64)
    pj = torch.where(chosen, torch.gather(p, 1, at), torch.zeros((), device=s.device))
    gj = dweights * case["scale"]
    if case["normalize"]:
        q = pj / pj.sum(dim=1, keepdim=True).clamp(min=1e-37)
        d = q * (gj - (gj * q).sum(dim=1, keepdim=True))
        if case["gate"] == "sigmoid":
            d = d * (1.0 - pj)
    elif case["gate"] == "sigmoid":
        d = pj * (1.0 - pj) * gj
    else:
        d = pj * gj
    d = torch.where(chosen, d, torch.zeros((), device=s.device))
    ds = torch.zeros_like(s).scatter_add_(1, at, d)
    if case["gate"] == "softmax" and not case["normalize"]:
        ds = ds - p * d.sum(dim=1, keepdim=True)
    return ds.to(scores.dtype)


def _dispatch(x, row_of_slot, out):
    t, k = row_of_slot.shape
    kept = row_of_slot >= 0
    token = torch.arange(t, device=x.device).unsqueeze(1).expand(t, k)
    out = torch.zeros_like(out)
    out[row_of_slot[kept].to(torch.int64)] = x[token[kept]]
    return out


def _combine(rows, row_of_slot, weights):
    t, k = row_of_slot.shape
    total = torch.zeros(t, rows.shape[1], dtype=torch.float32, device=rows.device)
    for j in range(k):
        r = row_of_slot[:, j].to(torch.int64)
        term = rows[r.clamp(min=0)].to(torch.float32)
        if weights is not None:
            term = term * weights[:, j : j + 1]
        total += torch.where((r >= 0).unsqueeze(1), term, torch.zeros((), device=rows.device))
    return total.to(rows.dtype)


def _combine_grad(dout, rows, row_of_slot, weights, out):
    t, k = row_of_slot.shape
    drows = torch.zeros_like(out)
    dweights = torch.zeros(t, k, dtype=torch.float32, device=rows.device)
    wide = dout.to(torch.float32)
    for j in range(k):
        r = row_of_slot[:, j].to(torch.int64)
        kept = r >= 0
        drows[r[kept]] = (wide * weights[:, j : j + 1])[kept].to(rows.dtype)
        dot = (wide * rows[r.clamp(min=0)].to(torch.float32)).sum(dim=1)
        dweights[:, j] = torch.where(kept, dot, torch.zeros((), device=rows.device))
    return drows, dweights


# ---- one pass -------------------------------------------------------------------------------
def run(state):
    case, op = state["case"], state["case"]["op"]
    if own:
        plan = state["plan"]
        if op == "select":
            return plan.select(state["scores"], state["bias"])
        if op == "select_grad":
            ids, weights = plan.select(state["scores"], state["bias"])
            return ids, weights, plan.select_backward(state["scores"], ids, state["dweights"], state["bias"])
        route = state["map"]
        if op == "order":
            plan.order(state["ids"], route)
            return route.row_of_slot, route.slot_of_row, route.counts, route.offsets
        if op == "dispatch":
            return plan.dispatch(state["x"], route, rows_out=state["out"])
        if op == "dispatch_grad":
            return plan.dispatch_backward(state["drows"], route)
        if op == "combine":
            return plan.combine(state["rows"], route, state["weights"])
        return plan.combine_backward(state["dout"], state["rows"], route, state["weights"], drows_out=state["out"])
    if op == "select":
        return _select(state["scores"], state["bias"], case)
    if op == "select_grad":
        ids, weights = _select(state["scores"], state["bias"], case)
        return ids, weights, _select_grad(state["scores"], state["bias"], ids, state["dweights"], case)
    if op == "order":
        return _order(state["ids"], case["experts"], case["align"], case["capacity"], _max_rows(case))
    if op == "dispatch":
        return _dispatch(state["x"], state["row_of_slot"], state["out"])
    if op == "dispatch_grad":
        return _combine(state["drows"], state["row_of_slot"], None)
    if op == "combine":
        return _combine(state["rows"], state["row_of_slot"], state["weights"])
    return _combine_grad(state["dout"], state["rows"], state["row_of_slot"], state["weights"], state["out"])


# ---- the definitions in 64 bits -------------------------------------------------------------
def _exact_select(state, case):
    """Chosen one after the other: the largest key left, at its lowest index."""
    scores, bias = state["scores"], state["bias"]
    t, e, k = case["tokens"], case["experts"], case["topk"]
    key = scores.float()
    if bias is not None:
        key = key + bias
    key = torch.where(key == key, key, torch.full_like(key, -math.inf))
    takes_part = torch.isfinite(key) | (key > 0)
    index = torch.arange(e, device=key.device).expand(t, e)
    left = key.clone()
    ids = torch.empty(t, k, dtype=torch.int64, device=key.device)
    for j in range(k):
        top = left.max(dim=1, keepdim=True).values
        at = torch.where(left == top, index, torch.full_like(index, e)).min(dim=1).values
        found = top.squeeze(1) > -math.inf
        ids[:, j] = torch.where(found, at, torch.full_like(at, -1))
        left.scatter_(1, at.unsqueeze(1), -math.inf)
    s = scores.double()
    s = torch.where(takes_part, s, torch.full_like(s, -math.inf))
    sel = torch.gather(s, 1, ids.clamp(min=0)).masked_fill(ids < 0, -math.inf)
    if case["gate"] == "softmax":
        base = sel if case["normalize"] else s
        q = torch.exp(sel - torch.logsumexp(base, dim=1, keepdim=True))
    else:
        log_p = torch.nn.functional.logsigmoid(sel)
        q = torch.exp(log_p - torch.logsumexp(log_p, dim=1, keepdim=True)) if case["normalize"] else torch.exp(log_p)
    q = torch.where(ids >= 0, q, torch.zeros_like(q))
    return ids, s, sel, q


def _exact_select_grad(s, sel, ids, q, dweights, case):
    """Row by row the Jacobian of the weights times their gradient."""
    g = torch.where(ids >= 0, dweights.double() * case["scale"], torch.zeros_like(q))
    keep = torch.sigmoid(-sel) if case["gate"] == "sigmoid" else torch.ones_like(q)
    if case["normalize"]:
        d = q * keep * (g - (g * q).sum(dim=1, keepdim=True))
    else:
        d = q * keep * g
    full = torch.zeros_like(s)
    for j in range(ids.shape[1]):
        row = torch.nonzero(ids[:, j] >= 0).squeeze(1)
        full[row, ids[row, j]] += d[row, j]
    if case["gate"] == "softmax" and not case["normalize"]:
        p = torch.exp(s - torch.logsumexp(s, dim=1, keepdim=True))
        full -= torch.nan_to_num(p) * (q * g).sum(dim=1, keepdim=True)
    return full


def _exact_order(ids, case):
    flat = ids.reshape(-1).cpu().numpy()
    rows = _max_rows(case)
    row_of_slot = np.full(flat.size, -1, dtype=np.int64)
    slot_of_row = np.full(rows, -1, dtype=np.int64)
    counts = np.zeros(case["experts"], dtype=np.int64)
    offsets = np.zeros(case["experts"] + 1, dtype=np.int64)
    at = 0
    for e in range(case["experts"]):
        slots = np.flatnonzero(flat == e)
        if case["capacity"]:
            slots = slots[: case["capacity"]]
        row_of_slot[slots] = at + np.arange(slots.size)
        slot_of_row[at : at + slots.size] = slots
        counts[e] = slots.size
        at += -(-slots.size // case["align"]) * case["align"]
        offsets[e + 1] = at
    return tuple(torch.from_numpy(a).to(_DEVICE, torch.int32)
                 for a in (row_of_slot.reshape(ids.shape), slot_of_row, counts, offsets))


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op in ("select", "select_grad"):
        ids, s, sel, q = _exact_select(state, case)
        weights = q * case["scale"]
        if op == "select":
            return ids.to(torch.int32), weights
        return ids.to(torch.int32), weights, _exact_select_grad(s, sel, ids, q, state["dweights"], case)
    if op == "order":
        return _exact_order(state["ids"], case)
    route = state["row_of_slot"].to(torch.int64)
    t, k = route.shape
    if op == "dispatch":
        out = state["out"].clone()
        for j in range(k):
            token = torch.nonzero(route[:, j] >= 0).squeeze(1)
            out[route[token, j]] = state["x"][token]
        return out if case["dtype"] == "u8" else out.double()
    rows = state["drows"] if op == "dispatch_grad" else state["rows"]
    weights = torch.ones(t, k, dtype=torch.float64, device=rows.device)
    if op != "dispatch_grad":
        weights = state["weights"].double()
    if op in ("combine", "dispatch_grad"):
        out = torch.zeros(t, rows.shape[1], dtype=torch.float64, device=rows.device)
        for j in range(k):
            token = torch.nonzero(route[:, j] >= 0).squeeze(1)
            out.index_add_(0, token, rows[route[token, j]].double() * weights[token, j].unsqueeze(1))
        return out
    dout = state["dout"].double()
    drows = torch.zeros(rows.shape, dtype=torch.float64, device=rows.device)
    dweights = torch.zeros(t, k, dtype=torch.float64, device=rows.device)
    for j in range(k):
        token = torch.nonzero(route[:, j] >= 0).squeeze(1)
        drows[route[token, j]] = dout[token] * weights[token, j].unsqueeze(1)
        dweights[token, j] = (dout[token] * rows[route[token, j]].double()).sum(dim=1)
    return drows, dweights
