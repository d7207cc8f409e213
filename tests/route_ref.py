"""Token routing in 64 bits on the CPU, written from the definitions in include/mrs.h."""
import torch

INF = float("inf")
U32 = 2.0**-24  # half a step of a float32, relative to the value


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Half the distance of two numbers where they no longer get finer."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def keys(scores, bias):
    k = scores.float()
    k = k + bias.float() if bias is not None else k
    return torch.where(k > -INF, k, torch.full_like(k, -INF))  # NaN does not take part


def select_ids(scores, bias, topk):
    k = keys(scores, bias)
    ids = torch.full((k.size(0), topk), -1, dtype=torch.int32)
    for t in range(k.size(0)):
        row = k[t].tolist()
        best = sorted((e for e in range(len(row)) if row[e] > -INF), key=lambda e: (-row[e], e))[:topk]
        ids[t, : len(best)] = torch.tensor(best, dtype=torch.int32)
    return ids


def _parts(scores, bias, ids):
    s = scores.double()
    part = keys(scores, bias) > -INF
    s = torch.where(part, s, torch.full_like(s, -INF))
    experts = s.size(1)
    ok = (ids >= 0) & (ids < experts)
    at = ids.clamp(0, experts - 1).long()
    ok = ok & torch.gather(part, 1, at)
    return s, part, ok, at


def _ratio(x, over):
    """exp(x) / sum of exp(over), rows with nothing in `over` 0.  The maximum goes first: a difference of two numbers of 1e38
    is exact, the logarithm of a sum would vanish beside them."""
    m = over.amax(1, keepdim=True)
    m = torch.where(m > -INF, m, torch.zeros_like(m))
    total = torch.exp(over - m).sum(1, keepdim=True)
    return torch.where(total > 0, torch.exp(x - m) / total, torch.zeros_like(x))


def weights(scores, bias, ids, gate, normalize, scale):
    s, part, ok, at = _parts(scores, bias, ids)
    sel = torch.where(ok, torch.gather(s, 1, at), torch.full_like(at, -INF, dtype=torch.float64))
    x = torch.nn.functional.logsigmoid(sel) if gate == "sigmoid" else sel
    if normalize:
        q = _ratio(x, x)
    elif gate == "softmax":
        q = _ratio(x, s)
    else:
        q = torch.exp(x)
    return torch.where(ok, q * scale, torch.zeros_like(q))


def scores_grad(scores, bias, ids, dw, gate, normalize, scale):
    """The formula of the derivative, slot by slot."""
    s, part, ok, at = _parts(scores, bias, ids)
    g = torch.where(ok, dw.double() * scale, torch.zeros(ids.shape, dtype=torch.float64))
    q = weights(scores, bias, ids, gate, normalize, 1.0)
    sel = torch.where(ok, torch.gather(s, 1, at), torch.zeros(ids.shape, dtype=torch.float64))
    away = torch.sigmoid(-sel) if gate == "sigmoid" else torch.ones_like(sel)
    if normalize:
        d = q * away * (g - (q * g).sum(1, keepdim=True))
    else:
        d = q * away * g
    d = torch.where(ok, d, torch.zeros_like(d))
    ds = torch.zeros_like(s)
    for j in range(ids.size(1)):
        ds.scatter_add_(1, at[:, j : j + 1], d[:, j : j + 1])
    if gate == "softmax" and not normalize:
        p = _ratio(s, s)
        ds = ds - p * d.sum(1, keepdim=True)
    return ds


def order(ids, experts, align, capacity, rows):
    flat = ids.reshape(-1).tolist()
    lists = [[] for _ in range(experts)]
    for slot, e in enumerate(flat):
        if 0 <= e < experts and (capacity == 0 or len(lists[e]) < capacity):
            lists[e].append(slot)
    row_of_slot = torch.full((len(flat),), -1, dtype=torch.int32)
    slot_of_row = torch.full((rows,), -1, dtype=torch.int32)
    offsets = [0]
    for slots in lists:
        at = offsets[-1]
        if slots:
            idx = torch.tensor(slots, dtype=torch.int64)
            row_of_slot[idx] = torch.arange(at, at + len(slots), dtype=torch.int32)
            slot_of_row[at : at + len(slots)] = idx.to(torch.int32)
        offsets.append(at + (len(slots) + align - 1) // align * align)
    counts = torch.tensor([len(x) for x in lists], dtype=torch.int32)
    return row_of_slot.reshape(ids.shape), slot_of_row, counts, torch.tensor(offsets, dtype=torch.int32)


def dispatch(x, row_of_slot, counts, offsets, before):
    out = before.clone()
    for e in range(counts.numel()):
        out[int(offsets[e]) + int(counts[e]) : int(offsets[e + 1])] = 0
    t, k = row_of_slot.shape
    for j in range(k):
        token = torch.nonzero(row_of_slot[:, j] >= 0).squeeze(1)
        out[row_of_slot[token, j].long()] = x[token]
    return out


def combine(rows, row_of_slot, w):
    """(sum, sum of magnitudes) in 64 bits."""
    t, k = row_of_slot.shape
    total = torch.zeros(t, rows.size(1), dtype=torch.float64)
    size = torch.zeros_like(total)
    for j in range(k):
        token = torch.nonzero(row_of_slot[:, j] >= 0).squeeze(1)
        term = rows[row_of_slot[token, j].long()].double()
        if w is not None:
            term = term * w[token, j : j + 1].double()
        total[token] += term
        size[token] += term.abs()
    return total, size


def combine_backward(dout, rows, row_of_slot, w, counts, offsets, before):
    """(gradient of rows in 64 bits, gradient of weights, sum of magnitudes of the latter)."""
    t, k = row_of_slot.shape
    drows = before.double().clone()
    for e in range(counts.numel()):
        drows[int(offsets[e]) + int(counts[e]) : int(offsets[e + 1])] = 0
    dw = torch.zeros(t, k, dtype=torch.float64)
    size = torch.zeros_like(dw)
    g = dout.double()
    for j in range(k):
        token = torch.nonzero(row_of_slot[:, j] >= 0).squeeze(1)
        r = row_of_slot[token, j].long()
        drows[r] = g[token] * w[token, j : j + 1].double()
        prod = g[token] * rows[r].double()
        dw[token, j] = prod.sum(1)
        size[token, j] = prod.abs().sum(1)
    return drows, dw, size
