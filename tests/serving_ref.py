"""Plain 64-bit forms of the serving operators (include/tarscuda_serve.h), on CPU tensors: the
definitions the GPU tests compare with. No code of the package."""
import math

import torch


def gather(pool, table, b, n, page_size):
    """The first n slots of sequence b [n, n_kv, head_dim]; and which of them lie in the pool."""
    slot = torch.arange(n)
    page = table[b].long()[slot // page_size]
    good = (page >= 0) & (page < pool.shape[0])
    rows = pool[page.clamp(0, pool.shape[0] - 1), slot % page_size]
    return torch.where(good[:, None, None], rows, torch.zeros_like(rows)), good


def visible(end, window, sinks):
    """Which of the slots 0 .. end-1 a row whose last visible slot is end-1 sees."""
    j = torch.arange(end)
    return torch.ones(end, dtype=torch.bool) if not window else (j >= end - window) | (j < sinks)


def attend_row(q, k, v, see, scale):
    """One row q [heads, hd] over k, v [n, n_kv, hd]: out [heads, hd], probabilities [heads, n]."""
    nh, n, kv = q.shape[0], k.shape[0], k.shape[1]
    out, prob = torch.zeros(nh, q.shape[1], dtype=torch.float64), torch.zeros(nh, n, dtype=torch.float64)
    idx = torch.nonzero(see)[:, 0]
    if idx.numel():
        for h in range(nh):
            g = h // (nh // kv)
            s = (k[idx, g].double() @ q[h].double()) * scale
            p = torch.softmax(s, 0)
            out[h] = p @ v[idx, g].double()
            prob[h, idx] = p
    return out, prob


def attend(k, v, table, length, q, scale, window, sinks, page_size):
    B, nh = q.shape[:2]
    out = torch.zeros(q.shape, dtype=torch.float64)
    weights = []
    for b in range(B):
        n = int(length[b])
        kk, good = gather(k, table, b, n, page_size)
        vv, _ = gather(v, table, b, n, page_size)
        out[b], p = attend_row(q[b], kk, vv, visible(n, window, sinks) & good, scale)
        weights.append(p.reshape(k.shape[2], nh // k.shape[2], n).sum(1))
    return out, weights


def attend_prompt(k, v, table, length, q, cu, scale, window, sinks, page_size):
    out = torch.zeros(q.shape, dtype=torch.float64)
    for b in range(len(length)):
        n, L = int(cu[b + 1] - cu[b]), int(length[b])
        kk, good = gather(k, table, b, L, page_size)
        vv, _ = gather(v, table, b, L, page_size)
        for i in range(n):
            end = L - n + i + 1
            if end > 0:
                out[int(cu[b]) + i] = attend_row(q[int(cu[b]) + i], kk[:end], vv[:end],
                                                 visible(end, window, sinks) & good[:end], scale)[0]
    return out


def rank_value(w):
    """Larger stays longer; a NaN before every number; -0 as 0."""
    return (1, 0.0) if math.isnan(w) else (0, w + 0.0)


def evict(weight, pos, length, seen, budget, sinks, recent):
    """Per (sequence, head): the kept slots of the new cache in slot order, as old slots."""
    out = []
    for b in range(weight.shape[0]):
        n = int(length[b])
        for h in range(weight.shape[1]):
            if n <= budget:
                out.append(list(range(n)))
                continue
            must = lambda s: int(pos[b, h, s]) < sinks or int(pos[b, h, s]) >= int(seen[b]) - recent  # noqa: E731
            rank = lambda s: (not must(s), (0, 0.0) if must(s) else tuple(-x for x in rank_value(float(weight[b, h, s]))), s)  # noqa: E731
            kept = set(sorted(range(n), key=rank)[:budget])
            arrive = iter(sorted(s for s in kept if s >= budget))
            out.append([s if s in kept else next(arrive) for s in range(budget)])
    return out


def adjust(x, hist, n_hist, n_prompt, rep, pres, freq, ids, bias, allowed):
    """One row of logits in 64 bits, and the pick (None: nothing allowed)."""
    x = x.double().clone()
    V = x.numel()
    seen, made = set(), {}
    for i in range(n_hist):
        t = int(hist[i])
        if 0 <= t < V:
            seen.add(t)
            if i >= n_prompt:
                made[t] = made.get(t, 0) + 1
    for t in seen:
        x[t] = x[t] / rep if x[t] > 0 else x[t] * rep
    for t, c in made.items():
        x[t] = x[t] - freq * c - pres
    last = {int(t): float(b) for t, b in zip(ids, bias) if 0 <= int(t) < V}
    for t, b in last.items():
        x[t] += b
    pick = None
    for t in torch.nonzero(allowed)[:, 0].tolist():
        v = float(x[t])
        if pick is None or (math.isnan(v) and not math.isnan(float(x[pick]))) or v > float(x[pick]):
            pick = t
    x[~allowed] = -math.inf
    return x, pick
