"""Trees of drafted tokens, accumulated attention weight and eviction, in 64 bits on the CPU, from their definitions."""
import torch

from . import paged


def path_to(parents, i):
    """The tokens on the way down to token i, itself the last."""
    path = [i]
    while 0 <= parents[path[0]] < path[0]:
        path.insert(0, int(parents[path[0]]))
    return path


def mask(parents):
    """[B, N] -> int32 [B, N, ceil(N / 32)]."""
    B, N = parents.shape
    out = torch.zeros(B, N, (N + 31) // 32, dtype=torch.int64)
    for b in range(B):
        for i in range(N):
            for j in path_to(parents[b].tolist(), i):
                out[b, i, j // 32] |= 1 << (j % 32)
    return torch.where(out >= 2 ** 31, out - 2 ** 32, out).int()


def seen_keys(t, place, table, starts, window=None, tree=None):
    """The positions that row t, of sequence and position `place`, sees."""
    b, pos = place
    j = torch.arange(max(0, pos + 1 - window) if window else 0, pos + 1)
    if tree is not None:
        at = j - (pos - (t - int(starts[b])))
        word = tree[t].long()[(at.clamp(min=0) // 32).clamp(max=tree.shape[1] - 1)]
        j = j[(at < 0) | (at >= 32 * tree.shape[1]) | ((word >> (at % 32)) & 1).bool()]
    return j


def attention(q, cache, table, lens, starts, scale, window=None, tree=None):
    """As paged.attention, with a tree and the logarithms: -> (o, bound, lse)."""
    k, v = paged.dense(cache, 0), paged.dense(cache, 1)
    T, heads, d = q.shape
    kv, page = k.shape[1], k.shape[2]
    o, mean = (torch.zeros(T, heads, d, dtype=torch.float64) for _ in range(2))
    size, most = (torch.zeros(T, heads, dtype=torch.float64) for _ in range(2))
    lse = torch.full((T, heads), -torch.inf, dtype=torch.float64)
    q = q.cpu().double()
    tree = tree.cpu() if tree is not None else None
    g = torch.arange(heads) * kv // heads
    for t, place in enumerate(paged.places(table, lens, starts, page, T)):
        if place is None or place[1] < 0:
            continue
        j = seen_keys(t, place, table, starts, window, tree)
        if len(j) == 0:
            continue
        rows = table[place[0]].cpu().long()[j // page]
        kj, vj = (x[rows, :, j % page][:, g] for x in (k, v))  # [keys, heads, d]
        x = torch.einsum("jhd,hd->jh", kj, q[t]) * scale
        w = torch.softmax(x, 0)
        lse[t] = torch.logsumexp(x, 0)
        o[t] = torch.einsum("jh,jhd->hd", w, vj)
        mean[t] = torch.einsum("jh,jhd->hd", w, vj.abs())
        size[t] = (torch.einsum("jhd,hd->jh", kj.abs(), q[t].abs()) * scale).amax(0)
        most[t] = vj.abs().amax((0, 2))
    return o, (mean, size, most), lse


def lse_tolerance(lse, size, d, eight_bit, keys):
    """How far a logarithm may be off: by the scores' error (paged.tolerance), the sum's (an addition a key and an exponential each,
    half a step or 2^-22 of their terms), and two roundings of the result and of the maximum in log2.  Over an 8-bit cache, the scales'."""
    return (2 * (d + 4) * 2.0 ** -24 * size + (2.0 ** -16 if eight_bit else 0.0) + 2.0 ** -20 + keys * 2.0 ** -24 +
            4 * 2.0 ** -24 * torch.where(torch.isfinite(lse), lse.abs(), 0.0))


def weights(before, q, cache, lse, table, lens, starts, scale, window=None):
    """-> (weights [pages, kv, page_size], tolerance): `before` with what the new tokens attend to.

    A term p = exp(x - lse) is off by p times the error of x (as in paged.tolerance; for bf16 queries over an 8-bit cache the query's
    numbers are kept to 2^-25 of the row's largest), of lse in log2, rounded once (2^-24 of it, and as much of x), and 2^-21 for the
    exponential; a sum of n terms by n half steps, and the number before it by one."""
    k = paged.dense(cache, 0)
    T, heads, d = q.shape
    kv, page = k.shape[1], k.shape[2]
    rescaled = q.dtype == torch.bfloat16 and len(cache) == 4
    out, tol, terms = before.cpu().double().clone(), torch.zeros(before.shape, dtype=torch.float64), torch.zeros(before.shape)
    q, lse = q.cpu().double(), lse.cpu().double()
    where = paged.places(table, lens, starts, page, T)
    for place in where:  # new tokens begin at 0
        if place is not None and place[1] >= 0:
            out[int(table[place[0], place[1] // page]), :, place[1] % page] = 0.0
    old = out.abs().clone()
    g = torch.arange(heads) * kv // heads
    for t, place in enumerate(where):
        if place is None or place[1] < 0:
            continue
        j = seen_keys(t, place, table, starts, window)
        rows = table[place[0]].cpu().long()[j // page]
        kj = k[rows, :, j % page][:, g]
        x = torch.einsum("jhd,hd->jh", kj, q[t]) * scale
        size = torch.einsum("jhd,hd->jh", kj.abs(), q[t].abs()) * scale
        kept = 2.0 ** -25 * scale * q[t].abs().amax(-1) * kj.abs().sum(-1) if rescaled else 0.0
        fine = torch.isfinite(lse[t])
        p = torch.where(fine, torch.exp(x - torch.where(fine, lse[t], 0.0)), 0.0)
        e = p * (2 * (d + 4) * 2.0 ** -24 * size + kept + 2.0 ** -21 + 4 * 2.0 ** -24 * (x.abs() + torch.where(fine, lse[t].abs(), 0.0)))
        for h in range(kv):
            mine = g == h
            out[rows, h, j % page] += p[:, mine].sum(1)
            tol[rows, h, j % page] += e[:, mine].nan_to_num(0.0).sum(1)
            terms[rows, h, j % page] += int(mine.sum())
    return out, tol + (terms + 2) * 2.0 ** -24 * out.abs() + 2.0 ** -24 * old


def verify(probs, tokens, parents, u):
    """-> (tokens out [B, N], path [B, N], counts [B])."""
    B, N = tokens.shape
    V = probs.shape[2]
    out = torch.full((B, N), -1, dtype=torch.int64)
    path = torch.full((B, N), -1, dtype=torch.int32)
    counts = torch.zeros(B, dtype=torch.int32)
    probs = torch.where(torch.isfinite(probs) & (probs > 0), probs, 0.0).double()
    for b in range(B):
        at, way = 0, [0]
        while True:
            rest, refused, taken = 1.0, [], None
            for c in range(at + 1, N):
                if int(parents[b, c]) != at:
                    continue
                x = int(tokens[b, c])
                p = float(probs[b, at, x]) if 0 <= x < V and x not in refused else 0.0
                if float(u[b, c]) * rest < p:
                    taken = c
                    break
                rest = max(rest - p, 0.0)
                refused.append(x)
            if taken is None:
                break
            at = taken
            way.append(at)
        w = probs[b, at].clone()
        for x in refused:
            if 0 <= x < V:
                w[x] = 0.0
        if not float(w.sum()) > 0:
            w = probs[b, at]
        for i, c in enumerate(way):
            path[b, i] = c
            if i > 0:
                out[b, i - 1] = tokens[b, c]
        counts[b] = len(way)
        if float(w.sum()) > 0:
            sums = w.cumsum(0)
            above = (sums > float(u[b, 0]) * float(sums[-1])).nonzero()
            out[b, len(way) - 1] = int(above[0]) if len(above) else int((w > 0).nonzero()[-1])
    return out, path, counts


def keep(planes, kept, counts, table, first=None, into=None):
    """planes: tensors [pages, kv, page_size, ..] on the CPU -> what they are after the moves."""
    into = table if into is None else into
    after = [x.clone() for x in planes]
    kv, page = planes[0].shape[1], planes[0].shape[2]
    for b in range(len(counts)):
        f = 0 if first is None else int(first[b])
        for h in range(kv):
            for i in range(min(max(int(counts[b]), 0), kept.shape[-1])):
                src = f + int(kept[b, i] if kept.dim() == 2 else kept[b, h, i])
                for x, y in zip(planes, after):
                    y[int(into[b, (f + i) // page]), h, (f + i) % page] = x[int(table[b, src // page]), h, src % page]
    return after


def choose(weights, table, lens, keep, recent):
    """-> (lengths, kept [B, kv, keep])."""
    B, kv, page = len(lens), weights.shape[1], weights.shape[2]
    kept = torch.full((B, kv, keep), -1, dtype=torch.int32)
    for b in range(B):
        n = int(lens[b])
        for h in range(kv):
            j = list(range(n))
            if n > keep:
                w = [float(weights[int(table[b, i // page]), h, i % page]) for i in j]
                w = [-float("inf") if x != x else x for x in w]
                nan = [float(weights[int(table[b, i // page]), h, i % page]) != float(weights[int(table[b, i // page]), h, i % page]) for i in j]
                order = sorted(j[: n - recent], key=lambda i: (nan[i], -w[i], i))
                j = sorted(order[: keep - recent]) + j[n - recent:]
            kept[b, h, : len(j)] = torch.tensor(j, dtype=torch.int32)
    return torch.tensor([min(int(n), keep) for n in lens], dtype=torch.int32), kept
