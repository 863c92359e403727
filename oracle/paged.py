"""The paged cache, the attention over it and the verification of drafted tokens, in 64 bits on the CPU, from their definitions."""
import torch


def places(table, lens, starts, page_size, rows):
    """For each row (sequence, position), or None where no sequence has it."""
    out = [None] * rows
    for b in range(len(lens)):
        for t in range(max(0, int(starts[b])), min(rows, int(starts[b + 1]))):
            out[t] = (b, int(lens[b]) - int(starts[b + 1]) + t)
    return out


def quantise(x):
    """x [..., d] -> (codes, exponents), bytes: the smallest e >= 1 with max |x| <= 448 * 2^(e - 127); NaN where not finite."""
    x = x.double()
    m, e = torch.frexp((x.abs().amax(-1) / 448.0).clamp(min=2.0 ** -126))
    e = e - (m == 0.5).to(e.dtype)
    y = torch.ldexp(x, -e[..., None])
    step = torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 4
    y = torch.ldexp(torch.round(torch.ldexp(y, -step)), step)
    fine = torch.isfinite(x).all(-1)
    codes = torch.where(fine[..., None], y, 0.0).to(torch.float32).to(torch.float8_e4m3fn).view(torch.uint8)
    codes = torch.where(fine[..., None], codes, 0x7F).to(torch.uint8)
    # zeros keep the sign of what was rounded to them
    codes = torch.where((codes == 0) & torch.signbit(x), 0x80, codes.int()).to(torch.uint8)
    return codes, torch.where(fine, e + 127, 255).to(torch.uint8)


def values(codes, exponents):
    return codes.view(torch.float8_e4m3fn).double() * torch.exp2(exponents.double() - 127.0)[..., None]


def dense(cache, i):
    """Keys (0) or values (1) of a cache [pages, kv, page_size, d], as numbers."""
    x = cache[i].cpu()
    return values(x.view(torch.uint8), cache[2 + i].cpu()) if len(cache) == 4 else x.double()


def attention(q, cache, table, lens, starts, scale, window=None):
    """-> (o, bound): bound is the sum of weight * |value|, and the largest scale * sum |q| |k| and |value| that a row meets."""
    k, v = dense(cache, 0), dense(cache, 1)
    T, heads, d = q.shape
    kv, page = k.shape[1], k.shape[2]
    o = torch.zeros(T, heads, d, dtype=torch.float64)
    mean = torch.zeros_like(o)
    size = torch.zeros(T, heads, dtype=torch.float64)
    most = torch.zeros(T, heads, dtype=torch.float64)
    q = q.cpu().double()
    for t, place in enumerate(places(table, lens, starts, page, T)):
        if place is None or place[1] < 0:
            continue
        b, pos = place
        j = torch.arange(max(0, pos + 1 - window) if window else 0, pos + 1)
        rows = table[b].cpu().long()[j // page]
        kj, vj = k[rows, :, j % page], v[rows, :, j % page]  # [keys, kv, d]
        for h in range(heads):
            g = h * kv // heads
            x = (kj[:, g] @ q[t, h]) * scale
            w = torch.softmax(x, 0)
            o[t, h] = w @ vj[:, g]
            mean[t, h] = w @ vj[:, g].abs()
            size[t, h] = ((kj[:, g].abs() @ q[t, h].abs()) * scale).max()
            most[t, h] = vj[:, g].abs().max()
    return o, (mean, size, most)


def verify(probs, drafts, u, draft_probs=None, counts=None):
    B, K = drafts.shape
    V = probs.shape[2]
    tokens = torch.full((B, K + 1), -1, dtype=torch.int64)
    n_out = torch.zeros(B, dtype=torch.int32)
    clean = lambda x: torch.where(torch.isfinite(x) & (x > 0), x, 0.0)
    probs = clean(probs)
    draft_probs = clean(draft_probs) if draft_probs is not None else None
    for b in range(B):
        mine = K if counts is None else min(max(int(counts[b]), 0), K)
        n = 0
        while n < mine:
            x = int(drafts[b, n])
            if not 0 <= x < V:
                break
            qx = 1.0 if draft_probs is None else float(draft_probs[b, n, x])
            if not float(u[b, n]) * qx < float(probs[b, n, x]):
                break
            tokens[b, n] = x
            n += 1
        w = p = probs[b, n].double()
        if n < mine:
            x = int(drafts[b, n])
            if draft_probs is not None:
                w = clean(p - draft_probs[b, n].double())
            elif 0 <= x < V:
                w = w.clone()
                w[x] = 0.0
            if not float(w.sum()) > 0:
                w = p
        if float(w.sum()) > 0:
            sums = w.cumsum(0)
            above = (sums > float(u[b, K]) * float(sums[-1])).nonzero()
            tokens[b, n] = int(above[0]) if len(above) else int((w > 0).nonzero()[-1])
        n_out[b] = n + 1
    return tokens, n_out


def tolerance(o, bound, dtype, d, eight_bit, keys):
    """How far a result of `dtype` may be from the 64-bit one, per number.

    Half a step of the output; half a step of each weight as the products take it (their 16-bit type: of q, or fp16 over an 8-bit
    cache), which moves the result by that much of the sum of weight * |value|, and the sum of weights in 32 bits by the rest; scores in
    32 bits: (d + 4) additions and products, each off by half a step (2^-24) of at most scale * sum |q| |k|, in numerator and sum of
    the weights, and 2^-21 for two exponentials; fp16 weights, the largest of them 1 or more, are off by up to half of its
    smallest number (2^-25) each.  Over an 8-bit cache a weight carries its value's scale, the sizes of a row's largest number
    and of its scale being less than 2^9 apart where 448 is not reached by a factor below 2: 2^-24 of the largest value; the scale's
    exponent (below 2^7) is added to the score, off by half a step of their sum (2^-17 with what the sum reaches)."""
    mean, size, most = bound
    eps = torch.finfo(dtype).eps
    weights = torch.finfo(torch.float16).eps if eight_bit else eps
    score = (2 * (d + 4) * 2.0 ** -24 * size + 2.0 ** -21 + (2.0 ** -16 if eight_bit else 0.0))[..., None]
    tol = eps / 2 * o.abs() + (weights / 2 + 2 * score + 2.0 ** -20) * mean
    if eight_bit or dtype == torch.float16:
        tol = tol + keys * 2.0 ** (-24 if eight_bit else -25) * most[..., None]
        tol = tol + 2.0 ** -25  # half of fp16's smallest number, of results that are smaller still
    return tol * (1 + eps)
