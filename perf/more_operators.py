"""Performance cases of trees of drafted tokens over a paged cache, and of eviction from it by accumulated attention weight.

A case's "op" names the operator:

    attend     ops.paged_attention with tree=    the tokens of drafted trees over the cache; "mask": behind ops.tree_mask,
                                                 as in a model's first layer, the others take the mask as it is
    verify     ops.verify_tree                   drafted trees against the target's probabilities
    keep       ops.paged_cache_keep              the cache's rows of the accepted paths, one behind the other
    weigh      ops.paged_attention_weights       what new tokens attend to, added to a weight for each key in the cache
    evict      ops.paged_cache_evict             the keys of the largest weights and the latest ones, in pages of their own or
                                                 ("in_place") the same

`run` computes a case with plain torch operations, or (`own`) by the framework's calls.  Both get the same
buffers: cache pages [pages, kv_heads, page_size, d], for an 8-bit cache an exponent byte a row, weights (fp32) a number a
row.  A batch is described by `starts` (first row of each sequence's new tokens), `lens` (keys of each sequence, the
new ones included) and `table` (its pages).  Token 0 of a tree is the last one that is certain.
"""
import math
import random

import torch

own = False

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # A single user's tree behind a short conversation, mask and all: latency.
        {"name": "attend tree one bf16", "op": "attend", "dtype": "bf16", "cache": "bf16", "B": 1, "N": 25, "len_lo": 777, "len_hi": 777,
         "kv": 8, "group": 4, "d": 128, "page": 16, "mask": True},
        # Trees of a small model's batch, of an odd size, heads in threes.
        {"name": "attend trees f16 d64", "op": "attend", "dtype": "f16", "cache": "f16", "B": 37, "N": 13, "len_lo": 33, "len_hi": 6000,
         "kv": 4, "group": 3, "d": 64, "page": 32, "mask": True},
        # A full server: trees of 33 tokens behind long sequences, 8-bit cache, one of many layers.
        {"name": "attend trees e4m3", "op": "attend", "dtype": "bf16", "cache": "e4m3", "B": 32, "N": 33, "len_lo": 1000, "len_hi": 16000,
         "kv": 8, "group": 8, "d": 128, "page": 64, "mask": False},
        # One user's tree over the vocabulary.
        {"name": "verify tree one", "op": "verify", "B": 1, "N": 25, "V": 49152},
        # A server's trees over a large vocabulary of an odd size.
        {"name": "verify trees batch", "op": "verify", "B": 60, "N": 33, "V": 130001},
        # The accepted path of one user's tree: nothing but latency.
        {"name": "keep path one bf16", "op": "keep", "dtype": "bf16", "cache": "bf16", "B": 1, "N": 25, "len_lo": 802, "len_hi": 802,
         "kv": 8, "d": 128, "page": 16, "weights": False},
        # The accepted paths of a server's trees, 8-bit cache, with the keys' weights.
        {"name": "keep paths e4m3", "op": "keep", "dtype": "bf16", "cache": "e4m3", "B": 128, "N": 61, "len_lo": 300, "len_hi": 5000,
         "kv": 8, "d": 128, "page": 64, "weights": True},
        # A single user's token, keys of a short conversation.
        {"name": "weigh one bf16", "op": "weigh", "dtype": "bf16", "cache": "bf16", "B": 1, "n_lo": 1, "n_hi": 1, "len_lo": 777,
         "len_hi": 777, "kv": 8, "group": 4, "d": 128, "page": 16, "window": 0},
        # A decoding step of an ordinary batch, sequences of very different lengths.
        {"name": "weigh decode bf16", "op": "weigh", "dtype": "bf16", "cache": "bf16", "B": 64, "n_lo": 1, "n_hi": 1, "len_lo": 33,
         "len_hi": 8000, "kv": 8, "group": 4, "d": 128, "page": 16, "window": 0},
        # A chunk of a long prompt behind what is in an 8-bit cache already: matrix products and exponentials.
        {"name": "weigh chunk e4m3", "op": "weigh", "dtype": "f16", "cache": "e4m3", "B": 1, "n_lo": 2048, "n_hi": 2048, "len_lo": 16384,
         "len_hi": 16384, "kv": 8, "group": 4, "d": 128, "page": 64, "window": 0},
        # One long document down to a fraction of itself, in its own pages.
        {"name": "evict one long e4m3", "op": "evict", "dtype": "bf16", "cache": "e4m3", "B": 1, "len_lo": 100001, "len_hi": 100001, "kv": 4,
         "d": 128, "page": 128, "keep": 8192, "recent": 1024, "in_place": True},
        # A batch down to what its share of memory holds, into other pages; some sequences are short enough as they are.
        {"name": "evict batch bf16", "op": "evict", "dtype": "bf16", "cache": "bf16", "B": 48, "len_lo": 1500, "len_hi": 9000, "kv": 8,
         "d": 128, "page": 16, "keep": 2048, "recent": 257, "in_place": False},
    ]


# ------------------------------------------------------------------------------- more of the same ranges
def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "verify", "keep", "weigh", "weigh", "evict"])
    if op == "verify":
        V, N = _spread(rng, 1000, 150000), rng.randint(1, 64)
        return {"op": op, "B": _spread(rng, 1, max(1, min(128, 250000000 // (V * N)))), "N": N, "V": V}
    dtype = rng.choice(["f16", "bf16"])
    c = {"op": op, "dtype": dtype, "cache": dtype if rng.random() < 0.5 else "e4m3", "B": _spread(rng, 1, 64), "kv": rng.choice([1, 2, 3, 4, 5, 8]),
         "d": rng.choice([64, 128, 128]), "page": rng.choice([16, 32, 64, 128])}
    if op in ("attend", "weigh"):
        c["group"] = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 16])
    rows = c["B"] * c["kv"] * c.get("group", 1)
    if op == "attend":
        c.update(N=_spread(rng, 1, 100), mask=rng.random() < 0.5)
        most = 130000000 // (rows * c["N"])
    elif op == "keep":
        c.update(N=_spread(rng, 1, 100), weights=rng.random() < 0.5)
        most = 3000000 // rows
    elif op == "weigh":
        c["n_hi"] = 1 if rng.random() < 0.4 else _spread(rng, 2, max(3, min(2048, 60000 // rows)))
        c["n_lo"] = max(1, c["n_hi"] // rng.choice([1, 2, 5]))
        c["window"] = 0
        most = min(3000000 // (c["B"] * c["kv"]), 250000000 // (rows * c["n_hi"]))
    else:
        most = 6000000 // rows
    least = c.get("N", c.get("n_hi", 1))
    c["len_hi"] = max(least, _spread(rng, 16, max(20, min(40000, most))))
    c["len_lo"] = max(least, c["len_hi"] // rng.choice([1, 2, 10, 50]))
    if op == "weigh" and rng.random() < 0.25:
        c["window"] = _spread(rng, 1, c["len_hi"])
    if op == "evict":
        c["keep"] = _spread(rng, 1, c["len_hi"])
        c.update(recent=rng.randint(0, c["keep"]), in_place=rng.random() < 0.5)
    return c


def _random(case):
    return random.Random(" ".join("%s" % case[k] for k in sorted(case) if k not in ("name", "op", "mask", "weights", "in_place")))


def _batch(case):
    """Lengths and numbers of new tokens of the case's sequences: the same for every seed."""
    r = _random(case)
    lens = [r.randint(case["len_lo"], case["len_hi"]) for _ in range(case["B"])]
    if "N" in case:
        return lens, [case["N"]] * case["B"]
    if case["op"] == "evict":
        return lens, [0] * case["B"]
    return lens, [r.randint(case["n_lo"], case["n_hi"]) for _ in lens]


def _trees(case):
    """Parents of each sequence's tree, [-1, ..]: a token comes behind its parent, early ones have more children."""
    r = _random(case)
    return [[-1] + [int(i * r.random() ** 1.5) for i in range(1, case["N"])] for _ in range(case["B"])]


def _path_to(parents, i):
    path = [i]
    while parents[path[0]] >= 0:
        path.insert(0, parents[path[0]])
    return path


def _paths(case):
    """An accepted path of each tree: from token 0 to a random one."""
    r = _random(case)
    return [_path_to(parents, r.randrange(case["N"])) for parents in _trees(case)]


# --------------------------------------------------------------------------------------------- inputs
def _quantise(x):
    """x [..., d] -> e4m3 codes (bytes) and exponents [...] (bytes): x = code * 2^(exponent - 127), |code| <= 448."""
    x = x.float()
    bits = x.abs().amax(-1).view(torch.int32)
    e = (bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()
    e = e.clamp(1, 254)
    inverse = ((254 - e.clamp(max=253)) << 23).view(torch.float32)
    return (x * inverse[..., None]).to(torch.float8_e4m3fn), e.to(torch.uint8)


def _keys(g, shape, dtype):
    """Numbers as keys and values have them: some channels larger than others, some tokens too."""
    x = torch.randn(shape, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(shape[-1], generator=g, device="cuda"))
    x *= torch.exp(0.3 * torch.randn(shape[:-1], generator=g, device="cuda"))[..., None]
    return x.to(dtype)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _padded(rows, width):
    return _ints([list(r) + [-1] * (width - len(r)) for r in rows])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    B = case["B"]
    if "N" in case:
        s["parents"] = _ints(_trees(case))
    if case["op"] == "verify":
        N, V = case["N"], case["V"]
        logits = 3.0 * torch.randn(B, N, V, generator=g, device="cuda")
        s["probs"] = torch.softmax(logits, -1)
        # a token's children: what a draft model thinks likeliest behind it, nearly what the target thinks
        rank = [[sum(p == parents[i] for p in parents[:i]) for i in range(N)] for parents in _trees(case)]
        likeliest = (logits + 0.7 * torch.randn(B, N, V, generator=g, device="cuda")).topk(1 + max(map(max, rank)), -1).indices
        b = torch.arange(B, device="cuda")[:, None]
        s["tokens"] = likeliest[b, s["parents"].clamp(min=0).long(), _ints(rank).long()]
        s["u"] = torch.rand(B, N, generator=g, device="cuda")
        return s
    lens, new = _batch(case)
    kv, d, page, dtype = case["kv"], case["d"], case["page"], _DTYPES[case["dtype"]]
    into = [min(n, case["keep"]) for n in lens] if case["op"] == "evict" and not case["in_place"] else []
    counts = [-(-n // page) for n in lens + into]
    pages = sum(counts) + 3
    order = torch.randperm(pages, generator=g, device="cuda").int()
    has = torch.arange(max(counts), device="cuda")[None, :] < _ints(counts)[:, None]
    tables = torch.full(has.shape, -1, dtype=torch.int32, device="cuda")
    tables[has] = order[: sum(counts)]
    s["table"], s["into"] = tables[:B], tables[B:, : max(counts[B:])].contiguous() if into else None
    s["lens"] = _ints(lens)
    s["starts"] = _ints([sum(new[:i]) for i in range(B + 1)])
    k, v = (_keys(g, (pages, kv, page, d), dtype) for _ in range(2))
    s["cache"] = (k, v)
    if case["cache"] == "e4m3":
        (kc, ke), (vc, ve) = _quantise(k), _quantise(v)
        s["cache"] = (kc, vc, ke, ve)
    s["scale"] = 1.0 / math.sqrt(d)
    if case["op"] in ("weigh", "evict", "keep"):  # of few keys much, of most of them little
        s["weights"] = torch.exp(2.0 * torch.randn(pages, kv, page, generator=g, device="cuda"))
    if case["op"] == "weigh":  # what about as many tokens in front have left
        s["weights"] *= 0.1 * case["group"] * case["n_hi"] / case["len_hi"]
    if case["op"] == "keep":
        paths = _paths(case)
        s["kept"], s["counts"], s["first"] = _padded(paths, case["N"]), _ints([len(p) for p in paths]), s["lens"] - case["N"]
        if not case["weights"]:
            s["weights"] = None
    if case["op"] in ("attend", "weigh"):
        # what the product in front gives: queries, keys and values of a token side by side
        s["rows"], s["most_new"] = sum(new), max(new)
        heads = kv * case["group"]
        qkv = torch.randn(s["rows"], (heads + 2 * kv) * d, generator=g, device="cuda").to(dtype)
        s["q"] = qkv[:, : heads * d].unflatten(1, (heads, d))
    if case["op"] == "attend":
        s["tree"] = _mask(s["parents"]).flatten(0, 1)
    if case["op"] == "weigh":  # from the attention in front
        s["lse"] = _unpadded(s, torch.logsumexp(_scores(s, _sees(s)), -1))
    return s


# ---------------------------------------------------------------------------------------- plain forms
def _places(s):
    """Sequence, number in it and position of every row of new tokens."""
    rows = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["starts"][1:].contiguous(), rows, right=True)
    first = s["starts"][seq]
    return seq, (rows - first).long(), s["lens"][seq] - (s["starts"][seq + 1] - first) + (rows - first)


def _whole(s, i):
    """Keys (0) or values (1) of all sequences, padded: fp32 [B, kv, W * page, d]."""
    table = s["table"].clamp(min=0).long()
    x = s["cache"][i]
    if len(s["cache"]) == 4:
        x = x.view(torch.uint8)[table].view(torch.float8_e4m3fn).float() * (s["cache"][2 + i][table].int() << 23).view(torch.float32)[..., None]
    else:
        x = x[table].float()
    return x.transpose(1, 2).flatten(2, 3)


def _sees(s):
    """Which keys a token sees: [B, most_new, W * page]."""
    seq, i, pos = _places(s)
    at = torch.full((s["B"], s["most_new"]), -1, dtype=pos.dtype, device="cuda")
    at[seq, i] = pos
    key = torch.arange(s["table"].shape[1] * s["page"], device="cuda")
    sees = key <= at[..., None]
    if s["op"] == "weigh":
        return sees & (key > at[..., None] - s["window"]) if s["window"] else sees
    j = key - (s["lens"] - s["N"])[:, None, None]  # of a key among the new ones
    mask = s["tree"].unflatten(0, (s["B"], s["N"]))
    word = mask.gather(2, (j.clamp(min=0, max=s["N"] - 1) // 32).expand(-1, s["N"], -1))
    return sees & ((j < 0) | ((word >> (j % 32).int()) & 1).bool())


def _scores(s, sees):
    """scale * q . k of all sequences, padded, -inf where a token does not see the key: [B, kv, most_new * group, W * page]."""
    seq, i, _ = _places(s)
    q = torch.zeros(s["B"], s["most_new"], s["kv"] * s["group"], s["d"], device="cuda")
    q[seq, i] = s["q"].float()
    q = q.unflatten(2, (s["kv"], s["group"])).permute(0, 2, 1, 3, 4).flatten(2, 3)
    x = (q @ _whole(s, 0).transpose(2, 3)).mul_(s["scale"])
    return x.masked_fill_(~sees.repeat_interleave(s["group"], 1)[:, None], -math.inf)


def _unpadded(s, x):
    """[B, kv, most_new * group, ..] -> [rows, heads, ..]."""
    seq, i, _ = _places(s)
    x = x.unflatten(2, (s["most_new"], s["group"])).transpose(1, 2).flatten(2, 3)
    return x[seq, i]


def _attend(s):
    x = _scores(s, _sees(s))
    x = torch.exp(x.sub_(x.amax(-1, keepdim=True).clamp(min=-3e38)))
    total = x.sum(-1, keepdim=True)
    key = torch.arange(x.shape[-1], device="cuda")
    v = _whole(s, 1).masked_fill_((key >= s["lens"][:, None])[:, None, :, None], 0.0)
    return _unpadded(s, (x @ v) / torch.where(total > 0, total, 1.0)).to(s["q"].dtype)


def _mask(parents):
    """[B, N] -> 32-bit words [B, N, ceil(N / 32)]: bit j of token i is 1 if j is i or one of the tokens on the way to it."""
    B, N = parents.shape
    i = torch.arange(N, device="cuda")
    to = (parents[..., None] == i).float()  # one step up
    on = torch.eye(N, device="cuda").expand(B, N, N)
    for _ in range(max(1, N.bit_length())):  # up to 2, 4, 8, .. steps
        on = ((on + on @ to) > 0).float()
        to = to @ to
    bits = torch.nn.functional.pad(on.long(), (0, -N % 32)).unflatten(2, (-1, 32)) << torch.arange(32, device="cuda")
    word = bits.sum(-1)
    return torch.where(word >= 2 ** 31, word - 2 ** 32, word).int()


def _verify(s):
    B, N, V = s["B"], s["N"], s["V"]
    tokens, parents, u = s["tokens"], s["parents"].long(), s["u"].double()
    b = torch.arange(B, device="cuda")
    p = s["probs"][b[:, None], parents.clamp(min=0), tokens].double()
    i = torch.arange(N, device="cuda")
    again = ((parents[:, :, None] == parents[:, None, :]) & (tokens[:, :, None] == tokens[:, None, :]) & (i[:, None] > i)).any(-1)
    p = torch.where(again, 0.0, p)
    at = torch.zeros(B, dtype=torch.long, device="cuda")
    rest = torch.ones(B, dtype=torch.float64, device="cuda")
    on = torch.zeros(B, N, dtype=torch.bool, device="cuda")
    on[:, 0] = True
    for c in range(1, N):  # a token comes behind its parent: what is drafted behind the one that the path is at
        asked = parents[:, c] == at
        taken = asked & (u[:, c] * rest < p[:, c])
        on[:, c] = taken
        at = torch.where(taken, c, at)
        rest = torch.where(taken, 1.0, torch.where(asked, (rest - p[:, c]).clamp(min=0.0), rest))
    w = s["probs"][b, at].double()
    refused = torch.zeros(B, V, device="cuda").scatter_add(1, tokens, (parents == at[:, None]).float()) > 0
    w = torch.where(refused, 0.0, w)
    w = torch.where(w.sum(1, keepdim=True) > 0, w, s["probs"][b, at].double())
    total = w.cumsum(1)
    token = (total <= u[:, :1] * total[:, -1:]).sum(1).clamp(max=V - 1)
    n = on.sum(1)
    path = torch.where(on, i, N).sort(1).values
    path = torch.where(path < N, path, -1)
    out = torch.where(path[:, 1:] >= 0, tokens.gather(1, path[:, 1:].clamp(min=0)), -1)
    out = torch.cat([out, torch.full((B, 1), -1, device="cuda")], 1)
    out[b, n - 1] = token
    return out, path.int(), n.int()


def _move(s, kept, counts, first, into):
    """Rows first + kept[.., i], i < counts, to first + i: kept [B, kv, K]."""
    page, K = s["page"], kept.shape[2]
    i = torch.arange(K, device="cuda")
    b, h, i = torch.nonzero((i < counts[:, None, None]) & (kept >= 0), as_tuple=True)
    src, dst = first[b].long() + kept[b, h, i], first[b].long() + i
    src_page, dst_page = s["table"][b, src // page].long(), into[b, dst // page].long()
    planes = list(s["cache"]) + ([s["weights"]] if s["weights"] is not None else [])
    for x in planes:
        x = x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x
        x[dst_page, h, dst % page] = x[src_page, h, src % page]
    return planes


def _weigh(s):
    seq, i, _ = _places(s)
    x = _scores(s, _sees(s))
    lse = torch.zeros(s["B"], s["most_new"], s["kv"] * s["group"], device="cuda")
    lse[seq, i] = s["lse"]
    lse = lse.unflatten(2, (s["kv"], s["group"])).permute(0, 2, 1, 3).flatten(2, 3)
    total = torch.exp(x.sub_(lse[..., None])).sum(2)  # [B, kv, W * page]
    key = torch.arange(total.shape[-1], device="cuda")
    new = s["starts"][1:] - s["starts"][:-1]
    b, j = torch.nonzero(key < s["lens"][:, None], as_tuple=True)
    page, off = s["table"][b, j // s["page"]].long(), j % s["page"]
    before = torch.where((j >= (s["lens"] - new)[b])[:, None], 0.0, s["weights"][page, :, off])
    s["weights"][page, :, off] = before + total[b, :, j]
    return s["weights"]


def _evict(s):
    B, kv, keep, recent, page = s["B"], s["kv"], s["keep"], s["recent"], s["page"]
    key = torch.arange(s["table"].shape[1] * page, device="cuda")
    w = s["weights"][s["table"].clamp(min=0).long()].transpose(1, 2).flatten(2, 3)
    lens = s["lens"][:, None]
    w = torch.where((key >= lens - recent)[:, None], math.inf, w)  # the latest ones first of all
    w = torch.where((key >= lens)[:, None], -math.inf, w)
    kept = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :keep]
    kept = torch.nn.functional.pad(kept, (0, keep - kept.shape[-1]), value=len(key))
    kept = torch.where(kept < lens[..., None], kept, len(key)).sort(-1).values
    kept = torch.where(kept < len(key), kept, -1)
    now = s["lens"].clamp(max=keep)
    planes = _move(s, kept, now, torch.zeros_like(s["lens"]), s["table"] if s["in_place"] else s["into"])
    return now, kept.int(), planes


def run(s):
    if own:
        from fractaltensor_b200 import ops
        if s["op"] == "verify":
            return ops.verify_tree(s["probs"], s["tokens"], s["parents"], s["u"])
        if s["op"] == "attend":
            tree = ops.tree_mask(s["parents"]) if s["mask"] else None
            o = ops.paged_attention(s["q"], s["cache"], s["table"], s["lens"], s["starts"], scale=s["scale"],
                                    tree=tree.flatten(0, 1) if s["mask"] else s["tree"])
            return (tree, o) if s["mask"] else o
        if s["op"] == "weigh":
            ops.paged_attention_weights(s["q"], s["cache"], s["weights"], s["lse"], s["table"], s["lens"], s["starts"],
                                        scale=s["scale"], window=s["window"] or None)
            return s["weights"]
        if s["op"] == "keep":
            ops.paged_cache_keep(s["cache"], s["kept"], s["counts"], s["table"], s["first"], weights=s["weights"])
            return list(s["cache"]) + ([s["weights"]] if s["weights"] is not None else [])
        now, kept = ops.paged_cache_evict(s["cache"], s["weights"], s["table"], s["lens"], s["keep"], s["recent"], into=s["into"])
        return now, kept, list(s["cache"]) + [s["weights"]]
    if s["op"] == "verify":
        return _verify(s)
    if s["op"] == "attend":
        tree = _mask(s["parents"]) if s["mask"] else None
        return (tree, _attend(dict(s, tree=tree.flatten(0, 1)))) if s["mask"] else _attend(s)
    if s["op"] == "weigh":
        return _weigh(s)
    if s["op"] == "keep":
        _move(s, s["kept"][:, None].expand(-1, s["kv"], -1), s["counts"], s["first"], s["table"])
        return list(s["cache"]) + ([s["weights"]] if s["weights"] is not None else [])
    now, kept, _ = _evict(s)
    return now, kept, list(s["cache"]) + [s["weights"]]


# ------------------------------------------------------------------------------------------ the floors
def work(case):
    B = case["B"]
    if case["op"] == "verify":  # a row of the token that the path ends with; tokens, parents, random numbers and their probabilities; results
        N, V = case["N"], case["V"]
        return {"bytes": B * (V * 4 + N * 20 + N * 12 + 4), "flops": B * V * 3}
    lens, new = _batch(case)
    kv, d = case["kv"], case["d"]
    row = d + 1 if case["cache"] == "e4m3" else 2 * d  # bytes of a key or value of a head
    if case["op"] == "keep":  # rows that change their place
        moved = sum(i != at for path in _paths(case) for i, at in enumerate(path)) * kv
        return {"bytes": max(1, 2 * moved * (2 * row + (4 if case["weights"] else 0)) + B * case["N"] * 4), "flops": 0}
    if case["op"] == "evict":  # the weights, and the rows that are kept
        kept = sum(min(n, case["keep"]) for n in lens if n > case["keep"] or not case["in_place"]) * kv
        return {"bytes": sum(lens) * kv * 4 + kept * (2 * (2 * row + 4) + 4) + B * 8, "flops": 0}
    heads = kv * case["group"]
    if case["op"] == "attend":
        N = case["N"]
        seen = sum(len(_path_to(parents, i)) for parents in _trees(case) for i in range(N))
        pairs = sum(n - N for n in lens) * N + seen
        mask = B * N * -(-N // 32) * 4 + (B * N * 4 if case["mask"] else 0)
        return {"bytes": sum(lens) * kv * 2 * row + sum(new) * heads * d * 4 + mask, "flops": 4 * pairs * heads * d}
    w = case["window"] or max(lens)
    pairs = sum(min(n - m + i + 1, w) for n, m in zip(lens, new) for i in range(m))
    keys = sum(min(n, w + m - 1) for n, m in zip(lens, new))
    return {"bytes": keys * kv * (row + 8) + sum(new) * heads * (2 * d + 4), "flops": 2 * pairs * heads * d}


# ----------------------------------------------------------------------- the definitions in 64 bits
def _of_sequence(s, i, b, first, last):
    """Positions first .. last - 1 of sequence b from the keys (0) or values (1): 64 bits [n, kv, d]."""
    at = torch.arange(first, last, device="cuda")
    page, off = s["table"][b, at // s["page"]].long(), at % s["page"]
    if len(s["cache"]) == 2:
        return s["cache"][i][page, :, off].double()
    codes = s["cache"][i].view(torch.uint8)[page, :, off].view(torch.float8_e4m3fn).double()
    return codes * torch.exp2(s["cache"][2 + i][page, :, off].double() - 127.0)[..., None]


def _exact_attend(case, s):
    lens, N, trees = _batch(case)[0], case["N"], _trees(case)
    o = torch.zeros(s["rows"], case["kv"] * case["group"], case["d"], dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        k, v = _of_sequence(s, 0, b, 0, n), _of_sequence(s, 1, b, 0, n)
        hidden = torch.zeros(N, n, dtype=torch.bool)
        hidden[:, n - N:] = True
        for i in range(N):
            hidden[i, [n - N + j for j in _path_to(trees[b], i)]] = False
        hidden = hidden.cuda()
        for h in range(case["kv"] * case["group"]):
            x = s["q"][b * N: (b + 1) * N, h].double() @ k[:, h // case["group"]].T * s["scale"]
            o[b * N: (b + 1) * N, h] = torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ v[:, h // case["group"]]
    return (None, o) if case["mask"] else o


def _exact_weights(case, s):
    lens, new = _batch(case)
    ends, weights = s["starts"].tolist(), s["weights"].double()
    for b, (n, m) in enumerate(zip(lens, new)):
        k = _of_sequence(s, 0, b, 0, n)
        key, pos = torch.arange(n, device="cuda"), torch.arange(n - m, n, device="cuda")[:, None]
        hidden = key > pos
        if case["window"]:
            hidden = hidden | (key <= pos - case["window"])
        page, off = s["table"][b, key // case["page"]].long(), key % case["page"]
        weights[page[n - m:], :, off[n - m:]] = 0.0
        for h in range(case["kv"] * case["group"]):
            x = s["q"][ends[b]: ends[b + 1], h].double() @ k[:, h // case["group"]].T * s["scale"]
            p = torch.exp(x - s["lse"][ends[b]: ends[b + 1], h, None].double()).masked_fill(hidden, 0.0)
            weights[page, h // case["group"], off] += p.sum(0)
    return weights


def exact(case, seed):
    if case["op"] == "verify":
        return None  # whole numbers, and the plain form computes in 64 bits
    s = prepare(case, seed)
    if case["op"] == "attend":
        return _exact_attend(case, s)
    if case["op"] == "weigh":
        return _exact_weights(case, s)
    # copies: what row goes where, one sequence at a time
    planes = list(s["cache"]) + ([s["weights"]] if s["weights"] is not None else [])
    before = [x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x for x in planes]
    after = [x.clone() for x in before]
    page, lens, kept = case["page"], _batch(case)[0], []
    if case["op"] == "keep":
        kept = [[path] * case["kv"] for path in _paths(case)]
    else:
        weights = s["weights"].cpu()
        for b, n in enumerate(lens):
            w = weights[s["table"][b].clamp(min=0).cpu().long()].transpose(0, 1).flatten(1)[:, : max(0, n - case["recent"])].numpy()
            order = (-w).argsort(axis=1, kind="stable")[:, : max(0, case["keep"] - case["recent"])]
            kept.append([sorted(o.tolist()) + list(range(max(0, n - case["recent"]), n)) for o in order])
    into = s["into"] if s["into"] is not None else s["table"]
    for b, heads in enumerate(kept):
        first = int(lens[b]) - case["N"] if case["op"] == "keep" else 0
        for h, rows in enumerate(heads):
            src = torch.tensor(rows, device="cuda") + first
            dst = torch.arange(first, first + len(rows), device="cuda")
            for x, y in zip(before, after):
                y[into[b, dst // page].long(), h, dst % page] = x[s["table"][b, src // page].long(), h, src % page]
    after = [(y.view(torch.float8_e4m3fn) if x.dtype == torch.float8_e4m3fn else y).double() if x.dtype != torch.uint8 else None
             for x, y in zip(planes, after)]
    return after if case["op"] == "keep" else (None, None, after)
