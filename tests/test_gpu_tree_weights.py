"""Trees of drafts beside eviction: the path's rows are what new tokens attend to, once the path has been kept."""
import math

import pytest
import torch

from oracle import tree

from test_gpu_paged import BF16, E4M3, _batch, _full_cache, _numbers
from test_gpu_tree import _forest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eight_bit", [False, True])
def test_weights_of_paths_and_eviction(eight_bit):
    from fractaltensor_b200 import ops
    kv, group, d, page, B, N, V = 2, 4, 64, 16, 3, 17, 200
    before = [70, 5, 123]
    lens = [n + N for n in before]
    table, ln, st, pages = _batch([N] * B, lens, page)
    cache = _full_cache(pages, kv, page, d, E4M3 if eight_bit else BF16, 3)
    probs, tokens, parents, u = _forest(B, N, V, 4)
    weights = torch.rand(pages, kv, page, generator=torch.Generator().manual_seed(1)).cuda()
    q = _numbers((B * N, kv * group, d), BF16, 5).cuda()
    scale = 1.0 / math.sqrt(d)
    lse = torch.empty(B * N, kv * group, device="cuda")
    device = (table.cuda(), ln.cuda(), st.cuda())
    ops.paged_attention(q, cache, *device, scale=scale, tree=ops.tree_mask(parents.cuda()).flatten(0, 1), lse=lse)
    out, path, counts = ops.verify_tree(probs.cuda(), tokens.cuda(), parents.cuda(), u.cuda())
    first = torch.tensor(before, dtype=torch.int32)
    ops.paged_cache_keep(cache, path, counts, device[0], first=first.cuda(), weights=weights)
    ops.check_status()
    n = counts.tolist()
    assert max(n) > 2
    rows = torch.cat([b * N + path[b, : n[b]].long() for b in range(B)])
    now, starts = first + counts.cpu(), torch.tensor([sum(n[:b]) for b in range(B + 1)], dtype=torch.int32)
    old = weights.clone()
    ops.paged_attention_weights(q[rows], cache, weights, lse[rows], device[0], now.cuda(), starts.cuda(), scale=scale)
    ops.check_status()
    # what the path's tokens see of the cache as it is now is what they saw of the tree: their logarithms are those of a plain call
    _, bound, plain = tree.attention(q[rows], cache, table, now, starts, scale)
    assert bool(((plain - lse[rows].double().cpu()).abs() <= tree.lse_tolerance(plain, bound[1], d, eight_bit, max(lens))).all())
    want, tol = tree.weights(old, q[rows], cache, lse[rows], table, now, starts, scale)
    assert bool(((weights.double().cpu() - want).abs() <= tol).all())
    keep, recent = 60, 10
    want_lens, want_kept = tree.choose(weights.cpu(), table, now.tolist(), keep, recent)
    got_lens, got_kept = ops.paged_cache_evict(cache, weights, device[0], now.cuda(), keep, recent)
    ops.check_status()
    assert torch.equal(got_lens.cpu(), want_lens) and torch.equal(got_kept.cpu(), want_kept)
