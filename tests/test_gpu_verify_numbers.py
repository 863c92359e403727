"""verify_drafts on numbers that are no probabilities: what is not positive and finite counts as 0, on either side."""
import pytest
import torch

from oracle import paged

INF, NAN = float("inf"), float("nan")

# (target row at the draft, draft's row, drafted token, u, u of the drawn token, expected tokens); a second target row [.25, .25, .5, 0]
CASES = [
    ([INF, 0.5, 0.5, 0.0], [0.1, 0.4, 0.5, 0.0], 0, 0.5, 0.0, [1, -1]),     # the target's infinity: 0, not taken; .1 is left of token 1
    ([0.0, 0.5, 0.5, 0.0], [-0.5, 0.5, 0.25, 0.0], 0, 0.9, 0.0, [2, -1]),   # 0 against a negative number: 0 < 0 is not
    ([-0.25, 0.5, 0.5, 0.0], [-0.5, 0.5, 0.25, 0.0], 0, 0.9, 0.0, [2, -1]),  # nor does -.25 weigh over -.5
    ([0.0, 0.5, 0.5, 0.0], [0.0, 0.7, -INF, 0.0], 1, 0.9, 0.3, [2, -1]),    # -inf in the draft's row: 0, and no infinite sum
    ([0.25, 0.5, 0.25, 0.0], [0.25, 0.7, INF, 0.0], 1, 0.9, 0.9, [2, -1]),  # +inf in it: 0
    ([0.25, 0.5, 0.25, 0.0], [NAN, 0.7, 0.5, 0.0], 1, 0.9, 0.9, [0, -1]),   # NaN in it: 0
    ([0.0, 0.5, 0.5, 0.0], [0.0, NAN, 0.25, 0.0], 1, 0.9, 0.0, [1, 0]),     # a draft that counts as 0: min(1, p / 0) is 1
    ([0.0, NAN, 0.5, 0.0], [0.0, 0.5, 0.25, 0.0], 1, 0.0, 0.0, [2, -1]),    # a target that does: not taken
    ([0.0, 0.5, 0.5, 0.0], [0.0, INF, 0.25, 0.0], 1, 0.9, 0.6, [1, 2]),
]


def _tensors(width):
    B, V = len(CASES), 4
    p, q = torch.zeros(B, 2, width), torch.zeros(B, 1, width)
    for b, (target, draft, *_) in enumerate(CASES):
        p[b, 0, :V], q[b, 0, :V] = torch.tensor(target), torch.tensor(draft)
        p[b, 1, :V] = torch.tensor([0.25, 0.25, 0.5, 0.0])
    drafts = torch.tensor([[c[2]] for c in CASES])
    u = torch.tensor([[c[3], c[4]] for c in CASES])
    want = torch.tensor([c[5] for c in CASES])
    return p, q, drafts, u, want, 1 + (want[:, 1] >= 0).int()


def test_oracle():
    p, q, drafts, u, want, counts = _tensors(4)
    got = paged.verify(p, drafts, u, q)
    assert torch.equal(got[0], want) and torch.equal(got[1], counts)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [4, 5001])  # a CTA a sequence, and a cluster
def test_kernel(width):
    from fractaltensor_b200 import ops
    p, q, drafts, u, want, counts = _tensors(width)
    got = ops.verify_drafts(p.cuda(), drafts.cuda(), u.cuda(), q.cuda())
    ops.check_status()
    assert torch.equal(got[0].cpu(), want) and torch.equal(got[1].cpu(), counts)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [700, 9001])
def test_kernel_like_the_oracle(V):
    from fractaltensor_b200 import ops
    B, K = 40, 3
    g = torch.Generator().manual_seed(5)
    p, q = torch.softmax(torch.randn(B, K + 1, V, generator=g), -1), torch.softmax(torch.randn(B, K, V, generator=g), -1)
    for x, bad in ((p, (NAN, INF, -INF, -0.5, 0.0)), (q, (NAN, INF, -INF, -0.5, 0.0))):
        for i, value in enumerate(bad):
            x.masked_fill_(torch.rand(x.shape, generator=g) < 0.05, value)
    drafts = torch.randint(0, V, (B, K), generator=g)
    u = torch.rand(B, K + 1, generator=g)
    want = paged.verify(p, drafts, u, q)
    got = ops.verify_drafts(p.cuda(), drafts.cuda(), u.cuda(), q.cuda())
    ops.check_status()
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
