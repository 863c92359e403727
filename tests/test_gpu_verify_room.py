"""Results of a verification in the room between the probabilities of two sequences, and behind the last."""
import pytest
import torch

from oracle import tree

from test_gpu_tree import _forest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("behind", [False, True])
def test_results_beside_the_probabilities(behind):
    from fractaltensor_b200 import ops
    from fractaltensor_b200._lib import check, lib
    B, N, V = 2, 3, 50
    probs, tokens, parents, u = _forest(B, N, V, 1)
    room = torch.zeros(4, 256, device="cuda")  # a sequence's 150 numbers, then 106 of others
    for b in range(B):
        room[b, : N * V] = probs[b].flatten().cuda()
    at = room[1, N * V + 2:] if behind else room[0, N * V + 2:]  # (on an 8-byte boundary)
    out, path, counts = at[:12].view(torch.int64).view(B, N), at[12:18].view(torch.int32).view(B, N), at[18:20].view(torch.int32)
    ws = ops.workspace(room.device)
    tokens, parents, u = tokens.cuda(), parents.cuda(), u.cuda()
    check(lib.ftb_verify_tree(room.data_ptr(), 256, V, tokens.data_ptr(), parents.data_ptr(), u.data_ptr(), out.data_ptr(), path.data_ptr(), counts.data_ptr(),
                              B, N, V, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream), "ftb_verify_tree")
    torch.cuda.synchronize()
    for x, y in zip((out, path, counts), tree.verify(probs, tokens.cpu(), parents.cpu(), u.cpu())):
        assert torch.equal(x.cpu(), y)
