"""DistillationLoss of values that are not numbers and of logits far from zero."""
import pytest
import torch

from neoml_b200 import ops

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _made(t, *shape, seed, std=2.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(t)


def _indices(rows, v, k):
    return (torch.arange(k, device="cuda", dtype=torch.int32) * (v // k) + torch.arange(rows, device="cuda", dtype=torch.int32)[:, None]) % v


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,v", [(5, 2003), (300, 1003), (2, 60001)])   # a block per row, a warp per row, a cluster per row
@pytest.mark.parametrize("k", [1, 8, 64, 100, 300, 1000])
def test_a_teacher_that_is_not_a_number(t, rows, v, k):
    """Wherever it is kept, such a row's loss and gradient say so; the other rows do not notice."""
    z, top, index = _made(t, rows, v, seed=1), _made(t, rows, k, seed=2), _indices(rows, v, k)
    want = ops.DistillationLoss(z, top, index)
    dloss = torch.ones(rows, device="cuda")
    grad = ops.DistillationLossBackward(dloss, z, top, index, want[1])
    for at in {0, 1 % k, k // 2, k - 1}:
        bad = top.clone()
        bad[1, at] = float("nan")
        loss, log_sum = ops.DistillationLoss(z, bad, index)
        others = torch.arange(rows, device="cuda") != 1
        assert loss[1].isnan() and torch.equal(loss[others], want[0][others]) and torch.equal(log_sum, want[1])
        got = ops.DistillationLossBackward(dloss, z, bad, index, log_sum)
        assert got[1].isnan().any() and torch.equal(got[others], grad[others])
    all_bad = top.clone()
    all_bad[1] = float("nan")
    assert ops.DistillationLoss(z, all_bad, index)[0][1].isnan()
    all_bad[1] = float("-inf")
    all_bad[1, k - 1] = float("nan")
    assert ops.DistillationLoss(z, all_bad, index)[0][1].isnan()
