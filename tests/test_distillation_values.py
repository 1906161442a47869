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


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,v,k", [(5, 2003, 64), (300, 1003, 9), (2, 60001, 300), (40, 777, 1)])
@pytest.mark.parametrize("offset,tau", [(1000.0, 1.0), (-1000.0, 1.0), (300.0, 0.3), (-20000.0, 3.0)])
def test_a_common_offset_of_the_students_logits(t, rows, v, k, offset, tau):
    """The loss does not know it, nor does its error: a student close to its teacher, so that the loss is small, and far from zero."""
    z = (_made(t, rows, v, seed=1).float() * min(tau, 1.0) + offset).to(t)
    index = _indices(rows, v, k)
    z.scatter_add_(1, index.long(), torch.full(index.shape, 16.0 * tau, dtype=t, device="cuda"))   # nearly all of the student's probability
    top = (z.gather(1, index.long()).float() - offset + 0.1 * _made(torch.float32, rows, k, seed=3)).to(t)
    loss, log_sum = ops.DistillationLoss(z, top, index, temperature=tau)
    zd, x = z.double() / tau, top.double() / tau
    log_p = torch.log_softmax(x, 1)
    want_sum = torch.logsumexp(zd, 1)
    log_q = zd.gather(1, index.long()) - want_sum[:, None]
    p = log_p.exp()
    want = tau ** 2 * (p * (log_p - log_q)).sum(1)
    # exponents are rounded at the size of the distances within a row, a hundred of them at most that count, and the terms as they are
    inside = (x - x.amax(1, keepdim=True)).abs().amax(1) + (zd - zd.amax(1, keepdim=True)).abs().clamp(max=100).amax(1)
    size = (p * (log_p.abs() + log_q.abs())).sum(1)
    # (c x is rounded at the teacher's own size, which the test keeps to that of its distances)
    bound = tau ** 2 * (32 + v / 256 + 4 * inside + 4 * x.abs().amax(1)) * 2.0 ** -24 * (1 + size)
    assert ((loss.double() - want).abs() <= bound).all()
    assert ((log_sum.double() - want_sum).abs() <= 2 * 2.0 ** -24 * want_sum.abs() + bound / tau ** 2).all()


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,v", [(5, 2003), (300, 1003)])
@pytest.mark.parametrize("k,at", [(2, 0), (2, 1), (9, 4), (300, 0), (300, 299)])
def test_kept_columns_that_a_student_masks(t, rows, v, k, at):
    """A column at the type's lowest value adds its probability times that, and nothing where the probability is nothing in fp32; the
    other terms are neither lost in it nor in its absence."""
    z, top, index = _made(t, rows, v, seed=1), _made(t, rows, k, seed=2), _indices(rows, v, k)
    lowest = torch.finfo(t).min
    z.scatter_(1, index[:, at:at + 1].long(), lowest)
    for far in (300.0, 24.0, 2.0):
        top[:, at] = -far
        loss, log_sum = ops.DistillationLoss(z, top, index)
        zd, x = z.double(), top.double()
        want_sum = torch.logsumexp(zd, 1)
        log_p = torch.log_softmax(x, 1)
        p = torch.where(log_p < -150, 0.0, log_p.exp())
        terms = torch.where(p > 0, p * (log_p - zd.gather(1, index.long()) + want_sum[:, None]), 0.0)
        # a probability is off by its logarithm's size, and so is the masked column's part of the loss
        assert ((loss.double() - terms.sum(1)).abs() <= (64 + 4 * far) * 2.0 ** -24 * terms.abs().sum(1)).all()
        assert ((log_sum.double() - want_sum).abs() <= 64 * 2.0 ** -24 * want_sum.abs()).all()
    z.fill_(lowest)   # all alike: log of how many, above the lowest value
    log_sum = ops.DistillationLoss(z, top, index)[1]
    want_sum = lowest + torch.log(torch.tensor(float(v), dtype=torch.float64, device="cuda"))
    assert ((log_sum.double() - want_sum).abs() <= 2.0 ** -22 * abs(lowest)).all()
