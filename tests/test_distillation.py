"""DistillationLoss and its backward pass against 64-bit arithmetic."""
import pytest
import torch

from neoml_b200 import _capi as capi
from neoml_b200 import ops

TYPES = [torch.float32, torch.float16, torch.bfloat16]
STEP = 2.0 ** -24


def _made(t, *shape, seed, std=2.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(t)


def _indices(rows, v, k, seed, low=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randint(low, v, (rows, k), generator=g, device="cuda", dtype=torch.int32)


def _reference(z, top, index, tau, dloss=None):
    z, v = z.double() / tau, z.shape[-1]
    used = (index >= 0) & (index < v)
    x = torch.where(used, top.double() / tau, -torch.inf)
    any_used = (x > -torch.inf).any(1) if index.shape[1] else torch.zeros(len(z), dtype=torch.bool, device=z.device)
    p = torch.where(any_used[:, None], torch.softmax(torch.where(any_used[:, None], x, 0.0), 1), 0.0) if index.shape[1] else x
    log_sum = torch.logsumexp(z, 1)
    at = torch.where(used, index, 0).long()
    log_q = z.gather(1, at) - log_sum[:, None]
    terms = torch.where(p > 0, p * (torch.log(p) - log_q), 0.0)
    size = torch.where(p > 0, p * (torch.log(p).abs() + z.gather(1, at).abs() + log_sum[:, None].abs()), 0.0)
    out = {"log_sum": log_sum, "loss": tau ** 2 * terms.sum(1), "size": tau ** 2 * size.sum(1)}
    if dloss is not None:
        target = torch.zeros_like(z).scatter_add_(1, at, p)
        q = torch.exp(z - log_sum[:, None]) * any_used[:, None]
        out["diff"] = tau * dloss.double()[:, None] * (q - target)
        # an exponential's argument is rounded at the size of the logits and of their sum
        noise = (16 + 2 * (torch.where(q > 0, z.abs(), 0.0) + log_sum.abs()[:, None])) * STEP   # nothing where q is zero
        worst = x.abs().nan_to_num(posinf=0.0).amax(1, keepdim=True) if index.shape[1] else 0.0
        out["off"] = (tau * dloss.double()[:, None]).abs() * (q * noise + target * (24 + 4 * worst) * STEP)
    return out


def _check(z, top, index, tau, **kw):
    dloss = _made(torch.float32, len(z), seed=99)
    loss, log_sum = ops.DistillationLoss(z, top, index, temperature=tau)
    got = ops.DistillationLossBackward(dloss, z, top, index, log_sum, temperature=tau, **kw)
    want = _reference(z, top, index, tau, dloss)
    assert loss.dtype == log_sum.dtype == torch.float32 and loss.shape == (len(z),)
    # partial sums of a thread (at most a few hundred terms each) are joined pairwise: relative 2^-24 apiece
    grow = 16 + z.shape[1] / 256
    # only the entries that add something count: masked ones are exact zeros
    adds = torch.exp(z.double() / tau - want["log_sum"][:, None]) > 0
    bound = (grow + 2 * torch.where(adds, z.double() / tau, 0.0).abs().amax(1) + 4 * want["log_sum"].abs()) * STEP
    assert ((log_sum.double() - want["log_sum"]).abs() <= bound).all()
    spread = (top.double() / tau).abs().nan_to_num(posinf=0.0).amax(1) if index.shape[1] else 0.0
    assert ((loss.double() - want["loss"]).abs() <= want["size"] * (32 + 4 * spread) * STEP + tau ** 2 * bound).all()
    t = got.dtype
    tiny = 2.0 ** -25 if t == torch.float16 else 2.0 ** -126
    off = want["off"] + (tau * dloss.double()).abs()[:, None] * torch.exp(z.double() / tau - want["log_sum"][:, None]) * bound[:, None]
    excess = (got.double() - want["diff"]).abs() - (torch.finfo(t).eps / 2 * want["diff"].abs() + off + tiny)
    assert got.shape == z.shape and excess.max().item() <= 0.0, excess.max().item()
    return loss, got


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,v,k", [(1, 1, 1), (3, 2, 2), (5, 100, 7), (1, 50257, 64), (17, 32003, 100), (300, 1001, 33), (2, 4096, 1024),
                                      (4, 130001, 256), (601, 513, 5), (700, 2049, 128), (200, 1024, 129), (500, 3, 2)])
def test_against_64_bits(t, rows, v, k):
    for seed, tau in ((1, 1.0), (2, 2.5)):
        _check(_made(t, rows, v, seed=seed), _made(t, rows, k, seed=seed + 10), _indices(rows, v, k, seed + 20), tau)
    # the teacher in fp32
    _check(_made(t, rows, v, seed=3), _made(torch.float32, rows, k, seed=13), _indices(rows, v, k, 23), 0.7)


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows", [40, 300])   # a block per row, a warp per row
def test_unused_repeated_and_masked_entries(t, rows):
    v, k = 777, 12
    z, top, index = _made(t, rows, v, seed=1), _made(t, rows, k, seed=2), _indices(rows, v, k, 3)
    index[0] = -1                        # a row without a teacher
    index[1, 3:] = v                     # behind the vocabulary: not used
    index[2] = index[2, 0]               # one column, twelve times
    index[3, 5] = index[3, 2]
    top[4] = float("-inf")               # a teacher that excludes all it kept
    top[5, 1:] = float("-inf")
    top[6, 0] = float("inf")
    index[6, 0] = -7                     # an infinite logit in an entry that is not used
    top[7, 0], index[7, 0] = float("nan"), v + 5
    mask = _indices(rows, v, 50, 5).long()
    masked = z.scatter(1, mask, float("-inf"))
    keep = masked.gather(1, index.clamp(0, v - 1).long()).isinf().any(1)   # a kept column that the student excludes: infinite loss
    masked[keep] = z[keep]
    loss, grad = _check(masked, top, index, 1.5)
    assert loss[0] == 0 and (grad[0] == 0).all() and loss[4] == 0 and (grad[4] == 0).all()
    low = z.clone()
    low.scatter_(1, mask, torch.finfo(t).min)
    low[keep] = z[keep]
    _check(low, top, index, 1.5)


@pytest.mark.gpu
def test_a_kept_column_that_the_student_excludes():
    z = torch.zeros(1, 10, device="cuda")
    z[0, 3] = float("-inf")
    top, index = torch.zeros(1, 2, device="cuda"), torch.tensor([[3, 4]], dtype=torch.int32, device="cuda")
    loss, log_sum = ops.DistillationLoss(z, top, index)
    assert loss[0] == float("inf")
    grad = ops.DistillationLossBackward(torch.ones(1, device="cuda"), z, top, index, log_sum)
    assert grad[0, 3] == -0.5 and abs(grad[0, 4].item() - (1 / 9 - 0.5)) < 1e-6


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows", [37, 411])
def test_views_in_place_and_repeats(t, rows):
    v, k = 1003, 20
    wide, top, index = _made(t, rows, v + 30, seed=1), _made(t, rows, k, seed=2), _indices(rows, v, k, 3)
    dloss = _made(torch.float32, rows, seed=4)
    for first in (0, 3, 8):
        z = wide[:, first:first + v]
        _check(z, top, index, 1.0)
        loss, log_sum = ops.DistillationLoss(z, top, index)
        want = ops.DistillationLossBackward(dloss, z, top, index, log_sum)
        assert torch.equal(want, ops.DistillationLossBackward(dloss, z, top, index, log_sum))
        held = wide.clone()
        into = held[:, first:first + v]
        assert ops.DistillationLossBackward(dloss, into, top, index, log_sum, result=into) is into
        assert torch.equal(into, want)
        into.copy_(z)
        assert torch.equal(held, wide)   # nothing around the rows was touched
    big = _made(t, 2, 60001, seed=5)     # split rows
    top, index = _made(t, 2, k, seed=6), _indices(2, 60001, k, 7)
    loss, log_sum = ops.DistillationLoss(big, top, index)
    want = ops.DistillationLossBackward(dloss[:2], big, top, index, log_sum)
    assert torch.equal(ops.DistillationLossBackward(dloss[:2], big, top, index, log_sum, result=big), want)


@pytest.mark.gpu
def test_empty_and_leading_dimensions():
    z = _made(torch.float32, 2, 3, 50, seed=1)
    top, index = _made(torch.float32, 2, 3, 4, seed=2), _indices(6, 50, 4, 3).view(2, 3, 4)
    loss, log_sum = ops.DistillationLoss(z, top, index)
    assert loss.shape == log_sum.shape == (2, 3)
    assert torch.equal(loss.view(6), ops.DistillationLoss(z.view(6, 50), top.view(6, 4), index.view(6, 4))[0])
    loss, log_sum = ops.DistillationLoss(z, top[..., :0].contiguous(), index[..., :0].contiguous())
    assert (loss == 0).all()
    assert (ops.DistillationLossBackward(log_sum, z, top[..., :0].contiguous(), index[..., :0].contiguous(), log_sum) == 0).all()
    none = torch.empty(0, 50, device="cuda")
    loss, log_sum = ops.DistillationLoss(none, torch.empty(0, 4, device="cuda"), index[0, :0])
    assert loss.shape == (0,) and ops.DistillationLossBackward(loss, none, torch.empty(0, 4, device="cuda"), index[0, :0], log_sum).shape == (0, 50)


@pytest.mark.gpu
def test_gradient_is_the_slope():
    z, top, index = _made(torch.float32, 4, 60, seed=1), _made(torch.float32, 4, 6, seed=2), _indices(4, 60, 6, 3)
    dloss, direction, h = _made(torch.float32, 4, seed=4), _made(torch.float32, 4, 60, seed=5, std=1.0), 2.0 ** -7
    _, log_sum = ops.DistillationLoss(z, top, index, temperature=1.5)
    grad = ops.DistillationLossBackward(dloss, z, top, index, log_sum, temperature=1.5)
    value = [(ops.DistillationLoss(z + s * h * direction, top, index, temperature=1.5)[0].double() * dloss.double()) for s in (1, -1)]
    slope = (value[0] - value[1]).sum() / (2 * h)
    want = (grad.double() * direction.double())
    # third derivative of a log-sum along a direction of ones: below ten, over six; differences of fp32 losses of about ten
    assert abs(slope - want.sum()) <= (10 * h * h + 2.0 ** -20 / h) * dloss.abs().sum().item() * 10


def test_refusals():
    z, top, index = torch.zeros(4, 8), torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int32)
    with pytest.raises(AssertionError, match="CUDA device"):
        ops.DistillationLoss(z, top, index)
    with pytest.raises(AssertionError, match="for every row"):
        ops.DistillationLoss(z, top[:3], index[:3])
    with pytest.raises(AssertionError, match="for every row"):
        ops.DistillationLoss(z, top, index[:, :1])
    with pytest.raises(AssertionError, match="teacher"):
        ops.DistillationLoss(z, top.half(), index)
    with pytest.raises(AssertionError, match="int32"):
        ops.DistillationLoss(z, top, index.long())
    for tau in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(AssertionError, match="temperature"):
            ops.DistillationLoss(z, top, index, temperature=tau)


def test_argument_validation_needs_no_device():
    lib = capi.load()
    forward = [None, 0, 0, 64, 4, 8, 8, 64, 64, 2, 1.0, 64, 64]
    for at, value in ((1, 5), (2, 2), (3, None), (3, 66), (4, -1), (5, 0), (6, 7), (7, None), (8, None), (9, -1), (10, 0.0), (10, float("nan")),
                      (10, float("inf")), (11, None), (12, None)):
        bad = list(forward)
        bad[at] = value
        assert lib.nb200_distillation_loss(*bad) == capi.EINVAL, (at, value)
    forward[9] = 1025
    assert lib.nb200_distillation_loss(*forward) == capi.ETOOBIG
    forward[4] = 0
    assert lib.nb200_distillation_loss(*forward) == capi.OK
    backward = [None, 1, 0, 64, 64, 4, 8, 8, 64, 64, 2, 1.0, 64, 64, 8]
    for at, value in ((1, -1), (2, 2), (3, None), (4, None), (4, 65), (7, 7), (8, None), (12, None), (13, None), (13, 65), (14, 7)):
        bad = list(backward)
        bad[at] = value
        assert lib.nb200_distillation_loss_backward(*bad) == capi.EINVAL, (at, value)


def test_vectors_off_word_boundaries_are_refused():
    lib = capi.load()
    calls = ((lib.nb200_distillation_loss, [None, 1, 1, 64, 4, 8, 8, 64, 64, 2, 1.0, 64, 64], (8, 11, 12)),
             (lib.nb200_distillation_loss_backward, [None, 1, 1, 64, 64, 4, 8, 8, 64, 64, 2, 1.0, 64, 64, 8], (3, 9, 12)))
    for function, good, places in calls:
        for at in places:
            bad = list(good)
            bad[at] = 66
            assert function(*bad) == capi.EINVAL, (function, at)
