"""What VocabularyCrossEntropy's 16-bit products lose in one direction: errors of a common sign, which norms of random data do not show."""
import pytest
import torch

from neoml_b200 import _capi as capi
from neoml_b200 import ops

HALVES = [torch.float16, torch.bfloat16]


def _made(t, *shape, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(t)


@pytest.mark.gpu
@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("rows,width,v", [(64, 4096, 2000), (300, 8200, 700), (3, 4104, 9000)])
def test_long_sums_of_one_sign(t, rows, width, v):
    """The tensor core's additions cut off: a sum of 512 elements is 32 of them, each of which loses about a unit in the last place (2^-23) of
    what has been summed, which on the way up comes to 16.5 of the whole.  Those sums are added up to nearest; the row's maximum, its
    logarithm and their sum round a few times more."""
    x, w = _made(t, rows, width, seed=1).abs(), (_made(torch.float32, v, width, seed=2).abs() * (20 / width)).to(t)
    labels = torch.arange(rows, device="cuda", dtype=torch.int32) % v
    loss, log_sum = ops.VocabularyCrossEntropy(x, w, labels)
    z = x.double() @ w.double().T
    want = torch.logsumexp(z, 1)
    bound = (16.5 * 2.0 ** -23 + (width / 512 + 16) * 2.0 ** -24) * want
    assert ((log_sum.double() - want).abs() <= bound).all()
    assert ((loss.double() - (want - z.gather(1, labels.long()[:, None])[:, 0])).abs() <= 2 * bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width,v", [(4096, 768, 30000), (5001, 520, 24001)])
def test_gradient_of_many_entries_of_one_sign(rows, width, v):
    """hidden_diff of positive weights whose labelled entry has a softmax of zero, so that its part of dz is exact, by
    enough rows for the sum not to be cut into parts.  The vocabulary is summed 1024 entries at a time in 64 additions of 17 addends each (16
    products and the sum so far), which are cut off at the last place of the largest: less than 17 units of 2^-23 of the sum so far, and as that
    grows evenly 32.5 times that of the whole.  A half's own rounding, which has no direction, is 2^-11 over the root of how many there are."""
    t = torch.float16
    x, w = _made(t, rows, width, seed=1), _made(t, v, width, seed=2).abs() * 0.05
    x[:, 0], w[:, 0], w[7, 0] = 4.0, 1.0, -8.0
    labels = torch.full((rows,), 7, dtype=torch.int32, device="cuda")
    dloss = torch.full((rows,), 1024.0, device="cuda")
    _, log_sum = ops.VocabularyCrossEntropy(x, w, labels)
    dx, _ = ops.VocabularyCrossEntropyBackward(dloss, x, w, labels, log_sum, weights_diff=False)
    part = 1024 * torch.cat([torch.softmax(cut.double() @ w.double().T, 1) @ w.double() for cut in x.split(1024)])[:, 1:]
    want = part - 1024 * w[7, 1:].double()
    lost = (dx[:, 1:].double() - want).sum() / part.sum()
    noise = 2.0 ** -11 * want.abs().max() / part.mean() / (rows * (width - 1)) ** 0.5
    assert lost.abs() <= 32.5 * 17 * 2.0 ** -23 + 64 * 2.0 ** -24 + 3 * noise


@pytest.mark.gpu
@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("rows,width,v", [(921, 512, 30000), (48, 1024, 32000), (1843, 200, 9001)])
@pytest.mark.parametrize("every", [1, 3])
def test_mean_losses(t, rows, width, v, every):
    """One loss_diff for all rows that count, 1 / their number as a mean has it, which 16 bits do not hold: neither gradient may be off in a
    common direction.  A rounding has a deviation of at most a half step over the root of three; dz rounds the softmax's part, a tenth
    of it here.  The label's element, p - 1, may round to -1, which is off by p; sums lose a few 2^-17 (above)."""
    x, w = _made(t, rows, width, seed=1), (_made(torch.float32, v, width, seed=2) * (2 / width ** 0.5)).to(t)
    labels = (torch.arange(rows, device="cuda", dtype=torch.int32) * 7919 % v // 16 * 16).int()   # many of them repeated
    labels[every::every + 1] = -1
    scale = 4096.0 if t == torch.float16 else 1.0
    dloss = torch.full((rows,), scale / (labels >= 0).sum().item(), device="cuda")
    _, log_sum = ops.VocabularyCrossEntropy(x, w, labels)
    dx, dw = ops.VocabularyCrossEntropyBackward(dloss, x, w, labels, log_sum)
    used = labels >= 0
    p = torch.softmax(x.double() @ w.double().T, 1)
    at = labels.clamp(min=0).long()[:, None]
    own = p.gather(1, at)[used].mean()
    dz = (p.scatter_add(1, at, torch.full_like(at, -1.0, dtype=torch.float64)) * dloss.double()[:, None])[used]
    half = torch.finfo(t).eps / 2
    for got, want in ((dx[used], dz @ w.double()), (dw[at[used][:, 0].unique()], (dz.T @ x[used].double())[at[used][:, 0].unique()])):
        off = got.double() - want
        tiny = 2.0 ** -25 * want.numel() ** 0.5 if t == torch.float16 else 0.0   # of halves below their normal numbers
        assert off.norm() <= 1.03 * half / 3 ** 0.5 * want.norm() + tiny
        lost = (off * want.sign()).sum() / want.abs().sum()
        assert lost.abs() <= 5 * half / (3 * want.numel()) ** 0.5 * want.norm() / want.abs().mean() / want.numel() ** 0.5 + own + 2.0 ** -15


def test_sizes_beyond_the_limits_are_named():
    """Their scratch memory has no size, so none can be given."""
    lib = capi.load()
    for rows, width, v in ((2 ** 24 + 1, 8, 10), (4, 2 ** 24 + 8, 10), (4, 8, 2 ** 28 + 1)):
        for t in (0, 2):
            assert lib.nb200_vocabulary_cross_entropy_scratch_bytes(t, 64, rows, width, width, 64, v, width, 1) == 0
            assert lib.nb200_vocabulary_cross_entropy(None, t, 64, rows, width, width, 64, v, width, 64, 64, 64, None) == capi.ETOOBIG
            assert lib.nb200_vocabulary_cross_entropy_backward(None, t, 64, 64, rows, width, width, 64, v, width, 64, 64, 64, width, 64, width,
                                                               None) == capi.ETOOBIG


@pytest.mark.gpu
@pytest.mark.parametrize("t", [torch.float32, *HALVES])
@pytest.mark.parametrize("rows,width,v", [(5, 64, 3000), (20, 64, 9600), (200, 96, 1001), (40, 130, 40000)])   # few rows, some, wide and narrow tiles
@pytest.mark.parametrize("offset", [0.0, 200.0, -500.0])
def test_losses_of_confident_rows(t, rows, width, v, offset):
    """The label has nearly all of the probability, all logits a common part: the loss is small and does not know that part.  What a
    product's rounding moves of the logits, a few units of their terms' size, counts as far as the other entries do.  The sum of
    exponentials is about one and rounded at that size: 8 + 2 additions of a thread's 32 columns, 4 of its groups of them (by the kernels for few
    rows, 16 entries one after another, twice each), 3 + 5 joins of the parts, the exponential and the logarithm two each: 48 at most."""
    x, w = _made(t, rows, width, seed=1), (_made(torch.float32, v, width, seed=2) / width ** 0.5).to(t)
    labels = torch.full((rows,), 5, dtype=torch.int32, device="cuda")
    x[:, 0], w[:, 0] = 8.0, offset / 8
    at = labels.long()[:, None]
    x[:, 1], w[:, 1], w[5, 1] = 4.0, 0.0, 4.0       # 16 above the others
    z = x.double() @ w.double().T
    loss, log_sum = ops.VocabularyCrossEntropy(x, w, labels)
    p = torch.softmax(z, 1)
    rest = p.scatter(1, at, 0.0).sum(1)
    want = -torch.log1p(-rest)
    moved = (x.double().abs() @ w.double().abs().T).amax(1) * 2.0 ** -20
    assert rest.max() < 0.2
    assert ((loss.double() - want).abs() <= 2 * rest * (moved + (32 + v / 128) * 2.0 ** -24) + 48 * 2.0 ** -24 * (1 + want)).all()
    assert ((log_sum.double() - torch.logsumexp(z, 1)).abs() <= moved + 2.0 ** -22 * (1 + log_sum.double().abs())).all()
