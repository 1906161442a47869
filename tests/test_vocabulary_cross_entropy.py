"""VocabularyCrossEntropy and its backward pass against 64-bit arithmetic."""
import math

import pytest
import torch

from neoml_b200 import _capi as capi
from neoml_b200 import ops

TYPES = [torch.float32, torch.float16, torch.bfloat16]
STEP = 2.0 ** -24


def _made(t, *shape, seed, std=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(t)


def _labels(rows, v, seed, unused=0.15):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    labels = torch.randint(0, v, (rows,), generator=g, device="cuda", dtype=torch.int32)
    labels[torch.rand(rows, generator=g, device="cuda") < unused] = -1
    return labels


def _case(t, rows, width, v, seed=0):
    return (_made(t, rows, width, seed=seed + 1), _made(t, v, width, seed=seed + 2, std=2.0 / math.sqrt(width)),
            _labels(rows, v, seed + 3))


def _check(x, w, labels, dloss=None, got_forward=None, **kw):
    """Bounds: a product's sum of `width` terms in fp32 is off by at most width / 2 of its roundings (half a unit each, by its
    terms' absolute sum; the split products of fp32 operands keep 21 bits of each factor); an exponential carries its
    argument's error; dz is rounded to the 16-bit type once; sums over rows or columns round as the first one does."""
    t, (rows, width), v = x.dtype, x.shape, len(w)
    dloss = _made(torch.float32, rows, seed=77).abs() + 0.1 if dloss is None else dloss
    loss, log_sum = ops.VocabularyCrossEntropy(x, w, labels)
    dx, dw = ops.VocabularyCrossEntropyBackward(dloss, x, w, labels, log_sum, **kw)
    assert loss.dtype == log_sum.dtype == torch.float32 and dx.dtype == dw.dtype == t and dx.shape == x.shape and dw.shape == w.shape
    used = (labels >= 0) & (labels < v)
    xd = torch.where((used & (dloss != 0))[:, None], x.double(), 0.0)   # what has no gradient is not looked at
    xf, wd = torch.where(used[:, None], x.double(), 0.0), w.double()
    at = torch.where(used, labels, 0).long()[:, None]
    z = xf @ wd.T
    product = (2.0 ** -20 if t == torch.float32 else 0.0) + min(width / 2, 64) * STEP   # sums of blocks of at most 128 terms meet
    z_off = (xf.abs() @ wd.abs().T) * product
    want_sum = torch.logsumexp(z, 1)
    p = torch.exp(z - want_sum[:, None])
    grow = (16 + v / 128) * STEP
    sum_off = (p * z_off).sum(1) + grow + 4 * STEP * (want_sum.abs() + z.abs().amax(1))
    assert ((log_sum.double() - want_sum).abs()[used] <= sum_off[used]).all()
    want = torch.where(used, want_sum - z.gather(1, at)[:, 0], 0.0)
    off = torch.where(used, sum_off + z_off.gather(1, at)[:, 0] + 2 * STEP * want.abs(), 0.0)
    assert ((loss.double() - want).abs() <= off).all()
    g = torch.where(used, dloss.double(), 0.0)[:, None]
    hot = torch.zeros_like(z).scatter_(1, at, 1.0)
    dz = g * (p - hot)
    half = torch.finfo(t).eps / 2
    dz_off = g.abs() * p * (z_off + sum_off[:, None] + (16 + 2 * (z.abs() + want_sum.abs()[:, None])) * STEP) + 4 * STEP * dz.abs()
    if t != torch.float32:
        # fp16: scaled to 2^14, so that half a step of its smallest numbers is 2^-25 / 2^14 of the largest loss_diff
        dz_off = dz_off + half * dz.abs() + (2.0 ** -38 * g.abs().max() if t == torch.float16 else 0.0)
    for name, got, a, a_off, b in (("dx", dx, dz, dz_off, wd), ("dw", dw, dz.T, dz_off.T, xd)):
        value = a @ b
        terms = min(a.shape[1] / 2, 64) + a.shape[1] / 2048
        # fp32 below 2^-126 counts as zero: a softmax value of that size is lost, times what it would have been multiplied by
        tiny = (2.0 ** -25 if t == torch.float16 else 2.0 ** -126) + 2.0 ** -126 * (1 + g.abs().max()) * b.abs().sum(0)
        bound = half * value.abs() + a_off @ b.abs() + (a.abs() @ b.abs()) * ((2.0 ** -20 if t == torch.float32 else 0.0) + (8 + terms) * STEP) + tiny
        excess = (got.double() - value).abs() - bound
        assert excess.max().item() <= 0.0, f"{name}: {excess.max().item()} more than allowed"
        # those bounds are for the worst case; roundings without a common direction stay far below
        if a.shape[1] * got.numel() > 10000:
            assert (got.double() - value).norm() <= (2.5 * half + (1e-5 if t == torch.float32 else 0.0)) * value.norm()
    assert (dx[~used] == 0).all()
    return loss, log_sum, dx, dw


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,width,v", [(1, 1, 1), (1, 8, 2), (3, 64, 256), (128, 64, 256), (129, 72, 300), (7, 129, 1000), (200, 1031, 515),
                                          (48, 256, 32000), (1, 512, 5003), (1000, 96, 257), (300, 640, 1500), (2049, 33, 77), (130, 2048, 700), (4, 203, 70001), (8, 31, 300), (9, 1001, 2000),
                                          (16, 130, 5000), (16, 4100, 64), (17, 203, 3000), (2, 3, 150000)])
def test_against_64_bits(t, rows, width, v):
    _check(*_case(t, rows, width, v))


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
def test_several_pieces(t, monkeypatch):
    """More columns than a piece holds: the sums over the vocabulary go on from piece to piece, the last of them ragged."""
    rows, width, v = (12000, 24, 12000) if t != torch.float32 else (6000, 24, 11001)
    x, w, labels = _case(t, rows, width, v)
    loss, log_sum = ops.VocabularyCrossEntropy(x, w, labels)
    dloss = _made(torch.float32, rows, seed=7)
    dx, dw = ops.VocabularyCrossEntropyBackward(dloss, x, w, labels, log_sum)
    used = labels >= 0
    for r in range(0, rows, 1500):    # 64-bit logits in parts
        cut = slice(r, r + 1500)
        z = x[cut].double() @ w.double().T
        want = torch.where(used[cut], torch.logsumexp(z, 1) - z.gather(1, labels[cut].clamp(min=0).long()[:, None])[:, 0], 0.0)
        assert (loss[cut].double() - want).abs().max() < 2e-5
        dz = torch.softmax(z, 1)
        dz.scatter_add_(1, labels[cut].clamp(min=0).long()[:, None], -torch.ones(len(z), 1, dtype=torch.float64, device="cuda"))
        dz *= torch.where(used[cut], dloss[cut], 0.0).double()[:, None]
        value = dz @ w.double()
        assert (dx[cut].double() - value).norm() <= (2.5 * torch.finfo(t).eps / 2 + 1e-5) * value.norm()
        total = dz.T @ x[cut].double() + (total if r else 0.0)
    assert (dw.double() - total).norm() <= (2.5 * torch.finfo(t).eps / 2 + 1e-5) * total.norm()


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("width,first,row", [(64, 8, 96), (64, 1, 77), (31, 2, 40)])
def test_views_of_columns(t, width, first, row):
    x, w = _made(t, 70, row, seed=1)[:, first:first + width], _made(t, 333, row, seed=2, std=0.3)[:, first:first + width]
    labels = _labels(70, 333, 3)
    room, room_w = torch.full((70, row), 5.0, dtype=t, device="cuda"), torch.full((333, row), 5.0, dtype=t, device="cuda")
    dx, dw = room[:, first:first + width], room_w[:, first:first + width]
    _, _, got, got_w = _check(x, w, labels, hidden_diff=dx, weights_diff=dw)
    assert got is dx and got_w is dw
    dx.fill_(5.0), dw.fill_(5.0)
    assert (room == 5.0).all() and (room_w == 5.0).all()   # nothing around the rows was touched


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
def test_rows_without_a_target(t):
    x, w, labels = _case(t, 150, 80, 400)
    labels[::3] = torch.tensor([-1, 400, -100, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda").repeat(10)
    dloss = _made(torch.float32, 150, seed=9)
    dloss[1] = 0.0
    first = _check(x, w, labels, dloss)
    x[::3] = float("nan")     # padding that was never written
    again = ops.VocabularyCrossEntropy(x, w, labels)
    assert torch.equal(again[0], first[0])
    grads = ops.VocabularyCrossEntropyBackward(dloss, x, w, labels, again[1])
    assert torch.equal(grads[0], first[2]) and torch.equal(grads[1], first[3]) and (grads[0][1] == 0).all()
    none = torch.full_like(labels, -1)
    loss, log_sum = ops.VocabularyCrossEntropy(x, w, none)
    assert (loss == 0).all()
    for g in ops.VocabularyCrossEntropyBackward(dloss, x, w, none, log_sum):
        assert (g == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("scale", [1e-6, 1.0, 3e4])
def test_sizes_of_the_gradient(t, scale):
    """loss_diff as a trainer scales it: the rounding of dz does not depend on it."""
    x, w, labels = _case(t, 64, 128, 3001)
    x, w = x / 16, w / 16 if scale == 3e4 else w
    dloss = torch.full((64,), scale / 64, device="cuda")
    if t == torch.float16 and scale == 1e-6:
        loss, log_sum = ops.VocabularyCrossEntropy(x, w, labels)
        small = ops.VocabularyCrossEntropyBackward(dloss, x, w, labels, log_sum)
        assert all(g.abs().max() < 1e-6 for g in small)     # below a half's smallest numbers, mostly
        return
    _check(x, w, labels, dloss)


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
def test_confident_and_repeated_rows(t):
    """Logits of a hundred: softmax zeros and ones, and one label on many rows."""
    x, w = _made(t, 200, 64, seed=1, std=4.0), _made(t, 500, 64, seed=2, std=3.0)
    labels = torch.full((200,), 17, dtype=torch.int32, device="cuda")
    labels[100:] = (x[100:].double() @ w.double().T).argmax(1).int()
    _check(x, w, labels)


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
def test_one_gradient_only_repeats_and_leading_dimensions(t):
    x, w, labels = _case(t, 60, 40, 600)
    dloss = _made(torch.float32, 60, seed=9)
    loss, log_sum = ops.VocabularyCrossEntropy(x.view(4, 15, 40), w, labels.view(4, 15))
    assert loss.shape == log_sum.shape == (4, 15)
    dx, dw = ops.VocabularyCrossEntropyBackward(dloss.view(4, 15), x.view(4, 15, 40), w, labels.view(4, 15), log_sum)
    assert dx.shape == (4, 15, 40)
    only, none = ops.VocabularyCrossEntropyBackward(dloss, x, w, labels, log_sum, weights_diff=False)
    assert none is None and torch.equal(only, dx.view(60, 40))
    none, only = ops.VocabularyCrossEntropyBackward(dloss, x, w, labels, log_sum, hidden_diff=False)
    assert none is None and torch.equal(only, dw)
    assert ops.VocabularyCrossEntropyBackward(dloss, x, w, labels, log_sum, hidden_diff=False, weights_diff=False) == (None, None)


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
def test_no_rows(t):
    x, w, labels = torch.empty(0, 16, dtype=t, device="cuda"), _made(t, 30, 16, seed=1), torch.empty(0, dtype=torch.int32, device="cuda")
    loss, log_sum = ops.VocabularyCrossEntropy(x, w, labels)
    dx, dw = ops.VocabularyCrossEntropyBackward(loss, x, w, labels, log_sum)
    assert loss.shape == (0,) and dx.shape == (0, 16) and (dw == 0).all()


@pytest.mark.gpu
def test_gradient_is_the_slope():
    x, w, labels = _case(torch.float32, 20, 12, 50)
    dloss, h = _made(torch.float32, 20, seed=9), 2.0 ** -6
    _, log_sum = ops.VocabularyCrossEntropy(x, w, labels)
    for k, grad in enumerate(ops.VocabularyCrossEntropyBackward(dloss, x, w, labels, log_sum)):
        direction = _made(torch.float32, *(x, w)[k].shape, seed=30 + k)
        value = []
        for sign in (1, -1):
            pair = [x, w]
            pair[k] = pair[k] + sign * h * direction
            value.append((ops.VocabularyCrossEntropy(*pair, labels)[0].double() * dloss.double()).sum())
        slope, want = (value[0] - value[1]) / (2 * h), grad.double() * direction.double()
        # third derivatives of a log-sum, logits moving by up to about ten: under a hundred, over six; fp32 losses of about ten
        assert abs(slope - want.sum()) <= (100 / 6 * h * h * 4 + 2.0 ** -18 / h) * dloss.abs().sum()


@pytest.mark.gpu
def test_graph_and_stream():
    x, w, labels = _case(torch.bfloat16, 300, 136, 1000)
    dloss = _made(torch.float32, 300, seed=9)

    def step():
        loss, log_sum = ops.VocabularyCrossEntropy(x, w, labels)
        return (loss, log_sum, *ops.VocabularyCrossEntropyBackward(dloss, x, w, labels, log_sum))
    first = step()
    assert all(torch.equal(a, b) for a, b in zip(first, step()))
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
            out = step()
        graphs.append((graph, out))
    x.copy_(_made(torch.bfloat16, 300, 136, seed=21))
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, step())) and not torch.equal(out[0], first[0])
    assert capi.load().nb200_device_status(None, 0) == 0


def test_refusals():
    x, w, labels = torch.zeros(4, 8), torch.zeros(10, 8), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(AssertionError, match="CUDA device"):
        ops.VocabularyCrossEntropy(x, w, labels)
    with pytest.raises(AssertionError, match="weights"):
        ops.VocabularyCrossEntropy(x, torch.zeros(10, 9), labels)
    with pytest.raises(AssertionError, match="weights"):
        ops.VocabularyCrossEntropy(x, w.half(), labels)
    with pytest.raises(AssertionError, match="a vocabulary"):
        ops.VocabularyCrossEntropy(x, torch.zeros(0, 8), labels)
    with pytest.raises(AssertionError, match="label"):
        ops.VocabularyCrossEntropy(x, w, labels[:3])
    with pytest.raises(AssertionError, match="fp32, fp16 or bf16"):
        ops.VocabularyCrossEntropy(x.double(), w.double(), labels)


def test_argument_validation_needs_no_device():
    lib = capi.load()
    forward = [None, 2, 64, 4, 8, 8, 64, 10, 8, 64, 64, 64, 256]
    for at, value in ((1, 3), (2, None), (2, 65), (3, -1), (4, 0), (5, 7), (6, None), (7, 0), (8, 7), (9, None), (10, None), (11, None),
                      (12, None), (12, 64)):
        bad = list(forward)
        bad[at] = value
        assert lib.nb200_vocabulary_cross_entropy(*bad) == capi.EINVAL, (at, value)
    forward[3] = 2 ** 24 + 1
    assert lib.nb200_vocabulary_cross_entropy(*forward) == capi.ETOOBIG
    forward[3] = 0
    assert lib.nb200_vocabulary_cross_entropy(*forward) == capi.OK
    backward = [None, 2, 64, 64, 4, 8, 8, 64, 10, 8, 64, 64, 64, 8, 64, 8, 256]
    for at, value in ((1, -1), (2, None), (3, None), (4, -1), (6, 7), (7, None), (9, 1), (10, None), (11, None), (12, 65), (13, 7), (14, 65), (15, 7),
                      (16, None)):
        bad = list(backward)
        bad[at] = value
        assert lib.nb200_vocabulary_cross_entropy_backward(*bad) == capi.EINVAL, (at, value)
    backward[12] = backward[14] = None
    assert lib.nb200_vocabulary_cross_entropy_backward(*backward) == capi.OK
    need = lib.nb200_vocabulary_cross_entropy_scratch_bytes
    assert need(2, 64, 0, 8, 8, 64, 10, 8, 1) == 0 and need(5, 64, 4, 8, 8, 64, 10, 8, 1) == 0
    # one piece of the gradient by the logits, however large the vocabulary
    assert 250e6 < need(2, 256, 8192, 64, 64, 256, 10 ** 7, 64, 1) < 300e6
    # a copy of weights that do not begin on a 16-byte boundary
    assert need(2, 256, 40, 64, 64, 258, 10 ** 6, 64, 0) - need(2, 256, 40, 64, 64, 256, 10 ** 6, 64, 0) == 128 * 10 ** 6
    # a few rows of fp32 take the weights as they lie
    assert need(0, 260, 4, 64, 64, 260, 10 ** 6, 64, 0) < 10 ** 5


def test_vectors_off_word_boundaries_are_refused():
    lib = capi.load()
    calls = ((lib.nb200_vocabulary_cross_entropy, [None, 2, 64, 4, 8, 8, 64, 10, 8, 64, 64, 64, 256], (9, 10, 11)),
             (lib.nb200_vocabulary_cross_entropy_backward, [None, 2, 64, 64, 4, 8, 8, 64, 10, 8, 64, 64, 64, 8, 64, 8, 256], (2, 10, 11)))
    for function, good, places in calls:
        for at in places:
            bad = list(good)
            bad[at] = 66
            assert function(*bad) == capi.EINVAL, (function, at)


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
def test_none_is_not_wanted(t):
    x, w, labels = _case(t, 30, 24, 100)
    dloss = _made(torch.float32, 30, seed=9)
    _, log_sum = ops.VocabularyCrossEntropy(x, w, labels)
    dx, dw = ops.VocabularyCrossEntropyBackward(dloss, x, w, labels, log_sum)
    only, none = ops.VocabularyCrossEntropyBackward(dloss, x, w, labels, log_sum, weights_diff=None)
    assert none is None and torch.equal(only, dx)
    none, only = ops.VocabularyCrossEntropyBackward(dloss, x, w, labels, log_sum, hidden_diff=None)
    assert none is None and torch.equal(only, dw)


def test_negated_views_are_refused():
    x, w, labels = torch.zeros(4, 8), torch.zeros(10, 8), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(AssertionError, match="negated"):
        ops.VocabularyCrossEntropy(torch._neg_view(x), w, labels)
    with pytest.raises(AssertionError, match="negated"):
        ops.LayerNormalization(torch._neg_view(x))
    with pytest.raises(AssertionError, match="negated"):
        ops.GatedRecurrence(x[None], torch._neg_view(x[None]))
    with pytest.raises(AssertionError, match="negated"):
        ops.DistillationLoss(torch._neg_view(x), torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int32))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width,v", [(9, 33, 9600), (12, 1, 40000), (16, 130, 20011), (17, 64, 30003), (24, 36, 12001), (25, 1031, 9500), (32, 206, 10007), (32, 512, 9999),
                                          (33, 206, 10007)])
def test_some_rows_of_fp32(rows, width, v):
    x, w, labels = _case(torch.float32, rows, width, v)
    labels[0], labels[-1] = 0, v - 1
    _check(x, w, labels)
    first = ops.VocabularyCrossEntropy(x, w, labels)
    assert all(torch.equal(a, b) for a, b in zip(first, ops.VocabularyCrossEntropy(x, w, labels)))


@pytest.mark.gpu
@pytest.mark.parametrize("first,row", [(0, 72), (2, 70), (1, 72), (2, 69)])
def test_some_rows_of_fp32_in_views(first, row):
    x, w, labels = _case(torch.float32, 20, row, 9700)
    x, w = x[:, first:first + 64], w[:, first:first + 64]
    got, want = (ops.VocabularyCrossEntropy(*pair, labels) for pair in ((x, w), (x.contiguous(), w.contiguous())))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # a row without a target, whatever it holds, and its neighbours
    x = x.clone()
    labels[3] = -1
    before = ops.VocabularyCrossEntropy(x, w, labels)
    x[3] = float("nan")
    after = ops.VocabularyCrossEntropy(x, w, labels)
    others = torch.arange(20, device="cuda") != 3
    assert torch.equal(before[0], after[0]) and torch.equal(before[1][others], after[1][others])

