"""LayerNormalization and its backward pass against 64-bit arithmetic, at the widths, alignments and types where they can
go wrong."""
import pytest
import torch

from neoml_b200 import _capi as capi
from neoml_b200 import ops

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _half_step(t):
    return torch.finfo(t).eps / 2


def _close(got, want, magnitude, extra=0.0):
    """One rounding to the output's type, and fp32 arithmetic of up to some twenty roundings on terms of `magnitude`."""
    t = got.dtype
    bound = _half_step(t) * want.abs() + (24 * 2.0 ** -24 + extra) * magnitude + (2.0 ** -25 if t == torch.float16 else 0.0)
    worst = ((got.double() - want).abs() - bound).max().item() if got.numel() else 0.0
    assert worst <= 0.0, f"off by {worst} more than allowed"


def _reference(x, scale, free, epsilon, dy=None):
    x = x.double()
    s = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if scale is None else scale.double()
    mean = x.mean(-1, keepdim=True)
    inv = 1.0 / (((x - mean) ** 2).mean(-1, keepdim=True) + epsilon).sqrt()
    u = (x - mean) * inv
    y = u * s + (0.0 if free is None else free.double())
    if dy is None:
        return y, mean[..., 0], inv[..., 0], u
    dy = dy.double()
    g = dy * s
    dx = inv * (g - g.mean(-1, keepdim=True) - u * (g * u).mean(-1, keepdim=True))
    size = inv * (g.abs() + g.abs().mean(-1, keepdim=True) + u.abs() * (g * u).abs().mean(-1, keepdim=True))
    rows = tuple(range(x.dim() - 1))
    return dx, (dy * u).sum(rows), dy.sum(rows), size, (dy * u).abs().sum(rows), dy.abs().sum(rows)


def _made(shape, t, seed, mean=0.5):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") + mean).to(t)


def _check(x, scale, free, dy, epsilon=1e-5, **kw):
    y, mean, inv = ops.LayerNormalization(x, scale, free, epsilon=epsilon)
    want, wmean, winv, u = _reference(x, scale, free, epsilon)
    assert y.shape == x.shape and y.dtype == x.dtype and mean.shape == x.shape[:-1] and mean.dtype == torch.float32
    top = x.double().abs().amax(-1)
    _close(mean, wmean, top)
    # a rounding of the mean moves x - mean by that much, over the deviation
    lost = top[..., None] * winv[..., None]
    s = 1.0 if scale is None else scale.double().abs()
    _close(inv, winv, winv * (1 + top * winv))
    _close(y, want, want.abs() + (u.abs() + lost) * s)
    dx, ds, db = ops.LayerNormalizationBackward(dy, x, mean, inv, scale, **kw)
    wdx, wds, wdb, size, sum_s, sum_b = _reference(x, scale, free, epsilon, dy)
    assert dx.shape == x.shape and dx.dtype == x.dtype
    _close(dx, wdx, size * (1 + lost))
    if ds is not None:
        # fp32 sums of up to a thousand terms in a row before they meet others
        rows = x.numel() // x.shape[-1]
        grow = min(rows, 1000) * 2.0 ** -24
        per_row = (dy.double().abs() * lost).reshape(-1, x.shape[-1]).sum(0)
        _close(ds, wds, sum_s + per_row, grow)
        _close(db, wdb, sum_b, grow)
    return y, dx, ds, db


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 2), (1, 7), (8, 768), (5, 31), (33, 129), (700, 1031), (1, 4096), (601, 2048),
                                        (9, 8200), (3, 16384), (2, 20011), (4, 70001), (4099, 65)])
def test_against_64_bits(t, rows, width):
    x, dy = _made((rows, width), t, 1), _made((rows, width), t, 2, 0.0)
    scale, free = _made((width,), torch.float32, 3, 1.0), _made((width,), torch.float32, 4)
    _check(x, scale, free, dy)


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("scale,free", [(True, False), (False, True), (False, False)])
def test_optional_parameters_of_the_rows_type(t, scale, free):
    x, dy = _made((3, 50, 96), t, 1), _made((3, 50, 96), t, 2)
    _check(x, _made((96,), t, 3) if scale else None, _made((96,), t, 4) if free else None, dy)


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("width,first,row", [(64, 1, 80), (100, 3, 129), (7, 0, 9), (768, 8, 800), (33, 5, 40)])
def test_views_of_columns(t, width, first, row):
    """Rows that begin anywhere: aligned alike with the gradient or not."""
    x = _made((77, row), t, 1)[:, first:first + width]
    dy = _made((77, width), t, 2)
    scale = _made((width,), torch.float32, 3, 1.0)
    _check(x, scale, None, dy)
    _check(x, scale, None, _made((77, row), t, 5)[:, first:first + width])
    _check(_made((154, width), t, 6)[::2], scale, None, dy)
    # the elements between the rows stay as they are
    room = torch.full((77, row), 7.0, dtype=t, device="cuda")
    out = room[:, first:first + width]
    got, _, inv = ops.LayerNormalization(x, scale, result=out)
    want, _, _, u = _reference(x, scale, None, 1e-5)
    # (not the bits of contiguous rows: where a row begins decides which elements a thread adds)
    _close(got, want, want.abs() + (u.abs() + (x.double().abs().amax(-1) * inv.double())[:, None]) * scale.double().abs())
    room[:, first:first + width] = 7.0
    assert (room == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
def test_in_place_and_repeated(t):
    for rows, width in ((1000, 513), (5, 40001)):
        x, dy = _made((rows, width), t, 1), _made((rows, width), t, 2)
        scale, free = _made((width,), torch.float32, 3), _made((width,), torch.float32, 4)
        y, mean, inv = ops.LayerNormalization(x, scale, free)
        grads = ops.LayerNormalizationBackward(dy, x, mean, inv, scale)
        again = ops.LayerNormalizationBackward(dy, x, mean, inv, scale)
        assert all(torch.equal(a, b) for a, b in zip(grads, again))   # no order of additions that varies
        into = dy.clone()
        assert torch.equal(ops.LayerNormalizationBackward(into, x, mean, inv, scale, source_diff=into)[0], grads[0])
        held = x.clone()
        assert torch.equal(ops.LayerNormalization(held, scale, free, result=held)[0], y)


@pytest.mark.gpu
def test_constant_and_infinite_rows():
    x = torch.full((3, 200), 5.0, device="cuda")
    x[2, 3] = float("inf")
    y, mean, inv = ops.LayerNormalization(x, epsilon=1e-5)
    assert (y[:2] == 0).all() and (mean[:2] == 5).all() and y[2].isnan().any()
    assert torch.allclose(inv[:2], torch.full((2,), 1e-5 ** -0.5, device="cuda"))
    # values near the largest of a half: neither sums nor squares overflow
    h = (_made((4, 300), torch.float16, 1) * 20000).clamp(-60000, 60000)
    _check(h, None, None, _made((4, 300), torch.float16, 2))


@pytest.mark.gpu
def test_no_rows():
    x = torch.empty(0, 16, device="cuda")
    y, mean, inv = ops.LayerNormalization(x)
    assert y.shape == (0, 16) and mean.shape == (0,)
    dx, ds, db = ops.LayerNormalizationBackward(x, x, mean, inv)
    assert dx.shape == (0, 16) and (ds == 0).all() and (db == 0).all()
    assert ops.LayerNormalizationBackward(x, x, mean, inv, parameters=False)[1:] == (None, None)


@pytest.mark.gpu
def test_gradient_is_the_slope():
    """fp32 differences of the forward pass along random directions."""
    x, dy = _made((6, 40), torch.float32, 1), _made((6, 40), torch.float32, 2)
    scale, free = _made((40,), torch.float32, 3), _made((40,), torch.float32, 4)
    y, mean, inv = ops.LayerNormalization(x, scale, free)
    for operand, grad in zip((x, scale, free), ops.LayerNormalizationBackward(dy, x, mean, inv, scale)):
        step = torch.randn_like(operand)
        h = 2.0 ** -7
        hi, lo = operand + h * step, operand - h * step
        args = [hi if o is operand else o for o in (x, scale, free)], [lo if o is operand else o for o in (x, scale, free)]
        slope = (dy.double() * (ops.LayerNormalization(*args[0])[0].double() - ops.LayerNormalization(*args[1])[0].double())).sum() / (2 * h)
        want = (grad.double() * step.double()).sum()
        size = (grad.double() * step.double()).abs().sum()
        # differences: h^2 / 6 times a third derivative of the size of a few dozen first ones, and 2^-22 / h of rounding
        assert abs(slope - want) <= (40 * h * h + 2.0 ** -22 / h * 8) * size


@pytest.mark.gpu
def test_graph_and_stream():
    x, scale = _made((300, 320), torch.bfloat16, 1), _made((320,), torch.float32, 2)
    dy = _made((300, 320), torch.bfloat16, 3)
    side = torch.cuda.Stream()

    def step():
        y, mean, inv = ops.LayerNormalization(x, scale)
        return (y, *ops.LayerNormalizationBackward(dy, x, mean, inv, scale))
    want = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step()
    x.copy_(_made((300, 320), torch.bfloat16, 9))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, step())) and not torch.equal(got[0], want[0])


def test_refusals():
    x, v = torch.zeros(4, 8), torch.zeros(4)
    with pytest.raises(AssertionError, match="CUDA device"):
        ops.LayerNormalization(x)
    with pytest.raises(AssertionError, match="fp32, fp16 or bf16"):
        ops.LayerNormalization(x.double())
    with pytest.raises(AssertionError, match="parameters"):
        ops.LayerNormalization(x, torch.zeros(8, dtype=torch.float16))
    with pytest.raises(AssertionError, match="at least one"):
        ops.LayerNormalization(torch.zeros(4, 0))
    with pytest.raises(AssertionError, match="overlap"):
        ops.LayerNormalization(torch.zeros(1, 8).expand(4, 8))
    with pytest.raises(AssertionError, match="overlap"):
        ops.LayerNormalization(torch.zeros(8, 4).t())
    with pytest.raises(AssertionError, match="like the source"):
        ops.LayerNormalizationBackward(torch.zeros(4, 9), x, v, v)


def test_argument_validation_needs_no_device():
    lib, e = capi.load(), 1e-5
    good = [None, 0, 0, 64, 4, 8, 8, None, None, e, 64, 8, None, None]
    for at, value in ((1, 3), (1, -1), (2, 1), (4, -1), (5, 0), (6, 7), (11, 7), (3, None), (10, None), (3, 65), (7, 66)):
        bad = list(good)
        bad[at] = value
        assert lib.nb200_layer_normalization(*bad) == capi.EINVAL, (at, value)
    assert lib.nb200_layer_normalization(None, 0, 0, None, 0, 8, 8, None, None, e, None, 8, None, None) == capi.OK
    good = [None, 1, 0, 64, 8, 64, 4, 8, 8, None, 64, 64, 64, 8, 64, 64, 64]
    for at, value in ((1, 7), (2, 2), (3, None), (3, 63), (4, 7), (5, None), (8, 7), (10, None), (11, None), (12, None), (13, 1),
                      (16, None), (14, 65)):
        bad = list(good)
        bad[at] = value
        assert lib.nb200_layer_normalization_backward(*bad) == capi.EINVAL, (at, value)
    assert lib.nb200_layer_normalization_backward_scratch_floats(0, 0, 8) == 0
    assert lib.nb200_layer_normalization_backward_scratch_floats(0, 5, 8) >= 16


def test_vectors_off_word_boundaries_are_refused():
    lib = capi.load()
    calls = ((lib.nb200_layer_normalization, [None, 1, 1, 64, 4, 8, 8, None, None, 1e-5, 64, 8, None, None], (12, 13)),
             (lib.nb200_layer_normalization_backward, [None, 1, 1, 64, 8, 64, 4, 8, 8, None, 64, 64, 64, 8, 64, 64, 64], (10, 11, 16)))
    for function, good, places in calls:
        for at in places:
            bad = list(good)
            bad[at] = 66
            assert function(*bad) == capi.EINVAL, (function, at)
