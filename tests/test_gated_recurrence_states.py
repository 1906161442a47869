"""GatedRecurrence's gradients of 16-bit types take the states in fp32, whatever the result's rounding: nothing but a gradient's own
rounding and fp32 arithmetic may show.  The shapes reach the kernels that are fed by TMA in blocks and clusters of every size, with
sequences that end inside a box, in front of one and nowhere."""
import ctypes

import pytest
import torch

from neoml_b200 import _capi as capi
from neoml_b200 import ops
from test_gated_recurrence import _close, _made, _reference

HALVES = [torch.float16, torch.bfloat16]
TYPES = [torch.float32, *HALVES]


def _exact(z, f, i, *rest):
    """The 64-bit recurrence with bounds for states that are not rounded to 16 bits."""
    return _reference(z.float(), f.float(), None if i is None else i.float(), *rest)


def _inputs(t, b, n, c, gate):
    return (_made(t, b, n, c, seed=1), _made(t, b, n, c, seed=2, mean=3.0, std=2.0), _made(t, b, n, c, seed=3) if gate else None,
            _made(torch.float32, b, c, seed=4), _made(t, b, n, c, seed=7), _made(torch.float32, b, c, seed=8))


def _check(z, f, i, h0, lengths, dh, last_diff):
    h, last = ops.GatedRecurrence(z, f, i, initial_state=h0, lengths=lengths)
    grads = ops.GatedRecurrenceBackward(dh, h, z, f, i, initial_state=h0, final_state_diff=last_diff, lengths=lengths)
    clean = [x if x is None or lengths is None else torch.where((torch.arange(z.shape[1], device="cuda") < lengths[:, None])[..., None], x, 0.0)
             for x in (z, f, i, dh)]
    want = _exact(*clean[:3], h0, lengths, clean[3], last_diff)
    for name, got in zip(("h", "last", "dz", "df", "di", "dh0"), (h, last, *grads)):
        if got is not None:
            _close(got, want[name], name)
    if lengths is not None:
        behind = torch.arange(z.shape[1], device="cuda") >= lengths[:, None]
        assert all(x is None or (x[behind] == 0).all() for x in (h, *grads[:3]))
    return h, last, *grads


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("b,n,c", [(1, 1, 4), (2, 8, 6), (2, 9, 64), (3, 17, 33), (2, 70, 2), (2, 260, 127), (36, 8, 46)])
def test_unrounded_states(t, gate, b, n, c):
    z, f, i, h0, dh, last_diff = _inputs(t, b, n, c, gate)
    _check(z, f, i, h0, None, dh, last_diff)
    # strided operands
    wide = _made(t, n, b, c + 2, seed=9)
    _check(wide[..., :c].transpose(0, 1), f, i, h0, None, wide[..., 2:].transpose(0, 1), None)


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("gate", [False, True])
# blocks of two warps; clusters of two, four and eight blocks of four; of eight blocks of eight (16-bit types; fp32 has others)
@pytest.mark.parametrize("b,n,c", [(32, 70, 2048), (16, 300, 1024), (8, 600, 1024), (4, 1100, 1024), (3, 2305, 64)])
def test_long_sequences(t, gate, b, n, c):
    z, f, i, h0, dh, last_diff = _inputs(t, b, n, c, gate)
    ends = [n, 0, n - 1, 1, 7, 8, 9, 15, 16, 17, n // 2, 33, 64, 65, 31, 32]
    lengths = torch.tensor((ends * 2)[:b], dtype=torch.int32, device="cuda")
    if b < 16:   # ends around those of a round
        more = torch.tensor([n, n // 2 + 1, 1025, 511, 513, 129, 15, 0], dtype=torch.int32, device="cuda").clamp(max=n)
        lengths = more[:b].clone()
    for x in (z, f, i, dh):
        if x is not None:
            x[torch.arange(n, device="cuda") >= lengths[:, None]] = float("nan")
    _check(z, f, i, h0, lengths, dh, last_diff)
    if b <= 8:
        z, f, i, h0, dh, last_diff = _inputs(t, b, n, c, gate)
        _check(z, f, i, None, None, dh, None)


@pytest.mark.gpu
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("n,c", [(40, 10), (40, 7), (2100, 64)])
def test_states_beyond_a_half(gate, n, c):
    """States that a half does not hold come out infinite, as it rounds them, and leave the gradients finite."""
    t = torch.float16
    z = _made(t, 2, n, c, seed=1).abs() * 1000 + 40000
    f = torch.full((2, n, c), 7.0, dtype=t, device="cuda")
    i = torch.full((2, n, c), 3.0, dtype=t, device="cuda") if gate else None
    h0 = torch.full((2, c), 1e5, device="cuda")
    dh = _made(t, 2, n, c, seed=2, std=2.0 ** -8)
    h, last = ops.GatedRecurrence(z, f, i, initial_state=h0)
    assert h[:, :8].isinf().all() and last.isfinite().all()
    grads = ops.GatedRecurrenceBackward(dh, h, z, f, i, initial_state=h0)
    want = _exact(z, f, i, h0, None, dh, None)
    for name, got in zip(("dz", "df", "di", "dh0"), grads):
        if got is not None:
            assert want[name][0].abs().max() < 65000
            _close(got, want[name], name)


@pytest.mark.gpu
@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("gate", [False, True])
def test_repeats_and_graph(t, gate):
    z, f, i, h0, dh, last_diff = _inputs(t, 4, 1100, 1024, gate)
    h, _ = ops.GatedRecurrence(z, f, i, initial_state=h0)

    def step():
        return ops.GatedRecurrenceBackward(dh, h, z, f, i, initial_state=h0, final_state_diff=last_diff)
    first = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        got = step()
    for _ in range(3):
        graph.replay()
        again = step()
        torch.cuda.synchronize()
        assert all((x is None and y is None) or (torch.equal(x, y) and torch.equal(x, w)) for x, y, w in zip(got, first, again))


def test_gradients_in_place_of_an_operand_are_refused():
    """Before any device is asked for."""
    lib, e = capi.load(), 2 * 3 * 4 * 2   # bytes of [2][3][4] halves
    desc = ctypes.byref(capi.RecurrenceDesc(2, 3, 4, 12, 4, 12, 4, 12, 4))
    far = 1 << 20
    good = [None, 1, desc, far, 12, 4, far + 2 * e, far + 4 * e, far + 6 * e, far + 8 * e, None, None, None, far + 10 * e, far + 12 * e, far + 14 * e, None]
    for operand in (3, 7, 8, 9):
        for off in (0, 2 - e, e - 2):
            bad = list(good)
            bad[13] = good[operand] + off
            assert lib.nb200_gated_recurrence_backward(*bad) == capi.EINVAL, (operand, off)
    for off in (-e, e):
        near = list(good)
        near[13] = good[7] + off
        if not torch.cuda.is_available():   # nothing to refuse but the device
            assert lib.nb200_gated_recurrence_backward(*near) == capi.ENODEVICE


def test_sizes_beyond_the_limits_are_refused():
    lib = capi.load()
    for head in ((65536, 3, 4), (1, 2 ** 30 + 1, 1), (1, 1, 2 ** 30 + 1), (1, 1, 2 ** 31 - 1)):
        desc = ctypes.byref(capi.RecurrenceDesc(*head, 0, 0, 0, 0, 0, 0))
        assert lib.nb200_gated_recurrence(None, 1, desc, 64, 64, None, None, None, 64, None) == capi.ETOOBIG, head
        backward = [None, 0, desc, 64, 0, 0, 64, 64, 64, None, None, None, None, 64, 64, None, None]
        assert lib.nb200_gated_recurrence_backward(*backward) == capi.ETOOBIG, head


@pytest.mark.gpu
def test_no_wait_gave_up():
    assert capi.load().nb200_device_status(None, 0) == 0
