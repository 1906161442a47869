"""GatedRecurrence and its backward pass against a step-by-step 64-bit recurrence, with bounds that follow each state's own
rounding errors through time."""
import ctypes

import pytest
import torch

from neoml_b200 import _capi as capi
from neoml_b200 import ops

TYPES = [torch.float32, torch.float16, torch.bfloat16]
STEP = 2.0 ** -24


def _made(t, *shape, seed, mean=0.0, std=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(t)


def _case(t, b, n, c, gate, ragged=False, seed=0):
    z, f = _made(t, b, n, c, seed=seed + 1), _made(t, b, n, c, seed=seed + 2, mean=3.0, std=2.0)
    i = _made(t, b, n, c, seed=seed + 3) if gate else None
    h0 = _made(torch.float32, b, c, seed=seed + 4)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed + 5)
    lengths = torch.randint(0, n + 1, (b,), generator=g, device="cuda", dtype=torch.int32) if ragged else None
    return z, f, i, h0, lengths


def _gates(f, i):
    f = f.double()
    a = torch.sigmoid(f)
    u = torch.sigmoid(-f) if i is None else torch.sigmoid(i.double())
    # exp's error grows with its argument; a sum, a quotient and the products around them
    noise = (16 + 3 * f.abs() + (0 if i is None else 3 * i.double().abs())) * STEP
    return a, u, noise


def _reference(z, f, i, h0, lengths, dh=None, last_diff=None):
    """Values and what each may be off by before its own rounding."""
    b, n, c = z.shape
    a, u, noise = _gates(f, i)
    zd = z.double()
    long = torch.full((b,), n, device=z.device) if lengths is None else lengths.long()
    on = (torch.arange(n, device=z.device) < long[:, None]).double()
    h = torch.zeros(b, c, dtype=torch.float64, device=z.device) if h0 is None else h0.double()
    off = torch.zeros_like(h)
    size = h.abs()
    states, offs, befores = [], [], []
    for t in range(n):
        m = on[:, t, None]
        befores.append((h, off, size))
        new = a[:, t] * h + u[:, t] * zd[:, t]
        new_size = a[:, t] * size + u[:, t] * zd[:, t].abs()
        new_off = a[:, t] * off + noise[:, t] * new_size
        h, size, off = m * new + (1 - m) * h, m * new_size + (1 - m) * size, m * new_off + (1 - m) * off
        states.append(m * new)
        offs.append(m * new_off)
    stack = lambda s: torch.stack(s, 1) if s else torch.zeros_like(zd)  # noqa: E731
    out = {"h": (stack(states), stack(offs)), "last": (h, off)}
    if dh is None:
        return out
    half = torch.finfo(z.dtype).eps / 2
    s = torch.zeros_like(h) if last_diff is None else last_diff.double()
    s_off, s_size = torch.zeros_like(s), s.abs()
    grads = {k: ([], []) for k in ("dz", "df", "di")}
    for t in reversed(range(n)):
        m = on[:, t, None]
        S, S_size = (s + dh[:, t].double()) * m, (s_size + dh[:, t].double().abs()) * m
        S_off = (s_off + STEP * S_size) * m
        before, b_off, b_size = befores[t]
        # the backward pass reads the states as they were rounded
        b_off = b_off + half * before.abs() + (2.0 ** -25 if z.dtype == torch.float16 else 0.0)
        slope, w = a[:, t] * (1 - a[:, t]), 2 * noise[:, t]
        value = before if i is not None else before - zd[:, t]
        v_size = before.abs() if i is not None else before.abs() + zd[:, t].abs()
        for name, v, o in (("dz", S * u[:, t], S_off * u[:, t] + w * S_size * u[:, t]),
                           ("df", S * value * slope, slope * (S_off * v_size + S_size * (b_off + w * v_size))),
                           ("di", S * zd[:, t] * u[:, t] * (1 - u[:, t]), (S_off + w * S_size) * zd[:, t].abs() * u[:, t] * (1 - u[:, t]))):
            grads[name][0].append(v)
            grads[name][1].append(o)
        s, s_size = m * a[:, t] * S + (1 - m) * s, m * a[:, t] * S_size + (1 - m) * s_size
        s_off = m * (a[:, t] * S_off + w * a[:, t] * S_size) + (1 - m) * s_off
    for name, (v, o) in grads.items():
        out[name] = (stack(v[::-1]), stack(o[::-1]))
    out["dh0"] = (s, s_off)
    return out


def _close(got, want, name=""):
    value, off = want
    # stretches of time are folded before they meet: every product is formed from two sides
    bound = torch.finfo(got.dtype).eps / 2 * value.abs() + 3 * off + 2.0 ** -100 + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    excess = (got.double() - value).abs() - bound
    assert got.shape == value.shape
    assert got.numel() == 0 or excess.max().item() <= 0.0, f"{name}: {excess.max().item()} more than allowed"


def _check(t, z, f, i, h0, lengths, dh, last_diff):
    h, last = ops.GatedRecurrence(z, f, i, initial_state=h0, lengths=lengths)
    assert h.dtype == t and last.dtype == torch.float32
    dz, df, di, dh0 = ops.GatedRecurrenceBackward(dh, h, z, f, i, initial_state=h0, final_state_diff=last_diff, lengths=lengths)
    want = _reference(z, f, i, h0, lengths, dh, last_diff)
    for name, got in (("h", h), ("last", last), ("dz", dz), ("df", df), ("di", di), ("dh0", dh0)):
        if got is not None:
            _close(got, want[name], name)
    assert (di is None) == (i is None)
    if lengths is not None:
        behind = torch.arange(z.shape[1], device="cuda") >= lengths[:, None]
        for got in (h, dz, df, di):
            assert got is None or (got[behind] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("b,n,c", [(1, 1, 1), (16, 1, 2048), (2, 2, 3), (3, 8, 64), (1, 9, 33), (5, 127, 65), (2, 129, 66), (1, 1031, 96),
                                   (3, 260, 127), (1, 2500, 5), (300, 17, 10)])
def test_against_64_bits(t, gate, b, n, c):
    _check(t, *_case(t, b, n, c, gate), _made(t, b, n, c, seed=7), _made(torch.float32, b, c, seed=8))


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("b,n,c", [(7, 33, 40), (3, 1500, 34), (40, 128, 130)])
def test_ragged(t, gate, b, n, c):
    z, f, i, h0, lengths = _case(t, b, n, c, gate, True)
    lengths[0], lengths[-1] = 0, n
    dh, last_diff = _made(t, b, n, c, seed=7), _made(torch.float32, b, c, seed=8)
    _check(t, z, f, i, h0, lengths, dh, last_diff)
    # what lies behind a sequence is not looked at
    before = ops.GatedRecurrence(z, f, i, initial_state=h0, lengths=lengths)
    grads = ops.GatedRecurrenceBackward(dh, before[0], z, f, i, initial_state=h0, final_state_diff=last_diff, lengths=lengths)
    behind = torch.arange(n, device="cuda") >= lengths[:, None]
    for x in (z, f, i, dh):
        if x is not None:
            x[behind] = float("nan")
    after = ops.GatedRecurrence(z, f, i, initial_state=h0, lengths=lengths)
    again = ops.GatedRecurrenceBackward(dh, after[0], z, f, i, initial_state=h0, final_state_diff=last_diff, lengths=lengths)
    for x, y in zip((*before, *grads), (*after, *again)):
        assert (x is None and y is None) or torch.equal(x, y)
    # lengths outside the range count as its ends
    outside = torch.where(lengths == 0, -5, torch.where(lengths == n, n + 9, lengths)).int()
    assert torch.equal(ops.GatedRecurrence(z, f, i, initial_state=h0, lengths=outside)[0], after[0])


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
def test_no_states_and_no_steps(t):
    z, f, i, h0, _ = _case(t, 2, 50, 31, True)
    _check(t, z, f, i, None, None, _made(t, 2, 50, 31, seed=7), None)
    none = torch.empty(2, 0, 31, dtype=t, device="cuda")
    h, last = ops.GatedRecurrence(none, none, initial_state=h0)
    assert h.shape == none.shape and torch.equal(last, h0)
    assert torch.equal(ops.GatedRecurrenceBackward(none, h, none, none, initial_state=h0, final_state_diff=h0)[3], h0)
    empty = torch.empty(0, 5, 31, dtype=t, device="cuda")
    assert ops.GatedRecurrence(empty, empty)[1].shape == (0, 31)


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
def test_strided_and_expanded(t):
    b, n, c = 3, 70, 48
    wide = _made(t, b, n, 3 * c + 1, seed=1, mean=1.0)
    z, f, i = wide[..., 1:c + 1], wide[..., c + 1:2 * c + 1], wide[..., 2 * c + 1:]
    dh, last_diff, h0 = _made(t, n, b, c, seed=7).transpose(0, 1), _made(torch.float32, b, c, seed=8), _made(torch.float32, b, c, seed=9)
    _check(t, z, f, i, h0, None, dh, last_diff)
    _check(t, z, f[:1, :1].expand(b, n, c), f[:, :1].expand(b, n, c), h0, None, dh[:1].expand(b, n, c), None)
    even = _made(t, b, n, 3 * c, seed=1)
    _check(t, even[..., :c], even[..., c:2 * c], even[..., 2 * c:], h0, None, dh, last_diff)


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("gate", [False, True])
def test_tokens_one_at_a_time(t, gate):
    """Serving: the state goes from call to call, in place, and arrives where one call over all steps arrives."""
    b, n, c = 4, 37, 130
    z, f, i, h0, _ = _case(t, b, n, c, gate)
    whole, last = ops.GatedRecurrence(z, f, i, initial_state=h0)
    state = h0.clone()
    want = _reference(z, f, i, h0, None)
    for k in range(n):
        cut = [None if x is None else x[:, k:k + 1] for x in (z, f, i)]
        got, same = ops.GatedRecurrence(*cut, initial_state=state, final_state=state)
        assert same is state
        _close(got[:, 0], tuple(w[:, k] for w in want["h"]))
    _close(state, want["last"])
    _close(last, want["last"])


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n", [24, 300, 2100])
def test_state_in_place_over_many_steps(t, n):
    """Few channels: several blocks share a sequence and read the state that one of them replaces."""
    b, c = 1, 64
    z, f, i, h0, _ = _case(t, b, n, c, True)
    want, last = ops.GatedRecurrence(z, f, i, initial_state=h0)
    for _ in range(20):
        state = h0.clone()
        got, same = ops.GatedRecurrence(z, f, i, initial_state=state, final_state=state)
        assert same is state and torch.equal(got, want) and torch.equal(state, last)


@pytest.mark.gpu
def test_extreme_gates():
    inf = float("inf")
    z = torch.full((1, 4, 3), 2.0, device="cuda")
    f = torch.tensor([inf, -inf, 200.0], device="cuda").expand(1, 4, 3).contiguous()
    h0 = torch.full((1, 3), 5.0, device="cuda")
    h, last = ops.GatedRecurrence(z, f, initial_state=h0)
    assert (h == torch.tensor([5.0, 2.0, 5.0], device="cuda")).all()
    grads = ops.GatedRecurrenceBackward(torch.ones_like(h), h, z, f, initial_state=h0)
    assert (grads[0] == torch.tensor([0.0, 1.0, 0.0], device="cuda")).all() and (grads[1] == 0).all()
    assert torch.equal(grads[3], torch.tensor([[4.0, 0.0, 4.0]], device="cuda"))


@pytest.mark.gpu
def test_gradient_is_the_slope():
    b, n, c = 2, 20, 6
    z, f, i, h0, _ = _case(torch.float32, b, n, c, True)
    f = f - 2.0
    dh, last_diff = _made(torch.float32, b, n, c, seed=7), _made(torch.float32, b, c, seed=8)
    h, _ = ops.GatedRecurrence(z, f, i, initial_state=h0)
    grads = ops.GatedRecurrenceBackward(dh, h, z, f, i, initial_state=h0, final_state_diff=last_diff)
    step = 2.0 ** -7
    for k, grad in enumerate(grads):
        operands = [z, f, i, h0]
        direction = _made(torch.float32, *operands[k].shape, seed=20 + k)
        value = []
        for sign in (1, -1):
            operands[k] = [z, f, i, h0][k] + sign * step * direction
            r, last = ops.GatedRecurrence(*operands[:3], initial_state=operands[3])
            value.append((r.double() * dh.double()).sum() + (last.double() * last_diff.double()).sum())
        slope, want = (value[0] - value[1]) / (2 * step), (grad.double() * direction.double()).sum()
        # third derivatives along a direction of ones: some thirty times the first, over six; differences of fp32 states
        assert abs(slope - want) <= (30 * step * step + 2.0 ** -22 / step * 8) * (grad.double() * direction.double()).abs().sum()


@pytest.mark.gpu
def test_graph_stream_and_repeats():
    t, b, n, c = torch.bfloat16, 2, 600, 128
    z, f, i, h0, _ = _case(t, b, n, c, True)
    dh = _made(t, b, n, c, seed=7)

    def step():
        h, last = ops.GatedRecurrence(z, f, i, initial_state=h0)
        return (h, last, *ops.GatedRecurrenceBackward(dh, h, z, f, i, initial_state=h0))
    first = step()
    assert all(torch.equal(x, y) for x, y in zip(first, step()))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        got = step()
    z.copy_(_made(t, b, n, c, seed=11))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, step())) and not torch.equal(got[0], first[0])


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("gate", [False, True])
def test_long_results_off_word_boundaries(t, gate):
    """Long sequences whose operands are aligned and whose results begin one element further."""
    b, n, c = 2, 2100, 64
    z, f, i, h0, _ = _case(t, b, n, c, gate)
    dh = _made(t, b, n, c, seed=7)

    def off():
        return torch.empty(b * n * c + 1, dtype=t, device="cuda")[1:].view(b, n, c)
    h, last = ops.GatedRecurrence(z, f, i, initial_state=h0, result=off())
    want = _reference(z, f, i, h0, None, dh, None)
    _close(h, want["h"], "h")
    _close(last, want["last"], "last")
    h = h.clone()
    dz, df, di, dh0 = off(), off(), off() if gate else None, torch.empty_like(h0)
    desc = capi.RecurrenceDesc(b, n, c, *(n * c, c) * 3)
    at = lambda x: None if x is None else x.data_ptr()  # noqa: E731
    assert capi.load().nb200_gated_recurrence_backward(
        torch.cuda.current_stream().cuda_stream, ops._TYPES[t], ctypes.byref(desc), at(dh), n * c, c, at(h), at(z), at(f), at(i), at(h0), None,
        None, at(dz), at(df), at(di), at(dh0)) == capi.OK
    for name, got in (("dz", dz), ("df", df), ("di", di), ("dh0", dh0)):
        if got is not None:
            _close(got, want[name], name)


def test_refusals():
    z, s = torch.zeros(2, 3, 4), torch.zeros(2, 4)
    with pytest.raises(AssertionError, match="CUDA device"):
        ops.GatedRecurrence(z, z)
    with pytest.raises(AssertionError, match=r"\[batch, length, channels\]"):
        ops.GatedRecurrence(s, s)
    with pytest.raises(AssertionError, match="fp32, fp16 or bf16"):
        ops.GatedRecurrence(z.double(), z.double())
    with pytest.raises(AssertionError, match="float32"):
        ops.GatedRecurrence(z, z.half())
    with pytest.raises(AssertionError, match=r"\[2, 3, 4\]"):
        ops.GatedRecurrence(z, torch.zeros(2, 3, 5))
    with pytest.raises(AssertionError, match="adjacent"):
        ops.GatedRecurrence(z.transpose(1, 2), z.transpose(1, 2))
    with pytest.raises(AssertionError, match="dense"):
        ops.GatedRecurrence(z, z, result=torch.zeros(2, 3, 8)[..., :4])


def test_argument_validation_needs_no_device():
    import ctypes as C
    lib = capi.load()

    def desc(*head, strides=(0,) * 6):
        return C.byref(capi.RecurrenceDesc(*head, *strides))
    forward = [None, 0, desc(2, 3, 4), 64, 64, None, None, None, 64, None]
    for at, value in ((1, 3), (2, None), (2, desc(-1, 3, 4)), (2, desc(2, -3, 4)), (2, desc(2, 3, 4, strides=(0, -1, 0, 0, 0, 0))), (3, None),
                      (4, None), (8, None), (3, 66), (5, 66), (6, 66), (9, 66)):
        bad = list(forward)
        bad[at] = value
        assert lib.nb200_gated_recurrence(*bad) == capi.EINVAL, (at, value)
    forward[2] = desc(70000, 3, 4)
    assert lib.nb200_gated_recurrence(*forward) == capi.ETOOBIG
    forward[2] = desc(0, 3, 4)
    assert lib.nb200_gated_recurrence(*forward) == capi.OK
    backward = [None, 1, desc(2, 3, 4), 64, 0, 0, 64, 64, 64, None, None, None, None, 64, 64, None, None]
    for at, value in ((1, -1), (3, None), (4, -2), (6, None), (7, None), (8, None), (9, 64), (13, None), (14, None), (15, 64), (6, 65), (16, 65)):
        bad = list(backward)
        bad[at] = value
        assert lib.nb200_gated_recurrence_backward(*bad) == capi.EINVAL, (at, value)


def test_vectors_off_word_boundaries_are_refused():
    lib = capi.load()
    desc = ctypes.byref(capi.RecurrenceDesc(2, 3, 4, 0, 0, 0, 0, 0, 0))
    calls = ((lib.nb200_gated_recurrence, [None, 1, desc, 64, 64, None, None, None, 64, None], (6, 7, 9)),
             (lib.nb200_gated_recurrence_backward, [None, 1, desc, 64, 0, 0, 64, 64, 64, None, None, None, None, 64, 64, None, None], (10, 11, 12, 16)))
    for function, good, places in calls:
        for at in places:
            bad = list(good)
            bad[at] = 66
            assert function(*bad) == capi.EINVAL, (function, at)
