"""The language-model operators one after another, as a training step and a serving step of a small recurrent model call them:
normalisation, recurrence, normalisation, the vocabulary's cross entropy, and distillation on logits of the library's product.
The step's gradients are compared with torch's automatic ones in 64 bits."""
import math

import pytest
import torch

from neoml_b200 import ops

TYPES = [torch.float32, torch.float16, torch.bfloat16]
B, L, C, V, K = 6, 75, 96, 1003, 9
TAU = 2.0


def _made(t, *shape, seed, std=1.0, mean=0.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(t)


def _model(t, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed + 50)
    return {
        "x": _made(t, B, L, C, seed=seed + 1), "gates": _made(t, B, L, C, seed=seed + 2, mean=2.0), "inputs": _made(t, B, L, C, seed=seed + 3),
        "scale1": _made(torch.float32, C, seed=seed + 4, std=0.2, mean=1.0), "free1": _made(torch.float32, C, seed=seed + 5, std=0.2),
        "scale2": _made(torch.float32, C, seed=seed + 6, std=0.2, mean=1.0), "free2": _made(torch.float32, C, seed=seed + 7, std=0.2),
        "head": _made(t, V, C, seed=seed + 8, std=2 / math.sqrt(C)), "state": _made(torch.float32, B, C, seed=seed + 9),
    }, {
        "lengths": torch.randint(1, L + 1, (B,), generator=g, device="cuda", dtype=torch.int32),
        "labels": torch.randint(0, V, (B, L), generator=g, device="cuda", dtype=torch.int32),
        "top": _made(t, B, L, K, seed=seed + 10, std=2.0),
        "index": torch.randint(0, V, (B, L, K), generator=g, device="cuda", dtype=torch.int32),
    }


def _step(m, d):
    """Losses per token and every gradient, the loss being the mean cross entropy plus the mean distillation."""
    inside = torch.arange(L, device="cuda") < d["lengths"][:, None]
    labels = torch.where(inside, d["labels"], -1).int()
    index = torch.where(inside[..., None], d["index"], -1).int()
    y1, mean1, inv1 = ops.LayerNormalization(m["x"], m["scale1"], m["free1"])
    h, last = ops.GatedRecurrence(y1, m["gates"], m["inputs"], initial_state=m["state"], lengths=d["lengths"])
    y2, mean2, inv2 = ops.LayerNormalization(h, m["scale2"], m["free2"])
    loss, log_sum = ops.VocabularyCrossEntropy(y2, m["head"], labels)
    # distillation wants the logits themselves: the library's product of fp32 matrices
    logits = ops.MultiplyMatrixByTransposedMatrix(y2.float().view(B * L, C), m["head"].float()).view(B, L, V)
    far, far_sum = ops.DistillationLoss(logits, d["top"].float(), index, temperature=TAU)
    each = inside / inside.sum()
    dy, dhead = ops.VocabularyCrossEntropyBackward(each.float(), y2, m["head"], labels, log_sum)
    dlogits = ops.DistillationLossBackward(each.float(), logits, d["top"].float(), index, far_sum, temperature=TAU).view(B * L, V)
    dy2 = dy.float() + ops.MultiplyMatrixByMatrix(dlogits, m["head"].float()).view(B, L, C)
    dhead2 = dhead.float() + ops.MultiplyMatrixByMatrix(dlogits.t().contiguous(), y2.float().view(B * L, C))
    dh, dscale2, dfree2 = ops.LayerNormalizationBackward(dy2.to(h.dtype), h, mean2, inv2, m["scale2"])
    dy1, dgates, dinputs, dstate = ops.GatedRecurrenceBackward(dh, h, y1, m["gates"], m["inputs"], initial_state=m["state"],
                                                               lengths=d["lengths"])
    dx, dscale1, dfree1 = ops.LayerNormalizationBackward(dy1, m["x"], mean1, inv1, m["scale1"])
    return loss, far, last, {"x": dx, "gates": dgates, "inputs": dinputs, "scale1": dscale1, "free1": dfree1, "scale2": dscale2,
                             "free2": dfree2, "head": dhead2, "state": dstate}


def _reference(m, d):
    p = {k: v.double().requires_grad_() for k, v in m.items()}
    inside = torch.arange(L, device="cuda") < d["lengths"][:, None]

    def norm(x, scale, free):
        centred = x - x.mean(-1, keepdim=True)
        return centred / torch.sqrt((centred ** 2).mean(-1, keepdim=True) + 1e-5) * scale + free
    y = norm(p["x"], p["scale1"], p["free1"])
    keep, take = torch.sigmoid(p["gates"]), torch.sigmoid(p["inputs"])
    h, states = p["state"], []
    for t in range(L):
        h = torch.where(inside[:, t, None], keep[:, t] * h + take[:, t] * y[:, t], h)
        states.append(torch.where(inside[:, t, None], h, 0.0))
    z = norm(torch.stack(states, 1), p["scale2"], p["free2"]) @ p["head"].T
    loss = torch.logsumexp(z, -1) - z.gather(-1, d["labels"].long()[..., None])[..., 0]
    q = torch.softmax(d["top"].double() / TAU, -1)
    log_q = torch.log_softmax(z / TAU, -1).gather(-1, d["index"].long())
    far = TAU ** 2 * (q * (torch.log(q) - log_q)).sum(-1)
    loss, far = torch.where(inside, loss, 0.0), torch.where(inside, far, 0.0)
    ((loss + far).sum() / inside.sum()).backward()
    return loss, far, h, {k: v.grad for k, v in p.items()}


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
def test_training_step(t):
    m, d = _model(t)
    loss, far, last, grads = _step(m, d)
    want = _reference(m, d)
    # what a rounding to the type at every operator's border leaves of a value: some ten in a row, each half a step, and the product's
    # 1e-5 in fp32; the norms of whole tensors average them
    bound = 10 * torch.finfo(t).eps / 2 + 2e-5
    for got, wanted in ((loss, want[0]), (far, want[1]), (last, want[2])):
        assert (got.double() - wanted).norm() <= bound * wanted.norm()
    for name, grad in grads.items():
        wanted = want[3][name]
        assert grad.shape == wanted.shape and grad.isfinite().all(), name
        assert (grad.double() - wanted).norm() <= bound * wanted.norm(), name


@pytest.mark.gpu
def test_training_step_in_a_graph():
    """Captured once, replayed on other data, while an eager step runs beside it on another stream."""
    m, d = _model(torch.bfloat16)
    _step(m, d)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        loss, far, last, grads = _step(m, d)
    other, _ = _model(torch.bfloat16, 100)
    for k in m:
        m[k].copy_(other[k])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph.replay()
    with torch.cuda.stream(side):
        eager = _step(m, d)
    torch.cuda.synchronize()
    assert torch.equal(loss, eager[0]) and torch.equal(far, eager[1]) and torch.equal(last, eager[2])
    for name in grads:
        assert torch.equal(grads[name], eager[3][name]), name


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
def test_tokens_one_at_a_time(t):
    """Serving: one token of every sequence per call, the states in place, against the same tokens in one call."""
    m, _ = _model(t)
    state, logs = m["state"].clone(), []
    y = ops.LayerNormalization(m["x"], m["scale1"], m["free1"])[0]
    h, last = ops.GatedRecurrence(y, m["gates"], m["inputs"], initial_state=m["state"])
    whole = ops.LayerNormalization(h, m["scale2"], m["free2"])[0]
    labels = torch.full((B, 1), 5, dtype=torch.int32, device="cuda")
    for k in range(L):
        cut = slice(k, k + 1)
        y = ops.LayerNormalization(m["x"][:, cut].contiguous(), m["scale1"], m["free1"])[0]
        h, _ = ops.GatedRecurrence(y, m["gates"][:, cut], m["inputs"][:, cut], initial_state=state, final_state=state)
        logs.append(ops.VocabularyCrossEntropy(ops.LayerNormalization(h, m["scale2"], m["free2"])[0], m["head"], labels)[0])
    want, _ = ops.VocabularyCrossEntropy(whole, m["head"], labels.expand(B, L).contiguous())
    # both round a state once per step, sometimes to the neighbouring value: a step of the type through the normalisation and the head
    step = torch.finfo(t).eps
    assert (torch.cat(logs, 1) - want).abs().max() <= 16 * step * want.abs().max() + 1e-5
    assert (state - last).abs().max() <= 2.0 ** -18 * last.abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
def test_same_bits_without_the_native_half(monkeypatch, t):
    m, d = _model(t)
    want = _step(m, d)
    monkeypatch.setattr(ops, "_native_module", ops._DeclinesAll())
    got = _step(m, d)
    for a, b in zip((*got[:3], *got[3].values()), (*want[:3], *want[3].values())):
        assert a.shape == b.shape and a.dtype == b.dtype and torch.equal(a, b)


@pytest.mark.gpu
def test_parameters_and_other_streams():
    """torch's parameters are taken like tensors, nothing is recorded for its automatic gradients, and a call runs on the stream
    that is current where it is made."""
    m, d = _model(torch.bfloat16)
    want = _step(m, d)
    p = {k: torch.nn.Parameter(v) for k, v in m.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, mean, inv = ops.LayerNormalization(p["x"], p["scale1"], p["free1"])
        h, last = ops.GatedRecurrence(y, p["gates"], p["inputs"], initial_state=p["state"], lengths=d["lengths"])
        z, _, _ = ops.LayerNormalization(h, p["scale2"], p["free2"])
        inside = torch.arange(L, device="cuda") < d["lengths"][:, None]
        loss, log_sum = ops.VocabularyCrossEntropy(z, p["head"], torch.where(inside, d["labels"], -1).int())
    side.synchronize()
    assert torch.equal(loss, want[0]) and torch.equal(last, want[2])
    assert not any(t.requires_grad for t in (y, mean, inv, h, last, loss, log_sum))
