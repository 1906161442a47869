"""What a language model's training step and its serving step ask of the library besides products and attention, as cases
that can be timed and compared.

A case is a dict of plain values with an `op`:
  normalization   LayerNormalization (pass "forward") and its backward pass (pass "step": both, as a layer in training runs)
  recurrence      GatedRecurrence over [batch, length, channels] (pass "forward": a prompt, or one token with its state;
                  pass "step": with the backward pass)
  entropy         VocabularyCrossEntropy of hidden rows against a vocabulary's weights (pass "forward": scoring a text;
                  pass "step": with the gradients of rows and weights)
  distillation    DistillationLoss of logits against a teacher's top logits (pass "forward" or "step")
`run` computes them in plain torch operations, or with `own` through neoml_b200.ops.
"""
from __future__ import annotations

import math

import torch

own = False

EPSILON = 1e-5
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed() -> list[dict]:
    return [
        # the rows of a few tokens that are decoded together: a launch or two, bound by latency
        {"name": "norm_token", "op": "normalization", "pass": "forward", "type": "bfloat16", "rows": 8, "width": 768},
        # the encoder of the benchmark (64 sequences of 512, 768 wide) in the library's own precision
        {"name": "norm_encoder_fp32", "op": "normalization", "pass": "forward", "type": "float32", "rows": 32768, "width": 768},
        # a training step of a wide layer whose parameters are kept in 32 bits
        {"name": "norm_step_wide", "op": "normalization", "pass": "step", "type": "bfloat16", "rows": 16384, "width": 4096},
        # one token of each of 16 conversations: the states go in and come out
        {"name": "recurrence_token", "op": "recurrence", "pass": "forward", "type": "bfloat16", "batch": 16, "length": 1,
         "channels": 2048, "input_gate": True, "ragged": False},
        # long prompts, few of them: the work has to be split along the time axis
        {"name": "recurrence_long", "op": "recurrence", "pass": "forward", "type": "bfloat16", "batch": 2, "length": 16384,
         "channels": 2048, "input_gate": False, "ragged": False},
        # a training step on a padded batch of texts with an odd channel count
        {"name": "recurrence_step_ragged", "op": "recurrence", "pass": "step", "type": "float32", "batch": 24, "length": 1021,
         "channels": 1025, "input_gate": True, "ragged": True},
        # a training step of ordinary sizes in mixed precision
        {"name": "recurrence_step", "op": "recurrence", "pass": "step", "type": "bfloat16", "batch": 16, "length": 2048,
         "channels": 2048, "input_gate": False, "ragged": False},
        # scoring one short text: few rows, the weights are read once
        {"name": "entropy_score", "op": "entropy", "pass": "forward", "type": "bfloat16", "rows": 48, "width": 1024, "vocabulary": 32000},
        # the head of a training step: a large batch of tokens, an odd vocabulary
        {"name": "entropy_step", "op": "entropy", "pass": "step", "type": "bfloat16", "rows": 8192, "width": 2048, "vocabulary": 50257},
        # the head of a small model in the library's own precision
        {"name": "entropy_step_fp32", "op": "entropy", "pass": "step", "type": "float32", "rows": 1023, "width": 768, "vocabulary": 30011},
        # a student's training step against 64 kept logits of its teacher
        {"name": "distillation_step", "op": "distillation", "pass": "step", "type": "bfloat16", "rows": 4096, "vocabulary": 50257, "kept": 64},
        # how far a student is from its teacher on a short text
        {"name": "distillation_score", "op": "distillation", "pass": "forward", "type": "float16", "rows": 17, "vocabulary": 32003, "kept": 100},
    ]


def _log_int(rng, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng) -> dict:
    op = rng.choice(["normalization", "recurrence", "entropy", "distillation"])
    case = {"op": op, "pass": rng.choice(["forward", "step"]), "type": rng.choice(list(TYPES))}
    while True:
        if op == "normalization":
            case.update(rows=_log_int(rng, 1, 40000), width=_log_int(rng, 1, 20000))
            if case["rows"] * case["width"] <= 16384 * 4096:
                return case
        elif op == "recurrence":
            case.update(batch=_log_int(rng, 1, 64), length=_log_int(rng, 1, 16384), channels=_log_int(rng, 1, 4096),
                        input_gate=rng.random() < 0.5, ragged=rng.random() < 0.5)
            if case["batch"] * case["length"] * case["channels"] <= 2 * 16384 * 2048:
                return case
        elif op == "entropy":
            case.update(rows=_log_int(rng, 1, 8192), width=_log_int(rng, 8, 4096), vocabulary=_log_int(rng, 50, 130000))
            # 32-bit products take several times as long as those of 16-bit operands
            most = 8192 * 2048 * 50257 // (8 if case["type"] == "float32" else 1)
            if case["rows"] * case["width"] * case["vocabulary"] <= most and case["rows"] * case["vocabulary"] <= 8192 * 50257:
                return case
        else:
            case.update(rows=_log_int(rng, 1, 8192), vocabulary=_log_int(rng, 300, 130000), kept=_log_int(rng, 1, 256))
            if case["rows"] * case["vocabulary"] <= 4096 * 50257:
                return case


def _loss_scale(case: dict) -> float:
    """What a trainer multiplies the loss by: half precision would otherwise lose small gradients."""
    return 4096.0 if case["type"] == "float16" else 1.0


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*size, mean=0.0, std=1.0, dtype=t):
        return torch.randn(*size, generator=g, device="cuda").mul_(std).add_(mean).to(dtype)

    def whole(low, high, *size):
        return torch.randint(low, high, size, generator=g, device="cuda", dtype=torch.int32)

    s = {"case": case}
    if case["op"] == "normalization":
        rows, width = case["rows"], case["width"]
        # activations of a residual stream: a common offset and rows of differing size
        s["x"] = (torch.randn(rows, width, generator=g, device="cuda") * torch.exp(torch.randn(rows, 1, generator=g, device="cuda") * 0.5)
                  + 0.5).to(t)
        # the parameters of a layer stay in 32 bits
        s["scale"] = normal(width, mean=1.0, std=0.2, dtype=torch.float32)
        s["free_term"] = normal(width, std=0.2, dtype=torch.float32)
        if case["pass"] == "step":
            s["dy"] = normal(rows, width)
    elif case["op"] == "recurrence":
        b, n, c = case["batch"], case["length"], case["channels"]
        s["z"] = normal(b, n, c)
        # forget gates between a half and 0.999: a memory of a few to a thousand tokens
        s["f"] = normal(b, n, c, mean=3.0, std=1.5)
        s["i"] = normal(b, n, c) if case["input_gate"] else None
        s["h0"] = normal(b, c, dtype=torch.float32)
        s["lengths"] = whole(0, n + 1, b) if case["ragged"] else None
        if case["pass"] == "step":
            s["dh"] = normal(b, n, c)
            s["d_last"] = normal(b, c, dtype=torch.float32)
    elif case["op"] == "entropy":
        rows, d, v = case["rows"], case["width"], case["vocabulary"]
        s["x"] = normal(rows, d)
        s["w"] = normal(v, d, std=2.0 / math.sqrt(d))   # logits of a deviation of two
        s["labels"] = whole(0, v, rows)
        s["labels"][torch.rand(rows, generator=g, device="cuda") < 0.1] = -1   # padding, prompts
        if case["pass"] == "step":
            s["dloss"] = torch.full((rows,), _loss_scale(case) / rows, device="cuda") * (s["labels"] >= 0)
    else:
        rows, v, k = case["rows"], case["vocabulary"], case["kept"]
        s["logits"] = normal(rows, v, std=2.0)
        s["top"] = normal(rows, k, mean=5.0, std=2.0).sort(dim=1, descending=True).values
        # distinct entries, spread over the vocabulary
        start, step = whole(0, v, rows, 1).long(), v // k
        s["index"] = ((start + step * torch.arange(k, device="cuda")) % v).int()
        s["temperature"] = 2.0
        if case["pass"] == "step":
            s["dloss"] = torch.full((rows,), _loss_scale(case) / rows, device="cuda")
    return s


def run(s: dict):
    case = s["case"]
    return (_own if own else _plain)[case["op"]](s, case["pass"] == "step")


# ---- the framework's operators ------------------------------------------------------------------------------------------

def _own_normalization(s, step):
    from neoml_b200 import ops
    y, mean, inv = ops.LayerNormalization(s["x"], s["scale"], s["free_term"], epsilon=EPSILON)
    if not step:
        return {"y": y, "mean": mean, "inv": inv}
    dx, dscale, dfree = ops.LayerNormalizationBackward(s["dy"], s["x"], mean, inv, s["scale"])
    return {"y": y, "dx": dx, "dscale": dscale, "dfree": dfree}


def _own_recurrence(s, step):
    from neoml_b200 import ops
    h, last = ops.GatedRecurrence(s["z"], s["f"], s["i"], initial_state=s["h0"], lengths=s["lengths"])
    if not step:
        return {"h": h, "last": last}
    dz, df, di, dh0 = ops.GatedRecurrenceBackward(s["dh"], h, s["z"], s["f"], s["i"], initial_state=s["h0"],
                                                  final_state_diff=s["d_last"], lengths=s["lengths"])
    return {"h": h, "last": last, "dz": dz, "df": df, **({} if di is None else {"di": di}), "dh0": dh0}


def _own_entropy(s, step):
    from neoml_b200 import ops
    loss, log_sum = ops.VocabularyCrossEntropy(s["x"], s["w"], s["labels"])
    if not step:
        return {"loss": loss, "log_sum": log_sum}
    dx, dw = ops.VocabularyCrossEntropyBackward(s["dloss"], s["x"], s["w"], s["labels"], log_sum)
    return {"loss": loss, "log_sum": log_sum, "dx": dx, "dw": dw}


def _own_distillation(s, step):
    from neoml_b200 import ops
    loss, log_sum = ops.DistillationLoss(s["logits"], s["top"], s["index"], temperature=s["temperature"])
    if not step:
        return {"loss": loss, "log_sum": log_sum}
    d = ops.DistillationLossBackward(s["dloss"], s["logits"], s["top"], s["index"], log_sum, temperature=s["temperature"])
    return {"loss": loss, "log_sum": log_sum, "dlogits": d}


_own = {"normalization": _own_normalization, "recurrence": _own_recurrence, "entropy": _own_entropy,
        "distillation": _own_distillation}


# ---- the plain form -----------------------------------------------------------------------------------------------------

def _plain_normalization(s, step):
    x = s["x"].float()
    mean = x.mean(dim=1, keepdim=True)
    centred = x - mean
    inv = 1.0 / torch.sqrt((centred * centred).mean(dim=1, keepdim=True) + EPSILON)
    unit = centred * inv
    y = (unit * s["scale"] + s["free_term"]).to(s["x"].dtype)
    if not step:
        return {"y": y, "mean": mean[:, 0], "inv": inv[:, 0]}
    dy = s["dy"].float()
    by_scale = dy * s["scale"]
    dx = inv * (by_scale - by_scale.mean(dim=1, keepdim=True) - unit * (by_scale * unit).mean(dim=1, keepdim=True))
    return {"y": y, "dx": dx.to(s["x"].dtype), "dscale": (dy * unit).sum(dim=0), "dfree": dy.sum(dim=0)}


def _scan(a, b):
    """h[:, t] = a[:, t] * h[:, t - 1] + b[:, t] from zero, by doubling the span that each step has summed."""
    span = 1
    while span < a.shape[1]:
        b = torch.cat([b[:, :span], b[:, span:] + a[:, span:] * b[:, :-span]], dim=1)
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], dim=1)
        span *= 2
    return b


def _plain_recurrence(s, step):
    z, h0, t = s["z"].float(), s["h0"], s["z"].dtype
    keep = torch.sigmoid(s["f"].float())
    take = torch.sigmoid(-s["f"].float()) if s["i"] is None else torch.sigmoid(s["i"].float())
    batch, length = z.shape[:2]
    inside = None
    if s["lengths"] is not None:   # behind a sequence's end the state stays as it is
        inside = (torch.arange(length, device=z.device) < s["lengths"][:, None])[:, :, None]
        keep_all, added = torch.where(inside, keep, 1.0), torch.where(inside, take * z, 0.0)
    else:
        keep_all, added = keep, take * z
    first = added[:, :1] + keep_all[:, :1] * h0[:, None]
    h = _scan(keep_all, torch.cat([first, added[:, 1:]], dim=1))
    last = h[:, -1]
    shown = h if inside is None else torch.where(inside, h, 0.0)
    out = {"h": shown.to(t), "last": last}
    if not step:
        return out
    dh = s["dh"].float() if inside is None else torch.where(inside, s["dh"].float(), 0.0)
    # the gradient of each state is its own plus what the next one hands back
    dh = torch.cat([dh[:, :-1], dh[:, -1:] + s["d_last"][:, None]], dim=1)
    back = torch.cat([keep_all[:, 1:], torch.zeros_like(keep_all[:, :1])], dim=1)
    ds = _scan(back.flip(1), dh.flip(1)).flip(1)
    before = torch.cat([h0[:, None], h[:, :-1]], dim=1)
    dz = ds * take
    if s["i"] is None:
        df = ds * (before - z) * keep * take
        grads = {"dz": dz, "df": df}
    else:
        grads = {"dz": dz, "df": ds * before * keep * (1.0 - keep), "di": ds * z * take * (1.0 - take)}
    for name, value in grads.items():
        out[name] = (value if inside is None else torch.where(inside, value, 0.0)).to(t)
    out["dh0"] = ds[:, 0] * keep_all[:, 0]
    return out


def _plain_entropy(s, step):
    x, w, t = s["x"].float(), s["w"].float(), s["x"].dtype
    z = x @ w.t()
    top = z.amax(dim=1, keepdim=True)
    log_sum = (torch.log(torch.exp(z - top).sum(dim=1, keepdim=True)) + top)
    used = s["labels"] >= 0
    at = s["labels"].clamp(min=0).long()[:, None]
    out = {"loss": torch.where(used, (log_sum - z.gather(1, at))[:, 0], 0.0), "log_sum": log_sum[:, 0]}
    if not step:
        return out
    z.sub_(log_sum).exp_()
    rows = torch.arange(z.shape[0], device=z.device)
    z[rows, at[:, 0]] -= 1.0
    z.mul_(torch.where(used, s["dloss"], 0.0)[:, None])
    out["dx"], out["dw"] = (z @ w).to(t), (z.t() @ x).to(t)
    return out


def _plain_distillation(s, step):
    tau, t = s["temperature"], s["logits"].dtype
    z = s["logits"].float() / tau
    top = s["top"].float() / tau
    log_sum = torch.log(torch.exp(z - z.amax(dim=1, keepdim=True)).sum(dim=1)) + z.amax(dim=1)
    log_p = top - (torch.log(torch.exp(top - top.amax(dim=1, keepdim=True)).sum(dim=1, keepdim=True)) + top.amax(dim=1, keepdim=True))
    p = torch.exp(log_p)
    at = s["index"].long()
    log_q = z.gather(1, at) - log_sum[:, None]
    out = {"loss": tau * tau * (p * (log_p - log_q)).sum(dim=1), "log_sum": log_sum}
    if not step:
        return out
    d = torch.exp(z - log_sum[:, None])
    d.scatter_add_(1, at, -p)
    out["dlogits"] = (d * (tau * s["dloss"])[:, None]).to(t)
    return out


_plain = {"normalization": _plain_normalization, "recurrence": _plain_recurrence, "entropy": _plain_entropy,
          "distillation": _plain_distillation}


# ---- from the definitions in 64 bits ------------------------------------------------------------------------------------

def exact(case: dict, seed: int):
    s = prepare(case, seed)
    return {"normalization": _exact_normalization, "recurrence": _exact_recurrence, "entropy": _exact_entropy,
            "distillation": _exact_distillation}[case["op"]](s, case["pass"] == "step")


def _exact_normalization(s, step):
    x, scale = s["x"].double(), s["scale"].double()
    variance, mean = torch.var_mean(x, dim=1, correction=0)
    inv = (variance + EPSILON).rsqrt()
    if not step:
        return {"y": (x - mean[:, None]) * inv[:, None] * scale + s["free_term"].double(), "mean": mean, "inv": inv}
    # the Jacobian of the unit rows: (1 - 1/n - u u^T / n) / deviation
    u, n = (x - mean[:, None]) * inv[:, None], x.shape[1]
    dy = s["dy"].double()
    du = dy * scale
    dx = (du - du.sum(dim=1, keepdim=True) / n - u * torch.einsum("ij,ij->i", du, u)[:, None] / n) * inv[:, None]
    return {"y": u * scale + s["free_term"].double(), "dx": dx, "dscale": torch.einsum("ij,ij->j", dy, u), "dfree": dy.sum(dim=0)}


def _exact_recurrence(s, step):
    z, f, h0 = s["z"].double(), s["f"].double(), s["h0"].double()
    a = 1.0 / (1.0 + torch.exp(-f))
    u = 1.0 - a if s["i"] is None else 1.0 / (1.0 + torch.exp(-s["i"].double()))
    b, n, c = z.shape
    lengths = torch.full((b,), n, device=z.device) if s["lengths"] is None else s["lengths"].long()
    states = torch.empty(n + 1, b, c, dtype=torch.float64, device=z.device)
    states[0] = h0
    valid = (torch.arange(n, device=z.device)[:, None] < lengths)[:, :, None].double()
    for t in range(n):
        states[t + 1] = torch.lerp(states[t], a[:, t] * states[t] + u[:, t] * z[:, t], valid[t])
    out = {"h": (states[1:] * valid).transpose(0, 1), "last": states[n].clone()}
    if not step:
        return out
    grad, dh = s["d_last"].double(), s["dh"].double()
    dz, df, di = torch.zeros_like(z), torch.zeros_like(z), torch.zeros_like(z)
    for t in reversed(range(n)):
        g = (grad + dh[:, t]) * valid[t]
        dz[:, t] = g * u[:, t]
        da, du = g * states[t], g * z[:, t]
        if s["i"] is None:
            da = da - du
        else:
            di[:, t] = du * u[:, t] * (1.0 - u[:, t])
        df[:, t] = da * a[:, t] * (1.0 - a[:, t])
        grad = grad * (1.0 - valid[t]) + g * a[:, t]
    out.update(dz=dz, df=df, **({} if s["i"] is None else {"di": di}), dh0=grad)
    return out


def _exact_entropy(s, step):
    x, w = s["x"].double(), s["w"].double()
    labels, rows = s["labels"].long(), s["x"].shape[0]
    loss, log_sum = torch.zeros(rows, dtype=torch.float64, device=x.device), torch.empty(rows, dtype=torch.float64, device=x.device)
    dx, dw = torch.empty_like(x) if step else None, torch.zeros_like(w) if step else None
    for r in range(0, rows, 1024):   # the rows of the batch in parts: 64-bit logits of all would take several GB
        part = slice(r, min(r + 1024, rows))
        z = x[part] @ w.T
        log_sum[part] = torch.logsumexp(z, dim=1)
        hot = torch.zeros_like(z)
        has = (labels[part] >= 0).nonzero()[:, 0]
        hot[has, labels[part][has]] = 1.0
        loss[part] = hot.sum(dim=1) * log_sum[part] - (hot * z).sum(dim=1)
        if step:
            dz = (torch.softmax(z, dim=1) * hot.sum(dim=1, keepdim=True) - hot) * s["dloss"][part].double()[:, None]
            dx[part] = dz @ w
            dw += dz.T @ x[part]
    return {"loss": loss, "log_sum": log_sum, **({"dx": dx, "dw": dw} if step else {})}


def _exact_distillation(s, step):
    tau = s["temperature"]
    rows, v = s["logits"].shape
    p = torch.softmax(s["top"].double() / tau, dim=1)
    z = s["logits"].double() / tau
    log_q = torch.log_softmax(z, dim=1)
    target = torch.zeros_like(z).index_put_((torch.arange(rows, device=z.device)[:, None], s["index"].long()), p, accumulate=True)
    # sum p log p - sum p log q over the kept entries
    loss = tau ** 2 * (torch.special.xlogy(p, p).sum(dim=1) - (target * log_q).sum(dim=1))
    out = {"loss": loss, "log_sum": torch.logsumexp(z, dim=1)}
    if step:
        out["dlogits"] = (log_q.exp() - target) * (tau * s["dloss"].double())[:, None]
    return out


# ---- what a pass cannot do without --------------------------------------------------------------------------------------

def work(case: dict) -> dict:
    size, step = TYPES[case["type"]].itemsize, case["pass"] == "step"
    if case["op"] == "normalization":
        n = case["rows"] * case["width"]
        # forward: x, y; backward: dy and x again (the layers behind it ran in between), dx
        return {"bytes": n * size * (5 if step else 2) + 8 * case["rows"] + 4 * case["width"] * (4 if step else 2),
                "flops": n * (19 if step else 8)}
    if case["op"] == "recurrence":
        n = case["batch"] * case["length"] * case["channels"]
        inputs = 3 if case["input_gate"] else 2
        state = 4 * case["batch"] * case["channels"]
        # forward: z, f, i, h; backward: dh, h, z, f, i and as many gradients as inputs
        return {"bytes": n * size * (inputs + 1 + (2 + 2 * inputs if step else 0)) + state * (5 if step else 2),
                "flops": n * (30 if step else 10)}
    if case["op"] == "entropy":
        rows, d, v = case["rows"], case["width"], case["vocabulary"]
        return {"bytes": (rows * d + v * d) * size * (2 if step else 1) + 12 * rows + (4 * rows if step else 0),
                "flops": 2 * rows * d * v * (3 if step else 1) + 4 * rows * v}
    n, kept = case["rows"] * case["vocabulary"], case["rows"] * case["kept"]
    return {"bytes": n * size * (3 if step else 1) + kept * (size + 4) * (2 if step else 1) + 8 * case["rows"], "flops": n * (9 if step else 4)}
