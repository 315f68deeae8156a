"""The operators that train a small draft model from a teacher and serve it
beside the model it drafts for, as measurable cases with a plain form beside
them.

  mlp           y = (silu(x Wg^T) * (x Wu^T)) Wd^T, the gated feed-forward
                block of a layer, and where ``keep`` the two projections'
                outputs for its backward pass (``gated_mlp``)
  mlp_grad      its gradients: dx and those of the three weights
                (``gated_mlp_backward``)
  distill       divergence of an LM head whose logits are never kept from the
                teacher's top logits: loss and log-sum-exp of every row, and
                the student's logits at the teacher's entries
                (``lm_head_distill``)
  distill_grad  its gradients of the rows and of the head
                (``lm_head_distill_backward``)
  verify        drafted tokens of many requests accepted or rejected against
                the target model's logits from given random numbers, and the
                token that follows the accepted ones (``draft_verify``)

``prepare`` makes what a step has in hand; ``run`` is one call.  ``limit`` is
the block's clamp (gate from above, up from both sides; 0: none).
"""
import math

import torch

own = False

# feed-forward blocks as (hidden, intermediate): Qwen3-8B, DeepSeek V4 Flash's
# shared expert, an expert of the 7168-wide MoE layer
BLOCKS = ((4096, 12288), (4096, 2048), (7168, 2048))
# LM heads as (vocabulary, hidden): Qwen3-0.6B, DeepSeek V4 Flash
HEADS = ((151936, 1024), (129280, 4096))
VOCABULARIES = (151936, 129280)
NONE = -1  # no teacher entry


def listed():
    return [
        # one request's decode step of a small block: the smallest call,
        # latency alone
        {"name": "mlp_decode_1", "kind": "mlp", "rows": 1, "hidden": 4096, "inter": 2048, "limit": 10.0, "keep": False},
        # a decode batch of concurrent requests
        {"name": "mlp_decode_57", "kind": "mlp", "rows": 57, "hidden": 4096, "inter": 12288, "limit": 0.0,
         "keep": False},
        # the forward pass of a training step of ragged samples
        {"name": "mlp_keep_4099", "kind": "mlp", "rows": 4099, "hidden": 4096, "inter": 12288, "limit": 0.0,
         "keep": True},
        # the backward pass of a few short samples, clamped
        {"name": "mlp_grad_509", "kind": "mlp_grad", "rows": 509, "hidden": 7168, "inter": 2048, "limit": 10.0},
        # the backward pass of 4096 tokens
        {"name": "mlp_grad_4096", "kind": "mlp_grad", "rows": 4096, "hidden": 4096, "inter": 12288, "limit": 0.0},
        # the divergence on a short held-out continuation
        {"name": "distill_33", "kind": "distill", "rows": 33, "vocab": 151936, "hidden": 1024, "top": 20,
         "temperature": 1.0, "tail": False},
        # the divergence on a 4096-token batch
        {"name": "distill_4096", "kind": "distill", "rows": 4096, "vocab": 129280, "hidden": 4096, "top": 64,
         "temperature": 2.0, "tail": False},
        # a training step of a ragged batch with a tied head, the teacher's
        # probabilities those of its whole vocabulary
        {"name": "distill_grad_1021", "kind": "distill_grad", "rows": 1021, "vocab": 151936, "hidden": 1024, "top": 32,
         "temperature": 1.0, "tail": True},
        # a training step over a large head, the largest call
        {"name": "distill_grad_2053", "kind": "distill_grad", "rows": 2053, "vocab": 129280, "hidden": 4096, "top": 64,
         "temperature": 2.0, "tail": False},
        # one request's five drafted tokens
        {"name": "verify_1", "kind": "verify", "sequences": 1, "drafts": 5, "vocab": 151936, "half": False, "soft": True},
        # a batch with none to seven drafted tokens each, looked up and not
        # drawn from a model; one request in eight is greedy
        {"name": "verify_57", "kind": "verify", "sequences": 57, "drafts": 7, "vocab": 129280, "half": True,
         "soft": False},
        # a large batch of a draft model's tokens
        {"name": "verify_256", "kind": "verify", "sequences": 256, "drafts": 4, "vocab": 151936, "half": False,
         "soft": True},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("mlp", "mlp", "mlp_grad", "distill", "distill_grad", "verify", "verify"))
    if kind in ("mlp", "mlp_grad"):
        hidden, inter = rng.choice(BLOCKS)
        case = {"kind": kind, "rows": _log_int(rng, 1, 8191 if kind == "mlp" else 4095), "hidden": hidden,
                "inter": inter, "limit": rng.choice((0.0, 10.0))}
        if kind == "mlp":
            case["keep"] = case["rows"] > 64 and rng.random() < 0.7
        return case
    if kind in ("distill", "distill_grad"):
        vocab, hidden = rng.choice(HEADS)
        return {"kind": kind, "rows": _log_int(rng, 1, 4095 if kind == "distill" else 2047), "vocab": vocab,
                "hidden": hidden, "top": _log_int(rng, 1, 128), "temperature": rng.choice((0.75, 1.0, 2.0, 4.0)),
                "tail": rng.random() < 0.5}
    return {"kind": kind, "sequences": _log_int(rng, 1, 255), "drafts": rng.randint(1, 8),
            "vocab": rng.choice(VOCABULARIES), "half": rng.random() < 0.3, "soft": rng.random() < 0.6}


# ------------------------------------------------------------------ inputs
def _gen(seed, device="cuda"):
    g = torch.Generator(device=device)
    g.manual_seed(0x4452_4146 + int(seed))
    return g


def _normal(g, shape, std=1.0):
    return (torch.randn(shape, device=g.device, generator=g) * std).to(torch.bfloat16)


def _block(case, seed):
    g = _gen(seed)
    rows, h, i = case["rows"], case["hidden"], case["inter"]
    # gates and ups about 2 wide, so that a clamp at 10 is met now and then
    # (by the rows of larger norm)
    size = 0.5 + 1.5 * torch.rand(rows, 1, device="cuda", generator=g)
    x = (torch.randn(rows, h, device="cuda", generator=g) * size).to(torch.bfloat16)
    t = {"x": x, "wg": _normal(g, (i, h), 2 * h ** -0.5), "wu": _normal(g, (i, h), 2 * h ** -0.5),
         "wd": _normal(g, (h, i), i ** -0.5)}
    if case["kind"] == "mlp_grad":
        t["gate"] = (x.float() @ t["wg"].float().T).to(torch.bfloat16)
        t["up"] = (x.float() @ t["wu"].float().T).to(torch.bfloat16)
        t["dy"] = _normal(g, (rows, h), 1e-3)
    return t


def _teacher(case, seed):
    g = _gen(seed)
    rows, v, h, k = case["rows"], case["vocab"], case["hidden"], case["top"]
    w = _normal(g, (v, h), 0.02)
    u = torch.rand(rows, device="cuda", generator=g)
    lean = w[(u * u * u * v).long().clamp_(max=v - 1)].float() * 5
    # a student on its way to the teacher: the same leaning, other noise
    shared = torch.randn(rows, h, device="cuda", generator=g)
    x = (shared + 0.5 * torch.randn(rows, h, device="cuda", generator=g) + lean).to(torch.bfloat16)
    teacher = (shared + lean * 1.2) @ w.float().T
    top = torch.topk(teacher, k, dim=1)
    # a teacher's list may be cut short, and one row in ten has none (padding)
    keep = torch.where(torch.rand(rows, device="cuda", generator=g) < 0.5, k,
                       (torch.rand(rows, device="cuda", generator=g) * k).long() + 1)
    keep = torch.where(torch.rand(rows, device="cuda", generator=g) < 0.1, 0, keep)
    there = torch.arange(k, device="cuda")[None, :] < keep[:, None]
    t = {"x": x, "w": w, "ids": torch.where(there, top.indices, NONE).to(torch.int32),
         "teacher": top.values.contiguous(), "teacher_lse": None}
    if case["tail"]:
        t["teacher_lse"] = torch.logsumexp(teacher / case["temperature"], 1)
    if case["kind"] == "distill_grad":
        logits = x.float() @ w.float().T
        t["lse"] = torch.logsumexp(logits / case["temperature"], 1)
        t["logits"] = torch.where(there, logits.gather(1, top.indices), 0.0)
        t["dloss"] = torch.where(keep > 0, 1.0 / (keep > 0).sum().clamp(min=1), 0.0).float()
    return t


def _drafts(case, seed):
    g, host = _gen(seed), _gen(seed, "cpu")
    b, most, v = case["sequences"], case["drafts"], case["vocab"]
    count = torch.full((b,), most) if b == 1 else torch.randint(0, most + 1, (b,), generator=host)
    offsets = torch.cat((torch.zeros(1, dtype=torch.int64), count.cumsum(0))).cuda()
    d, dtype = int(count.sum()), torch.bfloat16 if case["half"] else torch.float32
    common = -2.0 * torch.log1p(torch.randperm(v, device="cuda", generator=g).float() / 50)
    target = torch.randn(d + b, v, device="cuda", generator=g).mul_(1.5).add_(common)
    temperature = 0.6 + 0.7 * torch.rand(b, device="cuda", generator=g)
    temperature[7::8] = 0.0  # greedy
    row = torch.arange(d, device="cuda")
    seq = torch.bucketize(row, offsets[1:], right=True)
    # the draft model's logits stand near the target's of the same position
    draft = target[row + seq] + 0.5 * torch.randn(d, v, device="cuda", generator=g)
    tau = temperature[seq][:, None]
    noise = -torch.log(-torch.log(torch.rand(d, v, device="cuda", generator=g).clamp(min=1e-30, max=1 - 1e-7)))
    tokens = torch.where(tau > 0, draft / torch.where(tau > 0, tau, 1.0) + noise, draft).argmax(1)
    return {"target": target.to(dtype), "tokens": tokens.to(torch.int32), "offsets": offsets.to(torch.int32),
            "accept": torch.rand(d, device="cuda", generator=g), "sample": torch.rand(b, device="cuda", generator=g),
            "draft": draft.to(dtype) if case["soft"] else None, "temperature": temperature}


def _inputs(case, seed):
    if case["kind"] in ("mlp", "mlp_grad"):
        return _block(case, seed)
    if case["kind"] in ("distill", "distill_grad"):
        return _teacher(case, seed)
    return _drafts(case, seed)


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    state["flag"] = torch.zeros(1, dtype=torch.int32, device="cuda")  # the packs' error flag, one for a pipeline
    return state


# -------------------------------------------------------------- plain form
def _plain_mlp(t, case):
    x, wg, wu, wd = (t[n].float() for n in ("x", "wg", "wu", "wd"))
    limit = case["limit"] if case["limit"] > 0 else math.inf
    if case["kind"] == "mlp":
        gate, up = x @ wg.T, x @ wu.T
        g = gate.clamp(max=limit)
        y = (g / (1 + torch.exp(-g)) * up.clamp(min=-limit, max=limit)) @ wd.T
        return [y.to(torch.bfloat16)] + ([gate.to(torch.bfloat16), up.to(torch.bfloat16)] if case["keep"] else [])
    dy, gate, up = (t[n].float() for n in ("dy", "gate", "up"))
    g, u = gate.clamp(max=limit), up.clamp(min=-limit, max=limit)
    share = 1 / (1 + torch.exp(-g))
    dh = dy @ wd
    dg = torch.where(gate <= limit, dh * u * share * (1 + g * (1 - share)), 0.0)
    du = torch.where(up.abs() <= limit, dh * g * share, 0.0)
    return [o.to(torch.bfloat16) for o in (dg @ wg + du @ wu, dg.T @ x, du.T @ x, dy.T @ (g * share * u))]


def _plain_distill(t, case):
    tau = case["temperature"]
    logits = t["x"].float() @ t["w"].float().T
    there = t["ids"] >= 0
    at = t["ids"].clamp(min=0).long()
    scaled = torch.where(there, t["teacher"] / tau, -math.inf)
    if t["teacher_lse"] is None:
        top = scaled.amax(1, keepdim=True)
        top = torch.where(top == -math.inf, 0.0, top)
        log_q = scaled - top - torch.log(torch.exp(scaled - top).sum(1, keepdim=True).clamp(min=1e-30))
    else:
        log_q = scaled - t["teacher_lse"][:, None]
    q = torch.exp(log_q)
    if case["kind"] == "distill":
        top = logits.amax(1, keepdim=True)
        lse = top[:, 0] / tau + torch.log(torch.exp((logits - top) / tau).sum(1))
        z = torch.where(there, logits.gather(1, at), 0.0)
        loss = tau * tau * torch.where(there, q * (log_q - z / tau + lse[:, None]), 0.0).sum(1)
        return [loss, lse, z]
    d = torch.exp(logits / tau - t["lse"][:, None]) * q.sum(1, keepdim=True)
    d.scatter_add_(1, at, -q)
    d *= (tau * t["dloss"])[:, None]
    return [(d @ t["w"].float()).to(torch.bfloat16), (d.T @ t["x"].float()).to(torch.bfloat16)]


def _plain_verify(t, case):
    b, most = case["sequences"], case["drafts"]
    offsets, tokens = t["offsets"].long(), t["tokens"].long()
    d, count = tokens.shape[0], offsets[1:] - offsets[:-1]
    drafts, seqs = torch.arange(d, device="cuda"), torch.arange(b, device="cuda")
    seq = torch.bucketize(drafts, offsets[1:], right=True)
    greedy = t["temperature"] == 0
    tau = torch.where(greedy, 1.0, t["temperature"]).double()
    of_target = torch.bucketize(torch.arange(d + b, device="cuda"), offsets[1:] + seqs + 1, right=True)
    p = torch.exp((t["target"].double() - t["target"].double().amax(1, keepdim=True)) / tau[of_target][:, None])
    p /= p.sum(1, keepdim=True)
    best = t["target"].argmax(1)
    at = drafts + seq  # a drafted token's row of the target
    if case["soft"]:
        q = torch.exp((t["draft"].double() - t["draft"].double().amax(1, keepdim=True)) / tau[seq][:, None])
        q /= q.sum(1, keepdim=True)
        theirs = q.gather(1, tokens[:, None])[:, 0]
    else:
        theirs = torch.ones(d, dtype=torch.float64, device="cuda")
    drawn = t["accept"].double() * theirs < p[at].gather(1, tokens[:, None])[:, 0]
    right = torch.where(greedy[seq], tokens == best[at], drawn)
    place = torch.arange(most + 1, device="cuda")[None, :]
    there = place < count[:, None]
    index = (offsets[:-1, None] + place).clamp(max=max(d - 1, 0))
    fill = torch.zeros(1, dtype=torch.bool, device="cuda") if d == 0 else right
    accepted = (there & fill[index]).long().cumprod(1).sum(1)
    row = offsets[:-1] + seqs + accepted
    rest = p[row]
    if d:
        rejected = (accepted < count)[:, None]
        last = (offsets[:-1] + accepted).clamp(max=d - 1)
        if case["soft"]:
            left = (rest - q[last]).clamp(min=0)
        else:
            left = rest.scatter(1, tokens[last][:, None], 0.0)
        left = torch.where(rejected, left, rest)
        rest = torch.where(left.sum(1, keepdim=True) > 0, left, rest)
    run_up = rest.cumsum(1)
    threshold = t["sample"].double() * run_up[:, -1]
    token = torch.searchsorted(run_up, threshold[:, None], right=True)[:, 0].clamp(max=case["vocab"] - 1)
    token = torch.where(greedy, best[row], token)
    mine = torch.zeros(1, dtype=torch.int64, device="cuda") if d == 0 else tokens
    out = torch.where(place < accepted[:, None], mine[index], NONE)
    out = torch.where(place == accepted[:, None], token[:, None], out)
    return [out.to(torch.int32), accepted.to(torch.int32)]


def _calls(t, case):
    from pih_amd.device import engine_stream
    from pih_amd.linear import (draft_verify, gated_mlp, gated_mlp_backward, lm_head_distill, lm_head_distill_backward)

    kind = case["kind"]
    with engine_stream():
        if kind == "mlp":
            out = gated_mlp(t["x"], t["wg"], t["wu"], t["wd"], limit=case["limit"], keep=case["keep"])
            return list(out) if case["keep"] else [out]
        if kind == "mlp_grad":
            return list(gated_mlp_backward(t["dy"], t["x"], t["wg"], t["wu"], t["wd"], t["gate"], t["up"],
                                           limit=case["limit"]))
        if kind == "distill":
            return list(lm_head_distill(t["x"], t["w"], t["ids"], t["teacher"], case["temperature"],
                                        teacher_lse=t["teacher_lse"], flag=t["flag"])[:3])
        if kind == "distill_grad":
            return list(lm_head_distill_backward(t["x"], t["w"], t["ids"], t["teacher"], t["lse"], t["logits"],
                                                 t["dloss"], case["temperature"], teacher_lse=t["teacher_lse"],
                                                 flag=t["flag"])[:2])
        return list(draft_verify(t["target"], t["tokens"], t["offsets"], t["accept"], t["sample"], case["drafts"],
                                 draft_logits=t["draft"], temperature=t["temperature"], flag=t["flag"])[:2])


def run(state):
    case = state["case"]
    if own:
        return _calls(state, case)
    if case["kind"] in ("mlp", "mlp_grad"):
        return _plain_mlp(state, case)
    if case["kind"] in ("distill", "distill_grad"):
        return _plain_distill(state, case)
    return _plain_verify(state, case)


# ------------------------------------------------------------------ floors
def work(case):
    kind = case["kind"]
    if kind in ("mlp", "mlp_grad"):
        rows, h, i = case["rows"], case["hidden"], case["inter"]
        if kind == "mlp":
            return {"bytes": 6 * h * i + 4 * rows * h + (4 * rows * i if case["keep"] else 0), "flops": 6 * rows * h * i}
        return {"bytes": 12 * h * i + 6 * rows * h + 4 * rows * i, "flops": 12 * rows * h * i}
    if kind in ("distill", "distill_grad"):
        rows, v, h, k = case["rows"], case["vocab"], case["hidden"], case["top"]
        if kind == "distill":
            return {"bytes": 2 * h * (v + rows) + 12 * rows * k + 12 * rows, "flops": 2 * rows * v * h}
        return {"bytes": 4 * h * (v + rows) + 12 * rows * k + 12 * rows, "flops": 6 * rows * v * h}
    b, v = case["sequences"], case["vocab"]
    d = b * case["drafts"] if b == 1 else b * case["drafts"] // 2  # (the mean)
    size = 2 if case["half"] else 4
    elements = (d + b + (d if case["soft"] else 0)) * v
    return {"bytes": elements * size + 16 * d + 16 * b, "flops": 4 * elements}


# ------------------------------------------------------------- 64-bit form
def _exact_mlp(t, case):
    d = {n: v.double() for n, v in t.items()}
    x, wg, wu, wd = (d[n].requires_grad_() for n in ("x", "wg", "wu", "wd"))
    limit = case["limit"] or 1e30

    def act(gate, up):
        return torch.nn.functional.silu(torch.clamp(gate, max=limit)) * torch.clamp(up, -limit, limit)

    if case["kind"] == "mlp":
        with torch.no_grad():
            gate, up = x @ wg.T, x @ wu.T
            y = act(gate, up) @ wd.T
        return [y, gate, up] if case["keep"] else [y]
    # the activation is taken at the gate and up that were kept
    gate, up = d["gate"].requires_grad_(), d["up"].requires_grad_()
    y = act(gate, up) @ wd.T
    dgate, dup, dwd = torch.autograd.grad((y * d["dy"]).sum(), (gate, up, wd))
    with torch.no_grad():
        return [torch.cat((dgate, dup), 1) @ torch.cat((wg, wu), 0), dgate.T @ x, dup.T @ x, dwd]


def _exact_distill(t, case):
    tau = case["temperature"]
    x, w = t["x"].double(), t["w"].double()
    there, at = t["ids"] >= 0, t["ids"].clamp(min=0).long()
    weight = torch.exp(t["teacher"].double() / tau) * there
    if t["teacher_lse"] is None:
        q = weight / weight.sum(1, keepdim=True).clamp(min=1e-300)
    else:
        q = weight / torch.exp(t["teacher_lse"].double())[:, None]
    if case["kind"] == "distill":
        logits = x @ w.T
        log_p = torch.log_softmax(logits / tau, 1)
        lse = torch.logsumexp(logits / tau, 1)
        loss = (torch.special.xlogy(q, q) - q * log_p.gather(1, at)).sum(1) * tau ** 2
        return [loss, lse, logits.gather(1, at) * there]
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    for part in torch.arange(x.shape[0], device="cuda").split(512):
        xs = x[part]
        # d (tau^2 KL) / d logits
        g = torch.softmax(xs @ w.T / tau, 1) * q[part].sum(1, keepdim=True)
        g.scatter_add_(1, at[part], -q[part])
        g *= tau * t["dloss"][part].double()[:, None]
        dx[part] = g @ w
        dw += g.T @ xs
    return [dx, dw]


def exact(case, seed):
    if case["kind"] == "verify":
        return None  # whole numbers alone
    t = _inputs(case, seed)
    if case["kind"] in ("mlp", "mlp_grad"):
        return _exact_mlp(t, case)
    return _exact_distill(t, case)
