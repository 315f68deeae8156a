"""The operators that fine-tune and serve low-rank adapters over the packs'
frozen projections, as measurable cases with a plain form beside them.

  adapter      y = base + scale[a] (x A_a^T) B_a^T for the rows of many
               requests, each with an adapter a of its own or none, on top of
               a shared projection's output (``adapter_gemm``)
  adapter_grad its gradients: dx on top of the shared projection's, dA and dB
               of every adapter (``adapter_backward``)
  loss         softmax cross entropy of an LM head whose logits are never
               kept: loss and log-sum-exp of every row (``lm_head_loss``)
  loss_grad    its gradients of the rows and of the head
               (``lm_head_loss_backward``)
  router       a MoE router's balance loss with the experts' route counts,
               and where ``grad`` the gradient of the scores behind both that
               loss and the route weights (``router_balance``,
               ``router_backward``)

``prepare`` makes what a step has in hand; ``run`` is one call, or with the
router the two calls of one training step.  Every row belongs to a request.
"""
import math

import torch

own = False

# Qwen3-8B projections as (N, K): q, k/v, gate/up, down
PROJECTIONS = ((4096, 4096), (1024, 4096), (12288, 4096), (4096, 12288))
# LM heads as (vocabulary, hidden): Qwen3-0.6B, DeepSeek V4 Flash
HEADS = ((151936, 1024), (129280, 4096))
NONE = -1  # no adapter, or a row without a target


def listed():
    return [
        # one request's decode step on the query projection: the smallest call,
        # latency alone
        {"name": "adapter_decode_1", "kind": "adapter", "rows": 1, "requests": 1, "adapters": 1, "rank": 16, "n": 4096,
         "k": 4096},
        # a decode batch of concurrent requests over 16 adapters, up projection
        {"name": "adapter_decode_57", "kind": "adapter", "rows": 57, "requests": 57, "adapters": 16, "rank": 32,
         "n": 12288, "k": 4096},
        # ragged prompts of nine requests on the down projection, high rank
        {"name": "adapter_prompts_4099", "kind": "adapter", "rows": 4099, "requests": 9, "adapters": 4, "rank": 64,
         "n": 4096, "k": 12288},
        # a fine-tuning step of a few short samples, one adapter each
        {"name": "adapter_grad_509", "kind": "adapter_grad", "rows": 509, "requests": 5, "adapters": 3, "rank": 8,
         "n": 1024, "k": 4096},
        # a fine-tuning step of 8192 tokens of one adapter
        {"name": "adapter_grad_8192", "kind": "adapter_grad", "rows": 8192, "requests": 4, "adapters": 1, "rank": 16,
         "n": 4096, "k": 4096},
        # log-probabilities of a short continuation
        {"name": "loss_33", "kind": "loss", "rows": 33, "vocab": 151936, "hidden": 1024},
        # log-probabilities of a 4096-token batch
        {"name": "loss_4096", "kind": "loss", "rows": 4096, "vocab": 129280, "hidden": 4096},
        # a training step of a ragged batch with a tied head
        {"name": "loss_grad_1021", "kind": "loss_grad", "rows": 1021, "vocab": 151936, "hidden": 1024},
        # a training step of 4096 tokens, the largest call
        {"name": "loss_grad_4096", "kind": "loss_grad", "rows": 4096, "vocab": 129280, "hidden": 4096},
        # expert load of a decode batch
        {"name": "router_57", "kind": "router", "rows": 57, "experts": 256, "topk": 6, "softplus": True, "grad": False},
        # router training steps, both score functions
        {"name": "router_grad_4099", "kind": "router", "rows": 4099, "experts": 256, "topk": 6, "softplus": True,
         "grad": True},
        {"name": "router_grad_32768", "kind": "router", "rows": 32768, "experts": 256, "topk": 8, "softplus": False,
         "grad": True},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("adapter", "adapter", "adapter_grad", "loss", "loss_grad", "router"))
    if kind in ("adapter", "adapter_grad"):
        n, k = rng.choice(PROJECTIONS)
        rank = rng.choice((8, 16, 24, 32, 64, 128))
        if kind == "adapter" and rng.random() < 0.5:  # a decode batch
            rows = requests = _log_int(rng, 1, 256)
        else:
            rows = _log_int(rng, 17, 8192)
            requests = rng.randint(1, 12)
        return {"kind": kind, "rows": rows, "requests": requests, "adapters": rng.randint(1, min(16, 512 // rank)),
                "rank": rank, "n": n, "k": k}
    if kind in ("loss", "loss_grad"):
        vocab, hidden = rng.choice(HEADS)
        return {"kind": kind, "rows": _log_int(rng, 1, 4095), "vocab": vocab, "hidden": hidden}
    return {"kind": kind, "rows": _log_int(rng, 1, 32767), "experts": rng.choice((64, 128, 256, 384)),
            "topk": rng.randint(1, 8), "softplus": rng.random() < 0.5, "grad": rng.random() < 0.7}


# ------------------------------------------------------------------ inputs
def _gen(seed, device="cuda"):
    g = torch.Generator(device=device)
    g.manual_seed(0x4144_4150 + int(seed))
    return g


def _normal(g, shape, std=1.0):
    return (torch.randn(shape, device=g.device, generator=g) * std).to(torch.bfloat16)


def _requests(case, seed):
    """Row offsets of the requests and their adapters; with several requests
    one in eight has none."""
    g = _gen(seed, "cpu")
    rows, count = case["rows"], case["requests"]
    if rows == count:
        offsets = torch.arange(rows + 1)
    else:
        cuts = torch.randint(0, rows + 1, (count - 1,), generator=g).sort().values
        offsets = torch.cat((torch.zeros(1, dtype=torch.int64), cuts, torch.full((1,), rows)))
    adapters = torch.arange(count) % case["adapters"]
    adapters[7::8] = NONE
    adapters = adapters[torch.randperm(count, generator=g)]
    return offsets.to(torch.int32).cuda(), adapters.to(torch.int32).cuda()


def _inputs(case, seed):
    g = _gen(seed)
    kind, rows = case["kind"], case["rows"]
    if kind in ("adapter", "adapter_grad"):
        s, r, n, k = case["adapters"], case["rank"], case["n"], case["k"]
        offsets, adapters = _requests(case, seed)
        t = {"a": _normal(g, (s, r, k), k ** -0.5), "b": _normal(g, (s, n, r), 0.05), "x": _normal(g, (rows, k)),
             "scale": 0.5 + 1.5 * torch.rand(s, device="cuda", generator=g), "offsets": offsets, "adapters": adapters}
        if kind == "adapter":
            t["base"] = _normal(g, (rows, n))
        else:
            t["dy"] = _normal(g, (rows, n), 1e-3)
            t["base"] = _normal(g, (rows, k), 1e-3)
        return t
    if kind in ("loss", "loss_grad"):
        v, h = case["vocab"], case["hidden"]
        w = _normal(g, (v, h), 0.02)
        u = torch.rand(rows, device="cuda", generator=g)
        target = (u * u * u * v).long().clamp_(max=v - 1)
        # a row leans towards its target's weights, as a trained model's does
        x = (torch.randn(rows, h, device="cuda", generator=g) + w[target].float() * 5).to(torch.bfloat16)
        masked = torch.rand(rows, device="cuda", generator=g) < 0.1
        t = {"x": x, "w": w, "target": torch.where(masked, NONE, target).to(torch.int32)}
        if kind == "loss_grad":
            live = t["target"] >= 0
            t["lse"] = torch.logsumexp(x.float() @ w.float().T, 1)
            t["dloss"] = torch.where(live, 1.0 / live.sum().clamp(min=1), 0.0).float()
        return t
    e, k = case["experts"], case["topk"]
    rank = torch.randperm(e, device="cuda", generator=g)
    scores = torch.randn(rows, e, device="cuda", generator=g) - 1.1 * torch.log1p(rank.float())
    return {"scores": scores, "ids": torch.topk(scores, k, dim=1).indices.to(torch.int32),
            "coefficient": 0.01, "route_scale": 1.5 if case["softplus"] else 1.0,
            "dweights": torch.randn(rows, k, device="cuda", generator=g) * 1e-3,
            "dloss": torch.ones(1, device="cuda")}


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    state["flag"] = torch.zeros(1, dtype=torch.int32, device="cuda")  # the packs' error flag, one for a pipeline
    return state


# -------------------------------------------------------------- plain form
def _chosen(t, rows, count):
    """[rows, adapters, 1]: the scale of a row's adapter in its place, else 0."""
    at = torch.bucketize(torch.arange(rows, device="cuda"), t["offsets"][1:].long(), right=True)
    ids = t["adapters"].long()[at]
    hit = ids[:, None] == torch.arange(count, device="cuda")[None, :]
    return torch.where(hit, t["scale"][None, :], torch.zeros((), device="cuda"))[:, :, None]


def _plain_adapter(t, case):
    s, r, n, k, rows = case["adapters"], case["rank"], case["n"], case["k"], case["rows"]
    x, a = t["x"].float(), t["a"].float().view(s * r, k)
    chosen = _chosen(t, rows, s)
    h = ((x @ a.T).view(rows, s, r) * chosen).view(rows, s * r)
    bt = t["b"].float().permute(0, 2, 1).reshape(s * r, n)
    if case["kind"] == "adapter":
        return (t["base"].float() + h @ bt).to(torch.bfloat16)
    dy = t["dy"].float()
    dh = ((dy @ bt.T).view(rows, s, r) * chosen).view(rows, s * r)
    dx = (t["base"].float() + dh @ a).to(torch.bfloat16)
    da = (dh.T @ x).view(s, r, k)
    db = (dy.T @ h).view(n, s, r).permute(1, 0, 2).contiguous()
    return [dx, da, db]


def _plain_loss(t, case):
    logits = t["x"].float() @ t["w"].float().T
    target = t["target"].long()
    live = target >= 0
    at = target.clamp(min=0)[:, None]
    if case["kind"] == "loss":
        top = logits.amax(1, keepdim=True)
        lse = top[:, 0] + torch.log(torch.exp(logits - top).sum(1))
        loss = torch.where(live, lse - logits.gather(1, at)[:, 0], torch.zeros((), device="cuda"))
        return [loss, lse]
    d = torch.exp(logits - t["lse"][:, None])
    d.scatter_add_(1, at, torch.full_like(at, -1, dtype=torch.float32))
    d *= torch.where(live, t["dloss"], torch.zeros((), device="cuda"))[:, None]
    return [(d @ t["w"].float()).to(torch.bfloat16), (d.T @ t["x"].float()).to(torch.bfloat16)]


def _plain_router(t, case):
    rows, e = case["rows"], case["experts"]
    raw, ids = t["scores"], t["ids"].long()
    counts = torch.zeros(e, dtype=torch.int32, device="cuda")
    counts.index_add_(0, ids.reshape(-1), torch.ones(ids.numel(), dtype=torch.int32, device="cuda"))
    if case["softplus"]:
        base = torch.sqrt(torch.log1p(torch.exp(-raw.abs())) + raw.clamp(min=0))
        slope = 1 / (1 + torch.exp(-raw)) / (2 * base)  # d base / d raw
    else:
        base = torch.exp(raw - raw.amax(1, keepdim=True))
        slope = base
    p = base / base.sum(1, keepdim=True)
    mean = p.sum(0) / rows
    weight = t["coefficient"] * e / (rows * case["topk"])
    loss = (counts * mean).sum().view(1) * weight
    if not case["grad"]:
        return [loss, counts, mean]
    g = counts.float()[None, :] * (t["dloss"] * weight / rows)
    dscores = slope / base.sum(1, keepdim=True) * (g - (g * p).sum(1, keepdim=True))
    top = base.gather(1, ids)
    share = top / top.sum(1, keepdim=True)
    dtop = t["route_scale"] / top.sum(1, keepdim=True) * (t["dweights"] - (t["dweights"] * share).sum(1, keepdim=True))
    dscores.scatter_add_(1, ids, dtop * slope.gather(1, ids))
    return [loss, counts, mean, dscores]


def _calls(t, case):
    from pih_amd import abi
    from pih_amd.device import engine_stream
    from pih_amd.linear import (adapter_backward, adapter_gemm, lm_head_loss, lm_head_loss_backward, router_backward,
                                router_balance)

    kind, flag = case["kind"], t["flag"]
    with engine_stream():
        if kind == "adapter":
            return adapter_gemm(t["x"], t["a"], t["b"], t["scale"], t["offsets"], t["adapters"], base=t["base"],
                                flag=flag)[0]
        if kind == "adapter_grad":
            return adapter_backward(t["dy"], t["x"], t["a"], t["b"], t["scale"], t["offsets"], t["adapters"],
                                    base=t["base"], flag=flag)[:3]
        if kind == "loss":
            return lm_head_loss(t["x"], t["w"], t["target"], flag=flag)[:2]
        if kind == "loss_grad":
            return lm_head_loss_backward(t["x"], t["w"], t["target"], t["lse"], t["dloss"], flag=flag)[:2]
        mode = abi.ROUTER_SQRT_SOFTPLUS if case["softplus"] else abi.ROUTER_SOFTMAX
        loss, counts, mean, _ = router_balance(t["scores"], t["ids"], mode, t["coefficient"], flag=flag)
        if not case["grad"]:
            return [loss, counts, mean]
        dscores, _ = router_backward(t["scores"], t["ids"], counts, mode, t["coefficient"], t["dloss"],
                                     dweights=t["dweights"], route_scale=t["route_scale"], flag=flag)
        return [loss, counts, mean, dscores]


def run(state):
    case = state["case"]
    if own:
        return _calls(state, case)
    if case["kind"] in ("adapter", "adapter_grad"):
        return _plain_adapter(state, case)
    if case["kind"] in ("loss", "loss_grad"):
        return _plain_loss(state, case)
    return _plain_router(state, case)


# ------------------------------------------------------------------ floors
def work(case):
    kind, rows = case["kind"], case["rows"]
    if kind in ("adapter", "adapter_grad"):
        s, r, n, k = min(case["adapters"], case["requests"]), case["rank"], case["n"], case["k"]
        weights = 2 * s * r * (n + k)
        if kind == "adapter":
            return {"bytes": weights + 2 * rows * (k + 2 * n), "flops": 2 * rows * r * (n + k)}
        # every gradient of the stacks is written, in 32 bits
        return {"bytes": weights + 4 * case["adapters"] * r * (n + k) + 2 * rows * (3 * k + n),
                "flops": 2 * rows * r * (3 * k + 2 * n)}
    if kind in ("loss", "loss_grad"):
        v, h = case["vocab"], case["hidden"]
        if kind == "loss":
            return {"bytes": 2 * h * (v + rows) + 12 * rows, "flops": 2 * rows * v * h}
        return {"bytes": 4 * h * (v + rows) + 12 * rows, "flops": 6 * rows * v * h}
    e, k = case["experts"], case["topk"]
    if not case["grad"]:
        return {"bytes": 4 * rows * (e + k) + 8 * e + 4, "flops": 8 * rows * e}
    return {"bytes": 4 * rows * (2 * e + 2 * k) + 8 * e + 8, "flops": 20 * rows * e}


# ------------------------------------------------------------- 64-bit form
def _exact_adapter(t, case):
    d = {name: v.double() if v.is_floating_point() else v for name, v in t.items()}
    out = d["base"].clone()
    da, db = torch.zeros_like(d["a"]), torch.zeros_like(d["b"])
    bounds, which = t["offsets"].tolist(), t["adapters"].tolist()
    for i, a in enumerate(which):
        rows = slice(bounds[i], bounds[i + 1])
        if a < 0 or bounds[i] == bounds[i + 1]:
            continue
        down, up, scale = d["a"][a], d["b"][a], d["scale"][a]
        low = d["x"][rows] @ down.T
        if case["kind"] == "adapter":
            out[rows] += scale * (low @ up.T)
            continue
        dlow = scale * (d["dy"][rows] @ up)
        out[rows] += dlow @ down
        da[a] += dlow.T @ d["x"][rows]
        db[a] += scale * (d["dy"][rows].T @ low)
    return out if case["kind"] == "adapter" else [out, da, db]


def _exact_loss(t, case):
    x, w, target = t["x"].double(), t["w"].double(), t["target"].long()
    live = target >= 0
    index = torch.nonzero(live)[:, 0]
    if case["kind"] == "loss":
        lse = torch.logsumexp(x @ w.T, 1)
        loss = torch.zeros_like(lse)
        loss[index] = lse[index] - (x[index] * w[target[index]]).sum(1)
        return [loss, lse]
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    for part in index.split(1024):
        xs, g = x[part], t["dloss"][part].double()[:, None]
        p = torch.softmax(xs @ w.T, 1)
        dx[part] = g * (p @ w - w[target[part]])
        dw += p.T @ (g * xs)
        dw.index_add_(0, target[part], -g * xs)
    return [dx, dw]


def _exact_router(t, case):
    rows, e, k = case["rows"], case["experts"], case["topk"]
    raw = t["scores"].double().requires_grad_()
    ids = t["ids"].long()
    base = torch.sqrt(torch.nn.functional.softplus(raw, threshold=700)) if case["softplus"] else torch.exp(raw)
    counts = (ids.view(-1, 1) == torch.arange(e, device="cuda")).sum(0)
    mean = (base / base.sum(1, keepdim=True)).mean(0)
    loss = t["coefficient"] * e * (counts / (rows * k) * mean).sum().view(1)
    out = [loss.detach(), counts.to(torch.int32), mean.detach()]
    if case["grad"]:
        top = base.gather(1, ids)
        weights = top / top.sum(1, keepdim=True) * t["route_scale"]
        total = (loss * t["dloss"].double()).sum() + (weights * t["dweights"].double()).sum()
        out.append(torch.autograd.grad(total, raw)[0])
    return out


def exact(case, seed):
    t = _inputs(case, seed)
    if case["kind"] in ("adapter", "adapter_grad"):
        return _exact_adapter(t, case)
    if case["kind"] in ("loss", "loss_grad"):
        return _exact_loss(t, case)
    return _exact_router(t, case)
