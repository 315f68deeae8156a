"""A small draft model trained from a larger one's top logits and then used:
feed-forward block and LM head forward, distillation loss, both backward passes
and an update, eager and captured; then its drafts verified against the larger
model's logits."""
import pytest

from pih_amd import abi

pytestmark = pytest.mark.gpu

ROWS, HIDDEN, INTER, VOCAB, TOP, T = 96, 256, 512, 2048, 16, 2.0


@pytest.fixture(scope="module")
def eng():
    import torch

    from pih_amd.device import engine_stream

    with engine_stream() as s:
        yield s
        torch.cuda.synchronize()


def _model(seed, scale=1.0):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda s, *shape: (torch.randn(*shape, generator=g, device="cuda") * s).to(torch.bfloat16)  # noqa: E731
    return [n(2 * HIDDEN ** -0.5, INTER, HIDDEN), n(2 * HIDDEN ** -0.5, INTER, HIDDEN), n(INTER ** -0.5, HIDDEN, INTER),
            n(scale * HIDDEN ** -0.5, VOCAB, HIDDEN)]


def _hidden(x, model):
    from pih_amd.linear import gated_mlp

    y, gate, up = gated_mlp(x, *model[:3], keep=True)
    return x + y, gate, up


def _teacher(x, model):
    """The larger model's top logits, and the log-sum-exp of all of them."""
    import torch

    from pih_amd.linear import bf16_gemm

    logits = bf16_gemm(_hidden(x, model)[0], model[3], abi.OUTPUT_F32)
    top = torch.topk(logits, TOP, dim=1)
    return top.indices.to(torch.int32), top.values.contiguous(), torch.logsumexp(logits / T, 1)


def _loss(x, model, teacher, flag):
    from pih_amd.linear import lm_head_distill

    hidden, gate, up = _hidden(x, model)
    return (hidden, gate, up) + lm_head_distill(hidden, model[3], *teacher[:2], T, teacher_lse=teacher[2], flag=flag)[:3]


def _gradients(x, model, teacher, dloss, flag):
    """Gradients of the block's input, its three weights and the head."""
    from pih_amd.linear import gated_mlp_backward, lm_head_distill_backward

    hidden, gate, up, loss, lse, logits = _loss(x, model, teacher, flag)
    dh, dhead, _ = lm_head_distill_backward(hidden, model[3], *teacher[:2], lse, logits, dloss, T,
                                            teacher_lse=teacher[2], flag=flag)
    dx, dg, du, dd = gated_mlp_backward(dh, x, *model[:3], gate, up)
    return loss, dx + dh, [dg, du, dd, dhead]


def _inputs(seed):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(ROWS, HIDDEN, generator=g, device="cuda").to(torch.bfloat16)
    ids, values, lse = _teacher(x, _model(1, 3.0))
    ids[::7] = -1  # padding
    ids[1::5, TOP // 2:] = -1
    return x, (ids, values, lse)


def test_gradients_against_differences(eng):
    """The loss's change along each gradient.  The loss is a sum of fp32 values
    over bf16 activations: steps of 2 % of a tensor move it by far more than
    those round."""
    import torch

    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    x, teacher = _inputs(5)
    model = _model(2)
    dloss = torch.full((ROWS,), 1.0 / ROWS, device="cuda")
    _, dx, grads = _gradients(x, model, teacher, dloss, flag)
    everything = [x] + model
    for i, d in enumerate([dx] + grads):
        step = d.double() / d.double().norm() * everything[i].double().norm() * 0.02
        ends = [(everything[i].double() + s * step).to(torch.bfloat16) for s in (-1, 1)]
        value = []
        for e in ends:
            at = list(everything)
            at[i] = e
            value.append((_loss(at[0], at[1:], teacher, flag)[3].double() * dloss.double()).sum())
        moved = ((ends[1].double() - ends[0].double()) * d.double()).sum()
        print(f"{i}: {(value[1] - value[0]).item():.6f} against {moved.item():.6f}", flush=True)
        assert abs((value[1] - value[0] - moved) / moved) < 0.1
    assert int(flag.item()) == 0


def test_training_steps_captured(eng):
    """Three steps of a captured graph against three eager ones, other rows
    each time: the same weights to the bit."""
    import torch

    from pih_amd.device import engine_stream

    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    batches = [_inputs(s) for s in (5, 6, 7)]
    dloss = torch.full((ROWS,), 1.0 / ROWS, device="cuda")

    def step(x, teacher, model):
        loss, _, grads = _gradients(x, model, teacher, dloss, flag)
        for w, g in zip(model, grads):
            w.add_(g, alpha=-0.5)
        return loss

    with engine_stream() as s:
        eager, static = _model(2), _model(2)
        x = batches[0][0].clone()
        teacher = tuple(t.clone() for t in batches[0][1])
        step(x, teacher, _model(2))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            loss = step(x, teacher, static)
        for rows, entries in batches:
            x.copy_(rows)
            for t, e in zip(teacher, entries):
                t.copy_(e)
            graph.replay()
            want = step(rows, entries, eager)
            torch.cuda.synchronize()
            assert torch.equal(loss, want) and torch.isfinite(want).all()
            assert all(torch.equal(a, b) for a, b in zip(static, eager))
    assert int(flag.item()) == 0


def test_drafts_are_verified(eng):
    """Tokens drawn from the small model's logits, verified against the larger
    one's as a sequential restatement does it."""
    import numpy as np
    import torch

    from pih_amd.linear import bf16_gemm, draft_verify
    from tests.test_gpu_draft_verify import _reference

    teacher, model = _model(1, 3.0), _model(2, 3.0)
    counts = np.array([4, 0, 3, 5, 1, 2])
    offsets = np.concatenate(([0], counts.cumsum())).astype(np.int32)
    drafts, sequences = int(counts.sum()), len(counts)
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(drafts + sequences, HIDDEN, generator=g, device="cuda").to(torch.bfloat16)
    target = bf16_gemm(_hidden(x, teacher)[0], teacher[3], abi.OUTPUT_F32)
    row = np.concatenate([np.arange(c) + offsets[s] + s for s, c in enumerate(counts)]).astype(int)
    draft = bf16_gemm(_hidden(x, model)[0], model[3], abi.OUTPUT_F32)[torch.from_numpy(row).cuda()].contiguous()
    draft = (0.7 * target[torch.from_numpy(row).cuda()] + 0.3 * draft).contiguous()
    temperature = torch.tensor([1.0, 0.7, 0.0, 1.0, 0.9, 1.2])
    of = torch.from_numpy(np.repeat(np.arange(sequences), counts))
    tau = temperature[of][:, None].cuda()
    gumbel = -torch.log(-torch.log(torch.rand(draft.shape, generator=g, device="cuda").clamp(1e-20, 1 - 1e-7)))
    tokens = torch.where(tau > 0, draft / tau.clamp(min=1e-3) + gumbel, draft).argmax(1).to(torch.int32)
    accept = torch.rand(drafts, generator=g, device="cuda")
    sample = torch.rand(sequences, generator=g, device="cuda")
    out, accepted, flag = draft_verify(target, tokens, torch.from_numpy(offsets).cuda(), accept, sample, 5,
                                       draft_logits=draft, temperature=temperature.cuda())
    cpu = lambda t: t.cpu().numpy()  # noqa: E731
    want = _reference(cpu(target), cpu(tokens), offsets, cpu(accept), cpu(sample), 5, cpu(draft), temperature.numpy())
    np.testing.assert_array_equal(cpu(out), want[0])
    np.testing.assert_array_equal(cpu(accepted), want[1])
    assert int(flag.item()) == want[2] == 0
