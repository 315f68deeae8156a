"""The adapters, the LM-head loss and the router balance together, as a
fine-tuning step and the serving step after it use them: a frozen projection
(BF16 or FP8) with adapters on top of its output, the loss of a frozen head,
back through the head into the adapters, and the router's terms of the same
tokens.  Each stage is held to 64 bits on the stage's own inputs with the
bounds of its own test; the adapters' gradients also to autograd through all
of it."""
import pytest

from pih_amd import abi
from tests import test_gpu_adapter as adapter_test
from tests import test_gpu_lm_head_loss as loss_test

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    import torch

    from pih_amd.device import engine_stream

    with engine_stream() as s:
        yield s
        torch.cuda.synchronize()


LENGTHS, ADAPTERS, RANK, HIDDEN, VOCAB = [90, 7, 64, 40], [1, -1, 0, 1], 16, 256, 1500


def _state(seed):
    import torch

    g = torch.Generator().manual_seed(seed)
    c = adapter_test._case(seed, LENGTHS, ADAPTERS, RANK, HIDDEN, HIDDEN, 2)
    rows = sum(LENGTHS)
    c["w"] = (torch.randn(HIDDEN, HIDDEN, generator=g) * HIDDEN ** -0.5).to(torch.bfloat16)
    c["head"] = (torch.randn(VOCAB, HIDDEN, generator=g) * 0.1).to(torch.bfloat16)
    c["target"] = torch.randint(0, VOCAB, (rows,), generator=g).to(torch.int32)
    c["target"][::9] = -1
    live = c["target"] >= 0
    c["up"] = torch.where(live, 1.0 / live.sum(), 0.0).float()
    c["scores"] = torch.randn(rows, 64, generator=g)
    return c


def _base(d, kind):
    from pih_amd.linear import bf16_gemm, fp8_gemm, fp8_quant

    if kind == "bf16":
        return bf16_gemm(d["x"], d["w"])
    codes, scales, flag = fp8_quant(d["x"], abi.SCALE_F32)
    return fp8_gemm(codes, scales, d["w8"], d["w8_scale"], abi.SCALE_F32, flag=flag)[0]


def _step(d, kind, flag):
    from pih_amd.linear import (adapter_backward, adapter_gemm, lm_head_loss, lm_head_loss_backward, router_backward,
                                router_balance, router_topk)

    args = (d["a"], d["b"], d["scale"], d["offsets"], d["adapters"])
    base = _base(d, kind)
    y, _ = adapter_gemm(d["x"], *args, base=base, flag=flag)
    loss, lse, _ = lm_head_loss(y, d["head"], d["target"], flag=flag)
    dy, none, _ = lm_head_loss_backward(y, d["head"], d["target"], lse, d["up"], weight_gradient=False, flag=flag)
    dx, da, db, _ = adapter_backward(dy, d["x"], *args, flag=flag)
    ids, weights, _ = router_topk(d["scores"], 4, abi.ROUTER_SOFTMAX, flag=flag)
    balance, counts, mean, _ = router_balance(d["scores"], ids, abi.ROUTER_SOFTMAX, 0.01, flag=flag)
    dscores, _ = router_backward(d["scores"], ids, counts, abi.ROUTER_SOFTMAX, 0.01, d["one"], dweights=weights,
                                 flag=flag)
    return base, y, loss, lse, dy, dx, da, db, balance, counts, dscores


def _device(c):
    import torch

    d = {k: v.cuda() for k, v in c.items()}
    d["one"] = torch.ones(1, device="cuda")
    w = c["w"].float().view(HIDDEN // 128, 128, HIDDEN // 128, 128)
    s = w.abs().amax((1, 3)) / 448.0
    d["w8"] = (w / s[:, None, :, None]).view(HIDDEN, HIDDEN).to(torch.float8_e4m3fn).view(torch.uint8).cuda()
    d["w8_scale"] = s.contiguous().cuda()
    return d


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_step(eng, kind):
    import torch

    c = _state(3)
    d = _device(c)
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    base, y, loss, lse, dy, dx, da, db, balance, counts, dscores = _step(d, kind, flag)
    torch.cuda.synchronize()
    assert int(flag.item()) == 0 and int(counts.sum()) == 4 * sum(LENGTHS)
    # each stage on its own inputs
    at = dict(c, base=base.cpu(), dy=dy.cpu(), dbase=torch.zeros_like(c["x"]))
    ref, bound, _ = adapter_test._forward_ref(at, True)
    adapter_test._within(y, ref, bound, "y")
    _, _, rlse, elog, rloss, eloss, _, _ = loss_test._ref(y.cpu(), c["head"], c["target"])
    loss_test._within(loss, rloss, eloss, "loss")
    loss_test._within(lse, rlse, elog, "lse")
    (rdy, edy), _ = loss_test._grads_ref(y.cpu(), c["head"], c["target"], c["up"], lse.cpu())
    loss_test._within(dy, rdy, edy, "dy")
    (rdx, edx), (rda, eda), (rdb, edb) = adapter_test._backward_ref(at, False)
    adapter_test._within(dx, rdx, edx, "dx")
    adapter_test._within(da, rda, eda, "da")
    adapter_test._within(db, rdb, edb, "db")

    # autograd from the base on: y and dy are rounded to bf16 on the way (2^-8
    # of them each) and g once (2^-8): the gradients' norms are off by a few of
    # those at most
    a, b = c["a"].double().requires_grad_(), c["b"].double().requires_grad_()
    out = base.cpu().double()
    rows = []
    for lo, hi, i in adapter_test._segments(c):
        part = out[lo:hi]
        if i != abi.NO_ADAPTER:
            part = part + float(c["scale"][i]) * (c["x"][lo:hi].double() @ a[i].T) @ b[i].T
        rows.append(part)
    logits = torch.cat(rows) @ c["head"].double().T
    live = c["target"] >= 0
    torch.nn.functional.cross_entropy(logits[live], c["target"][live].long()).backward()
    for got, want in ((da, a.grad), (db, b.grad)):
        off = (got.double().cpu() - want).norm() / want.norm()
        assert float(off) <= 4 * 2.0 ** -8, float(off)


def test_step_captured_and_replayed(eng):
    import torch

    c = _state(5)
    d = _device(c)
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    _step(d, "bf16", flag)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.current_stream()):
        held = _step(d, "bf16", flag)
    for i in range(4):
        n = _state(11 + i)
        for k in ("x", "a", "target", "scores"):
            d[k].copy_(n[k].cuda())
        eager = _step(d, "bf16", flag)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(held, eager):
            assert torch.equal(p, q)
    assert int(flag.item()) == 0


def test_serving_after_an_update(eng):
    """The adapters as trained (fp32 gradients into bf16 stacks in place), then
    one decode token per request: the row of a prompt and the same row alone
    are both within the forward's bound."""
    import torch

    from pih_amd.linear import adapter_gemm

    c = _state(7)
    d = _device(c)
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    da, db = _step(d, "bf16", flag)[6:8]
    d["a"].sub_(da.to(torch.bfloat16))
    d["b"].sub_(db.to(torch.bfloat16))
    base = _base(d, "bf16")
    y, _ = adapter_gemm(d["x"], d["a"], d["b"], d["scale"], d["offsets"], d["adapters"], base=base, flag=flag)
    last = torch.tensor([89, 96, 160, 200])
    one = dict(c, a=d["a"].cpu(), b=d["b"].cpu(), x=c["x"][last], base=base.cpu()[last],
               offsets=torch.arange(5, dtype=torch.int32))
    alone, _ = adapter_gemm(d["x"][last], d["a"], d["b"], d["scale"], one["offsets"].cuda(), d["adapters"],
                            base=base[last], flag=flag)
    torch.cuda.synchronize()
    assert int(flag.item()) == 0
    ref, bound, _ = adapter_test._forward_ref(dict(one, dbase=one["x"]), True)
    adapter_test._within(alone, ref, bound, "alone")
    adapter_test._within(y[last.cuda()], ref, bound, "in the prompt")
