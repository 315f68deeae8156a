"""Router balance loss, route counts and the scores' gradient
(launch_router_balance, launch_router_backward) against 64 bits.

Counts are whole numbers and equal.  An affinity is a few fp32 functions
(expf, log1pf, sqrtf, a division: 2^-20 of it together, and |s| 2^-23 for the
shifted score), the row sums 10 additions, the sums over T rows at most
T / 4 + 300; the gradients are differences of such terms and are held to 2^-18
of the sum of the magnitudes in them."""
import numpy as np
import pytest

from pih_amd import abi

pytestmark = pytest.mark.gpu
MODES = [abi.ROUTER_SOFTMAX, abi.ROUTER_SQRT_SOFTPLUS]


@pytest.fixture(scope="module")
def eng():
    import torch

    from pih_amd.device import engine_stream

    with engine_stream() as s:
        yield s
        torch.cuda.synchronize()


def _case(seed, t, e, k, spread=1.0):
    import torch

    g = torch.Generator().manual_seed(seed)
    scores = torch.randn(t, e, generator=g) * spread - 1.1 * torch.log1p(torch.randperm(e, generator=g).float())
    ids = torch.topk(scores, k, dim=1).indices.to(torch.int32)
    return scores, ids, torch.randn(t, k, generator=g)


def _affinity(raw, mode):
    import torch

    if mode == abi.ROUTER_SOFTMAX:
        b = torch.exp(raw - raw.amax(1, keepdim=True).detach())
    else:
        b = torch.sqrt(torch.nn.functional.softplus(raw, threshold=700))
    return b


def _ref(scores, ids, mode, coefficient, dloss, dweights, scale):
    """loss, counts, mean affinities, the scores' gradient and its bound."""
    import torch

    t, e = scores.shape
    k = ids.shape[1]
    raw = scores.double().requires_grad_()
    b = _affinity(raw, mode)
    p = b / b.sum(1, keepdim=True)
    counts = torch.bincount(ids.reshape(-1).long(), minlength=e)
    loss = coefficient * e / (t * k) * (counts * p.mean(0)).sum()
    top = b.gather(1, ids.long())
    w = top / top.sum(1, keepdim=True) * scale
    total = loss * dloss + (w * dweights.double()).sum()
    grad = torch.autograd.grad(total, raw)[0]
    # magnitudes of the gradient's terms
    with torch.no_grad():
        slope = b if mode == abi.ROUTER_SOFTMAX else torch.sigmoid(raw) / (2 * b)
        weight = abs(coefficient * dloss) * e / (t * t * k)
        mag = slope / b.sum(1, keepdim=True) * weight * (counts + (counts * p).sum(1, keepdim=True))
        part = slope.gather(1, ids.long()) * scale / top.sum(1, keepdim=True)
        dw = dweights.double().abs()
        mag.scatter_add_(1, ids.long(), part * (dw + (dw * w / scale).sum(1, keepdim=True)))
    return loss.detach(), counts, p.mean(0).detach(), grad, mag * 2.0 ** -18 + 1e-37


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (1, 256, 8), (3, 64, 6), (57, 200, 5), (130, 384, 8), (1025, 256, 6),
                                   (67, 1024, 32), (4100, 128, 2)])
def test_against_64_bits(eng, t, e, k, mode):
    import torch

    from pih_amd.linear import router_backward, router_balance

    scores, ids, dweights = _case(t * 3 + e, t, e, k)
    coefficient, dloss, scale = 0.02, 0.7, 1.5
    loss, counts, mean, grad, bound = _ref(scores, ids, mode, coefficient, dloss, dweights, scale)
    s, i, dw = scores.cuda(), ids.cuda(), dweights.cuda()
    gl, gc, gm, flag = router_balance(s, i, mode, coefficient)
    up = torch.tensor([dloss], device="cuda")
    both, _ = router_backward(s, i, gc, mode, coefficient, up, dweights=dw, route_scale=scale, flag=flag)
    one, _ = router_backward(s, i, gc, mode, coefficient, up, flag=flag)
    two, _ = router_backward(s, i, None, mode, 0.0, None, dweights=dw, route_scale=scale, flag=flag)
    torch.cuda.synchronize()
    assert int(flag.item()) == 0
    assert torch.equal(gc.cpu().long(), counts)
    rel = 2.0 ** -19 + (t / 4 + 300) * 2.0 ** -24
    assert float(((gm.cpu().double() - mean).abs() / (mean + 1e-30)).max()) <= rel
    assert abs(float(gl) - float(loss)) <= (rel + e * 2.0 ** -23) * abs(float(loss))
    worst = float(((both.cpu().double() - grad).abs() / bound).max())
    print(f"worst {worst:.3f} of the bound", flush=True)
    assert worst <= 1.0
    # the two parts are what they add up to
    assert float((((one + two).cpu().double() - grad).abs() / bound).max()) <= 1.0


@pytest.mark.parametrize("mode", MODES)
def test_gradients_are_the_differences(eng, mode):
    import torch

    from pih_amd.linear import router_backward, router_balance

    scores, ids, dweights = _case(5, 7, 24, 3)
    s, i = scores.cuda(), ids.cuda()
    _, counts, _, _ = router_balance(s, i, mode, 0.3)
    got, _ = router_backward(s, i, counts, mode, 0.3, torch.ones(1, device="cuda"), dweights=dweights.cuda())

    def value(raw):
        b = _affinity(raw, mode)
        p = b / b.sum(1, keepdim=True)
        top = b.gather(1, ids.long())
        w = top / top.sum(1, keepdim=True)
        balance = 0.3 * 24 / (7 * 3) * (counts.cpu() * p.mean(0)).sum()
        return float(balance + (w * dweights.double()).sum())

    step = 1e-4  # the third derivative's step^2 / 6 is far below the bound
    for at in ((0, 0), (2, 7), (6, 23), (3, int(ids[3, 0])), (5, int(ids[5, 2]))):
        raw = scores.double()
        raw[at] += step
        high = value(raw)
        raw[at] -= 2 * step
        diff = (high - value(raw)) / (2 * step)
        assert abs(diff - float(got[at])) <= 1e-4 * abs(diff) + 1e-6, at


@pytest.mark.parametrize("mode", MODES)
def test_extreme_scores(eng, mode):
    """Scores where the affinities underflow or overflow a plain exp."""
    import torch

    from pih_amd.linear import router_backward, router_balance

    scores, ids, dweights = _case(9, 40, 64, 4, spread=30.0)
    scores[0], scores[1, :32] = -60.0, 80.0
    scores[2, 1:] = -80.0
    scores[2, 0] = 60.0
    ids = torch.topk(scores, 4, dim=1).indices.to(torch.int32)
    loss, counts, mean, grad, bound = _ref(scores, ids, mode, 0.02, 1.0, dweights, 1.0)
    s, i = scores.cuda(), ids.cuda()
    gl, gc, gm, flag = router_balance(s, i, mode, 0.02)
    got, _ = router_backward(s, i, gc, mode, 0.02, torch.ones(1, device="cuda"), dweights=dweights.cuda(), flag=flag)
    torch.cuda.synchronize()
    assert int(flag.item()) == 0 and torch.isfinite(got).all()
    # (a shifted score of s is rounded by |s| 2^-24: 140 2^-24 on top)
    assert float(((gm.cpu().double() - mean).abs() / (mean + 1e-12)).max()) <= 2.0 ** -16
    assert float(((got.cpu().double() - grad).abs() / (bound * 8 + 1e-12)).max()) <= 1.0


@pytest.mark.parametrize("mode", MODES)
def test_bad_rows_and_ids_are_flagged(eng, mode):
    import torch

    from pih_amd.linear import router_backward, router_balance

    scores, ids, dweights = _case(13, 20, 64, 4)
    clean = torch.ones(20, dtype=torch.bool)
    clean[[2, 5]] = False
    s, i, dw = scores.cuda(), ids.cuda(), dweights.cuda()
    up = torch.ones(1, device="cuda")
    s[2, 7], s[5, 0] = float("nan"), float("-inf")
    loss, counts, mean, flag = router_balance(s, i, mode, 0.02)
    got, flag2 = router_backward(s, i, counts, mode, 0.02, up, dweights=dw)
    torch.cuda.synchronize()
    assert int(flag.item()) == int(flag2.item()) == 1
    assert torch.equal(counts.cpu().long(), torch.bincount(ids.reshape(-1).long(), minlength=64))
    want = (_affinity(scores.double(), mode) / _affinity(scores.double(), mode).sum(1, keepdim=True))[clean].sum(0) / 20
    assert float(((mean.cpu().double() - want).abs() / want).max()) <= 2.0 ** -17
    assert torch.isfinite(got).all() and not got[[2, 5]].any()
    s.copy_(scores)
    i[4, 1], i[4, 2] = 64, -1
    loss, counts, mean, flag = router_balance(s, i, mode, 0.02)
    got, flag2 = router_backward(s, i, counts, mode, 0.02, up, dweights=dw)
    torch.cuda.synchronize()
    assert int(flag.item()) == int(flag2.item()) == 2
    keep = ids.reshape(-1)[[j for j in range(80) if j not in (17, 18)]]
    assert torch.equal(counts.cpu().long(), torch.bincount(keep.long(), minlength=64))
    assert torch.isfinite(got).all()
    if mode == abi.ROUTER_SQRT_SOFTPLUS:
        s[7] = -1e30  # every affinity 0
        loss, counts, mean, flag = router_balance(s, ids.cuda(), mode, 0.02)
        got, flag2 = router_backward(s, ids.cuda(), counts, mode, 0.02, up, dweights=dw)
        torch.cuda.synchronize()
        assert int(flag.item()) == int(flag2.item()) == 4 and not got[7].any() and torch.isfinite(loss).all()


def test_captured_and_replayed(eng):
    import torch

    from pih_amd.linear import router_backward, router_balance

    scores, ids, dw = [t.cuda() for t in _case(17, 700, 256, 8)]
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    up = torch.ones(1, device="cuda")

    def calls():
        loss, counts, mean, _ = router_balance(scores, ids, abi.ROUTER_SOFTMAX, 0.01, flag=flag)
        return loss, counts, mean, router_backward(scores, ids, counts, abi.ROUTER_SOFTMAX, 0.01, up, dweights=dw,
                                                   flag=flag)[0]

    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.current_stream()):
        held = calls()
    for i in range(4):
        ns, ni, _ = _case(70 + i, 700, 256, 8)
        scores.copy_(ns.cuda())
        ids.copy_(ni.cuda())
        eager = calls()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(held, eager):
            assert torch.equal(p, q)


def test_counts_are_the_route_plan_s(eng):
    """The counts against the expert offsets of launch_route_plan, after
    launch_router_topk on the same scores."""
    import torch

    from pih_amd.linear import route_plan, router_balance, router_topk

    scores = _case(19, 777, 256, 8)[0].cuda()
    ids, weights, flag = router_topk(scores, 8, abi.ROUTER_SOFTMAX)
    offsets = route_plan(ids, weights, 256, flag=flag)[0]
    _, counts, _, _ = router_balance(scores, ids, abi.ROUTER_SOFTMAX, 0.01, flag=flag)
    torch.cuda.synchronize()
    assert int(flag.item()) == 0
    np.testing.assert_array_equal(np.diff(offsets.cpu().numpy()), counts.cpu().numpy())


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("t,e,k", [(33, 67, 3), (5, 2, 2), (129, 301, 7), (40, 515, 9), (9, 1023, 31), (9001, 63, 2)])
def test_odd_expert_counts(eng, t, e, k, mode):
    """Rows that are not 16-byte aligned, and more rows than a round of blocks."""
    test_against_64_bits(eng, t, e, k, mode)


@pytest.mark.parametrize("mode", MODES)
def test_an_id_twice_is_two_routes(eng, mode):
    import torch

    from pih_amd.linear import router_backward, router_balance

    scores, ids, dweights = _case(61, 50, 96, 5)
    ids[:, 3] = ids[:, 1]
    loss, counts, mean, grad, bound = _ref(scores, ids, mode, 0.05, 1.25, dweights, 2.0)
    s, i = scores.cuda(), ids.cuda()
    _, gc, _, flag = router_balance(s, i, mode, 0.05)
    got, _ = router_backward(s, i, gc, mode, 0.05, torch.tensor([1.25], device="cuda"), dweights=dweights.cuda(),
                             route_scale=2.0, flag=flag)
    torch.cuda.synchronize()
    assert int(flag.item()) == 0 and torch.equal(gc.cpu().long(), counts)
    # (the two routes' magnitudes add up in the bound as their terms do)
    assert float(((got.cpu().double() - grad).abs() / bound).max()) <= 1.0


@pytest.mark.parametrize("mode", MODES)
def test_a_bad_row_is_zeros_whatever_its_upstream(eng, mode):
    import torch

    from pih_amd.linear import router_backward, router_balance

    scores, ids, dweights = _case(67, 21, 64, 4)
    want = _ref(scores, ids, mode, 0.1, 1.0, dweights, 1.0)[3]
    scores[8, 5] = float("nan")
    dweights[8] = torch.tensor([float("inf"), float("nan"), 1.0, -float("inf")])
    s, i, dw = scores.cuda(), ids.cuda(), dweights.cuda()
    _, counts, _, flag = router_balance(s, i, mode, 0.1)
    got, _ = router_backward(s, i, None, mode, 0.0, None, dweights=dw, flag=flag)
    nan, _ = router_backward(s, i, counts, mode, 0.1, torch.full((1,), float("nan"), device="cuda"), flag=flag)
    torch.cuda.synchronize()
    assert int(flag.item()) == 1
    assert torch.all(got[8] == 0) and torch.all(nan[8] == 0) and torch.all(nan[9].isnan())
    assert bool(torch.isfinite(got).all()) and want.shape == got.shape


def test_affinities_far_below_the_normal_exponentials(eng):
    """sqrt(softplus(s)) = e^(s/2) keeps its bits where e^s has none left
    (s < -87): rows that launch_router_topk takes, and lower ones."""
    import torch

    from pih_amd.linear import router_backward, router_balance, router_topk

    mode = abi.ROUTER_SQRT_SOFTPLUS
    g = torch.Generator().manual_seed(71)
    scores = torch.randn(96, 64, generator=g) * 3 - 95  # about -106 to -84
    scores[64:] -= 60
    assert float(scores.min()) > -172 and float(scores[:64].max()) > -90
    scores[1], scores[2, 5] = -100.0, -20.0
    dweights = torch.randn(96, 4, generator=g)
    s = scores.cuda()
    ids, _, flag = router_topk(s[:64].contiguous(), 4, mode)
    assert int(flag.item()) == 0
    ids = torch.cat((ids.cpu(), torch.topk(scores[64:], 4, dim=1).indices.to(torch.int32)))
    loss, counts, mean, grad, bound = _ref(scores, ids, mode, 0.02, 1.0, dweights, 1.5)
    i = ids.cuda()
    gl, gc, gm, _ = router_balance(s, i, mode, 0.02, flag=flag)
    got, _ = router_backward(s, i, gc, mode, 0.02, torch.ones(1, device="cuda"), dweights=dweights.cuda(),
                             route_scale=1.5, flag=flag)
    torch.cuda.synchronize()
    assert int(flag.item()) == 0 and torch.equal(gc.cpu().long(), counts)
    # an exponent of s / 2 log2 e is rounded twice: its affinity is off by |s| 2^-24
    far = 172 * 2.0 ** -24
    rel = 2.0 ** -19 + 2 * far + 324 * 2.0 ** -24
    assert float(((gm.cpu().double() - mean).abs() / mean).max()) <= rel
    assert abs(float(gl) - float(loss)) <= (rel + 64 * 2.0 ** -23) * float(loss)
    # (slope, sum, selected sum and their products: four such factors at most)
    assert float(((got.cpu().double() - grad).abs() / (bound * (1 + 4 * far * 2 ** 18))).max()) <= 1.0


@pytest.mark.parametrize("mode", MODES)
def test_routes_without_affinity_are_flagged(eng, mode):
    """A row whose routes have affinities of 0 has no route weights (bit 4 of
    launch_router_topk too, where a bias selects them): that part of its
    gradient is zeros, the balance loss's stays."""
    import torch

    from pih_amd.linear import router_backward, router_balance, router_topk

    scores, ids, dweights = _case(73, 30, 64, 4)
    scores[7, :8] = -1e30
    ids[7] = torch.tensor([0, 3, 5, 6], dtype=torch.int32)
    s, i, dw = scores.cuda(), ids.cuda(), dweights.cuda()
    one = torch.ones(1, device="cuda")
    _, counts, _, flag = router_balance(s, i, mode, 0.02)
    balance, _ = router_backward(s, i, counts, mode, 0.02, one, flag=flag)
    assert int(flag.item()) == 0  # (the whole row has affinities)
    both, flag = router_backward(s, i, counts, mode, 0.02, one, dweights=dw)
    part, flag2 = router_backward(s, i, None, mode, 0.0, None, dweights=dw)
    torch.cuda.synchronize()
    assert int(flag.item()) == int(flag2.item()) == 4
    assert not part[7].any() and torch.equal(both[7], balance[7])
    assert part[[6, 8]].any(1).all() and torch.isfinite(part).all()
    if mode == abi.ROUTER_SQRT_SOFTPLUS:
        bias = torch.zeros(64, device="cuda")
        bias[:8] = 100.0
        chosen, _, flag = router_topk(s[7:8].contiguous(), 4, mode, bias=bias)
        assert int(flag.item()) == 4 and int(chosen.max()) < 8
    # ids past the experts alone leave no route: bit 2, not 4
    i[7] = 64
    part, flag = router_backward(s, i, None, mode, 0.0, None, dweights=dw)
    torch.cuda.synchronize()
    assert int(flag.item()) == 2 and not part[7].any()
