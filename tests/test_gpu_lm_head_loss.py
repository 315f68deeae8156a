"""LM-head cross entropy without the logits (launch_lm_head_loss and its
backward) against 64 bits, element by element.

Bounds.  A logit, an fp32 sum of H products, is off by e = H 2^-23 of the sum
of their magnitudes.  The log-sum-exp moves by no more than the largest e of
its row; the sum of V exponentials (each off by 2^-21 of itself: expf and its
argument's rounding, |argument| < 8 within the values here that count) is off
by (V / 64 + 40) 2^-23 of itself in the order used (64 or more partial sums),
which the logarithm turns into an absolute error, and the result is rounded.
A gradient's element g = up (p - [target]) is off by |up| p (e + the error of
lse + 2^-21), and 2^-8 of itself for its rounding to bf16; dx and dw sum it
and round once to bf16."""
import pytest

from pih_amd import abi

pytestmark = pytest.mark.gpu
U = 2.0 ** -23
HALF_BF16 = 2.0 ** -8


@pytest.fixture(scope="module")
def eng():
    import torch

    from pih_amd.device import engine_stream

    with engine_stream() as s:
        yield s
        torch.cuda.synchronize()


def _case(seed, rows, vocab, hidden, masked=0.2, std=0.3):
    import torch

    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, hidden, generator=g).to(torch.bfloat16)
    w = (torch.randn(vocab, hidden, generator=g) * std * (64 / hidden) ** 0.5).to(torch.bfloat16)
    target = torch.randint(0, vocab, (rows,), generator=g).to(torch.int32)
    if rows > 1:
        target[torch.rand(rows, generator=g) < masked] = -1
    up = torch.randn(rows, generator=g)
    return x, w, target, up


def _ref(x, w, target):
    """lse, loss, the probabilities and the error of logits and lse."""
    import torch

    rows = x.shape[0]
    xd, wd = x.double(), w.double()
    logits = xd @ wd.T
    e = xd.abs() @ wd.abs().T * (x.shape[1] + 8) * U
    lse = torch.logsumexp(logits, 1)
    elog = e.max(1).values + (w.shape[0] / 64 + 48) * U + lse.abs() * 2 * U
    live = target >= 0
    at = target.clamp(min=0).long()
    loss = torch.where(live, lse - logits[torch.arange(rows, device=x.device), at], torch.zeros((), dtype=torch.float64, device=x.device))
    eloss = elog + e[torch.arange(rows, device=x.device), at] + loss.abs() * U
    return logits, e, lse, elog, loss, eloss, live, at


def _within(got, ref, bound, what):
    worst = ((got.double().cpu() - ref).abs() / bound).max().item()
    print(f"{what}: worst {worst:.3f} of the bound", flush=True)
    assert worst <= 1.0, (what, worst)


SIZES = [(1, 1, 8), (1, 1000, 64), (3, 5, 72), (2, 63, 256), (17, 64, 200), (33, 65, 128), (16, 257, 64), (65, 130, 320),
         (64, 1024, 512), (100, 513, 1024), (130, 2050, 192), (257, 777, 264), (300, 5000, 128), (515, 300, 64)]


@pytest.mark.parametrize("rows,vocab,hidden", SIZES)
def test_forward(eng, rows, vocab, hidden):
    import torch

    from pih_amd.linear import lm_head_loss

    x, w, target, _ = _case(rows * 7 + vocab, rows, vocab, hidden)
    _, _, lse, elog, loss, eloss, live, _ = _ref(x, w, target)
    got, glse, flag = lm_head_loss(x.cuda(), w.cuda(), target.cuda())
    torch.cuda.synchronize()
    assert int(flag.item()) == 0
    _within(glse, lse, elog, "lse")
    _within(got, loss, eloss, "loss")
    assert torch.all(got.cpu()[~live] == 0)


def _grads_ref(x, w, target, up, lse32):
    import torch

    logits, e, _, _, _, _, live, at = _ref(x, w, target)
    xd, wd = x.double(), w.double()
    rows, vocab = logits.shape
    p = torch.exp(logits - lse32.double()[:, None])
    upd = torch.where(live, up.double(), torch.zeros((), dtype=torch.float64, device=x.device))[:, None]
    g = p.clone()
    g[torch.arange(rows, device=x.device), at] -= 1
    g *= upd
    arg = (logits - lse32.double()[:, None]).abs()
    eg = upd.abs() * p * (1.1 * e + (arg + 4) * U + 2.0 ** -21) + g.abs() * (2 * U + HALF_BF16) + upd.abs() * U
    dx, dw = g @ wd, g.T @ xd
    ex = eg @ wd.abs() + (g.abs() + eg) @ wd.abs() * (2 * vocab + 64) * U
    ew = eg.T @ xd.abs() + (g.abs() + eg).T @ xd.abs() * (2 * rows + 64) * U
    return (dx, ex + (dx.abs() + ex) * HALF_BF16 + 1e-37), (dw, ew + (dw.abs() + ew) * HALF_BF16 + 1e-37)


@pytest.mark.parametrize("rows,vocab,hidden", SIZES)
def test_backward(eng, rows, vocab, hidden):
    import torch

    from pih_amd.linear import lm_head_loss_backward

    x, w, target, up = _case(rows * 5 + vocab, rows, vocab, hidden)
    lse = _ref(x, w, target)[2].float()
    (dx, ex), (dw, ew) = _grads_ref(x, w, target, up, lse)
    args = [t.cuda() for t in (x, w, target, lse, up)]
    gx, gw, flag = lm_head_loss_backward(*args)
    hx, hw, _ = lm_head_loss_backward(*args)
    only, none, _ = lm_head_loss_backward(*args, weight_gradient=False)
    torch.cuda.synchronize()
    assert int(flag.item()) == 0 and none is None
    _within(gx, dx, ex, "dx")
    _within(gw, dw, ew, "dw")
    assert torch.equal(gx, hx) and torch.equal(gw, hw) and torch.equal(gx, only)
    assert torch.all(gx.cpu()[target < 0] == 0)


def test_several_pieces_of_the_vocabulary(eng):
    """More columns than a piece holds (about 2^26 elements, 60928 columns at
    these rows); 64 bits on the GPU."""
    import torch

    from pih_amd.linear import lm_head_loss, lm_head_loss_backward

    x, w, target, up = [t.cuda() for t in _case(3, 1100, 60928 * 2 + 1003, 64)]
    target[0], target[1], target[2] = 60927, 60928, 60928 * 2 + 1002
    logits, e, lse, elog, loss, eloss, _, _ = _ref(x, w, target)
    del logits, e
    got, glse, _ = lm_head_loss(x, w, target)
    _within(glse, lse.cpu(), elog.cpu(), "lse")
    _within(got, loss.cpu(), eloss.cpu(), "loss")
    gx, gw, flag = lm_head_loss_backward(x, w, target, glse, up)
    (dx, ex), (dw, ew) = _grads_ref(x, w, target, up, glse)
    assert int(flag.item()) == 0
    _within(gx, dx.cpu(), ex.cpu(), "dx")
    _within(gw, dw.cpu(), ew.cpu(), "dw")


def test_gradients_are_the_differences(eng):
    """dx and dw against central differences of the 64-bit loss."""
    import torch

    from pih_amd.linear import lm_head_loss, lm_head_loss_backward

    x, w, target, up = _case(29, 6, 40, 64)
    args = [t.cuda() for t in (x, w, target)]
    _, lse, _ = lm_head_loss(*args)
    dx, dw, _ = lm_head_loss_backward(*args, lse, up.cuda())

    def value(xd, wd):
        return float((_ref(xd, wd, target)[4] * up.double()).sum())

    # the loss's third derivative times step^2 / 6 is below 1e-6 here (|w|, |x|
    # < 5); g's rounding and the output's, 2^-8 each of sums of magnitudes
    step = 1e-3
    for grad, which, places in ((dx, 0, ((0, 0), (3, 17), (5, 63))), (dw, 1, ((0, 1), (11, 30), (39, 63)))):
        scale = float(grad.double().abs().mean())
        for at in places:
            pair = []
            for sign in (1, -1):
                t = [x.double(), w.double()]
                t[which][at] += sign * step
                pair.append(value(*t))
            diff = (pair[0] - pair[1]) / (2 * step)
            assert abs(diff - float(grad[at])) <= 4 * HALF_BF16 * (abs(diff) + scale) + 1e-5, (which, at)


def test_rows_without_target_do_not_matter(eng):
    """NaN and infinities in masked rows, their lse and upstream gradient."""
    import torch

    from pih_amd.linear import lm_head_loss, lm_head_loss_backward

    x, w, target, up = [t.cuda() for t in _case(31, 70, 300, 128, masked=0.4)]
    loss, lse, _ = lm_head_loss(x, w, target)
    want = lm_head_loss_backward(x, w, target, lse, up)
    dead = target < 0
    x[dead], up[dead], lse2 = float("nan"), float("inf"), lse.clone()
    lse2[dead] = float("nan")
    got_loss, got_lse, flag = lm_head_loss(x, w, target)
    got = lm_head_loss_backward(x, w, target, lse2, up)
    torch.cuda.synchronize()
    assert int(flag.item()) == 0
    assert torch.equal(got_loss, loss) and torch.equal(got_lse[~dead], lse[~dead])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_no_target_at_all(eng):
    import torch

    from pih_amd.linear import lm_head_loss, lm_head_loss_backward

    x, w, target, up = [t.cuda() for t in _case(37, 19, 100, 64)]
    target.fill_(-1)
    loss, lse, flag = lm_head_loss(x, w, target)
    dx, dw, flag2 = lm_head_loss_backward(x, w, target, lse, up)
    torch.cuda.synchronize()
    assert int(flag.item()) == int(flag2.item()) == 0
    assert not loss.any() and not dx.any() and not dw.any() and torch.isfinite(lse).all()


def test_bad_targets_and_values_are_flagged(eng):
    import torch

    from pih_amd.linear import lm_head_loss, lm_head_loss_backward

    x, w, target, up = [t.cuda() for t in _case(41, 20, 100, 64, masked=0.0)]
    loss, lse, _ = lm_head_loss(x, w, target)
    target[3] = 100
    got, got_lse, flag = lm_head_loss(x, w, target)
    assert int(flag.item()) == 1 and float(got[3]) == 0.0 and torch.equal(got_lse, lse)
    dx, dw, flag = lm_head_loss_backward(x, w, target, lse, up)
    assert int(flag.item()) == 1 and not dx[3].any() and torch.isfinite(dw).all()
    target[3] = -1
    ref = lm_head_loss_backward(x, w, target, lse, up)
    assert torch.equal(dx, ref[0]) and torch.equal(dw, ref[1])
    x[5, 0] = float("inf")
    got, got_lse, flag = lm_head_loss(x, w, target)
    torch.cuda.synchronize()
    assert int(flag.item()) == 4 and not torch.isfinite(got[5]) and torch.isfinite(got[[0, 1, 2, 4, 6]]).all()


def test_large_logits(eng):
    """Logits up to about +-3000: the maximum is taken out, nothing overflows."""
    import torch

    from pih_amd.linear import lm_head_loss

    x, w, target, _ = _case(43, 40, 500, 256, std=60.0)
    _, _, lse, elog, loss, eloss, _, _ = _ref(x, w, target)
    got, glse, flag = lm_head_loss(x.cuda(), w.cuda(), target.cuda())
    torch.cuda.synchronize()
    assert int(flag.item()) == 0 and float(lse.abs().max()) > 1000
    _within(glse, lse, elog, "lse")
    _within(got, loss, eloss, "loss")


def test_loss_is_the_logits_log_probability(eng):
    """Beside the LM head that stores its logits (launch_lm_head, fp32)."""
    import torch

    from pih_amd.linear import deepseek_lm_head, lm_head_loss

    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(5, 4096, device="cuda", generator=g).to(torch.bfloat16)
    w = (torch.randn(129280, 4096, device="cuda", generator=g) * 0.02).to(torch.bfloat16)
    target = torch.tensor([0, 129279, 70000, 255, 256], dtype=torch.int32, device="cuda")
    logits, _ = deepseek_lm_head(x, w)
    loss, lse, flag = lm_head_loss(x, w, target)
    want = torch.log_softmax(logits.double(), 1).gather(1, target.long()[:, None])[:, 0]
    torch.cuda.synchronize()
    # each logit within 4096 2^-23 of its magnitudes' sum (about 0.016 x 4096 = 65)
    assert int(flag.item()) == 0 and float((loss.double() + want).abs().max()) <= 2 * 4096 * U * 80


def test_captured_and_replayed(eng):
    import torch

    from pih_amd.linear import lm_head_loss, lm_head_loss_backward

    x, w, target, up = [t.cuda() for t in _case(47, 200, 3000, 256)]
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")

    def calls():
        loss, lse, _ = lm_head_loss(x, w, target, flag=flag)
        return (loss, lse) + lm_head_loss_backward(x, w, target, lse, up, flag=flag)[:2]

    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.current_stream()):
        held = calls()
    for i in range(4):
        nx, _, nt, _ = _case(60 + i, 200, 3000, 256)
        x.copy_(nx.cuda())
        target.copy_(nt.cuda())
        eager = calls()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(held, eager):
            assert torch.equal(p, q)
    assert int(flag.item()) == 0


# tiles of 128 and 256 rows (the sizes above take 64), of every product: the
# logits' in the first two, dx's in the next two, whose columns are split too;
# and the logits in two launches, of 768 rows and the 22 behind them
@pytest.mark.parametrize("rows,vocab,hidden", [(1003, 8190, 64), (301, 29999, 64), (1000, 8200, 2048),
                                               (190, 16380, 2048), (790, 20400, 128)])
def test_taller_tiles(eng, rows, vocab, hidden):
    import torch

    from pih_amd.linear import lm_head_loss, lm_head_loss_backward

    x, w, target, up = (t.cuda() for t in _case(rows + vocab, rows, vocab, hidden))
    _, _, lse, elog, loss, eloss, live, _ = _ref(x, w, target)
    got, glse, flag = lm_head_loss(x, w, target)
    torch.cuda.synchronize()
    _within(glse, lse.cpu(), elog.cpu(), "lse")
    _within(got, loss.cpu(), eloss.cpu(), "loss")
    (dx, ex), (dw, ew) = _grads_ref(x, w, target, up, lse.float())
    gx, gw, _ = lm_head_loss_backward(x, w, target, lse.float(), up, flag=flag)
    torch.cuda.synchronize()
    assert int(flag.item()) == 0 and torch.all(got[~live] == 0) and torch.all(gx[~live] == 0)
    _within(gx, dx.cpu(), ex.cpu(), "dx")
    _within(gw, dw.cpu(), ew.cpu(), "dw")


def test_other_streams_at_once(eng):
    """Forward and backward on two streams, each with the workspaces of its own calls."""
    import torch

    from pih_amd.linear import lm_head_loss, lm_head_loss_backward

    cases = [[t.cuda() for t in _case(90 + i, 200, 3000, 256)] for i in range(2)]

    def call(x, w, target, up):
        loss, lse, flag = lm_head_loss(x, w, target)
        return (loss,) + lm_head_loss_backward(x, w, target, lse, up, flag=flag)[:2]

    want = [call(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(*cases[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(p, q) for g in got[i] for p, q in zip(g, want[i]))


def test_weights_past_4_gib(eng):
    """2^20 vocabulary entries of 2112 (4.4 GB), 1009 different ones over and
    over: the sums follow from those, each so many times."""
    import torch

    from pih_amd.linear import lm_head_loss, lm_head_loss_backward

    vocab, hidden, rows, kinds = 1 << 20, 2112, 5, 1009
    x, few, _, up = (t.cuda() for t in _case(97, rows, kinds, hidden))
    w = few.repeat((vocab + kinds - 1) // kinds, 1)[:vocab].contiguous()
    target = torch.tensor([0, vocab - 1, 123456, vocab // 2 + 7, vocab - 300], dtype=torch.int32, device="cuda")
    logits, e, _, _, _, _, _, _ = _ref(x, few, target % kinds)
    times = torch.bincount(torch.arange(vocab, device="cuda") % kinds, minlength=kinds).double()
    lse = torch.logsumexp(logits + times.log(), 1)
    elog = e.max(1).values + (vocab / 64 + 48) * U + lse.abs() * 2 * U
    at = (target.long() % kinds)[:, None]
    loss = lse - logits.gather(1, at)[:, 0]
    got, glse, flag = lm_head_loss(x, w, target)
    _within(glse, lse.cpu(), elog.cpu(), "lse")
    _within(got, loss.cpu(), (elog + e.gather(1, at)[:, 0] + loss.abs() * U).cpu(), "loss")
    gx, gw, _ = lm_head_loss_backward(x, w, target, glse, up, flag=flag)
    torch.cuda.synchronize()
    assert int(flag.item()) == 0
    # (an entry's gradient in the last 1009 of them and around the targets)
    for first in (0, 123456 - 4, vocab // 2, vocab - kinds):
        take = torch.arange(first, min(first + kinds, vocab), device="cuda")
        g = torch.exp(logits - glse.double()[:, None])[:, take % kinds]
        eg = up.double().abs()[:, None] * g * (1.1 * e[:, take % kinds] + 64 * U + 2.0 ** -21)
        g = (g - (take == target[:, None]).double()) * up.double()[:, None]
        eg += g.abs() * (2 * U + HALF_BF16) + up.double().abs()[:, None] * U
        ref = g.T @ x.double()
        err = eg.T @ x.double().abs() * 1.01
        err += ref.abs() * HALF_BF16 + 1e-37
        _within(gw[take], ref.cpu(), (err + 256 * U * (g.abs().T @ x.double().abs())).cpu(), f"dw from {first}")
    assert bool(torch.isfinite(gx).all())


@pytest.mark.parametrize("hidden", [64, 72])
def test_targets_beside_every_tile_s_edge(eng, hidden):
    """Targets in the last and the first column of every 256-column tile, and
    so on either side of wherever a piece of the vocabulary ends (a piece is
    whole tiles; these sizes have more columns than one holds: (4/3) 2^26
    elements, 81152 columns at 1100 rows).  64 bits on the GPU."""
    import torch

    from pih_amd.linear import lm_head_loss, lm_head_loss_backward

    rows, vocab = 1100, 122859
    x, w, target, up = [t.cuda() for t in _case(7, rows, vocab, hidden, masked=0.0)]
    edges = torch.arange(256, vocab, 256, dtype=torch.int32, device="cuda")
    target[:2 * len(edges)] = torch.stack((edges - 1, edges), 1).reshape(-1)
    target[-1] = vocab - 1
    _, e, lse, elog, loss, eloss, _, _ = _ref(x, w, target)
    got, glse, _ = lm_head_loss(x, w, target)
    _within(glse, lse.cpu(), elog.cpu(), "lse")
    _within(got, loss.cpu(), eloss.cpu(), "loss")
    del e
    gx, gw, flag = lm_head_loss_backward(x, w, target, glse, up)
    (dx, ex), (dw, ew) = _grads_ref(x, w, target, up, glse)
    torch.cuda.synchronize()
    assert int(flag.item()) == 0
    _within(gx, dx.cpu(), ex.cpu(), "dx")
    _within(gw, dw.cpu(), ew.cpu(), "dw")


# one piece of the vocabulary, and two whose sums of dx are added up
@pytest.mark.parametrize("vocab", [5000, 30011])
def test_input_gradient_in_two_launches(eng, vocab):
    """dx of 4096 rows and the 4 behind them: a round of 256 tiles of 256 x
    256, where one more row of tiles would cost a second round."""
    import torch

    from pih_amd.linear import lm_head_loss_backward

    x, w, target, up = [t.cuda() for t in _case(11, 4100, vocab, 4096)]
    lse = torch.logsumexp(x.double() @ w.double().T, 1).float()
    gx, gw, flag = lm_head_loss_backward(x, w, target, lse, up)
    (dx, ex), (dw, ew) = _grads_ref(x, w, target, up, lse)
    torch.cuda.synchronize()
    assert int(flag.item()) == 0 and torch.all(gx[target < 0] == 0)
    _within(gx, dx.cpu(), ex.cpu(), "dx")
    _within(gx[4090:], dx[4090:].cpu(), ex[4090:].cpu(), "dx around row 4096")
    _within(gw, dw.cpu(), ew.cpu(), "dw")


def test_input_gradient_of_weights_past_4_gib(eng):
    """dx over 2^20 entries of 2112 where two thirds of every row's probability
    lie past 2^32 bytes: 1009 different entries over and over up to there, 211
    others behind it, each five of which point along one of the rows of x.

    A term of dx is off as in _grads_ref, without up 2^-23 but for the target,
    whose 1 is subtracted; the sum runs in 16 parts or more."""
    import torch

    from pih_amd.linear import lm_head_loss_backward

    vocab, hidden, rows, kinds, late = 1 << 20, 2112, 5, 1009, 211
    x, few, _, up = (t.cuda() for t in _case(101, rows, kinds, hidden))
    g = torch.Generator(device="cuda").manual_seed(103)
    along = x[torch.arange(late, device="cuda") % rows].float() * 0.004
    along = (along + torch.randn(late, hidden, device="cuda", generator=g) * 0.002).to(torch.bfloat16)
    first = (1 << 32) // (2 * hidden) + 1
    every = torch.cat((few, along))
    v = torch.arange(vocab, device="cuda")
    kind = torch.where(v < first, v % kinds, kinds + v % late)
    w = every[kind].contiguous()
    target = torch.tensor([0, vocab - 1, first - 1, first, vocab - 300], dtype=torch.int32, device="cuda")
    times = torch.bincount(kind, minlength=kinds + late).double()
    logits, e, _, _, _, _, _, _ = _ref(x, every, kind[target.long()])
    lse = torch.logsumexp(logits + times.log(), 1).float()
    p = torch.exp(logits - lse.double()[:, None])
    assert float((p * times)[:, kinds:].sum(1).min()) > 0.3
    gx, none, flag = lm_head_loss_backward(x, w, target, lse, up, weight_gradient=False)
    torch.cuda.synchronize()
    assert int(flag.item()) == 0 and none is None
    u = up.double()[:, None]
    of = every[kind[target.long()]].double()
    ref = (u * p * times) @ every.double() - u * of
    arg = (logits - lse.double()[:, None]).abs()
    terms = u.abs() * p * (1 + 1.1 * e)
    eg = u.abs() * p * (1.1 * e + (arg + 4) * U + 2.0 ** -21) + terms * (2 * U + HALF_BF16)
    size = (terms * times) @ every.double().abs() + u.abs() * of.abs()
    err = (eg * times) @ every.double().abs() + u.abs() * of.abs() * (3 * U + HALF_BF16) + size * (vocab / 16 + 64) * U
    _within(gx, ref.cpu(), (err + (ref.abs() + err) * HALF_BF16 + 1e-37).cpu(), "dx")
    # (what lies past 2^32 bytes is most of the value: the bound holds it apart)
    lost = (u * (p * times)[:, kinds:]) @ along.double()
    assert float((lost.abs() / err).max()) > 4


@pytest.mark.parametrize("rows,vocab,hidden", [(33, 1000, 128), (300, 5000, 128), (1003, 8190, 64), (790, 20400, 128),
                                               (70, 1000, 72)])
def test_forward_stays_in_its_workspace(eng, rows, vocab, hidden):
    import torch

    from pih_amd import linear

    x, w, target, _ = (t.cuda() for t in _case(111, rows, vocab, hidden))
    want = linear.lm_head_loss(x, w, target)
    need = linear._workspace_bytes(abi.WORKSPACE_LM_HEAD_LOSS, rows, vocab, hidden)
    ws = torch.full((need + 65536,), 0x5A, dtype=torch.uint8, device="cuda")
    loss, lse = (torch.empty(rows, dtype=torch.float32, device="cuda") for _ in range(2))
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    linear._launch("launch_lm_head_loss", "lm_head_loss", x.data_ptr(), w.data_ptr(), target.data_ptr(), loss.data_ptr(),
                   lse.data_ptr(), ws.data_ptr(), need, flag.data_ptr(), linear.stream_handle(), rows, vocab, hidden)
    torch.cuda.synchronize()
    assert int(flag.item()) == 0 and torch.all(ws[need:] == 0x5A)
    assert torch.equal(loss, want[0]) and torch.equal(lse, want[1])


@pytest.mark.parametrize("rows,vocab,hidden", [(70, 300, 1024), (65, 500, 1000)])
def test_a_frozen_head_leaves_the_copy_of_the_rows_out(eng, rows, vocab, hidden):
    """Without dw the workspace's scaled copy of x, which only dw reads, is not
    written (its bytes, of rows up to a multiple of 64, keep their pattern), and
    dx has the bits that it has beside dw."""
    import torch

    from pih_amd import linear

    x, w, target, up = (t.cuda() for t in _case(113, rows, vocab, hidden))
    lse = torch.logsumexp(x.double() @ w.double().T, 1).float()
    target[5] = -1
    want = linear.lm_head_loss_backward(x, w, target, lse, up)[0]
    need = linear._workspace_bytes(abi.WORKSPACE_LM_HEAD_LOSS_BACKWARD, rows, vocab, hidden)
    ws = torch.full((need,), 0x5A, dtype=torch.uint8, device="cuda")
    dx, flag = torch.empty_like(x), torch.zeros(1, dtype=torch.int32, device="cuda")
    target[5] = vocab + 3
    linear._launch("launch_lm_head_loss_backward", "lm_head_loss_backward", x.data_ptr(), w.data_ptr(), target.data_ptr(),
                   lse.data_ptr(), up.data_ptr(), dx.data_ptr(), 0, ws.data_ptr(), need, flag.data_ptr(),
                   linear.stream_handle(), rows, vocab, hidden)
    torch.cuda.synchronize()
    assert int(flag.item()) == 1  # (a bad target is reported as ever)
    assert int((ws == 0x5A).sum()) >= (rows + 63) // 64 * 64 * hidden * 2
    assert torch.equal(dx, want)
