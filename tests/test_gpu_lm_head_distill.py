"""Divergence of an LM head from a teacher's top logits (launch_lm_head_distill
and its backward) against 64 bits, element by element.

Bounds.  A logit, an fp32 sum of H products, is off by e = (H + 8) 2^-23 of the
sum of their magnitudes.  The log-sum-exp over the temperature T moves by no
more than the largest e / T of its row; the sum of V exponentials is off by (V /
64 + 48) 2^-23 of itself as the cross entropy's is, and the result is rounded.
A teacher's s = logit / T is off by |s| 2^-22 and its log-normalizer by as much
and by 24 units of 2^-22 (its sum of at most 256 exponentials, the logarithm),
which its probabilities q = exp(s - normalizer) take as a relative error eq.  A
gradient's element g = up T (Q p - q) is off by |up| T (Q p (e / T + |argument|
2^-23 + 2^-20 + eq) + q eq), and 2^-8 of itself for its rounding to bf16; dx and
dw sum it and round once to bf16."""
import pytest

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


def _case(seed, rows, vocab, hidden, top_k, device="cpu", empty=0.2, std=0.3):
    """x, w, ids, teacher logits, the log-sum-exp of more logits than those,
    and an upstream gradient.  Entries are absent at random, rows are empty at
    random, and an id may come twice."""
    import torch

    g = torch.Generator(device=device).manual_seed(seed)
    rand = lambda *s: torch.rand(*s, generator=g, device=device)  # noqa: E731
    x = torch.randn(rows, hidden, generator=g, device=device).to(torch.bfloat16)
    w = (torch.randn(vocab, hidden, generator=g, device=device) * std * (64 / hidden) ** 0.5).to(torch.bfloat16)
    ids = (rand(rows, top_k) * vocab).long().clamp_(max=vocab - 1).to(torch.int32)
    if top_k > 2:
        ids[::3, 1] = ids[::3, 0]
    teacher = torch.randn(rows, top_k, generator=g, device=device) * 2
    ids[rand(rows, top_k) < 0.2] = -1
    if rows > 1:
        ids[rand(rows) < empty] = -1
    more = torch.randn(rows, 50, generator=g, device=device)
    return x, w, ids, teacher, more, torch.randn(rows, generator=g, device=device)


def _teacher_ref(ids, teacher, more, temperature, tail):
    """q, log q (0 where absent), their relative error, and the log-sum-exp
    that the call takes."""
    import torch

    there = ids >= 0
    s = torch.where(there, teacher.double() / temperature, -torch.inf)
    if tail:
        lse = torch.logsumexp(torch.cat((s, more.double() / temperature), 1), 1).float()
        norm = lse.double()
    else:
        lse = None
        norm = torch.logsumexp(s, 1)
    norm = torch.where(torch.isfinite(norm), norm, 0.0)[:, None]
    log_q = torch.where(there, s - norm, 0.0)
    q = torch.where(there, torch.exp(log_q), 0.0)
    size = torch.where(there, s.abs(), 0.0)
    eq = (size.amax(1, keepdim=True) + norm.abs() + 24) * 2.0 ** -22
    return there, q, log_q, eq, lse


def _forward_ref(x, w, ids, teacher, more, temperature, tail):
    import torch

    xd, wd = x.double(), w.double()
    logits = xd @ wd.T
    e = xd.abs() @ wd.abs().T * (x.shape[1] + 8) * U
    there, q, log_q, eq, teacher_lse = _teacher_ref(ids, teacher, more, temperature, tail)
    at = ids.clamp(min=0).long()
    lse = torch.logsumexp(logits / temperature, 1)
    elog = e.max(1).values / temperature + (w.shape[0] / 64 + 48) * U + (lse.abs() + (logits / temperature).abs().amax(1)) * 2 * U
    z = torch.where(there, logits.gather(1, at), 0.0)
    ez = torch.where(there, e.gather(1, at), 0.0)
    gap = log_q - z / temperature + lse[:, None]
    loss = temperature ** 2 * torch.where(there, q * gap, 0.0).sum(1)
    egap = ez / temperature + elog[:, None] + eq + (log_q.abs() + (z / temperature).abs() + lse.abs()[:, None]) * 2 * U
    part = q * (eq * (gap.abs() + egap) + egap)
    eloss = temperature ** 2 * (part + q * gap.abs() * (ids.shape[1] / 64 + 16) * U).sum(1) + loss.abs() * 8 * U + 1e-30
    return teacher_lse, (loss, eloss), (lse, elog), (z, ez + 1e-30)


def _within(got, want, what):
    value, bound = want
    assert got.shape == value.shape, what
    worst = ((got.double().to(value.device) - value).abs() / bound).max().item()
    print(f"{what}: worst {worst:.3f} of the bound", flush=True)
    assert worst <= 1.0, (what, worst)


def _grads_ref(x, w, ids, teacher, more, up, lse, temperature, tail):
    import torch

    xd, wd = x.double(), w.double()
    rows, vocab = x.shape[0], w.shape[0]
    logits = xd @ wd.T / temperature
    e = xd.abs() @ wd.abs().T * (x.shape[1] + 8) * U / temperature
    there, q, _, eq, _ = _teacher_ref(ids, teacher, more, temperature, tail)
    total = q.sum(1, keepdim=True)
    arg = logits - lse.double()[:, None]
    p = torch.exp(arg) * total
    upt = up.double()[:, None] * temperature
    at = ids.clamp(min=0).long()
    g = (p.clone().scatter_add_(1, at, -q)) * upt
    eg = p * (1.1 * e + (arg.abs() + lse.double().abs()[:, None] + logits.abs() + 4) * U + 2.0 ** -20 + eq)
    eg = eg.scatter_add_(1, at, q * eq) * upt.abs()
    eg += (g.abs() + eg) * (HALF_BF16 + 2 * U)
    live = there.any(1, keepdim=True)
    g, eg = torch.where(live, g, 0.0), torch.where(live, eg, 0.0)
    dx, dw = g @ wd, g.T @ xd
    ex = eg @ wd.abs() + (g.abs() + eg) @ wd.abs() * (2 * vocab + 64) * U
    ew = eg.T @ xd.abs() + (g.abs() + eg).T @ xd.abs() * (2 * rows + 64) * U
    return (dx, ex + (dx.abs() + ex) * HALF_BF16 + 1e-37), (dw, ew + (dw.abs() + ew) * HALF_BF16 + 1e-37)


SIZES = [(1, 1, 8, 1), (1, 1000, 64, 5), (3, 5, 72, 3), (2, 63, 256, 64), (17, 64, 200, 65), (33, 65, 128, 7),
         (16, 257, 64, 256), (65, 130, 320, 1), (64, 1024, 512, 20), (100, 513, 1024, 130), (130, 2050, 192, 32),
         (257, 777, 264, 9), (300, 5000, 128, 64), (515, 300, 64, 4)]


@pytest.mark.parametrize("rows,vocab,hidden,top_k", SIZES)
@pytest.mark.parametrize("temperature,tail", [(1.0, False), (2.0, True), (0.7, False)])
def test_forward(eng, rows, vocab, hidden, top_k, temperature, tail):
    import torch

    from pih_amd.linear import lm_head_distill

    case = _case(rows * 7 + vocab, rows, vocab, hidden, top_k)
    teacher_lse, loss, lse, z = _forward_ref(*case[:5], temperature, tail)
    x, w, ids, teacher = (t.cuda() for t in case[:4])
    got = lm_head_distill(x, w, ids, teacher, temperature, teacher_lse=None if teacher_lse is None else teacher_lse.cuda())
    torch.cuda.synchronize()
    assert int(got[3].item()) == 0
    _within(got[1], lse, "lse")
    _within(got[2], z, "logits")
    _within(got[0], loss, "loss")
    empty = (case[2] < 0).all(1)
    assert torch.all(got[0].cpu()[empty] == 0) and torch.all(got[2].cpu()[case[2] < 0] == 0)


@pytest.mark.parametrize("rows,vocab,hidden,top_k", SIZES)
@pytest.mark.parametrize("temperature,tail", [(1.0, False), (2.0, True), (0.7, False)])
def test_backward(eng, rows, vocab, hidden, top_k, temperature, tail):
    import torch

    from pih_amd.linear import lm_head_distill_backward

    case = _case(rows * 5 + vocab, rows, vocab, hidden, top_k)
    teacher_lse, _, lse, z = _forward_ref(*case[:5], temperature, tail)
    lse, z = lse[0].float(), z[0].float()
    dx, dw = _grads_ref(*case[:5], case[5], lse, temperature, tail)
    x, w, ids, teacher = (t.cuda() for t in case[:4])
    args = (x, w, ids, teacher, lse.cuda(), z.cuda(), case[5].cuda(), temperature)
    more = dict(teacher_lse=None if teacher_lse is None else teacher_lse.cuda())
    for n in (1 << 12, 1 << 16, 1 << 20, 1 << 24):
        torch.full((n,), float("nan"), device="cuda")  # freed: later allocations get it
    gx, gw, flag = lm_head_distill_backward(*args, **more)
    hx, hw, _ = lm_head_distill_backward(*args, **more)
    only, none, _ = lm_head_distill_backward(*args, weight_gradient=False, **more)
    torch.cuda.synchronize()
    assert int(flag.item()) == 0 and none is None
    _within(gx, dx, "dx")
    _within(gw, dw, "dw")
    assert torch.equal(gx, hx) and torch.equal(gw, hw) and torch.equal(gx, only)
    assert torch.all(gx.cpu()[(case[2] < 0).all(1)] == 0)


@pytest.mark.parametrize("rows,vocab,hidden,top_k", [(33, 151936, 1024, 20), (1100, 60928 * 2 + 1003, 64, 128),
                                                     (600, 32768, 2048, 64)])
def test_large(eng, rows, vocab, hidden, top_k):
    """More columns than a piece of the backward pass holds, 64 bits on the
    GPU; ids on either side of the pieces' and tiles' borders."""
    import torch

    from pih_amd.linear import lm_head_distill, lm_head_distill_backward

    case = _case(rows, rows, vocab, hidden, top_k, "cuda")
    ids = case[2]
    for i, v in enumerate((0, 255, 256, 60927, 60928, vocab - 1)):
        ids[i % rows, i % top_k] = min(v, vocab - 1)
    x, w, ids, teacher, more, up = case
    teacher_lse, loss, lse, z = _forward_ref(x, w, ids, teacher, more, 1.5, True)
    got = lm_head_distill(x, w, ids, teacher, 1.5, teacher_lse=teacher_lse)
    for what, a, b in (("loss", got[0], loss), ("lse", got[1], lse), ("logits", got[2], z)):
        _within(a, b, what)
    assert int(got[3].item()) == 0
    want = _grads_ref(x, w, ids, teacher, more, up, got[1], 1.5, True)
    grads = lm_head_distill_backward(x, w, ids, teacher, got[1], got[2], up, 1.5, teacher_lse=teacher_lse)
    _within(grads[0], want[0], "dx")
    _within(grads[1], want[1], "dw")


def test_one_certain_entry_is_the_cross_entropy(eng):
    """A teacher that is sure of one token: lm_head_loss."""
    import torch

    from pih_amd.linear import lm_head_distill, lm_head_distill_backward, lm_head_loss, lm_head_loss_backward

    x, w, ids, teacher, _, up = _case(11, 70, 3000, 256, 1)
    x, w, up = x.cuda(), w.cuda(), up.cuda()
    ids, teacher = ids.cuda(), teacher.cuda()
    loss, lse, z, _ = lm_head_distill(x, w, ids, teacher)
    want, want_lse, _ = lm_head_loss(x, w, ids[:, 0].contiguous())
    assert torch.equal(lse, want_lse)
    assert ((loss - want).abs() <= 1e-5 * (1 + want.abs())).all()
    dx, dw, _ = lm_head_distill_backward(x, w, ids, teacher, lse, z, up)
    ex, ew, _ = lm_head_loss_backward(x, w, ids[:, 0].contiguous(), lse, up)
    for a, b in ((dx, ex), (dw, ew)):
        assert ((a.double() - b.double()).norm() / b.double().norm()) < 2 * HALF_BF16


def test_gradient_against_differences(eng):
    """dx against the loss's own change along it; the loss is fp32."""
    import torch

    from pih_amd.linear import lm_head_distill, lm_head_distill_backward

    x, w, ids, teacher, _, up = (t.cuda() for t in _case(21, 40, 2000, 256, 16))
    _, lse, z, _ = lm_head_distill(x, w, ids, teacher, 2.0)
    grads = lm_head_distill_backward(x, w, ids, teacher, lse, z, up, 2.0)
    for i, (t, d) in enumerate(((x, grads[0]), (w, grads[1]))):
        step = d.double() / d.double().norm() * t.double().norm() * 0.02
        low, high = (t.double() - step).to(torch.bfloat16), (t.double() + step).to(torch.bfloat16)
        value = []
        for v in (low, high):
            loss = lm_head_distill(*((v, w) if i == 0 else (x, v)), ids, teacher, 2.0)[0]
            value.append((loss.double() * up.double()).sum())
        moved = ((high.double() - low.double()) * d.double()).sum()
        print(f"{i}: {(value[1] - value[0]).item():.5f} against {moved.item():.5f}", flush=True)
        assert abs((value[1] - value[0] - moved) / moved) < 0.05


def test_rows_without_a_teacher_reach_nothing(eng):
    """What rows whose entries are absent, or all of probability 0, hold (NaN,
    infinities) reaches no other row and not dw."""
    import torch

    from pih_amd.linear import lm_head_distill, lm_head_distill_backward

    inf, nan = float("inf"), float("nan")
    for rows, vocab, hidden, top_k in ((6, 300, 64, 4), (70, 1000, 256, 9), (9, 200, 72, 3)):
        x, w, ids, teacher, _, up = (t.cuda() for t in _case(rows, rows, vocab, hidden, top_k, empty=0.0))
        ids[1], teacher[1] = -1, nan  # nothing there, whatever the logits
        ids[2], teacher[2] = 5, -inf  # entries of probability 0
        clean = lm_head_distill(x, w, ids, teacher)
        assert int(clean[3].item()) == 0 and clean[0][1] == 0 and clean[0][2] == 0
        grads = lm_head_distill_backward(x, w, ids, teacher, clean[1], clean[2], up)
        x2, lse2, up2, z2 = x.clone(), clean[1].clone(), up.clone(), clean[2].clone()
        x2[1], x2[2], lse2[1], lse2[2], up2[1], up2[2], z2[1], z2[2] = nan, inf, nan, inf, inf, nan, inf, nan
        got = lm_head_distill(x2, w, ids, teacher)
        keep = torch.ones(rows, dtype=torch.bool, device="cuda")
        keep[1:3] = False
        for a, b in zip(clean[:3], got[:3]):
            assert torch.equal(a[keep], b[keep])
        assert got[0][1] == 0 and got[0][2] == 0 and int(got[3].item()) == 0
        dx, dw, _ = lm_head_distill_backward(x2, w, ids, teacher, lse2, z2, up2)
        assert torch.equal(dx, grads[0]) and torch.equal(dw, grads[1])
        assert torch.all(dx[1:3] == 0)


def test_error_bits(eng):
    import torch

    from pih_amd.linear import lm_head_distill, lm_head_distill_backward

    x, w, ids, teacher, _, up = (t.cuda() for t in _case(4, 6, 100, 64, 4, empty=0.0))
    ids[3] = torch.tensor([7, 100, 8, -1], dtype=torch.int32)
    clean = ids.clone()
    clean[3, 1] = -1
    want = lm_head_distill(x, w, clean, teacher)
    got = lm_head_distill(x, w, ids, teacher)
    assert int(want[3].item()) == 0 and int(got[3].item()) == 1
    for a, b in zip(want[:3], got[:3]):
        assert torch.equal(a, b)
    a = lm_head_distill_backward(x, w, clean, teacher, got[1], got[2], up)
    b = lm_head_distill_backward(x, w, ids, teacher, got[1], got[2], up)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and int(a[2].item()) == 0 and int(b[2].item()) == 1
    x[0] = float("nan")
    loss, _, _, flag = lm_head_distill(x, w, clean, teacher)
    assert int(flag.item()) == 4 and torch.isnan(loss[0]) and torch.equal(loss[1:], want[0][1:])
    # a probability above 0 where the head's logit is -infinity
    x, w, ids, teacher, _, _ = (t.cuda() for t in _case(4, 3, 100, 64, 2, empty=0.0))
    x, ids[:, 0] = x.abs() + 0.1, 9
    w[9] = float("-inf")
    loss, lse, _, flag = lm_head_distill(x, w, ids, teacher)
    assert int(flag.item()) == 4 and torch.all(loss == float("inf")) and torch.isfinite(lse).all()


def test_captured(eng):
    """Both passes in a graph, replayed between eager calls on new inputs."""
    import torch

    from pih_amd.device import engine_stream
    from pih_amd.linear import lm_head_distill, lm_head_distill_backward

    cases = [[t.cuda() for t in _case(s, 90, 3000, 256, 12)] for s in (1, 2, 3)]
    static = [t.clone() for t in cases[0]]
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")

    def step(x, w, ids, teacher, _, up):
        loss, lse, z, _ = lm_head_distill(x, w, ids, teacher, 1.5, flag=flag)
        return (loss, lse, z) + lm_head_distill_backward(x, w, ids, teacher, lse, z, up, 1.5, flag=flag)[:2]

    with engine_stream() as s:
        step(*static)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = step(*static)
        for case in cases + cases[:1]:
            for t, v in zip(static, case):
                t.copy_(v)
            graph.replay()
            want = step(*case)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert int(flag.item()) == 0


@pytest.mark.parametrize("rows,vocab,hidden,top_k", [(70, 600, 4096, 256), (190, 700, 2048, 200), (300, 300, 2048, 255),
                                                     (420, 5000, 2048, 100), (1000, 513, 1024, 128)])
def test_many_entries_in_a_tile(eng, rows, vocab, hidden, top_k):
    """Lists long enough for the tiles to write their logits, with many entries
    of a row in one tile, equal ones, none at all, and a certain id in all."""
    import torch

    from pih_amd.linear import lm_head_distill

    case = [t.cuda() for t in _case(rows, rows, vocab, hidden, top_k)]
    x, w, ids, teacher, more, _ = case
    ids[:, 3] = 255
    ids[1::4, 5:9] = vocab - 1
    ids[2] = 7
    _, loss, lse, z = _forward_ref(x, w, ids, teacher, more, 1.3, False)
    for n in (1 << 12, 1 << 16, 1 << 20):
        torch.full((n,), float("nan"), device="cuda")
    got = lm_head_distill(x, w, ids, teacher, 1.3)
    assert int(got[3].item()) == 0
    for what, a, b in (("logits", got[2], z), ("lse", got[1], lse), ("loss", got[0], loss)):
        _within(a, b, what)
    assert torch.all(got[2][ids < 0] == 0)


def test_rows_past_4_gib(eng):
    """2^20 rows, whose x has more than 2^32 bytes, that repeat 2047: so do the
    losses and dx, and the weights' gradient, of an upstream gradient that is zero
    before the last 2047 rows, is that of as many rows."""
    import torch

    from pih_amd.linear import lm_head_distill, lm_head_distill_backward

    rows, few, vocab, hidden, top_k = 1 << 20, 2047, 500, 4096, 8
    x, w, ids, teacher, more, up = _case(31, few, vocab, hidden, top_k, "cuda")
    times = -(-rows // few)
    long_x, long_ids, long_teacher = (t.repeat(times, 1)[-rows:].contiguous() for t in (x, ids, teacher))
    assert long_x.numel() * 2 > 1 << 32
    got = lm_head_distill(long_x, w, long_ids, long_teacher, 1.5)
    assert int(got[3].item()) == 0
    _, *want = _forward_ref(x, w, ids, teacher, more, 1.5, False)
    for at in (rows - few, rows - few * (times - 1)):
        for what, a, b in zip(("loss", "lse", "logits"), got, want):
            _within(a[at:at + few], b, what)
    long_up = torch.zeros(rows, device="cuda")
    long_up[-few:] = up
    dx, dw, _ = lm_head_distill_backward(long_x, w, long_ids, long_teacher, got[1], got[2], long_up, 1.5)
    want = _grads_ref(x, w, ids, teacher, more, up, got[1][-few:], 1.5, False)
    assert torch.all(dx[:-few] == 0)
    _within(dx[-few:], want[0], "dx")
    _within(dw, want[1], "dw")


def test_weights_past_4_gib(eng):
    """The largest vocabulary, whose weights and their gradient have more than
    2^32 bytes; entries at both ends of it."""
    import torch

    from pih_amd.linear import lm_head_distill, lm_head_distill_backward

    rows, vocab, hidden, top_k = 20, 1 << 20, 2112, 16
    x, w, ids, teacher, more, up = _case(32, rows, vocab, hidden, top_k, "cuda", std=1.0)
    assert w.numel() * 2 > 1 << 32
    ids[:, 2], ids[:, 7] = vocab - 1, 0
    got = lm_head_distill(x, w, ids, teacher)
    assert int(got[3].item()) == 0
    _, *want = _forward_ref(x, w, ids, teacher, more, 1.0, False)
    for what, a, b in zip(("loss", "lse", "logits"), got, want):
        _within(a, b, what)
    want = _grads_ref(x, w, ids, teacher, more, up, got[1], 1.0, False)
    dx, dw, _ = lm_head_distill_backward(x, w, ids, teacher, got[1], got[2], up)
    _within(dx, want[0], "dx")
    _within(dw, want[1], "dw")


@pytest.mark.parametrize("rows,vocab,hidden", [(1, 70, 64), (33, 1000, 128), (130, 2050, 192), (300, 5000, 256), (40, 777, 72),
                                               (16, 1024, 64)])
@pytest.mark.parametrize("loss", ["teacher", "target"])
def test_infinite_last_weight(eng, rows, vocab, hidden, loss):
    """The last vocabulary entry's weight holds an infinity at a column that is
    negative in every row: its logit is -inf, its probability 0.  Of the row whose
    teacher (or target) is sure of that entry, dx is -up times the weight there, an
    infinity; in the column 0 x inf of the other rows is NaN, and everything else is
    finite."""
    import torch

    from pih_amd.linear import (lm_head_distill, lm_head_distill_backward, lm_head_loss, lm_head_loss_backward)

    g = torch.Generator(device="cuda").manual_seed(rows + vocab)
    x = torch.randn(rows, hidden, generator=g, device="cuda").to(torch.bfloat16)
    w = (torch.randn(vocab, hidden, generator=g, device="cuda") * hidden ** -0.5).to(torch.bfloat16)
    up = torch.rand(rows, generator=g, device="cuda") + 0.5
    column, row = hidden // 3, rows // 2
    x[:, column] = -x[:, column].abs() - 0.1
    w[-1, column] = float("inf")
    target = torch.arange(rows, device="cuda", dtype=torch.int32) % (vocab - 1)
    target[row] = vocab - 1
    if loss == "target":
        _, lse, flag = lm_head_loss(x, w, target)
        dx, dw, _ = lm_head_loss_backward(x, w, target, lse, up)
    else:
        entries = target[:, None].contiguous(), torch.zeros(rows, 1, device="cuda")
        _, lse, z, flag = lm_head_distill(x, w, *entries)
        dx, dw, _ = lm_head_distill_backward(x, w, *entries, lse, z, up)
    torch.cuda.synchronize()
    assert int(flag.item()) == 4  # (that row's loss is infinite)
    assert torch.isfinite(lse).all() and torch.isfinite(dw).all()
    rest = torch.arange(hidden, device="cuda") != column
    assert torch.isfinite(dx[:, rest]).all()
    assert torch.isneginf(dx[row, column])
    others = torch.arange(rows, device="cuda") != row
    assert torch.isnan(dx[others, column]).all()


def test_lse_in_the_place_of_the_teachers(eng):
    """A row's place in teacher_lse is read before its lse (or loss) is written there."""
    import torch

    from pih_amd import abi, linear
    from pih_amd.device import error_flag, stream_handle

    rows, vocab, hidden, top_k = 70, 1000, 128, 5
    x, w, ids, teacher, _, _ = (t.cuda() for t in _case(8, rows, vocab, hidden, top_k))
    tail = torch.full((rows,), 4.0, device="cuda")
    want = linear.lm_head_distill(x, w, ids, teacher, 1.5, teacher_lse=tail)
    ws = linear._workspace(abi.WORKSPACE_LM_HEAD_DISTILL, rows, vocab, hidden, x.device)
    for place in (0, 1):
        out, flag = [torch.empty(rows, device="cuda") for _ in range(2)], error_flag()
        out[place] = tail.clone()
        z = torch.empty(rows, top_k, device="cuda")
        linear._launch("launch_lm_head_distill", "lm_head_distill",
                       *(t.data_ptr() for t in (x, w, ids, teacher, out[place], out[0], out[1], z, ws)), ws.numel(),
                       flag.data_ptr(), stream_handle(), rows, vocab, hidden, top_k, 1.5)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out + [z], want))


@pytest.mark.parametrize("rows,vocab,hidden,top_k", [(1100, 122859, 64, 128), (1021, 151936, 256, 8), (2053, 70001, 320, 3)])
def test_entries_at_every_tiles_border(eng, rows, vocab, hidden, top_k):
    """Ids on either side of every border of the tiles of 256 columns, those of the
    backward pass's pieces among them (2^26 elements of g or so in each, of the rows'
    135, 155 and 144 million), each in several rows."""
    import torch

    from pih_amd.linear import lm_head_distill, lm_head_distill_backward

    assert rows * vocab > (1 << 26) * 4 // 3  # more than a piece
    x, w, ids, teacher, more, up = _case(rows + 1, rows, vocab, hidden, top_k, "cuda", empty=0.0)
    edges = torch.arange(256, vocab, 256, device="cuda", dtype=torch.int32)
    edges = torch.cat((edges - 1, edges, torch.tensor([0, vocab - 1], device="cuda", dtype=torch.int32)))
    times = rows * top_k // edges.numel()
    assert times >= 2
    ids.view(-1)[:times * edges.numel()] = edges.repeat(times)
    teacher_lse, loss, lse, z = _forward_ref(x, w, ids, teacher, more, 1.5, True)
    got = lm_head_distill(x, w, ids, teacher, 1.5, teacher_lse=teacher_lse)
    for what, a, b in (("loss", got[0], loss), ("lse", got[1], lse), ("logits", got[2], z)):
        _within(a, b, what)
    assert int(got[3].item()) == 0
    want = _grads_ref(x, w, ids, teacher, more, up, got[1], 1.5, True)
    grads = lm_head_distill_backward(x, w, ids, teacher, got[1], got[2], up, 1.5, teacher_lse=teacher_lse)
    _within(grads[0], want[0], "dx")
    _within(grads[1], want[1], "dw")


def test_gradient_against_differences_along_the_formulas(eng):
    """The backward pass against the loss's own change along directions that do not
    come from it: the 64-bit gradient on a quarter of the tensor.  The losses are off
    by their bounds; what the change has beyond the first order is taken from the
    64-bit form, and the gradient's own error from its bound."""
    import torch

    from pih_amd.linear import lm_head_distill, lm_head_distill_backward

    case = [t.cuda() for t in _case(21, 40, 2000, 256, 16)]
    x, w, ids, teacher, more, up = case
    _, lse, z, _ = lm_head_distill(x, w, ids, teacher, 2.0)
    grads = lm_head_distill_backward(x, w, ids, teacher, lse, z, up, 2.0)
    refs = _grads_ref(x, w, ids, teacher, more, up, lse, 2.0, False)
    for i, (t, d) in enumerate(((x, grads[0]), (w, grads[1]))):
        ref, bound = refs[i]
        for rows in (0, 1):
            for columns in (0, 1):
                step = torch.zeros_like(ref)
                step[rows::2, columns::2] = ref[rows::2, columns::2]
                step *= t.double().norm() * 0.02 / step.norm()
                low, high = (t.double() - step).to(torch.bfloat16), (t.double() + step).to(torch.bfloat16)
                values, exact, noise = [], [], 0.0
                for v in (low, high):
                    xv, wv = (v, w) if i == 0 else (x, v)
                    values.append((lm_head_distill(xv, wv, ids, teacher, 2.0)[0].double() * up.double()).sum())
                    loss, eloss = _forward_ref(xv, wv, ids, teacher, more, 2.0, False)[1]
                    exact.append((loss * up.double()).sum())
                    noise = noise + (eloss * up.double().abs()).sum()
                moved = high.double() - low.double()
                first, change = (moved * d.double()).sum(), values[1] - values[0]
                beyond = (exact[1] - exact[0] - (moved * ref).sum()).abs()
                tolerance = noise + beyond + (moved.abs() * bound).sum()
                print(f"{i}.{rows}{columns}: {change.item():.6f} against {first.item():.6f}, tolerance "
                      f"{tolerance.item():.6f}", flush=True)
                assert tolerance < 0.2 * first.abs()
                assert (change - first).abs() <= tolerance


@pytest.mark.parametrize("rows,hidden", [(40, 64), (40, 72), (300, 128)])
@pytest.mark.parametrize("temperature", [4.25e-39, 1e-30, 1e-9])
def test_low_temperatures(eng, rows, hidden, temperature):
    """The head's and the teacher's softmax are their largest logits alone, which
    agree: no loss.  Of the gradients' two sides, each at most the temperature, the
    head's is as far off as its fp32 log-sum-exp over it, but never above that."""
    import torch

    from pih_amd.linear import lm_head_distill, lm_head_distill_backward

    vocab = 300
    g = torch.Generator(device="cuda").manual_seed(3)
    x = (torch.randn(rows, hidden, generator=g, device="cuda") * 0.02).to(torch.bfloat16)
    w = (torch.randn(vocab, hidden, generator=g, device="cuda") * 0.02).to(torch.bfloat16)
    best, second = (x.double() @ w.double().T).topk(2).indices.unbind(1)
    ids = torch.stack((best, second), 1).to(torch.int32)
    teacher = torch.tensor([0.25, 0.125], device="cuda").repeat(rows, 1)
    loss, lse, z, flag = lm_head_distill(x, w, ids, teacher, temperature)
    assert int(flag.item()) == 0 and torch.isfinite(lse).all()
    # (a row's loss is T^2 times a difference of numbers like lse)
    assert torch.all(loss.abs().double() <= temperature ** 2 * lse.abs().double() * 4 * U)
    dx, dw, flag = lm_head_distill_backward(x, w, ids, teacher, lse, z, torch.ones(rows, device="cuda"), temperature)
    assert int(flag.item()) == 0 and torch.isfinite(dx).all() and torch.isfinite(dw).all()
    # (two sides, rounded to bf16 twice)
    most = 2 * temperature * (1 + 4 * HALF_BF16)
    assert torch.all(dx.double().abs() <= most * w.double().abs().max())
    assert torch.all(dw.double().abs() <= most * x.double().abs().sum(0))


@pytest.mark.parametrize("rows,vocab,hidden,top_k", [(33, 65, 128, 7), (17, 64, 200, 65), (130, 2050, 192, 32),
                                                     (300, 5000, 128, 64), (515, 300, 64, 4)])
@pytest.mark.parametrize("temperature,tail", [(9e-4, False), (5e-4, True)])
def test_backward_below_a_thousandth(eng, rows, vocab, hidden, top_k, temperature, tail):
    import torch

    from pih_amd.linear import lm_head_distill_backward

    case = _case(rows * 3 + vocab, rows, vocab, hidden, top_k, std=0.02)
    # (the teacher's logits as far apart over the temperature as the head's)
    case = case[:3] + (case[3] * 0.01, case[4] * 0.01) + case[5:]
    teacher_lse, _, lse, z = _forward_ref(*case[:5], temperature, tail)
    lse, z = lse[0].float(), z[0].float()
    dx, dw = _grads_ref(*case[:5], case[5], lse, temperature, tail)
    x, w, ids, teacher = (t.cuda() for t in case[:4])
    gx, gw, flag = lm_head_distill_backward(x, w, ids, teacher, lse.cuda(), z.cuda(), case[5].cuda(), temperature,
                                            teacher_lse=None if teacher_lse is None else teacher_lse.cuda())
    torch.cuda.synchronize()
    assert int(flag.item()) == 0
    _within(gx, dx, "dx")
    _within(gw, dw, "dw")
