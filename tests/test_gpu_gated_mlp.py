"""The gated feed-forward block (launch_gated_mlp and its backward) against 64
bits, element by element.

Bounds.  A sum of K products of bf16 values in fp32 is off by (K + 8) 2^-23 of
the sum of their magnitudes.  The logistic function s of g, by a 2^x and a
reciprocal of one unit each at an argument rounded to fp32, is off by (|g| + 8)
2^-22 of itself at most, and so are silu(g) = g s and, of s + |silu|, silu'(g)
= s + silu (1 - s).  |silu'| <= 1.1, |silu''| <= 0.5.  A rounding to bf16 costs
2^-8 of the value, h, dgate and dup have one each before the products behind
them.  Numbers below 2^-126 may become 0."""
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -23
HALF_BF16 = 2.0 ** -8
TINY = 1e-36


@pytest.fixture(scope="module")
def eng():
    import torch

    from pih_amd.device import engine_stream

    with engine_stream() as s:
        yield s
        torch.cuda.synchronize()


def _poison():
    """Freed memory that later allocations get, full of NaN."""
    import torch

    for n in (1 << 12, 1 << 16, 1 << 20, 1 << 24):
        torch.full((n,), float("nan"), device="cuda")


def _case(seed, rows, hidden, inter, device="cpu", spread=2.0):
    import torch

    g = torch.Generator(device=device).manual_seed(seed)
    n = lambda s, *shape: (torch.randn(*shape, generator=g, device=device) * s).to(torch.bfloat16)  # noqa: E731
    x, wg, wu = n(1.0, rows, hidden), n(spread * hidden ** -0.5, inter, hidden), n(spread * hidden ** -0.5, inter, hidden)
    return x, wg, wu, n(inter ** -0.5, hidden, inter), n(0.1, rows, hidden)


def _clamped(gate, up, limit):
    import torch

    if limit <= 0:
        return gate, up
    return torch.clamp(gate, max=limit), torch.clamp(up, -limit, limit)


def _forward_ref(x, wg, wu, wd, limit):
    """(value, bound) of y, gate and up."""
    import torch

    x, wg, wu, wd = (t.double() for t in (x, wg, wu, wd))
    k = (x.shape[1] + 8) * U
    gate, up = x @ wg.T, x @ wu.T
    eg, eu = x.abs() @ wg.abs().T * k, x.abs() @ wu.abs().T * k
    g, u = _clamped(gate, up, limit)
    silu = g * torch.sigmoid(g)
    h = silu * u
    eh = 1.1 * eg * (u.abs() + eu) + silu.abs() * eu
    eh += (h.abs() + eh) * ((g.abs() + 10) * 2.0 ** -22 + HALF_BF16) + TINY
    y = h @ wd.T
    ey = eh @ wd.abs().T + (h.abs() + eh) @ wd.abs().T * (h.shape[1] + 8) * U
    half = lambda v, e: e + (v.abs() + e) * HALF_BF16 + TINY  # noqa: E731
    return (y, half(y, ey)), (gate, half(gate, eg)), (up, half(up, eu))


def _backward_ref(dy, x, wg, wu, wd, gate, up, limit):
    import torch

    dy, x, wg, wu, wd, gate, up = (t.double() for t in (dy, x, wg, wu, wd, gate, up))
    rows, hidden, inter = x.shape[0], x.shape[1], wg.shape[0]
    g, u = _clamped(gate, up, limit)
    s = torch.sigmoid(g)
    silu = g * s
    slope = s + silu * (1 - s)
    dh = dy @ wd
    ed = dy.abs() @ wd.abs() * (hidden + 8) * U
    eact = (g.abs() + 12) * 2.0 ** -22
    h, du, dg = silu * u, dh * silu, dh * u * slope
    eh = h.abs() * (eact + HALF_BF16) + TINY
    edu = ed * silu.abs()
    edu += (du.abs() + edu) * (eact + HALF_BF16) + TINY
    edg = ed * (u * slope).abs() + (dh.abs() + ed) * u.abs() * (s + silu.abs()) * eact
    edg += (dg.abs() + edg) * (HALF_BF16 + 4 * U) + TINY
    if limit > 0:
        for d, e, beyond in ((dg, edg, gate > limit), (du, edu, up.abs() > limit)):
            d[beyond] = 0
            e[beyond] = 0

    def product(a, ea, b, n):
        v = a @ b
        e = ea @ b.abs() + (a.abs() + ea) @ b.abs() * (n + 8) * U
        return v, e

    (p, ep), (q, eq) = product(dg, edg, wg, 2 * inter), product(du, edu, wu, 2 * inter)
    out = [(p + q, ep + eq), product(dg.T, edg.T, x, rows), product(du.T, edu.T, x, rows)]
    v, e = product(h.T, eh.T, dy, rows)
    out.append((v.T, e.T))
    return [(v, e + (v.abs() + e) * HALF_BF16 + TINY) for v, e in out]


def _within(got, want, what):
    value, bound = want
    assert got.shape == value.shape, what
    worst = ((got.double().to(value.device) - value).abs() / bound).max().item()
    print(f"{what}: worst {worst:.3f} of the bound", flush=True)
    assert worst <= 1.0, (what, worst)


# odd, below, at and above the tiles; sizes that are no multiple of 64
SIZES = [(1, 8, 8), (1, 64, 64), (2, 72, 136), (3, 64, 200), (5, 256, 128), (16, 128, 64), (17, 200, 264), (33, 512, 320),
         (63, 256, 512), (64, 64, 1024), (65, 1024, 64), (100, 192, 448), (129, 256, 1088), (130, 1000, 136),
         (257, 320, 640), (300, 128, 2048), (515, 640, 128), (700, 1088, 704)]


@pytest.mark.parametrize("rows,hidden,inter", SIZES)
@pytest.mark.parametrize("limit", [0.0, 1.5])
def test_forward(eng, rows, hidden, inter, limit):
    import torch

    from pih_amd.linear import gated_mlp

    x, wg, wu, wd, _ = _case(rows * 31 + hidden + inter, rows, hidden, inter)
    want = _forward_ref(x, wg, wu, wd, limit)
    args = [t.cuda() for t in (x, wg, wu, wd)]
    _poison()
    got = gated_mlp(*args, limit=limit, keep=True)
    alone = gated_mlp(*args, limit=limit)
    torch.cuda.synchronize()
    for what, g, w in zip(("y", "gate", "up"), got, want):
        _within(g, w, what)
    assert torch.equal(alone, got[0])


@pytest.mark.parametrize("rows,hidden,inter", SIZES)
@pytest.mark.parametrize("limit", [0.0, 1.5])
def test_backward(eng, rows, hidden, inter, limit):
    import torch

    from pih_amd.linear import gated_mlp_backward

    x, wg, wu, wd, dy = _case(rows * 29 + hidden + inter, rows, hidden, inter)
    gate, up = ((x.double() @ w.double().T).to(torch.bfloat16) for w in (wg, wu))
    gate.view(-1)[::7] = 1.5  # on the clamp's border, where the gradient still passes
    up.view(-1)[::11] = -1.5
    want = _backward_ref(dy, x, wg, wu, wd, gate, up, limit)
    args = [t.cuda() for t in (dy, x, wg, wu, wd, gate, up)]
    _poison()
    got = gated_mlp_backward(*args, limit=limit)
    again = gated_mlp_backward(*args, limit=limit)
    only = gated_mlp_backward(*args, limit=limit, weight_gradients=False)
    torch.cuda.synchronize()
    for what, g, w in zip(("dx", "dw_gate", "dw_up", "dw_down"), got, want):
        _within(g, w, what)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    assert torch.equal(only[0], got[0]) and only[1:] == (None, None, None)


LARGE = [(1, 4096, 2048), (7, 7168, 2048), (16, 4096, 12288), (40, 4096, 12288), (57, 4096, 2048), (128, 4096, 12288),
         (200, 7168, 2048), (509, 4096, 12288), (1021, 4096, 2048), (1030, 4096, 12288), (2100, 4096, 4096)]


@pytest.mark.parametrize("rows,hidden,inter", LARGE)
def test_large(eng, rows, hidden, inter):
    """The sizes of real blocks, 64 bits on the GPU."""
    import torch

    from pih_amd.linear import gated_mlp, gated_mlp_backward

    x, wg, wu, wd, dy = _case(rows + hidden, rows, hidden, inter, "cuda")
    _poison()
    y, gate, up = gated_mlp(x, wg, wu, wd, keep=True)
    alone = gated_mlp(x, wg, wu, wd)
    for what, g, w in zip(("y", "gate", "up"), (y, gate, up), _forward_ref(x, wg, wu, wd, 0.0)):
        _within(g, w, what)
    assert torch.equal(alone, y)
    want = _backward_ref(dy, x, wg, wu, wd, gate, up, 0.0)
    for what, g, w in zip(("dx", "dw_gate", "dw_up", "dw_down"), gated_mlp_backward(dy, x, wg, wu, wd, gate, up), want):
        _within(g, w, what)


def test_gradient_against_differences(eng):
    """The backward pass against the forward one's own change along a random
    direction.  y is bf16, so the step is long (0.5 of x's size) and central; the
    third derivative along it leaves less than a tenth of what is compared."""
    import torch

    from pih_amd.linear import gated_mlp, gated_mlp_backward

    x, wg, wu, wd, dy = (t.cuda() for t in _case(5, 64, 256, 512, spread=1.0))
    _, gate, up = gated_mlp(x, wg, wu, wd, keep=True)
    grads = gated_mlp_backward(dy, x, wg, wu, wd, gate, up)
    g = torch.Generator(device="cuda").manual_seed(9)
    for i, (t, d) in enumerate(zip((x, wg, wu, wd), grads)):
        # along the gradient's own direction, so that the change is far above
        # y's roundings
        step = (d.double() / d.double().norm() * t.double().norm() * 0.05)
        low, high = (t.double() - step).to(torch.bfloat16), (t.double() + step).to(torch.bfloat16)
        args = [x, wg, wu, wd]
        value = []
        for v in (low, high):
            args[i] = v
            value.append((gated_mlp(*args).double() * dy.double()).sum())
        moved = ((high.double() - low.double()) * d.double()).sum()
        change = value[1] - value[0]
        print(f"{i}: {change.item():.6f} against {moved.item():.6f}", flush=True)
        assert abs((change - moved) / moved) < 0.1
    del g


def test_a_row_keeps_to_itself(eng):
    """NaN and infinities of one row reach no other row of y, gate, up and dx."""
    import torch

    from pih_amd.linear import gated_mlp, gated_mlp_backward

    for rows, hidden, inter in ((3, 64, 128), (70, 256, 512), (300, 512, 256)):
        x, wg, wu, wd, dy = (t.cuda() for t in _case(rows, rows, hidden, inter))
        clean = gated_mlp(x, wg, wu, wd, keep=True)
        grad = gated_mlp_backward(dy, x, wg, wu, wd, *clean[1:])[0]
        bad = rows // 2
        x2, dy2 = x.clone(), dy.clone()
        x2[bad, ::2], x2[bad, 1::2] = float("nan"), float("inf")
        dy2[bad] = float("inf")
        got = gated_mlp(x2, wg, wu, wd, keep=True)
        dx = gated_mlp_backward(dy2, x2, wg, wu, wd, *got[1:])[0]
        keep = torch.arange(rows, device="cuda") != bad
        for a, b in zip(clean + (grad,), got + (dx,)):
            assert torch.equal(a[keep], b[keep])
            assert not torch.isfinite(b[bad]).any()


def test_extreme_gates(eng):
    """Gates far out on both sides: silu of them is 0 or the gate itself, and
    their gradients 0 or those of a product."""
    import torch

    from pih_amd.linear import gated_mlp_backward

    rows, hidden, inter = 4, 64, 64
    x, wg, wu, wd, dy = _case(3, rows, hidden, inter)
    gate = torch.zeros(rows, inter, dtype=torch.bfloat16)
    gate[0], gate[1], gate[2], gate[3] = -1000.0, 1000.0, -3e38, 3e38
    up = torch.ones(rows, inter, dtype=torch.bfloat16)
    got = gated_mlp_backward(*(t.cuda() for t in (dy, x, wg, wu, wd, gate, up)))
    dh = dy.double() @ wd.double()
    assert torch.isfinite(got[0].cpu()[:2]).all()
    assert torch.all(got[0].cpu()[0] == 0) and torch.all(got[0].cpu()[2] == 0)
    # row 1: dgate = dh, dup = 1000 dh
    want = dh[1] @ wg.double() + 1000 * dh[1] @ wu.double()
    assert ((got[0].cpu().double()[1] - want).abs() <= 0.02 * want.abs().max()).all()


def test_out_is_a_part_of_a_larger_tensor(eng):
    import torch

    from pih_amd.linear import gated_mlp

    x, wg, wu, wd, _ = (t.cuda() for t in _case(8, 37, 128, 256))
    whole = torch.full((50, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    y = gated_mlp(x, wg, wu, wd, out=whole[5:42])
    assert y.data_ptr() == whole[5:].data_ptr() and torch.equal(y, gated_mlp(x, wg, wu, wd))
    assert torch.all(whole[:5] == 7) and torch.all(whole[42:] == 7)
    # the halves of a fused gate/up weight
    fused = torch.cat((wg, wu))
    assert torch.equal(y, gated_mlp(x, fused[:256], fused[256:], wd))


@pytest.mark.parametrize("rows,hidden,inter", [(1, 256, 512), (40, 256, 512), (300, 320, 192)])
def test_captured(eng, rows, hidden, inter):
    """Both passes in a graph, replayed between eager calls on new inputs."""
    import torch

    from pih_amd.device import engine_stream
    from pih_amd.linear import gated_mlp, gated_mlp_backward

    cases = [[t.cuda() for t in _case(s, rows, hidden, inter)] for s in (1, 2, 3)]
    static = [t.clone() for t in cases[0]]

    def step(x, wg, wu, wd, dy):
        kept = gated_mlp(x, wg, wu, wd, limit=2.0, keep=True)
        return kept + gated_mlp_backward(dy, x, wg, wu, wd, *kept[1:], limit=2.0)

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


@pytest.mark.parametrize("rows,hidden,inter", [(40, 256, 512), (300, 320, 192), (7, 72, 136)])
def test_any_part_of_the_gradients(eng, rows, hidden, inter):
    """The entry's results that are left out (null) change nothing of the others."""
    import torch

    from pih_amd import abi, linear
    from pih_amd.device import stream_handle

    x, wg, wu, wd, dy = (t.cuda() for t in _case(12, rows, hidden, inter))
    _, gate, up = linear.gated_mlp(x, wg, wu, wd, keep=True)
    want = linear.gated_mlp_backward(dy, x, wg, wu, wd, gate, up)
    ws = linear._workspace(abi.WORKSPACE_GATED_MLP_BACKWARD, rows, inter, hidden, x.device)
    for parts in range(1, 16):
        got = [torch.full_like(w, 7.0) for w in want]
        linear._launch("launch_gated_mlp_backward", "gated_mlp_backward",
                       *(t.data_ptr() for t in (dy, x, wg, wu, wd, gate, up)),
                       *(t.data_ptr() if parts >> i & 1 else 0 for i, t in enumerate(got)), ws.data_ptr(), ws.numel(),
                       stream_handle(), rows, hidden, inter, 0.0)
        for i, (g, w) in enumerate(zip(got, want)):
            assert torch.equal(g, w if parts >> i & 1 else torch.full_like(w, 7.0)), (parts, i)


@pytest.mark.parametrize("hidden,inter", [(4096, 128), (128, 4096)])
def test_rows_past_4_gib(eng, hidden, inter):
    """2^20 rows, whose x and y or gate, up and h have more than 2^32 bytes.  All
    rows repeat the first 8191: y, gate, up and dx with them, and the weights'
    gradients, of an upstream gradient that is zero before the last 8191 rows, are
    those of as many rows."""
    import torch

    from pih_amd.linear import gated_mlp, gated_mlp_backward

    rows, few = 1 << 20, 8191
    x, wg, wu, wd, dy = _case(21, few, hidden, inter, "cuda")
    times = -(-rows // few)
    # (the last rows are the first ones, in order)
    long_x = x.repeat(times, 1)[-rows:].contiguous()
    assert long_x.numel() * 2 > 1 << 32 or rows * inter * 2 > 1 << 32
    y, gate, up = gated_mlp(long_x, wg, wu, wd, keep=True)
    for what, t, w in zip(("y", "gate", "up"), (y, gate, up), _forward_ref(x, wg, wu, wd, 0.0)):
        for at in (rows - few, rows - few * (times - 1)):
            _within(t[at:at + few], w, what)
    del y
    long_dy = torch.zeros_like(long_x)
    long_dy[-few:] = dy
    got = gated_mlp_backward(long_dy, long_x, wg, wu, wd, gate, up)
    want = _backward_ref(dy, x, wg, wu, wd, gate[-few:], up[-few:], 0.0)
    assert torch.all(got[0][:-few] == 0)
    # (their sums run over all rows, most of them zeros)
    for what, g, w in zip(("dx", "dw_gate", "dw_up", "dw_down"), (got[0][-few:],) + got[1:], want):
        _within(g, w, what)


def _same_nonfinite(got, want, what):
    """NaN and infinities where the 64-bit form has them, and nowhere else."""
    import torch

    for name, mask in (("NaN", torch.isnan), ("inf", torch.isposinf), ("-inf", torch.isneginf)):
        assert torch.equal(mask(got).cpu(), mask(want)), (what, name)


@pytest.mark.parametrize("rows,hidden,inter", [(1, 64, 64), (3, 64, 128), (70, 256, 512), (129, 320, 192), (300, 512, 256),
                                               (509, 1024, 512), (64, 64, 128), (5, 72, 136)])
@pytest.mark.parametrize("where", ["dy", "x"])
def test_infinity_in_the_last_row_of_the_weights_gradients(eng, rows, hidden, inter, where):
    """An infinite element of the last row: what the sums over the rows make of it is
    theirs alone, also where the rows are no multiple of the products' steps."""
    import torch

    from pih_amd.linear import gated_mlp_backward

    x, wg, wu, wd, dy = _case(rows + inter, rows, hidden, inter)
    gate, up = ((x.double() @ w.double().T).to(torch.bfloat16) for w in (wg, wu))
    (dy if where == "dy" else x)[-1, hidden // 3] = float("inf")
    want = _backward_ref(dy, x, wg, wu, wd, gate, up, 0.0)
    got = gated_mlp_backward(*(t.cuda() for t in (dy, x, wg, wu, wd, gate, up)))
    torch.cuda.synchronize()
    for what, g, (w, _) in zip(("dx", "dw_gate", "dw_up", "dw_down"), got, want):
        _same_nonfinite(g, w, what)
    assert torch.isinf(want[3][0] if where == "dy" else want[1][0]).any()


@pytest.mark.parametrize("rows,hidden,inter", [(1, 64, 16448), (8, 512, 2112), (24, 2048, 5696), (33, 1024, 4160), (64, 64, 16448),
                                               (65, 256, 4160), (130, 1024, 4160), (320, 512, 2112)])
def test_intermediate_sizes_off_128(eng, rows, hidden, inter):
    """Half a step of 128 behind the last whole one, on the kernels that take it."""
    import torch

    from pih_amd.linear import gated_mlp

    x, wg, wu, wd, _ = _case(rows + inter, rows, hidden, inter, "cuda")
    _poison()
    got = gated_mlp(x, wg, wu, wd, keep=True)
    alone = gated_mlp(x, wg, wu, wd)
    for what, g, w in zip(("y", "gate", "up"), got, _forward_ref(x, wg, wu, wd, 0.0)):
        _within(g, w, what)
    assert torch.equal(alone, got[0])


def test_gradient_against_differences_along_the_formulas(eng):
    """The backward pass against the forward one's own change along directions
    that do not come from it: the 64-bit gradient on a quarter of the tensor, for
    x also each of its two terms.  A value v = sum of y dy is off by y's and h's
    roundings, independent and at most 2^-8 of each element: six standard
    deviations of the two values' difference are 6 sqrt(2 / 3) 2^-8 sqrt(|y dy|^2 +
    |h dh|^2).  What the change has beyond the first order is taken from the 64-bit
    form, and the gradient's own error from its bound."""
    import torch

    from pih_amd.linear import gated_mlp, gated_mlp_backward

    x, wg, wu, wd, dy = (t.cuda() for t in _case(5, 64, 256, 512, spread=1.0))
    y, gate, up = gated_mlp(x, wg, wu, wd, keep=True)
    grads = gated_mlp_backward(dy, x, wg, wu, wd, gate, up)
    refs = _backward_ref(dy, x, wg, wu, wd, gate, up, 0.0)

    def value64(args):
        return (_forward_ref(*args, 0.0)[0][0] * dy.double()).sum()

    g, u, dh = gate.double(), up.double(), dy.double() @ wd.double()
    s = torch.sigmoid(g)
    h = g * s * u
    noise = 6 * (2 / 3) ** 0.5 * HALF_BF16 * ((y.double() * dy.double()).norm() ** 2 + (h * dh).norm() ** 2).sqrt()
    terms = ((dh * u * (s + g * s * (1 - s))) @ wg.double(), (dh * g * s) @ wu.double())
    for i, (t, d) in enumerate(zip((x, wg, wu, wd), grads)):
        ref, bound = refs[i]
        quarters = []
        for rows in (0, 1):
            for columns in (0, 1):
                part = torch.zeros_like(ref)
                part[rows::2, columns::2] = ref[rows::2, columns::2]
                quarters.append(part)
        for j, direction in enumerate(quarters + (list(terms) if i == 0 else [])):
            step = direction / direction.norm() * t.double().norm() * 0.05
            values, exact = [], []
            low, high = (t.double() - step).to(torch.bfloat16), (t.double() + step).to(torch.bfloat16)
            for v in (low, high):
                args = [x, wg, wu, wd]
                args[i] = v
                values.append((gated_mlp(*args).double() * dy.double()).sum())
                exact.append(value64(args))
            moved = high.double() - low.double()
            first, change = (moved * d.double()).sum(), values[1] - values[0]
            beyond = (exact[1] - exact[0] - (moved * ref).sum()).abs()
            tolerance = noise + beyond + (moved.abs() * bound).sum()
            print(f"{i}.{j}: {change.item():.6f} against {first.item():.6f}, tolerance {tolerance.item():.6f}", flush=True)
            assert tolerance < 0.2 * first.abs()
            assert (change - first).abs() <= tolerance
