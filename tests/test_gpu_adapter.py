"""Low-rank adapters over segments of rows (launch_adapter_gemm,
launch_adapter_backward) against 64 bits, element by element.

Bounds.  An fp32 sum of n products in any order is off by at most n 2^-23 of
the sum of their magnitudes (half a step per addition, twice over for an
accumulator that truncates).  The product between the two stages enters the
second as two bf16 values, off by 2^-16 of it.  A bf16 output is off by half a
step, 2^-8 of it, and the sum with base by 2^-23."""
import numpy as np
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


def _case(seed, lengths, adapters, rank, n, k, stacks, first=0, tail=0, scale=True):
    import torch

    g = torch.Generator().manual_seed(seed)
    rows = first + sum(lengths) + tail
    bf = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(torch.bfloat16)  # noqa: E731
    offsets = np.concatenate(([first], first + np.cumsum(lengths))).astype(np.int32)
    return dict(x=bf(rows, k), dy=bf(rows, n), a=bf(stacks, rank, k, std=k ** -0.5), b=bf(stacks, n, rank, std=0.1),
                scale=0.5 + torch.rand(stacks, generator=g) if scale else None, base=bf(rows, n), dbase=bf(rows, k),
                offsets=torch.from_numpy(offsets), adapters=torch.tensor(adapters, dtype=torch.int32))


def _dev(c):
    return {k: None if v is None else v.cuda() for k, v in c.items()}


def _segments(c):
    off, ad = c["offsets"].tolist(), c["adapters"].tolist()
    return [(off[i], off[i + 1], ad[i] & 0xFFFFFFFF) for i in range(len(ad))]


def _scale(c, a):
    return 1.0 if c["scale"] is None else float(c["scale"][a])


def _forward_ref(c, base):
    """(value, bound, written) of the output in 64 bits."""
    d = {k: None if v is None else v.double() for k, v in c.items()}
    rows, n, k, rank = c["x"].shape[0], c["b"].shape[1], c["a"].shape[2], c["a"].shape[1]
    out = d["base"].clone() if base else 0 * d["base"]
    err = 0 * out
    written = np.zeros(rows, bool)
    for lo, hi, a in _segments(c):
        if a == abi.NO_ADAPTER:
            written[lo:hi] = True
            continue
        if a >= c["a"].shape[0]:
            continue
        written[lo:hi] = True
        s, x, A, B = _scale(c, a), d["x"][lo:hi], d["a"][a], d["b"][a]
        h = x @ A.T
        eh = x.abs() @ A.abs().T * (k + 8) * U + h.abs() * (2.0 ** -16 + 2 * U)
        out[lo:hi] += s * (h @ B.T)
        err[lo:hi] += s * (eh @ B.abs().T + (h.abs() + eh) @ B.abs().T * (2 * rank + 2) * U)
    err += (out.abs() + err) * U
    return out, err + (out.abs() + err) * HALF_BF16 + 1e-37, written


def _backward_ref(c, base):
    import torch

    d = {k: None if v is None else v.double() for k, v in c.items()}
    n, k, rank = c["b"].shape[1], c["a"].shape[2], c["a"].shape[1]
    dx = d["dbase"].clone() if base else 0 * d["dbase"]
    ex = 0 * dx
    da, db = torch.zeros_like(d["a"]), torch.zeros_like(d["b"])
    ea, eb = 0 * da, 0 * db
    total = torch.zeros(c["a"].shape[0])
    for lo, hi, a in _segments(c):
        if a < c["a"].shape[0]:
            total[a] += hi - lo
    for lo, hi, a in _segments(c):
        if a >= c["a"].shape[0] or lo == hi:
            continue
        s, x, dy, A, B = _scale(c, a), d["x"][lo:hi], d["dy"][lo:hi], d["a"][a], d["b"][a]
        h, dh = s * (x @ A.T), s * (dy @ B)
        split = 2.0 ** -16 + 3 * U
        eh = s * (x.abs() @ A.abs().T) * (k + 8) * U + h.abs() * split
        edh = s * (dy.abs() @ B.abs()) * (n + 8) * U + dh.abs() * split
        dx[lo:hi] += dh @ A
        ex[lo:hi] += edh @ A.abs() + (dh.abs() + edh) @ A.abs() * (2 * rank + 2) * U
        t = (2 * float(total[a]) + 64) * U
        da[a] += dh.T @ x
        ea[a] += edh.T @ x.abs() + (dh.abs() + edh).T @ x.abs() * t
        db[a] += dy.T @ h
        eb[a] += dy.abs().T @ eh + dy.abs().T @ (h.abs() + eh) * t
    ex += (dx.abs() + ex) * U
    return (dx, ex + (dx.abs() + ex) * HALF_BF16 + 1e-37), (da, ea + 1e-37), (db, eb + 1e-37)


def _within(got, ref, bound, what):
    off = (got.double().cpu() - ref).abs()
    worst = (off / bound).max().item()
    print(f"{what}: worst {worst:.3f} of the bound", flush=True)
    assert worst <= 1.0, (what, worst)


# lengths of the segments, their adapters, rank, n, k, stacks, rows before and behind
CASES = [
    ([1], [0], 16, 64, 128, 1, 0, 0),  # a single token
    ([1] * 7, [2, 0, 1, 2, -1, 0, 2], 8, 40, 72, 3, 0, 0),  # a decode batch; sizes that are no multiple of 16 or 32
    ([1] * 70, [i % 5 for i in range(70)], 32, 136, 264, 5, 0, 0),  # more segments than a wave has lanes
    ([5, 0, 33, 16, 17], [1, 0, 1, -1, 0], 24, 200, 520, 2, 0, 3),  # an empty one, one without adapter, shared ones
    ([100, 31], [0, 1], 64, 512, 1000, 2, 5, 40),  # rows before and behind the segments
    ([129], [1], 128, 328, 648, 2, 0, 0),  # the largest rank, an adapter without rows
    ([15, 2, 64], [3, 3, 3], 48, 72, 4096, 4, 1, 0),  # long sums, one adapter throughout
    ([300, 1, 210], [0, 1, 0], 16, 4096, 96, 2, 0, 1),  # wide output
    ([700], [0], 16, 264, 392, 1, 0, 0),  # rows enough to split the gradients
]


@pytest.mark.parametrize("base", [True, False])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_forward(eng, case, base):
    import torch

    from pih_amd.linear import adapter_gemm

    c = _case(100 + case, *CASES[case], scale=case != 1)
    ref, bound, written = _forward_ref(c, base)
    d = _dev(c)
    out = torch.full_like(d["base"], 7.0)
    got, flag = adapter_gemm(d["x"], d["a"], d["b"], d["scale"], d["offsets"], d["adapters"],
                             base=d["base"] if base else None, out=out)
    torch.cuda.synchronize()
    assert int(flag.item()) == 0
    w = torch.from_numpy(written)
    assert torch.all(got.cpu()[~w] == 7.0)  # rows outside every segment
    _within(got[w.cuda()], ref[w], bound[w], f"case {case}")


@pytest.mark.parametrize("base", [True, False])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_backward(eng, case, base):
    import torch

    from pih_amd.linear import adapter_backward

    c = _case(200 + case, *CASES[case], scale=case != 1)
    _, _, written = _forward_ref(c, True)
    (dx, ex), (da, ea), (db, eb) = _backward_ref(c, base)
    d = _dev(c)
    out = torch.full_like(d["dbase"], 7.0)
    args = (d["dy"], d["x"], d["a"], d["b"], d["scale"], d["offsets"], d["adapters"])
    gx, ga, gb, flag = adapter_backward(*args, base=d["dbase"] if base else None, out=out)
    again = adapter_backward(*args, base=d["dbase"] if base else None, out=torch.full_like(out, 7.0))
    torch.cuda.synchronize()
    assert int(flag.item()) == 0
    w = torch.from_numpy(written)
    assert torch.all(gx.cpu()[~w] == 7.0)
    _within(gx[w.cuda()], dx[w], ex[w], f"dx {case}")
    _within(ga, da, ea, f"da {case}")
    _within(gb, db, eb, f"db {case}")
    for p, q in zip((gx, ga, gb), again):  # a fixed order of every sum
        assert torch.equal(p, q)


def test_gradients_are_the_differences(eng):
    """da, db and dx against central differences of the 64-bit forward."""
    import torch

    from pih_amd.linear import adapter_backward

    c = _case(7, [9, 4], [1, 0], 8, 24, 40, 2)
    d = _dev(c)
    dx, da, db, _ = adapter_backward(d["dy"], d["x"], d["a"], d["b"], d["scale"], d["offsets"], d["adapters"])
    torch.cuda.synchronize()

    def value(name, at, step):
        e = {k: v.double() for k, v in c.items()}
        e[name][at] += step
        y = 0.0
        for lo, hi, a in _segments(c):
            o = float(c["scale"][a]) * (e["x"][lo:hi] @ e["a"][a].T) @ e["b"][a].T
            y += float((o * e["dy"][lo:hi]).sum())
        return y

    # the function is a polynomial of degree 1 in each single entry, so that
    # the difference is exact but for 64-bit rounding; what is left is the
    # kernel's (fp32 sums, or bf16 for dx)
    for name, grad, rel in (("x", dx, HALF_BF16 + 1e-4), ("a", da, 1e-4), ("b", db, 1e-4)):
        g = grad.double().cpu()
        for at in ((0, 0, 0), (1, 3, 5), (1, 7, 2)) if g.dim() == 3 else ((0, 0), (8, 33), (12, 39)):
            diff = (value(name, at, 0.5) - value(name, at, -0.5))
            assert abs(diff - float(g[at])) <= rel * max(abs(diff), float(g.abs().mean())), (name, at)


def test_in_place_and_column_slices(eng):
    """base as its own output, and tensors that are columns of wider ones."""
    import torch

    from pih_amd.linear import adapter_backward, adapter_gemm

    c = _case(11, [17, 6], [1, 0], 16, 64, 128, 2)
    d = _dev(c)
    args = (d["a"], d["b"], d["scale"], d["offsets"], d["adapters"])
    want, _ = adapter_gemm(d["x"], *args, base=d["base"])
    wide_x = torch.randn(23, 200, device="cuda").to(torch.bfloat16)
    wide_y = torch.full((23, 152), 3.0, dtype=torch.bfloat16, device="cuda")
    wide_x[:, 40:168], wide_y[:, 8:72] = d["x"], d["base"]
    y = wide_y[:, 8:72]
    got, _ = adapter_gemm(wide_x[:, 40:168], *args, base=y, out=y)
    assert got is y and torch.equal(y, want)
    assert torch.all(wide_y[:, :8] == 3.0) and torch.all(wide_y[:, 72:] == 3.0)
    dx, da, db, _ = adapter_backward(d["dy"], d["x"], *args, base=d["dbase"])
    wide_dy = torch.randn(23, 96, device="cuda").to(torch.bfloat16)
    wide_dy[:, 16:80] = d["dy"]
    wide_dx = wide_x.clone()
    wide_dx[:, 40:168] = d["dbase"]
    z = wide_dx[:, 40:168]
    out = adapter_backward(wide_dy[:, 16:80], wide_x[:, 40:168], *args, base=z, out=z)
    torch.cuda.synchronize()
    assert torch.equal(z, dx) and torch.equal(out[1], da) and torch.equal(out[2], db)
    assert torch.equal(wide_dx[:, :40], wide_x[:, :40]) and torch.equal(wide_dx[:, 168:], wide_x[:, 168:])
    with pytest.raises(ValueError):
        adapter_gemm(d["x"].t().contiguous().t(), *args)


def test_values_outside_the_segments_do_not_matter(eng):
    """NaN in rows that belong to no segment, infinities and NaN in the
    stacks of adapters that no segment has."""
    import torch

    from pih_amd.linear import adapter_backward, adapter_gemm

    c = _case(13, [18, 30], [2, 0], 24, 72, 136, 4, first=3, tail=5)
    d = _dev(c)
    plain = adapter_gemm(d["x"], d["a"], d["b"], d["scale"], d["offsets"], d["adapters"])[0]
    grads = adapter_backward(d["dy"], d["x"], d["a"], d["b"], d["scale"], d["offsets"], d["adapters"])
    for t in ("x", "dy"):
        d[t][:3] = float("nan")
        d[t][51:] = float("inf")
    for t in ("a", "b"):
        d[t][1] = float("nan")
        d[t][3] = float("inf")
    d["scale"][1] = float("nan")
    got = adapter_gemm(d["x"], d["a"], d["b"], d["scale"], d["offsets"], d["adapters"])[0]
    bad = adapter_backward(d["dy"], d["x"], d["a"], d["b"], d["scale"], d["offsets"], d["adapters"])
    torch.cuda.synchronize()
    assert torch.equal(got[3:51], plain[3:51])
    assert torch.equal(bad[0][3:51], grads[0][3:51])
    for p, q in zip(bad[1:3], grads[1:3]):
        assert torch.equal(p, q) and torch.all(p[[1, 3]] == 0)


def test_a_row_without_adapter_keeps_its_base_bits(eng):
    import torch

    from pih_amd.linear import adapter_gemm

    c = _case(17, [4, 20], [-1, 0], 8, 48, 64, 1)
    d = _dev(c)
    d["x"][:4] = float("nan")
    d["base"][0, 0], d["base"][1, 3] = float("inf"), -0.0
    out, flag = adapter_gemm(d["x"], d["a"], d["b"], d["scale"], d["offsets"], d["adapters"], base=d["base"])
    torch.cuda.synchronize()
    assert int(flag.item()) == 0
    assert torch.equal(out[:4].view(torch.int16), d["base"][:4].view(torch.int16))


def test_bad_ids_and_offsets_are_flagged(eng):
    import torch

    from pih_amd.linear import adapter_backward, adapter_gemm

    c = _case(19, [4, 20, 7], [0, 1, 0], 8, 48, 64, 2)
    d = _dev(c)
    want = adapter_gemm(d["x"], d["a"], d["b"], d["scale"], d["offsets"], d["adapters"], base=d["base"])[0]
    d["adapters"][1] = 2
    out = torch.full_like(d["base"], 7.0)
    _, flag = adapter_gemm(d["x"], d["a"], d["b"], d["scale"], d["offsets"], d["adapters"], base=d["base"], out=out)
    torch.cuda.synchronize()
    assert int(flag.item()) == 1
    assert torch.all(out[4:24] == 7.0) and torch.equal(out[:4], want[:4]) and torch.equal(out[24:], want[24:])
    _, da, _, flag = adapter_backward(d["dy"], d["x"], d["a"], d["b"], d["scale"], d["offsets"], d["adapters"])
    assert int(flag.item()) == 1 and torch.all(da[1] == 0)
    d["adapters"][1] = 1
    d["offsets"][3] = 32  # past the 31 rows
    out.fill_(7.0)
    _, flag = adapter_gemm(d["x"], d["a"], d["b"], d["scale"], d["offsets"], d["adapters"], base=d["base"], out=out)
    torch.cuda.synchronize()
    assert int(flag.item()) == 2
    assert torch.equal(out[:24], want[:24]) and torch.all(out[24:] == 7.0)
    d["offsets"][3] = 20  # descends
    out.fill_(7.0)
    _, flag = adapter_gemm(d["x"], d["a"], d["b"], d["scale"], d["offsets"], d["adapters"], base=d["base"], out=out)
    torch.cuda.synchronize()
    assert int(flag.item()) == 2
    assert torch.equal(out[:24], want[:24]) and torch.all(out[24:] == 7.0)


def test_captured_and_replayed(eng):
    """Forward and backward in one graph, replayed on new inputs between
    eager calls of the same sizes."""
    import torch

    from pih_amd.linear import adapter_backward, adapter_gemm

    c = _case(23, [40, 1, 300], [0, 1, 1], 16, 256, 512, 2)
    d = _dev(c)
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")

    def calls():
        y, _ = adapter_gemm(d["x"], d["a"], d["b"], d["scale"], d["offsets"], d["adapters"], base=d["base"], flag=flag)
        return (y,) + adapter_backward(d["dy"], d["x"], d["a"], d["b"], d["scale"], d["offsets"], d["adapters"],
                                       base=d["dbase"], flag=flag)[:3]

    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.current_stream()):
        held = calls()
    for i in range(4):
        d["x"].copy_(_case(30 + i, [40, 1, 300], [0, 1, 1], 16, 256, 512, 2)["x"].cuda())
        eager = calls()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(held, eager):
            assert torch.equal(p, q)
    assert int(flag.item()) == 0


def test_other_streams_at_once(eng):
    """Calls on two streams, each with the workspace of its own call."""
    import torch

    from pih_amd.linear import adapter_gemm

    cases = [_dev(_case(50 + i, [200, 56], [0, 1], 32, 1024, 2048, 2)) for i in range(2)]
    call = lambda d: adapter_gemm(d["x"], d["a"], d["b"], d["scale"], d["offsets"], d["adapters"],  # noqa: E731
                                  base=d["base"])[0]
    want = [call(d) for d in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(cases[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def _mix(seed, count, adapters, longest=2, none=8):
    """Segments of 0 to `longest` rows and their adapters, every none-th without."""
    g = np.random.default_rng(seed)
    ids = g.integers(0, adapters, count)
    ids[none - 1::none] = -1
    return g.integers(0, longest + 1, count).tolist(), ids.tolist()


# as CASES: short segments, whose tiles take an adapter's rows from all of them
SHORT = [
    ([1] * 33, [0] * 33, 16, 72, 520, 1, 0, 0),  # one adapter, two tiles and a row
    ([1] * 300, [i % 3 for i in range(300)], 128, 136, 1032, 3, 0, 0),  # more segments than threads, tiles across them
    ([2] * 40, [-1] * 40, 8, 64, 64, 4, 0, 0),  # no adapter at all
    (*_mix(1, 900, 400), 8, 24, 40, 400, 7, 30),  # more adapters than threads, some without rows, empty segments
    (*_mix(2, 2048, 5), 24, 40, 264, 6, 0, 0),  # the most segments
    (*_mix(3, 2048, 1023), 8, 16, 24, 1023, 3, 0),  # and the most adapters
    ([1, 60] + [0] * 60, [1, 0] * 31, 64, 200, 136, 2, 1, 2),  # one segment has all tiles
    (*_mix(4, 2049, 9), 8, 32, 64, 9, 0, 0),  # one segment more than the groups take
]


@pytest.mark.parametrize("base", [True, False])
@pytest.mark.parametrize("case", range(len(SHORT)))
def test_short_segments(eng, case, base):
    import torch

    from pih_amd.linear import adapter_gemm

    c = _case(300 + case, *SHORT[case])
    ref, bound, written = _forward_ref(c, base)
    d = _dev(c)
    args = (d["x"], d["a"], d["b"], d["scale"], d["offsets"], d["adapters"])
    out = torch.full_like(d["base"], 7.0)
    got, flag = adapter_gemm(*args, base=d["base"] if base else None, out=out)
    w = torch.from_numpy(written)
    again = adapter_gemm(*args, base=d["base"] if base else None)[0]
    torch.cuda.synchronize()
    assert int(flag.item()) == 0
    assert torch.all(got.cpu()[~w] == 7.0)
    assert torch.equal(got[w.cuda()], again[w.cuda()])
    _within(got[w.cuda()], ref[w], bound[w], f"case {case}")


def test_short_segments_in_place_and_flagged(eng):
    import torch

    from pih_amd.linear import adapter_gemm

    c = _case(331, [1] * 64, [i % 3 - (i % 3 == 2) * 3 for i in range(64)], 16, 72, 136, 2)
    d = _dev(c)
    args = (d["x"], d["a"], d["b"], d["scale"], d["offsets"], d["adapters"])
    want = adapter_gemm(*args, base=d["base"])[0]
    y = d["base"].clone()
    assert torch.equal(adapter_gemm(*args, base=y, out=y)[0], want)
    d["adapters"][6] = 2  # past the stacks
    out = torch.full_like(want, 7.0)
    _, flag = adapter_gemm(*args, base=d["base"], out=out)
    torch.cuda.synchronize()
    rest = torch.arange(64, device="cuda") != 6
    assert int(flag.item()) == 1 and torch.all(out[6] == 7.0) and torch.equal(out[rest], want[rest])
    d["adapters"][6] = 0
    d["offsets"][64] = 65  # past the rows
    out.fill_(7.0)
    _, flag = adapter_gemm(*args, base=d["base"], out=out)
    torch.cuda.synchronize()
    assert int(flag.item()) == 2 and torch.all(out[63] == 7.0) and torch.equal(out[:63], want[:63])
    d["offsets"][64] = 62  # descends: the last two segments' rows are in question
    out.fill_(7.0)
    _, flag = adapter_gemm(*args, base=d["base"], out=out)
    torch.cuda.synchronize()
    assert int(flag.item()) == 2 and torch.equal(out[:62], want[:62])


def test_short_segments_captured(eng):
    """A decode batch whose segments change between replays."""
    import torch

    from pih_amd.linear import adapter_gemm

    c = _case(341, [1] * 96, [i % 4 for i in range(96)], 32, 264, 520, 4)
    d = _dev(c)
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    call = lambda: adapter_gemm(d["x"], d["a"], d["b"], d["scale"], d["offsets"], d["adapters"],  # noqa: E731
                                base=d["base"], flag=flag)[0]
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.current_stream()):
        held = call()
    for i in range(4):
        g = torch.Generator().manual_seed(350 + i)
        d["adapters"].copy_(torch.randint(-1, 4, (96,), generator=g).to(torch.int32))
        d["offsets"].copy_((torch.rand(97, generator=g) * 97).long().sort().values.clamp(max=96).to(torch.int32))
        d["offsets"][0], d["offsets"][96] = 0, 96
        eager = call()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, eager)
    assert int(flag.item()) == 0


def test_rows_more_than_4_gib_apart(eng):
    """x, base and output (in place), dy and dx as rows of one buffer each,
    whose last row lies past 2^32 bytes."""
    import torch

    from pih_amd.linear import adapter_backward, adapter_gemm

    c = _case(401, [2, 1], [1, 0], 16, 72, 136, 2)
    d = _dev(c)
    apart = (1 << 30) + 64
    far = {}
    for name in ("x", "base", "dy", "dbase"):
        flat = torch.empty(2 * apart + d[name].shape[1], dtype=torch.bfloat16, device="cuda")
        far[name] = flat.as_strided(d[name].shape, (apart, 1))
        far[name].copy_(d[name])
    args = (d["a"], d["b"], d["scale"], d["offsets"], d["adapters"])
    want = adapter_gemm(d["x"], *args, base=d["base"])[0]
    grads = adapter_backward(d["dy"], d["x"], *args, base=d["dbase"])
    got, flag = adapter_gemm(far["x"], *args, base=far["base"], out=far["base"])
    out = adapter_backward(far["dy"], far["x"], *args, base=far["dbase"], out=far["dbase"], flag=flag)
    torch.cuda.synchronize()
    assert int(flag.item()) == 0
    assert torch.equal(got, want)
    assert all(torch.equal(p, q) for p, q in zip(out[:3], grads[:3]))


def test_stacks_past_4_gib(eng):
    """The last of 530 adapters of 4.4 GB of A and of B (only two are filled)."""
    import torch

    from pih_amd.linear import adapter_gemm

    c = _case(409, [17, 30], [0, 1], 128, 32768, 32768, 2)
    d = _dev(c)
    want = adapter_gemm(d["x"], d["a"], d["b"], d["scale"], d["offsets"], d["adapters"], base=d["base"])[0]
    a = torch.empty(530, 128, 32768, dtype=torch.bfloat16, device="cuda")
    b = torch.empty(530, 32768, 128, dtype=torch.bfloat16, device="cuda")
    scale = torch.zeros(530, device="cuda")
    for at, i in ((529, 0), (3, 1)):
        a[at], b[at], scale[at] = d["a"][i], d["b"][i], d["scale"][i]
    ids = torch.tensor([529, 3], dtype=torch.int32, device="cuda")
    got, flag = adapter_gemm(d["x"], a, b, scale, d["offsets"], ids, base=d["base"])
    torch.cuda.synchronize()
    assert int(flag.item()) == 0 and torch.equal(got, want)


# as CASES: segments long enough for the tall tiles, ranks that fill none of
# their 32-rank pieces, rows enough for several splits of the gradients
LONG = [
    ([600, 3, 700, 0, 41], [1, 0, 1, 2, 0], 104, 136, 264, 3, 9, 5),
    ([130, 70, 65], [0, 1, -1], 40, 328, 72, 2, 0, 0),
    ([1100, 64], [1, 1], 128, 72, 520, 2, 0, 3),
    ([90, 200], [0, 0], 72, 40, 1032, 1, 1, 0),
]


@pytest.mark.parametrize("base", [True, False])
@pytest.mark.parametrize("case", range(len(LONG)))
def test_long_segments_of_odd_ranks(eng, case, base):
    import torch

    from pih_amd.linear import adapter_backward, adapter_gemm

    c = _case(500 + case, *LONG[case])
    ref, bound, written = _forward_ref(c, base)
    (dx, ex), (da, ea), (db, eb) = _backward_ref(c, base)
    d = _dev(c)
    w = torch.from_numpy(written)
    got, flag = adapter_gemm(d["x"], d["a"], d["b"], d["scale"], d["offsets"], d["adapters"],
                             base=d["base"] if base else None, out=torch.full_like(d["base"], 7.0))
    args = (d["dy"], d["x"], d["a"], d["b"], d["scale"], d["offsets"], d["adapters"])
    grads = adapter_backward(*args, base=d["dbase"] if base else None, out=torch.full_like(d["dbase"], 7.0), flag=flag)
    again = adapter_backward(*args, base=d["dbase"] if base else None, out=torch.full_like(d["dbase"], 7.0))
    torch.cuda.synchronize()
    assert int(flag.item()) == 0
    assert torch.all(got.cpu()[~w] == 7.0) and torch.all(grads[0].cpu()[~w] == 7.0)
    _within(got[w.cuda()], ref[w], bound[w], f"case {case}")
    _within(grads[0][w.cuda()], dx[w], ex[w], f"dx {case}")
    _within(grads[1], da, ea, f"da {case}")
    _within(grads[2], db, eb, f"db {case}")
    assert all(torch.equal(p, q) for p, q in zip(grads[:3], again[:3]))


# segment length, rank: tiles of 16 rows, and of 64 in each of the two products with B
@pytest.mark.parametrize("length,rank", [(1, 8), (40, 16), (70, 16), (70, 64), (66, 128)])
@pytest.mark.parametrize("bad", [64, 70, 98, 99])
def test_bad_offsets_behind_many_segments_are_flagged(eng, bad, length, rank):
    """Bit 2 for an offset that the block of the first tile need not read to
    find it, forward and backward: the end of segment `bad` of 100 passes the
    rows, and the next one's descends from there.  What is left out, and all
    else, is as with no adapter on those segments."""
    import torch

    from pih_amd.linear import adapter_backward, adapter_gemm

    stacks = 100 if length == 1 else 3  # (an adapter each: no tiles across segments)
    c = _case(600 + bad, [length] * 100, [i % stacks for i in range(100)], rank, 40, 72, stacks)
    d = _dev(c)
    args = (d["a"], d["b"], d["scale"])
    none = d["adapters"].clone()
    none[bad:bad + 2] = -1
    left = slice(bad * length, min(bad + 2, 100) * length)

    def calls(offsets, adapters):
        out, dx = torch.full_like(d["base"], 7.0), torch.full_like(d["dbase"], 7.0)
        _, flag = adapter_gemm(d["x"], *args, offsets, adapters, base=d["base"], out=out)
        _, da, db, back = adapter_backward(d["dy"], d["x"], *args, offsets, adapters, base=d["dbase"], out=dx)
        torch.cuda.synchronize()
        return out, dx, da, db, int(flag.item()), int(back.item())

    want = calls(d["offsets"], none)
    assert want[4:] == (0, 0)
    want[0][left], want[1][left] = 7.0, 7.0
    offsets = d["offsets"].clone()
    offsets[bad + 1] = 100 * length + 1
    got = calls(offsets, d["adapters"])
    assert got[4:] == (2, 2)
    for p, q in zip(got[:4], want[:4]):
        assert torch.equal(p, q)


# each kernel of the product with B: tiles of 16, 32 and 64 rows, of rows from all segments
@pytest.mark.parametrize("lengths,adapters,rank", [([9, 4], [1, 0], 24), ([70, 81], [1, 0], 16), ([70, 81], [0, 1], 72),
                                                   ([1] * 40, [i % 2 for i in range(40)], 16)])
def test_infinite_and_largest_products_with_a(eng, lengths, adapters, rank):
    """An infinite x . A (and dy . B) is infinite in out (dx) and in db (da),
    and a finite one past the largest bf16 stays finite: three rows with
    x[0] = +-inf or with x[:2] of the largest bf16 and 2^119 (a sum of
    0x1.ff * 2^127, which bf16 rounds to infinity), A[:, :2] = 1, B >= 0."""
    import torch

    from pih_amd.linear import adapter_backward, adapter_gemm

    c = _case(700 + rank, lengths, adapters, rank, 40, 72, 2, scale=False)
    rows = sum(lengths)
    plus, minus, large = 1, rows // 2, rows - 1
    for t in (c["x"], c["dy"]):
        t[plus, 0], t[minus, 0] = float("inf"), float("-inf")
        t[large] = 0
        t[large, 0], t[large, 1] = torch.finfo(torch.bfloat16).max, 2.0 ** 119
    # dx and db of the rows with infinite dy take A and x of one sign
    c["a"], c["b"] = c["a"].abs() + 2.0 ** -10, c["b"].abs() + 2.0 ** -10
    forward = {**c, "a": c["a"].clone()}
    forward["a"][:, :, :2] = 1
    forward["b"] = (c["b"] * 2.0 ** -4 / rank).to(torch.bfloat16)
    d = _dev(forward)
    args = (d["x"], d["a"], d["b"], None, d["offsets"], d["adapters"])
    out, flag = adapter_gemm(*args, base=d["base"])
    finite = c["dy"].clone()
    finite[[plus, minus, large]] = 1
    dx, da, db, _ = adapter_backward(finite.cuda(), *args, flag=flag)
    torch.cuda.synchronize()
    assert int(flag.item()) == 0
    out, dx, db = out.cpu(), dx.cpu(), db.cpu()
    assert torch.all(out[plus] == float("inf")) and torch.all(out[minus] == float("-inf"))
    rest = torch.ones(rows, dtype=torch.bool)
    rest[[plus, minus]] = False
    plain = {**forward, "x": forward["x"].clone(), "dy": finite}
    plain["x"][[plus, minus]] = 0
    ref, bound, _ = _forward_ref(plain, True)
    assert torch.isfinite(out[large]).all()
    _within(out[rest], ref[rest], bound[rest], "out")
    assert torch.isfinite(dx).all()  # (x takes no part in it)
    owner = {a: [r for lo, hi, i in _segments(c) if i == a for r in (plus, minus, large) if lo <= r < hi] for a in (0, 1)}
    for a, held in owner.items():
        if held and set(held) <= {plus}:
            assert torch.all(db[a] == float("inf"))
        if held and set(held) <= {minus}:
            assert torch.all(db[a] == float("-inf"))
        if held == [large]:
            assert torch.isfinite(db[a]).all()
    # the same of dy . B: dx and da
    back = {**c, "b": c["b"].clone(), "x": torch.ones_like(c["x"])}
    back["b"][:, :2] = 1
    back["a"] = (c["a"] * 2.0 ** -4 / rank).to(torch.bfloat16)
    d = _dev(back)
    dx, da, db, flag = adapter_backward(d["dy"], d["x"], d["a"], d["b"], None, d["offsets"], d["adapters"])
    torch.cuda.synchronize()
    dx, da = dx.cpu(), da.cpu()
    assert int(flag.item()) == 0
    assert torch.all(dx[plus] == float("inf")) and torch.all(dx[minus] == float("-inf"))
    assert torch.isfinite(dx[rest]).all()
    for a, held in owner.items():
        if held and set(held) <= {plus}:
            assert torch.all(da[a] == float("inf"))
        if held and set(held) <= {minus}:
            assert torch.all(da[a] == float("-inf"))
        if held == [large]:
            assert torch.isfinite(da[a]).all()


@pytest.mark.parametrize("lengths,rank", [([9], 24), ([140], 16), ([140], 72)])
def test_a_nan_stays_in_its_row_and_adapter(eng, lengths, rank):
    """NaN in x reaches all of its row's output and its adapter's db; in dy
    its row's dx and its adapter's da; and nothing else."""
    import torch

    from pih_amd.linear import adapter_backward, adapter_gemm

    c = _case(730 + rank, lengths + [5], [0, 1], rank, 40, 72, 2)
    c["a"], c["b"] = c["a"].abs() + 2.0 ** -10, c["b"].abs() + 2.0 ** -10
    for t in ("x", "dy"):
        bad = {**c, t: c[t].clone()}
        bad[t][3, 7] = float("nan")
        d = _dev(bad)
        args = (d["x"], d["a"], d["b"], d["scale"], d["offsets"], d["adapters"])
        out, flag = adapter_gemm(*args)
        dx, da, db, _ = adapter_backward(d["dy"], *args, flag=flag)
        torch.cuda.synchronize()
        assert int(flag.item()) == 0
        row = out if t == "x" else dx
        assert row[3].isnan().all() and torch.isfinite(row[:3]).all() and torch.isfinite(row[4:]).all()
        assert torch.isfinite(dx if t == "x" else out).all()
        whole, column = (db, da) if t == "x" else (da, db.transpose(1, 2))
        assert whole[0].isnan().all() and torch.isfinite(whole[1]).all()
        assert column[0, :, 7].isnan().all() and torch.isfinite(column[1]).all()
        rest = torch.arange(column.shape[2], device="cuda") != 7
        assert torch.isfinite(column[0][:, rest]).all()
