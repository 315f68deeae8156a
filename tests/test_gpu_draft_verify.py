"""Verification of drafted tokens (launch_draft_verify) against a sequential
restatement in 64 bits on the CPU: tokens and counts are equal.  (A token
differs only where a sum of probabilities comes within some 1e-13 of the
threshold, which for the sizes here happens once in 1e7 runs.)"""
import pytest

pytestmark = pytest.mark.gpu
NONE = -1


@pytest.fixture(scope="module")
def eng():
    import torch

    from pih_amd.device import engine_stream

    with engine_stream() as s:
        yield s
        torch.cuda.synchronize()


def _softmax(row, t):
    import numpy as np

    row = row.astype(np.float64)
    e = np.exp((row - row.max()) / t)
    return e / e.sum()


def _reference(target, tokens, offsets, accept, sample, most, draft=None, temperature=None):
    """(tokens, accepted, error bits), one sequence at a time."""
    import numpy as np

    vocab, count = target.shape[1], len(offsets) - 1
    out, accepted, bits = np.full((count, most + 1), NONE, np.int32), np.zeros(count, np.int32), 0
    for s in range(count):
        lo, hi = int(offsets[s]), int(offsets[s + 1])
        t = 1.0 if temperature is None else float(temperature[s])
        if not 0 <= lo <= hi <= len(tokens) or hi - lo > most:
            bits |= 2
            continue
        if not (t >= 0 and t < np.inf):
            bits |= 4
            continue
        for i in range(hi - lo + 1):
            row = target[lo + s + i]
            last = i == hi - lo
            soft = draft is not None and not last and t > 0
            bad = np.isnan(row).any() or row.max() == -np.inf or (t > 0 and row.max() == np.inf)
            if soft:
                q = draft[lo + i]
                bad = bad or np.isnan(q).any() or not np.isfinite(q.max())
            d = None if last else int(tokens[lo + i])
            outside = d is not None and not 0 <= d < vocab
            bits |= outside
            if bad:
                bits |= 4
                break
            if t == 0:
                best = int(row.argmax())
                if d == best:
                    out[s, i], accepted[s] = d, i + 1
                    continue
                out[s, i] = best
                break
            p = _softmax(row, t)
            rest = p
            if not last:
                q = _softmax(q, t) if soft else np.zeros(vocab)
                if not soft and not outside:
                    q[d] = 1.0
                if not outside and float(accept[lo + i]) * q[d] < p[d]:
                    out[s, i], accepted[s] = d, i + 1
                    continue
                if soft:
                    rest = np.maximum(p - q, 0)
                elif not outside:
                    rest = p.copy()
                    rest[d] = 0
                if not rest.sum() > 0:
                    rest = p
            run = np.cumsum(rest)
            v = int(np.searchsorted(run, float(sample[s]) * run[-1], side="right"))
            out[s, i] = min(v, int(np.nonzero(rest)[0][-1]))
            break
    return out, accepted, bits


def _case(seed, counts, vocab, dtype="float32", soft=True, spread=2.0, near=0.5, temperature=None, pad=0):
    """Logits on the CPU with what a draft model would have drawn from them."""
    import numpy as np
    import torch

    rng = np.random.default_rng(seed)
    counts = np.asarray(counts)
    offsets = np.concatenate(([0], counts.cumsum())).astype(np.int32)
    drafts, sequences = int(counts.sum()), len(counts)
    common = rng.normal(size=vocab) * spread
    target = (rng.normal(size=(drafts + sequences, vocab)) * spread + common).astype(np.float32)
    row = np.concatenate([np.arange(c) + offsets[s] + s for s, c in enumerate(counts)] + [np.zeros(0)]).astype(int)
    draft = (target[row] + near * rng.normal(size=(drafts, vocab))).astype(np.float32)
    as_type = lambda a: torch.from_numpy(a).to(getattr(torch, dtype))  # noqa: E731
    target, draft = as_type(target), as_type(draft)
    of = np.repeat(np.arange(sequences), counts)
    tau = np.ones(drafts) if temperature is None else np.asarray(temperature, np.float64)[of]
    d64 = draft.double().numpy()
    noise = rng.gumbel(size=d64.shape)
    with np.errstate(divide="ignore", invalid="ignore"):
        drawn = np.where((tau > 0)[:, None], d64 / tau[:, None] + noise, d64)
    tokens = drawn.argmax(1).astype(np.int32) if drafts else np.zeros(0, np.int32)
    return dict(target=target, tokens=tokens, offsets=offsets, accept=rng.random(drafts, np.float32),
                sample=rng.random(sequences, np.float32), draft=draft if soft else None,
                temperature=None if temperature is None else np.asarray(temperature, np.float32))


def _run(case, most, pad=0, sentinel=False):
    import numpy as np
    import torch

    from pih_amd.linear import draft_verify

    def rows(t):
        if t is None:
            return None
        wide = torch.full((t.shape[0], t.shape[1] + pad), float("nan"), dtype=t.dtype, device="cuda")
        wide[:, :t.shape[1]] = t.cuda()
        return wide[:, :t.shape[1]]

    dev = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    for n in (1 << 10, 1 << 14, 1 << 18, 1 << 22):
        torch.full((n,), float("nan"), device="cuda")  # freed: later allocations get it
    got = draft_verify(rows(case["target"]), dev(case["tokens"]), dev(case["offsets"]), dev(case["accept"]),
                       dev(case["sample"]), most, draft_logits=rows(case["draft"]), temperature=dev(case["temperature"]))
    torch.cuda.synchronize()
    return got[0].cpu().numpy(), got[1].cpu().numpy(), int(got[2].item())


def _check(case, most, pad=0):
    import numpy as np

    as_np = lambda t: None if t is None else t.float().numpy()  # noqa: E731
    want = _reference(as_np(case["target"]), case["tokens"], case["offsets"], case["accept"], case["sample"], most,
                      as_np(case["draft"]), case["temperature"])
    got = _run(case, most, pad)
    np.testing.assert_array_equal(got[1], want[1])
    np.testing.assert_array_equal(got[0], want[0])
    assert got[2] == want[2]
    return got


COUNTS = [[0], [1], [5], [3, 0, 4, 1], [0, 0], list(range(8)) * 4, [2] * 33, [255], [0, 17, 0, 60]]


@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: f"{len(c)}x{max(c)}")
@pytest.mark.parametrize("vocab", [1, 2, 255, 1000, 4096, 4097, 10007])
@pytest.mark.parametrize("soft", [True, False])
def test_sizes(eng, counts, vocab, soft):
    t = None if len(counts) == 2 else [0.7 + 0.1 * (i % 5) if i % 4 != 3 else 0.0 for i in range(len(counts))]
    _check(_case(len(counts) * 100 + vocab, counts, vocab, soft=soft, temperature=t), max(counts))


@pytest.mark.parametrize("vocab,pad", [(1000, 1), (1001, 0), (4099, 5), (4104, 8), (9000, 3)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("soft", [True, False])
def test_strides_and_types(eng, vocab, pad, dtype, soft):
    _check(_case(vocab, [4, 2, 0, 7, 3], vocab, dtype=dtype, soft=soft, temperature=[1.0, 0.0, 0.5, 2.0, 0.9]), 9, pad)


@pytest.mark.parametrize("dtype,soft", [("float32", True), ("bfloat16", False), ("bfloat16", True)])
def test_large_vocabulary(eng, dtype, soft):
    """Many seeds over a real vocabulary: most drafts are accepted, some not."""
    accepted = 0
    for seed in range(6):
        got = _check(_case(seed, [5, 3, 0, 4, 1, 2, 5, 5], 151936, dtype=dtype, soft=soft, spread=1.5,
                           temperature=[0.6, 1.0, 0.9, 1.3, 0.0, 0.8, 0.7, 1.0]), 5)
        accepted += got[1].sum()
    assert accepted > 0


@pytest.mark.parametrize("vocab,sequences", [(9000, 127), (9000, 129), (9000, 200), (300, 500), (40960, 45)])
@pytest.mark.parametrize("dtype,soft", [("float32", True), ("bfloat16", False)])
def test_many_sequences(eng, vocab, sequences, dtype, soft):
    """Enough of them that the walk and the draw are launches of their own, and
    just not: masks, greedy ones, hardly any randomness, tokens outside and broken
    rows among them."""
    import numpy as np

    counts = [i % 6 for i in range(sequences)]
    t = [(1.0, 0.0, 0.6, 1e-3, 1.4, 0.8, 1e5)[i % 7] for i in range(sequences)]
    case = _case(vocab + sequences, counts, vocab, dtype=dtype, soft=soft, temperature=t)
    case["target"][::5, 20:] = float("-inf")
    case["target"][3::17, 1:] = float("-inf")
    case["tokens"][5::40] = vocab
    case["target"][61] = float("-inf")
    case["target"][90, 7] = float("nan")
    case["accept"][1::9] = np.float32(1 - 2.0 ** -24)
    assert _check(case, 6)[2] == 5


def test_random_numbers_at_their_ends(eng):
    """0 accepts what has a probability and takes the first token that has one;
    the largest number below 1 the last."""
    import numpy as np

    top = np.float32(1 - 2.0 ** -24)
    for soft in (True, False):
        for u in (np.float32(0), top):
            for r in (np.float32(0), top):
                case = _case(5, [3, 3, 0], 5000, soft=soft)
                case["target"][:, :7] = float("-inf")
                case["target"][:, -3:] = float("-inf")
                case["target"][:, 4996] = 3.0  # (far above 2^-24 of the sum)
                case["tokens"][:] = 100 + np.arange(6)
                case["accept"][:], case["sample"][:] = u, r
                got = _check(case, 3)
                if u == 0:
                    assert (got[1] == [3, 3, 0]).all()
                    # behind all drafts, from p alone
                    assert (got[0][[0, 1, 2], [3, 3, 0]] == (7 if r == 0 else 4996)).all()


def test_equal_models_accept_everything(eng):
    """The same logits for both: p = q to the bit, accepted for every number
    below 1."""
    import numpy as np
    import torch

    case = _case(8, [6, 6, 2], 3001, near=0.0, temperature=[0.3, 1.0, 1.7])
    case["accept"][:] = np.float32(1 - 2.0 ** -24)
    at = np.concatenate([np.arange(c) + o + s for s, (c, o) in enumerate(zip((6, 6, 2), case["offsets"]))])
    case["draft"] = case["target"][torch.from_numpy(at)].clone()
    got = _check(case, 6)
    assert (got[1] == [6, 6, 2]).all()


def test_masked_logits(eng):
    """-infinity has probability 0: a masked draft is rejected, and nothing
    masked is put out, also where the mask leaves one token."""
    import numpy as np

    for soft in (True, False):
        case = _case(9, [4, 4, 4, 4], 2000, soft=soft, temperature=[1.0, 0.0, 0.5, 1.0])
        case["target"][::2, 10:] = float("-inf")
        case["target"][[17, 19], :1999] = float("-inf")
        if soft:
            case["draft"][1::3, ::2] = float("-inf")
        got = _check(case, 4)
        assert got[2] == 0
        # the draft's mask alone
        case = _case(10, [3, 3], 700, soft=soft)
        case["tokens"][0] = 5
        case["target"][0] = float("-inf")
        case["target"][0, 6] = 1.0
        got = _check(case, 3)
        assert got[0][0, 0] == 6 and got[1][0] == 0
        assert (got[0][0, 1:] == NONE).all()
        np.testing.assert_array_equal(got[0] < 700, True)


@pytest.mark.parametrize("soft", [True, False])
def test_extreme_temperatures(eng, soft):
    """Temperatures so low that the largest logit alone has a probability, or
    that a logit over it exceeds 64 bits' integers, and so high that all have the
    same; logits of every size."""
    import numpy as np

    for seed, spread in ((1, 1.0), (2, 50.0), (3, 1e-3)):
        t = [1e-45, 1e-38, 1e-30, 1e-20, 1e-12, 1e-8, 1e-5, 1e-3, 0.03, 30.0, 1e4, 1e20, 3e38]
        case = _case(seed, [3] * len(t), 9000, soft=soft, spread=spread, near=0.1 * spread, temperature=t)
        case["accept"][::4] = np.float32(1 - 2.0 ** -24)
        got = _check(case, 3)
        assert got[2] == 0
        # (equal models accept everything, at any of them)
        if soft:
            case["draft"] = case["target"][[4 * s + i for s in range(len(t)) for i in range(3)]].clone()
            tau = np.repeat(np.asarray(t, np.float32), 3)
            cold = tau < 0.1  # (a draft of probability 0 is rejected)
            case["tokens"][cold] = case["draft"].numpy()[cold].argmax(1)
            case["accept"][:] = np.float32(1 - 2.0 ** -24)
            got = _check(case, 3)
            assert (got[1] == 3).all()


def test_greedy_takes_the_first_of_equals(eng):
    case = _case(3, [3, 3], 9000, temperature=[0.0, 0.0])
    t = case["target"]
    t[0, 4095] = t[0, 4096] = t[0, 8999] = 50.0
    t[1, 17] = t[1, 8000] = 60.0
    t[4, 4097] = t[4, 4098] = float("inf")
    case["tokens"][:] = [4095, 8000, 3, 4098, 1, 2]
    got = _check(case, 3)
    assert got[0].tolist() == [[4095, 17, NONE, NONE], [4097, NONE, NONE, NONE]]
    assert got[2] == 0


def test_error_bits(eng):
    import numpy as np

    base = dict(counts=[2, 2, 2], vocab=600)
    # drafted tokens outside the vocabulary, reached and not
    case = _case(1, **base)
    case["tokens"][2] = 600
    case["tokens"][4] = -7
    got = _check(case, 2)
    assert got[2] == 1 and got[1][1] == 0 and got[1][2] == 0
    assert (got[0][1:, 0] >= 0).all()
    case = _case(1, **base, soft=False)
    case["tokens"][2] = 600
    assert _check(case, 2)[2] == 1
    # behind a rejected draft nothing counts
    case = _case(1, **base)
    case["target"][0, :] = float("-inf")
    case["target"][0, 3] = 0.0
    case["tokens"][:2] = [4, 10 ** 6]
    case["target"][1] = float("nan")
    case["draft"][1] = float("nan")
    got = _check(case, 2)
    assert got[2] == 0 and got[0][0].tolist() == [3, NONE, NONE]
    # rows without probabilities end their sequence
    for v in ("nan", "inf", "-inf"):
        case = _case(2, **base)
        case["accept"][:] = 0.0
        case["target"][1, :] = float(v)  # sequence 0, place 1
        case["target"][5, 5] = float("nan")  # sequence 1, behind its drafts
        case["draft"][4, 7] = float("nan" if v == "-inf" else "inf")  # sequence 2, place 0
        got = _check(case, 2)
        assert got[2] == 4 and got[1].tolist() == [1, 2, 0]
        assert got[0][0, 1:].tolist() == [NONE, NONE] and got[0][1, 2] == NONE and (got[0][2] == NONE).all()
    # temperatures
    case = _case(2, **base, temperature=[-1.0, float("nan"), float("inf")])
    got = _check(case, 2)
    assert got[2] == 4 and (got[0] == NONE).all() and (got[1] == 0).all()
    # a NaN in a greedy row
    case = _case(2, **base, temperature=[0.0, 1.0, 0.0])
    case["target"][0, 599] = float("nan")
    got = _check(case, 2)
    assert got[2] == 4 and (got[0][0] == NONE).all()
    # offsets
    for offsets in ([0, 2, 1, 6], [0, 2, 7, 6], [0, 5, 6, 6], [-1, 2, 4, 6]):
        case = _case(2, **base)
        case["offsets"] = np.asarray(offsets, np.int32)
        got = _check(case, 2)
        assert got[2] == 2


def test_rows_outside_are_left_as_they_are(eng):
    """Through the C entry: the results' own words and no others."""
    import torch

    from pih_amd import abi
    from pih_amd.device import stream_handle
    from pih_amd.linear import _workspace_bytes

    case = _case(6, [3, 1, 2], 777)
    most, drafts, sequences = 5, 6, 3
    dev = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    target, draft = case["target"].cuda(), case["draft"].cuda()
    tokens, offsets, accept, sample = (dev(case[n]) for n in ("tokens", "offsets", "accept", "sample"))
    out = torch.full((sequences * (most + 1) + 16,), 12345, dtype=torch.int32, device="cuda")
    accepted = torch.full((sequences + 16,), 12345, dtype=torch.int32, device="cuda")
    need = _workspace_bytes(abi.WORKSPACE_DRAFT_VERIFY, sequences, most, 777)
    ws = torch.full((need + 64,), 77, dtype=torch.uint8, device="cuda")
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    r = abi.request(abi.LN["draft_verify"], target_logits=target.data_ptr(), draft_logits=draft.data_ptr(),
                    draft_tokens_u32=tokens.data_ptr(), draft_offsets_u32=offsets.data_ptr(),
                    accept_random_f32=accept.data_ptr(), sample_random_f32=sample.data_ptr(),
                    tokens_u32=out[8:].data_ptr(), accepted_u32=accepted[8:].data_ptr(), workspace=ws.data_ptr(),
                    workspace_bytes=need, error_flag_u32=flag.data_ptr(), stream=stream_handle(),
                    sequence_count=sequences, draft_count=drafts, max_drafts=most, vocab=777, target_stride=777,
                    draft_stride=777, logits_type=abi.OUTPUT_F32)
    assert abi.linear_pack().call("launch_draft_verify", r).code == abi.OK
    torch.cuda.synchronize()
    want = _run(case, most)
    assert out[8:8 + 18].cpu().numpy().reshape(3, 6).tolist() == want[0].tolist()
    assert accepted[8:11].tolist() == want[1].tolist()
    for t, n in ((out, 18), (accepted, 3)):
        assert torch.all(t[:8] == 12345) and torch.all(t[8 + n:] == 12345)
    assert torch.all(ws[need:] == 77)


def test_the_tokens_are_distributed_as_the_targets(eng):
    """16384 sequences of one draft over 6 tokens: the first token put out has
    the target's probabilities, within 5 standard deviations."""
    import numpy as np
    import torch

    from pih_amd.linear import draft_verify

    n, rng = 16384, np.random.default_rng(77)
    p, q = rng.normal(size=6) * 1.5, rng.normal(size=6) * 1.5
    target = torch.from_numpy(np.tile(p.astype(np.float32), (2 * n, 1))).cuda()
    draft = torch.from_numpy(np.tile(q.astype(np.float32), (n, 1))).cuda()
    dev = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    drawn = rng.choice(6, size=n, p=_softmax(q.astype(np.float32), 1.0)).astype(np.int32)
    tokens, accepted, flag = draft_verify(target, dev(drawn), dev(np.arange(n + 1, dtype=np.int32)),
                                          dev(rng.random(n, np.float32)), dev(rng.random(n, np.float32)), 1,
                                          draft_logits=draft)
    got = np.bincount(tokens[:, 0].cpu().numpy(), minlength=6) / n
    want = _softmax(p.astype(np.float32), 1.0)
    assert int(flag.item()) == 0 and 0 < accepted.sum().item() < n
    assert (np.abs(got - want) <= 5 * np.sqrt(want * (1 - want) / n)).all(), (got, want)


def test_captured_and_beside_another_call(eng):
    """Two graphs, replayed in turn with an eager call, each on its own
    workspace; offsets change between replays."""
    import numpy as np
    import torch

    from pih_amd.device import engine_stream
    from pih_amd.linear import draft_verify

    cases = [_case(s, c, 5003, temperature=[1.0, 0.0, 0.8]) for s, c in ((1, [4, 1, 2]), (2, [0, 4, 3]), (3, [3, 3, 1]))]
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    make = lambda c: [c["target"].cuda(), dev(c["tokens"]), dev(c["offsets"]), dev(c["accept"]),  # noqa: E731
                      dev(c["sample"]), c["draft"].cuda(), dev(c["temperature"])]
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")

    def call(t):
        return draft_verify(*t[:5], 4, draft_logits=t[5], temperature=t[6], flag=flag)[:2]

    with engine_stream() as s:
        inputs = [make(c) for c in cases]
        static = [[t.clone() for t in inputs[0]] for _ in range(2)]
        graphs, outs = [], []
        call(static[0])
        torch.cuda.synchronize()
        for t in static:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                outs.append(call(t))
            graphs.append(g)
        for a, b in ((0, 1), (1, 2), (2, 0), (0, 0)):
            for t, i in zip(static, (a, b)):
                for x, y in zip(t, inputs[i]):
                    x.copy_(y)
            graphs[0].replay()
            eager = call(inputs[b])
            graphs[1].replay()
            torch.cuda.synchronize()
            for o, i in zip(outs, (a, b)):
                want = call(inputs[i])
                torch.cuda.synchronize()
                assert all(torch.equal(x, y) for x, y in zip(o, want))
            assert all(torch.equal(x, y) for x, y in zip(eager, outs[1]))
    assert int(flag.item()) == 0


def test_rows_past_4_gib(eng):
    """Logits of more than 2^32 bytes: the last sequences' rows lie behind."""
    import torch

    from pih_amd.linear import draft_verify

    vocab, sequences, most = 151936, 7200, 0
    target = torch.zeros(sequences, vocab, dtype=torch.float32, device="cuda")
    assert target.numel() * 4 > 1 << 32
    best = (torch.arange(sequences, device="cuda") * 7919) % vocab
    target.scatter_(1, best[:, None], 100.0)
    empty = torch.zeros(0, dtype=torch.int32, device="cuda")
    tokens, accepted, flag = draft_verify(target, empty, torch.zeros(sequences + 1, dtype=torch.int32, device="cuda"),
                                          empty.float(), torch.full((sequences,), 0.5, device="cuda"), most)
    assert int(flag.item()) == 0 and torch.equal(tokens[:, 0].long(), best) and torch.all(accepted == 0)


def test_results_between_strided_rows(eng):
    """The tokens and counts in the columns behind the logits of a wider tensor."""
    import torch

    from pih_amd import abi, linear
    from pih_amd.device import error_flag, stream_handle

    most, vocab = 4, 100
    case = _case(31, [3, 0, 4], vocab, soft=False)
    target = case["target"].cuda()
    tokens, offsets, accept, sample = (torch.from_numpy(case[n]).cuda() for n in ("tokens", "offsets", "accept", "sample"))
    drafts, sequences = tokens.shape[0], sample.shape[0]
    want = linear.draft_verify(target, tokens, offsets, accept, sample, most)
    wide = torch.zeros(drafts + sequences, 200, device="cuda")
    wide[:, :vocab] = target
    out, count = wide[0, vocab:].view(torch.int32), wide[1, vocab:].view(torch.int32)
    flag = error_flag()
    ws = linear._workspace(abi.WORKSPACE_DRAFT_VERIFY, sequences, most, vocab, target.device)
    linear._launch("launch_draft_verify", "draft_verify", wide.data_ptr(), 0,
                   *(t.data_ptr() for t in (tokens, offsets, accept, sample)), 0, out.data_ptr(), count.data_ptr(),
                   ws.data_ptr(), ws.numel(), flag.data_ptr(), stream_handle(), sequences, drafts, most, vocab, 200, 0,
                   abi.OUTPUT_F32)
    torch.cuda.synchronize()
    assert int(flag.item()) == 0 and torch.equal(wide[:, :vocab], target)
    assert torch.equal(out[:sequences * (most + 1)].view(sequences, most + 1), want[0])
    assert torch.equal(count[:sequences], want[1])
