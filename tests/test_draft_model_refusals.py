"""What the feed-forward block, the distillation loss and the verification of
drafted tokens refuse before any launch (no device work; the addresses are
never read)."""
import ctypes as C

import pytest

from pih_amd import abi
from tests.test_adapter_loss_refusals import _fill, _query, recorded  # noqa: F401


def _spread(r):
    """A request's addresses, all different, 16 MB apart."""
    at = 0x1000000
    for f, t in r._fields_:
        if t is abi.UPTR:
            setattr(r, f, at)
            at += 0x1000000
    return r


def _request(name, fields, over):
    r = _spread(_fill(name))
    for f, v in {**fields, **over}.items():
        setattr(r, f, getattr(r, v) if isinstance(v, str) else v)
    return r


def _mlp(**over):
    return "launch_gated_mlp", _request("gated_mlp", dict(workspace_bytes=1 << 40, rows=5, hidden=64, intermediate=128,
                                                          limit=0.0), over)


def _mlp_backward(**over):
    return "launch_gated_mlp_backward", _request("gated_mlp_backward", dict(
        workspace_bytes=1 << 40, rows=5, hidden=64, intermediate=128, limit=10.0), over)


def _distill(**over):
    return "launch_lm_head_distill", _request("lm_head_distill", dict(
        workspace_bytes=1 << 40, rows=5, vocab=100, hidden=64, top_k=4, temperature=1.0), over)


def _distill_backward(**over):
    return "launch_lm_head_distill_backward", _request("lm_head_distill_backward", dict(
        workspace_bytes=1 << 40, rows=5, vocab=100, hidden=64, top_k=4, temperature=1.0), over)


def _verify(**over):
    return "launch_draft_verify", _request("draft_verify", dict(
        workspace_bytes=1 << 40, sequence_count=3, draft_count=7, max_drafts=4, vocab=100, target_stride=100,
        draft_stride=100, logits_type=abi.OUTPUT_F32), over)


NAN, INF = float("nan"), float("inf")
BAD = []
for make in (_mlp, _mlp_backward):
    BAD += [(make, {f: 0}) for f in ("rows", "hidden", "intermediate", "input_bf16", "gate_weight_bf16",
                                     "up_weight_bf16", "down_weight_bf16", "workspace", "workspace_bytes", "stream")]
    BAD += [(make, {"hidden": 60}), (make, {"intermediate": 100}), (make, {"rows": (1 << 20) + 1}),
            (make, {"hidden": (1 << 17) + 8}), (make, {"intermediate": (1 << 17) + 8}), (make, {"limit": NAN}),
            (make, {"limit": INF}), (make, {"limit": -INF}), (make, {"gate_bf16": 0}), (make, {"up_bf16": 0})]
    BAD += [(make, {f: 0x1000008}) for f in ("input_bf16", "gate_weight_bf16", "up_weight_bf16", "down_weight_bf16",
                                             "gate_bf16", "up_bf16", "workspace")]
BAD += [(_mlp, {"output_bf16": 0}), (_mlp, {"output_bf16": 0x1000008}), (_mlp, {"output_bf16": "input_bf16"}),
        (_mlp, {"gate_bf16": "up_bf16"}), (_mlp, {"gate_bf16": "input_bf16"}), (_mlp, {"up_bf16": "output_bf16"})]
GRADS = ("input_grad_bf16", "gate_weight_grad_bf16", "up_weight_grad_bf16", "down_weight_grad_bf16")
BAD += [(_mlp_backward, {"output_grad_bf16": 0}), (_mlp_backward, {"output_grad_bf16": 0x1000008}),
        (_mlp_backward, {f: 0 for f in GRADS})]
BAD += [(_mlp_backward, {f: 0x1000008}) for f in GRADS]
BAD += [(_mlp_backward, {f: g}) for f, g in zip(GRADS, ("output_grad_bf16", "gate_weight_bf16", "gate_bf16",
                                                        "down_weight_bf16"))]
BAD += [(_mlp_backward, {"gate_weight_grad_bf16": "up_weight_grad_bf16"})]
for make in (_distill, _distill_backward):
    BAD += [(make, {f: 0}) for f in ("rows", "vocab", "hidden", "top_k", "temperature", "input_bf16", "weight_bf16",
                                     "teacher_ids_u32", "teacher_logits_f32", "lse_f32", "logits_f32", "workspace",
                                     "workspace_bytes", "error_flag_u32", "stream")]
    BAD += [(make, {"hidden": 60}), (make, {"rows": (1 << 20) + 1}), (make, {"vocab": (1 << 20) + 1}),
            (make, {"hidden": (1 << 20) + 8}), (make, {"top_k": 257}), (make, {"temperature": -1.0}),
            (make, {"temperature": NAN}), (make, {"temperature": INF}), (make, {"temperature": 1e-45})]
    BAD += [(make, {f: 0x1000008}) for f in ("input_bf16", "weight_bf16", "workspace")]
    BAD += [(make, {f: 0x1000002}) for f in ("teacher_ids_u32", "teacher_logits_f32", "teacher_lse_f32", "lse_f32",
                                             "logits_f32", "error_flag_u32")]
BAD += [(_distill, {"loss_f32": 0}), (_distill, {"loss_f32": 0x1000002}), (_distill, {"logits_f32": "teacher_logits_f32"}),
        (_distill, {"logits_f32": "teacher_ids_u32"}), (_distill, {"logits_f32": "teacher_lse_f32"}),
        (_distill_backward, {"loss_grad_f32": 0}), (_distill_backward, {"loss_grad_f32": 0x1000002}),
        (_distill_backward, {"input_grad_bf16": 0}), (_distill_backward, {"input_grad_bf16": 0x1000008}),
        (_distill_backward, {"weight_grad_bf16": 0x1000008}), (_distill_backward, {"weight_grad_bf16": "weight_bf16"})]
BAD += [(_verify, {f: 0}) for f in ("target_logits", "draft_tokens_u32", "draft_offsets_u32", "accept_random_f32",
                                    "sample_random_f32", "tokens_u32", "accepted_u32", "workspace", "workspace_bytes",
                                    "error_flag_u32", "stream", "sequence_count", "vocab", "target_stride",
                                    "logits_type")]
BAD += [(_verify, f) for f in ({"sequence_count": (1 << 14) + 1}, {"max_drafts": 256}, {"vocab": (1 << 20) + 1},
                               {"draft_count": (1 << 20) + 1}, {"target_stride": 99}, {"draft_stride": 99},
                               {"logits_type": 3}, {"tokens_u32": "draft_tokens_u32"},
                               {"accepted_u32": "draft_offsets_u32"}, {"tokens_u32": "accepted_u32"},
                               {"workspace": 0x1000008}, {"target_logits": 0x1000002}, {"draft_logits": 0x1000002},
                               {"target_logits": 0x1000001, "logits_type": abi.OUTPUT_BF16},
                               # more blocks than a grid has threads for
                               {"sequence_count": 1 << 14, "max_drafts": 255, "vocab": 1 << 20,
                                "target_stride": 1 << 20, "draft_stride": 1 << 20})]
BAD += [(_verify, {f: 0x1000002}) for f in ("draft_tokens_u32", "draft_offsets_u32", "accept_random_f32",
                                            "sample_random_f32", "temperature_f32", "tokens_u32", "accepted_u32",
                                            "error_flag_u32")]


@pytest.mark.parametrize("make,over", BAD, ids=lambda v: v.__name__ if callable(v) else str(v))
def test_refused(make, over):
    entry, r = make(**over)
    st = abi.linear_pack().call(entry, r)
    assert st.code == abi.INVALID_ARGUMENT, st


KINDS = ((_mlp, abi.WORKSPACE_GATED_MLP, (5, 128, 64)), (_mlp_backward, abi.WORKSPACE_GATED_MLP_BACKWARD, (5, 128, 64)),
         (_distill, abi.WORKSPACE_LM_HEAD_DISTILL, (5, 100, 64)),
         (_distill_backward, abi.WORKSPACE_LM_HEAD_DISTILL_BACKWARD, (5, 100, 64)),
         (_verify, abi.WORKSPACE_DRAFT_VERIFY, (3, 4, 100)))


@pytest.mark.parametrize("make,kind,shape", KINDS)
def test_workspace_one_byte_short(make, kind, shape):
    code, need = _query(kind, *shape)
    assert code == abi.OK and need > 0
    entry, r = make(workspace_bytes=need - 1)
    st = abi.linear_pack().call(entry, r)
    assert st.code == abi.INVALID_ARGUMENT and b"workspace" in st.message


@pytest.mark.parametrize("kind,shape", [(abi.WORKSPACE_GATED_MLP, (0, 128, 64)), (abi.WORKSPACE_GATED_MLP, (5, 100, 64)),
                                        (abi.WORKSPACE_GATED_MLP_BACKWARD, (5, 128, 60)),
                                        (abi.WORKSPACE_GATED_MLP_BACKWARD, ((1 << 20) + 1, 128, 64)),
                                        (abi.WORKSPACE_LM_HEAD_DISTILL, (5, 0, 64)),
                                        (abi.WORKSPACE_LM_HEAD_DISTILL_BACKWARD, (5, 100, 60)),
                                        (abi.WORKSPACE_DRAFT_VERIFY, (0, 4, 100)),
                                        (abi.WORKSPACE_DRAFT_VERIFY, (3, 256, 100)),
                                        (abi.WORKSPACE_DRAFT_VERIFY, (3, 4, 0))])
def test_workspace_query_refuses_shapes(kind, shape):
    assert _query(kind, *shape)[0] == abi.INVALID_ARGUMENT


def test_python_callers_refuse_wrong_types():
    import torch

    from pih_amd import linear

    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    f32 = torch.zeros
    with pytest.raises(ValueError, match="bfloat16"):
        linear.gated_mlp(f32(4, 64), bf(128, 64), bf(128, 64), bf(64, 128))
    with pytest.raises(ValueError, match="weights are gate"):
        linear.gated_mlp(bf(4, 64), bf(128, 64), bf(136, 64), bf(64, 128))
    with pytest.raises(ValueError, match="weights are gate"):
        linear.gated_mlp(bf(4, 64), bf(128, 64), bf(128, 64), bf(128, 64))
    with pytest.raises(ValueError, match="output is"):
        linear.gated_mlp(bf(4, 64), bf(128, 64), bf(128, 64), bf(64, 128), out=bf(4, 128))
    args = (bf(4, 64), bf(4, 64), bf(128, 64), bf(128, 64), bf(64, 128))
    with pytest.raises(ValueError, match="gate and up"):
        linear.gated_mlp_backward(*args, bf(4, 128), bf(5, 128))
    with pytest.raises(ValueError, match="upstream"):
        linear.gated_mlp_backward(bf(5, 64), *args[1:], bf(4, 128), bf(4, 128))
    with pytest.raises(ValueError, match="entries"):
        linear.lm_head_distill(bf(4, 64), bf(10, 64), i32(4, 3), f32(4, 2))
    with pytest.raises(ValueError, match="entries"):
        linear.lm_head_distill(bf(4, 64), bf(10, 64), i32(5, 3), f32(5, 3))
    with pytest.raises(ValueError, match="teacher_lse"):
        linear.lm_head_distill(bf(4, 64), bf(10, 64), i32(4, 3), f32(4, 3), teacher_lse=f32(3))
    with pytest.raises(ValueError, match="logits are float32"):
        linear.lm_head_distill_backward(bf(4, 64), bf(10, 64), i32(4, 3), f32(4, 3), f32(4), f32(4, 2), f32(4))
    good = dict(target_logits=f32(5, 9), draft_tokens=i32(3), draft_offsets=i32(3), accept_random=f32(3),
                sample_random=f32(2), max_drafts=2)
    for over, what in (({"target_logits": torch.zeros(5, 9, dtype=torch.float16)}, "float32 or bfloat16"),
                       ({"target_logits": f32(4, 9)}, "target's logits"), ({"draft_logits": bf(3, 9)}, "draft model"),
                       ({"draft_logits": f32(4, 9)}, "draft model"), ({"accept_random": f32(2)}, "random"),
                       ({"temperature": f32(3)}, "temperatures"), ({"max_drafts": -1}, "max_drafts"),
                       ({"draft_offsets": i32(1)}, "offsets"),
                       ({"target_logits": torch.zeros(9, 5).T}, "contiguous")):
        with pytest.raises(ValueError, match=what):
            linear.draft_verify(**{**good, **over})


def _past_32_bits():
    import torch

    from pih_amd import linear

    def meta(*shape, dtype=torch.bfloat16, stride=None):
        if stride is None:
            return torch.empty(shape, dtype=dtype, device="meta")
        return torch.empty_strided(shape, (stride, 1), dtype=dtype, device="meta")

    i32, f32, big = torch.int32, torch.float32, 1 << 32
    flag = meta(1, dtype=i32)

    def mlp(rows, inter):
        return lambda: linear.gated_mlp(meta(rows, 64), meta(inter, 64), meta(inter, 64), meta(64, inter))

    def mlp_backward(rows, inter):
        return lambda: linear.gated_mlp_backward(meta(rows, 64), meta(rows, 64), meta(inter, 64), meta(inter, 64),
                                                 meta(64, inter), meta(rows, inter), meta(rows, inter))

    def distill(rows, vocab):
        return lambda: linear.lm_head_distill(meta(rows, 64), meta(vocab, 64), meta(rows, 4, dtype=i32),
                                              meta(rows, 4, dtype=f32), flag=flag)

    def distill_backward(rows, vocab):
        return lambda: linear.lm_head_distill_backward(
            meta(rows, 64), meta(vocab, 64), meta(rows, 4, dtype=i32), meta(rows, 4, dtype=f32), meta(rows, dtype=f32),
            meta(rows, 4, dtype=f32), meta(rows, dtype=f32), flag=flag)

    def verify(vocab, stride=None, drafts=5, most=4):
        return lambda: linear.draft_verify(
            meta(drafts + 2, vocab, dtype=f32, stride=stride), meta(drafts, dtype=i32), meta(3, dtype=i32),
            meta(drafts, dtype=f32), meta(2, dtype=f32), most, draft_logits=meta(drafts, vocab, dtype=f32), flag=flag)

    good = [mlp(3, 128), mlp_backward(3, 128), distill(3, 5), distill_backward(3, 5), verify(9)]
    bad = [mlp(big + 3, 128), mlp(3, big + 128), mlp_backward(big + 3, 128), mlp_backward(3, big + 128),
           distill(big + 3, 5), distill(3, big + 5), distill_backward(big + 3, 5), distill_backward(3, big + 5),
           verify(big + 9), verify(9, stride=big + 9), verify(9, drafts=big + 5), verify(9, most=big + 4)]
    return good, bad


@pytest.mark.parametrize("case", range(12))
def test_sizes_past_32_bits_are_refused(recorded, case):  # noqa: F811
    good, bad = _past_32_bits()
    assert len(bad) == 12
    with pytest.raises(ValueError, match="32 bits"):
        bad[case]()
    assert not recorded.launched


def test_sizes_within_32_bits_are_launched(recorded):  # noqa: F811
    good, _ = _past_32_bits()
    for call in good:
        call()
    assert len(recorded.launched) == len(good)


def test_table_entries_follow_the_earlier_ones():
    table = abi.LN_API
    last = [n for n, _ in table._fields_][-5:]
    assert last == ["launch_gated_mlp", "launch_gated_mlp_backward", "launch_lm_head_distill",
                    "launch_lm_head_distill_backward", "launch_draft_verify"]
    assert table.launch_gated_mlp.offset == table.launch_router_backward.offset + C.sizeof(C.c_void_p)


def _overlaps():
    """A result that begins inside an input or another result, or ends there."""
    # (rows 5, hidden 64, intermediate 128: 640 bytes of rows, 1280 of gate and up, 16384 of a weight)
    x, inter, weight = 640, 1280, 16384
    out = []

    def pairs(make, results, inputs):
        for i, (r, size) in enumerate(results):
            for other, length in inputs + results[:i]:
                # (multiples of 16 for the rows, of 4 for the u32 and f32 arrays)
                step = 16 if "bf16" in r else 4
                out.extend((make, r, other, d) for d in (0, (length - 1) // step * step, -((size - 1) // step * step)))

    weights = [("gate_weight_bf16", weight), ("up_weight_bf16", weight), ("down_weight_bf16", weight)]
    kept = [("gate_bf16", inter), ("up_bf16", inter)]
    pairs(_mlp, [("output_bf16", x)] + kept, [("input_bf16", x)] + weights)
    pairs(_mlp_backward, [("input_grad_bf16", x)] + [(w.replace("_bf16", "_grad_bf16"), n) for w, n in weights],
          [("output_grad_bf16", x), ("input_bf16", x)] + weights + kept)
    # (5 rows of 4 entries, 100 x 64 weights)
    rows, entries, head = 20, 80, 12800
    teacher = [("teacher_ids_u32", entries), ("teacher_logits_f32", entries)]
    shared = [("input_bf16", x), ("weight_bf16", head)] + teacher
    pairs(_distill, [("loss_f32", rows), ("lse_f32", rows), ("logits_f32", entries)], shared)
    out.extend((_distill, r, "teacher_lse_f32", d) for r, d in
               (("loss_f32", 16), ("loss_f32", -16), ("lse_f32", 4), ("logits_f32", 0), ("logits_f32", -64)))
    pairs(_distill_backward, [("input_grad_bf16", x), ("weight_grad_bf16", head)],
          shared + [("teacher_lse_f32", rows), ("lse_f32", rows), ("logits_f32", entries), ("loss_grad_f32", rows)])
    # (3 sequences, 7 drafts, at most 4 a sequence, 100 columns of fp32)
    pairs(_verify, [("tokens_u32", 60), ("accepted_u32", 12)],
          [("target_logits", 4000), ("draft_logits", 2800), ("draft_tokens_u32", 28), ("draft_offsets_u32", 16),
           ("accept_random_f32", 28), ("sample_random_f32", 12), ("temperature_f32", 12)])
    return out


@pytest.mark.parametrize("make,result,other,offset", _overlaps(), ids=lambda v: v.__name__ if callable(v) else str(v))
def test_overlapping_results_are_refused(make, result, other, offset):
    entry, r = make()
    setattr(r, result, getattr(r, other) + offset)
    st = abi.linear_pack().call(entry, r)
    assert st.code == abi.INVALID_ARGUMENT and b"alias" in st.message, st.message


@pytest.mark.parametrize("offset", [396, 744])
def test_results_that_reach_into_strided_logits_are_refused(offset):
    """Rows 800 bytes apart, of which 400 are logits: 60 bytes of tokens from the
    last logit of a row on, or up to the first of the next (between them:
    test_gpu_draft_verify.py)."""
    entry, r = _verify(target_stride=200)
    r.tokens_u32 = r.target_logits + offset
    st = abi.linear_pack().call(entry, r)
    assert st.code == abi.INVALID_ARGUMENT and b"alias" in st.message, st.message


@pytest.mark.parametrize("make", [_distill, _distill_backward])
@pytest.mark.parametrize("temperature", [2.9e-39, 3.5e-39, 4.2e-39])
def test_temperatures_whose_exponents_have_no_scale_are_refused(make, temperature):
    """1 / T is finite from 2.94e-39 on, log2(e) / T, which the logits' differences
    are multiplied with, from 4.24e-39 on: below, 0 times it would be NaN."""
    entry, r = make(temperature=temperature)
    st = abi.linear_pack().call(entry, r)
    assert st.code == abi.INVALID_ARGUMENT and b"temperature" in st.message, st.message
