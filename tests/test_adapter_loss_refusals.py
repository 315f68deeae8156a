"""What the adapter, LM-head-loss and router-balance entries refuse before any
launch: null arguments, shapes, strides, alignments and workspaces (no device
work; the addresses are never read)."""
import ctypes as C

import pytest

from pih_amd import abi


def _query(kind, m, n, k):
    out = (C.c_uint64 * 1)()
    q = abi.request(abi.LN["workspace_query"], kind=kind, m=m, n=n, k=k, bytes_u64=C.addressof(out))
    st = abi.linear_pack().call("query_workspace", q)
    return st.code, int(out[0])


def _fill(name, **fields):
    """A request whose addresses are set and whose shape is right."""
    r = abi.request(abi.LN[name])
    for f, t in r._fields_:
        if t is abi.UPTR:
            setattr(r, f, 0x10000)
    for f, v in fields.items():
        setattr(r, f, v)
    return r


def _adapter_gemm(**over):
    f = dict(workspace_bytes=1 << 40, row_count=33, segment_count=2, adapter_count=3, rank=16, n=64, k=128,
             input_stride=128, base_stride=64, output_stride=64)
    f.update(over)
    return "launch_adapter_gemm", _fill("adapter_gemm", **f)


def _adapter_backward(**over):
    f = dict(workspace_bytes=1 << 40, row_count=33, segment_count=2, adapter_count=3, rank=16, n=64, k=128,
             output_grad_stride=64, input_stride=128, base_stride=128, input_grad_stride=128, input_bf16=0x20000,
             output_grad_bf16=0x30000)
    f.update(over)
    return "launch_adapter_backward", _fill("adapter_backward", **f)


def _loss(**over):
    f = dict(workspace_bytes=1 << 40, rows=5, vocab=100, hidden=64)
    f.update(over)
    return "launch_lm_head_loss", _fill("lm_head_loss", **f)


def _loss_backward(**over):
    f = dict(workspace_bytes=1 << 40, rows=5, vocab=100, hidden=64, weight_bf16=0x20000)
    f.update(over)
    return "launch_lm_head_loss_backward", _fill("lm_head_loss_backward", **f)


def _balance(**over):
    f = dict(workspace_bytes=1 << 40, token_count=5, expert_count=64, top_k=4, mode=1, coefficient=0.01)
    f.update(over)
    return "launch_router_balance", _fill("router_balance", **f)


def _router_backward(**over):
    f = dict(token_count=5, expert_count=64, top_k=4, mode=1, coefficient=0.01, route_scale=1.0)
    f.update(over)
    return "launch_router_backward", _fill("router_backward", **f)


NAN, INF = float("nan"), float("inf")
SHAPE = ("row_count", "segment_count", "adapter_count", "rank", "n", "k")
BAD = []
for make in (_adapter_gemm, _adapter_backward):
    BAD += [(make, {f: 0}) for f in SHAPE + ("workspace_bytes", "stream", "error_flag_u32", "segment_offsets_u32",
                                             "segment_adapter_u32", "input_bf16", "a_bf16", "b_bf16", "workspace")]
    BAD += [(make, {"rank": 12}), (make, {"rank": 136}), (make, {"n": 60}), (make, {"k": 100}),
            (make, {"row_count": 1 << 31}), (make, {"adapter_count": 1 << 15}), (make, {"n": (1 << 20) + 8}),
            (make, {"k": (1 << 20) + 8}), (make, {"input_stride": 120}), (make, {"input_stride": 132}),
            (make, {"base_stride": 56}), (make, {"base_stride": 132}), (make, {"input_bf16": 0x10008}),
            (make, {"a_bf16": 0x10008}), (make, {"b_bf16": 0x10002}), (make, {"base_bf16": 0x10008}),
            (make, {"scale_f32": 0x10002}), (make, {"segment_offsets_u32": 0x10001}), (make, {"workspace": 0x10008})]
BAD += [(_adapter_gemm, {f: v}) for f, v in (("output_bf16", 0), ("output_stride", 56), ("output_stride", 68),
                                             ("output_bf16", 0x10008), ("base_stride", 72))]
BAD += [(_adapter_backward, {f: v}) for f, v in
        (("output_grad_bf16", 0), ("input_grad_bf16", 0), ("a_grad_f32", 0), ("b_grad_f32", 0),
         ("output_grad_stride", 56), ("input_grad_stride", 120), ("a_grad_f32", 0x10008), ("b_grad_f32", 0x10004),
         ("base_stride", 136))]
for make in (_loss, _loss_backward):
    BAD += [(make, {f: 0}) for f in ("rows", "vocab", "hidden", "input_bf16", "weight_bf16", "target_u32", "lse_f32",
                                     "workspace", "workspace_bytes", "error_flag_u32", "stream")]
    BAD += [(make, {"hidden": 60}), (make, {"input_bf16": 0x10008}), (make, {"weight_bf16": 0x10008}),
            (make, {"target_u32": 0x10002}), (make, {"lse_f32": 0x10002}), (make, {"workspace": 0x10008}),
            (make, {"rows": (1 << 20) + 1}), (make, {"vocab": (1 << 20) + 1}), (make, {"hidden": (1 << 20) + 8})]
BAD += [(_loss, {"loss_f32": 0}), (_loss, {"loss_f32": 0x10002}), (_loss_backward, {"loss_grad_f32": 0}),
        (_loss_backward, {"input_grad_bf16": 0}), (_loss_backward, {"input_grad_bf16": 0x10008}),
        (_loss_backward, {"weight_grad_bf16": 0x10008})]
for make in (_balance, _router_backward):
    BAD += [(make, {f: 0}) for f in ("token_count", "expert_count", "top_k", "mode", "scores_f32", "topk_ids_u32",
                                     "error_flag_u32", "stream")]
    BAD += [(make, {"mode": 3}), (make, {"expert_count": 1025}), (make, {"top_k": 33}),
            (make, {"expert_count": 3}), (make, {"coefficient": NAN}), (make, {"coefficient": INF})]
BAD += [(_balance, {f: 0}) for f in ("loss_f32", "counts_u32", "mean_affinity_f32", "workspace", "workspace_bytes")]
BAD += [(_router_backward, f) for f in ({"scores_grad_f32": 0}, {"counts_u32": 0},
                                        {"loss_grad_f32": 0, "topk_weights_grad_f32": 0}, {"route_scale": 0.0},
                                        {"route_scale": -1.0}, {"route_scale": INF})]
# more tokens than the counts hold, rows than a grid has threads, segments than
# a block's search ends in; addresses between two words; results over inputs
BAD += [(make, {"token_count": 1 << 27}) for make in (_balance, _router_backward)]
BAD += [(make, {f: v}) for make in (_adapter_gemm, _adapter_backward)
        for f, v in (("row_count", (1 << 26) + 1), ("segment_count", (1 << 16) + 1))]
BAD += [(_balance, {f: 0x10002}) for f in ("scores_f32", "topk_ids_u32", "loss_f32", "counts_u32", "mean_affinity_f32",
                                           "error_flag_u32")]
BAD += [(_router_backward, {f: 0x10002}) for f in ("scores_f32", "topk_ids_u32", "counts_u32", "loss_grad_f32",
                                                   "topk_weights_grad_f32", "scores_grad_f32", "error_flag_u32")]
BAD += [(_adapter_backward, {"input_grad_bf16": 0x20000, "base_bf16": 0}),
        (_adapter_backward, {"input_grad_bf16": 0x30000, "base_bf16": 0}),
        (_loss_backward, {"weight_grad_bf16": 0x20000})]


@pytest.mark.parametrize("make,over", BAD, ids=lambda v: v.__name__ if callable(v) else str(v))
def test_refused(make, over):
    entry, r = make(**over)
    st = abi.linear_pack().call(entry, r)
    assert st.code == abi.INVALID_ARGUMENT, st


def test_workspace_one_byte_short():
    code, need = _query(abi.WORKSPACE_ADAPTER_GEMM, 33, 16, 128)
    assert code == abi.OK and need > 0
    entry, r = _adapter_gemm(workspace_bytes=need - 1)
    assert abi.linear_pack().call(entry, r).code == abi.INVALID_ARGUMENT
    for make, kind in ((_loss, abi.WORKSPACE_LM_HEAD_LOSS), (_loss_backward, abi.WORKSPACE_LM_HEAD_LOSS_BACKWARD)):
        code, need = _query(kind, 5, 100, 64)
        assert code == abi.OK and need > 0
        entry, r = make(workspace_bytes=need - 1)
        assert abi.linear_pack().call(entry, r).code == abi.INVALID_ARGUMENT
    code, need = _query(abi.WORKSPACE_ROUTER_BALANCE, 5, 4, 64)
    assert code == abi.OK and need > 0
    entry, r = _balance(workspace_bytes=need - 1)
    assert abi.linear_pack().call(entry, r).code == abi.INVALID_ARGUMENT
    out = (C.c_uint64 * 1)()
    _, r = _adapter_backward(required_bytes_u64=C.addressof(out))
    assert abi.linear_pack().call("query_adapter_backward_workspace", r).code == abi.OK and out[0] > 0
    r.workspace_bytes = out[0] - 1
    assert abi.linear_pack().call("launch_adapter_backward", r).code == abi.INVALID_ARGUMENT


@pytest.mark.parametrize("kind,shape", [(abi.WORKSPACE_ADAPTER_GEMM, (0, 16, 128)),
                                        (abi.WORKSPACE_ADAPTER_GEMM, (4, 200, 128)),
                                        (abi.WORKSPACE_LM_HEAD_LOSS, (4, 0, 64)),
                                        (abi.WORKSPACE_LM_HEAD_LOSS, (4, 10, 60)),
                                        (abi.WORKSPACE_LM_HEAD_LOSS_BACKWARD, (0, 10, 64)),
                                        (abi.WORKSPACE_ROUTER_BALANCE, (4, 9, 8)),
                                        (abi.WORKSPACE_ROUTER_BALANCE, (1 << 27, 4, 8)),
                                        (abi.WORKSPACE_ADAPTER_GEMM, ((1 << 26) + 1, 16, 128))])
def test_workspace_query_refuses_shapes(kind, shape):
    assert _query(kind, *shape)[0] == abi.INVALID_ARGUMENT


def test_adapter_backward_query_refuses():
    _, r = _adapter_backward(rank=4, required_bytes_u64=0x10000)
    assert abi.linear_pack().call("query_adapter_backward_workspace", r).code == abi.INVALID_ARGUMENT
    _, r = _adapter_backward(required_bytes_u64=0)
    assert abi.linear_pack().call("query_adapter_backward_workspace", r).code == abi.INVALID_ARGUMENT


def test_python_callers_refuse_host_tensors_and_wrong_types():
    import torch

    from pih_amd import linear

    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    a, b = bf(2, 8, 64), bf(2, 32, 8)
    with pytest.raises(ValueError, match="adapter stacks are A"):
        linear.adapter_gemm(bf(4, 64), a, bf(2, 32, 16), None, i32(2), i32(1), flag=i32(1))
    with pytest.raises(ValueError, match="int32"):
        linear.adapter_gemm(bf(4, 64), a, b, None, i32(3), i32(1), flag=i32(1))
    with pytest.raises(ValueError, match="float32"):
        linear.adapter_gemm(bf(4, 64), a, b, bf(2), i32(2), i32(1), flag=i32(1))
    with pytest.raises(ValueError, match="input is bfloat16"):
        linear.adapter_gemm(bf(4, 72), a, b, None, i32(2), i32(1), flag=i32(1))
    with pytest.raises(ValueError, match="bfloat16"):
        linear.lm_head_loss(torch.zeros(4, 64), bf(10, 64), i32(4), flag=i32(1))
    with pytest.raises(ValueError, match="targets"):
        linear.lm_head_loss(bf(4, 64), bf(10, 64), i32(5), flag=i32(1))
    with pytest.raises(ValueError, match="float32"):
        linear.router_balance(bf(4, 64), i32(4, 2), abi.ROUTER_SOFTMAX, 0.01, flag=i32(1))
    with pytest.raises(ValueError, match="counts"):
        linear.router_backward(torch.zeros(4, 64), i32(4, 2), None, abi.ROUTER_SOFTMAX, 0.01, torch.ones(1),
                               flag=i32(1))


class _Recorded:
    """The linear pack with its launches recorded in place of made."""

    def __init__(self):
        self.table, self.launched = self, []

    def call(self, entry, request):
        return abi.linear_pack().call(entry, request)

    def __getattr__(self, entry):
        def launch(request):
            self.launched.append(entry)
            return abi.Status(struct_size=C.sizeof(abi.Status), abi_version=1, code=abi.OK)
        return launch


@pytest.fixture
def recorded(monkeypatch):
    """Python callers over tensors that have sizes and strides but no memory."""
    from pih_amd import linear

    pack = _Recorded()
    monkeypatch.setattr(linear, "_ln", lambda: pack)
    monkeypatch.setattr(linear, "same_device", lambda *t: None)
    monkeypatch.setattr(linear, "device_ptrs", lambda *t: [0x10000 if v is not None else 0 for v in t])
    monkeypatch.setattr(linear, "stream_handle", lambda: 0x10000)
    linear._entry.cache_clear()
    yield pack
    linear._entry.cache_clear()


def _sizes_past_32_bits():
    import torch

    from pih_amd import linear

    def meta(*shape, dtype=torch.bfloat16, stride=None):
        if stride is None:
            return torch.empty(shape, dtype=dtype, device="meta")
        return torch.empty_strided(shape, (stride, 1), dtype=dtype, device="meta")

    i32, f32 = torch.int32, torch.float32
    a, b, flag, big = meta(2, 8, 64), meta(2, 32, 8), meta(1, dtype=i32), 1 << 32

    def gemm(rows=3, segments=1, x=None, base=None, out=None):
        return lambda: linear.adapter_gemm(meta(rows, 64, stride=x), a, b, None, meta(segments + 1, dtype=i32),
                                           meta(segments, dtype=i32), base=base and meta(rows, 32, stride=base),
                                           out=meta(rows, 32, stride=out or 32), flag=flag)

    def backward(rows=3, dy=None, x=None, base=None, out=None):
        return lambda: linear.adapter_backward(meta(rows, 32, stride=dy), meta(rows, 64, stride=x), a, b, None,
                                               meta(2, dtype=i32), meta(1, dtype=i32),
                                               base=base and meta(rows, 64, stride=base),
                                               out=meta(rows, 64, stride=out or 64), flag=flag)

    def loss(rows, vocab):
        return lambda: linear.lm_head_loss(meta(rows, 64), meta(vocab, 64), meta(rows, dtype=i32), flag=flag)

    def loss_backward(rows, vocab):
        return lambda: linear.lm_head_loss_backward(meta(rows, 64), meta(vocab, 64), meta(rows, dtype=i32),
                                                    meta(rows, dtype=f32), meta(rows, dtype=f32), flag=flag)

    def balance(tokens, mode):
        return lambda: linear.router_balance(meta(tokens, 8, dtype=f32), meta(tokens, 2, dtype=i32), mode, 0.1,
                                             flag=flag)

    def router_backward(tokens, mode):
        return lambda: linear.router_backward(meta(tokens, 8, dtype=f32), meta(tokens, 2, dtype=i32), None, mode, 0.1,
                                              None, dweights=meta(tokens, 2, dtype=f32), flag=flag)

    good = [gemm(x=64, base=32), backward(dy=32, x=64, base=64), loss(3, 5), loss_backward(3, 5), balance(3, 1),
            router_backward(3, 1)]
    bad = [gemm(x=big + 64), gemm(base=big + 40), gemm(out=big + 32), gemm(rows=big + 3), gemm(segments=big + 1),
           backward(dy=big + 32), backward(x=big + 72), backward(base=big + 64), backward(out=big + 64),
           backward(rows=big + 3), loss(big + 3, 5), loss(3, big + 5), loss_backward(big + 3, 5),
           loss_backward(3, big + 5), balance(big + 3, 1), balance(3, big + 1), router_backward(big + 3, 1),
           router_backward(3, big + 1)]
    return good, bad


@pytest.mark.parametrize("case", range(18))
def test_sizes_past_32_bits_are_refused(recorded, case):
    """Sizes and strides whose lower 32 bits alone are valid."""
    good, bad = _sizes_past_32_bits()
    assert len(bad) == 18
    with pytest.raises(ValueError, match="32 bits"):
        bad[case]()
    assert not recorded.launched


def test_sizes_within_32_bits_are_launched(recorded):
    good, _ = _sizes_past_32_bits()
    for call in good:
        call()
    assert len(recorded.launched) == len(good)


@pytest.mark.parametrize("rows,vocab,hidden", [(1, 1, 64), (33, 151936, 1024), (32768, 151936, 1024), (4096, 129281, 4096),
                                               (17, 1000, 72), (4096, 129280, 1000)])
def test_loss_workspace_is_what_is_written(rows, vocab, hidden):
    """A pair of 4-byte words per row and tile, of 256 columns or (hidden no
    multiple of 64) 64, and a word per row, each array in whole 256 bytes."""
    tile = 64 if hidden % 64 else 256
    up = lambda n: (n + 255) // 256 * 256  # noqa: E731
    assert _query(abi.WORKSPACE_LM_HEAD_LOSS, rows, vocab, hidden) == (
        abi.OK, up(rows * ((vocab + tile - 1) // tile) * 8) + up(rows * 4))
