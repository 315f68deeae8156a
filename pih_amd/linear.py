"""Python-side callers of the gfx950 pack tables (torch tensors in, torch
tensors out).  Every function goes through the C ABI of the built packs
(``pih_amd.abi``); there is no fallback: a missing pack or a non-OK status
raises.

Layouts (row-major):
  e4m3 codes   uint8 [rows, K], scales fp32 or uint8 (UE8M0) [rows, K/128]
  FP8 weights  uint8 [E, N, K], scales [E, N/128, K/128]
  MXFP4        uint8 [E, N, K/2] (low nibble = even k), UE8M0 [E, N, K/32]
"""
from __future__ import annotations

import functools
from typing import Optional, Tuple

import torch

from . import abi
from .device import device_ptrs, error_flag, ptr, same_device, stream_handle


class KernelError(RuntimeError):
    pass


def _check(status: abi.Status, what: str) -> None:
    if status.code != abi.OK:
        raise KernelError(f"{what}: {status!r}")


def _ln():
    return abi.linear_pack()


def _ds():
    return abi.deepseek_pack()


# ------------------------------------------------------------ route plan
def route_plan_workspace(tokens: int, topk: int, experts: int) -> int:
    out = (abi.C.c_uint64 * 1)()
    q = abi.request(abi.LN["workspace_query"], kind=abi.WORKSPACE_ROUTE_PLAN, m=tokens, n=topk, k=experts,
                    bytes_u64=abi.C.addressof(out))
    _check(_ln().call("query_workspace", q), "query_workspace")
    return int(out[0])


def bf16_gemm_workspace(m: int, n: int, k: int) -> int:
    """Scratch bytes launch_bf16_gemm can use at this shape (query_workspace;
    0: none).  A call that runs on the per-shape tiles leaves them alone."""
    out = (abi.C.c_uint64 * 1)()
    q = abi.request(abi.LN["workspace_query"], kind=abi.WORKSPACE_BF16_GEMM, m=m, n=n, k=k,
                    bytes_u64=abi.C.addressof(out))
    _check(_ln().call("query_workspace", q), "query_workspace")
    return int(out[0])


def route_plan(topk_ids: torch.Tensor, topk_weights: torch.Tensor, experts: int,
               flag: Optional[torch.Tensor] = None):
    """Returns (expert_offsets [E+1], row_token [R], row_weight [R],
    token_rows [T, k], flag)."""
    tokens, topk = topk_ids.shape
    dev = topk_ids.device
    ws = torch.empty(route_plan_workspace(tokens, topk, experts), dtype=torch.uint8, device=dev)
    offsets = torch.empty(experts + 1, dtype=torch.int32, device=dev)
    row_token = torch.empty(tokens * topk, dtype=torch.int32, device=dev)
    row_weight = torch.empty(tokens * topk, dtype=torch.float32, device=dev)
    token_rows = torch.empty(tokens, topk, dtype=torch.int32, device=dev)
    flag = error_flag() if flag is None else flag
    r = abi.request(abi.LN["route_plan"], topk_ids_u32=ptr(topk_ids), topk_weights_f32=ptr(topk_weights),
                    expert_offsets_u32=ptr(offsets), row_token_u32=ptr(row_token),
                    row_weight_f32=ptr(row_weight), token_rows_u32=ptr(token_rows), workspace=ptr(ws),
                    workspace_bytes=ws.numel(), error_flag_u32=ptr(flag), stream=stream_handle(),
                    token_count=tokens, top_k=topk, expert_count=experts)
    _check(_ln().call("launch_route_plan", r), "route_plan")
    return offsets, row_token, row_weight, token_rows, flag


def router_topk(scores: torch.Tensor, topk: int, mode: int, route_scale: float = 1.0,
                bias: Optional[torch.Tensor] = None, flag: Optional[torch.Tensor] = None,
                out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None):
    """Raw router scores f32 [T, E] -> (topk_ids int32 [T, k], topk_weights
    f32 [T, k], flag) on the device (``launch_router_topk``): softmax top-k
    renormalised (abi.ROUTER_SOFTMAX) or the V4 learned router's
    sqrt-softplus + bias selection (abi.ROUTER_SQRT_SOFTPLUS)."""
    tokens, experts = scores.shape
    if out is None:
        out = (torch.empty(tokens, topk, dtype=torch.int32, device=scores.device),
               torch.empty(tokens, topk, dtype=torch.float32, device=scores.device))
    ids, wts = out
    flag = error_flag() if flag is None else flag
    r = abi.request(abi.LN["router_topk"], scores_f32=ptr(scores), bias_f32=ptr(bias), topk_ids_u32=ptr(ids),
                    topk_weights_f32=ptr(wts), error_flag_u32=ptr(flag), stream=stream_handle(),
                    token_count=tokens, expert_count=experts, top_k=topk, mode=mode, route_scale=route_scale)
    _check(_ln().call("launch_router_topk", r), "router_topk")
    return ids, wts, flag


# ------------------------------------------------------------- FP8 quant
def fp8_quant(x: torch.Tensor, scale_format: int, rows: Optional[torch.Tensor] = None,
              flag: Optional[torch.Tensor] = None):
    """bf16 [R, K] (or gathered via rows) -> (codes uint8, scales, flag)."""
    n_out = x.shape[0] if rows is None else rows.numel()
    k = x.shape[1]
    codes = torch.empty(n_out, k, dtype=torch.uint8, device=x.device)
    sdt = torch.float32 if scale_format == abi.SCALE_F32 else torch.uint8
    scales = torch.empty(n_out, k // 128, dtype=sdt, device=x.device)
    flag = error_flag() if flag is None else flag
    r = abi.request(abi.LN["fp8_quant"], input_bf16=ptr(x), row_index_u32=ptr(rows), output_e4m3=ptr(codes),
                    scale=ptr(scales), error_flag_u32=ptr(flag), stream=stream_handle(), row_count=n_out,
                    logical_k=k, input_rows=x.shape[0], scale_format=scale_format)
    _check(_ln().call("launch_fp8_quant", r), "fp8_quant")
    return codes, scales, flag


def fp8_gemm(a, a_scale, w, w_scale, scale_format: int, output_type: int = abi.OUTPUT_BF16,
             flag: Optional[torch.Tensor] = None):
    m, k = a.shape
    n = w.shape[0]
    out = torch.empty(m, n, dtype=torch.bfloat16 if output_type == abi.OUTPUT_BF16 else torch.float32,
                      device=a.device)
    flag = error_flag() if flag is None else flag
    r = abi.request(abi.LN["fp8_gemm"], activation_e4m3=ptr(a), activation_scale=ptr(a_scale),
                    weight_e4m3=ptr(w), weight_scale=ptr(w_scale), output=ptr(out), error_flag_u32=ptr(flag),
                    stream=stream_handle(), m=m, n=n, k=k, scale_format=scale_format, output_type=output_type)
    _check(_ln().call("launch_fp8_gemm", r), "fp8_gemm")
    return out, flag


def moe_fp8_gemm(a, a_scale, row_token, w, w_scale, offsets, rows: int, scale_format: int,
                 output_type: int, row_weight=None, swiglu_limit: float = 0.0,
                 flag: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None):
    """Returns (out, flag); OUTPUT_SWIGLU_E4M3 returns ((codes, scales), flag)."""
    experts, n, k = w.shape
    e4m3 = output_type == abi.OUTPUT_SWIGLU_E4M3
    ncols = n // 2 if output_type in (abi.OUTPUT_SWIGLU_BF16, abi.OUTPUT_SWIGLU_E4M3) else n
    scales = None
    if e4m3:
        out = torch.empty(rows, ncols, dtype=torch.uint8, device=a.device) if out is None else out
        sdt = torch.float32 if scale_format == abi.SCALE_F32 else torch.uint8
        scales = torch.empty(rows, ncols // 128, dtype=sdt, device=a.device)
    elif out is None:
        out = torch.empty(rows, ncols, dtype=torch.float32 if output_type == abi.OUTPUT_F32 else torch.bfloat16,
                          device=a.device)
    flag = error_flag() if flag is None else flag
    r = abi.request(abi.LN["moe_fp8_gemm"], activation_e4m3=ptr(a), activation_scale=ptr(a_scale),
                    row_token_u32=ptr(row_token), weight_e4m3=ptr(w), weight_scale=ptr(w_scale),
                    expert_offsets_u32=ptr(offsets), row_weight_f32=ptr(row_weight), output=ptr(out),
                    error_flag_u32=ptr(flag), stream=stream_handle(), row_capacity=rows, expert_count=experts,
                    n=n, k=k, activation_rows=a.shape[0], scale_format=scale_format, output_type=output_type,
                    swiglu_limit=swiglu_limit, output_scale=ptr(scales))
    _check(_ln().call("launch_moe_fp8_gemm", r), "moe_fp8_gemm")
    return ((out, scales) if e4m3 else out), flag


def moe_mxfp4_gemm(a, a_scale, row_token, w_packed, w_scale, offsets, rows: int, activation_type: int,
                   output_type: int, row_weight=None, swiglu_limit: float = 0.0,
                   flag: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None):
    experts, n, k2 = w_packed.shape
    k = 2 * k2
    ncols = n // 2 if output_type == abi.OUTPUT_SWIGLU_BF16 else n
    if out is None:
        out = torch.empty(rows, ncols, dtype=torch.float32 if output_type == abi.OUTPUT_F32 else torch.bfloat16,
                          device=w_packed.device)
    flag = error_flag() if flag is None else flag
    r = abi.request(abi.LN["moe_mxfp4_gemm"], activation=ptr(a), activation_scale_ue8m0=ptr(a_scale),
                    row_token_u32=ptr(row_token), packed_weight=ptr(w_packed), weight_scale_ue8m0=ptr(w_scale),
                    expert_offsets_u32=ptr(offsets), row_weight_f32=ptr(row_weight), output=ptr(out),
                    error_flag_u32=ptr(flag), stream=stream_handle(), row_capacity=rows, expert_count=experts,
                    n=n, k=k, activation_rows=a.shape[0], activation_type=activation_type,
                    output_type=output_type, swiglu_limit=swiglu_limit)
    _check(_ln().call("launch_moe_mxfp4_gemm", r), "moe_mxfp4_gemm")
    return out, flag


def moe_combine(expert_out, token_rows, shared=None, flag: Optional[torch.Tensor] = None,
                out: Optional[torch.Tensor] = None):
    rows, hidden = expert_out.shape
    tokens, topk = token_rows.shape
    if out is None:
        out = torch.empty(tokens, hidden, dtype=torch.bfloat16, device=expert_out.device)
    flag = error_flag() if flag is None else flag
    r = abi.request(abi.LN["moe_combine"], expert_output_bf16=ptr(expert_out), token_rows_u32=ptr(token_rows),
                    shared_bf16=ptr(shared), output_bf16=ptr(out), error_flag_u32=ptr(flag),
                    stream=stream_handle(), token_count=tokens, top_k=topk, hidden_size=hidden, row_count=rows)
    _check(_ln().call("launch_moe_combine", r), "moe_combine")
    return out, flag


def bf16_gemm(a: torch.Tensor, w: torch.Tensor, output_type: int = abi.OUTPUT_BF16,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """C[m, n] = A[m, k] . W[n, k]^T through ``launch_bf16_gemm`` (the
    GemmPlan::execute replacement, src/backend/cuda/gemm_plan.cpp:169-198):
    bf16 in, fp32 accumulate, bf16 or fp32 out."""
    m, k = a.shape
    n = w.shape[0]
    if out is None:
        out = torch.empty(m, n, dtype=torch.bfloat16 if output_type == abi.OUTPUT_BF16 else torch.float32,
                          device=a.device)
    wsb = bf16_gemm_workspace(m, n, k)
    ws = torch.empty(wsb, dtype=torch.uint8, device=a.device) if wsb else None
    r = abi.request(abi.LN["bf16_gemm"], a_bf16=ptr(a), w_bf16=ptr(w), output=ptr(out),
                    workspace=ptr(ws) if ws is not None else 0, workspace_bytes=wsb, stream=stream_handle(),
                    m=m, n=n, k=k, output_type=output_type)
    _check(_ln().call("launch_bf16_gemm", r), "bf16_gemm")
    return out


def silu_mul(gate: torch.Tensor, up: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """bf16(silu(g) * u) elementwise (pih_qwen_silu_mul_bf16_v1)."""
    if out is None:
        out = torch.empty_like(gate)
    r = abi.request(abi.LN["silu_mul"], gate_bf16=ptr(gate), up_bf16=ptr(up), output_bf16=ptr(out),
                    stream=stream_handle(), count=gate.numel())
    _check(_ln().call("launch_silu_mul", r), "silu_mul")
    return out


class QwenMlpBlock:
    """The Qwen3 MLP block as the reference's model issues it per layer:
    gate = x.Wg^T and up = x.Wu^T (GemmPlan, bf16 out;
    plugins/model-qwen3/qwen3_bf16_execution_schedule.cpp:34-37), then
    silu_mul (qwen3_cpu_oracle.cpp:114-126 semantics), then down = h.Wd^T.
    Buffers and the workspace are allocated at construction and the four
    requests are built once per (input, stream), as a native host holds its
    GemmPlans, so ``forward`` only enqueues."""

    def __init__(self, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, tokens: int):
        self.wg, self.wu, self.wd = w_gate, w_up, w_down
        inter, hidden = w_gate.shape
        dev = w_gate.device
        self.tokens, self.inter, self.hidden = tokens, inter, hidden
        self.gate = torch.empty(tokens, inter, dtype=torch.bfloat16, device=dev)
        self.up = torch.empty(tokens, inter, dtype=torch.bfloat16, device=dev)
        self.h = torch.empty(tokens, inter, dtype=torch.bfloat16, device=dev)
        self.out = torch.empty(tokens, hidden, dtype=torch.bfloat16, device=dev)
        self.ws_gu = bf16_gemm_workspace(tokens, inter, hidden)
        self.ws_d = bf16_gemm_workspace(tokens, hidden, inter)
        wsb = max(self.ws_gu, self.ws_d)
        self.ws = torch.empty(wsb, dtype=torch.uint8, device=dev) if wsb else None
        self._key = None
        self._reqs = None

    def _gemm(self, a, w, out, m, n, k, wsb, s):
        return abi.request(abi.LN["bf16_gemm"], a_bf16=ptr(a), w_bf16=ptr(w), output=ptr(out),
                           workspace=ptr(self.ws) if wsb else 0, workspace_bytes=wsb, stream=s, m=m, n=n, k=k,
                           output_type=abi.OUTPUT_BF16)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape != (self.tokens, self.hidden) or x.dtype != torch.bfloat16:
            raise ValueError("Qwen MLP block input shape is invalid")
        s = stream_handle()
        key = (ptr(x), s)
        if key != self._key:
            t, i, h = self.tokens, self.inter, self.hidden
            self._reqs = (
                self._gemm(x, self.wg, self.gate, t, i, h, self.ws_gu, s),
                self._gemm(x, self.wu, self.up, t, i, h, self.ws_gu, s),
                abi.request(abi.LN["silu_mul"], gate_bf16=ptr(self.gate), up_bf16=ptr(self.up),
                            output_bf16=ptr(self.h), stream=s, count=t * i),
                self._gemm(self.h, self.wd, self.out, t, h, i, self.ws_d, s),
            )
            self._key = key
        ln = _ln()
        g, u, sm, d = self._reqs
        _check(ln.call("launch_bf16_gemm", g), "bf16_gemm")
        _check(ln.call("launch_bf16_gemm", u), "bf16_gemm")
        _check(ln.call("launch_silu_mul", sm), "silu_mul")
        _check(ln.call("launch_bf16_gemm", d), "bf16_gemm")
        return self.out


QWEN_VOCAB, QWEN_HIDDEN = 151936, 1024


class QwenLmHead:
    """The Qwen3-0.6B LM head as the reference's INT4 execution driver runs
    it (plugins/model-qwen3/nvidia_qwen3_int4_execution_driver.cpp:16-67): a
    bank of GemmPlans for 1..maximum_rows rows (at most 32) over the tied
    [151936, 1024] bf16 weight with fp32 logits; ``execute`` rejects a row
    count outside the bank.  Here every row count is the same
    ``launch_bf16_gemm`` call (one row the weight-streaming GEMV, more the 128 x
    256 tiles; no workspace)."""

    def __init__(self, maximum_rows: int):
        if not 1 <= maximum_rows <= 32:
            raise ValueError("NVIDIA Qwen INT4 workspace identity is invalid")
        self.maximum_rows = maximum_rows

    def execute(self, x: torch.Tensor, weight: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
        if x.dim() != 2 or x.shape[0] == 0 or x.shape[0] > self.maximum_rows:
            raise ValueError("NVIDIA Qwen INT4 LM head row count is invalid")
        if tuple(weight.shape) != (QWEN_VOCAB, QWEN_HIDDEN) or x.shape[1] != QWEN_HIDDEN:
            raise ValueError("Qwen LM head shape is invalid")
        return bf16_gemm(x, weight, abi.OUTPUT_F32, out=out)


def deepseek_lm_head(x: torch.Tensor, weight: torch.Tensor, out: Optional[torch.Tensor] = None,
                     flag: Optional[torch.Tensor] = None):
    """logits f32 [rows, 129280] through the DeepSeek table's
    ``launch_lm_head`` (plugins/kernels/deepseek-v4-sm89/native/
    deepseek_endpoint.cu:94-115,484-497): bit 128 of the flag for a
    non-finite logit, bit 64 for a non-finite x or W element."""
    rows, hidden = x.shape
    vocab = weight.shape[0]
    if out is None:
        out = torch.empty(rows, vocab, dtype=torch.float32, device=x.device)
    flag = error_flag() if flag is None else flag
    r = abi.request(abi.DS["lm_head"], input_bf16=ptr(x), weight_bf16=ptr(weight), logits_f32=ptr(out),
                    error_flag_u32=ptr(flag), stream=stream_handle(), output_rows=rows, vocab_size=vocab,
                    hidden_size=hidden)
    _check(abi.deepseek_pack().call("launch_lm_head", r), "lm_head")
    return out, flag


class MoeFp8Layer:
    """The BASELINE FP8 MoE expert layer on device, one launch per stage:
    route plan -> FP8 quant of the token rows -> grouped gate/up GEMM with
    the fused SwiGLU * route-weight epilogue that also quantises the
    intermediate to FP8 (as the quant entry would quantise its bf16 values)
    -> grouped down GEMM -> ordered combine.

    Buffers are allocated once at construction for ``tokens`` x ``topk``
    routes, so ``forward`` allocates nothing and can be timed or replayed.
    The stage order and rounding points are those of the reference's
    routed-expert chain (src/model/deepseek_routed_expert_oracle.cpp:50-95)
    with fp32 scales and a fused [2I, H] gate/up weight."""

    def __init__(self, w13, w13_scale, w2, w2_scale, tokens: int, topk: int, swiglu_limit: float = 0.0,
                 scale_format: int = abi.SCALE_F32):
        self.w13, self.w13_scale, self.w2, self.w2_scale = w13, w13_scale, w2, w2_scale
        self.experts, n13, self.hidden = w13.shape
        self.inter = n13 // 2
        self.tokens, self.topk = tokens, topk
        self.rows = tokens * topk
        self.limit = swiglu_limit
        self.fmt = scale_format
        dev = w13.device
        sdt = torch.float32 if scale_format == abi.SCALE_F32 else torch.uint8
        self.ws = torch.empty(route_plan_workspace(tokens, topk, self.experts), dtype=torch.uint8, device=dev)
        self.offsets = torch.empty(self.experts + 1, dtype=torch.int32, device=dev)
        self.row_token = torch.empty(self.rows, dtype=torch.int32, device=dev)
        self.row_weight = torch.empty(self.rows, dtype=torch.float32, device=dev)
        self.token_rows = torch.empty(tokens, topk, dtype=torch.int32, device=dev)
        self.xq = torch.empty(tokens, self.hidden, dtype=torch.uint8, device=dev)
        self.xs = torch.empty(tokens, self.hidden // 128, dtype=sdt, device=dev)
        self.mq = torch.empty(self.rows, self.inter, dtype=torch.uint8, device=dev)
        self.ms = torch.empty(self.rows, self.inter // 128, dtype=sdt, device=dev)
        self.y = torch.empty(self.rows, self.hidden, dtype=torch.bfloat16, device=dev)
        self.out = torch.empty(tokens, self.hidden, dtype=torch.bfloat16, device=dev)
        self.flag = error_flag()

    STAGES = ("route_plan", "quant_x", "gate_up", "down", "combine")

    def forward(self, x, topk_ids, topk_weights, shared=None, marks=None):
        """``marks``: optional list of len(STAGES)+1 events recorded on the
        launch stream around the stages (for per-kernel timing)."""
        L = _ln()
        s = stream_handle()
        f = ptr(self.flag)
        mark = (lambda i: marks[i].record()) if marks is not None else (lambda i: None)
        mark(0)
        st = L.call("launch_route_plan", abi.request(
            abi.LN["route_plan"], topk_ids_u32=ptr(topk_ids), topk_weights_f32=ptr(topk_weights),
            expert_offsets_u32=ptr(self.offsets), row_token_u32=ptr(self.row_token),
            row_weight_f32=ptr(self.row_weight), token_rows_u32=ptr(self.token_rows), workspace=ptr(self.ws),
            workspace_bytes=self.ws.numel(), error_flag_u32=f, stream=s, token_count=self.tokens,
            top_k=self.topk, expert_count=self.experts))
        _check(st, "route_plan")
        mark(1)
        st = L.call("launch_fp8_quant", abi.request(
            abi.LN["fp8_quant"], input_bf16=ptr(x), row_index_u32=0, output_e4m3=ptr(self.xq), scale=ptr(self.xs),
            error_flag_u32=f, stream=s, row_count=self.tokens, logical_k=self.hidden, input_rows=self.tokens,
            scale_format=self.fmt))
        _check(st, "fp8_quant(x)")
        mark(2)
        st = L.call("launch_moe_fp8_gemm", abi.request(
            abi.LN["moe_fp8_gemm"], activation_e4m3=ptr(self.xq), activation_scale=ptr(self.xs),
            row_token_u32=ptr(self.row_token), weight_e4m3=ptr(self.w13), weight_scale=ptr(self.w13_scale),
            expert_offsets_u32=ptr(self.offsets), row_weight_f32=ptr(self.row_weight), output=ptr(self.mq),
            output_scale=ptr(self.ms), error_flag_u32=f, stream=s, row_capacity=self.rows,
            expert_count=self.experts, n=2 * self.inter, k=self.hidden, activation_rows=self.tokens,
            scale_format=self.fmt, output_type=abi.OUTPUT_SWIGLU_E4M3, swiglu_limit=self.limit))
        _check(st, "moe_fp8_gemm(gate/up)")
        mark(3)
        st = L.call("launch_moe_fp8_gemm", abi.request(
            abi.LN["moe_fp8_gemm"], activation_e4m3=ptr(self.mq), activation_scale=ptr(self.ms),
            row_token_u32=0, weight_e4m3=ptr(self.w2), weight_scale=ptr(self.w2_scale),
            expert_offsets_u32=ptr(self.offsets), row_weight_f32=0, output=ptr(self.y), error_flag_u32=f,
            stream=s, row_capacity=self.rows, expert_count=self.experts, n=self.hidden, k=self.inter,
            activation_rows=self.rows, scale_format=self.fmt, output_type=abi.OUTPUT_BF16, swiglu_limit=0.0))
        _check(st, "moe_fp8_gemm(down)")
        mark(4)
        st = L.call("launch_moe_combine", abi.request(
            abi.LN["moe_combine"], expert_output_bf16=ptr(self.y), token_rows_u32=ptr(self.token_rows),
            shared_bf16=ptr(shared), output_bf16=ptr(self.out), error_flag_u32=f, stream=s,
            token_count=self.tokens, top_k=self.topk, hidden_size=self.hidden, row_count=self.rows))
        _check(st, "moe_combine")
        mark(5)
        return self.out


class MoeLayer:
    """One MoE expert layer per call through the pack's C++ layer entry
    (``launch_moe_layer``): the six stages of ``MoeFp8Layer`` enqueued by the
    native host code, for FP8 or MXFP4 weights.  Scratch is sized once with
    ``query_moe_layer_workspace`` and allocated at construction."""

    def __init__(self, w13, w13_scale, w2, w2_scale, tokens: int, topk: int, weight_format: int = abi.WEIGHT_FP8,
                 scale_format: int = abi.SCALE_F32, activation_type: int = abi.ACTIVATION_E4M3,
                 swiglu_limit: float = 0.0):
        self.w13, self.w13_scale, self.w2, self.w2_scale = w13, w13_scale, w2, w2_scale
        self.experts, n13, k13 = w13.shape
        self.hidden = k13 if weight_format == abi.WEIGHT_FP8 else 2 * k13
        self.inter = n13 // 2
        self.tokens, self.topk = tokens, topk
        self.fields = dict(token_count=tokens, top_k=topk, expert_count=self.experts, hidden_size=self.hidden,
                           intermediate_size=self.inter, weight_format=weight_format, scale_format=scale_format,
                           activation_type=activation_type, swiglu_limit=swiglu_limit)
        need = (abi.C.c_uint64 * 1)()
        q = abi.request(abi.LN["moe_layer"], required_bytes_u64=abi.C.addressof(need), **self.fields)
        _check(_ln().call("query_moe_layer_workspace", q), "query_moe_layer_workspace")
        self.ws = torch.empty(int(need[0]), dtype=torch.uint8, device=w13.device)
        self.out = torch.empty(tokens, self.hidden, dtype=torch.bfloat16, device=w13.device)
        self.flag = error_flag()

    def forward(self, x, topk_ids, topk_weights, shared=None):
        r = abi.request(abi.LN["moe_layer"], input_bf16=ptr(x), topk_ids_u32=ptr(topk_ids),
                        topk_weights_f32=ptr(topk_weights), w13=ptr(self.w13), w13_scale=ptr(self.w13_scale),
                        w2=ptr(self.w2), w2_scale=ptr(self.w2_scale), shared_bf16=ptr(shared),
                        output_bf16=ptr(self.out), workspace=ptr(self.ws), workspace_bytes=self.ws.numel(),
                        error_flag_u32=ptr(self.flag), stream=stream_handle(), **self.fields)
        _check(_ln().call("launch_moe_layer", r), "moe_layer")
        return self.out


# ------------------------------------------------ DeepSeek V4.1 32-block formats
def v41_linear(x: torch.Tensor, weight: torch.Tensor, weight_scales: torch.Tensor, weight_format: int,
               out: Optional[torch.Tensor] = None, quantized: Optional[torch.Tensor] = None,
               activation_scales: Optional[torch.Tensor] = None, flag: Optional[torch.Tensor] = None):
    """The V4.1 FP8 (32x32 weight blocks) or mixed FP8/FP4 linear
    (plugins/model-deepseek-v41/linear_fp8.cu:82-105) through
    ``launch_v41_linear``: per-32 activation quant into ``quantized`` /
    ``activation_scales`` (allocated when None), then the MX GEMM; returns
    (out bf16 [rows, N], quantized, activation_scales, flag)."""
    rows, k = x.shape
    n = weight.shape[0]
    dev = x.device
    if out is None:
        out = torch.empty(rows, n, dtype=torch.bfloat16, device=dev)
    if quantized is None:
        quantized = torch.empty(rows, k, dtype=torch.uint8, device=dev)
    if activation_scales is None:
        activation_scales = torch.empty(rows, k // 32, dtype=torch.uint8, device=dev)
    flag = error_flag() if flag is None else flag
    nbytes = lambda t: t.numel() * t.element_size()  # noqa: E731
    r = abi.request(abi.LN["v41_linear"], input_bf16=ptr(x), input_bytes=nbytes(x), weight=ptr(weight),
                    weight_bytes=nbytes(weight), weight_scales=ptr(weight_scales),
                    weight_scale_bytes=nbytes(weight_scales), quantized_e4m3=ptr(quantized),
                    quantized_bytes=nbytes(quantized), activation_scales=ptr(activation_scales),
                    activation_scale_bytes=nbytes(activation_scales), output_bf16=ptr(out),
                    output_bytes=nbytes(out), error_flag_u32=ptr(flag), error_flag_bytes=4,
                    stream=stream_handle(), rows=rows, in_features=k, out_features=n, weight_format=weight_format)
    _check(_ln().call("launch_v41_linear", r), "v41_linear")
    return out, quantized, activation_scales, flag


def v41_fp4_to_fp8(packed: torch.Tensor, scales: torch.Tensor, flag: Optional[torch.Tensor] = None):
    """V4.1 expert FP4 -> FP8 32x32 conversion on the device
    (weight_expert_convert.cpp:33-100): (e4m3 [rows, cols], UE8M0 [rows/32,
    cols/32], flag)."""
    rows, half = packed.shape
    cols = half * 2
    w = torch.empty(rows, cols, dtype=torch.uint8, device=packed.device)
    s = torch.empty(rows // 32, cols // 32, dtype=torch.uint8, device=packed.device)
    flag = error_flag() if flag is None else flag
    r = abi.request(abi.LN["v41_fp4_to_fp8"], packed=ptr(packed), scales=ptr(scales), weight_e4m3=ptr(w),
                    weight_scales=ptr(s), error_flag_u32=ptr(flag), stream=stream_handle(), rows=rows, columns=cols)
    _check(_ln().call("launch_v41_fp4_to_fp8", r), "v41_fp4_to_fp8")
    return w, s, flag


def v41_block_dequant(source: torch.Tensor, scales: torch.Tensor, block: int, out: Optional[torch.Tensor] = None,
                      flag: Optional[torch.Tensor] = None):
    """e4m3 [rows, cols] x per-block scale (uint8 UE8M0 or float32 tensor)
    -> bf16 (weight_dequantize.cpp:17-50, DequantizeWoATensor)."""
    rows, cols = source.shape
    if out is None:
        out = torch.empty(rows, cols, dtype=torch.bfloat16, device=source.device)
    flag = error_flag() if flag is None else flag
    storage = abi.V41_SCALE_F32 if scales.dtype == torch.float32 else abi.V41_SCALE_E8M0
    r = abi.request(abi.LN["v41_block_dequant"], source_e4m3=ptr(source), scales=ptr(scales), output_bf16=ptr(out),
                    error_flag_u32=ptr(flag), stream=stream_handle(), rows=rows, columns=cols, block=block,
                    scale_storage=storage)
    _check(_ln().call("launch_v41_block_dequant", r), "v41_block_dequant")
    return out, flag


# ------------------------------------ adapters, LM-head loss, router balance
@functools.lru_cache(maxsize=4096)
def _workspace_bytes(kind: int, m: int, n: int, k: int) -> int:
    out = abi.C.c_uint64()
    q = abi.request(abi.LN["workspace_query"], kind=kind, m=m, n=n, k=k, bytes_u64=abi.C.addressof(out))
    _check(_ln().call("query_workspace", q), "query_workspace")
    return out.value


def _workspace(kind: int, m: int, n: int, k: int, device) -> torch.Tensor:
    return torch.empty(_workspace_bytes(kind, m, n, k), dtype=torch.uint8, device=device)


@functools.lru_cache(maxsize=None)
def _entry(entry: str, name: str):
    t = abi.LN[name]
    # (the 32-bit sizes and strides, which follow one another in every request)
    words = [i for i, (_, kind) in enumerate(t._fields_[2:]) if kind is abi.U32]
    return getattr(_ln().table, entry), t, abi.C.sizeof(t), slice(words[0], words[-1] + 1)


_byref = abi.C.byref


def _launch(entry: str, name: str, *fields) -> None:
    """The entry called with its request's fields in order (one constructor
    call: 2 us less of host time than setting twenty fields by name)."""
    call, t, size, words = _entry(entry, name)
    if max(fields[words]) > 0xFFFFFFFF:  # (a request's field would keep the lower half)
        raise ValueError(f"pih_amd: {name} takes sizes and strides of 32 bits")
    status = call(_byref(t(size, 1, *fields)))
    if status.code:
        _check(status, name)


def _want(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError("pih_amd: " + what)


def _adapter_stacks(a, b, scale, offsets, adapters):
    # (plain comparisons: these callers' checks are a tenth of a small call)
    if a.dim() != 3 or b.dim() != 3 or a.dtype is not torch.bfloat16 or b.dtype is not torch.bfloat16:
        raise ValueError("pih_amd: adapter stacks are A [adapters, rank, k] and B [adapters, n, rank], bfloat16")
    count, rank, k = a.shape
    other, n, inner = b.shape
    if count != other or rank != inner:
        raise ValueError("pih_amd: adapter stacks are A [adapters, rank, k] and B [adapters, n, rank]")
    if scale is not None and (scale.dtype is not torch.float32 or scale.shape != (count,)):
        raise ValueError("pih_amd: adapter scales are float32 [adapters]")
    if offsets.dtype is not torch.int32 or adapters.dtype is not torch.int32 or adapters.dim() != 1 or \
            offsets.shape != (adapters.shape[0] + 1,):
        raise ValueError("pih_amd: segment offsets are int32 [segments + 1], segment adapters int32 [segments]")
    return count, rank, n, k


def _rows(t, rows: int, cols: int, what: str):
    """Address and row stride of a tensor whose rows are contiguous."""
    if t.shape != (rows, cols) or t.dtype is not torch.bfloat16:
        raise ValueError(f"pih_amd: {what} is bfloat16 [{rows}, {cols}]")
    row, col = t.stride()
    if col != 1 and cols > 1:
        raise ValueError("pih_amd: tensor rows must be contiguous")
    return t.data_ptr(), row if rows > 1 else cols


def adapter_gemm(x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, scale: Optional[torch.Tensor],
                 offsets: torch.Tensor, adapters: torch.Tensor, base: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None, flag: Optional[torch.Tensor] = None):
    """Low-rank adapters of many requests on top of a shared projection's
    output (``launch_adapter_gemm``): ``out[t] = base[t] + scale[i] *
    (x[t] . a[i]^T) . b[i]^T`` for the rows ``offsets[s] <= t <
    offsets[s + 1]`` of every segment ``s``, whose adapter is ``i =
    adapters[s]`` (-1: none).  ``x`` [rows, k], ``base`` and ``out``
    [rows, n] may be column slices of wider tensors; ``out`` may be ``base``
    itself; ``base`` None starts from zero.  Rows outside every segment are
    left as they are (in a new ``out`` they hold anything).  Returns (out,
    flag)."""
    count, rank, n, k = _adapter_stacks(a, b, scale, offsets, adapters)
    rows = x.shape[0]
    px, xs = _rows(x, rows, k, "the adapters' input")
    pbase, bs = (0, 0) if base is None else _rows(base, rows, n, "the adapters' base")
    if out is None:
        out = torch.empty(rows, n, dtype=torch.bfloat16, device=x.device)
    pout, os = _rows(out, rows, n, "the adapters' output")
    flag = error_flag() if flag is None else flag
    same_device(x, base, out)
    pa, pb, ps, po, pi, pflag = device_ptrs(a, b, scale, offsets, adapters, flag)
    ws = _workspace(abi.WORKSPACE_ADAPTER_GEMM, rows, rank, k, x.device)
    _launch("launch_adapter_gemm", "adapter_gemm", px, pa, pb, ps, po, pi, pbase, pout, ws.data_ptr(), ws.numel(),
            pflag, stream_handle(), rows, adapters.shape[0], count, rank, n, k, xs, bs, os)
    return out, flag


@functools.lru_cache(maxsize=4096)
def _adapter_backward_bytes(rows: int, segments: int, count: int, rank: int, n: int, k: int) -> int:
    out = abi.C.c_uint64()
    q = abi.request(abi.LN["adapter_backward"], row_count=rows, segment_count=segments, adapter_count=count, rank=rank,
                    n=n, k=k, required_bytes_u64=abi.C.addressof(out))
    _check(_ln().call("query_adapter_backward_workspace", q), "query_adapter_backward_workspace")
    return out.value


def adapter_backward(dy: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor,
                     scale: Optional[torch.Tensor], offsets: torch.Tensor, adapters: torch.Tensor,
                     base: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                     flag: Optional[torch.Tensor] = None):
    """Gradients of ``adapter_gemm`` for the upstream gradient ``dy`` [rows,
    n] (``launch_adapter_backward``): (dx bf16 [rows, k], da f32 like ``a``,
    db f32 like ``b``, flag).  ``base`` is the shared projection's gradient of
    x, on top of which dx comes (``out`` may be ``base`` itself).  Segments
    that share an adapter add up; an adapter without rows has zeros.  Rows of
    dx outside every segment are left as they are, as in ``adapter_gemm``."""
    count, rank, n, k = _adapter_stacks(a, b, scale, offsets, adapters)
    rows = x.shape[0]
    pdy, ys = _rows(dy, rows, n, "the upstream gradient")
    px, xs = _rows(x, rows, k, "the adapters' input")
    pbase, bs = (0, 0) if base is None else _rows(base, rows, k, "the gradient's base")
    if out is None:
        out = torch.empty(rows, k, dtype=torch.bfloat16, device=x.device)
    pout, os = _rows(out, rows, k, "the input's gradient")
    da = torch.empty(a.shape, dtype=torch.float32, device=x.device)
    db = torch.empty(b.shape, dtype=torch.float32, device=x.device)
    flag = error_flag() if flag is None else flag
    same_device(dy, x, base, out)
    pa, pb, ps, po, pi, pflag = device_ptrs(a, b, scale, offsets, adapters, flag)
    ws = torch.empty(_adapter_backward_bytes(rows, adapters.shape[0], count, rank, n, k), dtype=torch.uint8,
                     device=x.device)
    _launch("launch_adapter_backward", "adapter_backward", pdy, px, pa, pb, ps, po, pi, pbase, pout, da.data_ptr(),
            db.data_ptr(), ws.data_ptr(), ws.numel(), 0, pflag, stream_handle(), rows, adapters.shape[0], count, rank,
            n, k, ys, xs, bs, os)
    return out, da, db, flag


def _loss_inputs(x, weight, targets):
    _want(x.dim() == 2 and weight.dim() == 2 and x.shape[1] == weight.shape[1] and
          x.dtype == weight.dtype == torch.bfloat16, "the LM head is x [rows, hidden] . weight [vocab, hidden], bfloat16")
    _want(targets.dtype == torch.int32 and targets.shape == x.shape[:1], "targets are int32 [rows]")
    return x.shape[0], weight.shape[0], x.shape[1]


def lm_head_loss(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor,
                 flag: Optional[torch.Tensor] = None):
    """Softmax cross entropy of an LM head without its logits
    (``launch_lm_head_loss``): (loss f32 [rows], lse f32 [rows], flag) with
    ``lse`` the log-sum-exp of a row's logits and ``-loss`` the target's
    log-probability.  A target of -1 is none: loss 0."""
    rows, vocab, hidden = _loss_inputs(x, weight, targets)
    loss = torch.empty(rows, dtype=torch.float32, device=x.device)
    lse = torch.empty(rows, dtype=torch.float32, device=x.device)
    flag = error_flag() if flag is None else flag
    px, pw, pt, pflag = device_ptrs(x, weight, targets, flag)
    ws = _workspace(abi.WORKSPACE_LM_HEAD_LOSS, rows, vocab, hidden, x.device)
    _launch("launch_lm_head_loss", "lm_head_loss", px, pw, pt, loss.data_ptr(), lse.data_ptr(), ws.data_ptr(), ws.numel(),
            pflag, stream_handle(), rows, vocab, hidden)
    return loss, lse, flag


def lm_head_loss_backward(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, lse: torch.Tensor,
                          dloss: torch.Tensor, weight_gradient: bool = True, flag: Optional[torch.Tensor] = None):
    """Gradients of ``lm_head_loss`` for the losses' upstream gradient
    ``dloss`` f32 [rows] (``launch_lm_head_loss_backward``): (dx bf16 like
    ``x``, dweight bf16 like ``weight``, or None without
    ``weight_gradient``, flag)."""
    rows, vocab, hidden = _loss_inputs(x, weight, targets)
    _want(lse.dtype == dloss.dtype == torch.float32 and lse.shape == dloss.shape == x.shape[:1],
          "lse and dloss are float32 [rows]")
    flag = error_flag() if flag is None else flag
    px, pw, pt, pl, pd, pflag = device_ptrs(x, weight, targets, lse, dloss, flag)
    dx = torch.empty_like(x)
    dw = torch.empty_like(weight) if weight_gradient else None
    ws = _workspace(abi.WORKSPACE_LM_HEAD_LOSS_BACKWARD, rows, vocab, hidden, x.device)
    _launch("launch_lm_head_loss_backward", "lm_head_loss_backward", px, pw, pt, pl, pd, dx.data_ptr(),
            0 if dw is None else dw.data_ptr(), ws.data_ptr(), ws.numel(), pflag, stream_handle(), rows, vocab, hidden)
    return dx, dw, flag


def _router_inputs(scores, topk_ids):
    _want(scores.dim() == 2 and scores.dtype == torch.float32, "router scores are float32 [tokens, experts]")
    _want(topk_ids.dim() == 2 and topk_ids.dtype == torch.int32 and topk_ids.shape[0] == scores.shape[0],
          "expert ids are int32 [tokens, top_k]")
    return scores.shape[0], scores.shape[1], topk_ids.shape[1]


def router_balance(scores: torch.Tensor, topk_ids: torch.Tensor, mode: int, coefficient: float,
                   flag: Optional[torch.Tensor] = None):
    """A router's balance loss and its experts' load
    (``launch_router_balance``): (loss f32 [1], counts int32 [experts], mean
    affinity f32 [experts], flag) from the raw scores and the ids that
    ``router_topk`` chose; ``mode`` as there."""
    tokens, experts, topk = _router_inputs(scores, topk_ids)
    dev = scores.device
    loss = torch.empty(1, dtype=torch.float32, device=dev)
    counts = torch.empty(experts, dtype=torch.int32, device=dev)
    mean = torch.empty(experts, dtype=torch.float32, device=dev)
    flag = error_flag() if flag is None else flag
    ps, pi, pflag = device_ptrs(scores, topk_ids, flag)
    ws = _workspace(abi.WORKSPACE_ROUTER_BALANCE, tokens, topk, experts, dev)
    _launch("launch_router_balance", "router_balance", ps, pi, loss.data_ptr(), counts.data_ptr(), mean.data_ptr(),
            ws.data_ptr(), ws.numel(), pflag, stream_handle(), tokens, experts, topk, mode, coefficient)
    return loss, counts, mean, flag


def router_backward(scores: torch.Tensor, topk_ids: torch.Tensor, counts: Optional[torch.Tensor], mode: int,
                    coefficient: float, dloss: Optional[torch.Tensor], dweights: Optional[torch.Tensor] = None,
                    route_scale: float = 1.0, flag: Optional[torch.Tensor] = None):
    """Gradient of the raw scores (``launch_router_backward``): (dscores f32
    like ``scores``, flag), the sum of the balance loss's (``dloss`` f32 [1],
    with ``counts`` of ``router_balance``) and the route weights'
    (``dweights`` f32 [tokens, top_k], with ``router_topk``'s
    ``route_scale``); either may be None."""
    tokens, experts, topk = _router_inputs(scores, topk_ids)
    _want(dloss is None or (dloss.dtype == torch.float32 and dloss.numel() == 1 and counts is not None and
                            counts.dtype == torch.int32 and tuple(counts.shape) == (experts,)),
          "dloss is float32 [1] and comes with counts int32 [experts]")
    _want(dweights is None or (dweights.dtype == torch.float32 and dweights.shape == topk_ids.shape),
          "dweights is float32 [tokens, top_k]")
    flag = error_flag() if flag is None else flag
    ps, pi, pc, pl, pw, pflag = device_ptrs(scores, topk_ids, counts, dloss, dweights, flag)
    dscores = torch.empty_like(scores)
    _launch("launch_router_backward", "router_backward", ps, pi, pc, pl, pw, dscores.data_ptr(), pflag,
            stream_handle(), tokens, experts, topk, mode, coefficient, route_scale)
    return dscores, flag


# ------------------- feed-forward block, distillation, drafted tokens
def _mlp_inputs(x, w_gate, w_up, w_down):
    _want(x.dim() == w_gate.dim() == w_down.dim() == 2 and
          x.dtype == w_gate.dtype == w_up.dtype == w_down.dtype == torch.bfloat16,
          "the feed-forward block is x [rows, hidden] and three weights, bfloat16")
    rows, hidden = x.shape
    inter = w_gate.shape[0]
    _want(w_gate.shape == w_up.shape == (inter, hidden) and w_down.shape == (hidden, inter),
          "the block's weights are gate and up [intermediate, hidden] and down [hidden, intermediate]")
    return rows, hidden, inter


def gated_mlp(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, limit: float = 0.0,
              keep: bool = False, out: Optional[torch.Tensor] = None):
    """The gated feed-forward block ``(silu(x . w_gate^T) * (x . w_up^T)) .
    w_down^T`` (``launch_gated_mlp``): y bf16 [rows, hidden], or with
    ``keep`` (y, gate, up) with the two projections' outputs bf16 [rows,
    intermediate] that ``gated_mlp_backward`` takes.  ``limit`` above 0 clamps
    the gate from above and up from both sides.  Unlike ``QwenMlpBlock``,
    which issues the projections and the activation one by one as the
    reference's model does, the activation takes its inputs in fp32."""
    rows, hidden, inter = _mlp_inputs(x, w_gate, w_up, w_down)
    if out is None:
        out = torch.empty_like(x)
    _want(out.shape == x.shape and out.dtype == torch.bfloat16, "the block's output is bfloat16 [rows, hidden]")
    gate = up = None
    if keep:
        gate = torch.empty(rows, inter, dtype=torch.bfloat16, device=x.device)
        up = torch.empty(rows, inter, dtype=torch.bfloat16, device=x.device)
    px, pg, pu, pd, po = device_ptrs(x, w_gate, w_up, w_down, out)
    ws = _workspace(abi.WORKSPACE_GATED_MLP, rows, inter, hidden, x.device)
    _launch("launch_gated_mlp", "gated_mlp", px, pg, pu, pd, po, gate.data_ptr() if keep else 0,
            up.data_ptr() if keep else 0, ws.data_ptr(), ws.numel(), stream_handle(), rows, hidden, inter, limit)
    return (out, gate, up) if keep else out


def gated_mlp_backward(dy: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor,
                       w_down: torch.Tensor, gate: torch.Tensor, up: torch.Tensor, limit: float = 0.0,
                       weight_gradients: bool = True):
    """Gradients of ``gated_mlp`` for the upstream gradient ``dy`` of its
    output (``launch_gated_mlp_backward``), with ``gate`` and ``up`` as it
    kept them: (dx, dw_gate, dw_up, dw_down), bf16, the last three None
    without ``weight_gradients`` (frozen weights)."""
    rows, hidden, inter = _mlp_inputs(x, w_gate, w_up, w_down)
    _want(dy.shape == x.shape and dy.dtype == torch.bfloat16, "the upstream gradient is bfloat16 [rows, hidden]")
    _want(gate.shape == up.shape == (rows, inter) and gate.dtype == up.dtype == torch.bfloat16,
          "gate and up are bfloat16 [rows, intermediate]")
    py, px, pg, pu, pd, pa, pb = device_ptrs(dy, x, w_gate, w_up, w_down, gate, up)
    dx = torch.empty_like(x)
    grads = tuple(torch.empty_like(w) if weight_gradients else None for w in (w_gate, w_up, w_down))
    ws = _workspace(abi.WORKSPACE_GATED_MLP_BACKWARD, rows, inter, hidden, x.device)
    _launch("launch_gated_mlp_backward", "gated_mlp_backward", py, px, pg, pu, pd, pa, pb, dx.data_ptr(),
            *(0 if g is None else g.data_ptr() for g in grads), ws.data_ptr(), ws.numel(), stream_handle(), rows,
            hidden, inter, limit)
    return (dx,) + grads


def _teacher_inputs(x, weight, teacher_ids, teacher_logits, teacher_lse):
    _want(x.dim() == 2 and weight.dim() == 2 and x.shape[1] == weight.shape[1] and
          x.dtype == weight.dtype == torch.bfloat16, "the LM head is x [rows, hidden] . weight [vocab, hidden], bfloat16")
    _want(teacher_ids.dim() == 2 and teacher_ids.shape[0] == x.shape[0] and teacher_ids.dtype == torch.int32 and
          teacher_logits.shape == teacher_ids.shape and teacher_logits.dtype == torch.float32,
          "the teacher's entries are ids int32 and logits float32 [rows, top_k]")
    _want(teacher_lse is None or (teacher_lse.shape == x.shape[:1] and teacher_lse.dtype == torch.float32),
          "teacher_lse is float32 [rows]")
    return x.shape[0], weight.shape[0], x.shape[1], teacher_ids.shape[1]


def lm_head_distill(x: torch.Tensor, weight: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
                    temperature: float = 1.0, teacher_lse: Optional[torch.Tensor] = None,
                    flag: Optional[torch.Tensor] = None):
    """Divergence of an LM head from a teacher's top logits, without the
    head's own logits in memory (``launch_lm_head_distill``): (loss f32
    [rows], lse f32 [rows], logits f32 [rows, top_k], flag).  ``loss`` is
    ``temperature^2 * KL(teacher || head)`` of the softmaxes over
    ``temperature``, the teacher's over its entries, or with ``teacher_lse``
    (the log-sum-exp of all its logits over ``temperature``) over its whole
    vocabulary, of which the entries' part is summed.  An id of -1 is no
    entry; a row without entries has loss 0.  ``lse`` and ``logits`` (the
    head's, at the entries) are what the backward pass needs."""
    rows, vocab, hidden, top_k = _teacher_inputs(x, weight, teacher_ids, teacher_logits, teacher_lse)
    loss = torch.empty(rows, dtype=torch.float32, device=x.device)
    lse = torch.empty(rows, dtype=torch.float32, device=x.device)
    logits = torch.empty(rows, top_k, dtype=torch.float32, device=x.device)
    flag = error_flag() if flag is None else flag
    px, pw, pi, pt, pl, pflag = device_ptrs(x, weight, teacher_ids, teacher_logits, teacher_lse, flag)
    ws = _workspace(abi.WORKSPACE_LM_HEAD_DISTILL, rows, vocab, hidden, x.device)
    _launch("launch_lm_head_distill", "lm_head_distill", px, pw, pi, pt, pl, loss.data_ptr(), lse.data_ptr(),
            logits.data_ptr(), ws.data_ptr(), ws.numel(), pflag, stream_handle(), rows, vocab, hidden, top_k, temperature)
    return loss, lse, logits, flag


def lm_head_distill_backward(x: torch.Tensor, weight: torch.Tensor, teacher_ids: torch.Tensor,
                             teacher_logits: torch.Tensor, lse: torch.Tensor, logits: torch.Tensor,
                             dloss: torch.Tensor, temperature: float = 1.0,
                             teacher_lse: Optional[torch.Tensor] = None, weight_gradient: bool = True,
                             flag: Optional[torch.Tensor] = None):
    """Gradients of ``lm_head_distill`` for the losses' upstream gradient
    ``dloss`` f32 [rows], from the ``lse`` and ``logits`` it returned
    (``launch_lm_head_distill_backward``): (dx bf16 like ``x``, dweight bf16
    like ``weight``, or None without ``weight_gradient``, flag)."""
    rows, vocab, hidden, top_k = _teacher_inputs(x, weight, teacher_ids, teacher_logits, teacher_lse)
    _want(lse.dtype == dloss.dtype == torch.float32 and lse.shape == dloss.shape == x.shape[:1],
          "lse and dloss are float32 [rows]")
    _want(logits.dtype == torch.float32 and logits.shape == teacher_ids.shape, "logits are float32 [rows, top_k]")
    flag = error_flag() if flag is None else flag
    px, pw, pi, pt, pl, pe, pz, pd, pflag = device_ptrs(x, weight, teacher_ids, teacher_logits, teacher_lse, lse,
                                                        logits, dloss, flag)
    dx = torch.empty_like(x)
    dw = torch.empty_like(weight) if weight_gradient else None
    ws = _workspace(abi.WORKSPACE_LM_HEAD_DISTILL_BACKWARD, rows, vocab, hidden, x.device)
    _launch("launch_lm_head_distill_backward", "lm_head_distill_backward", px, pw, pi, pt, pl, pe, pz, pd, dx.data_ptr(),
            0 if dw is None else dw.data_ptr(), ws.data_ptr(), ws.numel(), pflag, stream_handle(), rows, vocab, hidden,
            top_k, temperature)
    return dx, dw, flag


def _logit_rows(t, rows: int, vocab: int, dtype, what: str):
    """Address and row stride of logits whose rows are contiguous."""
    if t.shape != (rows, vocab) or t.dtype is not dtype:
        raise ValueError(f"pih_amd: {what} are {dtype} [{rows}, {vocab}]")
    row, col = t.stride()
    if col != 1 and vocab > 1:
        raise ValueError("pih_amd: tensor rows must be contiguous")
    return t.data_ptr(), row if rows > 1 else vocab


def draft_verify(target_logits: torch.Tensor, draft_tokens: torch.Tensor, draft_offsets: torch.Tensor,
                 accept_random: torch.Tensor, sample_random: torch.Tensor, max_drafts: int,
                 draft_logits: Optional[torch.Tensor] = None, temperature: Optional[torch.Tensor] = None,
                 flag: Optional[torch.Tensor] = None):
    """Drafted tokens of many sequences against the target model's logits
    (``launch_draft_verify``): (tokens int32 [sequences, max_drafts + 1],
    accepted int32 [sequences], flag).  Sequence s drafted
    ``draft_tokens[draft_offsets[s]:draft_offsets[s + 1]]``, at most
    ``max_drafts``; its rows of ``target_logits`` [drafts + sequences, vocab]
    start at ``draft_offsets[s] + s``, one for each of them and one more.
    ``draft_logits`` [drafts, vocab] are what the drafts were drawn from (None:
    they were looked up); ``temperature`` f32 [sequences] (None: 1; 0: greedy)
    holds for both models.  ``accept_random`` f32 [drafts] and
    ``sample_random`` f32 [sequences] are uniform in [0, 1).  A row of
    ``tokens`` holds the accepted tokens, the one that follows them, and -1.
    Logits are float32 or bfloat16; their rows may be slices of wider ones."""
    _want(target_logits.dim() == 2 and target_logits.dtype in (torch.float32, torch.bfloat16),
          "logits are float32 or bfloat16 [rows, vocab]")
    _want(draft_tokens.dim() == 1 and draft_offsets.dim() == 1 and draft_offsets.shape[0] > 1 and
          draft_tokens.dtype == draft_offsets.dtype == torch.int32,
          "drafted tokens are int32 [drafts], their offsets int32 [sequences + 1]")
    drafts, sequences, vocab = draft_tokens.shape[0], draft_offsets.shape[0] - 1, target_logits.shape[1]
    _want(accept_random.dtype == sample_random.dtype == torch.float32 and accept_random.shape == (drafts,) and
          sample_random.shape == (sequences,), "random numbers are float32 [drafts] and [sequences]")
    _want(temperature is None or (temperature.dtype == torch.float32 and temperature.shape == (sequences,)),
          "temperatures are float32 [sequences]")
    _want(max_drafts >= 0, "max_drafts is not negative")
    pt, ts = _logit_rows(target_logits, drafts + sequences, vocab, target_logits.dtype, "the target's logits")
    pd, ds = 0, 0
    if draft_logits is not None and drafts:
        pd, ds = _logit_rows(draft_logits, drafts, vocab, target_logits.dtype, "the draft model's logits")
    dev = target_logits.device
    tokens = torch.empty(sequences, max_drafts + 1, dtype=torch.int32, device=dev)
    accepted = torch.empty(sequences, dtype=torch.int32, device=dev)
    flag = error_flag() if flag is None else flag
    same_device(target_logits, draft_logits)
    pk, po, pa, ps, pm, pflag = device_ptrs(draft_tokens, draft_offsets, accept_random, sample_random, temperature, flag)
    ws = _workspace(abi.WORKSPACE_DRAFT_VERIFY, sequences, max_drafts, vocab, dev)
    _launch("launch_draft_verify", "draft_verify", pt, pd, pk, po, pa, ps, pm, tokens.data_ptr(), accepted.data_ptr(),
            ws.data_ptr(), ws.numel(), pflag, stream_handle(), sequences, drafts, max_drafts, vocab, ts, ds,
            abi.OUTPUT_F32 if target_logits.dtype == torch.float32 else abi.OUTPUT_BF16)
    return tokens, accepted, flag
