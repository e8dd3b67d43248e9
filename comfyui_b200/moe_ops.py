"""Tensor-level wrappers around the C ABI (include/comfy_b200_moe.h).

PyTorch is used for device memory and streams only: every function here passes raw device pointers
of tensors it was given (or of workspaces it allocated through torch's caching allocator) to the
shared library and launches on ``torch.cuda.current_stream()``.  None of them has a PyTorch or CPU
implementation behind it.
"""
from __future__ import annotations

import ctypes
import weakref
from dataclasses import dataclass, field
from types import SimpleNamespace
from typing import Optional, Sequence, Tuple

import torch

from . import _native as N

_FP8 = torch.float8_e4m3fn


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _dtype_code(dt: torch.dtype) -> int:
    if dt == torch.bfloat16:
        return N.BF16
    if dt == torch.float32:
        return N.FP32
    if dt == _FP8:
        return N.FP8_E4M3
    raise ValueError(f"unsupported dtype {dt}")


def _need_cuda(*tensors: Optional[torch.Tensor]) -> None:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise ValueError("the sm_100a kernels need CUDA tensors; there is no CPU path")


# Status words (int32 [2]: [0] the sticky device status word, [1] a near-tie counter) that calls of this module
# have used and nobody has dropped yet; check_all_status() reads them all.
_status_words = weakref.WeakSet()
_device_status = {}


def _lasting_zeros(device) -> torch.Tensor:
    """A zeroed status block outside every CUDA graph: what a capture allocates belongs to the graph's memory pool, where the
    temporaries of other graphs may lie over it, and its zeroing would be repeated by every replay."""
    with torch.cuda.device(device):
        if not torch.cuda.is_current_stream_capturing():
            return torch.zeros((N.STATUS_WORDS,), dtype=torch.int32, device=device)
        relaxed, lib = ctypes.c_int(1), N.load()
        N.check("comfy_moe_relax_capture", lib.comfy_moe_relax_capture(relaxed))
        try:
            side = torch.cuda.Stream()
            with torch.cuda.stream(side):
                block = torch.zeros((N.STATUS_WORDS,), dtype=torch.int32, device=device)
            side.synchronize()
        finally:
            N.check("comfy_moe_relax_capture", lib.comfy_moe_relax_capture(relaxed))
        return block


def device_status(device) -> torch.Tensor:
    """The status word shared by every call on `device` that brings no workspace of its own (dense feed-forwards)."""
    st = _device_status.get(device)                # (a device object finds it without being spelled out)
    if st is None:
        st = _device_status.get(str(device))
        if st is None:
            st = _lasting_zeros(device)
            _device_status[str(device)] = st
            _status_words.add(st)
        _device_status[device] = st
    return st


def check_all_status() -> None:
    """Reads every live status word (one stream synchronisation each) and raises for the first code found.  Status
    words are sticky, so calling this once after a model forward covers every layer of it."""
    for st in list(_status_words):
        read_status(st)


def plan_sizes(n_tokens: int, n_experts: int, top_k: int = 2) -> Tuple[int, int]:
    """(rows_cap, n_blocks) for the permuted buffers and the per-block count scratch."""
    rows = ctypes.c_int64()
    blocks = ctypes.c_int()
    N.check("comfy_moe_plan_sizes", N.load().comfy_moe_plan_sizes(n_tokens, n_experts, top_k, rows, blocks))
    return rows.value, blocks.value


# --------------------------------------------------------------------------------------- weights
@dataclass
class FfnPack:
    """Device pointers of one FeedForwardSwiGLU; keeps the tensors alive."""

    w1: torch.Tensor
    w3: torch.Tensor
    w2: torch.Tensor
    scale_w1: Optional[torch.Tensor] = None
    scale_w3: Optional[torch.Tensor] = None
    scale_w2: Optional[torch.Tensor] = None
    scale_in13: Optional[torch.Tensor] = None
    scale_in2: Optional[torch.Tensor] = None
    max_sms: int = 0        # 0 = all; see ComfyMoeFfnWeights.max_sms

    def __post_init__(self):
        _need_cuda(self.w1, self.w2, self.w3)
        for w in (self.w1, self.w2, self.w3):
            if w.dim() != 2 or w.stride(1) != 1:
                raise ValueError("expert weights must be 2-D with a contiguous last dimension")
        if self.w1.shape != self.w3.shape or self.w1.stride(0) != self.w3.stride(0):
            raise ValueError("w1 and w3 must share shape and leading dimension")
        if self.w2.shape != (self.w1.shape[1], self.w1.shape[0]):
            raise ValueError("w2 must be [dim, hidden]")
        for s in (self.scale_w1, self.scale_w3, self.scale_w2, self.scale_in13, self.scale_in2):
            if s is not None and (s.dtype != torch.float32 or s.numel() != 1 or not s.is_cuda):
                raise ValueError("scales must be fp32 scalars on the device")

    @property
    def hidden(self) -> int:
        return self.w1.shape[0]

    @property
    def dim(self) -> int:
        return self.w1.shape[1]

    def fill(self, s: N.FfnWeights) -> None:
        s.w1, s.w3, s.w2 = self.w1.data_ptr(), self.w3.data_ptr(), self.w2.data_ptr()
        s.ld13, s.ld2 = self.w1.stride(0), self.w2.stride(0)
        s.hidden = self.hidden
        s.max_sms = self.max_sms
        for name in ("scale_w1", "scale_w3", "scale_w2", "scale_in13", "scale_in2"):
            t = getattr(self, name)
            setattr(s, name, None if t is None else t.data_ptr())

    def struct(self) -> N.FfnWeights:
        s = N.FfnWeights()
        self.fill(s)
        return s


@dataclass
class LayerPack:
    """Everything comfy_moe_forward needs to know about one MOEFeedForwardSwiGLU."""

    gate: torch.Tensor
    experts: Sequence[FfnPack]
    shared: FfnPack
    top_k: int = 2
    c_layer: N.Layer = field(init=False)

    def __post_init__(self):
        _need_cuda(self.gate)
        if not self.gate.is_contiguous():
            raise ValueError("gate weight must be contiguous")
        L = N.Layer()
        L.dim = self.gate.shape[1]
        L.n_experts = len(self.experts)
        L.top_k = self.top_k
        L.w_dtype = _dtype_code(self.experts[0].w1.dtype)
        L.gate_dtype = _dtype_code(self.gate.dtype)
        L.w_gate = self.gate.data_ptr()
        for i, e in enumerate(self.experts):
            e.fill(L.experts[i])
        self.shared.fill(L.shared)
        self.c_layer = L

    @property
    def dim(self) -> int:
        return self.gate.shape[1]

    @property
    def n_experts(self) -> int:
        return len(self.experts)

    @property
    def fp8(self) -> bool:
        return self.experts[0].w1.dtype == _FP8


# --------------------------------------------------------------------------------------- workspace
class Workspace:
    """Device buffers for one call of the layer at a given token count.  Owned by the caller."""

    def __init__(self, n_tokens: int, dim: int, n_experts: int, hidden: int, hidden_shared: int, fp8: bool,
                 device: torch.device, top_k: int = 2):
        self.n_tokens, self.dim, self.n_experts = n_tokens, dim, n_experts
        self.hidden, self.hidden_shared, self.fp8 = hidden, hidden_shared, fp8
        rows_cap, n_blocks = plan_sizes(n_tokens, n_experts, top_k)
        self.rows_cap, self.n_blocks = rows_cap, n_blocks
        act = _FP8 if fp8 else torch.bfloat16
        i32 = dict(dtype=torch.int32, device=device)
        self.topk_idx = torch.empty((n_tokens, top_k), **i32)
        self.topk_weight = torch.empty((n_tokens, top_k), dtype=torch.float32, device=device)
        self.block_counts = torch.empty((max(n_blocks, 1), n_experts), **i32)
        self.block_offsets = torch.empty((max(n_blocks, 1), n_experts), **i32)
        self.expert_counts = torch.zeros((n_experts,), **i32)
        self.expert_offsets = torch.zeros((n_experts + 1,), **i32)
        self.row_map = torch.empty((n_tokens, top_k), **i32)
        self.status = torch.zeros((N.STATUS_WORDS,), **i32)
        _status_words.add(self.status)
        self.x_perm = torch.empty((rows_cap, dim), dtype=act, device=device)
        self.x_q = torch.empty((n_tokens, dim), dtype=act, device=device) if fp8 else None
        self.h_perm = torch.empty((rows_cap, hidden), dtype=act, device=device)
        self.y_perm = torch.empty((rows_cap, dim), dtype=torch.bfloat16, device=device)
        self.h_shared = torch.empty((max(n_tokens, 1), hidden_shared), dtype=act, device=device)
        self.y_shared = torch.empty((max(n_tokens, 1), dim), dtype=torch.bfloat16, device=device)
        self.x_mod = None          # allocated on first use by moe_ffn_block
        ws = N.Workspace()
        for name in ("topk_idx", "topk_weight", "block_counts", "block_offsets", "expert_counts", "expert_offsets",
                     "row_map", "status", "x_perm", "x_q", "h_perm", "y_perm", "h_shared", "y_shared"):
            t = getattr(self, name)
            setattr(ws, name, None if t is None else t.data_ptr())
        ws.rows_cap = rows_cap
        ws.x_mod = None
        self.c_ws = ws

    def need_x_mod(self) -> None:
        if self.x_mod is None:
            self.x_mod = torch.empty((max(self.n_tokens, 1), self.dim), dtype=torch.bfloat16, device=self.x_perm.device)
            self.c_ws.x_mod = self.x_mod.data_ptr()

    @classmethod
    def for_layer(cls, layer: LayerPack, n_tokens: int) -> "Workspace":
        return cls(n_tokens, layer.dim, layer.n_experts, layer.experts[0].hidden, layer.shared.hidden, layer.fp8,
                   layer.gate.device, layer.top_k)

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in vars(self).values() if isinstance(t, torch.Tensor))


# --------------------------------------------------------------------------------------- kernels
def gate_topk(x: torch.Tensor, w_gate: torch.Tensor, *, neartie_eps: float = 1e-6, want_flags: bool = False,
              topk_idx: Optional[torch.Tensor] = None, topk_weight: Optional[torch.Tensor] = None,
              block_counts: Optional[torch.Tensor] = None):
    """Fused MoEGate.forward.  x: bf16 [N, D] contiguous; w_gate: bf16 or fp32 [E, D].

    Returns (topk_idx int32 [N,2], topk_weight fp32 [N,2], block_counts int32 [n_blocks,E],
    neartie_count int32 [1], neartie_flags uint8 [N] or None).
    """
    _need_cuda(x, w_gate)
    if x.dtype != torch.bfloat16 or x.dim() != 2 or not x.is_contiguous():
        raise ValueError("x must be a contiguous bf16 [N, D] tensor")
    n, d = x.shape
    e = w_gate.shape[0]
    w_gate = w_gate.contiguous()
    _, n_blocks = plan_sizes(n, e)
    dev = x.device
    if topk_idx is None:
        topk_idx = torch.empty((n, 2), dtype=torch.int32, device=dev)
    if topk_weight is None:
        topk_weight = torch.empty((n, 2), dtype=torch.float32, device=dev)
    if block_counts is None:
        block_counts = torch.empty((max(n_blocks, 1), e), dtype=torch.int32, device=dev)
    count = torch.zeros((1,), dtype=torch.int32, device=dev)
    flags = torch.zeros((n,), dtype=torch.uint8, device=dev) if want_flags else None
    rc = N.load().comfy_moe_gate_topk(_ptr(x), _ptr(w_gate), _dtype_code(w_gate.dtype), n, d, e, 2, _ptr(topk_idx),
                                      _ptr(topk_weight), _ptr(block_counts), _ptr(count), _ptr(flags),
                                      float(neartie_eps), _stream())
    N.check("comfy_moe_gate_topk", rc)
    return topk_idx, topk_weight, block_counts, count, flags


def route_count(topk_idx: torch.Tensor, n_experts: int) -> torch.Tensor:
    """Per-block expert counts of caller-supplied int32 routing [N, 2] (what the gate kernel emits itself)."""
    _need_cuda(topk_idx)
    if topk_idx.dtype != torch.int32 or not topk_idx.is_contiguous():
        raise ValueError("topk_idx must be a contiguous int32 tensor")
    n = topk_idx.numel() // 2
    _, n_blocks = plan_sizes(n, n_experts)
    block_counts = torch.empty((max(n_blocks, 1), n_experts), dtype=torch.int32, device=topk_idx.device)
    rc = N.load().comfy_moe_route_count(_ptr(topk_idx), n, n_experts, _ptr(block_counts), _stream())
    N.check("comfy_moe_route_count", rc)
    return block_counts


def route_plan(block_counts: torch.Tensor, n_tokens: int, n_experts: int):
    """Per-expert scan of the block counts.  Returns (block_offsets, expert_counts, expert_offsets)."""
    _need_cuda(block_counts)
    dev = block_counts.device
    block_offsets = torch.empty_like(block_counts)
    expert_counts = torch.empty((n_experts,), dtype=torch.int32, device=dev)
    expert_offsets = torch.empty((n_experts + 1,), dtype=torch.int32, device=dev)
    rc = N.load().comfy_moe_route_plan(_ptr(block_counts), n_tokens, n_experts, _ptr(block_offsets),
                                       _ptr(expert_counts), _ptr(expert_offsets), _stream())
    N.check("comfy_moe_route_plan", rc)
    return block_offsets, expert_counts, expert_offsets


def permute(x: torch.Tensor, topk_idx: torch.Tensor, block_offsets: torch.Tensor, expert_offsets: torch.Tensor,
            n_experts: int, *, fp8: bool = False, act_scale: Optional[torch.Tensor] = None,
            xq_scale: Optional[torch.Tensor] = None, want_xq: bool = False, zero_fill: bool = False,
            overflow_count: Optional[torch.Tensor] = None):
    """Row permutation into per-expert blocks.  Returns (x_perm, row_map, x_q or None).  ``overflow_count`` (int32 [1],
    fp8 with a scale only) grows by the number of elements the reference's unclamped cast turns into NaN."""
    _need_cuda(x, topk_idx)
    n, d = x.shape
    rows_cap, _ = plan_sizes(n, n_experts)
    act = _FP8 if fp8 else torch.bfloat16
    alloc = torch.zeros if zero_fill else torch.empty
    x_perm = alloc((rows_cap, d), dtype=act, device=x.device) if not fp8 else \
        alloc((rows_cap, d), dtype=torch.uint8, device=x.device).view(_FP8)
    row_map = torch.empty((n, 2), dtype=torch.int32, device=x.device)
    x_q = torch.empty((n, d), dtype=_FP8, device=x.device) if (fp8 and want_xq) else None
    rc = N.load().comfy_moe_permute(_ptr(x), _ptr(topk_idx), _ptr(block_offsets), _ptr(expert_offsets), n, d,
                                    n_experts, N.FP8_E4M3 if fp8 else N.BF16, _ptr(act_scale), _ptr(x_perm),
                                    _ptr(x_q), _ptr(xq_scale), _ptr(row_map), _ptr(overflow_count), _stream())
    N.check("comfy_moe_permute", rc)
    return x_perm, row_map, x_q


def plan_permute(x: torch.Tensor, topk_idx: torch.Tensor, block_counts: torch.Tensor, n_experts: int, *,
                 fp8: bool = False, zero_fill: bool = False):
    """route_plan + permute in one launch.  Returns (x_perm, row_map, expert_counts, expert_offsets)."""
    _need_cuda(x, topk_idx, block_counts)
    n, d = x.shape
    dev = x.device
    rows_cap, _ = plan_sizes(n, n_experts)
    alloc = torch.zeros if zero_fill else torch.empty
    x_perm = alloc((rows_cap, d), dtype=torch.uint8, device=dev).view(_FP8) if fp8 else \
        alloc((rows_cap, d), dtype=torch.bfloat16, device=dev)
    row_map = torch.empty((n, 2), dtype=torch.int32, device=dev)
    scratch = torch.empty_like(block_counts)
    counts = torch.empty((n_experts,), dtype=torch.int32, device=dev)
    offsets = torch.empty((n_experts + 1,), dtype=torch.int32, device=dev)
    rc = N.load().comfy_moe_plan_permute(_ptr(x), _ptr(topk_idx), _ptr(block_counts), n, d, n_experts,
                                         N.FP8_E4M3 if fp8 else N.BF16, None, _ptr(scratch), _ptr(counts),
                                         _ptr(offsets), _ptr(x_perm), None, None, _ptr(row_map), None, _stream())
    N.check("comfy_moe_plan_permute", rc)
    return x_perm, row_map, counts, offsets


def grouped_swiglu(experts: Sequence[FfnPack], shared: Optional[FfnPack], row_start: Optional[torch.Tensor],
                   row_count: Optional[torch.Tensor], x_perm: Optional[torch.Tensor],
                   x_shared: Optional[torch.Tensor], *, status: Optional[torch.Tensor] = None,
                   check_status: bool = True, h_perm: Optional[torch.Tensor] = None,
                   y_perm: Optional[torch.Tensor] = None, h_shared: Optional[torch.Tensor] = None,
                   y_shared: Optional[torch.Tensor] = None):
    """Both passes of the grouped expert GEMM.  Group g = rows [row_start[g], row_start[g] + row_count[g]) of
    x_perm with the weights experts[g] (int32 device tensors; the routing plan's expert_offsets and
    expert_counts on one GPU).  ``h_perm`` / ``y_perm`` may be given (buffers of x_perm's row count, e.g. a result
    buffer that peers read), and so may ``h_shared`` / ``y_shared`` ([n_tokens, hidden_s] / [n_tokens, dim]);
    otherwise they are allocated.  Returns (y_perm or None, y_shared or None, h_perm, h_shared)."""
    ref = experts[0] if experts else shared
    dim, fp8 = ref.dim, ref.w1.dtype == _FP8
    dev = ref.w1.device
    act = _FP8 if fp8 else torch.bfloat16
    n_e = len(experts)
    arr = (N.FfnWeights * max(n_e, 1))()
    for i, e in enumerate(experts):
        e.fill(arr[i])
    rows_cap = 0 if x_perm is None else x_perm.shape[0]
    if n_e:
        if h_perm is None:
            h_perm = torch.empty((rows_cap, experts[0].hidden), dtype=act, device=dev)
        if y_perm is None:
            y_perm = torch.empty((rows_cap, dim), dtype=torch.bfloat16, device=dev)
        if h_perm.shape != (rows_cap, experts[0].hidden) or y_perm.shape != (rows_cap, dim) or \
                not h_perm.is_contiguous() or not y_perm.is_contiguous():
            raise ValueError("h_perm / y_perm must be contiguous buffers with x_perm's row count")
    else:
        h_perm = y_perm = None
    n_tokens = 0 if x_shared is None else x_shared.shape[0]
    sh = h_sh = y_sh = None
    if shared is not None and n_tokens > 0:
        sh = shared.struct()
        h_sh = h_shared if h_shared is not None else torch.empty((n_tokens, shared.hidden), dtype=act, device=dev)
        y_sh = y_shared if y_shared is not None else torch.empty((n_tokens, dim), dtype=torch.bfloat16, device=dev)
        if h_sh.shape != (n_tokens, shared.hidden) or y_sh.shape != (n_tokens, dim) or not h_sh.is_contiguous() or \
                not y_sh.is_contiguous():
            raise ValueError("h_shared / y_shared must be contiguous [n_tokens, hidden] / [n_tokens, dim] buffers")
    if status is None:
        status = device_status(dev)
    rc = N.load().comfy_moe_grouped_swiglu(
        N.FP8_E4M3 if fp8 else N.BF16, n_e, arr, ctypes.byref(sh) if sh is not None else None,
        _ptr(row_start), _ptr(row_count), rows_cap, n_tokens, dim, _ptr(x_perm), _ptr(h_perm), _ptr(y_perm), _ptr(x_shared),
        _ptr(h_sh), _ptr(y_sh), _ptr(status), _stream())
    N.check("comfy_moe_grouped_swiglu", rc)
    if check_status:
        read_status(status)
    return y_perm, y_sh, h_perm, h_sh


def grouped_swiglu_scatter(groups: Sequence[FfnPack], row_start: torch.Tensor, row_count: torch.Tensor,
                           x_perm: torch.Tensor, h_perm: torch.Tensor, y_out_ptrs: Sequence[int],
                           y_row_shift: torch.Tensor, y_rows_cap: int, status: torch.Tensor) -> None:
    """Both passes of the grouped expert GEMM over routed groups, group i's results written to the buffer at address
    ``y_out_ptrs[i]`` (bf16 [y_rows_cap, dim], possibly another GPU's memory) at row + y_row_shift[i]."""
    n_g = len(groups)
    if len(y_out_ptrs) != n_g:
        raise ValueError("one output buffer per group")
    fp8 = groups[0].w1.dtype == _FP8
    arr = (N.FfnWeights * n_g)()
    for i, e in enumerate(groups):
        e.fill(arr[i])
    outs = (ctypes.c_void_p * n_g)(*[int(p) for p in y_out_ptrs])
    rc = N.load().comfy_moe_grouped_swiglu_scatter(
        N.FP8_E4M3 if fp8 else N.BF16, n_g, arr, _ptr(row_start), _ptr(row_count), x_perm.shape[0], groups[0].dim,
        _ptr(x_perm), _ptr(h_perm), outs, _ptr(y_row_shift), y_rows_cap, _ptr(status), _stream())
    N.check("comfy_moe_grouped_swiglu_scatter", rc)


def combine(y_perm: torch.Tensor, row_map: torch.Tensor, topk_weight: torch.Tensor,
            y_shared: Optional[torch.Tensor], out: Optional[torch.Tensor] = None,
            y_perm_b: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[t] = bf16(bf16(bf16(w0*y[r0]) + bf16(w1*y[r1])) + y_shared[t]); with y_perm_b every y is the bf16 sum of
    two partial results (hidden-split experts)."""
    _need_cuda(y_perm, row_map, topk_weight, y_shared, y_perm_b)
    n = row_map.shape[0]
    d = y_perm.shape[1]
    if out is None:
        out = torch.empty((n, d), dtype=torch.bfloat16, device=y_perm.device)
    lib = N.load()
    if y_perm_b is None:
        rc = lib.comfy_moe_combine(_ptr(y_perm), _ptr(row_map), _ptr(topk_weight), _ptr(y_shared), n, d, _ptr(out),
                                   _stream())
    else:
        rc = lib.comfy_moe_combine_partials(_ptr(y_perm), _ptr(y_perm_b), _ptr(row_map), _ptr(topk_weight),
                                            _ptr(y_shared), n, d, _ptr(out), _stream())
    N.check("comfy_moe_combine", rc)
    return out


def quantize_e4m3(x: torch.Tensor, scale: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                  overflow_count: Optional[torch.Tensor] = None) -> torch.Tensor:
    """bf16 -> e4m3 as the reference's fp8 Linear quantises its input: clamp and round without a scale; multiply by
    bf16(1 / scale) and cast without a clamp (overflow -> NaN, counted in ``overflow_count`` int32 [1]) with one."""
    _need_cuda(x, scale)
    if x.dtype != torch.bfloat16 or not x.is_contiguous():
        raise ValueError("x must be a contiguous bf16 tensor")
    if out is None:
        out = torch.empty(x.shape, dtype=_FP8, device=x.device)
    if overflow_count is None:
        overflow_count = device_status(x.device)[2:3]
    N.check("comfy_moe_quantize_e4m3", N.load().comfy_moe_quantize_e4m3(_ptr(x), _ptr(scale), x.numel(), _ptr(out),
                                                                        _ptr(overflow_count), _stream()))
    return out


def read_status(status: torch.Tensor) -> None:
    """Synchronises the current stream and raises if a device-side wait gave up."""
    h = ctypes.c_int32(0)
    rc = N.load().comfy_moe_read_status(_ptr(status), _stream(), h)
    if rc != N.OK:
        raise N.MoeError("comfy_moe_read_status", rc, f"device status word = {h.value}")


def validate_routing(ws: "Workspace") -> None:
    """Debug aid: checks the routing the last layer call left in ``ws`` on the device (ids, rows, offsets, counts) and
    raises if it is inconsistent.  One stream synchronisation."""
    rc = N.load().comfy_moe_validate_routing(_ptr(ws.topk_idx), _ptr(ws.row_map), _ptr(ws.expert_counts),
                                             _ptr(ws.expert_offsets), ws.n_tokens, ws.n_experts, ws.rows_cap,
                                             _ptr(ws.status), _stream())
    N.check("comfy_moe_validate_routing", rc)
    read_status(ws.status)


def moe_forward(layer: LayerPack, x: torch.Tensor, ws: Optional[Workspace] = None,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The whole layer through comfy_moe_forward.  x: bf16 [N, D] contiguous on the device."""
    _need_cuda(x)
    if x.dtype != torch.bfloat16 or x.dim() != 2 or not x.is_contiguous():
        raise ValueError("x must be a contiguous bf16 [N, D] tensor")
    n = x.shape[0]
    if ws is None or ws.n_tokens != n:
        ws = Workspace.for_layer(layer, n)
    if out is None:
        out = torch.empty_like(x)
    rc = N.load().comfy_moe_forward(ctypes.byref(layer.c_layer), ctypes.byref(ws.c_ws), _ptr(x), n, _ptr(out),
                                    _stream())
    N.check("comfy_moe_forward", rc)
    return out


# --------------------------------------------------------------------------------------- block glue
def _modulation(*vectors: torch.Tensor) -> int:
    """Common batch stride (elements) of bf16 [B, D] / [B, 1, D] modulation vectors that are views of one tensor."""
    strides = set()
    for v in vectors:
        _need_cuda(v)
        if v.dtype != torch.bfloat16 or v.stride(-1) != 1:
            raise ValueError("modulation vectors must be bf16 with a contiguous last dimension")
        strides.add(v.stride(0) if v.shape[0] > 1 else 0)
    if len(strides) != 1:
        raise ValueError("modulation vectors must share one batch stride")
    return strides.pop()


def ln_modulate(x: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, tokens_per_batch: int, eps: float = 1e-6,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """LayerNorm(x) * (1 + scale) + shift in one pass.  x: bf16 [N, D]; shift, scale: bf16 [B, D] views."""
    _need_cuda(x)
    n, d = x.shape
    stride = _modulation(shift, scale)
    if out is None:
        out = torch.empty_like(x)
    rc = N.load().comfy_moe_ln_modulate(_ptr(x), _ptr(shift), _ptr(scale), stride, n, tokens_per_batch, d, float(eps),
                                        _ptr(out), _stream())
    N.check("comfy_moe_ln_modulate", rc)
    return out


def ln_modulate_gate(x: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, tokens_per_batch: int,
                     w_gate: torch.Tensor, eps: float = 1e-6, *, neartie_eps: float = 1e-6, want_flags: bool = False):
    """ln_modulate and gate_topk of its output in one pass.  Returns (out, topk_idx, topk_weight, block_counts,
    neartie_count, neartie_flags or None), each bit-identical to what the two separate calls give."""
    _need_cuda(x, w_gate)
    n, d = x.shape
    e = w_gate.shape[0]
    stride = _modulation(shift, scale)
    _, n_blocks = plan_sizes(n, e)
    dev = x.device
    out = torch.empty_like(x)
    topk_idx = torch.empty((n, 2), dtype=torch.int32, device=dev)
    topk_weight = torch.empty((n, 2), dtype=torch.float32, device=dev)
    block_counts = torch.empty((max(n_blocks, 1), e), dtype=torch.int32, device=dev)
    count = torch.zeros((1,), dtype=torch.int32, device=dev)
    flags = torch.zeros((n,), dtype=torch.uint8, device=dev) if want_flags else None
    w_gate = w_gate.contiguous()
    rc = N.load().comfy_moe_ln_modulate_gate(_ptr(x), _ptr(shift), _ptr(scale), stride, n, tokens_per_batch, d, float(eps),
                                             _ptr(out), _ptr(w_gate), _dtype_code(w_gate.dtype), e, 2, _ptr(topk_idx),
                                             _ptr(topk_weight), _ptr(block_counts), _ptr(count), _ptr(flags),
                                             float(neartie_eps), _stream())
    N.check("comfy_moe_ln_modulate_gate", rc)
    return out, topk_idx, topk_weight, block_counts, count, flags


def gate_residual(y: torch.Tensor, gate: torch.Tensor, residual: torch.Tensor, tokens_per_batch: int) -> torch.Tensor:
    """gate * y + residual with PyTorch's bf16 rounding points.  y, residual: bf16 [N, D]; gate: bf16 [B, D] view."""
    _need_cuda(y, residual)
    n, d = y.shape
    out = torch.empty_like(y)
    rc = N.load().comfy_moe_gate_residual(_ptr(y), _ptr(gate), _modulation(gate), _ptr(residual), n, tokens_per_batch, d,
                                          _ptr(out), _stream())
    N.check("comfy_moe_gate_residual", rc)
    return out


def moe_ffn_block(layer: LayerPack, x: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, gate: torch.Tensor,
                  tokens_per_batch: int, eps: float = 1e-6, ws: Optional[Workspace] = None) -> torch.Tensor:
    """gate * MoE(LayerNorm(x) * (1 + scale) + shift) + x through comfy_moe_ffn_block.  x: bf16 [N, D]."""
    _need_cuda(x)
    n = x.shape[0]
    if ws is None or ws.n_tokens != n:
        ws = Workspace.for_layer(layer, n)
    ws.need_x_mod()
    out = torch.empty_like(x)
    rc = N.load().comfy_moe_ffn_block(ctypes.byref(layer.c_layer), ctypes.byref(ws.c_ws), _ptr(x), _ptr(shift),
                                      _ptr(scale), _ptr(gate), _modulation(shift, scale, gate), n, tokens_per_batch,
                                      float(eps), _ptr(out), _stream())
    N.check("comfy_moe_ffn_block", rc)
    return out


# --------------------------------------------------------------------------------------- GELU-MLP experts
@dataclass
class MlpPack:
    """Device pointers of one GELU feed-forward (Linear + bias, GELU, Linear + bias); keeps the tensors alive."""

    w1: torch.Tensor
    b1: Optional[torch.Tensor]
    w2: torch.Tensor
    b2: Optional[torch.Tensor]

    def __post_init__(self):
        _need_cuda(self.w1, self.w2, self.b1, self.b2)
        for w in (self.w1, self.w2):
            if w.dtype != torch.bfloat16 or w.dim() != 2 or w.stride(1) != 1:
                raise ValueError("expert weights must be 2-D bf16 with a contiguous last dimension")
        if self.w2.shape != (self.w1.shape[1], self.w1.shape[0]):
            raise ValueError("w2 must be [dim, hidden]")
        for b, n in ((self.b1, self.w1.shape[0]), (self.b2, self.w2.shape[0])):
            if b is not None and (b.dtype != torch.bfloat16 or b.shape != (n,) or not b.is_contiguous()):
                raise ValueError("biases must be contiguous bf16 vectors over the output features")

    @property
    def hidden(self) -> int:
        return self.w1.shape[0]

    @property
    def dim(self) -> int:
        return self.w1.shape[1]

    def fill(self, s: N.MlpWeights) -> None:
        s.w1, s.w2 = self.w1.data_ptr(), self.w2.data_ptr()
        s.b1 = None if self.b1 is None else self.b1.data_ptr()
        s.b2 = None if self.b2 is None else self.b2.data_ptr()
        s.ld1, s.ld2 = self.w1.stride(0), self.w2.stride(0)
        s.hidden = self.hidden
        s.reserved = 0

    def struct(self) -> N.MlpWeights:
        s = N.MlpWeights()
        self.fill(s)
        return s


@dataclass
class MlpLayerPack:
    """Everything comfy_moe_forward_gelu_mlp needs to know about one MoEBlock."""

    gate: torch.Tensor
    experts: Sequence[MlpPack]
    shared: MlpPack
    top_k: int = 2
    c_layer: N.MlpLayer = field(init=False)
    fp8 = False

    def __post_init__(self):
        _need_cuda(self.gate)
        if not self.gate.is_contiguous():
            raise ValueError("gate weight must be contiguous")
        L = N.MlpLayer()
        L.dim = self.gate.shape[1]
        L.n_experts = len(self.experts)
        L.top_k = self.top_k
        L.gate_dtype = _dtype_code(self.gate.dtype)
        L.w_gate = self.gate.data_ptr()
        for i, e in enumerate(self.experts):
            e.fill(L.experts[i])
        self.shared.fill(L.shared)
        self.c_layer = L

    @property
    def dim(self) -> int:
        return self.gate.shape[1]

    @property
    def n_experts(self) -> int:
        return len(self.experts)


def grouped_gelu_mlp(experts: Sequence[MlpPack], shared: Optional[MlpPack], row_start: Optional[torch.Tensor],
                     row_count: Optional[torch.Tensor], x_perm: Optional[torch.Tensor],
                     x_shared: Optional[torch.Tensor], *, check_status: bool = True):
    """Both passes of the grouped GELU-MLP expert GEMM; arguments as grouped_swiglu.
    Returns (y_perm or None, y_shared or None, h_perm, h_shared)."""
    ref = experts[0] if experts else shared
    dim, dev = ref.dim, ref.w1.device
    n_e = len(experts)
    arr = (N.MlpWeights * max(n_e, 1))()
    for i, e in enumerate(experts):
        e.fill(arr[i])
    rows_cap = 0 if x_perm is None else x_perm.shape[0]
    h_perm = y_perm = None
    if n_e:
        h_perm = torch.empty((rows_cap, experts[0].hidden), dtype=torch.bfloat16, device=dev)
        y_perm = torch.empty((rows_cap, dim), dtype=torch.bfloat16, device=dev)
    n_tokens = 0 if x_shared is None else x_shared.shape[0]
    sh = h_sh = y_sh = None
    if shared is not None and n_tokens > 0:
        sh = shared.struct()
        h_sh = torch.empty((n_tokens, shared.hidden), dtype=torch.bfloat16, device=dev)
        y_sh = torch.empty((n_tokens, dim), dtype=torch.bfloat16, device=dev)
    status = device_status(dev)
    rc = N.load().comfy_moe_grouped_gelu_mlp(
        n_e, arr, ctypes.byref(sh) if sh is not None else None, _ptr(row_start), _ptr(row_count), rows_cap, n_tokens,
        dim, _ptr(x_perm), _ptr(h_perm), _ptr(y_perm), _ptr(x_shared), _ptr(h_sh), _ptr(y_sh), _ptr(status), _stream())
    N.check("comfy_moe_grouped_gelu_mlp", rc)
    if check_status:
        read_status(status)
    return y_perm, y_sh, h_perm, h_sh


def moe_mlp_forward(layer: MlpLayerPack, x: torch.Tensor, ws: Optional[Workspace] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """MoEBlock.forward (eval) through comfy_moe_forward_gelu_mlp.  x: bf16 [N, D] contiguous on the device."""
    _need_cuda(x)
    if x.dtype != torch.bfloat16 or x.dim() != 2 or not x.is_contiguous():
        raise ValueError("x must be a contiguous bf16 [N, D] tensor")
    n = x.shape[0]
    if ws is None or ws.n_tokens != n:
        ws = Workspace.for_layer(layer, n)
    if out is None:
        out = torch.empty_like(x)
    rc = N.load().comfy_moe_forward_gelu_mlp(ctypes.byref(layer.c_layer), ctypes.byref(ws.c_ws), _ptr(x), n,
                                             _ptr(out), _stream())
    N.check("comfy_moe_forward_gelu_mlp", rc)
    return out


# --------------------------------------------------------------------------------------- attention glue
def rmsnorm_rope(x: torch.Tensor, weight: Optional[torch.Tensor], eps: float, rope: Optional[torch.Tensor],
                 heads: int, out: torch.Tensor, out_row_offset: int = 0, rope_row_offset: int = 0) -> torch.Tensor:
    """RMSNorm (optional) + rotary embedding (optional) of one projected tensor, written into rows
    [out_row_offset, out_row_offset + S) of every batch element of ``out`` [B, S_total, heads, head_dim].

    x: bf16 [B, S, heads * head_dim] (last dim contiguous, rows evenly strided); weight: bf16 [heads * head_dim] or
    None; rope: fp32 [B or 1, S_rope, 1, pairs, 2, 2] or None, rotated rows start at ``rope_row_offset``."""
    _need_cuda(x, weight, rope, out)
    b, s, inner = x.shape
    head_dim = inner // heads
    if x.dtype != torch.bfloat16 or x.stride(2) != 1 or x.stride(0) != s * x.stride(1):
        raise ValueError("x must be bf16 [B, S, inner] with evenly strided rows")
    if out.dtype != torch.bfloat16 or out.shape[0] != b or out.shape[2:] != (heads, head_dim) or \
            not out[0].is_contiguous() or out_row_offset + s > out.shape[1]:
        raise ValueError("out must be bf16 [B, S_total, heads, head_dim] with room for the rows")
    rope_stride = pairs = 0
    if rope is not None:
        if rope.dtype != torch.float32 or rope.dim() != 6 or rope.shape[2] != 1 or rope.shape[4:] != (2, 2) or \
                not rope[0].is_contiguous() or rope_row_offset + s > rope.shape[1]:
            raise ValueError("rope must be fp32 [B or 1, S_rope, 1, pairs, 2, 2]")
        pairs = rope.shape[3]
        rope_stride = rope.stride(0) if rope.shape[0] > 1 else 0
    rc = N.load().comfy_attn_rmsnorm_rope(_ptr(x), x.stride(1), _ptr(weight), eps, _ptr(rope), rope_stride,
                                          rope_row_offset, pairs, b * s, s, heads, head_dim, _ptr(out), out.stride(0),
                                          out_row_offset, _stream())
    N.check("comfy_attn_rmsnorm_rope", rc)
    return out


# --------------------------------------------------------------------------------------- weight ingest
def stochastic_round_e4m3(x: torch.Tensor, rand: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One slice of the reference's stochastic rounding to e4m3: x fp32 / bf16 / fp16 (contiguous), rand the fp16
    uniforms the reference would draw for it.  Returns the e4m3 tensor (``out`` if given)."""
    _need_cuda(x, rand, out)
    codes = {torch.float32: N.FP32, torch.bfloat16: N.BF16, torch.float16: N.FP16}
    if x.dtype not in codes or not x.is_contiguous() or rand.dtype != torch.float16 or rand.shape != x.shape or \
            not rand.is_contiguous():
        raise ValueError("x must be contiguous fp32 / bf16 / fp16 and rand fp16 of the same shape")
    if out is None:
        out = torch.empty(x.shape, dtype=_FP8, device=x.device)
    N.check("comfy_moe_stochastic_round_e4m3",
            N.load().comfy_moe_stochastic_round_e4m3(_ptr(x), codes[x.dtype], _ptr(rand), x.numel(), _ptr(out), _stream()))
    return out


def quantize_weight_e4m3(w: torch.Tensor):
    """Per-tensor scaled e4m3 of a weight: returns (wq e4m3 like w, scale fp32 scalar on the device) with
    scale = max|w| / 448 and wq = (w / scale) rounded to nearest even, the layout scaled-fp8 Linears load."""
    _need_cuda(w)
    codes = {torch.float32: N.FP32, torch.bfloat16: N.BF16, torch.float16: N.FP16}
    if w.dtype not in codes or not w.is_contiguous():
        raise ValueError("w must be a contiguous fp32 / bf16 / fp16 tensor")
    out = torch.empty(w.shape, dtype=_FP8, device=w.device)
    scale = torch.empty((), dtype=torch.float32, device=w.device)
    N.check("comfy_moe_quantize_weight_e4m3",
            N.load().comfy_moe_quantize_weight_e4m3(_ptr(w), codes[w.dtype], w.numel(), _ptr(scale), _ptr(out), _stream()))
    return out, scale


def grouped_linear(groups: Sequence[Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]],
                   outs: Optional[Sequence[torch.Tensor]] = None, status: Optional[torch.Tensor] = None):
    """Several ``F.linear(x, w, b)`` in one launch.  groups: (x [rows, in] bf16 with a contiguous last dimension,
    w [out, in] bf16, bias [out] bf16 or None); returns the list of outputs [rows, out] (``outs`` if given)."""
    if not groups:
        return []
    arr = (N.LinearGroup * len(groups))()
    res = []
    dev = groups[0][0].device
    for i, (x, w, b) in enumerate(groups):
        _need_cuda(x, w, b)
        if x.dtype != torch.bfloat16 or w.dtype != torch.bfloat16 or x.dim() != 2 or w.dim() != 2 or \
                x.stride(1) != 1 or w.stride(1) != 1 or x.shape[1] != w.shape[1]:
            raise ValueError("grouped_linear: x [rows, in] and w [out, in] must be bf16 with contiguous last dimensions")
        if b is not None and (b.dtype != torch.bfloat16 or b.shape != (w.shape[0],) or not b.is_contiguous()):
            raise ValueError("grouped_linear: bias must be a contiguous bf16 vector over the output features")
        out = outs[i] if outs is not None else torch.empty((x.shape[0], w.shape[0]), dtype=torch.bfloat16, device=dev)
        if out.shape != (x.shape[0], w.shape[0]) or out.dtype != torch.bfloat16 or out.stride(1) != 1:
            raise ValueError("grouped_linear: out must be bf16 [rows, out] with a contiguous last dimension")
        g = arr[i]
        g.x, g.w, g.out = x.data_ptr(), w.data_ptr(), out.data_ptr()
        g.bias = None if b is None else b.data_ptr()
        g.ld_x, g.ld_w, g.ld_out = x.stride(0), w.stride(0), out.stride(0)
        g.rows, g.in_features, g.out_features = x.shape[0], x.shape[1], w.shape[0]
        res.append(out)
    if status is None:
        status = device_status(dev)
    N.check("comfy_moe_grouped_linear", N.load().comfy_moe_grouped_linear(len(groups), arr, _ptr(status), _stream()))
    return res


def attention_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: Optional[float] = None,
                      status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(q k^T * scale) v per head.  q [B, Sq, H, 128], k / v [B, Skv, H, 128] bf16 contiguous ->
    [B, Sq, H * 128]; scale defaults to 1 / sqrt(128)."""
    _need_cuda(q, k, v)
    b, sq, h, d = q.shape
    if k.shape != v.shape or k.shape[0] != b or k.shape[2:] != (h, d):
        raise ValueError("attention_forward: k and v must be [B, Skv, H, D] matching q's batch, heads and head_dim")
    for t in (q, k, v):
        if t.dtype != torch.bfloat16 or not t.is_contiguous():
            raise ValueError("attention_forward: q, k, v must be contiguous bf16 tensors")
    out = torch.empty((b, sq, h * d), dtype=torch.bfloat16, device=q.device)
    if status is None:
        status = device_status(q.device)
    rc = N.load().comfy_attn_forward(_ptr(q), _ptr(k), _ptr(v), b, sq, k.shape[1], h, d,
                                     float(scale if scale is not None else d ** -0.5), _ptr(out), _ptr(status), _stream())
    N.check("comfy_attn_forward", rc)
    return out


# --------------------------------------------------------------------------------------- products over ragged rows
# These calls last from a few microseconds on, so the way to the C entry points is kept short: plain integers instead of
# ctypes objects, one pass of checks, no context manager where the tensors are on the current device.
_MAX_ROWS, _MAX_FEATURES = N.RAGGED_MAX_ROWS, N.RAGGED_MAX_FEATURES      # what C takes as int32: ctypes would cut more down
_MAX_BLOCKED = N.MAX_SCALE_BLOCKS * N.SCALE_BLOCK
_HALF_CODES = {torch.bfloat16: N.BF16, torch.float16: N.FP16}


def _raw_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream)       # the same without a Stream object
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)      # without looking whether CUDA is up


def _call(name: str, index: int, *args) -> None:
    """One C entry point on the current stream of the tensors' device, which need not be the current device."""
    fn = getattr(N.load(), name)
    if index == _current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        N.check(name, rc)


def _address(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _place(first: torch.Tensor, *others: Optional[torch.Tensor]) -> int:
    """Index of the one device that all tensors of a call live on."""
    index = first.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            if index >= 0 and t.is_cuda:
                raise ValueError(f"all tensors of a call live on one device, got {first.device} and {t.device}")
            index = -1
    if index < 0 or not first.is_cuda:
        raise ValueError("the sm_100a kernels need CUDA tensors; there is no CPU path")
    return index


def _row_stride(what: str, t: torch.Tensor, unit: int) -> int:
    """Elements from one row of t [.., rows, cols] to the next, where the kernels can read and write it as it is: `unit`
    elements are 16 bytes."""
    shape, strides = t.shape, t.stride()           # (as tuples: size(i) and stride(i) take twice as long each)
    cols = shape[-1]
    ld = cols if shape[-2] <= 1 else strides[-2]
    if cols % unit or ld % unit or ld < cols or t.data_ptr() % 16 or (strides[-1] != 1 and cols > 1):
        raise ValueError(f"{what}: rows must be contiguous, of a multiple of {unit} elements, and start on 16 bytes; "
                         f"got shape {tuple(t.shape)}, strides {t.stride()}")
    return ld


def _group_stride(what: str, t: torch.Tensor, unit: int) -> int:
    """Elements from one group of t [G, rows, cols] to the next."""
    if t.shape[0] <= 1:
        return 0
    step = t.stride()[0]
    if step <= 0 or step % unit:
        raise ValueError(f"{what}: groups must start on 16 bytes; got strides {t.stride()}")
    return step


def _readable(t: torch.Tensor) -> torch.Tensor:
    """A tensor as autograd hands it over (a gradient, possibly expanded or transposed; a saved tensor, in whatever layout a
    saved-tensor hook gives back), as rows that the kernels can read."""
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t
    unit, shape, strides = 16 // t.element_size(), t.shape, t.stride()
    ok = strides[-1] == 1 and (shape[-2] <= 1 or (strides[-2] >= shape[-1] and strides[-2] % unit == 0)) and \
        (len(shape) == 2 or shape[0] <= 1 or (strides[0] > 0 and strides[0] % unit == 0)) and t.data_ptr() % 16 == 0
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _unchanged(t: Optional[torch.Tensor], shape: tuple, strides: tuple, dtype: torch.dtype, index: int, unit: int = 1) -> bool:
    """Whether a saved tensor came back with the strides that the forward pass measured (a dimension of one element, whose
    stride it did not look at, says no: the checked calls then decide)."""
    return t is None or (t.stride() == strides and t.shape == shape and t.dtype == dtype and t.get_device() == index and
                         t.data_ptr() % unit == 0)


def _vector(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """Saved offsets, counts or scales, which the kernels read without strides."""
    return None if t is None else t.contiguous()


def _refuse_sizes(rows: int, *features: int) -> None:
    raise ValueError(f"at most {N.RAGGED_MAX_ROWS} rows and 1 to {N.RAGGED_MAX_FEATURES} features, got {rows} and {features}")


def _refuse_blocks(*sizes: int) -> None:
    raise ValueError(f"at most {N.MAX_SCALE_BLOCKS} blocks of {N.SCALE_BLOCK} along a dimension, got {sizes} elements")


def _check_ragged(offsets: torch.Tensor, counts: Optional[torch.Tensor], groups: int) -> None:
    if groups > N.RAGGED_MAX_GROUPS:
        raise ValueError(f"at most {N.RAGGED_MAX_GROUPS} groups, got {groups}")
    if offsets.dtype != torch.int32 or offsets.shape != (groups + 1,) or not offsets.is_contiguous():
        raise ValueError(f"offsets must be a contiguous int32 vector of {groups + 1} elements")
    if counts is not None and (counts.dtype != torch.int32 or counts.shape != (groups,) or not counts.is_contiguous()):
        raise ValueError(f"counts must be a contiguous int32 vector of {groups} elements")


def _extent(t: torch.Tensor) -> Tuple[int, int]:
    """First byte of t's elements, and the one behind the last."""
    size = t.element_size()
    return t.data_ptr(), t.data_ptr() + size * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))


def _check_apart(out: torch.Tensor, *operands: Optional[torch.Tensor]) -> None:
    """Tiles are written while others are still read: a result may stand between the columns of an operand's buffer, but
    share no element with it."""
    if out.numel() == 0:
        return
    first, last = _extent(out)
    for t in operands:
        if t is None or t.numel() == 0:
            continue
        begin, end = _extent(t)
        if end <= first or last <= begin:
            continue
        if t.dim() == 2 and out.dim() == 2:                                # columns of the same rows?
            pitch = {a.stride(0) * a.element_size() for a in (t, out) if a.size(0) > 1}
            ld = pitch.pop() if len(pitch) == 1 else 0
            shift = (first - begin) % ld if ld > 0 else 0
            if shift >= t.size(1) * t.element_size() and shift + out.size(1) * out.element_size() <= ld:
                continue
        raise ValueError("out must not overlap an operand")


def _result(out: Optional[torch.Tensor], like: torch.Tensor, rows: int, cols: int) -> torch.Tensor:
    if out is None:
        return like.new_empty((rows, cols))
    if out.shape != (rows, cols) or out.dtype != like.dtype or out.device != like.device:
        raise ValueError(f"out must be a {like.dtype} tensor of shape {(rows, cols)} on {like.device}")
    return out


def _rows_of(out: torch.Tensor, shape: Sequence[int]) -> torch.Tensor:
    """A result of any dimensions as rows, in place."""
    if out.shape != shape:
        raise ValueError(f"out must be of shape {tuple(shape)}, or its rows of {shape[-1]}, got {tuple(out.shape)}")
    try:
        return out.view(-1, shape[-1])
    except RuntimeError:
        raise ValueError(f"out: rows must be equally far apart; got strides {out.stride()}") from None


def _once(what: str) -> None:
    if torch.is_grad_enabled():
        raise RuntimeError(f"{what} is differentiable once: its gradient has no gradient")


# The level that is open, -1 for none (a torch without the name: every call looks at its tensors).
_forward_ad = torch.autograd.forward_ad if hasattr(torch.autograd.forward_ad, "_current_level") else \
    SimpleNamespace(_current_level=0)


def has_tangent(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether one of them is a dual tensor of a forward-mode derivative that is being taken."""
    return _forward_ad._current_level >= 0 and any(
        t is not None and t.is_floating_point() and torch.autograd.forward_ad.unpack_dual(t).tangent is not None
        for t in tensors)


def _no_tangents(what: str, *tensors: Optional[torch.Tensor]) -> None:
    """Dual tensors ask for a derivative without requires_grad; a result without a tangent would say that it is zero."""
    if has_tangent(*tensors):
        raise NotImplementedError(f"{what} has no forward-mode derivative")


def _grouped_sizes(a: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, counts: Optional[torch.Tensor],
                   width: int) -> tuple:
    """What the C entry points want to know of checked rows and weights: (device index, dtype code, rows, groups, N, K,
    row stride of a, row and group stride of w)."""
    shape, weights = a.shape, w.shape
    if len(shape) != 2 or len(weights) != 3 or shape[1] != weights[width]:
        raise ValueError(f"need rows [R, K] and weights [G, N, K] that fit, got {tuple(shape)} and {tuple(weights)}")
    index = _place(a, w, offsets, counts)
    code = _HALF_CODES.get(a.dtype)
    if code is None or w.dtype != a.dtype:
        raise ValueError(f"rows and weights must both be bf16 or both fp16, got {a.dtype} and {w.dtype}")
    r, (g, n, k) = shape[0], weights
    if not (r <= _MAX_ROWS and 0 < n <= _MAX_FEATURES and 0 < k <= _MAX_FEATURES):
        _refuse_sizes(r, n, k)
    _check_ragged(offsets, counts, g)
    return (index, code, r, g, n, k, _row_stride("rows", a, 8), _row_stride("weights", w, 8),
            _group_stride("weights", w, 8))


def _rows_by_group(name: str, sizes: tuple, a: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor,
                   counts: Optional[torch.Tensor], out: Optional[torch.Tensor], cols: int) -> torch.Tensor:
    index, code, r, g, n, k, ld_a, ld_w, step = sizes
    if out is None:
        res, ld = a.new_empty((r, cols)), cols
    else:
        res = _result(out, a, r, cols)
        ld = _row_stride("out", res, 8)
        _check_apart(res, a, w, offsets, counts)
    _call(name, index, a.data_ptr(), ld_a, w.data_ptr(), ld_w, step, code, r, g, n, k, offsets.data_ptr(), _address(counts),
          out is None, res.data_ptr(), ld, device_status(a.device).data_ptr())
    return res


def grouped_matmul(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, counts: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y[r] = x[r] @ w[g].T`` for the rows r of group g = rows offsets[g] .. offsets[g + 1], of which the first counts[g]
    where ``counts`` is given (the routing plan's expert_offsets and expert_counts).  x [R, K], w [G, N, K], both bf16 or
    both fp16, K and N multiples of 8, y [R, N]; offsets int32 [G + 1], counts int32 [G], on the device and never read by
    the host.  Rows of no group are zero in a result that this function makes, and stay as they were in ``out``, which
    overlaps no operand.
    Differentiable in x and w (once, in reverse mode); a group without rows has the gradient 0."""
    if _forward_ad._current_level >= 0:
        _no_tangents("grouped_matmul", x, w)
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad):
        if out is not None:
            raise ValueError("grouped_matmul: out cannot be given where a gradient is asked for")
        return _GroupedMatmul.apply(x, w, offsets, counts)
    sizes = _grouped_sizes(x, w, offsets, counts, 2)
    return _rows_by_group("comfy_moe_grouped_matmul", sizes, x, w, offsets, counts, out, sizes[4])


def grouped_matmul_dgrad(dy: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, counts: Optional[torch.Tensor] = None,
                         out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``dx[r] = dy[r] @ w[g]``: the gradient of grouped_matmul for x.  dy [R, N] -> [R, K]; rows of no group as there."""
    sizes = _grouped_sizes(dy, w, offsets, counts, 1)
    return _rows_by_group("comfy_moe_grouped_matmul_dgrad", sizes, dy, w, offsets, counts, out, sizes[5])


def grouped_matmul_wgrad(dy: torch.Tensor, x: torch.Tensor, offsets: torch.Tensor, counts: Optional[torch.Tensor] = None,
                         out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``dw[g] = sum over the rows r of group g of dy[r].T x[r]``: the gradient of grouped_matmul for w.  dy [R, N],
    x [R, K] -> [G, N, K] in ``out_dtype`` (x's dtype, or fp32), summed in fp32."""
    if dy.dim() != 2 or x.dim() != 2 or dy.size(0) != x.size(0):
        raise ValueError(f"need dy [R, N] and x [R, K], got {tuple(dy.shape)} and {tuple(x.shape)}")
    if offsets.numel() == 0:
        raise ValueError("offsets must have one element more than there are groups")
    g, (r, n), k = offsets.numel() - 1, dy.shape, x.size(1)
    if not (r <= _MAX_ROWS and 0 < n <= _MAX_FEATURES and 0 < k <= _MAX_FEATURES):
        _refuse_sizes(r, n, k)
    index = _place(x, dy, offsets, counts, out)
    code = _HALF_CODES.get(x.dtype)
    if code is None or dy.dtype != x.dtype:
        raise ValueError(f"dy and x must both be bf16 or both fp16, got {dy.dtype} and {x.dtype}")
    _check_ragged(offsets, counts, g)
    dt = out_dtype or (x.dtype if out is None else out.dtype)
    if dt not in (x.dtype, torch.float32):
        raise ValueError(f"the gradient of the weights comes in {x.dtype} or fp32, not {dt}")
    res = x.new_empty((g, n, k), dtype=dt) if out is None else out
    if res.shape != (g, n, k) or res.dtype != dt:
        raise ValueError(f"out must be a {dt} tensor of shape {(g, n, k)}")
    if g == 0:
        return res
    unit = 16 // res.element_size()
    ld, step = _row_stride("out", res, unit), _group_stride("out", res, unit)
    if g > 1 and step < n * ld:
        raise ValueError("out: groups must not overlap")
    if out is not None:
        _check_apart(out, dy, x, offsets, counts)
    _call("comfy_moe_grouped_matmul_wgrad", index, dy.data_ptr(), _row_stride("dy", dy, 8), x.data_ptr(),
          _row_stride("x", x, 8), code, r, g, n, k, offsets.data_ptr(), _address(counts),
          N.FP32 if dt == torch.float32 else code, res.data_ptr(), ld, step, device_status(x.device).data_ptr())
    return res


class _GroupedMatmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, offsets, counts):
        need_x, need_w = ctx.needs_input_grad[:2]         # each gradient reads the other operand: keep no more than that
        ctx.save_for_backward(x if need_w else None, w if need_x else None, offsets, counts)
        ctx.sizes = sizes = _grouped_sizes(x, w, offsets, counts, 2)
        return _rows_by_group("comfy_moe_grouped_matmul", sizes, x, w, offsets, counts, None, sizes[4])

    @staticmethod
    def backward(ctx, dy):
        _once("grouped_matmul")
        x, w, offsets, counts = ctx.saved_tensors
        index, code, r, g, n, k, ld_x, ld_w, step = ctx.sizes
        need_x, need_w = ctx.needs_input_grad[:2]
        dy, dtype, vec = _readable(dy), dy.dtype, torch.int32
        if not (_unchanged(x, (r, k), (ld_x, 1), dtype, index, 16) and _unchanged(offsets, (g + 1,), (1,), vec, index) and
                _unchanged(w, (g, n, k), (step, ld_w, 1), dtype, index, 16) and _unchanged(counts, (g,), (1,), vec, index)):
            # a saved-tensor hook (offloading, compression) gave back something else: the checked calls look at it anew
            offsets, counts = _vector(offsets), _vector(counts)
            return (grouped_matmul_dgrad(dy, _readable(w), offsets, counts) if need_x else None,
                    grouped_matmul_wgrad(dy, _readable(x), offsets, counts) if need_w else None, None, None)
        ld_dy = n if r <= 1 else dy.stride()[0]
        dx = dw = None
        if need_x:
            sizes = (index, code, r, g, n, k, ld_dy, ld_w, step)
            dx = _rows_by_group("comfy_moe_grouped_matmul_dgrad", sizes, dy, w, offsets, counts, None, k)
        if need_w:
            dw = x.new_empty((g, n, k))
            if g:
                _call("comfy_moe_grouped_matmul_wgrad", index, dy.data_ptr(), ld_dy, x.data_ptr(), ld_x, code, r, g, n, k,
                      offsets.data_ptr(), _address(counts), code, dw.data_ptr(), k, n * k,
                      device_status(x.device).data_ptr())
        return dx, dw, None, None


# --------------------------------------------------------------------------------------- e4m3 with block scales
def _blocks(n: int) -> int:
    return -(-n // N.SCALE_BLOCK)


_QUANT_CODES = {torch.bfloat16: N.BF16, torch.float16: N.FP16, torch.float32: N.FP32}


def quantize_blocks_e4m3(x: torch.Tensor):
    """Rows x [R, K] (bf16, fp16 or fp32, K a multiple of 16) as (xq e4m3 [R, K], scale fp32 [R, ceil(K / 128)]): a block of
    128 elements of a row with the largest magnitude m = max(max|x|, 2^-100) holds e4m3(x * 448 / m), rounded to nearest
    even, and the scale m / 448.  ``scale`` is the transposed view of what the product reads."""
    index = _place(x)
    if x.dim() != 2 or x.dtype not in _QUANT_CODES or x.shape[1] == 0 or x.shape[1] % 16:
        raise ValueError("x must be [R, K] in bf16, fp16 or fp32 with K a multiple of 16")
    r, k = x.shape
    if r > _MAX_ROWS or k > _MAX_BLOCKED:
        _refuse_sizes(r, k) if r > _MAX_ROWS else _refuse_blocks(k)
    q = torch.empty((r, k), dtype=_FP8, device=x.device)
    scale = torch.empty((_blocks(k), r), dtype=torch.float32, device=x.device)
    _call("comfy_moe_block_quantize", index, x.data_ptr(), _row_stride("x", x, 16 // x.element_size()),
          _QUANT_CODES[x.dtype], r, k, q.data_ptr(), k, scale.data_ptr(), r)
    return q, scale.t()


def quantize_weight_blocks_e4m3(w: torch.Tensor):
    """Weights w [N, K] or [G, N, K] (bf16, fp16 or fp32, K a multiple of 16) as (wq e4m3 like w, scale fp32
    [.., ceil(N / 128), ceil(K / 128)]) with one scale for each 128 x 128 block, by the rule of quantize_blocks_e4m3."""
    index = _place(w)
    if w.dim() not in (2, 3) or w.dtype not in _QUANT_CODES or w.shape[-1] == 0 or w.shape[-1] % 16 or w.shape[-2] == 0:
        raise ValueError("w must be [N, K] or [G, N, K] in bf16, fp16 or fp32 with K a multiple of 16")
    n, k = w.shape[-2:]
    groups = w.shape[0] if w.dim() == 3 else 1
    if max(n, k, groups * N.SCALE_BLOCK) > _MAX_BLOCKED:
        _refuse_blocks(n, k, groups * N.SCALE_BLOCK)
    unit = 16 // w.element_size()
    q = torch.empty(w.shape, dtype=_FP8, device=w.device)
    scale = torch.empty(w.shape[:-2] + (_blocks(n), _blocks(k)), dtype=torch.float32, device=w.device)
    _call("comfy_moe_block_quantize_weight", index, w.data_ptr(), _row_stride("w", w, unit),
          _group_stride("w", w, unit) if w.dim() == 3 else 0, _QUANT_CODES[w.dtype], groups, n, k, q.data_ptr(),
          scale.data_ptr())
    return q, scale


def _block_sizes(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, offsets: Optional[torch.Tensor],
                 counts: Optional[torch.Tensor], bias: Optional[torch.Tensor], transpose: bool) -> tuple:
    """What the C entry point wants to know of checked operands: (device index, dtype code, rows, groups, N, K, row stride
    of x, row and group stride of w).  offsets None: one group, w [N, K]; transpose: x is a gradient [R, N]."""
    shape, weights = x.shape, w.shape
    if len(weights) != (2 if offsets is None else 3) or len(shape) != 2 or shape[1] != weights[-2 if transpose else -1]:
        raise ValueError(f"need rows and weights that fit, got {tuple(shape)} and {tuple(weights)}")
    index = _place(x, w, w_scale, offsets, counts, bias)
    code = _HALF_CODES.get(x.dtype)
    if code is None or w.dtype != _FP8:
        raise ValueError(f"rows must be bf16 or fp16 and weights e4m3, got {x.dtype} and {w.dtype}")
    (r, contraction), (n, k) = shape, weights[-2:]
    if n % 8 or k % 16 or contraction % 16 or n == 0 or k == 0:
        raise ValueError(f"in_features must be a multiple of 16 and out_features of 8 (of 16 for a gradient), got {k} and {n}")
    if r > _MAX_ROWS or n > _MAX_FEATURES or k > _MAX_FEATURES:
        _refuse_sizes(r, n, k)
    if contraction > _MAX_BLOCKED:
        _refuse_blocks(contraction)
    nb, kb = _blocks(n), _blocks(k)
    if w_scale.dtype != torch.float32 or w_scale.shape != ((nb, kb) if offsets is None else (weights[0], nb, kb)) or \
            not w_scale.is_contiguous():
        raise ValueError(f"the scales must be a contiguous fp32 tensor [.., {nb}, {kb}] for each group")
    groups = step = 1
    if offsets is not None:
        groups = weights[0]
        _check_ragged(offsets, counts, groups)
        step = _group_stride("weights", w, 16)
    if bias is not None and (bias.dtype != x.dtype or bias.shape != (n,) or not bias.is_contiguous() or
                             bias.data_ptr() % 16):
        raise ValueError("bias must be a contiguous vector over the output features in the rows' dtype")
    return index, code, r, groups, n, k, _row_stride("rows", x, 8), _row_stride("weights", w, 16), step


def _block_product(sizes: tuple, x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, offsets: Optional[torch.Tensor],
                   counts: Optional[torch.Tensor], bias: Optional[torch.Tensor], out: Optional[torch.Tensor],
                   transpose: bool) -> torch.Tensor:
    index, code, r, groups, n, k, ld_x, ld_w, step = sizes
    contraction, cols = (n, k) if transpose else (k, n)
    if out is None:
        res, ld = x.new_empty((r, cols)), cols
    else:
        res = _result(out, x, r, cols)
        ld = _row_stride("out", res, 8)
        _check_apart(res, x, w, w_scale, offsets, counts, bias)
    work = None
    if transpose or r > N.FEW_ROWS_BLOCK or k > N.FEW_ROWS_BLOCK_MAX_K:      # the quantised rows and their scales
        work = x.new_empty((r * contraction + 255) // 256 * 256 + 4 * r * _blocks(contraction), dtype=torch.uint8)
    _call("comfy_moe_block_matmul", index, x.data_ptr(), ld_x, code, _address(work), w.data_ptr(), ld_w, step,
          w_scale.data_ptr(), transpose, r, groups, n, k, _address(offsets), _address(counts), _address(bias), out is None,
          res.data_ptr(), ld, device_status(x.device).data_ptr())
    return res


def _asks_for_gradient(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias: Optional[torch.Tensor],
                       out: Optional[torch.Tensor]) -> bool:
    if not torch.is_grad_enabled():
        return False
    if w.requires_grad or w_scale.requires_grad:
        raise ValueError("block-scaled weights are frozen: neither they nor their scales have a gradient")
    if not x.requires_grad and (bias is None or not bias.requires_grad):
        return False
    if out is not None:
        raise ValueError("out cannot be given where a gradient is asked for")
    if x.requires_grad and w.dim() > 1 and w.size(-2) % 16:
        raise ValueError(f"out_features must be a multiple of 16 for a gradient of the rows, got {w.size(-2)}")
    return True


def block_linear(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ (w * scales).T + bias`` in e4m3: x [.., K] (bf16 or fp16) is quantised by blocks of 128 on the way
    (quantize_blocks_e4m3), w is e4m3 [N, K] with w_scale [ceil(N / 128), ceil(K / 128)] (quantize_weight_blocks_e4m3),
    bias [N] in x's dtype; K a multiple of 16, N of 8 (of 16 where a gradient of x is asked for); sums in fp32, result
    [.., N] in x's dtype.  Differentiable (once, in reverse mode) in x, whose gradient is the same product with the gradient
    of the result quantised and the weight transposed, and in bias; w is frozen."""
    if _forward_ad._current_level >= 0:
        _no_tangents("block_linear", x, w, w_scale, bias)
    rows = x
    if x.dim() != 2 or x.size(1) == 0:
        if x.dim() == 0 or x.size(-1) == 0:
            raise ValueError(f"need rows [.., K] and weights [N, K] that fit, got {tuple(x.shape)} and {tuple(w.shape)}")
        rows = x.reshape(-1, x.size(-1))
    if _asks_for_gradient(x, w, w_scale, bias, out):
        y = _BlockLinear.apply(rows, w, w_scale, bias)
    else:
        flat = out
        if out is not None and out.dim() != 2:
            flat = _rows_of(out, x.shape[:-1] + w.shape[:1])
        sizes = _block_sizes(rows, w, w_scale, None, None, bias, False)
        y = _block_product(sizes, rows, w, w_scale, None, None, bias, flat, False)
        if out is not None:
            return out
    return y if rows is x else y.view(x.shape[:-1] + (w.shape[0],))


def block_linear_dgrad(dy: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
                       out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``dy @ (w * scales)`` in e4m3: the gradient of block_linear for x.  dy [R, N] -> [R, K]; N a multiple of 16."""
    return _block_product(_block_sizes(dy, w, w_scale, None, None, None, True), dy, w, w_scale, None, None, None, out, True)


def grouped_block_linear(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, offsets: torch.Tensor,
                         counts: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """block_linear by expert: ``y[r] = x[r] @ (w[g] * scales[g]).T`` for the rows r of group g.  x [R, K], w e4m3
    [G, N, K], w_scale [G, ceil(N / 128), ceil(K / 128)]; offsets, counts, out and rows of no group as for grouped_matmul,
    the quantised rows and the gradient (x only) as for block_linear."""
    if _forward_ad._current_level >= 0:
        _no_tangents("grouped_block_linear", x, w, w_scale)
    if _asks_for_gradient(x, w, w_scale, None, out):
        return _GroupedBlockLinear.apply(x, w, w_scale, offsets, counts)
    sizes = _block_sizes(x, w, w_scale, offsets, counts, None, False)
    return _block_product(sizes, x, w, w_scale, offsets, counts, None, out, False)


def grouped_block_linear_dgrad(dy: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, offsets: torch.Tensor,
                               counts: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``dx[r] = dy[r] @ (w[g] * scales[g])``: the gradient of grouped_block_linear for x.  dy [R, N] -> [R, K]."""
    sizes = _block_sizes(dy, w, w_scale, offsets, counts, None, True)
    return _block_product(sizes, dy, w, w_scale, offsets, counts, None, out, True)


def _block_backward(ctx, dy: torch.Tensor, w, w_scale, offsets, counts) -> torch.Tensor:
    index, code, r, g, n, k, _, ld_w, step = ctx.sizes
    scales, vec = (-(-n // N.SCALE_BLOCK), -(-k // N.SCALE_BLOCK)), torch.int32
    if offsets is None:
        shape, strides = (n, k), (ld_w, 1)
    else:
        shape, strides, scales = (g, n, k), (step, ld_w, 1), (g, *scales)
    dy = _readable(dy)
    if _unchanged(w, shape, strides, _FP8, index, 16) and _unchanged(offsets, (g + 1,), (1,), vec, index) and \
            _unchanged(counts, (g,), (1,), vec, index) and w_scale.is_contiguous() and w_scale.shape == scales and \
            w_scale.dtype == torch.float32 and w_scale.get_device() == index:
        sizes = (index, code, r, g, n, k, n if r <= 1 else dy.stride()[0], ld_w, step)
    else:                                         # a saved-tensor hook gave back something else
        w, w_scale, offsets, counts = _readable(w), _vector(w_scale), _vector(offsets), _vector(counts)
        sizes = _block_sizes(dy, w, w_scale, offsets, counts, None, True)
    return _block_product(sizes, dy, w, w_scale, offsets, counts, None, None, True)


class _BlockLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, w_scale, bias):
        if ctx.needs_input_grad[0]:
            ctx.save_for_backward(w, w_scale)
        ctx.sizes = sizes = _block_sizes(x, w, w_scale, None, None, bias, False)
        return _block_product(sizes, x, w, w_scale, None, None, bias, None, False)

    @staticmethod
    def backward(ctx, dy):
        _once("block_linear")
        dx = _block_backward(ctx, dy, *ctx.saved_tensors, None, None) if ctx.needs_input_grad[0] else None
        db = dy.sum(0, dtype=torch.float32).to(dy.dtype) if ctx.needs_input_grad[3] else None
        return dx, None, None, db


class _GroupedBlockLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, w_scale, offsets, counts):
        ctx.save_for_backward(w, w_scale, offsets, counts)
        ctx.sizes = sizes = _block_sizes(x, w, w_scale, offsets, counts, None, False)
        return _block_product(sizes, x, w, w_scale, offsets, counts, None, None, False)

    @staticmethod
    def backward(ctx, dy):
        _once("grouped_block_linear")
        return _block_backward(ctx, dy, *ctx.saved_tensors), None, None, None, None
