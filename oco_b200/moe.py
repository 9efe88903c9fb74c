"""Host-side mirror of the reference's expert-layer operators over the C ABI.

Names and argument meaning follow the reference (Rust, `src/weights/compute/feed_forward.rs`,
`src/weights/compute/nemotron.rs`, `src/weights/state.rs`, `src/weights/gpt_oss.rs`,
`src/weights/nemotron.rs`):

    ExpertPlan.new(hidden, ffn_width)                      <- ExpertPlan::new
    ReluExpertPlan.new(hidden, expert_width, shared_width, experts, active, normalize, scale)
                                                          <- ReluExpertPlan::new
    Experts / ReluExperts                                  <- the weight structs (device buffers)
    Routing                                                <- Routing{ids, plan, prob}: side outputs
    Bindings(scratch).experts(w, plan, routing, residual, rows)
    Bindings(scratch).relu_experts(w, plan, routing, residual, rows)

The input rows are `scratch.norm` (bf16 [rows, hidden]) and the result is accumulated into the
bf16 residual rows in place, as in the reference. PyTorch is used only to own device memory and
streams; every computation happens inside liboco_moe.so.
"""
from __future__ import annotations

import ctypes as C
import struct
import warnings
from dataclasses import dataclass
from typing import Optional

import numpy as np
import torch

from . import _lib, synth
from ._lib import OcoError

ACTIVE_EXPERTS = 4   # reference src/weights/gpt_oss.rs:15
EXPERT_COUNT = 32    # reference src/weights/gpt_oss.rs:14


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else C.c_void_p(t.data_ptr())


# torch.cuda.current_stream() builds an object for the handle, 3 us a call; torch's own shortcut is not a public name
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream_ptr(device: Optional[int] = None):
    """The current stream of the current device (`device`: its number, where the caller has it already)."""
    if _raw_stream is None:
        return C.c_void_p(torch.cuda.current_stream().cuda_stream)
    return C.c_void_p(_raw_stream(torch.cuda.current_device() if device is None else device))


def _dev_bytes(a: Optional[np.ndarray], device, misalign: int = 0) -> Optional[torch.Tensor]:
    """Stages a host array on the device byte for byte (the GGUF spans stay unchanged).
    `misalign` places the first byte that many bytes past a 256-byte boundary, the way GGUF tensors
    sit at arbitrary offsets of a mapped file (reference test: src/weights/dispatch_tests/mxfp4.rs:16)."""
    if a is None:
        return None
    a = np.ascontiguousarray(a)
    with warnings.catch_warnings():
        # views of a read-only file map are only read here (copied to the device)
        warnings.simplefilter("ignore", UserWarning)
        flat = torch.from_numpy(a.view(np.uint8).reshape(-1))
    if not misalign:
        return flat.to(device)
    buf = torch.full((flat.numel() + misalign + 64,), 0xA5, dtype=torch.uint8, device=device)
    buf[misalign:misalign + flat.numel()] = flat.to(device)
    return buf[misalign:misalign + flat.numel()]


class StepGraph:
    """A recorded forward step (oco_moe_graph_*); keeps its plan and buffers alive."""

    def __init__(self, plan, handle, keep):
        self.plan, self.handle, self._keep = plan, handle, keep

    def replay(self):
        self.plan._check(_lib.lib().oco_moe_graph_launch(self.handle, _stream_ptr()))

    def __del__(self):
        try:
            if self.handle:
                _lib.lib().oco_moe_graph_destroy(self.handle)
                self.handle = C.c_void_p()
        except Exception:
            pass


class _Plan:
    """Owns the C plan object, its workspace and the bound weights."""

    def __init__(self, arch, hidden, ffn, experts, top_k, fmt, shared_ffn=0, normalize=False, scale=1.0,
                 gemm_impl=0, numerics=0):
        self.desc = _lib.Desc(arch=arch, hidden=hidden, ffn=ffn, experts=experts, top_k=top_k,
                              shared_ffn=shared_ffn, weight_format=fmt, normalize=int(bool(normalize)),
                              scale=float(scale), gemm_impl=gemm_impl, numerics=numerics)
        self.handle = C.c_void_p()
        rc = _lib.lib().oco_moe_plan_create(C.byref(self.desc), C.byref(self.handle))
        if rc != _lib.OK:
            msg = _lib.lib().oco_moe_last_error(self.handle).decode() if self.handle else "plan_create failed"
            if self.handle:
                _lib.lib().oco_moe_plan_destroy(self.handle)
                self.handle = C.c_void_p()
            raise OcoError(rc, msg)
        self.workspace = None
        self.max_rows = 0
        self._weights = None

    def _check(self, rc):
        if rc != _lib.OK:
            raise OcoError(rc, _lib.lib().oco_moe_last_error(self.handle).decode())

    def reserve(self, max_rows: int, device="cuda"):
        """Session-time workspace (reference `Memory::new`, src/weights/gpt_oss.rs:48-91)."""
        if self.workspace is not None and max_rows <= self.max_rows:
            return
        nbytes = _lib.lib().oco_moe_workspace_bytes(self.handle, max_rows)
        self.workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
        self._check(_lib.lib().oco_moe_bind_workspace(self.handle, _ptr(self.workspace), nbytes, max_rows))
        self.max_rows = max_rows

    def bind(self, w: "_Weights"):
        if self._weights is w:
            return
        cw = _lib.Weights(**{k: (getattr(w, k).data_ptr() if getattr(w, k) is not None else None)
                             for k, _ in _lib.Weights._fields_})
        self._check(_lib.lib().oco_moe_bind_weights(self.handle, C.byref(cw)))
        self._weights = w

    def forward(self, x: torch.Tensor, residual: torch.Tensor, rows: int):
        self._check(_lib.lib().oco_moe_forward(self.handle, _ptr(x), _ptr(residual), rows, _stream_ptr()))

    def add_norm_forward(self, hidden: torch.Tensor, projected: Optional[torch.Tensor], norm_weight: torch.Tensor,
                         epsilon: float, full_layer: bool, rows: int):
        """hidden += projected; x = rmsnorm(hidden) * norm_weight; hidden += MoE(x) (reference
        `Bindings::add_norm` + `Bindings::experts`, src/weights/compute.rs:100-117, gpt_oss.rs:122-123)."""
        self._check(_lib.lib().oco_moe_add_norm_forward(self.handle, _ptr(hidden), _ptr(projected) if projected is not None else None,
                                                        _ptr(norm_weight), C.c_float(epsilon), int(bool(full_layer)), rows,
                                                        _stream_ptr()))

    def forward_host(self, x: np.ndarray, residual: np.ndarray, rows: int):
        self._check(_lib.lib().oco_moe_forward_host(self.handle, x.ctypes.data_as(C.c_void_p),
                                                    residual.ctypes.data_as(C.c_void_p), rows, _stream_ptr()))

    def forward_host_begin(self, x: np.ndarray, residual: np.ndarray, rows: int):
        """Queue the layer on host buffers (up to two calls in flight); `residual` is the caller's again after
        the matching forward_host_end."""
        self._check(_lib.lib().oco_moe_forward_host_begin(self.handle, x.ctypes.data_as(C.c_void_p),
                                                          residual.ctypes.data_as(C.c_void_p), rows, _stream_ptr()))

    def forward_host_end(self):
        self._check(_lib.lib().oco_moe_forward_host_end(self.handle))

    def repack(self, device="cuda"):
        """The optional second form of the expert tensors for numerics 2 (oco_moe_bind_repacked)."""
        nbytes = _lib.lib().oco_moe_repack_bytes(self.handle)
        if nbytes == 0:
            raise OcoError(_lib.UNSUPPORTED_SHAPE, "this plan has no use for repacked weights")
        self._repacked = torch.empty(nbytes + 1024, dtype=torch.uint8, device=device)
        base = (self._repacked.data_ptr() + 1023) & ~1023
        self._check(_lib.lib().oco_moe_bind_repacked(self.handle, C.c_void_p(base), nbytes, _stream_ptr()))
        return base, nbytes

    def capture(self, x: torch.Tensor, residual: torch.Tensor, rows: int) -> "StepGraph":
        """The forward call on these buffers as a graph of the library (one launch per replay)."""
        g = C.c_void_p()
        self._check(_lib.lib().oco_moe_graph_capture(self.handle, _ptr(x), _ptr(residual), rows, C.byref(g)))
        return StepGraph(self, g, (x, residual))

    def capture_host(self, x: np.ndarray, residual: np.ndarray, rows: int) -> "StepGraph":
        """The forward call on these pinned host buffers, copies included, as a graph of the library."""
        g = C.c_void_p()
        self._check(_lib.lib().oco_moe_graph_capture_host(self.handle, x.ctypes.data_as(C.c_void_p),
                                                          residual.ctypes.data_as(C.c_void_p), rows, C.byref(g)))
        return StepGraph(self, g, (x, residual))

    def poll(self):
        self._check(_lib.lib().oco_moe_poll(self.handle, _stream_ptr()))

    def launch_count(self) -> int:
        return _lib.lib().oco_moe_last_launch_count(self.handle)

    def set_profiling(self, enabled: bool):
        """Per-kernel device timestamps (reference `OCO_PROFILE`, src/gpu/profile.rs)."""
        self._check(_lib.lib().oco_moe_set_profiling(self.handle, int(enabled)))

    def phase_times(self) -> dict:
        """Milliseconds per phase of the last forward call; the stream must have been waited for."""
        ms = (C.c_float * 16)()
        names = (C.c_char_p * 16)()
        n = _lib.lib().oco_moe_phase_times(self.handle, 16, ms, names)
        return {names[i].decode(): float(ms[i]) for i in range(max(n, 0))}

    def __del__(self):
        try:
            if self.handle:
                _lib.lib().oco_moe_plan_destroy(self.handle)
        except Exception:
            pass


class ExpertPlan(_Plan):
    """gpt-oss expert geometry (reference `ExpertPlan`, feed_forward.rs:34-77)."""

    @classmethod
    def new(cls, hidden: int, ffn_width: int, experts: int = EXPERT_COUNT, active: int = ACTIVE_EXPERTS,
            gemm_impl: int = 0, numerics: int = 0) -> "ExpertPlan":
        return cls(synth.ARCH_GPT_OSS, hidden, ffn_width, experts, active, synth.FMT_MXFP4, gemm_impl=gemm_impl, numerics=numerics)

    def width(self) -> int:
        return self.desc.ffn


class ReluExpertPlan(_Plan):
    """Routed relu^2 expert geometry (reference `ReluExpertPlan`, compute/nemotron.rs:131-198)."""

    @classmethod
    def new(cls, hidden, expert_width, shared_width, experts, active, normalize, scale, gemm_impl=0):
        return cls(synth.ARCH_NEMOTRON, hidden, expert_width, experts, active, synth.FMT_Q4_0,
                   shared_ffn=shared_width, normalize=normalize, scale=scale, gemm_impl=gemm_impl)

    def active(self) -> int:
        return self.desc.top_k

    def experts(self) -> int:
        return self.desc.experts

    def expert_width(self) -> int:
        return self.desc.ffn


class GatedExpertPlan(_Plan):
    """SiLU-gated Q4_K experts with softmax-all / top-k-renormalised routing (Qwen3-MoE shaped).
    The reference has no operator for this family; the plan follows the other two."""

    @classmethod
    def new(cls, hidden, expert_width, experts, active, gemm_impl=0):
        return cls(synth.ARCH_QWEN, hidden, expert_width, experts, active, synth.FMT_Q4_K, gemm_impl=gemm_impl)


@dataclass
class _Weights:
    router_w: Optional[torch.Tensor] = None
    router_b: Optional[torch.Tensor] = None
    gate_w: Optional[torch.Tensor] = None
    up_w: Optional[torch.Tensor] = None
    down_w: Optional[torch.Tensor] = None
    gate_b: Optional[torch.Tensor] = None
    up_b: Optional[torch.Tensor] = None
    down_b: Optional[torch.Tensor] = None
    shared_up_w: Optional[torch.Tensor] = None
    shared_down_w: Optional[torch.Tensor] = None
    gate_up_w: Optional[torch.Tensor] = None   # one tensor, rows interleaved: 2c = gate row c, 2c + 1 = up row c
    gate_up_b: Optional[torch.Tensor] = None

    @classmethod
    def from_layer(cls, layer: synth.Layer, device="cuda", misalign: int = 0, interleaved: bool = False):
        """Uploads a host layer unchanged (reference `import()` / `MappedRegions::new`,
        src/gpu/buffer.rs:151-194: the GGUF bytes are registered, never repacked). `misalign`
        applies to the packed expert banks only; f32 tensors keep their natural alignment.
        `interleaved` stages gate and up as one tensor with alternating rows (and biases)."""
        packed = ("gate_w", "up_w", "down_w", "shared_up_w", "shared_down_w")
        names = ["router_w", "router_b", "gate_w", "up_w", "down_w", "gate_b", "up_b", "down_b", "shared_up_w", "shared_down_w"]
        if interleaved and layer.gate_w is not None:
            E, F, rb = layer.gate_w.shape
            both = np.empty((E, 2 * F, rb), np.uint8)
            both[:, 0::2], both[:, 1::2] = layer.gate_w, layer.up_w
            out = cls(**{k: _dev_bytes(getattr(layer, k), device, misalign if k in packed else 0)
                         for k in names if k not in ("gate_w", "up_w", "gate_b", "up_b")})
            out.gate_up_w = _dev_bytes(both, device, misalign)
            if layer.gate_b is not None:
                bias = np.empty((E, 2 * F), np.float32)
                bias[:, 0::2], bias[:, 1::2] = layer.gate_b, layer.up_b
                out.gate_up_b = _dev_bytes(bias, device)
            return out
        return cls(**{k: _dev_bytes(getattr(layer, k), device, misalign if k in packed else 0) for k in names})


class Experts(_Weights):
    """reference `Experts{gate, up, down, router}` (src/weights/gpt_oss.rs:33-38)."""


class ReluExperts(_Weights):
    """reference `ReluExperts{router, up, down, shared_up, shared_down}` (src/weights/nemotron.rs:60-66)."""


def operand_order(fmt: int, n: int) -> np.ndarray:
    """Column of element k in rows kept in the tile kernels' operand order: a packed code byte holds
    elements j and j + h of its block (h = 16, or 32 for Q4_K), and the tiles keep the two adjacent."""
    k = np.arange(n)
    if fmt == synth.FMT_Q4_K:
        return (k & ~63) + (((k & 31) << 1) | ((k >> 5) & 1))
    return (k & ~31) + (((k & 15) << 1) | ((k >> 4) & 1))


class Routing:
    """Expert selections and combination weights of the last call (reference `Routing`,
    src/weights/state.rs:112-117), read back from the plan's workspace."""

    def __init__(self):
        self.plan: Optional[_Plan] = None
        self.rows = 0

    def _view(self):
        v = _lib.RoutingView()
        rc = _lib.lib().oco_moe_routing(self.plan.handle, C.byref(v))
        if rc != _lib.OK:
            raise OcoError(rc, "no routing available")
        return v

    def _read(self, ptr, count, dtype):
        out = np.empty(count, dtype)
        torch.cuda.current_stream().synchronize()
        rc = _lib.lib().oco_cuda_download(out.ctypes.data_as(C.c_void_p), C.c_void_p(ptr), out.nbytes, _stream_ptr())
        if rc != _lib.OK:
            raise OcoError(rc, "download failed")
        torch.cuda.current_stream().synchronize()
        return out

    def read(self) -> dict:
        d = self.plan.desc
        v = self._view()
        R = self.rows * d.top_k
        out = dict(ids=self._read(v.ids, R, np.uint32).reshape(self.rows, d.top_k),
                   prob=self._read(v.probs, R, np.float32).reshape(self.rows, d.top_k),
                   logits=self._read(v.logits, self.rows * d.experts, np.float32).reshape(self.rows, d.experts),
                   y=self._read(v.y, R * d.hidden, np.uint16).reshape(R, d.hidden),
                   norm=self._read(v.norm, self.rows * d.hidden, np.uint16).reshape(self.rows, d.hidden))
        if self.rows > 1:
            out["offsets"] = self._read(v.offsets, d.experts + 1, np.uint32)
            out["row_of_route"] = self._read(v.row_of_route, R, np.uint32)
            out["route_of_row"] = self._read(v.route_of_row, R, np.uint32)
            n = int(self._read(v.tile_count, 1, np.uint32)[0])
            out["tiles"] = self._read(v.tiles, 2 * n, np.uint32).reshape(n, 2)
            act = self._read(v.act, R * d.ffn, np.uint16).reshape(R, d.ffn)
            out["act"] = act[:, operand_order(d.weight_format, d.ffn)]   # back to element order
        return out


BF16, F32, IDS = (torch.bfloat16,), (torch.float32,), (torch.int32, torch.uint32)


def need(t: torch.Tensor, name: str, types: tuple, count: int, device: int):
    """Refuses a tensor that is not `count` or more contiguous elements of one of the types on the CUDA device of that
    number."""
    if t.get_device() != device or t.dtype not in types or not t.is_contiguous() or t.numel() < count:
        if device < 0 and t.is_cuda:
            raise OcoError(_lib.INVALID_ARGUMENT, "reserve a workspace first")
        raise OcoError(_lib.INVALID_ARGUMENT, f"{name}: a contiguous CUDA tensor of {count} elements of {types[0]} on cuda:{device} is needed, "
                                              f"got {tuple(t.shape)} {t.dtype} on {t.device}")


def _current_device() -> int:
    return torch.cuda.current_device() if torch.cuda.is_initialized() else -2


def same_device(weights, workspace: torch.Tensor):
    """Refuses a workspace on another device than the weights (a dict or tuple of tensors, or of pairs of them), whichever
    of the two came first."""
    for t in (weights.values() if isinstance(weights, dict) else weights or ()):
        for part in t if isinstance(t, tuple) else (t,):
            if part is not None and part.get_device() != workspace.get_device():
                raise OcoError(_lib.INVALID_ARGUMENT, f"the workspace is on {workspace.device}, the weights are on another device")


def _staged(a, device) -> torch.Tensor:
    if isinstance(a, np.ndarray):
        return _dev_bytes(a, device)
    return a if a.is_cuda else a.to(device)


def f8_matrix(codes, scales, lead, n: int, k: int, device, name: str):
    """Codes [*lead, n, k] of one byte and f32 scales [*lead, ceil(n / 128), ceil(k / 128)] on the device, checked."""
    if codes is None or scales is None:
        raise OcoError(_lib.INVALID_ARGUMENT, f"{name}: codes and scales are required")
    count, blocks = n * k, -(-n // 128) * -(-k // 128)
    for d in lead:
        count, blocks = count * d, blocks * d
    codes, scales = _staged(codes, device), _staged(scales, device)
    if scales.dtype == torch.uint8 and scales.numel() == 4 * blocks:      # bytes of a host array
        scales = scales.view(torch.float32)
    for t, types, want, what in ((codes, (torch.float8_e4m3fn, torch.uint8, torch.int8), count, "codes"), (scales, (torch.float32,), blocks, "scales")):
        if t.numel() != want or t.dtype not in types or not t.is_contiguous():
            raise OcoError(_lib.INVALID_ARGUMENT, f"{name} {what}: {want} contiguous elements of {types[0]} are needed, got {tuple(t.shape)} {t.dtype}")
    for t, what in ((codes, "codes"), (scales, "scales")):
        if t.get_device() != _current_device():
            raise OcoError(_lib.INVALID_ARGUMENT, f"{name} {what}: on {t.device}, the current device is cuda:{_current_device()}")
    return codes, scales


class _GroupPlan:
    """What the plans of grouped routing and of 8-bit float experts share: handle, workspace, errors."""
    _prefix = ""

    def _open(self, create, desc):
        self.desc, self.handle = desc, C.c_void_p()
        self._fn = {n: getattr(_lib.lib(), self._prefix + n) for n in ("workspace_bytes", "bind_workspace", "bind_weights", "forward", "poll",
                                                                      "last_error", "last_launch_count")}
        self.workspace, self.max_rows, self._weights, self._bias = None, 0, None, None
        self.device = -2                                                   # of the workspace
        rc = create(C.byref(desc), C.byref(self.handle))
        if rc != _lib.OK:
            raise OcoError(rc, self._fn["last_error"](self.handle).decode())

    def _check(self, rc):
        if rc != _lib.OK:
            raise OcoError(rc, self._fn["last_error"](self.handle).decode())

    def reserve(self, max_rows: int, device="cuda"):
        if self.workspace is not None and max_rows <= self.max_rows:
            return
        nbytes = self._fn["workspace_bytes"](self.handle, max_rows)
        ws = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=device)
        same_device(self._weights, ws)
        self._check(self._fn["bind_workspace"](self.handle, _ptr(ws), nbytes, max_rows))
        self.workspace, self.max_rows, self.device = ws, max_rows, ws.get_device()

    def poll(self):
        self._check(self._fn["poll"](self.handle, _stream_ptr()))

    def launch_count(self) -> int:
        return self._fn["last_launch_count"](self.handle)

    def __del__(self):
        try:
            if self.handle:
                getattr(_lib.lib(), self._destroy)(self.handle)
                self.handle = C.c_void_p()
        except Exception:
            pass


SCORES = {"sigmoid": 0, "softmax": 1}


class RouterPlan(_GroupPlan):
    """Routing with groups of experts (oco_moe_router_*): rows or logits -> expert ids and weights. The definition stands
    at the declarations in include/oco_moe.h."""
    _prefix, _destroy = "oco_moe_router_", "oco_moe_router_destroy"

    @classmethod
    def new(cls, hidden: int, experts: int, active: int, score: str = "sigmoid", groups: int = 1, top_groups: int = 1,
            group_best: int = 1, normalize: bool = True, scale: float = 1.0) -> "RouterPlan":
        """hidden 0: a plan that selects from given logits only."""
        if score not in SCORES:
            raise OcoError(_lib.INVALID_ARGUMENT, f"score is one of {sorted(SCORES)}")
        self = cls()
        self._open(_lib.lib().oco_moe_router_create,
                   _lib.RouterDesc(hidden=hidden, experts=experts, top_k=active, score=SCORES[score], groups=groups, top_groups=top_groups,
                                   group_best=group_best, normalize=int(bool(normalize)), scale=float(scale)))
        return self

    def bind(self, router_w: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None):
        """f32 CUDA tensors [experts, hidden] and [experts]; they must stay unchanged."""
        d = self.desc
        for t, name, count in ((router_w, "router_w", d.experts * d.hidden), (bias, "bias", d.experts)):
            if t is not None:
                need(t, name, F32, count, self.device if self.workspace is not None else _current_device())
        self._check(self._fn["bind_weights"](self.handle, _ptr(router_w), _ptr(bias)))
        self._weights, self._bias = (router_w, bias), bias

    def forward(self, x: torch.Tensor, ids: torch.Tensor, probs: torch.Tensor, rows: int, logits: Optional[torch.Tensor] = None):
        """x bf16 [rows, hidden] -> ids (32-bit) and probs f32 [rows, active], and the logits f32 [rows, experts] if asked for."""
        d, dev = self.desc, self.device
        k = rows * d.top_k
        need(x, "x", BF16, rows * d.hidden, dev)
        need(ids, "ids", IDS, k, dev)
        need(probs, "probs", F32, k, dev)
        if logits is not None:
            need(logits, "logits", F32, rows * d.experts, dev)
            logits = logits.data_ptr()
        rc = self._fn["forward"](self.handle, x.data_ptr(), rows, ids.data_ptr(), probs.data_ptr(), logits, _stream_ptr())
        if rc:
            self._check(rc)

    def select(self, logits: torch.Tensor, ids: torch.Tensor, probs: torch.Tensor, rows: int):
        """The selection alone, from logits f32 [rows, experts] of any origin."""
        d, dev = self.desc, _current_device()
        if self._bias is not None and self._bias.get_device() != dev:
            raise OcoError(_lib.INVALID_ARGUMENT, f"the bias is on {self._bias.device}, the current device is cuda:{dev}")
        k = rows * d.top_k
        need(logits, "logits", F32, rows * d.experts, dev)
        need(ids, "ids", IDS, k, dev)
        need(probs, "probs", F32, k, dev)
        rc = _lib.lib().oco_moe_router_select(self.handle, logits.data_ptr(), rows, ids.data_ptr(), probs.data_ptr(), _stream_ptr())
        if rc:
            self._check(rc)


@dataclass
class F8Experts:
    """Codes (e4m3, or their bytes) [experts, ffn, hidden] (gate, up) and [experts, hidden, ffn] (down) with the f32 scales
    [experts, ceil(rows / 128), ceil(columns / 128)] of the same matrices."""
    gate_w: object
    gate_s: object
    up_w: object
    up_s: object
    down_w: object
    down_s: object


class F8ExpertPlan(_GroupPlan):
    """SiLU-gated experts with e4m3 weights and block scales (oco_moe_f8_*)."""
    _prefix, _destroy = "oco_moe_f8_", "oco_moe_f8_plan_destroy"

    @classmethod
    def new(cls, hidden: int, ffn: int, experts: int, active: int) -> "F8ExpertPlan":
        self = cls()
        self._open(_lib.lib().oco_moe_f8_plan_create, _lib.F8Desc(hidden=hidden, ffn=ffn, experts=experts, top_k=active))
        return self

    def bind(self, w: F8Experts, device="cuda"):
        d = self.desc
        got = {}
        for name, n, k in (("gate", d.ffn, d.hidden), ("up", d.ffn, d.hidden), ("down", d.hidden, d.ffn)):
            got[name + "_w"], got[name + "_s"] = f8_matrix(getattr(w, name + "_w"), getattr(w, name + "_s"), (d.experts,), n, k, device, name)
        if self.workspace is not None:
            same_device(got, self.workspace)
        cw = _lib.F8Weights(**{n: t.data_ptr() for n, t in got.items()})
        self._check(self._fn["bind_weights"](self.handle, C.byref(cw)))
        self._weights = got

    def forward(self, x: torch.Tensor, ids: torch.Tensor, probs: torch.Tensor, residual: torch.Tensor, rows: int,
                out: Optional[torch.Tensor] = None):
        """out = residual + the weighted expert outputs (bf16 rows; out None: in place). Ids outside 0 .. experts - 1 are left out."""
        d, dev = self.desc, self.device
        out = residual if out is None else out
        n, k = rows * d.hidden, rows * d.top_k
        need(x, "x", BF16, n, dev)
        need(ids, "ids", IDS, k, dev)
        need(probs, "probs", F32, k, dev)
        need(residual, "residual", BF16, n, dev)
        need(out, "out", BF16, n, dev)
        rc = self._fn["forward"](self.handle, x.data_ptr(), ids.data_ptr(), probs.data_ptr(), residual.data_ptr(), out.data_ptr(), rows, _stream_ptr())
        if rc:
            self._check(rc)


_NORM_ARGS = struct.Struct("@6i4f9P5q")     # oco_moe_block_norm_args
NORMS = {"rms": 0, "layer": 1}
GATE_ACTS = {"none": 0, "sigmoid": 1, "tanh": 2}


def block_norm(hidden: torch.Tensor, block: Optional[torch.Tensor] = None, *, hidden_out: Optional[torch.Tensor] = None,
               norm_out: Optional[torch.Tensor] = None, pre_weight=None, pre_bias=None, post_weight=None, post_bias=None,
               gate: Optional[torch.Tensor] = None, gate_rows: Optional[int] = None, gate_act: str = "none", kind: str = "rms",
               weight_offset: float = 0.0, residual_scale: float = 1.0, block_scale: float = 1.0, epsilon: float = 1e-6):
    """The step between two blocks (oco_moe_block_norm): h = residual_scale * hidden + block_scale * act(gate) * post(block)
    into hidden_out, pre(h) into norm_out; hidden_out may be hidden, norm_out may be block. Rows are [rows, width] with unit
    stride inside a row; hidden bf16 or f32, block and norm_out bf16, weights f32 [width]. The gate is [width] (for all rows)
    or [gates, width], of which row r takes gate r // gate_rows (default: rows / gates), bf16 or f32."""
    def refuse(text):
        raise OcoError(_lib.INVALID_ARGUMENT, text)

    dev = hidden.get_device()
    wide = hidden.dtype is torch.float32
    if hidden.dim() != 2 or dev < 0 or not (wide or hidden.dtype is torch.bfloat16):
        refuse("hidden: CUDA rows [rows, width], bf16 or f32")
    if dev != (current := _current_device()):
        refuse(f"hidden is on {hidden.device}, the current device is cuda:{current}")
    rows, width = shape = hidden.shape
    if kind not in NORMS or gate_act not in GATE_ACTS:
        refuse(f"kind is one of {sorted(NORMS)}, gate_act one of {sorted(GATE_ACTS)}")

    for t, name, dtype in ((block, "block", torch.bfloat16), (hidden_out, "hidden_out", hidden.dtype), (norm_out, "norm_out", torch.bfloat16)):
        if t is not None and (t.shape != shape or t.dtype is not dtype or t.get_device() != dev):
            refuse(f"{name}: rows {tuple(shape)} of {dtype} on {hidden.device} are needed")
    strides = []
    for t in (hidden, block, hidden_out, norm_out):
        if t is None or t.is_contiguous():
            strides.append(0)
        elif t.stride(1) == 1:
            if 0 < rows != 1 and t.stride(0) < width:      # expanded rows: a stride of 0 would be read as the width
                refuse("the rows must not overlap")
            strides.append(t.stride(0) if rows > 1 else 0)
        else:
            refuse("the elements of a row must be neighbours")
    for t, name in ((post_weight, "post_weight"), (post_bias, "post_bias"), (pre_weight, "pre_weight"), (pre_bias, "pre_bias")):
        if t is not None:
            need(t, name, F32, width, dev)
    gs = gate_type = per = 0
    if gate is not None:
        if gate.dim() not in (1, 2) or gate.dtype not in (torch.bfloat16, torch.float32) or gate.get_device() != dev or gate.shape[-1] != width or gate.stride(-1) != 1:
            refuse("gate: [width] or [gates, width], bf16 or f32, unit stride inside a row")
        gate_type = 2 if gate.dtype is torch.float32 else 1
        if gate.dim() == 2:
            gates = gate.shape[0]
            per = gate_rows if gate_rows is not None else (rows // gates if gates and rows % gates == 0 else 0)
            if rows and (per < 1 or (rows - 1) // per >= gates):
                refuse("gate: fewer gate rows than the rows need")
            gs = gate.stride(0) if gates > 1 else 0
            if gates > 1 and gs == 0:                      # an expanded row: one gate for all
                per = 0
    at = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    args = _NORM_ARGS.pack(width, NORMS[kind], wide, gate_type, per, GATE_ACTS[gate_act], epsilon, weight_offset, residual_scale, block_scale,
                           hidden.data_ptr(), at(block), at(post_weight), at(post_bias), at(pre_weight), at(pre_bias), at(gate), at(hidden_out), at(norm_out),
                           strides[0], strides[1], gs, strides[2], strides[3])
    if rows == 0:      # an empty tensor has no address
        return
    rc = _lib.lib().oco_moe_block_norm(args, rows, _stream_ptr(dev), None, 0)
    if rc:
        err = C.create_string_buffer(160)
        if rc in (_lib.INVALID_ARGUMENT, _lib.UNSUPPORTED_SHAPE):      # refused before anything ran: asked again for the reason
            _lib.lib().oco_moe_block_norm(args, rows, _stream_ptr(dev), err, len(err))
        raise OcoError(rc, err.value.decode())


@dataclass
class Scratch:
    """The slice of the reference's `CommonScratch` this path reads (src/weights/state.rs:148-177)."""
    norm: torch.Tensor  # bf16 [rows, hidden]: the layer's input rows


class Bindings:
    """reference `Bindings{kernels, scratch, encoder}` (src/weights/compute.rs:58-62): the encoder
    is the current CUDA stream."""

    def __init__(self, scratch: Scratch):
        self.scratch = scratch

    def _run(self, w: _Weights, plan: _Plan, routing: Optional[Routing], residual: torch.Tensor, rows: int):
        if rows < 1:
            raise OcoError(_lib.INVALID_ARGUMENT, "rows must be at least 1")
        plan.reserve(max(rows, plan.max_rows), residual.device)
        plan.bind(w)
        plan.forward(self.scratch.norm, residual, rows)
        if routing is not None:
            routing.plan, routing.rows = plan, rows

    def experts(self, w: Experts, plan: ExpertPlan, routing: Optional[Routing], residual: torch.Tensor, rows: int):
        """Route each token to its experts and add their weighted contributions to its features
        (reference `Bindings::experts`, feed_forward.rs:106-114)."""
        self._run(w, plan, routing, residual, rows)

    def relu_experts(self, w: ReluExperts, plan: ReluExpertPlan, routing: Optional[Routing],
                     residual: torch.Tensor, rows: int):
        """Add the shared expert and the weighted routed experts to the residual rows
        (reference `Bindings::relu_experts`, compute/nemotron.rs:285-293)."""
        self._run(w, plan, routing, residual, rows)

    def gated_experts(self, w: _Weights, plan: GatedExpertPlan, routing: Optional[Routing],
                      residual: torch.Tensor, rows: int):
        self._run(w, plan, routing, residual, rows)


def plan_for(layer: synth.Layer, gemm_impl: int = 0, numerics: int = 0) -> _Plan:
    if layer.arch == synth.ARCH_GPT_OSS:
        return ExpertPlan.new(layer.hidden, layer.ffn, layer.experts, layer.top_k, gemm_impl, numerics)
    if layer.arch == synth.ARCH_NEMOTRON:
        return ReluExpertPlan.new(layer.hidden, layer.ffn, layer.shared_ffn, layer.experts, layer.top_k,
                                  layer.normalize, layer.scale, gemm_impl)
    return GatedExpertPlan.new(layer.hidden, layer.ffn, layer.experts, layer.top_k, gemm_impl)


def run_layer(layer: synth.Layer, x_bits: np.ndarray, residual_bits: np.ndarray, gemm_impl: int = 0,
              device="cuda", state: Optional[dict] = None, misalign: int = 0, interleaved: bool = False, numerics: int = 0,
              repacked: bool = False):
    """Convenience used by tests and the benchmark: uploads (or reuses) a layer, runs it on bf16
    bit patterns given as uint16 arrays and returns (residual bits, routing dict)."""
    state = state if state is not None else {}
    if "plan" not in state:
        state["plan"] = plan_for(layer, gemm_impl, numerics)
        state["weights"] = _Weights.from_layer(layer, device, misalign, interleaved)
    plan, w = state["plan"], state["weights"]
    if repacked and not state.get("repacked"):
        plan.reserve(x_bits.shape[0], device)
        plan.bind(w)
        plan.repack(device)
        state["repacked"] = True
    rows = x_bits.shape[0]
    x = torch.from_numpy(np.ascontiguousarray(x_bits).view(np.int16)).to(device)
    res = torch.from_numpy(np.ascontiguousarray(residual_bits).view(np.int16).copy()).to(device)
    routing = Routing()
    b = Bindings(Scratch(norm=x))
    b._run(w, plan, routing, res, rows)
    plan.poll()
    return res.cpu().numpy().view(np.uint16), routing.read()


def dequant(fmt: int, packed: np.ndarray, n_elems: int, half: bool = False, device="cuda") -> np.ndarray:
    w = _dev_bytes(packed, device)
    out = torch.empty(n_elems, dtype=torch.int16 if half else torch.float32, device=device)
    fn = _lib.lib().oco_moe_dequant_f16 if half else _lib.lib().oco_moe_dequant_f32
    rc = fn(fmt, _ptr(w), n_elems, _ptr(out), _stream_ptr())
    if rc != _lib.OK:
        raise OcoError(rc, "dequant failed")
    torch.cuda.synchronize()
    r = out.cpu().numpy()
    return r.view(np.uint16) if half else r
