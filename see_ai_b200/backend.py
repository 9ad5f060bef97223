"""ctypes binding of libsee_cuda.so and a thin `CudaBackend` mirroring the
reference's backend seam (Bind / BindSource / Execute / BeginRange / EndRange /
Flush; reference: runtime/executor/backend.h:82-166).

The library is the product; this module adds nothing to the arithmetic.  If the
shared library is missing, importing `CudaBackend` still works but constructing
one raises — there is no CPU path here.
"""

from __future__ import annotations

import ctypes
import os
from typing import Optional, Sequence

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libsee_cuda.so")

SEE_OK, SEE_ERROR, SEE_REFUSED = 0, 1, 2
COHERENCE_STRICT, COHERENCE_LAZY = 0, 1

# Every symbol include/see_cuda.h declares.
EXPORTED_SYMBOLS = [
    "see_cuda_create", "see_cuda_create_error", "see_cuda_destroy", "see_cuda_name",
    "see_cuda_device", "see_cuda_last_error", "see_cuda_bind", "see_cuda_bind_source",
    "see_cuda_begin_range", "see_cuda_execute", "see_cuda_end_range", "see_cuda_flush",
    "see_cuda_run_range", "see_cuda_set_coherence", "see_cuda_host_wrote",
    "see_cuda_host_needs", "see_cuda_counters_get", "see_cuda_set_stream",
    "see_cuda_device_arena", "see_cuda_set_relaxed_allowed", "see_cuda_set_epilogue_fusion",
    "see_cuda_set_gradient_gather",
    "see_cuda_set_profiling", "see_cuda_take_profile",
    "see_cuda_xent_forward_static", "see_cuda_static_max_rows", "see_cuda_static_last_error",
    "see_cuda_quantize_columns", "see_cuda_set_lora_fold", "see_cuda_set_product_groups", "see_cuda_set_adapter_fma", "see_cuda_set_split_gemm", "see_cuda_set_cta_pairs", "see_cuda_set_adapter_tensor_backward", "see_cuda_set_attention_one_walk",
    "see_cuda_set_attention_slices", "see_cuda_attention_slices",
    "see_cuda_norm_forward", "see_cuda_norm_backward", "see_cuda_norm_backward_workspace", "see_cuda_adamw_step",
    "see_cuda_gated_forward", "see_cuda_gated_backward", "see_cuda_gated_backward_workspace",
    "see_cuda_join_forward", "see_cuda_join_backward", "see_cuda_join_backward_workspace",
    "see_cuda_grad_norm", "see_cuda_grad_clip", "see_cuda_grad_workspace",
    "see_cuda_preference_loss", "see_cuda_preference_workspace", "see_cuda_policy_loss", "see_cuda_policy_workspace",
]

# Element types, norms and activations of the operators below.
F32, BF16, F16 = 0, 1, 2
TYPES = {"f32": F32, "bf16": BF16, "f16": F16}
NORM_LAYER, NORM_RMS = 0, 1
ACT_RELU, ACT_GELU, ACT_SILU = 1, 2, 3
ACTS = {"relu": ACT_RELU, "gelu": ACT_GELU, "silu": ACT_SILU}
ADAMW_BLOCK, ADAMW_NO_DECAY = 256, 1
PREFERENCE_SIGMOID, PREFERENCE_HINGE, PREFERENCE_SQUARE = 0, 1, 2
PREFERENCES = {"sigmoid": PREFERENCE_SIGMOID, "hinge": PREFERENCE_HINGE, "square": PREFERENCE_SQUARE}


class StepParams(ctypes.Structure):
    _fields_ = [("lr", ctypes.c_float), ("beta1", ctypes.c_float), ("beta2", ctypes.c_float),
                ("eps", ctypes.c_float), ("weight_decay", ctypes.c_float),
                ("pad", ctypes.c_uint32), ("step", ctypes.c_uint64)]


class Counters(ctypes.Structure):
    _fields_ = [(n, ctypes.c_uint64) for n in
                ("relaxed_executions", "fused_dispatches", "kernel_launches", "h2d_bytes",
                 "d2h_bytes", "instructions", "split_executions")]


class ProfileRecord(ctypes.Structure):
    _fields_ = [("opcode", ctypes.c_uint16), ("absorbed", ctypes.c_uint16), ("index", ctypes.c_uint32),
                ("ms", ctypes.c_float), ("kernel_ms", ctypes.c_float), ("m", ctypes.c_uint64),
                ("n", ctypes.c_uint64), ("k", ctypes.c_uint64)]


class NormShape(ctypes.Structure):
    _fields_ = [("kind", ctypes.c_int32), ("x_type", ctypes.c_int32), ("y_type", ctypes.c_int32), ("eps", ctypes.c_float),
                ("rows", ctypes.c_uint64), ("cols", ctypes.c_uint64), ("x_stride", ctypes.c_uint64),
                ("y_stride", ctypes.c_uint64)]


class GatedShape(ctypes.Structure):
    _fields_ = [("type", ctypes.c_int32), ("act", ctypes.c_int32)] + [
        (n, ctypes.c_uint64) for n in ("rows", "d_in", "d_hidden", "x_stride", "hidden_stride")]


class AdamWTensor(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("p", "g", "m", "v", "m_scale", "v_scale", "copy")] + [
        ("n", ctypes.c_uint64), ("g_type", ctypes.c_int32), ("copy_type", ctypes.c_int32), ("flags", ctypes.c_uint32),
        ("pad", ctypes.c_uint32)]


class GradTensor(ctypes.Structure):
    _fields_ = [("g", ctypes.c_void_p), ("out", ctypes.c_void_p), ("n", ctypes.c_uint64), ("type", ctypes.c_int32),
                ("pad", ctypes.c_uint32)]


class JoinShape(ctypes.Structure):
    _fields_ = [("kind", ctypes.c_int32), ("x_type", ctypes.c_int32), ("y_type", ctypes.c_int32), ("eps", ctypes.c_float),
                ("residual_scale", ctypes.c_float), ("pad", ctypes.c_uint32)] + [
        (n, ctypes.c_uint64) for n in ("rows", "cols", "x_stride", "y_stride")]


class JoinWeights(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("post_gamma", "post_beta", "gate", "pre_gamma", "pre_beta")]


class JoinStats(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("post_mean", "post_rstd", "pre_mean", "pre_rstd")]


class PreferenceShape(ctypes.Structure):
    _fields_ = [("type", ctypes.c_int32), ("kind", ctypes.c_int32)] + [
        (n, ctypes.c_float) for n in ("beta", "smoothing", "margin", "logit_scale")] + [
        ("average", ctypes.c_int32), ("pad", ctypes.c_uint32)] + [(n, ctypes.c_uint64) for n in ("rows", "classes", "stride", "pairs")]


class PolicyShape(ctypes.Structure):
    _fields_ = [("type", ctypes.c_int32)] + [(n, ctypes.c_float) for n in ("logit_scale", "clip_low", "clip_high", "kl_coef")] + [
        ("pad", ctypes.c_uint32)] + [(n, ctypes.c_uint64) for n in ("rows", "classes", "stride")]


class BackendError(RuntimeError):
    pass


class Refusal(BackendError):
    """The step was refused (non-finite gradient norm or a bad clip threshold)."""


_lib = None


def load_library() -> ctypes.CDLL:
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise BackendError(
            f"{LIB_PATH} is missing: build it with `python -m see_ai_b200.build` "
            "(there is no CPU fallback)")
    lib = ctypes.CDLL(LIB_PATH)
    vp, u64, i32 = ctypes.c_void_p, ctypes.c_uint64, ctypes.c_int
    lib.see_cuda_create.argtypes = [i32, ctypes.POINTER(vp)]
    lib.see_cuda_create_error.restype = ctypes.c_char_p
    lib.see_cuda_destroy.argtypes = [vp]
    lib.see_cuda_destroy.restype = None
    for name in ("see_cuda_name", "see_cuda_device", "see_cuda_last_error"):
        getattr(lib, name).argtypes = [vp]
        getattr(lib, name).restype = ctypes.c_char_p
    lib.see_cuda_bind.argtypes = [vp, vp, u64, vp, u64]
    lib.see_cuda_bind_source.argtypes = [vp, vp, u64]
    lib.see_cuda_begin_range.argtypes = [vp, vp, u64, u64, u64]
    lib.see_cuda_execute.argtypes = [vp, vp, ctypes.POINTER(StepParams)]
    lib.see_cuda_end_range.argtypes = [vp]
    lib.see_cuda_flush.argtypes = [vp]
    lib.see_cuda_run_range.argtypes = [vp, vp, u64, u64, u64, ctypes.POINTER(StepParams),
                                       ctypes.POINTER(u64)]
    lib.see_cuda_set_coherence.argtypes = [vp, i32]
    lib.see_cuda_host_wrote.argtypes = [vp, u64, u64]
    lib.see_cuda_host_needs.argtypes = [vp, u64, u64]
    lib.see_cuda_counters_get.argtypes = [vp, ctypes.POINTER(Counters)]
    lib.see_cuda_set_stream.argtypes = [vp, vp]
    lib.see_cuda_device_arena.argtypes = [vp]
    lib.see_cuda_device_arena.restype = vp
    lib.see_cuda_set_relaxed_allowed.argtypes = [vp, i32]
    lib.see_cuda_set_epilogue_fusion.argtypes = [vp, i32]
    lib.see_cuda_set_gradient_gather.argtypes = [vp, i32, vp, u64, u64]
    lib.see_cuda_set_profiling.argtypes = [vp, i32]
    lib.see_cuda_take_profile.argtypes = [vp, ctypes.POINTER(ProfileRecord), u64]
    lib.see_cuda_take_profile.restype = ctypes.c_int64
    lib.see_cuda_quantize_columns.argtypes = [vp, vp, u64, u64, vp, vp]
    lib.see_cuda_set_lora_fold.argtypes = [vp, i32]
    lib.see_cuda_set_product_groups.argtypes = [vp, i32]
    lib.see_cuda_set_adapter_fma.argtypes = [vp, i32]
    lib.see_cuda_set_split_gemm.argtypes = [vp, i32]
    lib.see_cuda_set_cta_pairs.argtypes = [i32]
    lib.see_cuda_set_adapter_tensor_backward.argtypes = [i32]
    lib.see_cuda_set_attention_one_walk.argtypes = [vp, i32]
    lib.see_cuda_set_attention_slices.argtypes = [vp, i32]
    lib.see_cuda_attention_slices.argtypes = [vp]
    lib.see_cuda_attention_slices.restype = u64
    lib.see_cuda_norm_forward.argtypes = [vp, ctypes.POINTER(NormShape)] + [vp] * 6
    lib.see_cuda_norm_backward.argtypes = [vp, ctypes.POINTER(NormShape)] + [vp] * 10 + [u64]
    lib.see_cuda_norm_backward_workspace.argtypes = [u64, u64]
    lib.see_cuda_norm_backward_workspace.restype = u64
    lib.see_cuda_gated_forward.argtypes = [vp, ctypes.POINTER(GatedShape)] + [vp] * 6
    lib.see_cuda_gated_backward.argtypes = [vp, ctypes.POINTER(GatedShape)] + [vp] * 10 + [u64]
    lib.see_cuda_gated_backward_workspace.argtypes = [u64, u64, u64]
    lib.see_cuda_gated_backward_workspace.restype = u64
    lib.see_cuda_adamw_step.argtypes = [vp, ctypes.POINTER(AdamWTensor), u64, i32, ctypes.POINTER(StepParams), vp]
    lib.see_cuda_join_forward.argtypes = [vp, ctypes.POINTER(JoinShape), vp, vp, ctypes.POINTER(JoinWeights), vp, vp, ctypes.POINTER(JoinStats)]
    lib.see_cuda_join_backward.argtypes = [vp, ctypes.POINTER(JoinShape)] + [vp] * 4 + [
        ctypes.POINTER(JoinWeights), ctypes.POINTER(JoinStats), vp, vp, ctypes.POINTER(JoinWeights), vp, u64]
    lib.see_cuda_join_backward_workspace.argtypes = [u64, u64]
    lib.see_cuda_join_backward_workspace.restype = u64
    lib.see_cuda_preference_loss.argtypes = [vp, ctypes.POINTER(PreferenceShape)] + [vp] * 10 + [u64]
    lib.see_cuda_preference_workspace.argtypes = [u64, u64]
    lib.see_cuda_preference_workspace.restype = u64
    lib.see_cuda_policy_loss.argtypes = [vp, ctypes.POINTER(PolicyShape)] + [vp] * 11 + [u64]
    lib.see_cuda_policy_workspace.argtypes = [u64]
    lib.see_cuda_policy_workspace.restype = u64
    for name in ("see_cuda_grad_norm", "see_cuda_grad_clip"):
        getattr(lib, name).argtypes = [vp, ctypes.POINTER(GradTensor), u64, ctypes.c_float] + [vp] * 4 + [u64]
    lib.see_cuda_grad_workspace.argtypes = []
    lib.see_cuda_grad_workspace.restype = u64
    lib.see_cuda_xent_forward_static.argtypes = [vp, vp, vp, vp, u64, u64, i32, vp]
    lib.see_cuda_static_max_rows.restype = u64
    lib.see_cuda_static_last_error.restype = ctypes.c_char_p
    _lib = lib
    return lib


def xent_forward_static(logits_ptr: int, labels_ptr: int, loss_ptr: int, probs_ptr: int,
                        rows: int, classes: int, masked: bool = False, stream: int = 0) -> None:
    """Softmax cross-entropy forward over DEVICE pointers with no allocation:
    the scratch is a fixed array inside the library (at most
    see_cuda_static_max_rows() rows).  For callers that may not call cudaMalloc."""
    lib = load_library()
    rc = lib.see_cuda_xent_forward_static(ctypes.c_void_p(logits_ptr), ctypes.c_void_p(labels_ptr),
                                          ctypes.c_void_p(loss_ptr), ctypes.c_void_p(probs_ptr),
                                          rows, classes, int(masked), ctypes.c_void_p(stream))
    if rc != SEE_OK:
        raise BackendError(lib.see_cuda_static_last_error().decode())


def norm_backward_workspace(rows: int, cols: int) -> int:
    """Bytes that `CudaBackend.norm_backward` needs beside its operands."""
    return int(load_library().see_cuda_norm_backward_workspace(rows, cols))


def gated_backward_workspace(rows: int, d_in: int, d_hidden: int) -> int:
    """Bytes that `CudaBackend.gated_backward` needs beside its operands."""
    return int(load_library().see_cuda_gated_backward_workspace(rows, d_in, d_hidden))


def adamw_tensors(tensors):
    """The table `CudaBackend.adamw_step` takes, of dicts of DEVICE pointers p, g, m, v (and m_scale, v_scale with 8-bit
    moments; copy), the number of elements n, g_type, copy_type and no_decay."""
    table = (AdamWTensor * len(tensors))()
    for entry, t in zip(table, tensors):
        for key in ("p", "g", "m", "v", "m_scale", "v_scale", "copy"):
            setattr(entry, key, t.get(key) or None)
        entry.n, entry.g_type, entry.copy_type = t["n"], t.get("g_type", F32), t.get("copy_type", F32)
        entry.flags = ADAMW_NO_DECAY if t.get("no_decay") else 0
    return table


def join_backward_workspace(rows: int, cols: int) -> int:
    """Bytes that `CudaBackend.join_backward` needs beside its operands."""
    return int(load_library().see_cuda_join_backward_workspace(rows, cols))


def join_weights(pre_gamma: int, pre_beta: int = 0, gate: int = 0, post_gamma: int = 0, post_beta: int = 0):
    """The weights `CudaBackend.join_forward` and `join_backward` take, or their gradients: DEVICE pointers, 0 for what is not there."""
    return JoinWeights(post_gamma or None, post_beta or None, gate or None, pre_gamma or None, pre_beta or None)


def join_stats(pre_rstd: int, pre_mean: int = 0, post_rstd: int = 0, post_mean: int = 0):
    """Where `CudaBackend.join_forward` keeps each row's statistics for `join_backward`: DEVICE pointers, 0 for what is not there."""
    return JoinStats(post_mean or None, post_rstd or None, pre_mean or None, pre_rstd or None)


def preference_workspace(rows: int, pairs: int) -> int:
    """Bytes that `CudaBackend.preference_loss` needs beside its operands."""
    return int(load_library().see_cuda_preference_workspace(rows, pairs))


def policy_workspace(rows: int) -> int:
    """Bytes that `CudaBackend.policy_loss` needs beside its operands."""
    return int(load_library().see_cuda_policy_workspace(rows))


def grad_workspace() -> int:
    """Bytes that `CudaBackend.grad_norm` and `grad_clip` need beside their operands."""
    return int(load_library().see_cuda_grad_workspace())


def grad_tensors(tensors):
    """The table `CudaBackend.grad_norm` and `grad_clip` take, of dicts of DEVICE pointers g (and out, where the clipped
    gradients go; 0 or left out: g itself), the number of elements n and their type."""
    table = (GradTensor * len(tensors))()
    for entry, t in zip(table, tensors):
        entry.g, entry.out, entry.n, entry.type = t.get("g") or None, t.get("out") or None, t["n"], t.get("type", F32)
    return table


def program_bytes(program) -> bytes:
    if isinstance(program, (bytes, bytearray, memoryview)):
        return bytes(program)
    return b"".join(i.pack() for i in program)


class CudaBackend:
    """One handle per GPU.  `arena` passed to bind() is mutated in place by
    flush() (strict coherence) or host_needs() (lazy)."""

    def __init__(self, device: int = 0):
        self.lib = load_library()
        h = ctypes.c_void_p()
        if self.lib.see_cuda_create(device, ctypes.byref(h)) != SEE_OK:
            raise BackendError(self.lib.see_cuda_create_error().decode())
        self.h = h
        self._keep = []
        self._prog = None

    def close(self):
        if getattr(self, "h", None):
            self.lib.see_cuda_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check(self, rc: int):
        if rc == SEE_OK:
            return
        msg = self.lib.see_cuda_last_error(self.h).decode()
        raise (Refusal if rc == SEE_REFUSED else BackendError)(msg)

    @property
    def name(self) -> str:
        return self.lib.see_cuda_name(self.h).decode()

    @property
    def device(self) -> str:
        return self.lib.see_cuda_device(self.h).decode()

    def bind(self, arena: np.ndarray, rodata: Optional[np.ndarray] = None):
        assert arena.dtype == np.uint8 and arena.flags.c_contiguous
        if rodata is not None:
            rodata = np.ascontiguousarray(rodata)
        self._keep = [arena, rodata]
        self._check(self.lib.see_cuda_bind(
            self.h, arena.ctypes.data, arena.size,
            rodata.ctypes.data if rodata is not None and rodata.size else None,
            rodata.size if rodata is not None else 0))

    def bind_source(self, data: Optional[np.ndarray]):
        if data is None:
            self._check(self.lib.see_cuda_bind_source(self.h, None, 0))
            return
        data = np.ascontiguousarray(data)
        self._check(self.lib.see_cuda_bind_source(self.h, data.ctypes.data, data.size))

    def set_program(self, program):
        raw = program_bytes(program)
        self._prog = (ctypes.create_string_buffer(raw, len(raw)), len(raw) // 64)

    def run(self, program=None, params: Optional[StepParams] = None, begin: int = 0,
            end: Optional[int] = None):
        """BeginRange, Execute each instruction of [begin, end), Flush, EndRange."""
        if program is not None:
            self.set_program(program)
        buf, n = self._prog
        end = n if end is None else end
        params = params or StepParams(1e-3, 0.9, 0.999, 1e-8, 0.01, 0, 1)
        failed = ctypes.c_uint64(0)
        self._check(self.lib.see_cuda_run_range(self.h, buf, n, begin, end, ctypes.byref(params),
                                                ctypes.byref(failed)))

    def begin_range(self, begin: int, end: int):
        buf, n = self._prog
        self._check(self.lib.see_cuda_begin_range(self.h, buf, n, begin, end))

    def execute(self, index: int, params: StepParams):
        buf, n = self._prog
        ptr = ctypes.cast(ctypes.addressof(buf) + 64 * index, ctypes.c_void_p)
        self._check(self.lib.see_cuda_execute(self.h, ptr, ctypes.byref(params)))

    def end_range(self):
        self._check(self.lib.see_cuda_end_range(self.h))

    def flush(self):
        self._check(self.lib.see_cuda_flush(self.h))

    def set_coherence(self, mode: int):
        self._check(self.lib.see_cuda_set_coherence(self.h, mode))

    def host_wrote(self, offset: int, nbytes: int):
        self._check(self.lib.see_cuda_host_wrote(self.h, offset, nbytes))

    def host_needs(self, offset: int, nbytes: int):
        self._check(self.lib.see_cuda_host_needs(self.h, offset, nbytes))

    def counters(self) -> Counters:
        c = Counters()
        self._check(self.lib.see_cuda_counters_get(self.h, ctypes.byref(c)))
        return c

    def set_stream(self, stream_handle: int):
        self._check(self.lib.see_cuda_set_stream(self.h, ctypes.c_void_p(stream_handle)))

    def device_arena(self) -> int:
        return int(self.lib.see_cuda_device_arena(self.h) or 0)

    def set_relaxed_allowed(self, allowed: bool):
        self._check(self.lib.see_cuda_set_relaxed_allowed(self.h, int(allowed)))

    def set_epilogue_fusion(self, enabled: bool):
        self._check(self.lib.see_cuda_set_epilogue_fusion(self.h, int(enabled)))

    def set_product_groups(self, enabled: bool):
        self._check(self.lib.see_cuda_set_product_groups(self.h, int(enabled)))

    def set_lora_fold(self, enabled: bool):
        self._check(self.lib.see_cuda_set_lora_fold(self.h, int(enabled)))

    def set_adapter_fma(self, enabled: bool):
        self._check(self.lib.see_cuda_set_adapter_fma(self.h, int(enabled)))

    def set_split_gemm(self, mode: int):
        """-1: exact f32 products on the tensor cores in lazy coherence only; 0 never; 1 always."""
        self._check(self.lib.see_cuda_set_split_gemm(self.h, mode))

    def set_attention_one_walk(self, enabled: bool):
        self._check(self.lib.see_cuda_set_attention_one_walk(self.h, int(enabled)))

    def set_attention_slices(self, use: int):
        """0: exact attention never by digits on the tensor cores; 1: where that is the shorter way; 2: wherever it can be."""
        self._check(self.lib.see_cuda_set_attention_slices(self.h, use))

    def attention_slices(self) -> int:
        """Instructions that ran so since creation."""
        return int(self.lib.see_cuda_attention_slices(self.h))

    def set_cta_pairs(self, enabled: bool):
        """Process-wide: large tensor-core products on CTA pairs (default) or one CTA per tile."""
        self._check(self.lib.see_cuda_set_cta_pairs(int(enabled)))

    def set_adapter_tensor_backward(self, enabled: bool):
        """Process-wide: adapter backward sites on the tcgen05 tensor cores (default) or the legacy instruction."""
        self._check(self.lib.see_cuda_set_adapter_tensor_backward(int(enabled)))

    def set_gradient_gather(self, ranks: int, gathered_ptr: int, block_offset: int,
                            block_bytes: int):
        self._check(self.lib.see_cuda_set_gradient_gather(
            self.h, ranks, ctypes.c_void_p(gathered_ptr), block_offset, block_bytes))

    def quantize_columns(self, w_ptr: int, K: int, N: int, levels_ptr: int, scales_ptr: int):
        """Per-column int8 quantisation of W [K, N] over DEVICE pointers."""
        self._check(self.lib.see_cuda_quantize_columns(self.h, ctypes.c_void_p(w_ptr), K, N,
                                                       ctypes.c_void_p(levels_ptr), ctypes.c_void_p(scales_ptr)))

    def norm_forward(self, kind: int, rows: int, cols: int, x: int, gamma: int, beta: int, y: int, mean: int, rstd: int,
                     x_type: int = F32, y_type: int = F32, eps: float = 1e-5, x_stride: int = 0, y_stride: int = 0):
        """Layer norm (NORM_LAYER) or root-mean-square norm (NORM_RMS: beta and mean are 0) over DEVICE pointers."""
        shape = NormShape(kind, x_type, y_type, eps, rows, cols, x_stride, y_stride)
        self._check(self.lib.see_cuda_norm_forward(self.h, shape, x or None, gamma or None, beta or None, y or None, mean or None,
                                                   rstd or None))

    def norm_backward(self, kind: int, rows: int, cols: int, dy: int, x: int, gamma: int, mean: int, rstd: int, dx: int,
                      dgamma: int, dbeta: int, workspace: int, workspace_bytes: int, addend: int = 0, x_type: int = F32,
                      y_type: int = F32, x_stride: int = 0, y_stride: int = 0):
        """Its backward pass with the gradients of gamma and beta (NORM_RMS: mean and dbeta are 0); `addend` joins dx.
        The workspace has norm_backward_workspace(rows, cols) bytes."""
        shape = NormShape(kind, x_type, y_type, 0.0, rows, cols, x_stride, y_stride)
        self._check(self.lib.see_cuda_norm_backward(self.h, shape, dy or None, x or None, gamma or None, mean or None, rstd or None,
                                                    addend or None, dx or None, dgamma or None, dbeta or None, workspace or None,
                                                    workspace_bytes))

    def gated_forward(self, rows: int, d_in: int, d_hidden: int, x: int, w_gate: int, w_up: int, hidden: int, gate: int = 0,
                      up: int = 0, type: int = BF16, act: int = ACT_SILU, x_stride: int = 0, hidden_stride: int = 0):
        """hidden = act(x w_gate) * (x w_up) over DEVICE pointers of a 16-bit type; gate and up are the two products, kept for
        the backward pass (0: not kept)."""
        shape = GatedShape(type, act, rows, d_in, d_hidden, x_stride, hidden_stride)
        self._check(self.lib.see_cuda_gated_forward(self.h, shape, x or None, w_gate or None, w_up or None, hidden or None,
                                                    gate or None, up or None))

    def gated_backward(self, rows: int, d_in: int, d_hidden: int, dhidden: int, x: int, w_gate: int, w_up: int, gate: int, up: int,
                       dx: int, dw_gate: int, dw_up: int, workspace: int, workspace_bytes: int, type: int = BF16,
                       act: int = ACT_SILU, x_stride: int = 0, hidden_stride: int = 0):
        """Its backward pass; dx, or dw_gate and dw_up, may be 0 (not wanted).  The workspace has
        gated_backward_workspace(rows, d_in, d_hidden) bytes."""
        shape = GatedShape(type, act, rows, d_in, d_hidden, x_stride, hidden_stride)
        self._check(self.lib.see_cuda_gated_backward(self.h, shape, dhidden or None, x or None, w_gate or None, w_up or None,
                                                     gate or None, up or None, dx or None, dw_gate or None, dw_up or None,
                                                     workspace or None, workspace_bytes))

    def adamw_step(self, tensors, params: StepParams, state_bits: int = 32, grad_scale: int = 0):
        """One AdamW step over a table of adamw_tensors, moments in 8 bits or in 32."""
        self._check(self.lib.see_cuda_adamw_step(self.h, tensors, len(tensors), state_bits, params, grad_scale or None))

    def join_forward(self, kind: int, rows: int, cols: int, x: int, block: int, weights: JoinWeights, x_out: int, y: int, stats: JoinStats,
                     x_type: int = F32, y_type: int = F32, eps: float = 1e-5, residual_scale: float = 1.0, x_stride: int = 0, y_stride: int = 0):
        """x_out = residual_scale x + gate * N1(block), y = N2(x_out) over DEVICE pointers: the norm after a block (join_weights without
        post_gamma: none), its gate (without gate: 1), the scaled residual and the norm before the next block."""
        shape = JoinShape(kind, x_type, y_type, eps, residual_scale, 0, rows, cols, x_stride, y_stride)
        self._check(self.lib.see_cuda_join_forward(self.h, shape, x or None, block or None, weights, x_out or None, y or None, stats))

    def join_backward(self, kind: int, rows: int, cols: int, dy: int, dx_out: int, x_out: int, block: int, weights: JoinWeights,
                      stats: JoinStats, dx: int, dblock: int, gradients: JoinWeights, workspace: int, workspace_bytes: int,
                      x_type: int = F32, y_type: int = F32, residual_scale: float = 1.0, x_stride: int = 0, y_stride: int = 0):
        """Its backward pass with the gradients of the weights; `dx_out` is what reaches x_out past the norm (0: nothing).  The
        workspace has join_backward_workspace(rows, cols) bytes."""
        shape = JoinShape(kind, x_type, y_type, 0.0, residual_scale, 0, rows, cols, x_stride, y_stride)
        self._check(self.lib.see_cuda_join_backward(self.h, shape, dy or None, dx_out or None, x_out or None, block or None, weights, stats,
                                                    dx or None, dblock or None, gradients, workspace or None, workspace_bytes))

    def preference_loss(self, rows: int, classes: int, pairs: int, logits: int, labels: int, starts: int, loss: int, margins: int,
                        sequence_logp: int, workspace: int, workspace_bytes: int, ref_logp: int = 0, loss_grad: int = 0, dlogits: int = 0,
                        type: int = F32, kind: int = PREFERENCE_SIGMOID, beta: float = 0.1, smoothing: float = 0.0, margin: float = 0.0,
                        logit_scale: float = 1.0, average: bool = False, stride: int = 0):
        """A preference loss of `pairs` of sequences (2 i chosen, 2 i + 1 rejected; sequence s is the rows starts[s] up to
        starts[s + 1]) over DEVICE pointers, with the gradient of the logits (dlogits 0: not wanted; logits: in place; rows that no
        sequence has stay as they were).  The workspace has preference_workspace(rows, pairs) bytes."""
        shape = PreferenceShape(type, kind, beta, smoothing, margin, logit_scale, int(average), 0, rows, classes, stride, pairs)
        self._check(self.lib.see_cuda_preference_loss(self.h, shape, logits or None, labels or None, starts or None, ref_logp or None,
                                                      loss_grad or None, loss or None, margins or None, sequence_logp or None,
                                                      dlogits or None, workspace or None, workspace_bytes))

    def policy_loss(self, rows: int, classes: int, logits: int, labels: int, old_logp: int, advantages: int, loss: int, logp: int,
                    workspace: int, workspace_bytes: int, ref_logp: int = 0, weights: int = 0, loss_grad: int = 0, dlogits: int = 0,
                    type: int = F32, logit_scale: float = 1.0, clip_low: float = 0.2, clip_high: float = 0.2, kl_coef: float = 0.0,
                    stride: int = 0):
        """A clipped policy loss with a KL term over DEVICE pointers, with the gradient of the logits (dlogits 0: not wanted;
        logits: in place); loss [3]: the loss, the KL term, the clipped rows, each summed by the rows' weights.  The workspace
        has policy_workspace(rows) bytes."""
        shape = PolicyShape(type, logit_scale, clip_low, clip_high, kl_coef, 0, rows, classes, stride)
        self._check(self.lib.see_cuda_policy_loss(self.h, shape, logits or None, labels or None, old_logp or None, ref_logp or None,
                                                  advantages or None, weights or None, loss_grad or None, loss or None, logp or None,
                                                  dlogits or None, workspace or None, workspace_bytes))

    def grad_norm(self, tensors, max_norm: float, norm: int, factor: int, workspace: int, workspace_bytes: int, grad_scale: int = 0):
        """The norm of all gradients of a table of grad_tensors, and the factor that adamw_step takes as its grad_scale to clip
        them (grad_scale included).  The workspace has grad_workspace() bytes."""
        self._check(self.lib.see_cuda_grad_norm(self.h, tensors, len(tensors), max_norm, grad_scale or None, norm or None, factor or None,
                                                workspace or None, workspace_bytes))

    def grad_clip(self, tensors, max_norm: float, norm: int, factor: int, workspace: int, workspace_bytes: int, grad_scale: int = 0):
        """The same, and the gradients times the factor to each tensor's out."""
        self._check(self.lib.see_cuda_grad_clip(self.h, tensors, len(tensors), max_norm, grad_scale or None, norm or None, factor or None,
                                                workspace or None, workspace_bytes))

    def set_profiling(self, on: bool):
        self._check(self.lib.see_cuda_set_profiling(self.h, int(on)))

    def take_profile(self, capacity: int = 65536, with_absorbed: bool = False):
        """(opcode, index, ms, m, n, k, kernel_ms) per executed instruction; with
        `with_absorbed` an eighth field: how many following instructions the
        instruction also did (epilogue fusion)."""
        arr = (ProfileRecord * capacity)()
        n = self.lib.see_cuda_take_profile(self.h, arr, capacity)
        if with_absorbed:
            return [(r.opcode, r.index, r.ms, r.m, r.n, r.k, r.kernel_ms, r.absorbed) for r in arr[:n]]
        return [(r.opcode, r.index, r.ms, r.m, r.n, r.k, r.kernel_ms) for r in arr[:n]]
