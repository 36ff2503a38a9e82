"""gemmkit_b200 -- gemmkit's quantized-inference GEMM path on NVIDIA B200 (sm_100a).

A Python mirror of gemmkit's Rust API (gemmkit/src/lib.rs:98-148 re-exports) over the C ABI of
``libgemmkit_cuda.so``: the same entry names, argument meaning, view rules and ``gemmkit:``
error messages (raised as :class:`GemmkitError` where gemmkit panics). Matrices are views
over flat CUDA tensors; calls are enqueued on the current torch stream, and the checked
entries synchronise like gemmkit's blocking calls unless ``sync=False``.

All arithmetic runs in the engine's sm_100a kernels; there is no CPU or PyTorch fallback.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass, field
from typing import Optional, Sequence

from . import _lib
from ._lib import (AXIS_COL, AXIS_NONE, AXIS_ROW, FP4_MX, FP4_NV, GK_EINVAL, GK_ENODEV, GK_ENOMEM, GK_ETIMEOUT,
                   GK_OK, MatMutC, MatRefC, ProblemC, RequantC)

__all__ = [
    "GemmkitError", "Parallelism", "MatRef", "MatMut", "Workspace", "RequantScale", "Requantize",
    "PackedRhs", "gemm_i8", "gemm_i8_with", "gemm_i8_unchecked", "gemm_i8_requant",
    "gemv_i8_requant",
    "gemm_i8_requant_u8", "gemm_i8_requant_unchecked", "gemm_i8_requant_u8_unchecked",
    "prepack_rhs_i8", "prepack_rhs_i8_unchecked", "gemm_i8_packed_b", "gemm_i8_packed_b_unchecked",
    "gemm_i8_packed_b_requant", "gemm_i8_requant_batched", "gemm_i8_requant_batched_ptr",
    "gemm_half_f32", "gemm_bf16_f32_unchecked", "gemm_f16_f32_unchecked",
    "gemm_half_f32_batched", "gemm_half_f32_fused", "gemm_i8_fused", "gemm_i8_fused_unchecked", "Activation", "quantize_f32_i8", "gemm_i8_noalloc_unchecked", "set_tile_n", "knob_names", "knob_get",
    "gemm_half_grouped", "gemm_half_grouped_wgrad", "scratch_release", "Fp4Matrix", "quantize_fp4", "dequantize_fp4",
    "gemm_fp4", "gemm_half_epilogue", "gemm_half_dact", "act_backward", "Act8Matrix",
    "quantize_act8", "dequantize_act8", "gemm_act8_wgrad", "MoeBalance", "moe_balance",
    "moe_balance_backward", "FP4_MX", "FP4_NV", "knob_set", "device_status", "selftest_wait_timeout",
]


class GemmkitError(RuntimeError):
    """A rejected call: the engine's status code plus gemmkit's message."""

    def __init__(self, code: int, msg: str):
        super().__init__(msg)
        self.code = code


def _check(rc: int) -> None:
    if rc != GK_OK:
        raise GemmkitError(rc, _lib.last_error())


# ---- Parallelism (gemmkit/src/parallel.rs:25-39) -------------------------------------------

class Parallelism:
    """Accepted for API parity; the device engine always uses the whole GPU."""

    def __init__(self, kind: int = 0, threads: int = 0):
        self.kind, self.threads = kind, threads

    @staticmethod
    def Serial() -> "Parallelism":
        return Parallelism(0, 0)

    @staticmethod
    def Rayon(n: int = 0) -> "Parallelism":
        return Parallelism(1, n)

    def c(self) -> _lib.Parallelism:
        return _lib.Parallelism(self.kind, self.threads)


SERIAL = Parallelism.Serial()


_cuda = None  # (torch, current-device call, raw-stream call), once torch has a CUDA context


def _cuda_calls():
    """torch's current-device and current-stream calls, without building a Stream object per
    call (that and torch.cuda.is_available() cost several microseconds); None without CUDA."""
    global _cuda
    if _cuda is None:
        try:
            import torch
        except ImportError:
            return None
        if not torch.cuda.is_available():
            return None
        torch.cuda.init()
        dev = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
        raw = getattr(torch._C, "_cuda_getCurrentRawStream",
                      lambda d: torch.cuda.current_stream(d).cuda_stream)
        _cuda = (torch, dev, raw)
    return _cuda


def _stream(stream):
    if stream is not None:
        return C.c_void_p(int(stream))
    calls = _cuda or _cuda_calls()
    return C.c_void_p(calls[2](calls[1]()) if calls else 0)


def _sync(stream) -> None:
    import torch
    if torch.cuda.is_available():
        if stream is None:
            torch.cuda.current_stream().synchronize()
        else:
            torch.cuda.synchronize()


# ---- views (gemmkit/src/api.rs:99-186) -------------------------------------------------------

def _flat(data):
    """(pointer, length in elements) of a flat tensor / (ptr, len) pair."""
    if type(data) is tuple:
        return int(data[0]), int(data[1])
    return data.data_ptr(), data.numel()


class MatRef:
    """An immutable strided view: element (i, j) at data[i*rs + j*cs] (gemmkit MatRef)."""

    def __init__(self, data, rows: int, cols: int, rs: int, cs: int):
        self.data, self.rows, self.cols, self.rs, self.cs = data, rows, cols, rs, cs

    @classmethod
    def new(cls, data, rows, cols, rs, cs):
        return cls(data, rows, cols, rs, cs)

    @classmethod
    def from_row_major(cls, data, rows, cols):
        return cls(data, rows, cols, cols, 1)

    @classmethod
    def from_col_major(cls, data, rows, cols):
        return cls(data, rows, cols, 1, rows)

    def c(self) -> MatRefC:
        d = self.data
        if type(d) is tuple:
            return MatRefC(int(d[0]), int(d[1]), self.rows, self.cols, self.rs, self.cs)
        return MatRefC(d.data_ptr(), d.numel(), self.rows, self.cols, self.rs, self.cs)

    def ptr(self) -> int:
        return _flat(self.data)[0]


class MatMut(MatRef):
    """A mutable strided view (gemmkit MatMut), the output C."""

    def c(self) -> MatMutC:
        d = self.data
        if type(d) is tuple:
            return MatMutC(int(d[0]), int(d[1]), self.rows, self.cols, self.rs, self.cs)
        return MatMutC(d.data_ptr(), d.numel(), self.rows, self.cols, self.rs, self.cs)


class Workspace:
    """gemmkit::Workspace: reusable device scratch for operand packs (one per stream)."""

    def __init__(self):
        h = C.c_void_p()
        _check(_lib.load().gk_workspace_create(C.byref(h)))
        self.h = h

    def __del__(self):
        try:
            if getattr(self, "h", None) is not None and self.h.value:
                _lib.load().gk_workspace_free(self.h)
                self.h = None
        except Exception:  # interpreter shutdown
            pass


def _ws(ws: Optional[Workspace]):
    return ws.h if ws is not None else None


# ---- requant descriptors (gemmkit/src/api/int8.rs:185-209) ---------------------------------

@dataclass
class RequantScale:
    """PerTensor(s) or PerRow(vector) as gemmkit; PerCol(vector) is the extension."""
    value: float = 1.0
    vector: object = None
    axis: int = AXIS_NONE

    @staticmethod
    def PerTensor(s: float) -> "RequantScale":
        return RequantScale(float(s), None, AXIS_NONE)

    @staticmethod
    def PerRow(v) -> "RequantScale":
        return RequantScale(0.0, v, AXIS_ROW)

    @staticmethod
    def PerCol(v) -> "RequantScale":
        return RequantScale(0.0, v, AXIS_COL)


@dataclass
class Requantize:
    """gemmkit::Requantize plus the extension fields ``bias_axis`` and ``relu``."""
    scale: RequantScale
    zero_point: int = 0
    bias: object = None
    bias_axis: int = AXIS_ROW
    relu: bool = False

    def c(self) -> RequantC:
        key = (self.scale.value, self.scale.axis, id(self.scale.vector), self.zero_point,
               id(self.bias), self.bias_axis, self.relu)
        cached = self.__dict__.get("_c_cache")
        if cached is not None and cached[0] == key:
            return cached[1]
        r = self._build_c()
        self.__dict__["_c_cache"] = (key, r)
        return r

    def _build_c(self) -> RequantC:
        r = RequantC()
        r.scale = self.scale.value
        r.scale_axis = self.scale.axis
        if self.scale.vector is not None:
            p, n = _flat(self.scale.vector)
            r.scales, r.scales_len = p, n
        r.zero_point = int(self.zero_point)
        if self.bias is not None:
            p, n = _flat(self.bias)
            r.bias, r.bias_len, r.bias_axis = p, n, self.bias_axis
        r.relu = 1 if self.relu else 0
        return r


# ---- i8 -> i32 ----------------------------------------------------------------------------

def gemm_i8_with(ws, alpha: int, a: MatRef, b: MatRef, beta: int, c: MatMut,
                 par: Parallelism = SERIAL, stream=None, sync: bool = True) -> None:
    """gemm_i8_with (gemmkit/src/api/int8.rs:38): C(i32) <- alpha*A*B + beta*C, wrapping."""
    _check(_lib.load().gk_gemm_i8(_ws(ws), alpha, a.c(), b.c(), beta, c.c(), par.c(),
                                  _stream(stream)))
    if sync:
        _sync(stream)


def gemm_i8(alpha: int, a: MatRef, b: MatRef, beta: int, c: MatMut,
            par: Parallelism = SERIAL, stream=None, sync: bool = True) -> None:
    """gemm_i8 (gemmkit/src/api/int8.rs:22)."""
    gemm_i8_with(None, alpha, a, b, beta, c, par, stream, sync)


def gemm_i8_unchecked(m, k, n, alpha, a, rsa, csa, b, rsb, csb, beta, c, rsc, csc,
                      par: Parallelism = SERIAL, ws=None, stream=None) -> None:
    """gemm_i8_unchecked (gemmkit/src/api/int8.rs:86): raw device pointers (ints)."""
    _check(_lib.load().gk_gemm_i8_unchecked(_ws(ws), m, k, n, alpha, a, rsa, csa, b, rsb, csb,
                                            beta, c, rsc, csc, par.c(), _stream(stream)))


# ---- requant ------------------------------------------------------------------------------

def _requant(a, b, req, c, out_u8, par, ws, stream, sync):
    r = req.c()
    _check(_lib.load().gk_gemm_i8_requant(_ws(ws), a.c(), b.c(), C.byref(r), c.c(), int(out_u8),
                                          par.c(), _stream(stream)))
    if sync:
        _sync(stream)


def gemm_i8_requant(a: MatRef, b: MatRef, req: Requantize, c: MatMut,
                    par: Parallelism = SERIAL, ws=None, stream=None, sync: bool = True) -> None:
    """gemm_i8_requant (gemmkit/src/api/int8.rs:230): i8 output, clamp band [-128, 127]."""
    _requant(a, b, req, c, False, par, ws, stream, sync)


def gemm_i8_requant_u8(a: MatRef, b: MatRef, req: Requantize, c: MatMut,
                       par: Parallelism = SERIAL, ws=None, stream=None, sync: bool = True) -> None:
    """gemm_i8_requant_u8 (gemmkit/src/api/int8.rs:479): u8 output, clamp band [0, 255]."""
    _requant(a, b, req, c, True, par, ws, stream, sync)


def gemm_i8_requant_unchecked(m, k, n, a, rsa, csa, b, rsb, csb, scale, row_scales,
                              has_row_scales, zero_point, bias, has_bias, c, rsc, csc,
                              par: Parallelism = SERIAL, ws=None, stream=None) -> None:
    """gemm_i8_requant_unchecked (gemmkit/src/api/int8.rs:347)."""
    _check(_lib.load().gk_gemm_i8_requant_unchecked(
        _ws(ws), m, k, n, a, rsa, csa, b, rsb, csb, scale, row_scales, int(has_row_scales),
        zero_point, bias, int(has_bias), c, rsc, csc, par.c(), _stream(stream)))


def gemm_i8_requant_u8_unchecked(m, k, n, a, rsa, csa, b, rsb, csb, scale, row_scales,
                                 has_row_scales, zero_point, bias, has_bias, c, rsc, csc,
                                 par: Parallelism = SERIAL, ws=None, stream=None) -> None:
    """gemm_i8_requant_u8_unchecked (gemmkit/src/api/int8.rs:562)."""
    _check(_lib.load().gk_gemm_i8_requant_u8_unchecked(
        _ws(ws), m, k, n, a, rsa, csa, b, rsb, csb, scale, row_scales, int(has_row_scales),
        zero_point, bias, int(has_bias), c, rsc, csc, par.c(), _stream(stream)))


def gemm_i8_requant_ex_unchecked(m, k, n, a, rsa, csa, b, rsb, csb, req: Requantize, c, rsc,
                                 csc, out_u8=False, par: Parallelism = SERIAL, ws=None,
                                 stream=None) -> None:
    r = req.c()
    _check(_lib.load().gk_gemm_i8_requant_ex_unchecked(
        _ws(ws), m, k, n, a, rsa, csa, b, rsb, csb, C.byref(r), c, rsc, csc, int(out_u8),
        par.c(), _stream(stream)))


# ---- prepacked B (gemmkit/src/api/packed.rs) ----------------------------------------------

class PackedRhs:
    """gemmkit::PackedRhs<i8>: B packed once on the device (K-major tile layout)."""

    def __init__(self, handle: C.c_void_p):
        self.h = handle

    def rows(self) -> int:
        return _lib.load().gk_packed_rhs_rows(self.h)

    def cols(self) -> int:
        return _lib.load().gk_packed_rhs_cols(self.h)

    def to_bytes(self) -> bytes:
        """Extension: the serialized packed B (header + device-ready bytes)."""
        lib = _lib.load()
        need = C.c_size_t()
        _check(lib.gk_packed_rhs_serialize(self.h, None, 0, C.byref(need)))
        buf = C.create_string_buffer(need.value)
        _check(lib.gk_packed_rhs_serialize(self.h, buf, need.value, C.byref(need)))
        return buf.raw

    @staticmethod
    def from_bytes(data: bytes, stream=None) -> "PackedRhs":
        """Extension: a packed B loaded back from `to_bytes` output onto the current device."""
        h = C.c_void_p()
        _check(_lib.load().gk_packed_rhs_deserialize(data, len(data), _stream(stream),
                                                     C.byref(h)))
        return PackedRhs(h)

    def __del__(self):
        try:
            if getattr(self, "h", None) is not None and self.h.value:
                _lib.load().gk_packed_rhs_free(self.h)
                self.h = None
        except Exception:  # interpreter shutdown: the library may already be unloaded
            pass


def prepack_rhs_i8(b: MatRef, stream=None, sync: bool = True) -> PackedRhs:
    """prepack_rhs_i8 (gemmkit/src/api/packed.rs:372)."""
    h = C.c_void_p()
    _check(_lib.load().gk_prepack_rhs_i8(b.c(), _stream(stream), C.byref(h)))
    if sync:
        _sync(stream)
    return PackedRhs(h)


def prepack_rhs_i8_unchecked(b: int, rsb: int, csb: int, k: int, n: int, stream=None) -> PackedRhs:
    """prepack_rhs_i8_unchecked (gemmkit/src/api/packed.rs:386)."""
    h = C.c_void_p()
    _check(_lib.load().gk_prepack_rhs_i8_unchecked(b, rsb, csb, k, n, _stream(stream),
                                                   C.byref(h)))
    return PackedRhs(h)


def gemm_i8_packed_b(alpha: int, a: MatRef, packed: PackedRhs, beta: int, c: MatMut,
                     par: Parallelism = SERIAL, ws=None, stream=None, sync: bool = True) -> None:
    """gemm_i8_packed_b (gemmkit/src/api/packed.rs:473)."""
    _check(_lib.load().gk_gemm_i8_packed_b(_ws(ws), alpha, a.c(), packed.h, beta, c.c(), par.c(),
                                           _stream(stream)))
    if sync:
        _sync(stream)


def gemm_i8_packed_b_unchecked(alpha, m, a, rsa, csa, packed: PackedRhs, beta, c, rsc, csc,
                               par: Parallelism = SERIAL, ws=None, stream=None) -> None:
    """gemm_i8_packed_b_unchecked (gemmkit/src/api/packed.rs:584)."""
    _check(_lib.load().gk_gemm_i8_packed_b_unchecked(_ws(ws), alpha, m, a, rsa, csa, packed.h,
                                                     beta, c, rsc, csc, par.c(), _stream(stream)))


def gemm_i8_packed_b_requant(m, a, rsa, csa, packed: PackedRhs, req: Requantize, c, rsc, csc,
                             out_u8=False, par: Parallelism = SERIAL, ws=None,
                             stream=None) -> None:
    """Extension: requantized product with a prepacked B (raw device pointers)."""
    r = req.c()
    _check(_lib.load().gk_gemm_i8_packed_b_requant_unchecked(
        _ws(ws), m, a, rsa, csa, packed.h, C.byref(r), c, rsc, csc, int(out_u8), par.c(),
        _stream(stream)))


def gemv_i8_requant(m, a, rsa, csa, packed: PackedRhs, req: Requantize, c, rsc, csc,
                    out_u8=False, ws=None, stream=None) -> None:
    """The decode-step GEMV: gemm_i8_packed_b_requant for 1 <= m <= 64 activation rows on the
    small-M streaming kernel (gemmkit's internal small-shape route,
    gemmkit/src/special/small_mn.rs:834-1060, given an entry of its own)."""
    r = req.c()
    _check(_lib.load().gk_gemv_i8_requant_unchecked(
        _ws(ws), m, a, rsa, csa, packed.h, C.byref(r), c, rsc, csc, int(out_u8),
        _stream(stream)))


# ---- batched (extension of gemmkit/src/api/batched.rs to i8) ------------------------------

def gemm_i8_requant_batched(batch, m, k, n, a, rsa, csa, a_bs, b, rsb, csb, b_bs,
                            req: Requantize, bias_bs, scales_bs, c, rsc, csc, c_bs,
                            out_u8=False, par: Parallelism = SERIAL, ws=None,
                            stream=None) -> None:
    r = req.c()
    _check(_lib.load().gk_gemm_i8_requant_batched_unchecked(
        _ws(ws), batch, m, k, n, a, rsa, csa, a_bs, b, rsb, csb, b_bs, C.byref(r), bias_bs,
        scales_bs, c, rsc, csc, c_bs, int(out_u8), par.c(), _stream(stream)))


@dataclass
class GemmProblem:
    """One pointer-array batch element (gemmkit GemmProblem, gemmkit/src/dispatch.rs:135)."""
    m: int
    k: int
    n: int
    a: int
    rsa: int
    csa: int
    b: int
    rsb: int
    csb: int
    c: int
    rsc: int
    csc: int
    req: Requantize = field(default_factory=lambda: Requantize(RequantScale.PerTensor(1.0)))


def gemm_i8_requant_batched_ptr(problems: Sequence[GemmProblem], out_u8=False,
                                par: Parallelism = SERIAL, ws=None, stream=None) -> None:
    arr = (ProblemC * len(problems))()
    for i, p in enumerate(problems):
        arr[i] = ProblemC(p.m, p.k, p.n, p.a, p.rsa, p.csa, p.b, p.rsb, p.csb, p.c, p.rsc, p.csc,
                          p.req.c())
    _check(_lib.load().gk_gemm_i8_requant_batched_ptr_unchecked(
        _ws(ws), arr, len(problems), int(out_u8), par.c(), _stream(stream)))


# ---- half -> f32 ----------------------------------------------------------------------------

def gemm_half_f32(alpha: float, a: MatRef, b: MatRef, beta: float, c: MatMut, is_f16=False,
                  par: Parallelism = SERIAL, ws=None, stream=None, sync: bool = True) -> None:
    """bf16 / f16 inputs, f32 accumulate and output: C <- alpha*A*B + beta*C."""
    _check(_lib.load().gk_gemm_half_f32(_ws(ws), int(is_f16), alpha, a.c(), b.c(), beta, c.c(),
                                        par.c(), _stream(stream)))
    if sync:
        _sync(stream)


class Activation:
    """gemmkit::Activation (gemmkit/src/api.rs:63): ReLU or LeakyReLU(slope); and, for the
    feed-forward layers' entries (gemm_half_epilogue and the like) only, GELU, its tanh form and
    SiLU."""

    def __init__(self, kind: int, slope: float = 0.0):
        self.kind, self.slope = kind, slope

    @staticmethod
    def Relu() -> "Activation":
        return Activation(_lib.ACT_RELU)

    @staticmethod
    def LeakyRelu(slope: float) -> "Activation":
        return Activation(_lib.ACT_LEAKY_RELU, float(slope))

    @staticmethod
    def Gelu() -> "Activation":
        return Activation(_lib.ACT_GELU)

    @staticmethod
    def GeluTanh() -> "Activation":
        return Activation(_lib.ACT_GELU_TANH)

    @staticmethod
    def Silu() -> "Activation":
        return Activation(_lib.ACT_SILU)


def gemm_half_f32_fused(alpha: float, a: MatRef, b: MatRef, beta: float, c: MatMut, bias=None,
                        bias_dim: int = AXIS_ROW, act: Optional[Activation] = None, is_f16=False,
                        par: Parallelism = SERIAL, ws=None, stream=None,
                        sync: bool = True) -> None:
    """gemm_fused (gemmkit/src/api/fused.rs) on bf16 / f16 inputs with f32 output:
    C <- act(alpha*A*B + beta*C + bias), the bias per row (AXIS_ROW, length m) or per column
    (AXIS_COL, length n)."""
    bp, bn = _flat(bias) if bias is not None else (0, 0)
    _check(_lib.load().gk_gemm_half_f32_fused(
        _ws(ws), int(is_f16), alpha, a.c(), b.c(), beta, c.c(), C.c_void_p(bp or None), bn,
        bias_dim, act.kind if act else _lib.ACT_NONE, act.slope if act else 0.0, par.c(),
        _stream(stream)))
    if sync:
        _sync(stream)


def gemm_i8_fused(alpha: int, a: MatRef, b: MatRef, beta: int, c: MatMut, bias=None,
                  bias_dim: int = AXIS_ROW, act: Optional[Activation] = None,
                  par: Parallelism = SERIAL, ws=None, stream=None, sync: bool = True) -> None:
    """The i8 -> i32 GEMM with a fused integer epilogue (extension; gemmkit's gemm_fused is
    float-only): C <- act(alpha*A*B + beta*C + bias), wrapping i32 arithmetic, the i32 bias
    per row (AXIS_ROW, length m) or per column (AXIS_COL, length n), act None or ReLU."""
    bp, bn = _flat(bias) if bias is not None else (0, 0)
    _check(_lib.load().gk_gemm_i8_fused(
        _ws(ws), int(alpha), a.c(), b.c(), int(beta), c.c(), C.c_void_p(bp or None), bn,
        bias_dim, act.kind if act else _lib.ACT_NONE, par.c(), _stream(stream)))
    if sync:
        _sync(stream)


def gemm_i8_fused_unchecked(m, k, n, alpha, a, rsa, csa, b, rsb, csb, beta, c, rsc, csc,
                            bias=None, bias_dim: int = AXIS_ROW, act: int = 0,
                            par: Parallelism = SERIAL, ws=None, stream=None) -> None:
    """Raw-pointer tier of gemm_i8_fused (device pointers as ints; bias a device pointer or
    None; act one of _lib.ACT_NONE / _lib.ACT_RELU)."""
    _check(_lib.load().gk_gemm_i8_fused_unchecked(
        _ws(ws), m, k, n, alpha, a, rsa, csa, b, rsb, csb, beta, c, rsc, csc,
        C.c_void_p(bias) if bias else None, bias_dim, 1 if bias else 0, act, par.c(),
        _stream(stream)))


def quantize_f32_i8(rows, cols, x, rsx, csx, q, rsq, csq, scale: float = 1.0,
                    zero_point: int = 0, row_scales=None, stream=None) -> None:
    """Extension: f32 -> i8 activations (raw device pointers). Per-tensor scale / zero point,
    or per-row symmetric scales written to `row_scales` (a device pointer) when given."""
    _check(_lib.load().gk_quantize_f32_i8_unchecked(
        rows, cols, C.c_void_p(x), rsx, csx, C.c_void_p(q), rsq, csq, float(scale),
        int(zero_point), C.c_void_p(row_scales) if row_scales else None, _stream(stream)))


def gemm_bf16_f32_unchecked(m, k, n, alpha, a, rsa, csa, b, rsb, csb, beta, c, rsc, csc,
                            par: Parallelism = SERIAL, ws=None, stream=None) -> None:
    _check(_lib.load().gk_gemm_bf16_f32_unchecked(_ws(ws), m, k, n, alpha, a, rsa, csa, b, rsb,
                                                  csb, beta, c, rsc, csc, par.c(),
                                                  _stream(stream)))


def gemm_f16_f32_unchecked(m, k, n, alpha, a, rsa, csa, b, rsb, csb, beta, c, rsc, csc,
                           par: Parallelism = SERIAL, ws=None, stream=None) -> None:
    _check(_lib.load().gk_gemm_f16_f32_unchecked(_ws(ws), m, k, n, alpha, a, rsa, csa, b, rsb,
                                                 csb, beta, c, rsc, csc, par.c(),
                                                 _stream(stream)))


def gemm_half_f32_batched(is_f16, batch, m, k, n, alpha, a, rsa, csa, a_bs, b, rsb, csb, b_bs,
                          beta, c, rsc, csc, c_bs, par: Parallelism = SERIAL, ws=None,
                          stream=None) -> None:
    _check(_lib.load().gk_gemm_half_f32_batched_unchecked(
        _ws(ws), int(is_f16), batch, m, k, n, alpha, a, rsa, csa, a_bs, b, rsb, csb, b_bs, beta,
        c, rsc, csc, c_bs, par.c(), _stream(stream)))


# ---- products of rows grouped by expert ------------------------------------------------------

_ELEM = {"torch.float32": _lib.DT_F32, "torch.float16": _lib.DT_F16,
         "torch.bfloat16": _lib.DT_BF16, "torch.int16": None, "torch.uint16": None}
_elem = {}  # the same by dtype object, filled as they are met


def _elem_type(data, default: int) -> int:
    """The C ABI's element type of a tensor (``default`` for a (pointer, length) pair, or for the
    int16 / uint16 tensors that carry 16-bit floats)."""
    if isinstance(data, tuple):
        return default
    dt = data.dtype
    if dt not in _elem:
        if str(dt) not in _ELEM:
            raise GemmkitError(GK_EINVAL, f"gemmkit: elements of type {dt} are not supported here")
        _elem[dt] = _ELEM[str(dt)]
    t = _elem[dt]
    return default if t is None else t


def _same_device(*named) -> None:
    """The engine launches on the current device: refuse tensors that lie elsewhere. Takes names
    and tensors in turn; (pointer, length) pairs and None are not looked at."""
    calls = _cuda or _cuda_calls()
    cur = calls[1]() if calls else -2
    for i in range(1, len(named), 2):
        t = named[i]
        if t is None or isinstance(t, tuple) or t.get_device() == cur:
            continue
        if t.get_device() < 0:
            raise GemmkitError(GK_EINVAL, f"gemmkit: {named[i - 1]} is not in device memory")
        raise GemmkitError(GK_EINVAL, f"gemmkit: {named[i - 1]} is on cuda:{t.get_device()}, the "
                                      f"current device is cuda:{cur}")


def _one_device(*named):
    """The parts of one matrix lie in the memory of one device (names and tensors in turn, as in
    _same_device): the first tensor among them, which stands for all when the matrix is used."""
    at = first = None
    for i in range(1, len(named), 2):
        t = named[i]
        if t is None or isinstance(t, tuple):
            continue
        dev = t.get_device()
        if dev < 0:
            raise GemmkitError(GK_EINVAL, f"gemmkit: {named[i - 1]} is not in device memory")
        if first is None:
            at, first = (named[i - 1], dev), t
        elif dev != at[1]:
            raise GemmkitError(GK_EINVAL, f"gemmkit: {named[i - 1]} is on cuda:{dev}, {at[0]} is on "
                                          f"cuda:{at[1]}")
    return first


def _offsets(offsets):
    """(pointer, groups) of an int32 offsets tensor or a (pointer, groups + 1) pair."""
    if isinstance(offsets, tuple):
        return int(offsets[0]), int(offsets[1]) - 1
    if offsets.dim() != 1 or str(offsets.dtype) != "torch.int32" or not offsets.is_contiguous():
        raise GemmkitError(GK_EINVAL, "gemmkit: offsets must be a contiguous 1-D int32 tensor")
    return offsets.data_ptr(), offsets.numel() - 1


def _grouped_args(a, b, offsets, c, is_f16):
    half = _lib.DT_F16 if is_f16 else _lib.DT_BF16
    _same_device("A", a.data, "B", b.data, "C", c.data, "offsets", offsets)
    for name, d in (("A", a.data), ("B", b.data)):
        if _elem_type(d, half) != half:
            raise GemmkitError(GK_EINVAL, f"gemmkit: {name} must hold "
                                          f"{'f16' if is_f16 else 'bf16'} elements")
    ptr, groups = _offsets(offsets)
    if groups < 0:
        groups = 0
    return ptr, groups, _elem_type(c.data, half)


def gemm_half_grouped(alpha: float, a: MatRef, b: MatRef, b_gs: int, offsets, beta: float,
                      c: MatMut, is_f16=False, par: Parallelism = SERIAL, stream=None,
                      sync: bool = True) -> None:
    """The experts' products (extension): C[i, :] <- alpha*A[i, :]*B[g] + beta*C[i, :] for the rows
    offsets[g] <= i < offsets[g + 1]. A (rows x k) holds bf16 (f16 with is_f16), `b` views group 0's
    k x n matrix inside a slice that holds all groups at stride b_gs (elements, 0 = shared);
    `offsets` is an int32 device tensor of groups + 1 entries that the host never reads. C holds
    f32 or the operands' type, by its tensor's dtype (16-bit for a (pointer, length) pair). Rows
    outside the groups are left as they are. With C's gradient as A and B viewed transposed the
    same call is the gradient of A."""
    ptr, groups, out = _grouped_args(a, b, offsets, c, is_f16)
    _check(_lib.load().gk_gemm_half_grouped(int(is_f16), groups, ptr, float(alpha), a.c(), b.c(),
                                            int(b_gs), float(beta), c.c(), out, par.c(),
                                            _stream(stream)))
    if sync:
        _sync(stream)


def gemm_half_grouped_wgrad(alpha: float, a: MatRef, b: MatRef, offsets, beta: float, c: MatMut,
                            c_gs: int, is_f16=False, par: Parallelism = SERIAL, stream=None,
                            sync: bool = True) -> None:
    """The experts' weight gradients (extension): C[g] <- alpha*A_g^T*B_g + beta*C[g] with A (rows x
    m) and B (rows x n) grouped by `offsets` as in gemm_half_grouped; `c` views group 0's m x n
    matrix inside a slice that holds all groups at stride c_gs. An empty group's C[g] becomes
    beta*C[g]."""
    ptr, groups, out = _grouped_args(a, b, offsets, c, is_f16)
    _check(_lib.load().gk_gemm_half_grouped_wgrad(int(is_f16), groups, ptr, float(alpha), a.c(),
                                                  b.c(), float(beta), c.c(), int(c_gs), out,
                                                  par.c(), _stream(stream)))
    if sync:
        _sync(stream)


def scratch_release(device: int = 0) -> None:
    """Give the scratch that the grouped products keep for operands that they had to realign back
    to the device (at most 1/64 of its memory stays with the engine otherwise); synchronises it."""
    _check(_lib.load().gk_scratch_release(device))


# ---- microscaled 4-bit floating point --------------------------------------------------------

class Fp4Matrix:
    """A rows x cols matrix in microscaled 4-bit floats (extension; see gk_fp4_matrix in the C
    header): e2m1 codes with a scale per 32 (FP4_MX) or 16 (FP4_NV) elements of a row. Made by
    quantize_fp4, from_codes, or empty; holds its device tensors `data` and `scales`.

    `groups` equal groups make a stack of matrices (rows / groups rows each); `offsets` (an int32
    device tensor of groups + 1 entries) ragged groups. `scale` is the FP4_NV format's matrix
    scale (1 for FP4_MX)."""

    def __init__(self, rows: int, cols: int, fmt: int, scale: float, groups: int, offsets, data,
                 scales):
        self.rows, self.cols, self.fmt, self.scale = int(rows), int(cols), fmt, float(scale)
        self.groups, self.offsets = groups, offsets
        self._data, self._scales = data, scales
        self._where = _one_device("data", data, "scales", scales, "offsets", offsets)
        off = None
        if offsets is not None:
            off, n = _offsets(offsets)
            if n != groups:  # the kernels read groups + 1 offsets
                raise GemmkitError(GK_EINVAL, f"gemmkit: {groups} groups take {groups + 1} offsets "
                                              f"(has {n + 1})")
        self.c = _lib.Fp4MatrixC(fmt, self.scale, groups, off, self.rows, self.cols, *_flat(data),
                                 *_flat(scales))

    @property
    def data(self):
        """The codes (uint8): rows at a pitch of whole 16-byte pieces."""
        d = self._data
        return d if self._scales is not None else d[:self.c.data_len]

    @property
    def scales(self):
        """The block scales (uint8) in the engine's tile order."""
        return self._scales if self._scales is not None else self._data[self.c.data_len:]

    @staticmethod
    def empty(rows: int, cols: int, fmt: int, scale: float = 1.0, groups: int = 1, offsets=None,
              device=None, stream=None) -> "Fp4Matrix":
        """An unwritten matrix on the current device (a destination for quantize_fp4), its memory
        allocated for torch's current stream or for `stream`."""
        off = None
        if offsets is not None:
            off, groups = _offsets(offsets)
        calls = _cuda or _cuda_calls()
        if calls is None:
            _one_device("offsets", offsets)
            raise GemmkitError(GK_ENODEV, "gemmkit: no CUDA device")
        torch = calls[0]
        if fmt not in (FP4_MX, FP4_NV) or groups < 1 or rows < 0 or cols < 0:
            raise GemmkitError(GK_EINVAL, f"gemmkit: no 4-bit matrix of {rows}x{cols}, format {fmt}, "
                                          f"{groups} groups")
        # one allocation: codes, then scales (both parts whole 16-byte pieces)
        nd, ns = _fp4_sizes(rows, cols, fmt, groups, offsets is not None)
        device = device or torch.device("cuda", calls[1]())
        if stream is None:
            buf = torch.empty(nd + ns, dtype=torch.uint8, device=device)
        else:  # not what the current stream may still be writing
            with torch.cuda.stream(torch.cuda.ExternalStream(int(stream), device=device)):
                buf = torch.empty(nd + ns, dtype=torch.uint8, device=device)
        if offsets is not None:
            _one_device("the matrix", buf, "offsets", offsets)
        q = Fp4Matrix.__new__(Fp4Matrix)
        q._where = buf
        q.rows, q.cols, q.fmt, q.scale = rows, cols, fmt, float(scale)
        q.groups, q.offsets, q._data, q._scales = groups, offsets, buf, None
        at = buf.data_ptr()
        q.c = _lib.Fp4MatrixC(fmt, q.scale, groups, off, rows, cols, at, nd, at + nd, ns)
        return q

    @staticmethod
    def from_codes(codes, block_scales, rows: int, cols: int, fmt: int, scale: float = 1.0,
                   groups: int = 1, offsets=None, stream=None, sync: bool = True) -> "Fp4Matrix":
        """A matrix from plain row-major parts, as checkpoints hold them: uint8 tensors of codes
        (rows x ceil(cols / 2), the first element of a pair in the low nibble) and of block scales
        (rows x blocks: e8m0 or e4m3 bytes), both with contiguous rows."""
        _same_device("codes", codes, "block_scales", block_scales, "offsets", offsets)
        for name, t in (("codes", codes), ("block_scales", block_scales)):
            if t.dim() != 2 or t.shape[0] != rows or t.element_size() != 1 or \
                    (t.shape[1] > 1 and t.stride(1) != 1):
                raise GemmkitError(GK_EINVAL, f"gemmkit: {name} must hold {rows} contiguous rows of "
                                              "bytes")
        q = Fp4Matrix.empty(rows, cols, fmt, scale, groups, offsets, codes.device, stream)

        def part(t):
            ld = t.stride(0) if rows > 1 else t.shape[1]
            return t.data_ptr(), (rows - 1) * ld + t.shape[1] if rows else 0, ld
        _check(_lib.load().gk_fp4_import(*part(codes), *part(block_scales), C.byref(q.c),
                                         _stream(stream)))
        if sync:
            _sync(stream)
        return q


def _fp4_sizes(rows, cols, fmt, groups, ragged):
    """gk_fp4_data_bytes and gk_fp4_scale_bytes."""
    groups = max(groups, 1)
    blocks = (rows + 127) // 128 + groups if ragged else groups * ((rows // groups + 127) // 128)
    pitch = ((cols + 1) // 2 + 15) // 16 * 16
    return rows * pitch, blocks * ((cols + 255) // 256) * (1024 if fmt == FP4_MX else 2048)


def quantize_fp4(x: MatRef, fmt: int, scale: float = 1.0, offsets=None, groups: int = 1,
                 x_gs: int = 0, x_type: Optional[int] = None, out: Optional[Fp4Matrix] = None,
                 stream=None, sync: bool = True) -> Fp4Matrix:
    """x (f32, f16 or bf16) in 4 bits along its columns (extension): e2m1 codes, a scale per 32
    (FP4_MX) or 16 (FP4_NV, times `scale`) consecutive elements of a row. Activations (rows x k) as
    they are; weights with a column per output as the transposed view (n x k). With `offsets` the
    rows form ragged groups; with groups > 1 `x` views the first of `groups` matrices that lie
    x_gs elements apart. `out` reuses a matrix of the same shape, format and groups (its scale and
    groups then hold), otherwise the result's memory is allocated for the call's stream; x_type names
    the element type of a (pointer, length) pair."""
    _same_device("X", x.data, "offsets", offsets, "out", None if out is None else out._where)
    if out is None:
        stacked = offsets is None and groups > 1
        out = Fp4Matrix.empty(x.rows * groups if stacked else x.rows, x.cols, fmt, scale, groups,
                              offsets, stream=stream)
    elif out.fmt != fmt:
        raise GemmkitError(GK_EINVAL, "gemmkit: the output is held in another 4-bit format")
    if x_type is None:
        x_type = _elem_type(x.data, -1)
    _check(_lib.load().gk_quantize_fp4(x.c(), x_type, x_gs, C.byref(out.c), _stream(stream)))
    if sync:
        _sync(stream)
    return out


def dequantize_fp4(q: Fp4Matrix, out: MatMut, stream=None, sync: bool = True) -> None:
    """The f32 values that a 4-bit matrix stands for (extension)."""
    _same_device("Q", q._where, "C", out.data)
    if _elem_type(out.data, _lib.DT_F32) != _lib.DT_F32:
        raise GemmkitError(GK_EINVAL, "gemmkit: C must hold f32 elements")
    _check(_lib.load().gk_dequantize_fp4(C.byref(q.c), out.c(), _stream(stream)))
    if sync:
        _sync(stream)


def gemm_fp4(alpha: float, a: Fp4Matrix, b: Fp4Matrix, beta: float, c: MatMut,
             c_type: Optional[int] = None, par: Parallelism = SERIAL, stream=None,
             sync: bool = True) -> None:
    """C <- alpha*A*B^T + beta*C with both operands in 4 bits (extension): A (rows x k), B (n x k),
    C f32, f16 or bf16 by its tensor's dtype (c_type for a (pointer, length) pair). With groups,
    row i of A's group g is multiplied by B's g-th matrix: A ragged (offsets) or equal groups, B a
    stack of as many."""
    _same_device("A", a._where, "B", b._where, "C", c.data)
    if c_type is None:
        c_type = _elem_type(c.data, -1)
    _check(_lib.load().gk_gemm_fp4(float(alpha), C.byref(a.c), C.byref(b.c), float(beta), c.c(),
                                   c_type, par.c(), _stream(stream)))
    if sync:
        _sync(stream)


# ---- feed-forward layers, dense or by expert ---------------------------------------------------

_NO_MUT = MatMutC()


def _half_type(name: str, data, half: int, f32_too: bool = False) -> int:
    t = half if type(data) is tuple else _elem.get(data.dtype, -1)
    if t == half:
        return t
    t = _elem_type(data, half)
    if t != half and not (f32_too and t == _lib.DT_F32):
        raise GemmkitError(GK_EINVAL, f"gemmkit: {name} must hold "
                                      f"{'f16' if half == _lib.DT_F16 else 'bf16'} elements"
                                      f"{' or f32' if f32_too else ''}")
    return t


def _groups_of(offsets):
    """(pointer, groups) of optional offsets."""
    if offsets is None:
        return None, 1
    ptr, groups = _offsets(offsets)
    return ptr, max(groups, 0)


def _vector(name, t, half, n, gs):
    """(pointer, length, group stride, type) of a bias or its gradient."""
    if type(t) is not tuple and not t.is_contiguous():
        raise GemmkitError(GK_EINVAL, f"gemmkit: {name} must be contiguous")
    return (*_flat(t), n if gs is None else int(gs), _half_type(name, t, half, True))


def gemm_half_epilogue(alpha: float, a: MatRef, b: MatRef, c: MatMut, bias=None,
                       act: Optional[Activation] = None, residual: Optional[MatRef] = None,
                       z: Optional[MatMut] = None, offsets=None, b_gs: int = 0,
                       bias_gs: Optional[int] = None, is_f16=False, par: Parallelism = SERIAL,
                       stream=None, sync: bool = True) -> None:
    """A feed-forward layer's product (extension): z = alpha*A*B + bias, C <- act(z) + residual, in
    f32 on the accumulators and rounded once. A (rows x k) and B (k x n) hold bf16 (f16 with is_f16),
    C f32 or their type; `residual` has C's type and may be C itself; `z`, where the activation's
    input is kept for the backward pass, and `bias` (n elements; f32 allowed) the operands' type.
    With `offsets` the rows form groups as in gemm_half_grouped, `b` views group 0's matrix in a
    stack at stride b_gs, and group g's bias lies g * bias_gs (default n) elements on. Rows outside
    the groups are left as they are."""
    half = _lib.DT_F16 if is_f16 else _lib.DT_BF16
    rd, zd = residual and residual.data, z and z.data
    _same_device("A", a.data, "B", b.data, "C", c.data, "offsets", offsets, "bias", bias,
                 "residual", rd, "z", zd)
    _half_type("A", a.data, half)
    _half_type("B", b.data, half)
    if zd is not None:
        _half_type("z", zd, half)
    out = _elem_type(c.data, half)
    if rd is not None and _elem_type(rd, out) != out:
        raise GemmkitError(GK_EINVAL, "gemmkit: the residual must have C's type")
    ptr, groups = _groups_of(offsets)
    epi = _lib.EpilogueC()  # (no activation, bias, residual or z)
    if act:
        epi.act, epi.slope = act.kind, act.slope
    if bias is not None:
        epi.bias, epi.bias_len, epi.bias_gs, epi.bias_type = _vector("bias", bias, half, c.cols, bias_gs)
    if residual:
        epi.residual = residual.c()
    if z:
        epi.z = z.c()
    _check(_lib.load().gk_gemm_half_epilogue(int(is_f16), groups, ptr, float(alpha), a.c(), b.c(),
                                             int(b_gs), C.byref(epi), c.c(), out, par.c(),
                                             _stream(stream)))
    if sync:
        _sync(stream)


def _epilogue_bwd(z, act, dbias, dbias_gs, half, n):
    epi = _lib.EpilogueBwdC()  # (no activation, z or dbias)
    if act:
        epi.act, epi.slope = act.kind, act.slope
    if isinstance(z, Act8Matrix):
        epi.z8 = C.pointer(z.c)
    elif z is not None:
        _half_type("z", z.data, half)
        epi.z = z.c()
    if dbias is not None:
        epi.dbias, epi.dbias_len, epi.dbias_gs, epi.dbias_type = \
            _vector("dbias", dbias, half, n, dbias_gs)
    return epi


def _z_data(z):
    return None if z is None else z._where if isinstance(z, Act8Matrix) else z.data


def gemm_half_dact(alpha: float, a: MatRef, b: MatRef, z, act: Optional[Activation], c: MatMut,
                   dbias=None, offsets=None, b_gs: int = 0, dbias_gs: Optional[int] = None,
                   is_f16=False, par: Parallelism = SERIAL, stream=None, sync: bool = True) -> None:
    """The gradient through such a layer's activation (extension): C <- alpha*A*B * act'(z), A the
    gradient of the next layer's output, B its weights viewed transposed (k x n), `z` the activation's
    input as a MatRef in the operands' type or an Act8Matrix (None with act None). `dbias` (n
    elements a group, f32 or the operands' type) gets the sums of C over each group's rows. C may be
    z itself. Offsets, groups and types as in gemm_half_epilogue."""
    half = _lib.DT_F16 if is_f16 else _lib.DT_BF16
    _same_device("A", a.data, "B", b.data, "C", c.data, "offsets", offsets, "z", _z_data(z),
                 "dbias", dbias)
    _half_type("A", a.data, half)
    _half_type("B", b.data, half)
    ptr, groups = _groups_of(offsets)
    epi = _epilogue_bwd(z, act, dbias, dbias_gs, half, c.cols)
    _check(_lib.load().gk_gemm_half_dact(int(is_f16), groups, ptr, float(alpha), a.c(), b.c(),
                                         int(b_gs), C.byref(epi), c.c(), _elem_type(c.data, half),
                                         par.c(), _stream(stream)))
    if sync:
        _sync(stream)


def act_backward(dy: MatRef, z, act: Optional[Activation], dz: Optional[MatMut], dbias=None,
                 offsets=None, dbias_gs: Optional[int] = None, is_f16=False, stream=None,
                 sync: bool = True) -> None:
    """The same without a product (extension): dz <- dy * act'(z) and the sums of dz over each
    group's rows in `dbias`; either may be None. dy holds bf16 (f16 with is_f16), dz f32 or that
    type; dz may be dy or z itself."""
    half = _lib.DT_F16 if is_f16 else _lib.DT_BF16
    dzd = dz and dz.data
    _same_device("dY", dy.data, "dZ", dzd, "offsets", offsets, "z", _z_data(z), "dbias", dbias)
    _half_type("dY", dy.data, half)
    out = half if dzd is None else _elem_type(dzd, half)
    ptr, groups = _groups_of(offsets)
    epi = _epilogue_bwd(z, act, dbias, dbias_gs, half, dy.cols)
    _check(_lib.load().gk_act_backward(int(is_f16), groups, ptr, dy.c(), C.byref(epi),
                                       dz.c() if dz else _NO_MUT, out, _stream(stream)))
    if sync:
        _sync(stream)


_devices = {}  # torch.device objects by index


def _buffer(n, dtype, stream):
    """n unwritten elements on the current device, for torch's current stream or for `stream`."""
    torch, current = _cuda[0], _cuda[1]()
    device = _devices.get(current)
    if device is None:
        device = _devices[current] = torch.device("cuda", current)
    if stream is None:
        return torch.empty(n, dtype=dtype, device=device)
    # not what the current stream may still be writing
    with torch.cuda.stream(torch.cuda.ExternalStream(int(stream), device=device)):
        return torch.empty(n, dtype=dtype, device=device)


class Act8Matrix:
    """A rows x cols matrix of activations kept in 8 bits for the backward pass (extension; see
    gk_act8_matrix in the C header): int8 codes with a power of two per 32 elements of a row. Made by
    quantize_act8 or empty, or from tensors: `codes` int8, rows at a pitch that is a multiple of 32,
    and `exponents` uint8, ceil(cols / 32) a row. A run of rows of a matrix is one too (`rows_of`)."""

    def __init__(self, rows: int, cols: int, codes, exponents):
        self.rows, self.cols = int(rows), int(cols)
        nb = (self.cols + 31) // 32
        for name, t, types, n in (("codes", codes, ("torch.int8",), self.cols),
                                  ("exponents", exponents, ("torch.uint8",), nb)):
            if str(t.dtype) not in types or t.dim() != 2 or tuple(t.shape) != (self.rows, n) or \
                    (n > 1 and self.rows and t.stride(1) != 1):
                raise GemmkitError(GK_EINVAL, f"gemmkit: {name} must be {self.rows}x{n} "
                                              f"{types[0][6:]} with contiguous rows")
        self._where = _one_device("codes", codes, "exponents", exponents)
        self._codes, self._exps = codes, exponents
        lds = [t.stride(0) if self.rows > 1 else up
               for t, up in ((codes, (self.cols + 31) // 32 * 32), (exponents, nb))]
        # what lies behind the first element in its storage: the codes' last block may pass the row
        ends = [t.untyped_storage().nbytes() - t.storage_offset() for t in (codes, exponents)]
        self.c = _lib.Act8MatrixC(self.rows, self.cols, codes.data_ptr(),
                                  min(ends[0], self.rows * lds[0]), lds[0], exponents.data_ptr(),
                                  min(ends[1], self.rows * lds[1]), lds[1])

    @property
    def codes(self):
        """The codes (rows x cols, int8)."""
        if self._codes is None:  # parts of one buffer (empty), cut when they are asked for
            n = self.c.codes_len
            self._codes = self._where[:n].view(_cuda[0].int8).view(self.rows, -1 if n else 0)[:, :self.cols]
        return self._codes

    @property
    def exponents(self):
        """The exponent bytes (rows x ceil(cols / 32), uint8): 127 is a largest magnitude in [1, 2)."""
        if self._exps is None:
            part = self._where[self.c.codes_len:]
            self._exps = part.view(self.rows, -1 if part.numel() else 0)[:, :(self.cols + 31) // 32]
        return self._exps

    @staticmethod
    def empty(rows: int, cols: int, stream=None) -> "Act8Matrix":
        """An unwritten matrix on the current device, its memory allocated for torch's current stream
        or for `stream`."""
        calls = _cuda or _cuda_calls()
        if calls is None:
            raise GemmkitError(GK_ENODEV, "gemmkit: no CUDA device")
        if rows < 0 or cols < 0:
            raise GemmkitError(GK_EINVAL, f"gemmkit: no 8-bit matrix of {rows}x{cols}")
        torch = calls[0]
        nb = (cols + 31) // 32
        pitch = (nb + 15) // 16 * 16  # of the exponents: whole 16-byte pieces, as the codes' rows
        n = rows * nb * 32
        buf = _buffer(n + rows * pitch, torch.uint8, stream)
        q = Act8Matrix.__new__(Act8Matrix)
        q.rows, q.cols, q._where = rows, cols, buf
        q._codes = q._exps = None
        at = buf.data_ptr()
        q.c = _lib.Act8MatrixC(rows, cols, at, n, nb * 32, at + n, rows * pitch, pitch)
        return q

    def rows_of(self, first: int, last: int) -> "Act8Matrix":
        """Rows first .. last - 1, the same memory."""
        if not 0 <= first <= last <= self.rows:
            raise GemmkitError(GK_EINVAL, f"gemmkit: no rows {first} to {last} of {self.rows}")
        q = Act8Matrix.__new__(Act8Matrix)
        q.rows, q.cols, q._where = last - first, self.cols, self._where
        q._codes, q._exps = self.codes[first:last], self.exponents[first:last]
        c = self.c
        a, b = first * c.codes_ld, first * c.exps_ld
        q.c = _lib.Act8MatrixC(q.rows, q.cols, (c.codes or 0) + a, max(0, c.codes_len - a), c.codes_ld,
                               (c.exps or 0) + b, max(0, c.exps_len - b), c.exps_ld)
        return q


def quantize_act8(x: MatRef, out: Optional[Act8Matrix] = None, x_type: Optional[int] = None,
                  stream=None, sync: bool = True) -> Act8Matrix:
    """x (f32, f16 or bf16) in 8 bits (extension): per 32 consecutive elements of a row a power of two,
    codes rounded half to even in [-127, 127]. `out` reuses a matrix of the same shape, otherwise the
    result's memory is allocated for the call's stream; x_type names the element type of a (pointer,
    length) pair."""
    _same_device("X", x.data, "out", None if out is None else out._where)
    if out is None:
        out = Act8Matrix.empty(x.rows, x.cols, stream=stream)
    if x_type is None:
        x_type = _elem_type(x.data, -1)
    _check(_lib.load().gk_quantize_act8(x.c(), x_type, C.byref(out.c), _stream(stream)))
    if sync:
        _sync(stream)
    return out


def dequantize_act8(q: Act8Matrix, out: MatMut, out_type: Optional[int] = None, stream=None,
                    sync: bool = True) -> None:
    """The values that an 8-bit matrix stands for, in f32, bf16 (both exact) or f16 (exact where the
    source was f16)."""
    _same_device("Q", q._where, "C", out.data)
    if out_type is None:
        out_type = _elem_type(out.data, -1)
    _check(_lib.load().gk_dequantize_act8(C.byref(q.c), out.c(), out_type, _stream(stream)))
    if sync:
        _sync(stream)


def gemm_act8_wgrad(alpha: float, a: Act8Matrix, b: MatRef, beta: float, c: MatMut, offsets=None,
                    c_gs: int = 0, is_f16=False, par: Parallelism = SERIAL, stream=None,
                    sync: bool = True) -> None:
    """The weight gradient from a layer's input kept in 8 bits (extension): C[g] <- alpha*A_g^T*B_g +
    beta*C[g], A (rows x m) an Act8Matrix, B (rows x n) in bf16 (f16 with is_f16), C f32 or B's
    type; groups, offsets (None: all rows) and the stack of C as in gemm_half_grouped_wgrad."""
    half = _lib.DT_F16 if is_f16 else _lib.DT_BF16
    _same_device("A", a._where, "B", b.data, "C", c.data, "offsets", offsets)
    _half_type("B", b.data, half)
    ptr, groups = _groups_of(offsets)
    _check(_lib.load().gk_gemm_act8_wgrad(int(is_f16), groups, ptr, float(alpha), C.byref(a.c), b.c(),
                                          float(beta), c.c(), int(c_gs), _elem_type(c.data, half),
                                          par.c(), _stream(stream)))
    if sync:
        _sync(stream)


# ---- the router's balance loss ------------------------------------------------------------------

class MoeBalance:
    """What moe_balance gives, device tensors: `loss` (f32, one), `counts` (int32, a router's experts),
    `offsets` (int32, one more: the offsets of the products by expert), `rates` (f32, for
    moe_balance_backward)."""

    def __init__(self, loss, counts, offsets, rates):
        e = counts.numel()
        for name, t, dt, n in (("loss", loss, "torch.float32", 1), ("counts", counts, "torch.int32", e),
                               ("offsets", offsets, "torch.int32", e + 1),
                               ("rates", rates, "torch.float32", e)):
            if str(t.dtype) != dt or t.numel() != n or not t.is_contiguous():
                raise GemmkitError(GK_EINVAL, f"gemmkit: {name} must hold {n} contiguous {dt[6:]}")
        self.experts, self._parts = e, [loss, counts, offsets, rates]
        self._where = _one_device("loss", loss, "counts", counts, "offsets", offsets, "rates", rates)
        self._at = [t.data_ptr() for t in self._parts]

    def _part(self, i):
        if self._parts is None:  # parts of one buffer (empty), cut when they are asked for
            e, f32 = self.experts, _cuda[0].float32
            loss, counts, offsets, rates = self._where.split_with_sizes((1, e, e + 1, e))
            self._parts = [loss.view(f32), counts, offsets, rates.view(f32)]
        return self._parts[i]

    loss = property(lambda self: self._part(0))
    counts = property(lambda self: self._part(1))
    offsets = property(lambda self: self._part(2))
    rates = property(lambda self: self._part(3))

    @staticmethod
    def empty(experts: int, stream=None) -> "MoeBalance":
        """Unwritten results on the current device, allocated for torch's current stream or `stream`."""
        calls = _cuda or _cuda_calls()
        if calls is None:
            raise GemmkitError(GK_ENODEV, "gemmkit: no CUDA device")
        buf = _buffer(3 * experts + 2, calls[0].int32, stream)
        b = MoeBalance.__new__(MoeBalance)
        b.experts, b._where, b._parts = experts, buf, None
        at = buf.data_ptr()
        b._at = [at, at + 4, at + 4 * (experts + 1), at + 4 * (2 * experts + 2)]
        return b


def _ids(ids, tokens):
    """(pointer, length, ids a token, 64-bit) of a tokens x top tensor."""
    torch = (_cuda or _cuda_calls() or (None,))[0]
    wide = 0 if torch and ids.dtype is torch.int32 else 1 if torch and ids.dtype is torch.int64 else None
    shape = ids.shape
    if wide is None or len(shape) != 2 or shape[0] != tokens or not ids.is_contiguous():
        raise GemmkitError(GK_EINVAL, f"gemmkit: ids must be a contiguous {tokens} x top tensor of int32 "
                                      "or int64")
    return ids.data_ptr(), shape[0] * shape[1], shape[1], wide


def moe_balance(logits: MatRef, ids, coef: float = 1.0, out: Optional[MoeBalance] = None,
                x_type: Optional[int] = None, stream=None, sync: bool = True) -> MoeBalance:
    """A router's balance loss and the experts' counts and offsets (extension): `logits` (tokens x
    experts, f32, f16 or bf16), `ids` (tokens x top, int32 or int64, contiguous) the experts that each
    token goes to, a negative id for none; a token without any is padding. loss = coef * experts *
    sum_e (counts_e / routed) * (mean of softmax(logits)_e over the live tokens)."""
    _same_device("logits", logits.data, "ids", ids, "out", None if out is None else out._where)
    i = _ids(ids, logits.rows)
    if out is None:
        out = MoeBalance.empty(logits.cols, stream=stream)
    elif out.experts != logits.cols:
        raise GemmkitError(GK_EINVAL, f"gemmkit: the results are not of {logits.cols} experts")
    if x_type is None:
        x_type = _elem_type(logits.data, -1)
    _check(_lib.load().gk_moe_balance(logits.c(), x_type, *i, float(coef), *out._at, _stream(stream)))
    if sync:
        _sync(stream)
    return out


def moe_balance_backward(logits: MatRef, ids, balance: MoeBalance, dloss, dlogits: MatMut,
                         x_type: Optional[int] = None, stream=None, sync: bool = True) -> None:
    """The loss's gradient by the logits (extension), times `dloss` (one f32 on the device); padding
    gets zeros. dlogits has the logits' type and may be the logits themselves."""
    _same_device("logits", logits.data, "ids", ids, "balance", balance._where, "dloss", dloss,
                 "dlogits", dlogits.data)
    i = _ids(ids, logits.rows)
    if balance.experts != logits.cols:
        raise GemmkitError(GK_EINVAL, f"gemmkit: the results are not of {logits.cols} experts")
    if dloss.dtype is not _cuda[0].float32 or dloss.numel() != 1:
        raise GemmkitError(GK_EINVAL, "gemmkit: dloss must be one f32")
    if x_type is None:
        x_type = _elem_type(logits.data, -1)
    if _elem_type(dlogits.data, x_type) != x_type:
        raise GemmkitError(GK_EINVAL, "gemmkit: dlogits must have the logits' type")
    _check(_lib.load().gk_moe_balance_backward(logits.c(), x_type, *i, balance._at[3], dloss.data_ptr(),
                                               dlogits.c(), _stream(stream)))
    if sync:
        _sync(stream)


# ---- i8 -> i32 without allocation ---------------------------------------------------------

NOALLOC_SCRATCH_BYTES = 16 << 20


def gemm_i8_noalloc_unchecked(m, k, n, alpha, a, rsa, csa, b, rsb, csb, beta, c, rsc, csc,
                              stream=None) -> None:
    """gemm_i8_unchecked for callers that must not allocate device memory: operand packs use
    the library's fixed 16 MiB device scratch (shared by all calls; order calls on one
    stream). Raises GemmkitError(GK_EINVAL) when the packs need more than that."""
    _check(_lib.load().gk_gemm_i8_noalloc_unchecked(m, k, n, alpha, a, rsa, csa, b, rsb, csb,
                                                    beta, c, rsc, csc, _stream(stream)))


# ---- misc -----------------------------------------------------------------------------------

def set_tile_n(bn: int) -> None:
    """Force the MMA tile width (16/32/64/128/192/256) on this thread; 0 drops the override
    (the GEMMKIT_CUDA_BN knob, by default chosen per shape)."""
    _check(_lib.load().gk_set_tile_n(bn))


def knob_names() -> list[str]:
    """The engine's knobs (gemmkit's tuning knobs, gemmkit/src/tuning.rs:585-690)."""
    return _lib.load().gk_knob_names().decode().split(",")


def knob_get(name: str) -> int:
    """The value in effect: the run-time override, else the environment, else the default."""
    v = C.c_int64()
    _check(_lib.load().gk_knob_get(name.encode(), C.byref(v)))
    return int(v.value)


def knob_set(name: str, value: int) -> None:
    """Process-wide run-time override of a knob; a negative value drops the override."""
    _check(_lib.load().gk_knob_set(name.encode(), int(value)))


def device_status(device: int = 0, clear: bool = True) -> int:
    v = C.c_uint32()
    _check(_lib.load().gk_device_status(device, int(clear), C.byref(v)))
    return v.value


def selftest_wait_timeout(timeout_ns: int, stream=None) -> int:
    """Run the bounded-wait self test; returns the status code (GK_ETIMEOUT expected)."""
    return _lib.load().gk_selftest_wait_timeout(timeout_ns, _stream(stream))
