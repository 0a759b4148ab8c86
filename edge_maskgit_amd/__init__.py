"""edge_maskgit_amd — MI355X (gfx950) backend for the edge_maskgit Q8_0/Q4_K FC hot path.

The product is the native code: ``lib/libmgh.so`` (HIP kernels + the C ABI declared in
``include/mgh.h``) and ``lib/libmg_hip.so`` (the C++ mg tensor/graph API and HipRuntime).
This module is a thin ctypes binding used by tests and bench.py. It never falls back to
a CPU implementation: if the native library is missing or no gfx950 device is present,
calls raise.
"""
from __future__ import annotations

import ctypes
import os

import numpy as np

PKG = os.path.dirname(os.path.abspath(__file__))
LIB_DIR = os.path.join(PKG, "lib")
LIBMGH = os.path.join(LIB_DIR, "libmgh.so")

WTYPE_F32 = 0
WTYPE_Q8_0 = 8
WTYPE_Q4_K = 12
ACT_NONE, ACT_GELU, ACT_SILU = 0, 1, 2
EMIT_NONE, EMIT_INT8, EMIT_DEQ_F16 = 0, 1, 2
ALGO_AUTO, ALGO_INT8, ALGO_DEQ_F16 = 0, 1, 2
ROPE_HALVES, ROPE_PAIRS, ROPE_AXIS_HALVES = 0, 1, 2

# every entry point include/mgh.h declares (checked by tests/test_abi.py)
MGH_SYMBOLS = [
    "mgh_create", "mgh_destroy", "mgh_last_error", "mgh_device_name", "mgh_version",
    "mgh_alloc", "mgh_free", "mgh_h2d", "mgh_d2h", "mgh_fill_u32", "mgh_sync",
    "mgh_timer_start", "mgh_timer_stop",
    "mgh_quantize_act_q8", "mgh_gemm_q", "mgh_gemm_q_f32in", "mgh_debug_block_dots",
    "mgh_graph_begin", "mgh_graph_end", "mgh_graph_launch", "mgh_graph_destroy",
    "mgh_quantize_act_q8_codes16",
    "mgh_packed_weight_bytes", "mgh_pack_weights", "mgh_gemm_q_packed", "mgh_debug_block_dots_packed",
    "mgh_gemm_q_packed_f32in",
    "mgh_layernorm_affine", "mgh_flash_attn_f16kv", "mgh_gemm_f32", "mgh_get_rows", "mgh_add",
    "mgh_copy_strided", "mgh_decode_state_bytes", "mgh_decode_work_bytes", "mgh_decode_init",
    "mgh_decode_step", "mgh_packed_weight_bytes_f16", "mgh_pack_weights_f16", "mgh_f32_to_f16",
    "mgh_gemm_h16", "mgh_gemm_h16_f32in", "mgh_gemm_h16_y16", "mgh_gemm_h16_ln", "mgh_flash_attn_f16kv_o16", "mgh_flash_attn_f16in",
    "mgh_softmax", "mgh_binary", "mgh_scale", "mgh_unary", "mgh_gemm_f32_batched",
    "mgh_gemm_h16_f32in_noalloc", "mgh_conv2d", "mgh_group_norm", "mgh_upscale", "mgh_conv2d_ex",
    "mgh_conv2d_packed_bytes", "mgh_conv2d_pack_weights", "mgh_conv2d_i8_weight_bytes",
    "mgh_conv2d_i8_pack_weights", "mgh_conv2d_i8",
    "mgh_packed_weight_bytes_dq", "mgh_pack_weights_dq", "mgh_gemm_dq", "mgh_gemm_dq_f32in",
    "mgh_gemm_dq_y16", "mgh_gemm_dq_ln", "mgh_dequant_weights_f32",
    "mgh_attn_masked", "mgh_kv8_code_bytes", "mgh_kv8_scale_bytes", "mgh_kv8_tail_bytes", "mgh_kv8_append",
    "mgh_kv8_advance", "mgh_kv8_attn", "mgh_kv8_read", "mgh_logits_process",
    "mgh_rope", "mgh_kv8_append_rope", "mgh_kv8_attn_shared", "mgh_sample",
]

_lib = None


class MghError(RuntimeError):
    pass


def build_native(verbose: bool = False) -> None:
    """Compile the native libraries in-tree (see edge_maskgit_amd/build.py)."""
    import importlib
    importlib.import_module(__name__ + ".build").build(verbose=verbose, force=True)


def lib():
    """Load libmgh.so (raises if it was not built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIBMGH):
            raise MghError(f"native library missing: {LIBMGH} — run __graft_entry__.build()")
        L = ctypes.CDLL(LIBMGH)
        P, I, SZ = ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t
        L.mgh_create.argtypes = [I, ctypes.POINTER(P)]
        L.mgh_destroy.argtypes = [P]
        L.mgh_destroy.restype = None
        L.mgh_last_error.argtypes = [P]
        L.mgh_last_error.restype = ctypes.c_char_p
        L.mgh_device_name.argtypes = [P]
        L.mgh_device_name.restype = ctypes.c_char_p
        L.mgh_alloc.argtypes = [P, SZ, ctypes.POINTER(P)]
        L.mgh_free.argtypes = [P, P]
        L.mgh_h2d.argtypes = [P, P, P, SZ]
        L.mgh_d2h.argtypes = [P, P, P, SZ]
        L.mgh_fill_u32.argtypes = [P, P, ctypes.c_uint32, SZ]
        L.mgh_sync.argtypes = [P]
        L.mgh_timer_start.argtypes = [P]
        L.mgh_timer_stop.argtypes = [P, ctypes.POINTER(ctypes.c_float)]
        L.mgh_quantize_act_q8.argtypes = [P, P, I, I, P, P, P]
        L.mgh_gemm_q.argtypes = [P, I, P, I, I, P, P, P, I, P, I, P, P]
        L.mgh_gemm_q_f32in.argtypes = [P, I, I, P, I, I, P, I, P, I, P, P]
        L.mgh_debug_block_dots.argtypes = [P, I, P, I, I, P, I, P]
        L.mgh_quantize_act_q8_codes16.argtypes = [P, P, I, I, P, P, P]
        L.mgh_packed_weight_bytes.argtypes = [I, I, I]
        L.mgh_packed_weight_bytes.restype = SZ
        L.mgh_pack_weights.argtypes = [P, I, P, I, I, P]
        L.mgh_gemm_q_packed.argtypes = [P, I, P, I, I, P, P, P, I, P, I, P, P]
        L.mgh_debug_block_dots_packed.argtypes = [P, I, P, I, I, P, I, P]
        L.mgh_gemm_q_packed_f32in.argtypes = [P, I, I, P, I, I, P, I, P, I, P, P]
        I64 = ctypes.c_int64
        L.mgh_layernorm_affine.argtypes = [P, P, P, P, I, I, ctypes.c_float, P, I, P, P, P]
        L.mgh_flash_attn_f16kv.argtypes = [P, P, P, P, P, I, I, I, I, ctypes.c_float, P, P]
        L.mgh_gemm_f32.argtypes = [P, P, I, I, P, I, P, I, P, P]
        L.mgh_get_rows.argtypes = [P, P, I64, I64, P, I64, P]
        L.mgh_add.argtypes = [P, P, P, I64, P, I64]
        L.mgh_copy_strided.argtypes = [P, P, P, P, P]
        L.mgh_packed_weight_bytes_f16.argtypes = [I, I]
        L.mgh_packed_weight_bytes_f16.restype = SZ
        L.mgh_pack_weights_f16.argtypes = [P, I, P, I, I, P]
        L.mgh_f32_to_f16.argtypes = [P, P, I64, P]
        L.mgh_gemm_h16.argtypes = [P, P, I, I, P, I, P, I, P, P]
        L.mgh_gemm_h16_f32in.argtypes = [P, P, I, I, P, I, P, I, P, P]
        L.mgh_gemm_h16_y16.argtypes = [P, P, I, I, P, I, P, I, P, P]
        L.mgh_gemm_h16_ln.argtypes = [P, P, I, I, P, I, P, I, P, P, P, P, ctypes.c_float, P, I, P, P, P]
        L.mgh_gemm_h16_f32in_noalloc.argtypes = [P, P, I, I, P, I, P, I, P, P]
        L.mgh_packed_weight_bytes_dq.argtypes = [I, I, I]
        L.mgh_packed_weight_bytes_dq.restype = SZ
        L.mgh_pack_weights_dq.argtypes = [P, I, P, I, I, P]
        L.mgh_dequant_weights_f32.argtypes = [P, I, P, I, I, P]
        L.mgh_gemm_dq.argtypes = [P, I, P, I, I, P, I, P, I, P, P]
        L.mgh_gemm_dq_f32in.argtypes = [P, I, P, I, I, P, I, P, I, P, P]
        L.mgh_gemm_dq_y16.argtypes = [P, I, P, I, I, P, I, P, I, P, P]
        L.mgh_gemm_dq_ln.argtypes = [P, I, P, I, I, P, I, P, I, P, P, P, P, ctypes.c_float, P, I, P, P, P]
        L.mgh_flash_attn_f16kv_o16.argtypes = [P, P, P, P, P, I, I, I, I, ctypes.c_float, P, P]
        L.mgh_flash_attn_f16in.argtypes = [P, P, P, P, P, I, I, I, I, ctypes.c_float, P, P, P]
        L.mgh_decode_state_bytes.argtypes = [I]
        L.mgh_decode_state_bytes.restype = SZ
        L.mgh_decode_work_bytes.argtypes = [I, I]
        L.mgh_decode_work_bytes.restype = SZ
        L.mgh_decode_init.argtypes = [P, I, P, P]
        L.mgh_decode_step.argtypes = [P, P, P, P, I, I, I, I, I, I, I, I, ctypes.c_float, P, P]
        L.mgh_softmax.argtypes = [P, P, I64, I, ctypes.c_float, P]
        L.mgh_binary.argtypes = [P, I, P, P, P, P, P, P, P]
        L.mgh_scale.argtypes = [P, P, I64, ctypes.c_float, P]
        L.mgh_unary.argtypes = [P, I, P, I64, P]
        L.mgh_gemm_f32_batched.argtypes = [P, P, P, P, P, P, P, P, I, P, P]
        L.mgh_conv2d.argtypes = [P, P, I, I, I, I, P, I, I, I, I, I, P]
        L.mgh_conv2d_ex.argtypes = [P, P, I, I, I, I, P, P, I, I, I, I, I, P, P, P]
        L.mgh_conv2d_packed_bytes.argtypes = [I, I, I, I]
        L.mgh_conv2d_packed_bytes.restype = ctypes.c_size_t
        L.mgh_conv2d_pack_weights.argtypes = [P, P, I, I, I, I, P]
        L.mgh_conv2d_i8_weight_bytes.argtypes = [I, I, I, I]
        L.mgh_conv2d_i8_weight_bytes.restype = ctypes.c_size_t
        L.mgh_conv2d_i8_pack_weights.argtypes = [P, P, I, I, I, I, P]
        L.mgh_conv2d_i8.argtypes = [P, P, I, I, I, I, P, I, I, I, I, I, P, P, P]
        L.mgh_group_norm.argtypes = [P, P, I, I, I, I, I, ctypes.c_float, P, P, P]
        L.mgh_upscale.argtypes = [P, P, I, I, I, I, I, P]
        F = ctypes.c_float
        L.mgh_attn_masked.argtypes = [P, P, P, P, I, P, P, I, I, I, I, I, I, F, P, P, P, P]
        L.mgh_kv8_code_bytes.argtypes = [I64, I, I]
        L.mgh_kv8_code_bytes.restype = SZ
        L.mgh_kv8_scale_bytes.argtypes = [I64, I]
        L.mgh_kv8_scale_bytes.restype = SZ
        L.mgh_kv8_tail_bytes.argtypes = [I, I, I]
        L.mgh_kv8_tail_bytes.restype = SZ
        L.mgh_kv8_append.argtypes = [P, P, P, P, I, P, I, P, P]
        L.mgh_kv8_advance.argtypes = [P, P, P, I, I]
        L.mgh_kv8_attn.argtypes = [P, P, P, I, P, I, P, P, I, F, F, P, P, P, P]
        L.mgh_kv8_read.argtypes = [P, P, P, I, P, P, P, P, P]
        L.mgh_logits_process.argtypes = [P, P, I, I64, I, I, P, P, I64]
        L.mgh_rope.argtypes = [P, P, P, I, P, I, I, I, I, P, P, P, P, P]
        L.mgh_kv8_append_rope.argtypes = [P, P, P, P, P, I, P, I, P, P, P, P, I, P, P]
        L.mgh_kv8_attn_shared.argtypes = [P, P, P, I, P, I, P, P, I, P, I, I, F, F, P, P, P, P]
        L.mgh_sample.argtypes = [P, P, I, I64, I, I, P, P, P, P]
        L.mgh_graph_begin.argtypes = [P]
        L.mgh_graph_end.argtypes = [P, ctypes.POINTER(P)]
        L.mgh_graph_launch.argtypes = [P, P]
        L.mgh_graph_destroy.argtypes = [P]
        L.mgh_graph_destroy.restype = None
        _lib = L
    return _lib


def packed_weight_bytes_f16(N: int, K: int) -> int:
    return int(lib().mgh_packed_weight_bytes_f16(N, K))


def packed_weight_bytes_dq(wtype: int, N: int, K: int) -> int:
    """bytes of the K-loop-dequant weight layout (GGUF-sized: 1.0625 / 0.5625 bytes per weight
    for N % 16 == 0)"""
    return int(lib().mgh_packed_weight_bytes_dq(wtype, N, K))


def decode_state_bytes(B: int) -> int:
    return int(lib().mgh_decode_state_bytes(B))


def decode_work_bytes(B: int, S: int) -> int:
    return int(lib().mgh_decode_work_bytes(B, S))


def packed_weight_bytes(wtype: int, N: int, K: int) -> int:
    """Size of mgh_pack_weights' output (0 for an invalid type/shape)."""
    return int(lib().mgh_packed_weight_bytes(wtype, N, K))


class DeviceBuffer:
    """Owned device allocation (freed with the context)."""

    def __init__(self, ctx: "Context", nbytes: int):
        self.ctx = ctx
        self.nbytes = int(nbytes)
        p = ctypes.c_void_p()
        ctx._check(lib().mgh_alloc(ctx.h, self.nbytes, ctypes.byref(p)))
        self.ptr = p.value

    def free(self):
        if self.ptr:
            lib().mgh_free(self.ctx.h, ctypes.c_void_p(self.ptr))
            self.ptr = None

    @property
    def p(self):
        return ctypes.c_void_p(self.ptr)


class _AttnOpts(ctypes.Structure):
    _fields_ = [("cap", ctypes.c_float), ("causal", ctypes.c_int), ("d_slopes", ctypes.c_void_p),
                ("d_prefix", ctypes.c_void_p), ("d_docs", ctypes.c_void_p), ("doc_stride", ctypes.c_int64)]


class _LogitsOpts(ctypes.Structure):
    _fields_ = [("d_hist", ctypes.c_void_p), ("hist_stride", ctypes.c_int64), ("max_hist", ctypes.c_int),
                ("d_hist_len", ctypes.c_void_p), ("d_rep", ctypes.c_void_p), ("d_freq", ctypes.c_void_p),
                ("d_pres", ctypes.c_void_p), ("d_bias", ctypes.c_void_p), ("bias_stride", ctypes.c_int64),
                ("d_allowed", ctypes.c_void_p), ("allowed_stride", ctypes.c_int64)]


def _addr(b):
    """address of a DeviceBuffer, an int or None, as a ctypes structure's pointer field takes it"""
    return b.ptr if isinstance(b, DeviceBuffer) else b


class Kv8(ctypes.Structure):
    """mgh_kv8: a key / value cache in 8 bits over buffers that the caller owns (include/mgh.h has their
    layout and sizes). table: B rows of max_blocks page numbers (int32), table_stride apart."""

    _fields_ = [("d_k", ctypes.c_void_p), ("d_v", ctypes.c_void_p), ("d_scales", ctypes.c_void_p),
                ("d_k_tail", ctypes.c_void_p), ("d_v_tail", ctypes.c_void_p), ("d_table", ctypes.c_void_p),
                ("table_stride", ctypes.c_int64), ("pages", ctypes.c_int64), ("max_blocks", ctypes.c_int),
                ("Hkv", ctypes.c_int), ("D", ctypes.c_int), ("B", ctypes.c_int)]

    def __init__(self, k, v, scales, k_tail, v_tail, table, max_blocks, pages, Hkv, D, B, table_stride=None):
        super().__init__(*map(_addr, (k, v, scales, k_tail, v_tail, table)),
                         max_blocks if table_stride is None else table_stride, pages, max_blocks, Hkv, D, B)


class Rope(ctypes.Structure):
    """mgh_rotation: how pairs of features turn with their token's positions (include/mgh.h has the orders). pairs: of each
    axis; freqs: angle per unit of position of each pair; pos: whole positions (int32) on the device, pos_strides apart
    (token, sequence, axis), or None: consecutive ones."""

    _fields_ = [("axes", ctypes.c_int), ("pairs", ctypes.c_int * 4), ("order", ctypes.c_int), ("h_freqs", ctypes.c_void_p),
                ("d_pos", ctypes.c_void_p), ("pos_strides", ctypes.c_int64 * 3)]

    def __init__(self, pairs, freqs, order=ROPE_HALVES, pos=None, pos_strides=(0, 0, 0)):
        if not 1 <= len(pairs) <= 4:
            raise MghError("a rotation has 1 to 4 axes")
        if len(freqs) < sum(pairs):
            raise MghError("a frequency for every pair is needed")
        self._freqs = (ctypes.c_double * max(len(freqs), 1))(*freqs)
        super().__init__(len(pairs), (ctypes.c_int * 4)(*pairs), order, ctypes.addressof(self._freqs), _addr(pos),
                         (ctypes.c_int64 * 3)(*pos_strides))


class _SampleOpts(ctypes.Structure):
    _fields_ = [("d_temp", ctypes.c_void_p), ("d_top_k", ctypes.c_void_p), ("d_top_p", ctypes.c_void_p),
                ("d_min_p", ctypes.c_void_p)]


def kv8_code_bytes(pages: int, Hkv: int, D: int) -> int:
    """bytes of a Kv8's k, and of its v"""
    return int(lib().mgh_kv8_code_bytes(pages, Hkv, D))


def kv8_scale_bytes(pages: int, Hkv: int) -> int:
    return int(lib().mgh_kv8_scale_bytes(pages, Hkv))


def kv8_tail_bytes(B: int, Hkv: int, D: int) -> int:
    """bytes of a Kv8's k_tail, and of its v_tail"""
    return int(lib().mgh_kv8_tail_bytes(B, Hkv, D))


class Context:
    """One mgh_ctx (device + stream). Not thread-safe, like the reference runtime."""

    def __init__(self, device: int = 0):
        h = ctypes.c_void_p()
        rc = lib().mgh_create(device, ctypes.byref(h))
        if rc != 0:
            raise MghError(f"mgh_create({device}) failed with {rc} (no gfx950 device?)")
        self.h = h
        self._bufs: list[DeviceBuffer] = []

    def close(self):
        if self.h:
            for b in self._bufs:
                b.free()
            self._bufs.clear()
            lib().mgh_destroy(self.h)
            self.h = None

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.close()

    def _check(self, rc):
        if rc != 0:
            raise MghError(f"mgh error {rc}: {lib().mgh_last_error(self.h).decode()}")

    @property
    def device_name(self) -> str:
        return lib().mgh_device_name(self.h).decode()

    # ---- memory ----
    def alloc(self, nbytes: int) -> DeviceBuffer:
        b = DeviceBuffer(self, nbytes)
        self._bufs.append(b)
        return b

    def upload(self, arr: np.ndarray) -> DeviceBuffer:
        arr = np.ascontiguousarray(arr)
        b = self.alloc(max(arr.nbytes, 1))
        self._check(lib().mgh_h2d(self.h, b.p, arr.ctypes.data_as(ctypes.c_void_p), arr.nbytes))
        return b

    def write(self, buf: DeviceBuffer, arr: np.ndarray):
        """Copy a host array into the start of an existing device buffer."""
        arr = np.ascontiguousarray(arr)
        if arr.nbytes > buf.nbytes:
            raise ValueError("write: array larger than the buffer")
        self._check(lib().mgh_h2d(self.h, buf.p, arr.ctypes.data_as(ctypes.c_void_p), arr.nbytes))

    def download(self, buf: DeviceBuffer, shape, dtype) -> np.ndarray:
        out = np.empty(shape, dtype)
        self._check(lib().mgh_d2h(self.h, out.ctypes.data_as(ctypes.c_void_p), buf.p, out.nbytes))
        return out

    def free(self, buf: DeviceBuffer):
        buf.free()
        if buf in self._bufs:
            self._bufs.remove(buf)

    def sync(self):
        self._check(lib().mgh_sync(self.h))

    def timer_start(self):
        self._check(lib().mgh_timer_start(self.h))

    def timer_stop(self) -> float:
        ms = ctypes.c_float()
        self._check(lib().mgh_timer_stop(self.h, ctypes.byref(ms)))
        return ms.value

    # ---- kernels (device pointers in, device pointers out; stream-ordered) ----
    @staticmethod
    def _ptr(b):
        if b is None:
            return None
        return b.p if isinstance(b, DeviceBuffer) else ctypes.c_void_p(int(b))

    def fill_u32(self, buf, value, n_words):
        self._check(lib().mgh_fill_u32(self.h, self._ptr(buf), value, n_words))

    def quantize_act_q8(self, x, M, K, qx, dx, sx=None):
        P = self._ptr
        self._check(lib().mgh_quantize_act_q8(self.h, P(x), M, K, P(qx), P(dx), P(sx)))

    def gemm_q(self, wtype, w, N, K, qx, dx, sx, M, bias, act, resid, y):
        P = self._ptr
        self._check(lib().mgh_gemm_q(self.h, wtype, P(w), N, K, P(qx), P(dx), P(sx), M,
                                     P(bias), act, P(resid), P(y)))

    def quantize_act_q8_codes16(self, x, M, K, qx16, dx, sx=None):
        P = self._ptr
        self._check(lib().mgh_quantize_act_q8_codes16(self.h, P(x), M, K, P(qx16), P(dx), P(sx)))

    def pack_weights(self, wtype, w, N, K, wp):
        P = self._ptr
        self._check(lib().mgh_pack_weights(self.h, wtype, P(w), N, K, P(wp)))

    def gemm_q_packed(self, wtype, wp, N, K, qx16, dx, sx, M, bias, act, resid, y):
        P = self._ptr
        self._check(lib().mgh_gemm_q_packed(self.h, wtype, P(wp), N, K, P(qx16), P(dx), P(sx), M,
                                            P(bias), act, P(resid), P(y)))

    def layernorm_affine(self, x, gamma, beta, rows, D, eps, y, emit=0, codes=None, dx=None, s4=None):
        P = self._ptr
        self._check(lib().mgh_layernorm_affine(self.h, P(x), P(gamma), P(beta), rows, D, eps, P(y),
                                               emit, P(codes), P(dx), P(s4)))

    def flash_attn_f16kv(self, q, k, v, strides, D, S, H, B, scale, o, o_strides=None):
        P = self._ptr
        st = (ctypes.c_int64 * 4)(*strides)
        ost = (ctypes.c_int64 * 4)(*o_strides) if o_strides is not None else None
        self._check(lib().mgh_flash_attn_f16kv(self.h, P(q), P(k), P(v), st, D, S, H, B, scale,
                                               P(o), ost))

    def gemm_f32(self, w, N, K, x, M, bias, act, resid, y):
        P = self._ptr
        self._check(lib().mgh_gemm_f32(self.h, P(w), N, K, P(x), M, P(bias), act, P(resid), P(y)))

    def get_rows(self, a, E, R, ids, n, out):
        P = self._ptr
        self._check(lib().mgh_get_rows(self.h, P(a), E, R, P(ids), n, P(out)))

    def add(self, a, b, nb, out, n):
        P = self._ptr
        self._check(lib().mgh_add(self.h, P(a), P(b), nb, P(out), n))

    def copy_strided(self, a, ne, strides, out):
        P = self._ptr
        self._check(lib().mgh_copy_strided(self.h, P(a), (ctypes.c_int64 * 4)(*ne),
                                           (ctypes.c_int64 * 4)(*strides), P(out)))

    def pack_weights_f16(self, wtype, w, N, K, wp16):
        self._check(lib().mgh_pack_weights_f16(self.h, wtype, self._ptr(w), N, K, self._ptr(wp16)))

    def f32_to_f16(self, x, n, x16):
        self._check(lib().mgh_f32_to_f16(self.h, self._ptr(x), n, self._ptr(x16)))

    def gemm_h16(self, wp16, N, K, x16, M, bias, act, resid, y):
        P = self._ptr
        self._check(lib().mgh_gemm_h16(self.h, P(wp16), N, K, P(x16), M, P(bias), act, P(resid), P(y)))

    def gemm_h16_ln(self, wp16, N, K, x16, M, bias, act, resid, y, gamma, beta, eps, y_ln, emit=0, codes=None,
                    dx=None, s4=None):
        """gemm_h16 into y, then the LayerNorm-affine of y's rows into y_ln (and the emitted
        operand), as gemm_h16 followed by layernorm_affine(y)."""
        P = self._ptr
        self._check(lib().mgh_gemm_h16_ln(self.h, P(wp16), N, K, P(x16), M, P(bias), act, P(resid), P(y), P(gamma),
                                          P(beta), eps, P(y_ln), emit, P(codes), P(dx), P(s4)))

    def gemm_h16_y16(self, wp16, N, K, x16, M, bias, act, resid, y16):
        P = self._ptr
        self._check(lib().mgh_gemm_h16_y16(self.h, P(wp16), N, K, P(x16), M, P(bias), act, P(resid), P(y16)))

    def flash_attn_f16kv_o16(self, q, k, v, strides, D, S, H, B, scale, o16, o_strides=None):
        P = self._ptr
        st = (ctypes.c_int64 * 4)(*strides)
        ost = None if o_strides is None else (ctypes.c_int64 * 4)(*o_strides)
        self._check(lib().mgh_flash_attn_f16kv_o16(self.h, P(q), P(k), P(v), st, D, S, H, B, scale, P(o16), ost))

    def flash_attn_f16in(self, q16, k16, v16, strides, D, S, H, B, scale, o=None, o16=None, o_strides=None):
        """Attention on fp16 q/k/v (element strides as for flash_attn_f16kv); exactly one of
        o (fp32) and o16 (fp16) is given."""
        P = self._ptr
        st = (ctypes.c_int64 * 4)(*strides)
        ost = None if o_strides is None else (ctypes.c_int64 * 4)(*o_strides)
        self._check(lib().mgh_flash_attn_f16in(self.h, P(q16), P(k16), P(v16), st, D, S, H, B, scale,
                                               P(o), P(o16), ost))

    def gemm_h16_f32in(self, wp16, N, K, x, M, bias, act, resid, y):
        P = self._ptr
        self._check(lib().mgh_gemm_h16_f32in(self.h, P(wp16), N, K, P(x), M, P(bias), act, P(resid), P(y)))

    def dequant_weights_f32(self, wtype, w, N, K, out):
        self._check(lib().mgh_dequant_weights_f32(self.h, wtype, self._ptr(w), N, K, self._ptr(out)))

    def pack_weights_dq(self, wtype, w, N, K, wdq):
        self._check(lib().mgh_pack_weights_dq(self.h, wtype, self._ptr(w), N, K, self._ptr(wdq)))

    def gemm_dq(self, wtype, wdq, N, K, x16, M, bias, act, resid, y):
        P = self._ptr
        self._check(lib().mgh_gemm_dq(self.h, wtype, P(wdq), N, K, P(x16), M, P(bias), act, P(resid), P(y)))

    def gemm_dq_f32in(self, wtype, wdq, N, K, x, M, bias, act, resid, y):
        P = self._ptr
        self._check(lib().mgh_gemm_dq_f32in(self.h, wtype, P(wdq), N, K, P(x), M, P(bias), act, P(resid), P(y)))

    def gemm_dq_y16(self, wtype, wdq, N, K, x16, M, bias, act, resid, y16):
        P = self._ptr
        self._check(lib().mgh_gemm_dq_y16(self.h, wtype, P(wdq), N, K, P(x16), M, P(bias), act, P(resid), P(y16)))

    def gemm_dq_ln(self, wtype, wdq, N, K, x16, M, bias, act, resid, y, gamma, beta, eps, y_ln, emit=0,
                   codes=None, dx=None, s4=None):
        P = self._ptr
        self._check(lib().mgh_gemm_dq_ln(self.h, wtype, P(wdq), N, K, P(x16), M, P(bias), act, P(resid), P(y),
                                         P(gamma), P(beta), eps, P(y_ln), emit, P(codes), P(dx), P(s4)))

    def gemm_h16_f32in_noalloc(self, wp16, N, K, x, M, bias, act, resid, y):
        """mgh_gemm_h16_f32in with its scratch in the library's fixed per-GPU array."""
        P = self._ptr
        self._check(lib().mgh_gemm_h16_f32in_noalloc(self.h, P(wp16), N, K, P(x), M, P(bias), act, P(resid),
                                                     P(y)))

    def decode_init(self, seeds, state):
        """seeds: host sequence of B uint64 seeds; state: mgh_decode_state_bytes(B) bytes."""
        sd = (ctypes.c_uint64 * len(seeds))(*[int(v) for v in seeds])
        self._check(lib().mgh_decode_init(self.h, len(seeds), sd, self._ptr(state)))

    def decode_step(self, state, work, logits, B, S, V, codebook, mask_id, n_tokens, step, n_steps,
                    choice_temp, tokens, result):
        P = self._ptr
        self._check(lib().mgh_decode_step(self.h, P(state), P(work), P(logits), B, S, V, codebook,
                                          mask_id, n_tokens, step, n_steps, choice_temp, P(tokens),
                                          P(result)))

    def gemm_q_packed_f32in(self, algo, wtype, wp, N, K, x, M, bias, act, resid, y):
        P = self._ptr
        self._check(lib().mgh_gemm_q_packed_f32in(self.h, algo, wtype, P(wp), N, K, P(x), M,
                                                  P(bias), act, P(resid), P(y)))

    def debug_block_dots_packed(self, wtype, wp, N, K, qx16, M, out):
        P = self._ptr
        self._check(lib().mgh_debug_block_dots_packed(self.h, wtype, P(wp), N, K, P(qx16), M, P(out)))

    def gemm_q_f32in(self, algo, wtype, w, N, K, x, M, bias, act, resid, y):
        P = self._ptr
        self._check(lib().mgh_gemm_q_f32in(self.h, algo, wtype, P(w), N, K, P(x), M,
                                           P(bias), act, P(resid), P(y)))

    def softmax(self, x, rows, D, scale, y):
        self._check(lib().mgh_softmax(self.h, self._ptr(x), rows, D, scale, self._ptr(y)))

    def binary(self, op, a, a_strides, b, b_ne, b_strides, ne, out):
        P, A = self._ptr, (lambda v: (ctypes.c_int64 * 4)(*v))
        self._check(lib().mgh_binary(self.h, op, P(a), A(a_strides), P(b), A(b_ne), A(b_strides), A(ne), P(out)))

    def scale(self, x, n, s, y):
        self._check(lib().mgh_scale(self.h, self._ptr(x), n, s, self._ptr(y)))

    def unary(self, act, x, n, y):
        self._check(lib().mgh_unary(self.h, act, self._ptr(x), n, self._ptr(y)))

    def gemm_f32_batched(self, w, w_ne, w_strides, x, x_ne, x_strides, bias, act, resid, y):
        P, A = self._ptr, (lambda v: (ctypes.c_int64 * 4)(*v))
        self._check(lib().mgh_gemm_f32_batched(self.h, P(w), A(w_ne), A(w_strides), P(x), A(x_ne), A(x_strides),
                                               P(bias), act, P(resid), P(y)))

    # ---- VQGAN decoder ops, layout {W, H, C, N} ----
    def conv2d(self, x, IW, IH, IC, N, ker, KW, KH, OC, stride, pad, y):
        P = self._ptr
        self._check(lib().mgh_conv2d(self.h, P(x), IW, IH, IC, N, P(ker), KW, KH, OC, stride, pad, P(y)))

    def conv2d_ex(self, x, IW, IH, IC, N, ker, packed, KW, KH, OC, stride, pad, bias, resid, y):
        P = self._ptr
        self._check(lib().mgh_conv2d_ex(self.h, P(x), IW, IH, IC, N, P(ker), P(packed), KW, KH, OC, stride, pad,
                                        P(bias), P(resid), P(y)))

    @staticmethod
    def conv2d_packed_bytes(KW, KH, IC, OC) -> int:
        return lib().mgh_conv2d_packed_bytes(KW, KH, IC, OC)

    def conv2d_pack_weights(self, ker, KW, KH, IC, OC, packed):
        P = self._ptr
        self._check(lib().mgh_conv2d_pack_weights(self.h, P(ker), KW, KH, IC, OC, P(packed)))

    @staticmethod
    def conv2d_i8_weight_bytes(KW, KH, IC, OC) -> int:
        return lib().mgh_conv2d_i8_weight_bytes(KW, KH, IC, OC)

    def conv2d_i8_pack_weights(self, ker, KW, KH, IC, OC, wq):
        P = self._ptr
        self._check(lib().mgh_conv2d_i8_pack_weights(self.h, P(ker), KW, KH, IC, OC, P(wq)))

    def conv2d_i8(self, x, IW, IH, IC, N, wq, KW, KH, OC, stride, pad, bias, resid, y):
        P = self._ptr
        self._check(lib().mgh_conv2d_i8(self.h, P(x), IW, IH, IC, N, P(wq), KW, KH, OC, stride, pad, P(bias),
                                        P(resid), P(y)))

    def group_norm(self, x, W, H, C, N, groups, eps, gamma, beta, y):
        P = self._ptr
        self._check(lib().mgh_group_norm(self.h, P(x), W, H, C, N, groups, eps, P(gamma), P(beta), P(y)))

    def upscale(self, x, W, H, C, N, factor, y):
        self._check(lib().mgh_upscale(self.h, self._ptr(x), W, H, C, N, factor, self._ptr(y)))

    # ---- generating token by token: masked attention, the 8-bit cache, logits ----
    def attn_masked(self, q, k, v, q_strides, kv_strides, D, Sq, Sk, H, Hkv, B, scale, o=None, o16=None, o_strides=None,
                    in16=True, cap=0.0, slopes=None, causal=False, prefix=None, docs=None, doc_stride=0):
        """Attention of {D, Sq, H, B} queries at positions Sk - Sq + i over {D, Sk, Hkv, B} keys (fp16, or
        fp32 with in16=False); exactly one of o (fp32) and o16 (fp16) is given."""
        P = self._ptr
        op = _AttnOpts(cap, bool(causal), _addr(slopes), _addr(prefix), _addr(docs), doc_stride)
        ost = None if o_strides is None else (ctypes.c_int64 * 4)(*o_strides)
        self._check(lib().mgh_attn_masked(self.h, P(q), P(k), P(v), int(in16), (ctypes.c_int64 * 4)(*q_strides),
                                          (ctypes.c_int64 * 4)(*kv_strides), D, Sq, Sk, H, Hkv, B, scale,
                                          ctypes.byref(op), P(o), P(o16), ost))

    def kv8_append(self, cache, k, v, strides, S, lens, new=None, in16=True):
        """The keys and values of up to S new tokens per sequence ({D, S, Hkv, B} views) into the cache at
        positions lens[b] + i."""
        P = self._ptr
        self._check(lib().mgh_kv8_append(self.h, ctypes.byref(cache), P(k), P(v), int(in16),
                                         (ctypes.c_int64 * 4)(*strides), S, P(lens), P(new)))

    def kv8_advance(self, lens, new, B, S):
        """lens[b] += new[b] (S where new is None); numbers that append refuses leave lens[b] as it is"""
        self._check(lib().mgh_kv8_advance(self.h, self._ptr(lens), self._ptr(new), B, S))

    def kv8_attn(self, cache, q, q_strides, S, lens, new, H, scale, o=None, o16=None, o_strides=None, in16=True, cap=0.0,
                 slopes=None):
        """Attention of up to S new tokens per sequence ({D, S, H, B} queries at positions lens[b] + i) over
        the cache, which already holds them; exactly one of o and o16 is given."""
        P = self._ptr
        ost = None if o_strides is None else (ctypes.c_int64 * 4)(*o_strides)
        self._check(lib().mgh_kv8_attn(self.h, ctypes.byref(cache), P(q), int(in16), (ctypes.c_int64 * 4)(*q_strides), S,
                                       P(lens), P(new), H, scale, cap, P(slopes), P(o), P(o16), ost))

    def kv8_read(self, cache, first, n, lens, k=None, v=None, k16=None, v16=None):
        """The values at positions first[b] + i (first None: i), i < n, of sequences of lens[b] tokens, to
        [B][Hkv][n][D] in k and v (fp32) or k16 and v16 (fp16)."""
        P = self._ptr
        self._check(lib().mgh_kv8_read(self.h, ctypes.byref(cache), P(first), n, P(lens), P(k), P(v), P(k16), P(v16)))

    def logits_process(self, x, rows, V, y, f16=False, x_stride=None, y_stride=None, hist=None, hist_stride=None,
                       max_hist=0, hist_len=None, rep=None, freq=None, pres=None, bias=None, bias_stride=0, allowed=None,
                       allowed_stride=0):
        """Penalties for the tokens of a history, a bias and a bit mask of allowed tokens on rows of V logits."""
        op = _LogitsOpts(_addr(hist), max_hist if hist_stride is None else hist_stride, max_hist, _addr(hist_len),
                         _addr(rep), _addr(freq), _addr(pres), _addr(bias), bias_stride, _addr(allowed), allowed_stride)
        self._check(lib().mgh_logits_process(self.h, self._ptr(x), int(f16), V if x_stride is None else x_stride, rows, V,
                                             ctypes.byref(op), self._ptr(y), V if y_stride is None else y_stride))

    def rope(self, rot, x, x_strides, D, S, H, B, y=None, y16=None, y_strides=None, first=None, new=None, in16=True):
        """Pairs of features of {D, S, H, B} heads turned by their tokens' positions (a Rope); exactly one of y (fp32) and y16
        (fp16) is given, y_strides None: as x's."""
        P = self._ptr
        self._check(lib().mgh_rope(self.h, ctypes.byref(rot), P(x), int(in16), (ctypes.c_int64 * 4)(*x_strides), D, S, H, B,
                                   P(first), P(new), P(y), P(y16),
                                   (ctypes.c_int64 * 4)(*(x_strides if y_strides is None else y_strides))))

    def kv8_append_rope(self, cache, rot, k, v, strides, S, lens, new=None, in16=True, q=None, q_strides=None, H=0, q_out=None,
                        qo_strides=None):
        """kv8_append with the keys turned by a Rope on the way, and the H heads of queries q ({D, S, H, B}, as k's type) to
        fp16 rows in q_out; positions None: lens[b] + i."""
        P = self._ptr
        four = lambda st: None if st is None else (ctypes.c_int64 * 4)(*st)  # noqa: E731
        self._check(lib().mgh_kv8_append_rope(self.h, ctypes.byref(cache), ctypes.byref(rot), P(k), P(v), int(in16), four(strides), S,
                                              P(lens), P(new), P(q), four(q_strides), H, P(q_out), four(qo_strides)))

    def kv8_attn_shared(self, cache, q, q_strides, S, lens, new, group, shared, max_shared, H, scale, o=None, o16=None,
                        o_strides=None, in16=True, cap=0.0, slopes=None):
        """kv8_attn where each `group` sequences in a row share their first shared[g] blocks (at most max_shared), which are
        read once for all of them."""
        P = self._ptr
        ost = None if o_strides is None else (ctypes.c_int64 * 4)(*o_strides)
        self._check(lib().mgh_kv8_attn_shared(self.h, ctypes.byref(cache), P(q), int(in16), (ctypes.c_int64 * 4)(*q_strides), S,
                                              P(lens), P(new), group, P(shared), max_shared, H, scale, cap, P(slopes), P(o), P(o16), ost))

    def sample(self, x, rows, V, u, ids, f16=False, x_stride=None, temp=None, top_k=None, top_p=None, min_p=None, prob=None):
        """A token drawn from each of rows of V logits (temperature, top-k, top-p, min-p of each row) with the random numbers
        u [rows] in [0, 1): ids (int32), prob its probability among the kept ones. x_stride 0: one row for all draws."""
        op = _SampleOpts(_addr(temp), _addr(top_k), _addr(top_p), _addr(min_p))
        self._check(lib().mgh_sample(self.h, self._ptr(x), int(f16), V if x_stride is None else x_stride, rows, V,
                                     ctypes.byref(op), self._ptr(u), self._ptr(ids), self._ptr(prob)))

    # ---- graphs ----
    def graph_begin(self):
        self._check(lib().mgh_graph_begin(self.h))

    def graph_end(self) -> "Graph":
        g = ctypes.c_void_p()
        self._check(lib().mgh_graph_end(self.h, ctypes.byref(g)))
        return Graph(self, g)

    def debug_block_dots(self, wtype, w, N, K, qx, M, out):
        P = self._ptr
        self._check(lib().mgh_debug_block_dots(self.h, wtype, P(w), N, K, P(qx), M, P(out)))


class Graph:
    """A captured, instantiated sequence of calls (mgh_graph)."""

    def __init__(self, ctx: Context, h):
        self.ctx = ctx
        self.h = h

    def launch(self):
        self.ctx._check(lib().mgh_graph_launch(self.ctx.h, self.h))

    def destroy(self):
        if self.h:
            lib().mgh_graph_destroy(self.h)
            self.h = None


def gpu_available() -> bool:
    """True if libmgh.so loads and a gfx950 device can be opened."""
    try:
        with Context(0):
            return True
    except Exception:
        return False
