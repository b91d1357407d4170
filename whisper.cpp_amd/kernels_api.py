"""ctypes binding of include/mi355x_kernels.h (the kernel library's C ABI).

Used by tests/ and bench.py to drive the HIP kernels directly with device memory owned by PyTorch-ROCm
(torch is only the allocator / stream plumbing here).  Fails loudly when the library is missing.
"""
from __future__ import annotations

import ctypes as C
from pathlib import Path

import numpy as np

from . import KERNELS_SO

F32, F16, Q4_0, Q5_0, Q8_0, Q4_K, I32, BF16 = 0, 1, 2, 6, 8, 12, 26, 30      # BF16: the paged K/V cache and its attentions only
TYPE_NAMES = {"f32": F32, "f16": F16, "q4_0": Q4_0, "q5_0": Q5_0, "q8_0": Q8_0, "q4_k": Q4_K, "i32": I32}
_BLOCK = {F32: (1, 4), F16: (1, 2), I32: (1, 4), Q4_0: (32, 18), Q5_0: (32, 22), Q8_0: (32, 34), Q4_K: (256, 144)}

# every symbol declared in include/mi355x_kernels.h (tests/test_abi.py checks header <-> library <-> this list)
SYMBOLS = [
    "mi355x_device_count", "mi355x_ctx_create", "mi355x_ctx_destroy", "mi355x_ctx_stream", "mi355x_ctx_synchronize", "mi355x_flush", "mi355x_norm_prep", "mi355x_flash_attn_ext_prep", "mi355x_gemm_f16act_prep",
    "mi355x_last_error", "mi355x_eager_count", "mi355x_prof_enable", "mi355x_prof_report",
    "mi355x_prof_reset", "mi355x_type_is_quantized", "mi355x_type_row_bytes", "mi355x_repack_to_planar",
    "mi355x_repack_from_planar", "mi355x_mul_mat", "mi355x_prep_act", "mi355x_gemm_f16act", "mi355x_dequant_f16", "mi355x_gemv_fused",
    "mi355x_flash_attn_ext", "mi355x_flash_attn_ext_exact", "mi355x_flash_attn_partial", "mi355x_flash_attn_combine", "mi355x_norm", "mi355x_binary", "mi355x_scale", "mi355x_gelu", "mi355x_cpy",
    "mi355x_last_launch_mirrored", "mi355x_act_planes_bytes", "mi355x_act_prepare", "mi355x_act_scratch", "mi355x_flash_attn_partial_multi", "mi355x_flash_attn_planes", "mi355x_decode_head_multi",
    "mi355x_argmax_top2", "mi355x_act_rows_bytes", "mi355x_gemm_q8act", "mi355x_gemm_q8act_prep", "mi355x_flash_attn_ext_prep_rows", "mi355x_unary", "mi355x_pad_reflect_1d", "mi355x_get_rows", "mi355x_get_rows_add", "mi355x_im2col_1d", "mi355x_soft_max", "mi355x_rope", "mi355x_concat", "mi355x_memset", "mi355x_checksum", "mi355x_log_mel", "mi355x_log_mel_n_len", "mi355x_debug_read_stamps", "mi355x_wake", "mi355x_test_option",
    "mi355x_kv_work_bytes", "mi355x_kv_reset", "mi355x_kv_append", "mi355x_kv_truncate", "mi355x_kv_fork", "mi355x_kv_compact",
    "mi355x_attn_paged_work_bytes", "mi355x_attn_paged", "mi355x_attn_packed",
]


class Tensor(C.Structure):
    _fields_ = [("data", C.c_void_p), ("type", C.c_int32), ("reserved", C.c_int32), ("ne", C.c_int64 * 4), ("nb", C.c_int64 * 4)]


class Epilogue(C.Structure):
    _fields_ = [("bias", C.c_void_p), ("scale", C.c_float), ("has_scale", C.c_int32), ("gelu", C.c_int32), ("bias_per_col", C.c_int32),
                ("residual", C.c_void_p), ("residual_nb1", C.c_int64)]

    def __init__(self, bias=None, scale=0.0, has_scale=0, gelu=0, residual=None, residual_nb1=0, bias_per_col=0):
        # positional order of the struct BEFORE bias_per_col took the padding slot behind `gelu` (round 3): callers that fill the
        # struct positionally keep meaning what they meant
        super().__init__()
        self.bias, self.scale, self.has_scale, self.gelu = bias or None, scale, has_scale, gelu
        self.residual, self.residual_nb1, self.bias_per_col = residual or None, residual_nb1, bias_per_col


class GemvSeg(C.Structure):
    _fields_ = [("w", C.c_void_p), ("wtype", C.c_int32), ("N", C.c_int32), ("ep", Epilogue), ("dst", C.c_void_p),
                ("dst_type", C.c_int32), ("reserved", C.c_int32), ("dst_nb1", C.c_int64)]


class GemvDesc(C.Structure):
    _fields_ = [("x", C.c_void_p), ("x_nb1", C.c_int64), ("K", C.c_int32), ("T", C.c_int32), ("has_norm", C.c_int32),
                ("eps", C.c_float), ("ln_w", C.c_void_p), ("ln_b", C.c_void_p), ("nseg", C.c_int32), ("reserved", C.c_int32),
                ("seg", GemvSeg * 3), ("attn_part_o", C.c_void_p), ("attn_part_ml", C.c_void_p), ("attn_nparts", C.c_int32),
                ("reserved2", C.c_int32), ("x_planes", C.c_void_p), ("planes_out", C.c_void_p), ("planes_out_only", C.c_int32),
                ("reserved3", C.c_int32), ("cols", C.c_void_p)]


MAX_COLS = 32          # mi355x_kernels.h: MI355X_MAX_COLS (more than IMG_COLS = 8 columns travel as images of 8)
IMG_COLS = 8


class GemvCols(C.Structure):          # mi355x_gemv_cols: [segment][column] destinations / residuals
    _fields_ = [("dst", (C.c_void_p * MAX_COLS) * 3), ("res", (C.c_void_p * MAX_COLS) * 3), ("mirror", C.c_void_p * MAX_COLS)]


class ActDesc(C.Structure):
    _fields_ = [("x", C.c_void_p), ("x_nb1", C.c_int64), ("xcol", C.c_void_p * MAX_COLS), ("K", C.c_int32), ("T", C.c_int32),
                ("wtype", C.c_int32), ("has_norm", C.c_int32), ("eps", C.c_float), ("reserved", C.c_int32), ("ln_w", C.c_void_p),
                ("ln_b", C.c_void_p), ("attn_part_o", C.c_void_p), ("attn_part_ml", C.c_void_p), ("attn_nparts", C.c_int32),
                ("reserved2", C.c_int32)]


class AttnState(C.Structure):
    _fields_ = [("q", C.c_void_p), ("k", C.c_void_p), ("v", C.c_void_p), ("mask", C.c_void_p), ("n_kv", C.c_int32), ("reserved", C.c_int32)]


class HeadState(C.Structure):
    _fields_ = [("tok", C.c_void_p), ("pos", C.c_void_p), ("dst", C.c_void_p), ("mask_f32", C.c_void_p), ("mask_f16", C.c_void_p),
                ("n_mask", C.c_int32), ("reserved", C.c_int32)]


class AttnPartials(C.Structure):
    _fields_ = [("part_o", C.c_void_p), ("part_ml", C.c_void_p), ("nparts", C.c_int32), ("T", C.c_int32), ("H", C.c_int32), ("reserved", C.c_int32)]


class RopeParams(C.Structure):
    _fields_ = [("n_dims", C.c_int32), ("mode", C.c_int32), ("n_ctx_orig", C.c_int32), ("freq_base", C.c_float),
                ("freq_scale", C.c_float), ("ext_factor", C.c_float), ("attn_factor", C.c_float), ("beta_fast", C.c_float),
                ("beta_slow", C.c_float), ("sections", C.c_int32 * 4)]


class KvCache(C.Structure):           # mi355x_kv_cache
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("type", C.c_int32), ("head_dim", C.c_int32), ("n_head_kv", C.c_int32), ("page_size", C.c_int32),
                ("n_pages", C.c_int32), ("n_seq", C.c_int32), ("max_pages", C.c_int32), ("reserved", C.c_int32), ("nb_key", C.c_int64), ("nb_head", C.c_int64),
                ("nb_page", C.c_int64), ("table", C.c_void_p), ("len", C.c_void_p), ("ref", C.c_void_p), ("status", C.c_void_p), ("work", C.c_void_p)]


KV_BAD_ARG, KV_ROW_FULL, KV_OUT_OF_PAGES = 1, 2, 4      # enum mi355x_kv_status


class AttnPagedDesc(C.Structure):
    _fields_ = [("q", Tensor), ("dst", Tensor), ("seq", C.c_void_p), ("scale", C.c_float), ("window", C.c_int32), ("max_len", C.c_int32), ("reserved", C.c_int32),
                ("work", C.c_void_p), ("work_bytes", C.c_size_t)]


class AttnPackedDesc(C.Structure):
    _fields_ = [("q", Tensor), ("k", Tensor), ("v", Tensor), ("dst", Tensor), ("cu_q", C.c_void_p), ("cu_k", C.c_void_p), ("cache", C.POINTER(KvCache)),
                ("seq", C.c_void_p), ("n", C.c_int32), ("causal", C.c_int32), ("window", C.c_int32), ("max_q", C.c_int32), ("scale", C.c_float), ("reserved", C.c_int32)]


class ProfRow(C.Structure):
    _fields_ = [("name", C.c_char_p), ("calls", C.c_uint64), ("total_ms", C.c_double), ("algo_bytes", C.c_double), ("algo_flops", C.c_double)]


_lib = None


def lib() -> C.CDLL:
    global _lib
    if _lib is None:
        if not Path(KERNELS_SO).exists():
            raise RuntimeError(f"{KERNELS_SO} is missing: run `python whisper.cpp_amd/build.py` (no CPU fallback exists)")
        L = C.CDLL(str(KERNELS_SO), mode=C.RTLD_GLOBAL)
        L.mi355x_ctx_create.restype = C.c_void_p
        L.mi355x_ctx_create.argtypes = [C.c_int]
        L.mi355x_ctx_stream.restype = C.c_void_p
        L.mi355x_last_error.restype = C.c_char_p
        L.mi355x_type_row_bytes.restype = C.c_size_t
        L.mi355x_type_row_bytes.argtypes = [C.c_int, C.c_int64]
        for name in ("mi355x_ctx_destroy", "mi355x_ctx_synchronize", "mi355x_ctx_stream", "mi355x_prof_reset", "mi355x_flush", "mi355x_eager_count", "mi355x_last_launch_mirrored"):
            getattr(L, name).argtypes = [C.c_void_p]
        L.mi355x_eager_count.restype = C.c_uint64
        L.mi355x_prof_enable.argtypes = [C.c_void_p, C.c_int]
        L.mi355x_prof_report.argtypes = [C.c_void_p, C.POINTER(ProfRow), C.c_int]
        L.mi355x_repack_to_planar.argtypes = [C.c_int, C.c_void_p, C.c_void_p, C.c_int64]
        L.mi355x_repack_from_planar.argtypes = [C.c_int, C.c_void_p, C.c_void_p, C.c_int64]
        TP = C.POINTER(Tensor)
        L.mi355x_mul_mat.argtypes = [C.c_void_p, TP, TP, TP, C.POINTER(Epilogue)]
        L.mi355x_prep_act.argtypes = [C.c_void_p, C.c_void_p, C.c_int64, C.c_int, C.c_void_p, C.c_int, C.c_int64, C.c_int]
        L.mi355x_gemm_f16act.argtypes = [C.c_void_p, TP, C.c_void_p, C.c_int64, C.c_int64, C.c_void_p, C.c_int64, C.c_int, C.POINTER(Epilogue)]
        L.mi355x_gemm_f16act_prep.argtypes = [C.c_void_p, TP, C.c_void_p, C.c_int64, C.c_int64, C.c_void_p, C.c_int64, C.POINTER(Epilogue), C.c_void_p]
        L.mi355x_dequant_f16.argtypes = [C.c_void_p, TP, C.c_void_p]
        L.mi355x_act_rows_bytes.restype = C.c_size_t
        L.mi355x_act_rows_bytes.argtypes = [C.c_int, C.c_int64, C.c_int64]
        L.mi355x_gemm_q8act.argtypes = [C.c_void_p, TP, C.c_void_p, C.c_int64, C.c_void_p, C.c_int64, C.c_int, C.POINTER(Epilogue)]
        L.mi355x_gemm_q8act_prep.argtypes = [C.c_void_p, TP, C.c_void_p, C.c_int64, C.c_void_p, C.c_int64, C.POINTER(Epilogue), C.c_void_p]
        L.mi355x_flash_attn_ext_prep_rows.argtypes = [C.c_void_p, TP, TP, TP, TP, TP, C.c_float, C.c_void_p]
        L.mi355x_gemv_fused.argtypes = [C.c_void_p, C.POINTER(GemvDesc)]
        L.mi355x_flash_attn_ext.argtypes = [C.c_void_p, TP, TP, TP, TP, TP, C.c_float]
        L.mi355x_flash_attn_ext_prep.argtypes = [C.c_void_p, TP, TP, TP, TP, TP, C.c_float, C.c_void_p]
        L.mi355x_flash_attn_ext_exact.argtypes = [C.c_void_p, TP, TP, TP, TP, TP, C.c_float, C.c_int]
        L.mi355x_flash_attn_partial.argtypes = [C.c_void_p, TP, TP, TP, TP, C.c_float, C.POINTER(AttnPartials)]
        L.mi355x_flash_attn_combine.argtypes = [C.c_void_p, C.POINTER(AttnPartials), TP]
        L.mi355x_act_planes_bytes.restype = C.c_size_t
        L.mi355x_act_planes_bytes.argtypes = [C.c_int, C.c_int, C.c_int]
        L.mi355x_act_prepare.argtypes = [C.c_void_p, C.POINTER(ActDesc), C.c_void_p]
        L.mi355x_act_scratch.restype = C.c_void_p
        L.mi355x_act_scratch.argtypes = [C.c_void_p, C.c_int]
        L.mi355x_flash_attn_partial_multi.argtypes = [C.c_void_p, C.c_int, C.POINTER(AttnState), TP, TP, TP, C.c_float, C.POINTER(AttnPartials)]
        L.mi355x_flash_attn_planes.argtypes = [C.c_void_p, C.c_int, C.POINTER(AttnState), TP, TP, TP, C.c_float, C.c_void_p]
        L.mi355x_decode_head_multi.argtypes = [C.c_void_p, C.c_int, C.POINTER(HeadState), TP, TP]
        L.mi355x_norm.argtypes = [C.c_void_p, TP, TP, C.c_float, C.c_void_p, C.c_void_p]
        L.mi355x_norm_prep.argtypes = [C.c_void_p, TP, TP, C.c_float, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int]
        L.mi355x_binary.argtypes = [C.c_void_p, C.c_int, TP, TP, TP]
        L.mi355x_scale.argtypes = [C.c_void_p, TP, TP, C.c_float, C.c_float]
        L.mi355x_gelu.argtypes = [C.c_void_p, TP, TP]
        L.mi355x_argmax_top2.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p]
        L.mi355x_unary.argtypes = [C.c_void_p, C.c_int, TP, TP]
        L.mi355x_pad_reflect_1d.argtypes = [C.c_void_p, TP, TP, C.c_int, C.c_int]
        L.mi355x_cpy.argtypes = [C.c_void_p, TP, TP]
        L.mi355x_get_rows.argtypes = [C.c_void_p, TP, TP, TP]
        L.mi355x_get_rows_add.argtypes = [C.c_void_p, TP, TP, TP, TP, TP]
        L.mi355x_im2col_1d.argtypes = [C.c_void_p, TP, TP, C.c_int, C.c_int, C.c_int, C.c_int]
        L.mi355x_soft_max.argtypes = [C.c_void_p, TP, TP, TP, C.c_float, C.c_float]
        L.mi355x_rope.argtypes = [C.c_void_p, TP, TP, C.c_void_p, TP, C.POINTER(RopeParams)]
        L.mi355x_concat.argtypes = [C.c_void_p, TP, TP, TP, C.c_int]
        L.mi355x_checksum.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t, C.c_void_p]
        L.mi355x_log_mel_n_len.argtypes = [C.c_int]
        L.mi355x_log_mel.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_int, C.c_int, C.c_void_p, C.c_int]
        CP = C.POINTER(KvCache)
        L.mi355x_kv_work_bytes.restype = C.c_size_t
        L.mi355x_kv_work_bytes.argtypes = [C.c_int, C.c_int]
        L.mi355x_kv_reset.argtypes = [C.c_void_p, CP]
        L.mi355x_kv_append.argtypes = [C.c_void_p, CP, C.c_int, C.c_void_p, C.c_void_p, TP, TP]
        L.mi355x_kv_truncate.argtypes = [C.c_void_p, CP, C.c_int, C.c_void_p, C.c_void_p]
        L.mi355x_kv_fork.argtypes = [C.c_void_p, CP, C.c_int, C.c_void_p, C.c_void_p]
        L.mi355x_kv_compact.argtypes = [C.c_void_p, CP, CP]
        L.mi355x_attn_paged_work_bytes.restype = C.c_size_t
        L.mi355x_attn_paged_work_bytes.argtypes = [CP, C.c_int, C.c_int, C.c_int]
        L.mi355x_attn_paged.argtypes = [C.c_void_p, CP, C.POINTER(AttnPagedDesc)]
        L.mi355x_attn_packed.argtypes = [C.c_void_p, C.POINTER(AttnPackedDesc)]
        L.mi355x_memset.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_size_t]
        L.mi355x_debug_read_stamps.argtypes = [C.c_void_p, C.POINTER(C.c_uint64)]
        _lib = L
    return _lib


def row_bytes(t: int, ne0: int) -> int:
    blk, sz = _BLOCK[t]
    assert ne0 % blk == 0
    return ne0 // blk * sz


def tensor(ptr: int, t: int, ne, nb=None) -> Tensor:
    """Describe a device tensor.  ne: up to 4 dims (ggml order, fastest first); nb: byte strides (default contiguous)."""
    ne = list(ne) + [1] * (4 - len(ne))
    if nb is None:
        nb = [_BLOCK[t][1], row_bytes(t, ne[0])]
        nb.append(nb[1] * ne[1])
        nb.append(nb[2] * ne[2])
    nb = list(nb) + [0] * (4 - len(nb))
    m = Tensor()
    m.data, m.type = ptr, t
    for i in range(4):
        m.ne[i], m.nb[i] = ne[i], nb[i]
    return m


def repack_to_planar(t: int, blocks: np.ndarray, nelements: int) -> np.ndarray:
    src = np.ascontiguousarray(blocks).view(np.uint8).ravel()
    dst = np.empty_like(src)
    rc = lib().mi355x_repack_to_planar(t, src.ctypes.data, dst.ctypes.data, nelements)
    if rc != 0:
        raise RuntimeError(f"repack_to_planar failed: {rc}")
    return dst


def repack_from_planar(t: int, planar: np.ndarray, nelements: int) -> np.ndarray:
    src = np.ascontiguousarray(planar).view(np.uint8).ravel()
    dst = np.empty_like(src)
    rc = lib().mi355x_repack_from_planar(t, src.ctypes.data, dst.ctypes.data, nelements)
    if rc != 0:
        raise RuntimeError(f"repack_from_planar failed: {rc}")
    return dst


# ---- the paged K/V cache and its attentions, on device arrays (torch tensors or anything with data_ptr / shape / stride / dtype) ----
_DTYPE = {"torch.float32": F32, "torch.float16": F16, "torch.bfloat16": BF16}


def _rows(t) -> Tensor:
    """[rows, heads, dim] as the C side's [dim, heads, rows]"""
    if t.dim() != 3 or str(t.dtype) not in _DTYPE:
        raise ValueError(f"expected [rows, heads, dim] of float32, float16 or bfloat16, got {list(t.shape)} {t.dtype}")
    b = t.element_size()
    return tensor(t.data_ptr(), _DTYPE[str(t.dtype)], [t.shape[2], t.shape[1], t.shape[0]], [t.stride(2) * b, t.stride(1) * b, t.stride(0) * b])


def _ints(t, n: int, what: str):
    """the address of at least n contiguous 32-bit integers"""
    if t is None:
        return None
    if str(t.dtype) != "torch.int32" or not t.is_contiguous() or t.numel() < n:
        raise ValueError(f"{what}: {n} contiguous int32 values wanted, got {list(t.shape)} {t.dtype}")
    return t.data_ptr()


def _device(t):
    """of an array, as (type, number); None where it does not say"""
    d = getattr(t, "device", None)
    return None if d is None else (d.type, d.index)


def kv_work_bytes(n_seq: int, n_pages: int) -> int:
    return lib().mi355x_kv_work_bytes(n_seq, n_pages)


def kv_cache(k, v, table, length, ref, status, work) -> KvCache:
    """Describe a paged cache: pools k, v [page, head, key, dim] (any order of heads and keys in memory), table [sequence, page], length [sequence],
    ref [page], status [1] int32, work: kv_work_bytes() bytes.  The description holds on to the arrays."""
    if k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype or k.dim() != 4 or str(k.dtype) not in _DTYPE or k.stride(3) != 1:
        raise ValueError("k and v: [page, head, key, dim] of one shape, type and layout, dims contiguous")
    if table.dim() != 2:
        raise ValueError("table: [sequence, page]")
    if len({_device(t) for t in (k, v, table, length, ref, status, work)}) > 1:
        raise ValueError("the arrays of a cache lie on one device")
    b, need = k.element_size(), kv_work_bytes(table.shape[0], k.shape[0])
    if work.numel() * work.element_size() < need or not work.is_contiguous():
        raise ValueError(f"work: {need} bytes wanted")
    c = KvCache()
    c.k, c.v, c.type, c.head_dim, c.n_head_kv, c.page_size = k.data_ptr(), v.data_ptr(), _DTYPE[str(k.dtype)], k.shape[3], k.shape[1], k.shape[2]
    c.n_pages, c.n_seq, c.max_pages = k.shape[0], table.shape[0], table.shape[1]
    c.nb_key, c.nb_head, c.nb_page = k.stride(2) * b, k.stride(1) * b, k.stride(0) * b
    c.table, c.len, c.ref = _ints(table, 0, "table"), _ints(length, c.n_seq, "length"), _ints(ref, c.n_pages, "ref")
    c.status, c.work = _ints(status, 1, "status"), work.data_ptr()
    c.device, c.arrays = _device(k), (k, v, table, length, ref, status, work)
    return c


def attn_paged_work_bytes(cache: KvCache, n: int, n_head: int, max_len: int = 0) -> int:
    """for a call of exactly this shape; an area for several shapes is as large as the largest of their answers (fewer queries can need more)"""
    return lib().mi355x_attn_paged_work_bytes(C.byref(cache), n, n_head, max_len)


class Call:
    """A call of the C ABI with its arguments made once: a decode loop repeats it with new contents of the same arrays."""

    def __init__(self, ctx, name: str, *args, keep=()):
        self.ctx, self.name, self.fn, self.args, self.keep = ctx, name, getattr(lib(), name), (ctx.h, *args), (args, keep)

    def __call__(self):
        if not self.ctx.h:
            raise RuntimeError(f"{self.name}: the context is closed")
        rc = self.fn(*self.args)
        if rc:
            self.ctx.check(rc, self.name)


class Ctx:
    """One kernel context (HIP stream + scratch).  Raises if no gfx950 device is usable."""

    def __init__(self, device: int = 0):
        self.h = lib().mi355x_ctx_create(device)
        if not self.h:
            raise RuntimeError("mi355x_ctx_create failed: " + (lib().mi355x_last_error() or b"").decode())
        self.device = device

    def sync(self):
        rc = lib().mi355x_ctx_synchronize(self.h)
        if rc:
            raise RuntimeError(f"sync failed rc={rc}: {lib().mi355x_last_error().decode()}")

    @property
    def stream(self) -> int:
        """The stream (hipStream_t) that every call is launched on.  It waits for no other, torch's among them: work on the same arrays belongs on it too
        (torch.cuda.stream(torch.cuda.ExternalStream(ctx.stream))), or events between the two."""
        if not self.h:
            raise RuntimeError("the context is closed")
        return lib().mi355x_ctx_stream(self.h)

    def check(self, rc: int, what: str = "op"):
        if rc != 0:
            raise RuntimeError(f"{what} failed rc={rc}: {(lib().mi355x_last_error() or b'').decode()}")

    def close(self):
        if self.h:
            lib().mi355x_ctx_destroy(self.h)
            self.h = None

    # ---- the paged cache: each returns a Call (arrays as in kv_cache(); lists int32 on the device), made on this context's `stream` ----
    def _here(self, *arrays):
        """Kernels read what they are given as memory of the context's device: host arrays and those of another one are refused."""
        for t in arrays:
            d = None if t is None else t.__dict__.get("device") if isinstance(t, KvCache) else _device(t)
            if d is not None and d != ("cuda", self.device):
                raise ValueError(f"an array on {d[0]}{'' if d[1] is None else f':{d[1]}'}, where one on the context's device, {self.device}, is wanted")

    def kv_reset_call(self, cache: KvCache) -> Call:
        self._here(cache)
        return Call(self, "mi355x_kv_reset", C.byref(cache), keep=cache)

    def kv_append_call(self, cache: KvCache, seq, cu, k, v) -> Call:
        self._here(cache, seq, cu, k, v)
        n, tk, tv = seq.numel(), _rows(k), _rows(v)
        return Call(self, "mi355x_kv_append", C.byref(cache), n, _ints(seq, n, "seq"), _ints(cu, n + 1, "cu"), C.byref(tk), C.byref(tv), keep=(cache, seq, cu, k, v))

    def kv_truncate_call(self, cache: KvCache, seq, keep) -> Call:
        self._here(cache, seq, keep)
        n = seq.numel()
        return Call(self, "mi355x_kv_truncate", C.byref(cache), n, _ints(seq, n, "seq"), _ints(keep, n, "keep"), keep=(cache, seq, keep))

    def kv_fork_call(self, cache: KvCache, src, dst) -> Call:
        self._here(cache, src, dst)
        n = src.numel()
        return Call(self, "mi355x_kv_fork", C.byref(cache), n, _ints(src, n, "src"), _ints(dst, n, "dst"), keep=(cache, src, dst))

    def kv_compact_call(self, cache: KvCache, to: KvCache) -> Call:
        self._here(cache, to)
        return Call(self, "mi355x_kv_compact", C.byref(cache), C.byref(to), keep=(cache, to))

    def attn_paged_call(self, cache: KvCache, q, out, seq=None, scale: float = 1.0, window: int = 0, max_len: int = 0, work=None) -> Call:
        self._here(cache, q, out, seq, work)
        d = AttnPagedDesc()
        d.q, d.dst, d.seq, d.scale, d.window, d.max_len = _rows(q), _rows(out), _ints(seq, q.shape[0], "seq"), scale, window, max_len
        d.work, d.work_bytes = (work.data_ptr() or None, work.numel() * work.element_size()) if work is not None else (None, 0)
        return Call(self, "mi355x_attn_paged", C.byref(cache), C.byref(d), keep=(cache, d, q, out, seq, work))

    def attn_packed_call(self, q, out, cu_q, k=None, v=None, cu_k=None, cache=None, seq=None, scale: float = 1.0, causal: bool = True, window: int = 0, max_q: int = 0) -> Call:
        self._here(q, out, cu_q, k, v, cu_k, cache, seq)
        d, n = AttnPackedDesc(), cu_q.numel() - 1
        d.q, d.dst, d.cu_q, d.n = _rows(q), _rows(out), _ints(cu_q, 1, "cu_q"), n
        if cache is not None:
            d.cache, d.seq = C.pointer(cache), _ints(seq, n, "seq")
        else:
            d.k, d.v, d.cu_k = _rows(k), _rows(v), _ints(cu_k, n + 1, "cu_k")
        d.scale, d.causal, d.window, d.max_q = scale, causal, window, max_q
        return Call(self, "mi355x_attn_packed", C.byref(d), keep=(cache, d, q, out, cu_q, k, v, cu_k, seq))

    def prof(self, on: bool):
        lib().mi355x_prof_enable(self.h, 1 if on else 0)

    def prof_reset(self):
        lib().mi355x_prof_reset(self.h)

    def prof_report(self):
        rows = (ProfRow * 64)()
        n = lib().mi355x_prof_report(self.h, rows, 64)
        return [dict(name=rows[i].name.decode(), calls=rows[i].calls, total_ms=rows[i].total_ms,
                     algo_bytes=rows[i].algo_bytes, algo_flops=rows[i].algo_flops) for i in range(n)]
