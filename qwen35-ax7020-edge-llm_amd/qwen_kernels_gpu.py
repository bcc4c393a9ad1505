"""Python side of the MI355X BFP8 GEMV library.

Mirrors how the reference engine binds its operator library
(04/qwen_real_engine.py:656-725 loads libqwen_kernels.so with ctypes, calls
init_kernels() and declares argtypes; :848-866 rebinds the fast-path symbols;
:1221-1240 ``gemv_bfp8`` calls ``bfp8_gemv(y, x, mant, exps, M, K)`` on numpy
views of the weight mmap).  ``bind`` declares exactly those argtypes, so an
engine that loads this library gets the same ctypes behaviour.

On top of that, device-resident helpers (PyTorch tensors as plain device
memory, torch's current stream as the HIP stream) expose the ``bfp8_dev_*``
and ``bfp8_plan_*`` entry points used by the tests and the benchmark.

There is no CPU fallback: every entry point runs on the GPU, and a missing
library raises.
"""
from __future__ import annotations

import contextlib
import ctypes
import math
import struct
from ctypes import POINTER, c_double, c_float, c_int, c_int64, c_size_t, c_uint64, c_void_p
from pathlib import Path
from typing import Optional, Sequence

import numpy as np

LIB_PATH = Path(__file__).resolve().parent / "libqwen_kernels.so"

BFP8_OK, BFP8_EINVAL, BFP8_EHIP, BFP8_ENOMEM = 0, -1, -2, -3

# Reference symbols whose signatures the engine binds (04/qwen_real_engine.py).
REFERENCE_SYMBOLS = ("add_residual", "bfp8_gemv", "causal_conv1d_update_silu", "forward_linear_layer",
                     "forward_mlp", "forward_token_c", "gdn_gates", "gdn_recurrent_step", "init_kernels",
                     "lm_head_argmax", "qk_l2norm", "qwen_prof_count", "qwen_prof_enable", "qwen_prof_get",
                     "qwen_prof_name", "qwen_prof_reset", "rmsnorm", "rmsnorm_gated", "swiglu")


class bfp8_plan_item(ctypes.Structure):
    """Mirror of ``bfp8_plan_item`` (include/qwen_kernels.h)."""

    _fields_ = [
        ("x", c_void_p), ("y", c_void_p), ("mant_gpu", c_void_p), ("exps_gpu", c_void_p),
        ("M", c_int), ("K", c_int), ("topk", c_int),
        ("out_ids", c_void_p), ("out_scores", c_void_p), ("out_count", c_void_p),
        ("out_argmax", c_void_p),
    ]


# void (*)(int layer, float* h, void* ctx), 04/qwen_real_engine.py:979
FULL_ATTN_CALLBACK = ctypes.CFUNCTYPE(None, c_int, c_void_p, c_void_p)


class LinearLayerPlan(ctypes.Structure):
    """Mirror of ``LinearLayerPlan`` (include/qwen_kernels.h), field for field
    the engine's ``LinearLayerPlanC`` (04/qwen_real_engine.py:20-56)."""

    _fields_ = [
        ("in_ln_w", c_void_p), ("mant_qkv", c_void_p), ("exp_qkv", c_void_p), ("M_qkv", c_int), ("K_qkv", c_int),
        ("conv_w", c_void_p), ("conv_s", c_void_p), ("wa", c_void_p), ("wb", c_void_p), ("nea", c_void_p),
        ("dt", c_void_p), ("state", c_void_p), ("mant_z", c_void_p), ("exp_z", c_void_p), ("M_z", c_int),
        ("K_z", c_int), ("norm_w", c_void_p), ("mant_o", c_void_p), ("exp_o", c_void_p), ("M_o", c_int),
        ("K_o", c_int), ("post_ln_w", c_void_p), ("mant_gate", c_void_p), ("exp_gate", c_void_p),
        ("M_gate", c_int), ("K_gate", c_int), ("mant_up", c_void_p), ("exp_up", c_void_p), ("M_up", c_int),
        ("K_up", c_int), ("mant_down", c_void_p), ("exp_down", c_void_p), ("M_down", c_int), ("K_down", c_int),
    ]


class MlpPlan(ctypes.Structure):
    """Mirror of ``MlpPlan`` (include/qwen_kernels.h; the engine's ``MlpPlanC``)."""

    _fields_ = [
        ("post_ln_w", c_void_p), ("mant_gate", c_void_p), ("exp_gate", c_void_p), ("M_gate", c_int),
        ("K_gate", c_int), ("mant_up", c_void_p), ("exp_up", c_void_p), ("M_up", c_int), ("K_up", c_int),
        ("mant_down", c_void_p), ("exp_down", c_void_p), ("M_down", c_int), ("K_down", c_int),
    ]


QWEN_F32, QWEN_BF16 = 0, 1


class gdn_dev_args(ctypes.Structure):
    """Mirror of ``gdn_dev_args`` (include/qwen_kernels.h)."""

    _fields_ = [
        ("out", c_void_p), ("q", c_void_p), ("k", c_void_p), ("v", c_void_p), ("alpha", c_void_p),
        ("beta", c_void_p), ("state_in", c_void_p), ("state_out", c_void_p), ("slots", c_void_p),
        ("starts", c_void_p), ("work", c_void_p), ("work_bytes", c_size_t),
        ("q_row", c_int64), ("k_row", c_int64), ("v_row", c_int64), ("out_row", c_int64), ("gate_row", c_int64),
        ("rows", c_int), ("n_seq", c_int), ("n_slots", c_int), ("heads_k", c_int), ("heads_v", c_int),
        ("dim_k", c_int), ("dim_v", c_int), ("dtype", c_int), ("scale", c_float), ("zero_rest", c_int),
    ]


# gdn_dev_args in one packing: its 27 fields set one by one take longer than a short kernel
_GDN_PACK = struct.Struct("@11PN5q8ifi")


class lm_head_loss_args(ctypes.Structure):
    """Mirror of ``lm_head_loss_args`` (include/qwen_kernels.h)."""

    _fields_ = [
        ("loss", c_void_p), ("lse", c_void_p), ("grad_h", c_void_p), ("grad_table", c_void_p), ("h", c_void_p),
        ("table", c_void_p), ("targets", c_void_p), ("grad_loss", c_void_p), ("work", c_void_p),
        ("work_bytes", c_size_t), ("h_row", c_int64), ("table_row", c_int64), ("grad_h_row", c_int64),
        ("grad_table_row", c_int64), ("rows", c_int), ("vocab", c_int), ("hidden", c_int), ("dtype", c_int),
    ]


class rope_dev_args(ctypes.Structure):
    """Mirror of ``rope_dev_args`` (include/qwen_kernels.h)."""

    _fields_ = [
        ("out", c_void_p), ("x", c_void_p), ("positions", c_void_p), ("freqs", c_void_p),
        ("out_row", c_int64), ("out_head", c_int64), ("x_row", c_int64), ("x_head", c_int64),
        ("rows", c_int), ("heads", c_int), ("dim", c_int), ("rot", c_int), ("dtype", c_int), ("interleaved", c_int),
        ("amplitude", c_float),
    ]


class kv_dev_append_args(ctypes.Structure):
    """Mirror of ``kv_dev_append_args`` (include/qwen_kernels.h)."""

    _fields_ = [
        ("key_cache", c_void_p), ("value_cache", c_void_p), ("q_out", c_void_p), ("k", c_void_p), ("v", c_void_p),
        ("q", c_void_p), ("tables", c_void_p), ("cached", c_void_p), ("starts", c_void_p), ("positions", c_void_p),
        ("freqs", c_void_p),
        ("cache_page", c_int64), ("cache_token", c_int64), ("cache_head", c_int64), ("table_row", c_int64),
        ("k_row", c_int64), ("k_head", c_int64), ("v_row", c_int64), ("v_head", c_int64), ("q_row", c_int64),
        ("q_head", c_int64), ("q_out_row", c_int64), ("q_out_head", c_int64),
        ("rows", c_int), ("n_seq", c_int), ("pages", c_int), ("page", c_int), ("table_pages", c_int),
        ("heads_q", c_int), ("heads_k", c_int), ("dim", c_int), ("rot", c_int), ("dtype", c_int), ("interleaved", c_int),
        ("amplitude", c_float),
    ]


class attn_dev_args(ctypes.Structure):
    """Mirror of ``attn_dev_args`` (include/qwen_kernels.h)."""

    _fields_ = [
        ("out", c_void_p), ("q", c_void_p), ("key_cache", c_void_p), ("value_cache", c_void_p), ("tables", c_void_p),
        ("cached", c_void_p), ("starts", c_void_p), ("mask", c_void_p), ("work", c_void_p), ("work_bytes", c_size_t),
        ("cache_page", c_int64), ("cache_token", c_int64), ("cache_head", c_int64), ("table_row", c_int64),
        ("q_row", c_int64), ("q_head", c_int64), ("out_row", c_int64), ("out_head", c_int64),
        ("rows", c_int), ("n_seq", c_int), ("pages", c_int), ("page", c_int), ("table_pages", c_int),
        ("heads_q", c_int), ("heads_k", c_int), ("dim", c_int), ("mask_words", c_int), ("dtype", c_int),
        ("scale", c_float), ("zero_rest", c_int),
    ]


class attn_dev_tree_args(ctypes.Structure):
    """Mirror of ``attn_dev_tree_args`` (include/qwen_kernels.h)."""

    _fields_ = [
        ("mask", c_void_p), ("positions", c_void_p), ("parents", c_void_p), ("cached", c_void_p), ("starts", c_void_p),
        ("rows", c_int), ("n_seq", c_int), ("words", c_int),
    ]


# these in one packing, as _GDN_PACK
_ROPE_PACK = struct.Struct("@4P4q6if4x")
_APPEND_PACK = struct.Struct("@11P12q11if")
_ATTN_PACK = struct.Struct("@9PN8q10ifi")
_TREE_PACK = struct.Struct("@5P3i4x")


def bind(lib: ctypes.CDLL) -> ctypes.CDLL:
    """Declare argtypes/restypes of every exported symbol."""
    vp, i = c_void_p, c_int
    # reference symbols, as the engine declares them (04/qwen_real_engine.py:680-685, :864-866)
    lib.init_kernels.argtypes = []
    lib.init_kernels.restype = None
    lib.bfp8_gemv.argtypes = [vp, vp, vp, vp, i, i]
    lib.bfp8_gemv.restype = None
    lib.qwen_prof_enable.argtypes = [i]
    lib.qwen_prof_enable.restype = None
    lib.qwen_prof_reset.argtypes = []
    lib.qwen_prof_reset.restype = None
    lib.qwen_prof_count.argtypes = []
    lib.qwen_prof_count.restype = i
    lib.qwen_prof_get.argtypes = [i]
    lib.qwen_prof_get.restype = c_double
    lib.qwen_prof_name.argtypes = [i]
    lib.qwen_prof_name.restype = ctypes.c_char_p
    # new host-pointer symbols
    lib.bfp8_lm_head_topk.argtypes = [vp, vp, vp, i, i, i, vp, vp]
    lib.bfp8_lm_head_topk.restype = i
    lib.bfp8_lm_head_argmax.argtypes = [vp, vp, vp, i, i]
    lib.bfp8_lm_head_argmax.restype = i
    lib.bfp8_gemv_batch.argtypes = [vp, vp, vp, vp, i, i, i]
    lib.bfp8_gemv_batch.restype = None
    lib.bfp8_gemv_fallback.argtypes = [vp, vp, vp, vp, i, i, i]
    lib.bfp8_gemv_fallback.restype = i
    lib.bfp8_dev_gemv_fallback.argtypes = [vp, vp, vp, vp, i, i, i, vp]
    lib.bfp8_dev_gemv_fallback.restype = i
    # the bf16 tied-embedding lm_head (04/qwen_real_engine.py:691-696) and sampler
    lib.lm_head_argmax.argtypes = [vp, vp, i, i]
    lib.lm_head_argmax.restype = i
    lib.qwen_lm_head_topk_bf16.argtypes = [vp, vp, i, i, i, vp, vp]
    lib.qwen_lm_head_topk_bf16.restype = i
    lib.qwen_sample_from_topk.argtypes = [vp, vp, i, c_float, i, c_float, vp]
    lib.qwen_sample_from_topk.restype = i
    # the decode runtime and forward loop, as the engine binds them
    # (04/qwen_real_engine.py:676-725, :852-880, :978-985)
    f = c_float
    lib.rmsnorm.argtypes = [vp, vp, vp, i, f]
    lib.swiglu.argtypes = [vp, vp, vp, i]
    lib.add_residual.argtypes = [vp, vp, i]
    lib.causal_conv1d_update_silu.argtypes = [vp, vp, vp, vp, i]
    lib.qk_l2norm.argtypes = [vp, vp, i, i]
    lib.gdn_gates.argtypes = [vp, vp, vp, vp, vp, vp, vp, i, i]
    lib.gdn_recurrent_step.argtypes = [vp, vp, vp, vp, vp, vp, vp, i, i]
    lib.rmsnorm_gated.argtypes = [vp, vp, vp, vp, i, i, f]
    lib.forward_linear_layer.argtypes = [vp, vp]
    lib.forward_mlp.argtypes = [vp, vp]
    for name in ("rmsnorm", "swiglu", "add_residual", "causal_conv1d_update_silu", "qk_l2norm", "gdn_gates",
                 "gdn_recurrent_step", "rmsnorm_gated", "forward_linear_layer", "forward_mlp"):
        getattr(lib, name).restype = None
    lib.forward_token_c.argtypes = [i, vp, vp, vp, vp, vp, vp, FULL_ATTN_CALLBACK, vp]
    lib.forward_token_c.restype = i
    lib.qwen_forward_state_resident.argtypes = [i]
    lib.qwen_forward_state_resident.restype = i
    lib.qwen_forward_reset_state.argtypes = []
    lib.qwen_forward_reset_state.restype = None
    lib.qwen_forward_sync_state.argtypes = []
    lib.qwen_forward_sync_state.restype = None
    # the weight-image loader
    lib.qwen_weights_scan.argtypes = [ctypes.c_char_p, c_size_t, vp, vp, vp, vp]
    lib.qwen_weights_scan.restype = i
    lib.qwen_weights_preload.argtypes = [vp, c_size_t, ctypes.c_char_p]
    lib.qwen_weights_preload.restype = i
    lib.qwen_weights_find.argtypes = [ctypes.c_char_p, vp, vp, vp, vp]
    lib.qwen_weights_find.restype = i
    lib.bfp8_dev_pack_rows.argtypes = [vp, vp, vp, i, i, vp]
    lib.bfp8_dev_pack_rows.restype = i
    lib.bfp8_last_error.argtypes = []
    lib.bfp8_last_error.restype = ctypes.c_char_p
    lib.bfp8_gpu_ready.argtypes = []
    lib.bfp8_gpu_ready.restype = ctypes.c_int
    lib.bfp8_cache_clear.argtypes = []
    lib.bfp8_cache_clear.restype = None
    lib.bfp8_device_bytes.argtypes = []
    lib.bfp8_device_bytes.restype = ctypes.c_size_t
    lib.bfp8_debug_device_limit.argtypes = [ctypes.c_size_t]
    lib.bfp8_debug_device_limit.restype = None
    lib.qwen_debug_chain_wait.argtypes = [ctypes.c_longlong]
    lib.qwen_debug_chain_wait.restype = None
    lib.qwen_debug_chain_rest.argtypes = [i]
    lib.qwen_debug_chain_rest.restype = i
    lib.qwen_debug_chain_runs.argtypes = [ctypes.POINTER(ctypes.c_longlong)] * 2
    lib.qwen_debug_chain_runs.restype = None
    # device level
    for name in ("bfp8_dev_mant_bytes", "bfp8_dev_exps_bytes"):
        getattr(lib, name).argtypes = [i, i]
        getattr(lib, name).restype = c_size_t
    lib.bfp8_dev_xsplit_bytes.argtypes = [i]
    lib.bfp8_dev_xsplit_bytes.restype = c_size_t
    lib.bfp8_dev_pack.argtypes = [vp, vp, vp, vp, i, i, vp]
    lib.bfp8_dev_unpack.argtypes = [vp, vp, vp, vp, i, i, vp]
    lib.bfp8_dev_quantize.argtypes = [vp, vp, vp, vp, i, vp]
    lib.bfp8_dev_gemv.argtypes = [vp, vp, vp, vp, vp, i, i, vp, vp]
    lib.bfp8_dev_gemv_float.argtypes = [vp, vp, vp, vp, i, i, vp]
    lib.bfp8_dev_gemv_batch.argtypes = [vp, vp, vp, vp, vp, i, i, i, vp]
    lib.bfp8_dev_gemv_batch_kernel_name.argtypes = [i, i, i]
    lib.bfp8_dev_gemv_batch_kernel_name.restype = ctypes.c_char_p
    lib.bfp8_dev_lm_head_topk.argtypes = [vp, vp, vp, vp, vp, vp, vp, vp, i, i, i, vp]
    lib.bfp8_dev_lm_head_topk_noalloc.argtypes = [vp, vp, vp, vp, vp, vp, vp, vp, i, i, i, vp]
    lib.bfp8_dev_synth_planes.argtypes = [vp, vp, i, i, c_uint64, i, i, vp]
    lib.bfp8_dev_read_probe.argtypes = [vp, c_size_t, vp, vp]
    lib.bfp8_dev_copy_probe.argtypes = [vp, vp, c_size_t, vp]
    lib.bf16_dev_lm_head.argtypes = [vp, vp, vp, vp, vp, vp, vp, i, i, i, i, vp]
    lib.bf16_dev_tiles_bytes.argtypes = [i, i]
    lib.bf16_dev_tiles_bytes.restype = c_size_t
    lib.bf16_dev_tile_table.argtypes = [vp, vp, i, i, vp]
    lib.bf16_dev_lm_head_tiles.argtypes = [vp, vp, vp, vp, vp, vp, vp, i, i, i, vp]
    lib.bfp8_dev_sample_from_topk.argtypes = [vp, vp, vp, vp, i, c_float, i, c_float, vp, vp, vp]
    for name in ("bf16_dev_lm_head", "bf16_dev_tile_table", "bf16_dev_lm_head_tiles", "bfp8_dev_sample_from_topk", "bfp8_dev_pack", "bfp8_dev_unpack", "bfp8_dev_quantize", "bfp8_dev_gemv",
                 "bfp8_dev_gemv_float", "bfp8_dev_gemv_batch", "bfp8_dev_lm_head_topk", "bfp8_dev_lm_head_topk_noalloc",
                 "bfp8_dev_synth_planes", "bfp8_dev_read_probe", "bfp8_dev_copy_probe"):
        getattr(lib, name).restype = i
    lib.bfp8_plan_create.argtypes = [POINTER(bfp8_plan_item), i]
    lib.bfp8_plan_create.restype = vp
    for name in ("bfp8_plan_run", "bfp8_plan_run_gemv", "bfp8_plan_quantize"):
        getattr(lib, name).argtypes = [vp, vp]
        getattr(lib, name).restype = i
    lib.bfp8_plan_launch.argtypes = [vp, i, vp]
    lib.bfp8_plan_launch.restype = i
    lib.bfp8_plan_kernel_name.argtypes = [vp, i]
    lib.bfp8_plan_kernel_name.restype = ctypes.c_char_p
    lib.bfp8_plan_destroy.argtypes = [vp]
    lib.bfp8_plan_destroy.restype = None
    lib.bfp8_synth_planes_host.argtypes = [vp, vp, i, i, c_uint64, i, i]
    lib.bfp8_synth_planes_host.restype = None
    lib.bfp8_synth_normal.argtypes = [vp, i, c_uint64]
    lib.bfp8_synth_normal.restype = None
    lib.bfp8_synth_swiglu.argtypes = [vp, i, c_uint64, c_double, c_float]
    lib.bfp8_synth_swiglu.restype = None
    lib.gdn_dev_prompt_work_bytes.argtypes = [POINTER(gdn_dev_args)]
    lib.gdn_dev_prompt_work_bytes.restype = c_size_t
    for name in ("gdn_dev_prompt", "gdn_dev_step"):
        getattr(lib, name).argtypes = [POINTER(gdn_dev_args), vp]
        getattr(lib, name).restype = i
    for name in ("bf16_dev_lm_head_loss", "bf16_dev_lm_head_loss_grad"):
        getattr(lib, name + "_work_bytes").argtypes = [POINTER(lm_head_loss_args)]
        getattr(lib, name + "_work_bytes").restype = c_size_t
        getattr(lib, name).argtypes = [POINTER(lm_head_loss_args), vp]
        getattr(lib, name).restype = i
    lib.attn_dev_paged_work_bytes.argtypes = [POINTER(attn_dev_args)]
    lib.attn_dev_paged_work_bytes.restype = c_size_t
    for name, args in (("rope_dev_apply", rope_dev_args), ("rope_dev_grad", rope_dev_args),
                       ("kv_dev_append", kv_dev_append_args), ("attn_dev_paged", attn_dev_args),
                       ("attn_dev_tree", attn_dev_tree_args)):
        getattr(lib, name).argtypes = [POINTER(args), vp]
        getattr(lib, name).restype = i
    lib.bfp8_stream.argtypes = []
    lib.bfp8_stream.restype = vp
    return lib


_LIB: Optional[ctypes.CDLL] = None


def load(path: Optional[str] = None) -> ctypes.CDLL:
    """Load and bind libqwen_kernels.so (raises if it has not been built)."""
    global _LIB
    if path is None and _LIB is not None:
        return _LIB
    p = Path(path) if path else LIB_PATH
    if not p.exists():
        raise FileNotFoundError(f"{p} not built: run qwen35-ax7020-edge-llm_amd/build_lib.py")
    lib = bind(ctypes.CDLL(str(p)))
    if path is None:
        _LIB = lib
    return lib


SAMPLING_PATH = LIB_PATH.with_name("libqwen_sampling.so")
_SAMPLING: Optional[ctypes.CDLL] = None


def load_sampling() -> ctypes.CDLL:
    """libqwen_sampling.so, bound as 04/chat_v3.py:150-159 binds the reference's."""
    global _SAMPLING
    if _SAMPLING is None:
        if not SAMPLING_PATH.exists():
            raise FileNotFoundError(f"{SAMPLING_PATH} not built: run qwen35-ax7020-edge-llm_amd/build_lib.py")
        load()
        lib = ctypes.CDLL(str(SAMPLING_PATH))
        lib.lm_head_topk.restype = ctypes.c_int
        lib.lm_head_topk.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int, ctypes.c_int, ctypes.c_int,
                                     ctypes.POINTER(ctypes.c_int), ctypes.POINTER(ctypes.c_float)]
        lib.sample_from_topk.restype = ctypes.c_int
        lib.sample_from_topk.argtypes = [ctypes.POINTER(ctypes.c_int), ctypes.POINTER(ctypes.c_float), ctypes.c_int,
                                         ctypes.c_float, ctypes.c_int, ctypes.c_float, ctypes.POINTER(ctypes.c_uint)]
        _SAMPLING = lib
    return _SAMPLING


def check(rc: int, what: str = "call") -> None:
    if rc != BFP8_OK:
        msg = load().bfp8_last_error().decode(errors="replace")
        raise RuntimeError(f"{what} failed ({rc}): {msg}")


def _ptr(a: np.ndarray) -> int:
    return a.ctypes.data


# ---- synthetic inputs (host) ------------------------------------------------------
def synth_planes(M: int, K: int, seed: int, e_lo: int, e_hi: int):
    """Reference-format planes (int8 [M, K], uint8 [M, K/64]) from the counter hash."""
    lib = load()
    mant = np.empty((M, K), dtype=np.int8)
    exps = np.empty((M, K // 64), dtype=np.uint8)
    lib.bfp8_synth_planes_host(_ptr(mant), _ptr(exps), M, K, seed, e_lo, e_hi)
    return mant, exps


def synth_normal(n: int, seed: int) -> np.ndarray:
    out = np.empty(n, dtype=np.float32)
    load().bfp8_synth_normal(_ptr(out), n, seed)
    return out


def synth_swiglu(n: int, seed: int, outlier_frac: float = 0.01, mag: float = 20.0) -> np.ndarray:
    out = np.empty(n, dtype=np.float32)
    load().bfp8_synth_swiglu(_ptr(out), n, seed, outlier_frac, mag)
    return out


# ---- host-pointer API (engine-style) ---------------------------------------------------
class Bfp8Kernels:
    """The engine's view of the library: numpy in, numpy out, synchronous.

    ``gemv_bfp8`` mirrors QwenRealEngine.gemv_bfp8 (04/qwen_real_engine.py:1221-1240)
    on explicit planes instead of a tensor name.
    """

    def __init__(self, path: Optional[str] = None):
        self.lib = load(path)
        self.lib.init_kernels()

    def gemv_bfp8(self, x: np.ndarray, mantissas: np.ndarray, exps: np.ndarray, M: int, K: int,
                  y: Optional[np.ndarray] = None) -> np.ndarray:
        x = np.ascontiguousarray(x, dtype=np.float32)
        if y is None:
            y = np.empty(M, dtype=np.float32)
        self.lib.bfp8_gemv(_ptr(y), _ptr(x), _ptr(mantissas), _ptr(exps), M, K)
        return y

    def gemv_fallback(self, x: np.ndarray, mantissas: np.ndarray, exps: np.ndarray, M: int, K: int,
                      pairwise: bool = True) -> np.ndarray:
        """The engine's numpy fallback (04/qwen_real_engine.py:1230-1238) on the GPU."""
        x = np.ascontiguousarray(x, dtype=np.float32)
        y = np.empty(M, dtype=np.float32)
        check(self.lib.bfp8_gemv_fallback(_ptr(y), _ptr(x), _ptr(mantissas), _ptr(exps), M, K, int(pairwise)),
              "bfp8_gemv_fallback")
        return y

    def gemv_batch(self, X: np.ndarray, mantissas: np.ndarray, exps: np.ndarray, M: int, K: int) -> np.ndarray:
        X = np.ascontiguousarray(X, dtype=np.float32)
        B = X.shape[0]
        Y = np.empty((B, M), dtype=np.float32)
        self.lib.bfp8_gemv_batch(_ptr(Y), _ptr(X), _ptr(mantissas), _ptr(exps), M, K, B)
        return Y

    def lm_head_topk(self, h: np.ndarray, mantissas: np.ndarray, exps: np.ndarray, vocab: int,
                     hidden: int, k: int):
        h = np.ascontiguousarray(h, dtype=np.float32)
        ids = np.full(max(k, 1), -1, dtype=np.int32)
        scores = np.zeros(max(k, 1), dtype=np.float32)
        n = self.lib.bfp8_lm_head_topk(_ptr(h), _ptr(mantissas), _ptr(exps), vocab, hidden, k,
                                       _ptr(ids), _ptr(scores))
        return ids[:n], scores[:n]

    def lm_head_argmax(self, h: np.ndarray, mantissas: np.ndarray, exps: np.ndarray, vocab: int,
                       hidden: int) -> int:
        h = np.ascontiguousarray(h, dtype=np.float32)
        return self.lib.bfp8_lm_head_argmax(_ptr(h), _ptr(mantissas), _ptr(exps), vocab, hidden)


# ---- device-resident API (torch tensors as device memory) ------------------------------
def _torch():
    import torch  # noqa: local import keeps the CPU-only paths torch-free

    return torch


def _stream():
    torch = _torch()  # (its current_stream() makes an object: 2.6 us of a call's 10)
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


def _dp(t) -> int:
    return t.data_ptr()


class DeviceMatrix:
    """A BFP8 matrix resident in HBM in the GPU layout."""

    def __init__(self, M: int, K: int, mant_gpu, exps_gpu):
        self.M, self.K, self.mant, self.exps = M, K, mant_gpu, exps_gpu

    @staticmethod
    def empty(M: int, K: int, device="cuda"):
        torch = _torch()
        lib = load()
        mg = torch.empty(max(lib.bfp8_dev_mant_bytes(M, K), 1), dtype=torch.int8, device=device)
        eg = torch.empty(max(lib.bfp8_dev_exps_bytes(M, K), 1), dtype=torch.uint8, device=device)
        return DeviceMatrix(M, K, mg, eg)

    @staticmethod
    def from_soa(mant, exps, device="cuda") -> "DeviceMatrix":
        """Convert reference planes (numpy or device tensors) to the GPU layout."""
        torch = _torch()
        M, K = mant.shape
        ms = torch.as_tensor(np.ascontiguousarray(mant)) if isinstance(mant, np.ndarray) else mant
        es = torch.as_tensor(np.ascontiguousarray(exps)) if isinstance(exps, np.ndarray) else exps
        ms, es = ms.to(device).contiguous(), es.to(device).contiguous()
        dm = DeviceMatrix.empty(M, K, device)
        check(load().bfp8_dev_pack(_dp(dm.mant), _dp(dm.exps), _dp(ms), _dp(es), M, K, _stream()), "pack")
        return dm

    @staticmethod
    def synth(M: int, K: int, seed: int, e_lo: int, e_hi: int, device="cuda") -> "DeviceMatrix":
        """Synthetic planes generated on the GPU (same bytes as synth_planes)."""
        torch = _torch()
        ms = torch.empty(M * K, dtype=torch.int8, device=device)
        es = torch.empty(max(M * (K // 64), 1), dtype=torch.uint8, device=device)
        lib = load()
        check(lib.bfp8_dev_synth_planes(_dp(ms), _dp(es), M, K, seed, e_lo, e_hi, _stream()), "synth")
        dm = DeviceMatrix.empty(M, K, device)
        check(lib.bfp8_dev_pack(_dp(dm.mant), _dp(dm.exps), _dp(ms), _dp(es), M, K, _stream()), "pack")
        del ms, es
        return dm

    def unpack(self):
        torch = _torch()
        ms = torch.empty((self.M, self.K), dtype=torch.int8, device=self.mant.device)
        es = torch.empty((self.M, self.K // 64), dtype=torch.uint8, device=self.mant.device)
        check(load().bfp8_dev_unpack(_dp(ms), _dp(es), _dp(self.mant), _dp(self.exps), self.M, self.K,
                                     _stream()), "unpack")
        return ms, es

    @property
    def weight_bytes(self) -> int:
        """Algorithmic bytes: M*K mantissas + M*K/64 exponents."""
        return self.M * self.K + self.M * (self.K // 64)


def quantize(x):
    """x (device float32 [K]) -> (xq int16 [K], xscale f32 [K/64], xsplit int32 words)."""
    torch = _torch()
    K = x.numel()
    nb = K // 64
    xq = torch.empty(max(nb * 64, 1), dtype=torch.int16, device=x.device)
    xs = torch.empty(max(nb, 1), dtype=torch.float32, device=x.device)
    xsp = torch.empty(max(nb * 32, 1), dtype=torch.int32, device=x.device)
    check(load().bfp8_dev_quantize(_dp(xq), _dp(xs), _dp(xsp), _dp(x), K, _stream()), "quantize")
    return xq[: nb * 64], xs[:nb], xsp


def gemv(mat: DeviceMatrix, xsplit, xscale, y=None, lane_sums: bool = False):
    torch = _torch()
    if y is None:
        y = torch.empty(mat.M, dtype=torch.float32, device=mat.mant.device)
    lanes = None
    if lane_sums:
        lanes = torch.empty((mat.M, mat.K // 64, 4), dtype=torch.int32, device=mat.mant.device)
    check(load().bfp8_dev_gemv(_dp(y), _dp(xsplit), _dp(xscale), _dp(mat.mant), _dp(mat.exps), mat.M, mat.K,
                               _dp(lanes) if lanes is not None else None, _stream()), "gemv")
    return (y, lanes) if lane_sums else y


def gemv_float(mat: DeviceMatrix, x, y=None):
    torch = _torch()
    if y is None:
        y = torch.empty(mat.M, dtype=torch.float32, device=mat.mant.device)
    check(load().bfp8_dev_gemv_float(_dp(y), _dp(x), _dp(mat.mant), _dp(mat.exps), mat.M, mat.K, _stream()),
          "gemv_float")
    return y


def gemv_batch(mat: DeviceMatrix, xsplit, xscale, B: int, Y=None):
    torch = _torch()
    if Y is None:
        Y = torch.empty((B, mat.M), dtype=torch.float32, device=mat.mant.device)
    check(load().bfp8_dev_gemv_batch(_dp(Y), _dp(xsplit), _dp(xscale), _dp(mat.mant), _dp(mat.exps), mat.M,
                                     mat.K, B, _stream()), "gemv_batch")
    return Y


def lm_head_topk(mat: DeviceMatrix, xsplit, xscale, k: int):
    """Fused lm_head on the device -> (ids, scores, count, argmax) device tensors."""
    torch = _torch()
    dev = mat.mant.device
    ids = torch.empty(k, dtype=torch.int32, device=dev)
    scores = torch.empty(k, dtype=torch.float32, device=dev)
    cnt = torch.empty(2, dtype=torch.int32, device=dev)
    check(load().bfp8_dev_lm_head_topk(_dp(ids), _dp(scores), _dp(cnt), _dp(cnt) + 4, _dp(xsplit), _dp(xscale),
                                       _dp(mat.mant), _dp(mat.exps), mat.M, mat.K, k, _stream()), "lm_head_topk")
    return ids, scores, cnt[0:1], cnt[1:2]


class SweepPlan:
    """Grouped GEMV plan: per run the persistent streaming launches (the
    lm_head's tiles, a launch that also quantizes every activation, then every
    other GEMV's, whose workgroup 0 also merges the lm_head's top-k); plans
    without an lm_head quantize in a launch of their own first.

    items: sequence of dicts with keys x (device f32 [K]), mat (DeviceMatrix) and either
    y (device f32 [M]) or topk (int) for the fused lm_head (outputs allocated here).
    """

    def __init__(self, items: Sequence[dict]):
        torch = _torch()
        self.items = list(items)
        arr = (bfp8_plan_item * len(self.items))()
        self.topk_out = None
        for i, it in enumerate(self.items):
            m: DeviceMatrix = it["mat"]
            a = arr[i]
            a.x, a.mant_gpu, a.exps_gpu, a.M, a.K = _dp(it["x"]), _dp(m.mant), _dp(m.exps), m.M, m.K
            a.topk = int(it.get("topk", 0))
            if a.topk > 0:
                dev = m.mant.device
                ids = torch.empty(a.topk, dtype=torch.int32, device=dev)
                sc = torch.empty(a.topk, dtype=torch.float32, device=dev)
                cnt = torch.zeros(2, dtype=torch.int32, device=dev)
                self.topk_out = (ids, sc, cnt)
                a.out_ids, a.out_scores, a.out_count, a.out_argmax = _dp(ids), _dp(sc), _dp(cnt), _dp(cnt) + 4
                a.y = None
            else:
                a.y = _dp(it["y"])
        self._arr = arr
        self.handle = load().bfp8_plan_create(arr, len(self.items))
        if not self.handle:
            raise RuntimeError("bfp8_plan_create: " + load().bfp8_last_error().decode())

    def run(self):
        check(load().bfp8_plan_run(self.handle, _stream()), "plan_run")

    def topk_result(self):
        """(ids, scores, argmax) of the lm_head item after run(), waiting for
        the stream; raises when the run reports its top-k invalid (count -1:
        the single launch's merge gave up waiting for a tile's list)."""
        ids, sc, cnt = self.topk_out
        _torch().cuda.current_stream().synchronize()
        n, am = (int(v) for v in cnt.cpu().tolist())
        if n < 0:
            raise RuntimeError("bfp8 plan: the lm_head top-k of this run is invalid (count -1)")
        return ids[:n], sc[:n], am

    def quantize(self):
        check(load().bfp8_plan_quantize(self.handle, _stream()), "plan_quantize")

    def run_gemv(self):
        check(load().bfp8_plan_run_gemv(self.handle, _stream()), "plan_run_gemv")

    def kernel_name(self, stage):
        """Name of the kernel a stage launches ("" if the stage is empty)."""
        return load().bfp8_plan_kernel_name(self.handle, stage).decode()

    def launch(self, stage):
        """One GEMV stage: 0 lm_head tiles, 1 other tiles + merge, 2 tails."""
        check(load().bfp8_plan_launch(self.handle, stage, _stream()), "plan_launch")

    def close(self):
        if self.handle:
            load().bfp8_plan_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ---- a text's tokens -------------------------------------------------------------------
_HERE = contextlib.nullcontext()


def _same_device(first, *tensors):
    """Every tensor on the device of `first`, a GPU; a context that makes it current."""
    device = first.get_device()
    if device < 0:
        raise ValueError("the tensors have to be on a GPU")
    for t in tensors:
        if t is not None and t.get_device() != device:
            raise ValueError(f"a tensor of shape {tuple(t.shape)} is on {t.device}, not on {first.device}")
    cuda = _torch().cuda
    return _HERE if device == cuda.current_device() else cuda.device(device)


def _no_graph(who, why):
    """Refuses inputs whose gradient autograd would be asked for: the results have no graph behind them."""
    raise ValueError(f"{who}: an input requires a gradient, and {why}: detach it, or call under torch.no_grad()")


def _rows_of(t, name, shape, dtype):
    """t of this shape and type, each of its rows contiguous -> the stride between rows."""
    if t.shape != shape or t.dtype != dtype:
        raise ValueError(f"{name} has to be {tuple(shape)} of {dtype}, not {tuple(t.shape)} of {t.dtype}")
    if t.is_contiguous():
        return t.stride()[0]  # (of one row: anything, and not used)
    stride, step = t.stride(), 1
    for n, s in zip(shape[:0:-1], stride[:0:-1]):
        if n != 1 and s != step:
            raise ValueError(f"{name}: a row's elements have to be contiguous")
        step *= n
    if shape[0] < 2:
        return step
    if stride[0] < step:
        raise ValueError(f"{name}: its rows overlap")
    return stride[0]


def _like(t):
    """A contiguous tensor of t's shape and type."""
    torch = _torch()
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _flat(t, name, shape, dtype):
    if t.shape != shape or t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{name} has to be a contiguous {tuple(shape)} of {dtype}")


def _work_of(work):
    """Address and bytes of a caller's work buffer (None: 0, 0)."""
    if work is None:
        return 0, 0
    if not work.is_contiguous():  # (an expanded or strided one has fewer bytes of its own, or others' between)
        raise ValueError("work has to be contiguous")
    return work.data_ptr(), work.numel() * work.element_size()


def _gdn_args(q, k, v, alpha, beta, scale, state_in, state_out, slots, starts, n_seq, work, out, zero_rest):
    """The arguments of either form of the attention."""
    torch = _torch()
    dtype = q.dtype
    if q.dim() != 3 or v.dim() != 3 or dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("q, k, v are [rows, heads, dim] in float32 or bfloat16")
    rows, hk, dk = keys = q.shape
    n_v, hv, dv = values = v.shape
    if n_v != rows:
        raise ValueError("q and v have to have the same rows")
    gates = (rows, hv)
    n_slots = state_out.size(0)
    _flat(state_out, "state_out", (n_slots, hv, dk * dv), torch.float32)
    if state_in is not None and state_in is not state_out:
        _flat(state_in, "state_in", (n_slots, hv, dk * dv), torch.float32)
    if slots is None:
        if n_slots < n_seq:
            raise ValueError("fewer states than sequences")
    else:
        _flat(slots, "slots", (n_seq,), torch.int32)
    f32 = torch.float32
    if (q.is_contiguous() and k.is_contiguous() and v.is_contiguous() and out.is_contiguous() and alpha.is_contiguous()
            and k.shape == keys and out.shape == values and alpha.shape == gates
            and k.dtype == dtype and v.dtype == dtype and out.dtype == dtype and alpha.dtype == f32
            and (beta is None or beta.is_contiguous() and beta.shape == gates and beta.dtype == f32)):
        q_row = k_row = hk * dk  # (the usual step's, whose host time is its time: without a call for each)
        v_row = out_row = hv * dv
        gate_row = hv
    else:
        q_row, k_row = _rows_of(q, "q", keys, dtype), _rows_of(k, "k", keys, dtype)
        v_row, out_row = _rows_of(v, "v", values, dtype), _rows_of(out, "out", values, dtype)
        gate_row = _rows_of(alpha, "alpha", gates, f32)
        if beta is not None and _rows_of(beta, "beta", gates, f32) != gate_row and rows > 1:
            raise ValueError("alpha and beta have to have the same row stride")
    return gdn_dev_args.from_buffer_copy(_GDN_PACK.pack(
        out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), alpha.data_ptr(),
        0 if beta is None else beta.data_ptr(), 0 if state_in is None else state_in.data_ptr(), state_out.data_ptr(),
        0 if slots is None else slots.data_ptr(), 0 if starts is None else starts.data_ptr(),
        *_work_of(work),
        q_row, k_row, v_row, out_row, gate_row, rows, n_seq, n_slots, hk, hv, dk, dv,
        QWEN_F32 if dtype == f32 else QWEN_BF16, scale, zero_rest))


def linear_attention_prompt(q, k, v, alpha, beta=None, starts=None, *, scale=1.0, state_in=None, state_out=None,
                            slots=None, out=None, work=None):
    """Gated linear attention over the tokens of packed sequences -> (out, state_out).

    q, k [rows, heads_k, dim_k], v [rows, heads_v, dim_v] (float32 or bfloat16;
    parts of one projection's row are fine), alpha and beta float32 [rows,
    heads_v]; beta None: no delta rule.  Sequence s is rows starts[s] to
    starts[s + 1] (int32 on the device; None: one sequence).  States are float32
    [slots, heads_v, dim_k * dim_v] in the decode runtime's blocks; a sequence
    starts from its slot of state_in (None: zeros) and leaves its state in that
    slot of state_out (None: a new tensor; it may be state_in).  slots: int32 on
    the device, None: slot s for sequence s.  work: uint8 scratch of at least
    linear_attention_prompt_work_bytes, for callers that keep one.  Rows of out of
    skipped sequences, and rows that no sequence holds, are left as they were where out is
    given; in a new one they are 0 if slots are given, else undefined.  There is no
    backward pass: tensors that require a gradient are refused unless it is off.  The
    rest is gdn_dev_prompt's contract (include/qwen_kernels.h)."""
    torch = _torch()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or alpha.requires_grad or any(
            t is not None and t.requires_grad for t in (beta, state_in, state_out))):
        _no_graph("linear_attention_prompt", "there is no backward pass")
    with _same_device(q, k, v, alpha, beta, starts, state_in, state_out, slots, out, work):
        n_seq = 1 if starts is None else starts.numel() - 1
        if starts is not None:
            _flat(starts, "starts", (max(n_seq, 0) + 1,), torch.int32)
        zero_rest = out is None and slots is not None
        if out is None:
            out = _like(v) if n_seq else v.new_zeros(v.shape)  # (without sequences nothing is launched)
        if state_out is None:
            if slots is not None:
                raise ValueError("slots need a state_out that holds them")
            if q.dim() != 3 or v.dim() != 3:
                raise ValueError("q, k, v are [rows, heads, dim]")
            state_out = alpha.new_empty((n_seq, v.size(1), q.size(2) * v.size(2)), dtype=torch.float32)
        a = _gdn_args(q, k, v, alpha, beta, scale, state_in, state_out, slots, starts, n_seq, work, out, zero_rest)
        lib = load()
        if work is None:
            need = lib.gdn_dev_prompt_work_bytes(a)
            if need:
                work = q.new_empty(need, dtype=torch.uint8)
                a.work, a.work_bytes = work.data_ptr(), need
        check(lib.gdn_dev_prompt(a, _stream()), "linear_attention_prompt")
    return out, state_out


def _sizes_of(a, dtype, **sizes):
    """Sets the sizes of arguments `a` and its type (a c_int takes a larger number's lower half without a word)."""
    torch = _torch()
    if dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"float32 or bfloat16, not {dtype}")
    for name, n in sizes.items():
        if not 0 <= n < 1 << 31:
            raise ValueError(f"{name}: {n} is not a size")
        setattr(a, name, n)
    a.dtype = QWEN_F32 if dtype == torch.float32 else QWEN_BF16


def linear_attention_prompt_work_bytes(rows, n_seq, heads_k, heads_v, dim_k, dim_v, dtype) -> int:
    """Bytes of linear_attention_prompt's work for these sizes (dtype: of q, k, v)."""
    a = gdn_dev_args()
    _sizes_of(a, dtype, rows=rows, n_seq=n_seq, heads_k=heads_k, heads_v=heads_v, dim_k=dim_k, dim_v=dim_v)
    n = load().gdn_dev_prompt_work_bytes(a)
    if not n:
        check(BFP8_EINVAL, "linear_attention_prompt_work_bytes")
    return n


def linear_attention_step(q, k, v, alpha, beta, state, *, scale=1.0, slots=None, out=None):
    """One token for each sequence: row s of q, k, v updates the state in slot
    slots[s] (None: s) of `state` in place -> out.  Rows that are skipped (a slot
    outside the states, or an earlier sequence's) are left as they were in an out that is
    given and are 0 in a new one.  Types, layouts and refusals as in
    linear_attention_prompt; gdn_dev_step (include/qwen_kernels.h)."""
    if (q.requires_grad or k.requires_grad or v.requires_grad or alpha.requires_grad or state.requires_grad
            or beta is not None and beta.requires_grad) and _torch().is_grad_enabled():
        _no_graph("linear_attention_step", "there is no backward pass")
    with _same_device(q, k, v, alpha, beta, state, slots, out):
        zero_rest = out is None and slots is not None
        if out is None:
            out = _like(v)
        a = _gdn_args(q, k, v, alpha, beta, scale, state, state, slots, None, q.shape[0], None, out, zero_rest)
        check(load().gdn_dev_step(a, _stream()), "linear_attention_step")
    return out


def _loss_args(h, table, targets):
    torch = _torch()
    if h.dim() != 2 or table.dim() != 2 or h.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("h is [rows, hidden] in float32 or bfloat16, table [vocab, hidden] in bfloat16")
    a = lm_head_loss_args()
    a.rows, a.hidden = h.shape
    a.vocab = table.shape[0]
    a.h_row = _rows_of(h, "h", (a.rows, a.hidden), h.dtype)
    a.table_row = _rows_of(table, "table", (a.vocab, a.hidden), torch.bfloat16)
    _flat(targets, "targets", (a.rows,), torch.int32)
    a.h, a.table, a.targets = _dp(h), _dp(table), _dp(targets)
    a.dtype = QWEN_F32 if h.dtype == torch.float32 else QWEN_BF16
    return a


def _loss_call(name, a, work, h):
    """Runs entry point `name` with the caller's work or a new one."""
    lib = load()
    need = getattr(lib, name + "_work_bytes")(a)
    if need and work is None:
        work = h.new_empty(need, dtype=_torch().uint8)
    a.work, a.work_bytes = _work_of(work)
    check(getattr(lib, name)(a, _stream()), name)


def lm_head_loss(h, table, targets, *, work=None):
    """Negative log-likelihood of each row's target under the tied-embedding head
    -> (loss, lse), float32 [rows]; the logits are not kept.

    h [rows, hidden] float32 or bfloat16, table [vocab, hidden] bfloat16, targets
    int32 [rows]: below 0 the row is ignored (loss and lse 0), vocab or more
    gives NaN.  work: uint8 scratch of at least lm_head_loss_work_bytes.  No autograd
    graph is built: inputs that require a gradient are refused unless it is off, and
    lm_head_loss_grad has the gradients.  The rest is bf16_dev_lm_head_loss's contract
    (include/qwen_kernels.h)."""
    torch = _torch()
    if (h.requires_grad or table.requires_grad) and torch.is_grad_enabled():
        _no_graph("lm_head_loss", "its gradients are lm_head_loss_grad's")
    with _same_device(h, table, targets, work):
        a = _loss_args(h, table, targets)
        loss, lse = h.new_empty((2, a.rows), dtype=torch.float32)
        a.loss, a.lse = _dp(loss), _dp(lse)
        _loss_call("bf16_dev_lm_head_loss", a, work, h)
    return loss, lse


def lm_head_loss_grad(h, table, targets, lse, grad_loss, *, need_h=True, need_table=True, grad_h=None,
                      grad_table=None, work=None):
    """The gradients of sum(grad_loss * loss) -> (grad_h, grad_table), in h's and the
    table's type, overwritten where given; None for one that is not needed.
    lse is lm_head_loss's; grad_loss float32 [rows].  The gradients have no graph
    behind them, as autograd's own without create_graph."""
    torch = _torch()
    with _same_device(h, table, targets, lse, grad_loss, grad_h, grad_table, work):
        a = _loss_args(h, table, targets)
        _flat(lse, "lse", (a.rows,), torch.float32)
        _flat(grad_loss, "grad_loss", (a.rows,), torch.float32)
        if need_h and grad_h is None:
            grad_h = _like(h)
        if need_table and grad_table is None:
            grad_table = _like(table)
        a.lse, a.grad_loss = _dp(lse), _dp(grad_loss)
        if need_h:
            a.grad_h, a.grad_h_row = _dp(grad_h), _rows_of(grad_h, "grad_h", h.shape, h.dtype)
        if need_table:
            a.grad_table = _dp(grad_table)
            a.grad_table_row = _rows_of(grad_table, "grad_table", table.shape, table.dtype)
        _loss_call("bf16_dev_lm_head_loss_grad", a, work, h)
    return grad_h if need_h else None, grad_table if need_table else None


def lm_head_loss_work_bytes(rows, vocab, hidden, dtype, *, grad=False, need_h=True) -> int:
    """Bytes of lm_head_loss's work for these sizes (dtype: of h), or of lm_head_loss_grad's."""
    a = lm_head_loss_args()
    _sizes_of(a, dtype, rows=rows, vocab=vocab, hidden=hidden)
    a.grad_h = 1 if need_h else None  # only whether it is there
    lib = load()
    n = (lib.bf16_dev_lm_head_loss_grad_work_bytes if grad else lib.bf16_dev_lm_head_loss_work_bytes)(a)
    if not n:
        check(BFP8_EINVAL, "lm_head_loss_work_bytes")
    return n


# ---- positions, the paged cache and the attention over it ---------------------------------
def rotary_frequencies(rot, base=10000.0, *, scaling=None, factor=1.0, original=None, fast=32.0, slow=1.0,
                       device="cuda"):
    """Radians a position of each of rot / 2 pairs, base^(-2 i / rot) -> (freqs, amplitude): freqs float64 on
    the device, amplitude for the rotation.

    scaling, for contexts `factor` times as long as the model was trained on:
    "linear": every frequency divided by it; "ntk": the base grown, so that the slowest is;
    "yarn": pairs that turn more than `fast` times over the `original` context keep their frequency, those
    that turn less than `slow` times are divided, in between a linear ramp over the pairs,
    and the amplitude is 0.1 ln factor + 1 (Peng et al., 2023)."""
    torch = _torch()
    if rot < 2 or rot % 2 or not base > 0 or not factor > 0:
        raise ValueError("rot is even and at least 2, base and factor are above 0")
    if scaling == "ntk":
        if rot < 4:
            raise ValueError("ntk needs at least two pairs")
        base = base * factor ** (rot / (rot - 2))
    freqs = torch.tensor(float(base), dtype=torch.float64) ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    amplitude = 1.0
    if scaling == "linear":
        freqs /= factor
    elif scaling == "yarn":
        if not original or not fast > slow > 0 or not base > 1:
            raise ValueError("yarn needs the original context's length, fast above slow above 0, and a base above 1")
        # the pair, as a number with a fraction, that turns so many times over the original context
        pair = lambda turns: rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), rot - 1)
        ramp = ((torch.arange(rot // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        freqs = freqs * (1 - ramp) + freqs / factor * ramp
        amplitude = 0.1 * math.log(factor) + 1 if factor > 1 else 1.0
    elif scaling not in (None, "ntk"):
        raise ValueError(f"scaling is None, linear, ntk or yarn, not {scaling}")
    return freqs.to(device), amplitude


def _heads_of(t, name, shape, dtype):
    """t of this [rows, heads, dim] and type, each head's elements contiguous -> strides of rows and heads."""
    if t.shape != shape or t.dtype != dtype:
        raise ValueError(f"{name} has to be {tuple(shape)} of {dtype}, not {tuple(t.shape)} of {t.dtype}")
    row, head, one = t.stride()
    if one != 1 and shape[2] > 1:
        raise ValueError(f"{name}: a head's elements have to be contiguous")
    return row, head


def _rotate(who, x, positions, freqs, interleaved, amplitude, out):
    torch = _torch()
    with _same_device(x, positions, freqs, out):
        if x.dim() != 3 or x.dtype not in (torch.float32, torch.bfloat16):
            raise ValueError("x is [rows, heads, dim] in float32 or bfloat16")
        shape = rows, heads, dim = x.shape
        if out is None:
            out = _like(x)
        _flat(positions, "positions", (rows,), torch.int32)
        _flat(freqs, "freqs", (freqs.numel(),), torch.float64)
        a = rope_dev_args.from_buffer_copy(_ROPE_PACK.pack(
            out.data_ptr(), x.data_ptr(), positions.data_ptr(), freqs.data_ptr(), *_heads_of(out, "out", shape, x.dtype),
            *_heads_of(x, "x", shape, x.dtype), rows, heads, dim, 2 * freqs.numel(),
            QWEN_F32 if x.dtype == torch.float32 else QWEN_BF16, bool(interleaved), amplitude))
        check(getattr(load(), who)(a, _stream()), who)
    return out


def rotary(x, positions, freqs, *, interleaved=False, amplitude=1.0, out=None):
    """Rotary positions: each pair of a head's first 2 len(freqs) elements turned by position times
    frequency -> out (a new contiguous tensor, or the one given, which may be x).

    x [rows, heads, dim] float32 or bfloat16, with any strides of rows and heads; positions int32 [rows];
    freqs float64, radians a position (rotary_frequencies).  Pairs are elements i and i + len(freqs), or with
    interleaved 2 i and 2 i + 1; the rotation is multiplied by amplitude.  No autograd graph is built: an x that
    requires a gradient is refused unless gradients are off, and rotary_grad has it.  The rest is rope_dev_apply's
    contract (include/qwen_kernels.h)."""
    if x.requires_grad and _torch().is_grad_enabled():
        _no_graph("rotary", "its gradient is rotary_grad's")
    return _rotate("rope_dev_apply", x, positions, freqs, interleaved, amplitude, out)


def rotary_grad(grad, positions, freqs, *, interleaved=False, amplitude=1.0, out=None):
    """The gradient to rotary's x from that of its result: the transposed rotation -> out (it may be grad)."""
    return _rotate("rope_dev_grad", grad, positions, freqs, interleaved, amplitude, out)


def _cache_of(key_cache, value_cache, dtype):
    """Both caches [pages, page, heads, dim] with the same strides -> their shape and strides."""
    shape = key_cache.shape
    if len(shape) != 4 or value_cache.shape != shape or key_cache.dtype != dtype or value_cache.dtype != dtype:
        raise ValueError(f"the caches have to be [pages, page, heads_k, dim] of {dtype}, both the same")
    strides = key_cache.stride()
    if value_cache.stride() != strides or strides[3] != 1:
        raise ValueError("the caches have to have the same strides, a head's elements contiguous")
    return shape, strides


def _sequences_of(tables, cached, starts):
    """-> the number of sequences, the tables' columns, the stride of their rows."""
    int32 = _torch().int32
    n = cached.numel()
    _flat(cached, "cached", (n,), int32)
    if starts is not None:
        _flat(starts, "starts", (n + 1,), int32)
    if tables.dim() != 2 or tables.size(0) != n or tables.dtype != int32:
        raise ValueError("tables has to be [sequences, pages of a sequence] of int32")
    row, one = tables.stride()
    if one != 1 and tables.size(1) > 1:
        raise ValueError("tables: a row's elements have to be contiguous")
    return n, tables.size(1), row


def kv_cache_append(k, v, key_cache, value_cache, tables, cached, starts=None, *, positions=None, freqs=None,
                    interleaved=False, amplitude=1.0, q=None, q_out=None):
    """Writes a call's keys and values to their places in the paged caches, the keys rotated on the way where
    freqs is given; q is rotated in the same launch -> q_out (a new contiguous tensor, or the one
    given, which may be q; None without q).

    k, v [rows, heads_k, dim] float32 or bfloat16, q [rows, heads_q, dim]; key_cache and
    value_cache [pages, page, heads_k, dim] of the same type, with any strides that are multiples of 16 bytes (the
    same in both).  Sequence s has rows starts[s] to starts[s + 1] (int32 on the device; None: the same number each), its pages
    in tables[s] (int32 [sequences, pages], -1: none), and held cached[s] tokens before (int32, below 0: skipped);
    its row i goes to place cached[s] + i.  positions int32 [rows]: of the rotation, None: the
    places.  Rows of q_out of skipped sequences, and that no sequence holds, are left as they were (undefined in a new
    one).  There is no backward pass: tensors that require a gradient are refused unless it is off.  The rest is
    kv_dev_append's contract (include/qwen_kernels.h)."""
    torch = _torch()
    if (k.requires_grad or v.requires_grad or key_cache.requires_grad or value_cache.requires_grad
            or q is not None and q.requires_grad) and torch.is_grad_enabled():
        _no_graph("kv_cache_append", "there is no backward pass")
    with _same_device(k, v, key_cache, value_cache, tables, cached, starts, positions, freqs, q, q_out):
        dtype = k.dtype
        if k.dim() != 3 or dtype not in (torch.float32, torch.bfloat16):
            raise ValueError("k and v are [rows, heads_k, dim] in float32 or bfloat16")
        shape = rows, heads, dim = k.shape
        cache, strides = _cache_of(key_cache, value_cache, dtype)
        if cache[2] != heads or cache[3] != dim:
            raise ValueError(f"the caches' heads are {tuple(cache[2:])}, not {(heads, dim)}")
        n_seq, columns, table_row = _sequences_of(tables, cached, starts)
        if positions is not None:
            _flat(positions, "positions", (rows,), torch.int32)
        if freqs is not None:
            _flat(freqs, "freqs", (freqs.numel(),), torch.float64)
        heads_q, q_strides = 0, (0, 0, 0, 0)
        if q is not None:
            if freqs is None:
                raise ValueError("q is given to be rotated, and there are no freqs")
            if q.dim() != 3:
                raise ValueError("q is [rows, heads_q, dim]")
            heads_q = q.size(1)
            if q_out is None:
                q_out = _like(q)
            q_strides = (*_heads_of(q, "q", (rows, heads_q, dim), dtype),
                         *_heads_of(q_out, "q_out", (rows, heads_q, dim), dtype))
        elif q_out is not None:
            raise ValueError("q_out without q")
        ptr = _ptr_or_0
        a = kv_dev_append_args.from_buffer_copy(_APPEND_PACK.pack(
            key_cache.data_ptr(), value_cache.data_ptr(), ptr(q_out), k.data_ptr(), v.data_ptr(), ptr(q),
            tables.data_ptr(), cached.data_ptr(), ptr(starts), ptr(positions), ptr(freqs), *strides[:3], table_row,
            *_heads_of(k, "k", shape, dtype), *_heads_of(v, "v", shape, dtype), *q_strides,
            rows, n_seq, cache[0], cache[1], columns, heads_q, heads, dim, 0 if freqs is None else 2 * freqs.numel(),
            QWEN_F32 if dtype == torch.float32 else QWEN_BF16, bool(interleaved), amplitude))
        check(load().kv_dev_append(a, _stream()), "kv_cache_append")
    return q_out


def _ptr_or_0(t):
    return 0 if t is None else t.data_ptr()


def draft_tree(parents, cached, starts=None, *, longest=None, mask=None, positions=None):
    """Drafted tokens' masks and positions from their tree -> (mask, positions), once for all layers of a step.

    parents int32 [rows]: for each drafted token the place, among its sequence's rows, of the token that it follows,
    an earlier one (below 0: the cached text).  mask int32 [rows, words]: bit j of a row (word j / 32,
    bit j % 32) is set for the row's own place and its ancestors'; positions int32 [rows]: cached[s] plus the
    number of its ancestors.  cached and starts as in kv_cache_append.  longest: the most rows that a sequence
    has, for the words of a new mask (None: as many as there are rows, or without starts each has).
    attn_dev_tree (include/qwen_kernels.h)."""
    torch = _torch()
    with _same_device(parents, cached, starts, mask, positions):
        rows, n_seq = parents.numel(), cached.numel()
        _flat(parents, "parents", (rows,), torch.int32)
        _flat(cached, "cached", (n_seq,), torch.int32)
        if starts is not None:
            _flat(starts, "starts", (n_seq + 1,), torch.int32)
        if mask is None:
            if longest is None:
                longest = rows if starts is not None or not n_seq else rows // n_seq
            mask = parents.new_empty((rows, max(1, (longest + 31) // 32)))
        words = mask.size(1) if mask.dim() == 2 else 0
        _flat(mask, "mask", (rows, words), torch.int32)
        if positions is None:
            positions = parents.new_empty((rows,))
        _flat(positions, "positions", (rows,), torch.int32)
        a = attn_dev_tree_args.from_buffer_copy(_TREE_PACK.pack(
            mask.data_ptr(), positions.data_ptr(), parents.data_ptr(), cached.data_ptr(), _ptr_or_0(starts),
            rows, n_seq, words))
        check(load().attn_dev_tree(a, _stream()), "draft_tree")
    return mask, positions


def paged_attention(q, key_cache, value_cache, tables, cached, starts=None, *, scale=None, mask=None, out=None, work=None):
    """Attention of a call's tokens over the paged caches, their own keys and values in them already
    (kv_cache_append) -> out.

    q [rows, heads_q, dim], float32 or bfloat16 as the caches, heads_q a multiple of their heads; tables, cached
    and starts as in kv_cache_append (cached: without this call's tokens, as there).  Row i of a sequence sees
    the places up to cached[s] + i, or with a mask (draft_tree's, or any int32 [rows, words]) the cached ones and those of
    the sequence's rows whose bit is set.  scale: of the scores, None: dim^-0.5.  work: uint8 scratch of at least
    paged_attention_work_bytes, 256-byte aligned.  Rows of skipped sequences are left as they were where out is given, and 0 in a
    new one; rows that no sequence holds are left as they were, undefined in a new one.  There is no backward
    pass: tensors that require a gradient are refused unless it is off.  The rest is attn_dev_paged's contract
    (include/qwen_kernels.h)."""
    torch = _torch()
    if (q.requires_grad or key_cache.requires_grad or value_cache.requires_grad) and torch.is_grad_enabled():
        _no_graph("paged_attention", "there is no backward pass")
    with _same_device(q, key_cache, value_cache, tables, cached, starts, mask, out, work):
        dtype = q.dtype
        if q.dim() != 3 or dtype not in (torch.float32, torch.bfloat16):
            raise ValueError("q is [rows, heads_q, dim] in float32 or bfloat16")
        shape = rows, heads_q, dim = q.shape
        cache, strides = _cache_of(key_cache, value_cache, dtype)
        if cache[3] != dim:
            raise ValueError(f"the caches' heads have {cache[3]} elements, not {dim}")
        n_seq, columns, table_row = _sequences_of(tables, cached, starts)
        words = 0
        if mask is not None:
            words = mask.size(1) if mask.dim() == 2 else 0
            _flat(mask, "mask", (rows, words), torch.int32)
            if not words:
                raise ValueError("mask has no words")
        zero_rest = out is None
        if out is None:
            out = _like(q)
        a = attn_dev_args.from_buffer_copy(_ATTN_PACK.pack(
            out.data_ptr(), q.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), tables.data_ptr(),
            cached.data_ptr(), _ptr_or_0(starts), _ptr_or_0(mask), *_work_of(work), *strides[:3], table_row,
            *_heads_of(q, "q", shape, dtype), *_heads_of(out, "out", shape, dtype),
            rows, n_seq, cache[0], cache[1], columns, heads_q, cache[2], dim, words,
            QWEN_F32 if dtype == torch.float32 else QWEN_BF16, dim ** -0.5 if scale is None else scale, zero_rest))
        lib = load()
        if work is None:
            need = lib.attn_dev_paged_work_bytes(a)
            if need:
                work = q.new_empty(need, dtype=torch.uint8)
                a.work, a.work_bytes = work.data_ptr(), need
        check(lib.attn_dev_paged(a, _stream()), "paged_attention")
    return out


def paged_attention_work_bytes(rows, n_seq, heads_q, heads_k, dim, dtype) -> int:
    """Bytes of paged_attention's work for these sizes (dtype: of q and the caches)."""
    a = attn_dev_args()
    _sizes_of(a, dtype, rows=rows, n_seq=n_seq, heads_q=heads_q, heads_k=heads_k, dim=dim)
    n = load().attn_dev_paged_work_bytes(a)
    if not n:
        check(BFP8_EINVAL, "paged_attention_work_bytes")
    return n
