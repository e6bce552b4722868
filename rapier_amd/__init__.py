"""rapier_amd - MI355X-native exact-verify MTP hot path for the qwen35 hybrid (Rapier's engine, gfx950).

The compute lives in ``librapier_mi.so`` (hand-written HIP, C ABI declared in ``include/rapier_mi.h``).  This module
is the host-side mirror of the reference's ``strata::kernels`` launch surface: the same function names, argument
meaning and error behaviour (``ValueError`` where the reference throws ``std::invalid_argument``, ``RuntimeError``
for ``std::runtime_error``).  Device memory and streams come from PyTorch (``torch.Tensor`` arguments); nothing
here computes on the CPU.  A missing library is an ``ImportError``-style failure, never a fallback.
"""
from __future__ import annotations

import array
import ctypes
import functools
import operator
import os
import subprocess
import sys

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "librapier_mi.so")
CSRC = os.path.join(_HERE, "csrc")

RMI_OK, RMI_ERR_SHAPE, RMI_ERR_POINTER, RMI_ERR_STREAM, RMI_ERR_LAUNCH, RMI_ERR_UNSUPPORTED, RMI_ERR_STATE = range(7)
GGML_Q8_0, GGML_Q6_K = 8, 14
KV_F16, KV_I8, KV_I4 = range(3)   # K/V cache types
TREE_SHORT = 1 << 24              # a split's flag (gqa_tree_nsub)
ROPE_HALF, ROPE_NEIGHBOURS = range(2)                        # dims (i, i + n_rot / 2) or (2 i, 2 i + 1) of a pair
PAGES_OK, PAGES_BAD_LENGTH, PAGES_NONE_LEFT = range(3)       # a request's status in a page plan
Q6K_BYTES, Q8_0_BYTES, Q8_1_BYTES = 210, 34, 36

_lib = None
_vp, _i, _f, _sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_size_t

# name -> (restype, argtypes); every int-returning entry is a status code checked by _call
SIGNATURES = {
    "rmi_last_error": (ctypes.c_char_p, []),
    "rmi_version": (ctypes.c_char_p, []),
    "rmi_native_q8_1_bytes": (_sz, [_i, _i]),
    "rmi_native_quantize_q8_1": (_i, [_vp, _vp, _i, _i, _vp]),
    "rmi_native_q6_k_mmvq": (_i, [_vp, _vp, _vp, _i, _i, _i, _vp]),
    "rmi_native_q6_k_mmvq_res": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _i, _vp]),
    "rmi_native_q6_k_mmvq_res_n": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _vp]),
    "rmi_native_q4_k_mmvq": (_i, [_vp, _vp, _vp, _i, _i, _i, _vp]),
    "rmi_native_q5_k_mmvq": (_i, [_vp, _vp, _vp, _i, _i, _i, _vp]),
    "rmi_native_q4_k_mmvq_res_n": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _vp]),
    "rmi_native_q5_k_mmvq_res_n": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _vp]),
    "rmi_native_q4_k_mmvq_res": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _i, _vp]),
    "rmi_native_q5_k_mmvq_res": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _i, _vp]),
    "rmi_q6_k_packed_bytes": (_sz, [_i, _i]),
    "rmi_q6_k_pack": (_i, [_vp, _vp, _i, _i, _vp]),
    "rmi_native_q6_k_pack_copy": (_i, [_vp, _i, _i]),
    "rmi_native_q6_k_unpack": (_i, [_vp]),
    "rmi_native_q6_k_packed_copies": (_i, []),
    "rmi_q6_k_pack_swiglu": (_i, [_vp, _vp, _i, _i, _vp]),
    "rmi_native_q6_k_swiglu_packed": (_i, [_vp, _vp, _vp, _i, _i, _i, _vp]),
    "rmi_rms_quant_apply_self": (_i, [_vp, _vp, _vp, _i, _f, _i, _vp]),
    "rmi_native_q6_k_mmvq_packed": (_i, [_vp, _vp, _vp, _i, _i, _i, _vp]),
    "rmi_native_q6_k_mmvq_packed_res_n": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _vp]),
    "rmi_q6_k_gemm_workspace_bytes": (_sz, [_i, _i]),
    "rmi_q6_k_gemm_packed": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _vp, _vp]),
    "rmi_q6_k_block_dots": (_i, [_vp, _vp, _vp, _i, _i, _vp]),
    "rmi_native_q6_k_mmvq_packed_norm": (_i, [_vp, _vp, _vp, _vp, _f, _vp, _i, _i, _i, _vp]),
    "rmi_native_q6_k_swiglu_packed_norm": (_i, [_vp, _vp, _vp, _vp, _f, _vp, _i, _i, _i, _vp]),
    "rmi_q6_k_packed_norm_preferred": (_i, [_i, _i, _i]),
    "rmi_gen_q6_k": (_i, [_vp, _sz, ctypes.c_uint64, _f, _vp]),
    "rmi_gen_q8_0": (_i, [_vp, _sz, ctypes.c_uint64, _f, _vp]),
    "rmi_gen_normal": (_i, [_vp, _sz, ctypes.c_uint64, _f, _f, _vp]),
    "rmi_gen_normal_f16": (_i, [_vp, _sz, ctypes.c_uint64, _f, _f, _vp]),
    "rmi_stream_read": (_i, [_vp, _sz, _i, _vp, _vp]),
    "rmi_gdn_exchange_timeouts": (ctypes.c_uint, []),
    "rmi_gdn_exchange_test": (_i, [ctypes.c_uint, _i]),
    "rmi_gdn_exchange_bytes": (_sz, [_i]),
    "rmi_gdn_layer_tokens_x": (_i, [_vp, _vp, _vp, _vp, _vp, _vp, _i, _vp, _i, _vp, _vp, _vp, _vp, _f, _vp, _i, _vp,
                                    _i, _i, _i, _i, _vp, _vp]),
    "rmi_rms_quant_apply": (_i, [_vp, _vp, _vp, _vp, _i, _f, _i, _vp]),
    "rmi_rms_quant_apply_pair": (_i, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, _f, _i, _vp]),
    "rmi_rms_norm_out": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _f, _i, _vp]),
    "rmi_rms_norm_out_strided": (_i, [_vp, _vp, _vp, _vp, _i, _vp, _i, _f, _i, _vp]),
    "rmi_row_sum_partials": (_i, [_vp, _vp, _i, _i, _vp]),
    "rmi_add_partials": (_i, [_vp, _vp, _vp, _i, _i, _vp]),
    "rmi_swiglu_quant": (_i, [_vp, _vp, _vp, _i, _i, _i, _vp]),
    "rmi_swiglu_quant_interleaved": (_i, [_vp, _vp, _i, _i, _i, _vp]),
    "rmi_sig_mul_quant": (_i, [_vp, _vp, _vp, _i, _i, _i, _i, _vp]),
    "rmi_beta_gate": (_i, [_vp, _vp, _vp, _vp, _i, _i, _i, _vp]),
    "rmi_argmax_workspace_bytes": (_sz, [_i]),
    "rmi_argmax": (_i, [_vp, _i, _i, _i, _vp, _vp, _vp]),
    "rmi_topk_workspace_bytes": (_sz, [_i]),
    "rmi_topk": (_i, [_vp, _i, _i, _vp, _vp, _vp, _vp]),
    "rmi_embed_q6_k": (_i, [_vp, _vp, _vp, _vp, _i, _i, _i, _vp]),
    "rmi_embed": (_i, [_i, _vp, _vp, _vp, _vp, _i, _i, _i, _vp]),
    "rmi_embed_quant_apply_pair": (_i, [_i, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _f, _i, _vp]),
    "rmi_fused_gdn_conv_l2": (_i, [_vp, _vp, _vp, _vp, _i, _i, _f, _vp]),
    "rmi_fused_gdn_step_norm_silu_q8": (_i, [_vp] * 8 + [_f, _vp, _vp, _i, _i, _vp]),
    "rmi_gdn_layer_tokens": (_i, [_vp, _vp, _vp, _vp, _vp, _vp, _i, _vp, _i, _vp, _vp, _vp, _vp, _f, _vp, _i, _vp,
                                  _i, _i, _i, _i, _vp]),
    "rmi_attn_prep": (_i, [_vp, _i, _vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _f, _f, _i, _i, _vp]),
    "rmi_attn_prep_rope": (_i, [_vp, _i, _vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _vp, _f, _i, _i, _vp]),
    "rmi_gqa_flash_decode_prep": (_i, [_vp, _i, _vp, _vp, _vp, _vp, _vp, _vp, _i, _vp, _i, _vp, _i, _i, _i, _i, _vp,
                                       _f, _i, _i, _i, _f, _vp]),
    "rmi_gqa_rope_table_bytes": (ctypes.c_size_t, [_i]),
    "rmi_gqa_flash_decode_prep_rt": (_i, [_vp, _i, _vp, _vp, _vp, _vp, _vp, _vp, _i, _vp, _i, _vp, _i, _i, _i, _i,
                                          _vp, _f, _i, _i, _i, _f, _vp, _i, _vp]),
    "rmi_rms_norm_weighted": (_i, [_vp, _vp, _i, _i, _f, _vp]),
    "rmi_native_rope_apply": (_i, [_vp, _vp, _i, _i, _i, _vp, _vp, _vp]),
    "rmi_add_inplace": (_i, [_vp, _vp, _i, _vp]),
    "rmi_scale_inplace": (_i, [_vp, _i, _f, _vp]),
    "rmi_silu_inplace": (_i, [_vp, _i, _vp]),
    "rmi_gqa_workspace_bytes": (_sz, [_i, _i, _i]),
    "rmi_gqa_noalloc_scratch_bytes": (_sz, [_i, _i, _i, _i]),
    "rmi_gqa_noalloc_scratch_max": (_sz, []),
    "rmi_gqa_flash_decode_noalloc": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _vp, _i, _vp, _i, _i, _i, _i, _i, _i, _i, _f,
                                          _vp]),
    "rmi_gqa_flash_decode": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _vp, _i, _vp, _i, _vp, _i, _i, _i, _i, _i, _i, _f,
                                  _vp]),
    "rmi_kv_cache_bytes": (_sz, [_i, _i, _i, _i]),
    "rmi_kv_write": (_i, [_i, _vp, _i, _i, _vp, _i, _i, _i, _i, _i, _vp]),
    "rmi_kv_read": (_i, [_i, _vp, _vp, _i, _i, _i, _i, _i, _i, _i, _vp]),
    "rmi_kv_compact": (_i, [_i, _vp, _i, _vp, _vp, _vp, _i, _i, _i, _i, _vp]),
    "rmi_attn_prep_axes": (_i, [_vp, _i, _vp, _vp, _i, _vp, _i, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _vp, _vp, _f, _i,
                                _i, _vp]),
    "rmi_gqa_tree_nsub": (_i, [_i, _i, _i, _i, _i]),
    "rmi_gqa_tree_workspace_bytes": (_sz, [_i, _i, _i, _i, _i, _i]),
    "rmi_gqa_tree_decode": (_i, [_vp, _i, _vp, _i, _vp, _vp, _vp, _vp, _i, _vp, _i, _vp, _i, _vp, _i, _i, _i, _i, _i,
                                 _i, _f, _vp]),
    "rmi_page_plan": (_i, [_vp, _vp, _i, _i, _i, _vp, _vp, _vp, _i, _i, _vp, _vp, _vp, _vp, _vp, _vp, _vp]),
    "rmi_page_trim": (_i, [_vp, _vp, _i, _i, _i, _vp, _i, _vp, _vp, _vp, _vp]),
    "rmi_kv_page_read": (_i, [_i, _vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _i, _vp]),
    "rmi_attn_prep_paged": (_i, [_vp, _i, _vp, _vp, _i, _vp, _i, _vp, _vp, _vp, _i, _vp, _i, _i, _i, _i, _vp, _i, _f,
                                 _i, _i, _i, _vp]),
    "rmi_gqa_paged_split": (_i, [ctypes.c_longlong, _i, _i, _i, _i, _i, _i, _i]),
    "rmi_gqa_paged_workspace_bytes": (_sz, [_i, _i, _i, _i, _i]),
    "rmi_gqa_paged_attn": (_i, [_i, _vp, _i, _vp, _i, _vp, _vp, _i, _vp, _vp, _vp, _i, _vp, _i, _vp, _i, _vp, _i, _i,
                                _i, _i, _i, _i, _i, _i, _i, _i, _f, _vp]),
    "rmi_gqa_prompt_attn": (_i, [_i, _vp, _i, _vp, _i, _vp, _i, _vp, _vp, _i, _vp, _i, _vp, _i, _i, _i, _i, _i, _i, _i,
                                 _f, _vp]),
    "rmi_logits_process": (_i, [_vp, _i, _i, _i, _vp, _i, _vp, _vp, _i, _vp, _vp, _i, _vp, _vp, _vp, _i, _vp, _i,
                                _vp]),
}


class RapierError(RuntimeError):
    pass


def build(force: bool = False, jobs: int = 8) -> str:
    """Compile librapier_mi.so for gfx950 with hipcc (cross-compiles without a GPU)."""
    cmd = ["make", f"-j{jobs}"] + (["-B"] if force else [])
    subprocess.run(cmd, cwd=CSRC, check=True)
    return LIB_PATH


def lib():
    """The loaded HIP library.  Raises if it has not been built: there is no CPU fallback."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(f"rapier_amd: {LIB_PATH} is missing; run __graft_entry__.build() first")
        # One HIP runtime per process: torch bundles its own libamdhip64 (soname libamdhip64.so.7).  Loading torch
        # first makes our NEEDED libamdhip64.so.7 bind to that copy, so device pointers and streams are shared;
        # loading ours first would start a second runtime that does not see torch's allocations.
        try:
            import torch  # noqa: F401
        except ImportError:
            pass
        L = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _lib = L
    return _lib


def last_error() -> str:
    return lib().rmi_last_error().decode()


def _check(rc):
    if rc != RMI_OK:
        msg = last_error()
        if rc in (RMI_ERR_SHAPE, RMI_ERR_POINTER, RMI_ERR_STREAM, RMI_ERR_UNSUPPORTED):
            raise ValueError(msg)
        raise RapierError(msg)


_entries = {}   # entry points by name


def _call(name, *args):
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(lib(), name)
    rc = fn(*args)
    if rc:
        _check(rc)


def _p(t):
    """Device pointer of a torch tensor (None -> NULL)."""
    return None if t is None else ctypes.c_void_p(t.data_ptr())


_raw_stream = None   # torch's current stream handle, once its GPU state exists


def _current_stream():
    global _raw_stream
    import torch
    s = torch.cuda.current_stream().cuda_stream
    if torch.cuda.is_initialized() and hasattr(torch._C, "_cuda_getCurrentRawStream"):
        # the handle itself: current_stream() builds a Stream object for it at every call, 3 us
        device, raw = torch.cuda.current_device, torch._C._cuda_getCurrentRawStream
        _raw_stream = lambda: raw(device())  # noqa: E731
    return s


def _stream(stream):
    if stream is None:
        return ctypes.c_void_p(_raw_stream() if _raw_stream else _current_stream())
    if isinstance(stream, int):
        return ctypes.c_void_p(stream)
    return ctypes.c_void_p(stream.cuda_stream)


# ---- strata::kernels mirror -----------------------------------------------------------------------------------------

def native_q8_1_bytes(n_in: int, ncols: int) -> int:
    n = lib().rmi_native_q8_1_bytes(n_in, ncols)
    if n == 0:
        raise ValueError(last_error())
    return n


def native_quantize_q8_1(x, x_q8_1, n_in: int, ncols: int, stream=None):
    _call("rmi_native_quantize_q8_1", _p(x), _p(x_q8_1), n_in, ncols, _stream(stream))


def native_q6_k_mmvq(w, x_q8_1, y, n_in: int, n_out: int, ncols: int, stream=None):
    _call("rmi_native_q6_k_mmvq", _p(w), _p(x_q8_1), _p(y), n_in, n_out, ncols, _stream(stream))


def native_q6_k_mmvq_res(w, x_q8_1, y, res, partials, n_in: int, n_out: int, stream=None):
    _call("rmi_native_q6_k_mmvq_res", _p(w), _p(x_q8_1), _p(y), _p(res), _p(partials), n_in, n_out, _stream(stream))


def native_q6_k_mmvq_res_n(w, x_q8_1, y, res, partials, n_in: int, n_out: int, ncols: int, stream=None):
    _call("rmi_native_q6_k_mmvq_res_n", _p(w), _p(x_q8_1), _p(y), _p(res), _p(partials), n_in, n_out, ncols,
          _stream(stream))


def native_kquant_mmvq(ggml_type, w, x_q8_1, y, n_in: int, n_out: int, ncols: int = 1, stream=None):
    """Q4_K (12) / Q5_K (13) x Q8_1 GEMV"""
    name = {12: "rmi_native_q4_k_mmvq", 13: "rmi_native_q5_k_mmvq"}[ggml_type]
    _call(name, _p(w), _p(x_q8_1), _p(y), n_in, n_out, ncols, _stream(stream))


def native_kquant_mmvq_res_n(ggml_type, w, x_q8_1, y, res, partials, n_in: int, n_out: int, ncols: int = 1,
                             stream=None):
    name = {12: "rmi_native_q4_k_mmvq_res_n", 13: "rmi_native_q5_k_mmvq_res_n"}[ggml_type]
    _call(name, _p(w), _p(x_q8_1), _p(y), _p(res), _p(partials), n_in, n_out, ncols, _stream(stream))


def q6_k_packed_bytes(n_in: int, n_out: int) -> int:
    n = lib().rmi_q6_k_packed_bytes(n_in, n_out)
    if n == 0:
        raise ValueError(last_error())
    return n


def q6_k_pack(w, w_packed, n_in: int, n_out: int, stream=None):
    _call("rmi_q6_k_pack", _p(w), _p(w_packed), n_in, n_out, _stream(stream))


def native_q6_k_pack(w, n_in: int, n_out: int) -> bool:
    """native_q6_k_pack (mmvq:2930-2960): a library-owned packed copy of the GGUF-layout matrix ``w`` that
    native_q6_k_mmvq / _res / _res_n then run on (the same bits); False where the packed layout does not take the
    shape, as the reference returns false."""
    rc = lib().rmi_native_q6_k_pack_copy(_p(w), n_in, n_out)
    if rc == RMI_ERR_UNSUPPORTED:
        return False
    _check(rc)
    return True


def native_q6_k_unpack(w):
    _call("rmi_native_q6_k_unpack", _p(w))


def native_q6_k_packed_copies() -> int:
    return int(lib().rmi_native_q6_k_packed_copies())


def q6_k_pack_swiglu(w, w_packed, n_in: int, n_ff: int, stream=None):
    """pack an up||gate Q6_K matrix ([up n_ff rows | gate n_ff rows]) in the SwiGLU row order"""
    _call("rmi_q6_k_pack_swiglu", _p(w), _p(w_packed), n_in, n_ff, _stream(stream))


def native_q6_k_swiglu_packed(w_packed, x_q8_1, y_q8_1, n_in: int, n_ff: int, ncols: int, stream=None):
    """Q8_1 of silu(gate) * up from an up||gate matrix packed by q6_k_pack_swiglu (one launch)"""
    _call("rmi_native_q6_k_swiglu_packed", _p(w_packed), _p(x_q8_1), _p(y_q8_1), n_in, n_ff, ncols, _stream(stream))


def native_q6_k_mmvq_packed(w_packed, x_q8_1, y, n_in: int, n_out: int, ncols: int, stream=None):
    _call("rmi_native_q6_k_mmvq_packed", _p(w_packed), _p(x_q8_1), _p(y), n_in, n_out, ncols, _stream(stream))


def native_q6_k_mmvq_packed_norm(w_packed, x, w_norm, partials, eps, y, n_in: int, n_out: int, ncols: int,
                                 stream=None):
    """rms_quant_apply + packed GEMV in one launch (the norm quantized in the GEMV's stage); same bits as the pair"""
    _call("rmi_native_q6_k_mmvq_packed_norm", _p(w_packed), _p(x), _p(w_norm), _p(partials), eps, _p(y), n_in, n_out,
          ncols, _stream(stream))


def native_q6_k_swiglu_packed_norm(w_packed, x, w_norm, partials, eps, y_q8_1, n_in: int, n_ff: int, ncols: int,
                                   stream=None):
    """rms_quant_apply + the fused up||gate SwiGLU GEMV in one launch; same bits as the pair"""
    _call("rmi_native_q6_k_swiglu_packed_norm", _p(w_packed), _p(x), _p(w_norm), _p(partials), eps, _p(y_q8_1), n_in,
          n_ff, ncols, _stream(stream))


def native_q6_k_mmvq_packed_res_n(w_packed, x_q8_1, y, res, partials, n_in: int, n_out: int, ncols: int,
                                  stream=None):
    _call("rmi_native_q6_k_mmvq_packed_res_n", _p(w_packed), _p(x_q8_1), _p(y), _p(res), _p(partials), n_in, n_out,
          ncols, _stream(stream))


def q6_k_gemm_workspace_bytes(n_in: int, ncols: int) -> int:
    n = lib().rmi_q6_k_gemm_workspace_bytes(n_in, ncols)
    if n == 0:
        raise ValueError(last_error())
    return n


def q6_k_gemm_packed(w_packed, x_q8_1, y, res, partials, n_in: int, n_out: int, ncols: int, ws, stream=None):
    """the packed GEMV over 1..4096 columns in one weight pass; each column bitwise the GEMV's"""
    _call("rmi_q6_k_gemm_packed", _p(w_packed), _p(x_q8_1), _p(y), _p(res), _p(partials), n_in, n_out, ncols, _p(ws),
          _stream(stream))


def q6_k_block_dots(w, x_q8_1, out, n_in: int, n_out: int, stream=None):
    _call("rmi_q6_k_block_dots", _p(w), _p(x_q8_1), _p(out), n_in, n_out, _stream(stream))


# ---- seeded synthetic tensors in HBM (random-init stand-in for a GGUF file) -----------------------------------------

def gen_q6_k(w, nblocks: int, seed: int, d_std: float = 1e-3, stream=None):
    """Fill ``nblocks`` Q6_K blocks: codes U{0..63}, sub-scales U[-32,31], d = fp16(|N(0, d_std)|)."""
    _call("rmi_gen_q6_k", _p(w), nblocks, seed, d_std, _stream(stream))


def gen_q8_0(w, nblocks: int, seed: int, d_std: float = 1e-2, stream=None):
    _call("rmi_gen_q8_0", _p(w), nblocks, seed, d_std, _stream(stream))


def gen_normal(out, n: int, seed: int, mean: float = 0.0, std: float = 1.0, stream=None):
    _call("rmi_gen_normal", _p(out), n, seed, mean, std, _stream(stream))


def gen_normal_f16(out, n: int, seed: int, mean: float = 0.0, std: float = 1.0, stream=None):
    _call("rmi_gen_normal_f16", _p(out), n, seed, mean, std, _stream(stream))


def stream_read(buf, nbytes: int, grid: int, out, stream=None):
    """the single-launch read-bandwidth reference: streams nbytes of buf with grid x 256 lanes and discards them"""
    _call("rmi_stream_read", _p(buf), nbytes, grid, _p(out), _stream(stream))


# ---- norm / activation epilogues (qw:602-715) ----------------------------------------------------------------------

def rms_quant_apply(x, w, partials, y_q8_1, cols, eps, ncols=1, stream=None):
    _call("rmi_rms_quant_apply", _p(x), _p(w), _p(partials), _p(y_q8_1), cols, eps, ncols, _stream(stream))


def rms_quant_apply_self(x, w, y_q8_1, cols, eps, ncols=1, stream=None):
    """row_sum_partials(x) + rms_quant_apply in one launch (same bytes)"""
    _call("rmi_rms_quant_apply_self", _p(x), _p(w), _p(y_q8_1), cols, eps, ncols, _stream(stream))


def rms_quant_apply_pair(x0, w0, partials0, x1, w1, partials1, y_q8_1, cols, eps, ncols=1, stream=None):
    _call("rmi_rms_quant_apply_pair", _p(x0), _p(w0), _p(partials0), _p(x1), _p(w1), _p(partials1), _p(y_q8_1), cols,
          eps, ncols, _stream(stream))


def rms_norm_out(x, w, partials, out, out_partials, cols, eps, ncols=1, stream=None):
    _call("rmi_rms_norm_out", _p(x), _p(w), _p(partials), _p(out), _p(out_partials), cols, eps, ncols,
          _stream(stream))


def rms_norm_out_strided(x, w, partials, out, out_stride, out_partials, cols, eps, ncols=1, stream=None):
    _call("rmi_rms_norm_out_strided", _p(x), _p(w), _p(partials), _p(out), out_stride, _p(out_partials), cols, eps,
          ncols, _stream(stream))


def row_sum_partials(x, partials, n, ncols=1, stream=None):
    _call("rmi_row_sum_partials", _p(x), _p(partials), n, ncols, _stream(stream))


def add_partials(x, o, partials, n, ncols=1, stream=None):
    _call("rmi_add_partials", _p(x), _p(o), _p(partials), n, ncols, _stream(stream))


def swiglu_quant(up, gate, y_q8_1, n, ncols=1, col_stride=None, stream=None):
    _call("rmi_swiglu_quant", _p(up), _p(gate), _p(y_q8_1), n, ncols, n if col_stride is None else col_stride,
          _stream(stream))


def swiglu_quant_interleaved(up_gate, y_q8_1, n, ncols=1, col_stride=None, stream=None):
    _call("rmi_swiglu_quant_interleaved", _p(up_gate), _p(y_q8_1), n, ncols, 2 * n if col_stride is None else col_stride,
          _stream(stream))


def sig_mul_quant(o, g, y_q8_1, n, ncols=1, o_stride=None, g_stride=None, stream=None):
    _call("rmi_sig_mul_quant", _p(o), _p(g), _p(y_q8_1), n, ncols, n if o_stride is None else o_stride,
          n if g_stride is None else g_stride, _stream(stream))


def beta_gate(beta_alpha, dt, ssm_a, ggate, n, ncols=1, ab_stride=None, stream=None):
    _call("rmi_beta_gate", _p(beta_alpha), _p(dt), _p(ssm_a), _p(ggate), n, ncols,
          2 * n if ab_stride is None else ab_stride, _stream(stream))


def argmax_workspace_bytes(ncols):
    return lib().rmi_argmax_workspace_bytes(ncols)


def argmax(logits, n, out_idx, workspace, ncols=1, col_stride=None, stream=None):
    _call("rmi_argmax", _p(logits), n, ncols, n if col_stride is None else col_stride, _p(out_idx), _p(workspace),
          _stream(stream))


def topk_workspace_bytes(n):
    return lib().rmi_topk_workspace_bytes(n)


def topk(logits, n, k, out_idx, out_val, workspace, stream=None):
    """the k largest of n logits: out_idx (int32) and out_val (fp32), logit descending, lower id first on ties"""
    _call("rmi_topk", _p(logits), n, k, _p(out_idx), _p(out_val), _p(workspace), _stream(stream))


def embed_q6_k(emb, tokens, x, partials, n_embd, n_vocab, ncols=1, stream=None):
    _call("rmi_embed_q6_k", _p(emb), _p(tokens), _p(x), _p(partials), n_embd, n_vocab, ncols, _stream(stream))


def embed(ggml_type, emb, tokens, x, partials, n_embd, n_vocab, ncols=1, stream=None):
    """token rows of a GGUF type 14 (Q6_K) / 13 (Q5_K) / 12 (Q4_K) table, dequantized on the device"""
    _call("rmi_embed", ggml_type, _p(emb), _p(tokens), _p(x), _p(partials), n_embd, n_vocab, ncols, _stream(stream))


def embed_quant_apply_pair(ggml_type, emb, tokens, w0, x1, w1, partials1, y_q8_1, cols, n_vocab, eps, ncols=1,
                           stream=None):
    """embed + rms_quant_apply_pair(embedding rows, w0, .., x1, w1, partials1) in one launch (same bytes)"""
    _call("rmi_embed_quant_apply_pair", ggml_type, _p(emb), _p(tokens), _p(w0), _p(x1), _p(w1), _p(partials1),
          _p(y_q8_1), cols, n_vocab, eps, ncols, _stream(stream))


# ---- Gated DeltaNet (fgdn:40-133) ----------------------------------------------------------------------------------

def fused_gdn_conv_l2(history, qkv, conv_w, h, channels, qk_heads, eps, stream=None):
    _call("rmi_fused_gdn_conv_l2", _p(history), _p(qkv), _p(conv_w), _p(h), channels, qk_heads, eps, _stream(stream))


def fused_gdn_step_norm_silu_q8(state, q, k, v, gate, beta, z, gamma, eps, y, q8, h_k, h_v, stream=None):
    _call("rmi_fused_gdn_step_norm_silu_q8", _p(state), _p(q), _p(k), _p(v), _p(gate), _p(beta), _p(z), _p(gamma),
          eps, _p(y), _p(q8), h_k, h_v, _stream(stream))


def gdn_exchange_timeouts() -> int:
    """bounded waits of the split GDN kernel that ran out (0 in every correct run)"""
    return lib().rmi_gdn_exchange_timeouts()


def gdn_exchange_test(spin_limit: int = 0, force_miss: bool = False) -> None:
    """test hook: the split GDN kernel's wait bound (0 = default) and a switch that makes every wait time out"""
    _call("rmi_gdn_exchange_test", spin_limit, 1 if force_miss else 0)


def gdn_exchange_bytes(h_v: int) -> int:
    return lib().rmi_gdn_exchange_bytes(h_v)


def gdn_layer_tokens_x(state_a, state_b, hist_a, hist_b, sel, qkvz, qkvz_stride, ab, ab_stride, conv_w, dt, ssm_a,
                       gamma, eps, y, y_stride, q8, q8_stride, h_k, h_v, ntok, xch, stream=None):
    """gdn_layer_tokens with 1 / 2-token launches on four workgroups per value head (xch: zeroed exchange buffer)"""
    _call("rmi_gdn_layer_tokens_x", _p(state_a), _p(state_b), _p(hist_a), _p(hist_b), _p(sel), _p(qkvz), qkvz_stride,
          _p(ab), ab_stride, _p(conv_w), _p(dt), _p(ssm_a), _p(gamma), eps, _p(y), y_stride, _p(q8), q8_stride, h_k,
          h_v, ntok, _p(xch), _stream(stream))


def gdn_layer_tokens(state_a, state_b, hist_a, hist_b, sel, qkvz, qkvz_stride, ab, ab_stride, conv_w, dt, ssm_a,
                     gamma, eps, y, y_stride, q8, q8_stride, h_k, h_v, ntok, stream=None):
    _call("rmi_gdn_layer_tokens", _p(state_a), _p(state_b), _p(hist_a), _p(hist_b), _p(sel), _p(qkvz), qkvz_stride,
          _p(ab), ab_stride, _p(conv_w), _p(dt), _p(ssm_a), _p(gamma), eps, _p(y), y_stride, _p(q8), q8_stride, h_k,
          h_v, ntok, _stream(stream))


# ---- attention --------------------------------------------------------------------------------------------------------

def attn_prep(q3, q3_stride, qn, kn, kcache, vcache, pos, qout, n_head, n_kv, head_dim, n_rot, theta, eps, ntok,
              max_ctx, stream=None):
    _call("rmi_attn_prep", _p(q3), q3_stride, _p(qn), _p(kn), _p(kcache), _p(vcache), _p(pos), _p(qout), n_head,
          n_kv, head_dim, n_rot, theta, eps, ntok, max_ctx, _stream(stream))


class RopeParams(ctypes.Structure):
    """rmi_rope_params: YaRN as the reference configures it (qw:1991-1999)"""
    _fields_ = [(n, ctypes.c_float) for n in ("freq_base", "factor", "orig_ctx", "ext_factor", "attn_factor",
                                              "beta_fast", "beta_slow")]


def attn_prep_rope(q3, q3_stride, qn, kn, kcache, vcache, pos, qout, n_head, n_kv, head_dim, n_rot, freq_base, factor,
                   orig_ctx, eps, ntok, max_ctx, ext_factor=1.0, attn_factor=1.0, beta_fast=32.0, beta_slow=1.0,
                   stream=None):
    rope = RopeParams(freq_base, factor, orig_ctx, ext_factor, attn_factor, beta_fast, beta_slow)
    _call("rmi_attn_prep_rope", _p(q3), q3_stride, _p(qn), _p(kn), _p(kcache), _p(vcache), _p(pos), _p(qout), n_head,
          n_kv, head_dim, n_rot, ctypes.byref(rope), eps, ntok, max_ctx, _stream(stream))


def gqa_flash_decode_prep(q3, q3_stride, qn, kn, kcache, vcache, pos, y, y_stride, q8, q8_stride, workspace, n_head,
                          n_kv, head_dim, n_rot, freq_base, factor, orig_ctx, eps, ntok, max_ctx, nsub, scale,
                          ext_factor=1.0, attn_factor=1.0, beta_fast=32.0, beta_slow=1.0, stream=None):
    """attn_prep folded into the split-K decode attention (one slot group: decode and verify)"""
    rope = RopeParams(freq_base, factor, orig_ctx, ext_factor, attn_factor, beta_fast, beta_slow)
    _call("rmi_gqa_flash_decode_prep", _p(q3), q3_stride, _p(qn), _p(kn), _p(kcache), _p(vcache), _p(pos), _p(y),
          y_stride, _p(q8), q8_stride, _p(workspace), n_head, n_kv, head_dim, n_rot, ctypes.byref(rope), eps, ntok,
          max_ctx, nsub, scale, _stream(stream))


def gqa_rope_table_bytes(n_rot: int) -> int:
    return lib().rmi_gqa_rope_table_bytes(n_rot)


def gqa_flash_decode_prep_rt(q3, q3_stride, qn, kn, kcache, vcache, pos, y, y_stride, q8, q8_stride, workspace,
                             n_head, n_kv, head_dim, n_rot, freq_base, factor, orig_ctx, eps, ntok, max_ctx, nsub,
                             scale, rope_table, table_mode, ext_factor=1.0, attn_factor=1.0, beta_fast=32.0,
                             beta_slow=1.0, stream=None):
    """gqa_flash_decode_prep with the forward pass's RoPE table (table_mode 0 compute, 1 compute and store, 2 load)"""
    rope = RopeParams(freq_base, factor, orig_ctx, ext_factor, attn_factor, beta_fast, beta_slow)
    _call("rmi_gqa_flash_decode_prep_rt", _p(q3), q3_stride, _p(qn), _p(kn), _p(kcache), _p(vcache), _p(pos), _p(y),
          y_stride, _p(q8), q8_stride, _p(workspace), n_head, n_kv, head_dim, n_rot, ctypes.byref(rope), eps, ntok,
          max_ctx, nsub, scale, _p(rope_table), table_mode, _stream(stream))


def rms_norm_weighted(x, w, rows, cols, eps, stream=None):
    """per-row RMSNorm in place (strata::kernels::rms_norm_weighted, qw:971-975)"""
    _call("rmi_rms_norm_weighted", _p(x), _p(w), rows, cols, eps, _stream(stream))


def native_rope_apply(x, y, heads, head_dim, n_rot, pos, freq_base, factor=1.0, orig_ctx=0.0, ext_factor=1.0,
                      attn_factor=1.0, beta_fast=32.0, beta_slow=1.0, stream=None):
    """NEOX / YaRN RoPE of each head at its device position pos[h] (strata::kernels::native_rope_apply)"""
    rope = RopeParams(freq_base, factor, orig_ctx, ext_factor, attn_factor, beta_fast, beta_slow)
    _call("rmi_native_rope_apply", _p(x), _p(y), heads, head_dim, n_rot, ctypes.byref(rope), _p(pos), _stream(stream))


def add_inplace(x, y, n, stream=None):
    _call("rmi_add_inplace", _p(x), _p(y), n, _stream(stream))


def scale_inplace(x, n, s, stream=None):
    _call("rmi_scale_inplace", _p(x), n, s, _stream(stream))


def silu_inplace(x, n, stream=None):
    _call("rmi_silu_inplace", _p(x), n, _stream(stream))


def gqa_workspace_bytes(max_ctx, n_kv, nsub):
    return lib().rmi_gqa_workspace_bytes(max_ctx, n_kv, nsub)


def gqa_flash_decode(q, kcache, vcache, pos, gate_src, gate_stride, y, y_stride, q8, q8_stride, workspace, n_head,
                     n_kv, head_dim, ntok, max_ctx, nsub, scale, stream=None):
    _call("rmi_gqa_flash_decode", _p(q), _p(kcache), _p(vcache), _p(pos), _p(gate_src), gate_stride, _p(y), y_stride,
          _p(q8), q8_stride, _p(workspace), n_head, n_kv, head_dim, ntok, max_ctx, nsub, scale, _stream(stream))


def gqa_flash_decode_noalloc(q, kcache, vcache, pos, gate_src, gate_stride, y, y_stride, q8, q8_stride, n_head, n_kv,
                             head_dim, ntok, max_ctx, nsub, scale, stream=None):
    """rmi_gqa_flash_decode without a workspace argument: the split-K records live in the library's own per-GPU
    scratch array (rmi_gqa_noalloc_scratch_max() bytes); no allocation.  Calls that overlap on one GPU race."""
    _call("rmi_gqa_flash_decode_noalloc", _p(q), _p(kcache), _p(vcache), _p(pos), _p(gate_src), gate_stride, _p(y),
          y_stride, _p(q8), q8_stride, n_head, n_kv, head_dim, ntok, max_ctx, nsub, scale, _stream(stream))


# ---- K/V caches in 16, 8 or 4 bits, attention for drafted trees over them, logits of a tree's nodes ---------------------

# Short calls of many arguments: addresses go as plain integers (an argument of a declared c_void_p takes one; building the
# c_void_p objects first costs 0.1 us each).

def _a(t):
    return None if t is None else t.data_ptr()


_gpu = None   # torch's current device and raw stream, without the checks (0.5 us each) around them


def _s(stream, at, *tensors):
    """the stream's handle, for a call on the tensor `at` and these (None: an argument left out): all on the current GPU, whose
    kernels and streams these are"""
    global _gpu
    at = at.get_device()   # -1: host memory
    for t in tensors:
        if t is not None and t.get_device() != at:
            raise ValueError("a tensor that is not on the current GPU")
    if at < 0:
        raise ValueError("a tensor that is not on the current GPU")
    if _gpu is None:
        c = sys.modules["torch"]._C
        _gpu = c._cuda_getDevice, c._cuda_getCurrentRawStream
    if at != _gpu[0]():
        raise ValueError("a tensor that is not on the current GPU")
    if stream is None:
        return _gpu[1](at)
    if isinstance(stream, int):
        return stream
    if getattr(stream, "device_index", at) != at:
        raise ValueError("a stream that is not the current GPU's")
    return stream.cuda_stream


# element types that an argument may have (filled when torch is known to be there); uint8: raw memory
_F32, _I32, _I64 = {}, {}, {}


def _another_type(kind, t):
    """an argument whose type is not in `kind`: the first one of all, or an error"""
    if not kind:
        torch = sys.modules["torch"]
        for k, names in ((_F32, ("float32", "uint8")), (_I32, ("int32", "uint32", "uint8")), (_I64, ("int64", "uint64", "uint8"))):
            k.update((getattr(torch, name), names[0]) for name in names)
    if t.dtype not in kind:
        raise ValueError(f"a tensor of {t.dtype} where the library takes {next(iter(kind.values()))}")


# addresses of such arguments (None: left out)

def _f32(t):
    if t is None:
        return None
    if t.dtype not in _F32:
        _another_type(_F32, t)
    return t.data_ptr()


def _i32(t):
    if t is None:
        return None
    if t.dtype not in _I32:
        _another_type(_I32, t)
    return t.data_ptr()


def _i64(t):
    if t is None:
        return None
    if t.dtype not in _I64:
        _another_type(_I64, t)
    return t.data_ptr()


def kv_cache_bytes(type_, max_ctx, n_kv, head_dim) -> int:
    n = lib().rmi_kv_cache_bytes(type_, max_ctx, n_kv, head_dim)
    if n == 0:
        raise ValueError(last_error())
    return n


_ROWS = {}   # dtypes of rows -> whether they are 16-bit


def _is_f16(t):
    """1 for float16 rows (or int16 / uint16 that hold their bits), 0 for float32"""
    f16 = _ROWS.get(t.dtype)
    if f16 is None:
        torch = sys.modules["torch"]
        _ROWS.update({torch.float32: 0, torch.float16: 1, torch.int16: 1, torch.uint16: 1})
        f16 = _ROWS.get(t.dtype)
        if f16 is None:
            raise ValueError(f"rows of float32 or float16, not {t.dtype}")
    return f16


def _rows(t, n, cache):
    """the rows' address; no rows (an empty tensor has no address) are as well anywhere"""
    return t.data_ptr() or (cache.data_ptr() if n == 0 else None)


def kv_write(type_, src, src_stride, cache, first, n, n_kv, head_dim, max_ctx, stream=None):
    """n rows [n_kv x head_dim] of float32 or float16, src_stride elements apart, to positions [first, first + n)"""
    _call("rmi_kv_write", type_, _rows(src, n, cache), _is_f16(src), src_stride, _a(cache), first, n, n_kv, head_dim, max_ctx,
          _s(stream, cache, src))


def kv_read(type_, cache, out, out_stride, first, n, n_kv, head_dim, max_ctx, stream=None):
    """positions [first, first + n) of a cache back to float32 or float16 rows"""
    _call("rmi_kv_read", type_, _a(cache), _rows(out, n, cache), _is_f16(out), out_stride, first, n, n_kv, head_dim, max_ctx,
          _s(stream, cache, out))


def kv_compact(type_, caches, pos, path, count, max_path, n_kv, head_dim, max_ctx, stream=None):
    """rows pos[0] + path[i] -> pos[0] + i, i < min(count[0], max_path), in each of the caches (a list of tensors)"""
    ptrs = array.array("Q", [c.data_ptr() for c in caches] or [0])
    _call("rmi_kv_compact", type_, ptrs.buffer_info()[0], len(caches), _i32(pos), _i32(path), _i32(count), max_path, n_kv,
          head_dim, max_ctx, _s(stream, pos, path, count, *caches))


class RopeAxes(ctypes.Structure):
    """rmi_rope_axes: the pairs of each axis and how they are dealt out"""
    _fields_ = [("section", ctypes.c_int * 3), ("interleaved", ctypes.c_int)]


class _NotAValue(Exception):
    """an argument that is kept by its identity, whatever it holds later (a tensor's element)"""


def _by_value(values):
    if not all(isinstance(v, (int, float)) for v in values):
        raise _NotAValue   # and nothing is kept


@functools.lru_cache(maxsize=64)
def _rope_args(sections, interleaved, *rope):
    """the argument blocks of these values, which the library only reads (building them costs as much as the call)"""
    _by_value(sections + rope)
    return ctypes.byref(RopeParams(*rope)), ctypes.byref(RopeAxes((ctypes.c_int * 3)(*sections), interleaved))


def attn_prep_axes(q3, q3_stride, qn, kn, ktype, kcache, vtype, vcache, pos, axis_pos, qout, n_head, n_kv, head_dim,
                   n_rot, freq_base, factor, orig_ctx, sections, interleaved, eps, ntok, max_ctx, ext_factor=1.0,
                   attn_factor=1.0, beta_fast=32.0, beta_slow=1.0, stream=None):
    """per-head norm, rotation at axis_pos ([3][ntok]; None: the slots) and the cache write at slots pos[0] + t"""
    values = freq_base, factor, orig_ctx, ext_factor, attn_factor, beta_fast, beta_slow
    try:
        rope, axes = _rope_args(tuple(sections), bool(interleaved), *values)
    except _NotAValue:
        rope, axes = _rope_args(tuple(map(operator.index, sections)), bool(interleaved), *map(float, values))
    _call("rmi_attn_prep_axes", _f32(q3), q3_stride, _f32(qn), _f32(kn), ktype, _a(kcache), vtype, _a(vcache),
          _i32(pos), _i32(axis_pos), _f32(qout), n_head, n_kv, head_dim, n_rot, rope, axes, eps, ntok, max_ctx,
          _s(stream, kcache, vcache, q3, qn, kn, pos, axis_pos, qout))


def gqa_tree_nsub(ctx, n_head, n_kv, head_dim, ntok) -> int:
    """the split of a context of ctx positions: chunks of 128 * nsub, with TREE_SHORT added where groups of 16 rows pay"""
    n = lib().rmi_gqa_tree_nsub(ctx, n_head, n_kv, head_dim, ntok)
    if n == 0:
        raise ValueError(last_error())
    return n


def gqa_tree_workspace_bytes(max_ctx, n_head, n_kv, head_dim, ntok, nsub) -> int:
    n = lib().rmi_gqa_tree_workspace_bytes(max_ctx, n_head, n_kv, head_dim, ntok, nsub)
    if n == 0:
        raise ValueError(last_error())
    return n


def gqa_tree_decode(q, ktype, kcache, vtype, vcache, pos, masks, gate_src, gate_stride, y, y_stride, q8, q8_stride,
                    workspace, n_head, n_kv, head_dim, ntok, max_ctx, nsub, scale, stream=None):
    """attention of ntok drafted tokens at slots pos[0] + t: all of the context before them, and of each other what
    masks[t] (int64 bit patterns) says; masks None: the chain j <= t"""
    _call("rmi_gqa_tree_decode", _f32(q), ktype, _a(kcache), vtype, _a(vcache), _i32(pos), _i64(masks), _f32(gate_src),
          gate_stride, _f32(y), y_stride, _a(q8), q8_stride, _a(workspace), n_head, n_kv, head_dim, ntok, max_ctx, nsub,
          scale, _s(stream, q, kcache, vcache, pos, masks, gate_src, y, q8, workspace))


class Penalties(ctypes.Structure):
    """rmi_penalties"""
    _fields_ = [("repetition", ctypes.c_float), ("presence", ctypes.c_float), ("frequency", ctypes.c_float),
                ("window", ctypes.c_int)]


@functools.lru_cache(maxsize=64)
def _penalties(*values):
    """the argument block of these values"""
    _by_value(values)
    return ctypes.byref(Penalties(*values))


def logits_process(logits, n, ncols, col_stride, out, out_stride, history, history_len, max_history, window=0,
                   draft=None, masks=None, ndraft=0, repetition=1.0, presence=0.0, frequency=0.0, bias_ids=None,
                   bias_vals=None, n_bias=0, allow=None, allow_stride=0, stream=None):
    """biases, penalties over history (+ the draft path of each column's mask) and grammar masks, before argmax / topk"""
    try:
        pen = _penalties(repetition, presence, frequency, window)
    except _NotAValue:
        pen = _penalties(float(repetition), float(presence), float(frequency), operator.index(window))
    _call("rmi_logits_process", _f32(logits), n, ncols, col_stride, _f32(out), out_stride, _i32(history), _i32(history_len),
          max_history, _i32(draft), _i64(masks), ndraft, pen, _i32(bias_ids), _f32(bias_vals), n_bias, _i32(allow),
          allow_stride, _s(stream, logits, out, history, history_len, draft, masks, bias_ids, bias_vals, allow))


# ---- several requests at once: caches in pages, attention for a ragged batch --------------------------------------------

def page_plan(past, count, n_req, page_size, n_pages, free_pages, n_free, table, table_stride, max_tok, row_start, kv_len, slot,
              pos, n_left, status, stream=None):
    """row starts, lengths, slots and positions of count[i] new tokens of each request, and the pages they need (int32 tensors)"""
    _call("rmi_page_plan", _i32(past), _i32(count), n_req, page_size, n_pages, _i32(free_pages), _i32(n_free), _i32(table),
          table_stride, max_tok, _i32(row_start), _i32(kv_len), _i32(slot), _i32(pos), _i32(n_left), _i32(status),
          _s(stream, table, past, count, free_pages, n_free, row_start, kv_len, slot, pos, n_left, status))


def page_trim(length, keep, n_req, page_size, n_pages, table, table_stride, n_free, free_pages, n_out, stream=None):
    """the pages past the first keep[i] of length[i] positions of each request, back to the free list (after a plan, length is the
    larger of kv_len and past: a request that it refused has kv_len 0 and still holds its pages)"""
    _call("rmi_page_trim", _i32(length), _i32(keep), n_req, page_size, n_pages, _i32(table), table_stride, _i32(n_free),
          _i32(free_pages), _i32(n_out), _s(stream, table, length, keep, n_free, free_pages, n_out))


def kv_page_read(type_, pool, slot, out, out_stride, n, n_kv, head_dim, page_size, n_pages, stream=None):
    """the rows of n slots of a pool to float32 or float16 rows"""
    _call("rmi_kv_page_read", type_, _a(pool), _i32(slot), _rows(out, n, pool), _is_f16(out), out_stride, n, n_kv, head_dim,
          page_size, n_pages, _s(stream, pool, slot, out))


_ROWS16 = {}   # dtypes of 16-bit rows -> the library's name of them


def _row_type(*tensors):
    """RMI_ROWS_F16 or RMI_ROWS_BF16, the type of all of these (None: an argument left out)"""
    kind = None
    for t in tensors:
        if t is None:
            continue
        k = _ROWS16.get(t.dtype)
        if k is None:
            torch = sys.modules["torch"]
            _ROWS16.update({torch.float16: 0, torch.bfloat16: 1})
            k = _ROWS16.get(t.dtype)
            if k is None:
                raise ValueError(f"rows of float16 or bfloat16, not {t.dtype}")
        if kind is None:
            kind = k
        elif k != kind:
            raise ValueError("rows of one type, float16 or bfloat16")
    return kind


@functools.lru_cache(maxsize=64)
def _rope_values(*rope):
    """the argument block of these values"""
    _by_value(rope)
    return ctypes.byref(RopeParams(*rope))


def attn_prep_paged(q3, q3_stride, qn, kn, ktype, kpool, vtype, vpool, slot, pos, qout, n_head, n_kv, head_dim, n_rot, pairs,
                    freq_base, eps, ntok, page_size, n_pages, factor=1.0, orig_ctx=0.0, ext_factor=1.0, attn_factor=1.0,
                    beta_fast=32.0, beta_slow=1.0, stream=None):
    """per-head norm (qn / kn None: none), rotation of row t at pos[t], q to float16 or bfloat16 rows, K and V to slot[t]"""
    values = freq_base, factor, orig_ctx, ext_factor, attn_factor, beta_fast, beta_slow
    try:
        rope = _rope_values(*values)
    except _NotAValue:
        rope = _rope_values(*map(float, values))
    _call("rmi_attn_prep_paged", _f32(q3), q3_stride, _f32(qn), _f32(kn), ktype, _a(kpool), vtype, _a(vpool), _i32(slot),
          _i32(pos), _row_type(qout), _a(qout), n_head, n_kv, head_dim, n_rot, rope, pairs, eps, ntok, page_size, n_pages,
          _s(stream, kpool, vpool, q3, qn, kn, slot, pos, qout))


def gqa_paged_split(total_ctx, max_ctx, n_req, ntok, max_new, n_head, n_kv, head_dim) -> int:
    """the positions of a chunk, for a batch of total_ctx positions and ntok new tokens in all"""
    n = lib().rmi_gqa_paged_split(total_ctx, max_ctx, n_req, ntok, max_new, n_head, n_kv, head_dim)
    if n == 0:
        raise ValueError(last_error())
    return n


def gqa_paged_workspace_bytes(ntok, max_ctx, n_head, head_dim, split) -> int:
    n = lib().rmi_gqa_paged_workspace_bytes(ntok, max_ctx, n_head, head_dim, split)
    if n == 0:
        raise ValueError(last_error())
    return n


def gqa_paged_attn(q, ktype, kpool, vtype, vpool, table, table_stride, row_start, kv_len, gate_src, gate_stride, y, y_stride, q8,
                   q8_stride, workspace, n_req, ntok, max_new, max_ctx, n_head, n_kv, head_dim, page_size, n_pages, split, scale,
                   stream=None):
    """attention of each request's new tokens (rows row_start[i] .. of q) over its pages, up to position kv_len[i] - 1"""
    _call("rmi_gqa_paged_attn", _row_type(q, y), _a(q), ktype, _a(kpool), vtype, _a(vpool), _i32(table), table_stride,
          _i32(row_start), _i32(kv_len), _f32(gate_src), gate_stride, _a(y), y_stride, _a(q8), q8_stride, _a(workspace), n_req,
          ntok, max_new, max_ctx, n_head, n_kv, head_dim, page_size, n_pages, split, scale,
          _s(stream, q, kpool, vpool, table, row_start, kv_len, gate_src, y, q8, workspace))


def gqa_prompt_attn(q, q_stride, k, k_stride, v, v_stride, row_start, gate_src, gate_stride, y, y_stride, q8, q8_stride, n_req,
                    ntok, max_len, n_head, n_kv, head_dim, scale, stream=None):
    """causal attention over whole prompts packed row by row (float16 or bfloat16)"""
    _call("rmi_gqa_prompt_attn", _row_type(q, k, v, y), _a(q), q_stride, _a(k), k_stride, _a(v), v_stride, _i32(row_start),
          _f32(gate_src), gate_stride, _a(y), y_stride, _a(q8), q8_stride, n_req, ntok, max_len, n_head, n_kv, head_dim, scale,
          _s(stream, q, k, v, row_start, gate_src, y, q8))
