"""ctypes binding of libm1moe_hip.so (the C ABI declared in include/m1moe_hip.h).

The library is built in-tree (``make -C m1moe_amd/csrc``) and loaded from
this package directory only.  There is no fallback: if the shared library is
missing, importing the binding raises, so a GPU run can never silently take
another code path.
"""
from __future__ import annotations

import ctypes
import os
from ctypes import POINTER, c_char_p, c_float, c_int32, c_uint16, c_uint64, c_void_p

LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libm1moe_hip.so")

M1MOE_OK = 0
M1MOE_ERR_INVALID = 1
M1MOE_ERR_HIP = 2
M1MOE_ERR_OOM = 3
M1MOE_ERR_DEVICE = 4

M1MOE_F32 = 0
M1MOE_BF16 = 1

PROJ_GATE, PROJ_UP, PROJ_DOWN = 0, 1, 2


class MoEShape(ctypes.Structure):
    """m1moe_moe_shape: ModelSpec.hiddenDim/numLayers + MoESpec + QuantSpec.groupSize."""

    _fields_ = [
        ("hidden", c_int32),
        ("num_experts", c_int32),
        ("top_k", c_int32),
        ("intermediate", c_int32),
        ("group_size", c_int32),
        ("num_layers", c_int32),
        ("norm_topk_prob", c_int32),
    ]


class DecShape(ctypes.Structure):
    """m1moe_dec_shape: ModelSpec.vocabSize/rmsNormEps + AttentionSpec (ModelSpec.swift:19-22,
    62-75); qk_norm = the OLMoE per-head q/k RMSNorm (InferenceEngine.swift:55)."""

    _fields_ = [
        ("vocab", c_int32),
        ("num_heads", c_int32),
        ("num_kv_heads", c_int32),
        ("head_dim", c_int32),
        ("max_seq", c_int32),
        ("qk_norm", c_int32),
        ("rope_theta", c_float),
        ("rms_eps", c_float),
    ]


def _address(p):
    """A device address (int, c_void_p, DeviceBuffer or None) as ctypes stores it."""
    p = getattr(p, "ptr", p)
    return p.value if isinstance(p, c_void_p) else None if p is None else int(p)


def dtype_code(dtype) -> int:
    """M1MOE_F32 or M1MOE_BF16 from "f32" / "bf16" or the code itself."""
    if dtype in ("bf16", M1MOE_BF16):
        return M1MOE_BF16
    if dtype in ("f32", M1MOE_F32):
        return M1MOE_F32
    raise ValueError(f"unknown dtype {dtype!r}")


class PagedKV(ctypes.Structure):
    """m1moe_paged_kv: a KV cache in pages, in the caller's memory."""

    _fields_ = [
        ("d_k", c_void_p),
        ("d_v", c_void_p),
        ("dtype", c_int32),
        ("num_pages", c_int32),
        ("page_size", c_int32),
        ("num_kv_heads", c_int32),
        ("head_dim", c_int32),
    ]

    @staticmethod
    def make(k, v, dtype, num_pages: int, page_size: int, num_kv_heads: int,
             head_dim: int) -> "PagedKV":
        return PagedKV(_address(k), _address(v), dtype_code(dtype), num_pages, page_size,
                       num_kv_heads, head_dim)


class PagedBatch(ctypes.Structure):
    """m1moe_paged_batch: the rows, lengths and page tables of one call."""

    _fields_ = [
        ("num_seqs", c_int32),
        ("num_rows", c_int32),
        ("table_stride", c_int32),
        ("prefix_len", c_int32),
        ("d_row_start", c_void_p),
        ("d_kv_len", c_void_p),
        ("d_pages", c_void_p),
        ("d_prefix_pages", c_void_p),
    ]

    @staticmethod
    def make(num_seqs: int, num_rows: int, row_start, kv_len, pages, table_stride: int,
             prefix_len: int = 0, prefix_pages=None) -> "PagedBatch":
        return PagedBatch(num_seqs, num_rows, table_stride, prefix_len, _address(row_start),
                          _address(kv_len), _address(pages), _address(prefix_pages))


class KVAppend(ctypes.Structure):
    """m1moe_kv_append_args: what an append reads and writes besides the cache."""

    _fields_ = [
        ("dtype", c_int32),
        ("num_heads", c_int32),
        ("d_q", c_void_p),
        ("d_k", c_void_p),
        ("d_v", c_void_p),
        ("d_q_out", c_void_p),
        ("q_stride", ctypes.c_int64),
        ("k_stride", ctypes.c_int64),
        ("v_stride", ctypes.c_int64),
        ("q_out_stride", ctypes.c_int64),
        ("d_q_norm", c_void_p),
        ("d_k_norm", c_void_p),
        ("eps", c_float),
        ("rotary_dim", c_int32),
        ("interleaved", c_int32),
        ("rope_amplitude", c_float),
        ("d_inv_freq", c_void_p),
    ]

    @staticmethod
    def make(dtype, num_heads: int, q, k, v, q_stride: int, k_stride: int, v_stride: int, q_out,
             q_out_stride: int, q_norm=None, k_norm=None, eps: float = 0.0, rotary_dim: int = 0,
             interleaved: bool = False, inv_freq=None, amplitude: float = 1.0) -> "KVAppend":
        return KVAppend(dtype_code(dtype), num_heads, _address(q), _address(k), _address(v),
                        _address(q_out), q_stride, k_stride, v_stride, q_out_stride,
                        _address(q_norm), _address(k_norm), eps, rotary_dim,
                        1 if interleaved else 0, amplitude, _address(inv_freq))


class SampleParams(ctypes.Structure):
    """m1moe_sample_params: per-row settings in device memory."""

    _fields_ = [
        ("d_u", c_void_p),
        ("d_temperature", c_void_p),
        ("d_top_k", c_void_p),
        ("d_top_p", c_void_p),
        ("d_min_p", c_void_p),
    ]

    @staticmethod
    def make(u, temperature=None, top_k=None, top_p=None, min_p=None) -> "SampleParams":
        return SampleParams(_address(u), _address(temperature), _address(top_k), _address(top_p),
                            _address(min_p))


# dtypes of the on-disk manifest (m1moe_store_tensor)
DT_BF16, DT_F32, DT_U32 = 0, 1, 2

# dense tensor ids of m1moe_dec_upload
(W_EMBED, W_LM_HEAD, W_FINAL_NORM, W_IN_NORM, W_POST_NORM, W_Q, W_K, W_V, W_O, W_Q_NORM,
 W_K_NORM) = range(11)
W_PER_LAYER = (W_IN_NORM, W_POST_NORM, W_Q, W_K, W_V, W_O, W_Q_NORM, W_K_NORM)


class M1MoEError(RuntimeError):
    """A non-zero status from the C ABI, with m1moe_last_error()'s message."""

    def __init__(self, code: int, where: str, message: str):
        super().__init__(f"{where} -> status {code}: {message}")
        self.code = code
        self.where = where
        self.message = message


# (name, restype, argtypes) of every exported function of include/m1moe_hip.h
_PROTOTYPES = [
    ("m1moe_abi_version", c_int32, []),
    ("m1moe_last_error", c_char_p, []),
    ("m1moe_check_shape", c_int32, [POINTER(MoEShape)]),
    ("m1moe_expert_bytes", c_int32, [POINTER(MoEShape), POINTER(c_uint64)]),
    ("m1moe_expert_offsets", c_int32, [POINTER(MoEShape), POINTER(c_uint64)]),
    ("m1moe_decode_kernel_for", c_int32, [POINTER(MoEShape), c_int32, c_int32, POINTER(c_int32)]),
    ("m1moe_create", c_int32, [c_int32, POINTER(MoEShape), POINTER(c_void_p)]),
    ("m1moe_destroy", None, [c_void_p]),
    ("m1moe_upload_layer_experts", c_int32, [c_void_p, c_int32, c_void_p, c_uint64]),
    ("m1moe_upload_router", c_int32, [c_void_p, c_int32, POINTER(c_uint16), c_uint64]),
    ("m1moe_set_logit_bias", c_int32, [c_void_p, c_int32, POINTER(c_float), c_int32]),
    ("m1moe_expert_block", c_int32, [c_void_p, c_int32, c_int32, POINTER(c_void_p)]),
    ("m1moe_alloc", c_int32, [c_void_p, c_uint64, POINTER(c_void_p)]),
    ("m1moe_free", c_int32, [c_void_p, c_void_p]),
    ("m1moe_copy_h2d", c_int32, [c_void_p, c_void_p, c_void_p, c_uint64]),
    ("m1moe_copy_d2h", c_int32, [c_void_p, c_void_p, c_void_p, c_uint64]),
    ("m1moe_copy_d2d", c_int32, [c_void_p, c_void_p, c_void_p, c_uint64]),
    ("m1moe_set_stream", c_int32, [c_void_p, c_void_p]),
    ("m1moe_get_stream", c_int32, [c_void_p, POINTER(c_void_p)]),
    ("m1moe_sync", c_int32, [c_void_p]),
    ("m1moe_event_create", c_int32, [c_void_p, POINTER(c_void_p)]),
    ("m1moe_event_record", c_int32, [c_void_p, c_void_p]),
    ("m1moe_event_elapsed_ms", c_int32, [c_void_p, c_void_p, POINTER(c_float)]),
    ("m1moe_event_destroy", None, [c_void_p]),
    ("m1moe_graph_begin", c_int32, [c_void_p]),
    ("m1moe_graph_end", c_int32, [c_void_p, POINTER(c_void_p)]),
    ("m1moe_graph_launch", c_int32, [c_void_p, c_void_p]),
    ("m1moe_graph_destroy", None, [c_void_p]),
    ("m1moe_router_topk", c_int32,
     [c_void_p, c_int32, c_int32, c_void_p, c_int32, c_void_p, c_void_p, c_void_p]),
    ("m1moe_moe_decode", c_int32,
     [c_void_p, c_int32, c_void_p, c_int32, c_void_p, c_void_p, c_void_p, c_void_p]),
    ("m1moe_moe_decode_given_topk", c_int32,
     [c_void_p, c_int32, c_void_p, c_int32, c_void_p, c_void_p, c_void_p, c_void_p]),
    ("m1moe_moe_prefill", c_int32,
     [c_void_p, c_int32, c_int32, c_void_p, c_int32, c_void_p, c_void_p, c_void_p, c_void_p]),
    ("m1moe_moe_prefill_noalloc", c_int32,
     [c_void_p, c_int32, c_int32, c_void_p, c_int32, c_void_p, c_void_p, c_void_p, c_void_p]),
    ("m1moe_dequant_debug", c_int32, [c_void_p, c_int32, c_int32, c_int32, c_void_p]),
    ("m1moe_rmsnorm", c_int32, [c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_float]),
    ("m1moe_matvec_bf16", c_int32,
     [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_int32]),
    ("m1moe_attention_decode", c_int32,
     [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_int32, c_int32, c_int32]),
    ("m1moe_argmax", c_int32, [c_void_p, c_void_p, c_int32, c_void_p]),
    ("m1moe_dec_create", c_int32, [c_void_p, POINTER(DecShape), POINTER(c_void_p)]),
    ("m1moe_dec_destroy", None, [c_void_p]),
    ("m1moe_dec_upload", c_int32, [c_void_p, c_int32, c_int32, POINTER(c_uint16), c_uint64]),
    ("m1moe_dec_reset", c_int32, [c_void_p]),
    ("m1moe_dec_step", c_int32, [c_void_p, c_void_p, c_void_p, c_void_p]),
    ("m1moe_dec_step_seq", c_int32, [c_void_p, c_void_p, c_int32, c_int32, c_void_p]),
    ("m1moe_dec_prefill", c_int32, [c_void_p, c_void_p, c_int32, c_void_p, c_void_p]),
    ("m1moe_dec_position", c_int32, [c_void_p, POINTER(c_int32)]),
    ("m1moe_check_paged", c_int32, [POINTER(PagedKV), POINTER(PagedBatch)]),
    ("m1moe_kv_append", c_int32,
     [c_void_p, POINTER(PagedKV), POINTER(PagedBatch), POINTER(KVAppend)]),
    ("m1moe_paged_attention", c_int32,
     [c_void_p, POINTER(PagedKV), POINTER(PagedBatch), c_void_p, ctypes.c_int64, c_void_p,
      ctypes.c_int64, c_int32, c_int32]),
    ("m1moe_sample", c_int32,
     [c_void_p, c_void_p, c_int32, c_int32, ctypes.c_int64, POINTER(SampleParams), c_void_p,
      c_void_p]),
    ("m1moe_store_open", c_int32, [c_char_p, c_char_p, POINTER(c_void_p)]),
    ("m1moe_store_close", None, [c_void_p]),
    ("m1moe_store_count", c_int32, [c_void_p, POINTER(c_int32)]),
    ("m1moe_store_tensor", c_int32,
     [c_void_p, c_char_p, POINTER(c_void_p), POINTER(c_int32), POINTER(ctypes.c_int64),
      POINTER(c_int32)]),
    ("m1moe_load_model", c_int32, [c_void_p, c_void_p, c_char_p, c_int32]),
    ("m1moe_quantize_4bit", c_int32,
     [c_void_p, ctypes.c_int64, ctypes.c_int64, c_int32, c_void_p, c_void_p, c_void_p, c_int32]),
    ("m1moe_quantize_expert", c_int32,
     [POINTER(MoEShape), c_void_p, c_void_p, c_void_p, c_void_p, c_uint64, c_int32]),
    ("m1moe_f32_to_bf16", c_int32, [c_void_p, c_uint64, c_void_p]),
    ("m1moe_tokenizer_load", c_int32, [c_char_p, POINTER(c_void_p)]),
    ("m1moe_tokenizer_free", None, [c_void_p]),
    ("m1moe_tokenizer_info", c_int32,
     [c_void_p, POINTER(c_int32), POINTER(c_uint64), POINTER(c_uint64)]),
    ("m1moe_tokenizer_encode", c_int32,
     [c_void_p, c_char_p, c_uint64, c_int32, ctypes.c_uint32, c_void_p, c_uint64,
      POINTER(c_uint64)]),
    ("m1moe_tokenizer_decode", c_int32,
     [c_void_p, c_void_p, c_uint64, c_int32, c_void_p, c_uint64, POINTER(c_uint64)]),
    ("m1moe_synth_normal_bf16", c_int32,
     [c_uint64, c_uint64, c_uint64, c_float, c_int32, c_void_p]),
    ("m1moe_synth_normal_f32", c_int32, [c_uint64, c_uint64, c_uint64, c_float, c_void_p]),
    ("m1moe_synth_layer_image", c_int32,
     [POINTER(MoEShape), c_uint64, c_int32, c_float, c_float, c_void_p, c_uint64, c_int32]),
]

EXPORTED_NAMES = [p[0] for p in _PROTOTYPES]

_lib = None


def load() -> ctypes.CDLL:
    """Loads the in-tree library once; raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise ImportError(
            f"{LIB_PATH} is missing: build it with `make -C m1moe_amd/csrc` "
            "(or __graft_entry__.build()); there is no fallback implementation")
    lib = ctypes.CDLL(LIB_PATH)
    for name, restype, argtypes in _PROTOTYPES:
        fn = getattr(lib, name)
        fn.restype = restype
        fn.argtypes = argtypes
    _lib = lib
    return lib


def last_error() -> str:
    msg = load().m1moe_last_error()
    return msg.decode() if msg else ""


def check(code: int, where: str) -> None:
    """Raises M1MoEError for a non-zero status."""
    if code != M1MOE_OK:
        raise M1MoEError(code, where, last_error())
