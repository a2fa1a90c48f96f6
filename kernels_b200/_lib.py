"""ctypes binding of libcuda-graft.so (include/cuda_graft.h).

The library is the product; this module only loads it and declares argument
types.  Loading fails loudly: there is no CPU or PyTorch fallback for any entry
point.
"""
from __future__ import annotations

import ctypes as C
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent / "lib" / "libcuda-graft.so"

GRAFT_OK, GRAFT_EINVAL, GRAFT_ECUDA, GRAFT_ENCCL, GRAFT_ETIMEDOUT, GRAFT_ENOTSUP = range(6)
STATUS_NAMES = {0: "GRAFT_OK", 1: "GRAFT_EINVAL", 2: "GRAFT_ECUDA", 3: "GRAFT_ENCCL",
                4: "GRAFT_ETIMEDOUT", 5: "GRAFT_ENOTSUP"}


class GemvParams(C.Structure):
    """GemvParams, int4-gemv/src/kernels.metal:42-49."""
    _fields_ = [("M", C.c_uint32), ("K", C.c_uint32), ("G", C.c_uint32),
                ("words_pr", C.c_uint32), ("groups_pr", C.c_uint32), ("chunks_pg", C.c_uint32)]


class VQParams(C.Structure):
    """VQParams, vq-gemv/src/kernels.metal:32-37."""
    _fields_ = [("M", C.c_uint32), ("K", C.c_uint32), ("chunks_pr", C.c_uint32),
                ("cb_size", C.c_uint32)]


class VQQuantParams(C.Structure):
    """GraftVQQuantParams: the quantiser's shape, passes, sample size and seed."""
    _fields_ = [("M", C.c_uint32), ("K", C.c_uint32), ("iters", C.c_uint32),
                ("sub", C.c_uint32), ("seed", C.c_uint64)]


class MoEParams(C.Structure):
    """MoEParams, moe-fused/src/kernels.metal:22-35 (u64 block at byte 40)."""
    _fields_ = [("hidden", C.c_uint32), ("inter", C.c_uint32), ("n_experts", C.c_uint32),
                ("top_k", C.c_uint32), ("quads_hid", C.c_uint32), ("quads_int", C.c_uint32),
                ("groups_hid", C.c_uint32), ("groups_int", C.c_uint32),
                ("chunks_pg", C.c_uint32),
                ("blob", C.c_uint64), ("off_gate", C.c_uint64), ("off_up", C.c_uint64),
                ("off_down", C.c_uint64), ("sub_w", C.c_uint64), ("sub_s", C.c_uint64),
                ("sub_b", C.c_uint64), ("sub_bi", C.c_uint64)]


class MoEFormat(C.Structure):
    _fields_ = [("scale_f16", C.c_uint32), ("has_bias_out", C.c_uint32),
                ("act_f16", C.c_uint32), ("y_f16", C.c_uint32),
                ("expert_lo", C.c_uint32), ("expert_hi", C.c_uint32)]


class MoEScratch(C.Structure):
    _fields_ = [("idx", C.c_void_p), ("wgt", C.c_void_p), ("local", C.c_void_p),
                ("xh", C.c_void_p), ("h", C.c_void_p), ("xsh", C.c_void_p),
                ("ypart", C.c_void_p), ("sync", C.c_void_p)]


class ExpertParams(C.Structure):
    """ExpertParams, moe-pipeline/src/main.mm:53."""
    _fields_ = [("M", C.c_uint32), ("K", C.c_uint32), ("G", C.c_uint32),
                ("quads_pr", C.c_uint32), ("groups_pr", C.c_uint32), ("chunks_pg", C.c_uint32)]


class ExpertScratch(C.Structure):
    _fields_ = [("xs_x", C.c_void_p), ("gate", C.c_void_p), ("up", C.c_void_p),
                ("h", C.c_void_p), ("xs_h", C.c_void_p)]


class KVCacheDesc(C.Structure):
    """GraftKVCache: codes and scales of a paged 8-bit key/value cache."""
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_scale", C.c_void_p),
                ("v_scale", C.c_void_p), ("n_blocks", C.c_uint32), ("kv_heads", C.c_uint32),
                ("block_tokens", C.c_uint32), ("head_dim", C.c_uint32), ("format", C.c_uint32)]


class KVRangeDesc(C.Structure):
    """GraftKVRange: consecutive tokens of each sequence, and where they are."""
    _fields_ = [("block_table", C.c_void_p), ("start", C.c_void_p), ("cu_tokens", C.c_void_p),
                ("n_seqs", C.c_uint32), ("table_stride", C.c_uint32),
                ("max_tokens", C.c_uint32), ("max_len", C.c_uint32)]


class Heads(C.Structure):
    """GraftHeads: a strided [tokens][heads][head_dim] buffer."""
    _fields_ = [("data", C.c_void_p), ("token_stride", C.c_uint64), ("head_stride", C.c_uint64),
                ("tokens", C.c_uint32), ("dtype", C.c_uint32)]


class AttnParams(C.Structure):
    _fields_ = [("q_heads", C.c_uint32), ("window", C.c_uint32), ("scale", C.c_float)]


class LogprobParams(C.Structure):
    _fields_ = [("rows", C.c_uint32), ("vocab", C.c_uint32), ("top_k", C.c_uint32),
                ("dtype", C.c_uint32), ("row_stride", C.c_uint64), ("scale", C.c_float)]


P = C.c_void_p
U32 = C.c_uint32
U64 = C.c_uint64
INT = C.c_int
SIZE = C.c_size_t

# name -> (restype, argtypes); every name here is declared in include/cuda_graft.h
SIGNATURES: dict[str, tuple] = {
    "graft_last_error_string": (C.c_char_p, []),
    "graft_version": (C.c_char_p, []),
    "graft_gemv_params": (INT, [U32, U32, U32, C.POINTER(GemvParams)]),
    "graft_xsum32": (INT, [P, P, C.POINTER(GemvParams), P]),
    "graft_gemv_int4_wide_unroll": (INT, [P, P, P, P, P, P, C.POINTER(GemvParams), P]),
    "graft_gemv_int4_simd": (INT, [P, P, P, P, P, P, C.POINTER(GemvParams), P]),
    "graft_gemv_int4_sb_f16out": (INT, [P, P, P, P, C.POINTER(GemvParams), P]),
    "graft_stream_read": (INT, [P, P, U64, P]),
    "graft_gemm_int4_sb_f16": (INT, [P, P, P, P, U32, C.POINTER(GemvParams), P]),
    "graft_expert_params": (INT, [U32, U32, U32, C.POINTER(ExpertParams)]),
    "graft_xsum32_f32": (INT, [P, P, C.POINTER(ExpertParams), P]),
    "graft_gemv_int4_bf16": (INT, [P, P, P, P, P, P, P, C.POINTER(ExpertParams), P]),
    "graft_expert_stream_create": (INT, [P, U32, U64, C.POINTER(P)]),
    "graft_expert_stream_destroy": (INT, [P]),
    "graft_expert_stream_slot": (P, [P, U32]),
    "graft_expert_stream_fetch": (INT, [P, U32, P]),
    "graft_expert_stream_acquire": (INT, [P, U32, P]),
    "graft_expert_stream_release": (INT, [P, U32, P]),
    "graft_expert_stream_sync": (INT, [P]),
    "graft_expert_forward": (INT, [P, P, P, C.POINTER(MoEParams), C.POINTER(ExpertScratch), P]),
    "graft_device_errors": (INT, [C.POINTER(U32), INT]),
    "graft_set_gemv_engine": (INT, [INT]),
    "graft_get_gemv_engine": (INT, []),
    "graft_gemv_vq_wide": (INT, [P, P, P, P, P, C.POINTER(VQParams), P]),
    "graft_gemv_vq_ex": (INT, [P, P, P, U32, P, P, INT, C.POINTER(VQParams), P]),
    "graft_vq_decode": (INT, [P, P, P, U64, P]),
    "graft_vq_quantize_workspace": (U64, [C.POINTER(VQQuantParams)]),
    "graft_vq_quantize": (INT, [P, P, P, P, C.POINTER(VQQuantParams), P, U64, P]),
    "graft_moe_params": (INT, [U32, U32, U32, U32, C.POINTER(MoEParams)]),
    "graft_moe_router_topk": (INT, [P, P, P, P, C.POINTER(MoEParams), P, P, P]),
    "graft_moe_fused_gate_up_swiglu": (INT, [P, P, P, P, C.POINTER(MoEParams), P]),
    "graft_moe_fused_down_combine": (INT, [P, P, P, P, P, C.POINTER(MoEParams), P]),
    "graft_moe_fused_gate_up_swiglu_at": (INT, [P, P, P, P, C.POINTER(MoEParams), P, P]),
    "graft_moe_fused_down_combine_at": (INT, [P, P, P, P, P, C.POINTER(MoEParams), P, P]),
    "graft_moe_scratch_bytes": (SIZE, [C.POINTER(MoEParams)]),
    "graft_moe_scratch_carve": (INT, [P, SIZE, C.POINTER(MoEParams), C.POINTER(MoEScratch)]),
    "graft_moe_set_one_launch": (INT, [INT]),
    "graft_moe_set_down_pass": (INT, [INT]),
    "graft_gemm_set_tcgen05": (INT, [INT]),
    "graft_moe_scratch_init": (INT, [C.POINTER(MoEParams), C.POINTER(MoEScratch), P]),
    "graft_moe_block": (INT, [P, P, P, P, C.POINTER(MoEParams), C.POINTER(MoEScratch), P]),
    "graft_moe_block_ex": (INT, [P, P, P, P, C.POINTER(MoEParams), C.POINTER(MoEFormat),
                                 C.POINTER(MoEScratch), P]),
    "graft_moe_block_noalloc": (INT, [P, P, P, P, C.POINTER(MoEParams), C.POINTER(MoEFormat),
                                      P]),
    "graft_comm_get_unique_id": (INT, [P]),
    "graft_comm_init": (INT, [C.POINTER(P), P, INT, INT]),
    "graft_comm_destroy": (INT, [P]),
    "graft_comm_info": (INT, [P, C.POINTER(INT), C.POINTER(INT)]),
    "graft_comm_alloc": (INT, [P, SIZE, C.POINTER(P)]),
    "graft_comm_free": (INT, [P, P]),
    "graft_comm_fused": (INT, [P]),
    "graft_comm_set_fused": (INT, [P, INT]),
    "graft_comm_status": (INT, [P]),
    "graft_comm_set_wait_limit": (INT, [P, U64]),
    "graft_gemv_int4_sharded": (INT, [P, P, P, P, P, C.POINTER(GemvParams), P]),
    "graft_gemm_int4_sharded": (INT, [P, P, P, P, P, U32, C.POINTER(GemvParams), P]),
    "graft_moe_block_ep": (INT, [P, P, P, P, P, C.POINTER(MoEParams), C.POINTER(MoEFormat),
                                 C.POINTER(MoEScratch), P]),
    "graft_kv_write": (INT, [C.POINTER(KVCacheDesc), C.POINTER(Heads), C.POINTER(Heads),
                             C.POINTER(KVRangeDesc), P]),
    "graft_kv_read": (INT, [C.POINTER(KVCacheDesc), C.POINTER(Heads), C.POINTER(Heads),
                            C.POINTER(KVRangeDesc), P]),
    "graft_kv_device_errors": (INT, [C.POINTER(U32), INT]),
    "graft_attn_kv8_workspace": (SIZE, [C.POINTER(KVCacheDesc), C.POINTER(KVRangeDesc),
                                        C.POINTER(AttnParams)]),
    "graft_attn_kv8_init": (INT, [P, SIZE, P]),
    "graft_attn_kv8": (INT, [C.POINTER(KVCacheDesc), C.POINTER(Heads), C.POINTER(Heads),
                             C.POINTER(KVRangeDesc), P, P, C.POINTER(AttnParams), P, SIZE, P]),
    "graft_logprobs_workspace": (SIZE, [C.POINTER(LogprobParams)]),
    "graft_logprobs_init": (INT, [P, SIZE, P]),
    "graft_logprobs": (INT, [P, P, P, P, P, P, C.POINTER(LogprobParams), P, SIZE, P]),
}

_lib: C.CDLL | None = None


def load() -> C.CDLL:
    """Loads the in-tree library once; raises if it is missing or incomplete."""
    global _lib
    if _lib is not None:
        return _lib
    if not LIB_PATH.exists():
        raise RuntimeError(
            f"{LIB_PATH} is missing: build it with `python -m kernels_b200.build` "
            "(there is no fallback implementation)")
    lib = C.CDLL(str(LIB_PATH))
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)  # AttributeError = the library lacks a declared symbol
        fn.restype = res
        fn.argtypes = args
    _lib = lib
    return lib


class GraftError(RuntimeError):
    def __init__(self, fn: str, code: int, msg: str):
        super().__init__(f"{fn}: {STATUS_NAMES.get(code, code)}: {msg}")
        self.code = code


def call(name: str, *args):
    lib = _lib or load()
    rc = getattr(lib, name)(*args)
    if rc != GRAFT_OK:
        raise GraftError(name, rc, lib.graft_last_error_string().decode())
    return rc
