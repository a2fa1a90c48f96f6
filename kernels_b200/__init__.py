"""kernels_b200 -- B200 (sm_100a) decode hot path of agastya-choudhary123/kernels.

Host-side mirror of the reference's kernel interface over libcuda-graft.so:
each function below has the name of the Metal kernel it replaces and takes its
buffers in the kernel's [[buffer(i)]] order (params struct included), e.g.

    P = gemv_params(M, K, G)                        # GemvParams
    xsum32(x, xs, P)                                # int4-gemv/src/kernels.metal:54
    gemv_int4_wide_unroll(W, SB, None, x, y, xs, P) # int4-gemv/src/kernels.metal:399

Buffers are device tensors (anything with .data_ptr()) or raw device
addresses (int).  Work is enqueued on the current torch CUDA stream unless a
stream handle is given.  A non-zero library status raises GraftError.  There is
no CPU fallback: if the library is missing, every call raises.
"""
from __future__ import annotations

import ctypes as C

from ._lib import (AttnParams, ExpertParams, ExpertScratch, GemvParams, GraftError, Heads,
                   KVCacheDesc, KVRangeDesc, LogprobParams, MoEFormat, MoEParams, MoEScratch,
                   VQParams, VQQuantParams, call, load)

__all__ = [
    "GemvParams", "VQParams", "MoEParams", "MoEFormat", "MoEScratch", "GraftError",
    "load", "version", "gemv_params", "xsum32", "gemv_int4_wide_unroll", "gemv_int4_fused",
    "gemv_int4_simd", "gemv_int4_sb_f16out", "gemm_int4_sb_f16", "gemm_int4_sharded", "stream_read", "set_gemv_engine", "get_gemv_engine",
    "device_errors",
    "ENGINE_TENSOR", "ENGINE_CUDA_CORE", "expert_params", "xsum32_f32", "gemv_int4_bf16",
    "ExpertScratchBuffers", "expert_forward", "ExpertStream", "vq_params", "gemv_vq_wide",
    "gemv_vq_ex", "vq_decode", "vq_quantize", "moe_params", "moe_router_topk", "moe_fused_gate_up_swiglu",
    "moe_fused_down_combine", "moe_fused_gate_up_swiglu_at", "moe_fused_down_combine_at",
    "MoEWorkspace", "moe_block", "moe_block_ex", "moe_format",
    "KVCache", "kv_range", "kv_write", "kv_read", "kv_device_errors", "AttnParams",
    "attn_params", "AttnWorkspace", "attn_kv8", "LogprobParams", "logprob_params",
    "LogprobWorkspace", "logprobs",
]


def _p(t) -> int | None:
    if t is None:
        return None
    if isinstance(t, int):
        return t
    return t.data_ptr()


def _s(stream) -> int | None:
    if stream is not None:
        return stream if isinstance(stream, int) else stream.cuda_stream
    import torch
    return torch.cuda.current_stream().cuda_stream


def version() -> str:
    return load().graft_version().decode()


# ------------------------------------------------------------------- int4 --
def gemv_params(M: int, K: int, G: int) -> GemvParams:
    P = GemvParams()
    call("graft_gemv_params", M, K, G, C.byref(P))
    return P


def xsum32(x, xs, P: GemvParams, stream=None) -> None:
    call("graft_xsum32", _p(x), _p(xs), C.byref(P), _s(stream))


def gemv_int4_wide_unroll(W, SB, unused, x, y, xs, P: GemvParams, stream=None) -> None:
    call("graft_gemv_int4_wide_unroll", _p(W), _p(SB), _p(unused), _p(x), _p(y), _p(xs),
         C.byref(P), _s(stream))


gemv_int4_fused = gemv_int4_wide_unroll   # v4 computes the same y from the same buffers


def gemv_int4_simd(W, S, B, x, y, xs, P: GemvParams, stream=None) -> None:
    call("graft_gemv_int4_simd", _p(W), _p(S), _p(B), _p(x), _p(y), _p(xs), C.byref(P),
         _s(stream))


def gemv_int4_sb_f16out(W, SB, x, y, P: GemvParams, stream=None) -> None:
    call("graft_gemv_int4_sb_f16out", _p(W), _p(SB), _p(x), _p(y), C.byref(P), _s(stream))


def gemm_int4_sb_f16(W, SB, X, Y, B: int, P: GemvParams, stream=None) -> None:
    """The int4 GEMV for B = 1..16 tokens at once: X fp16 [B][K], Y fp16 [B][M]."""
    call("graft_gemm_int4_sb_f16", _p(W), _p(SB), _p(X), _p(Y), B, C.byref(P), _s(stream))


def stream_read(src, sink, nquads: int, stream=None) -> None:
    call("graft_stream_read", _p(src), _p(sink), nquads, _s(stream))


# --------------------------------------------------------------------- VQ --
ENGINE_TENSOR, ENGINE_CUDA_CORE = 0, 1
_ENGINES = {"tensor": ENGINE_TENSOR, "cuda-core": ENGINE_CUDA_CORE}


def set_gemv_engine(engine) -> None:
    """Selects the engine of the dense GEMVs (int4 and VQ), process-wide:
    "tensor" (default: TMA-fed mma.sync tiles) or "cuda-core" (register-direct
    fp32 FMAs, no tensor cores)."""
    call("graft_set_gemv_engine", _ENGINES.get(engine, engine))


def device_errors(clear: bool = False) -> dict:
    """The kernels' device-side error bits (graft_device_errors), per kernel file."""
    b = C.c_uint32()
    call("graft_device_errors", C.byref(b), int(clear))
    v = b.value
    return {"int4": v & 0xFF, "vq": (v >> 8) & 0xFF, "moe": (v >> 16) & 0xFF}


def get_gemv_engine() -> str:
    e = load().graft_get_gemv_engine()
    return {v: k for k, v in _ENGINES.items()}[e]


def expert_params(M: int, K: int, G: int) -> ExpertParams:
    P = ExpertParams()
    call("graft_expert_params", M, K, G, C.byref(P))
    return P


def xsum32_f32(x, xs, P: ExpertParams, stream=None) -> None:
    call("graft_xsum32_f32", _p(x), _p(xs), C.byref(P), _s(stream))


def gemv_int4_bf16(W, S, B, BI, x, y, xs, P: ExpertParams, stream=None) -> None:
    """gemv_int4_bf16 (moe-pipeline/src/kernels.metal:53-83), buffers in the reference's order."""
    call("graft_gemv_int4_bf16", _p(W), _p(S), _p(B), _p(BI), _p(x), _p(y), _p(xs), C.byref(P),
         _s(stream))


class ExpertScratchBuffers:
    """fp32 scratch of expert_forward, owned by torch."""

    def __init__(self, P: MoEParams, device="cuda"):
        import torch
        f = dict(dtype=torch.float32, device=device)
        self.xs_x = torch.empty(P.hidden // 32, **f)
        self.gate = torch.empty(P.inter, **f)
        self.up = torch.empty(P.inter, **f)
        self.h = torch.empty(P.inter, **f)
        self.xs_h = torch.empty(P.inter // 32, **f)
        self.s = ExpertScratch(_p(self.xs_x), _p(self.gate), _p(self.up), _p(self.h),
                               _p(self.xs_h))


def expert_forward(blob, x, y, P: MoEParams, scratch: ExpertScratchBuffers, stream=None) -> None:
    """One expert (encode_expert, moe-pipeline/src/main.mm:201-239); blob is a device
    tensor or address holding one experts.bin blob."""
    call("graft_expert_forward", blob if isinstance(blob, int) else _p(blob), _p(x), _p(y),
         C.byref(P), C.byref(scratch.s), _s(stream))


class ExpertStream:
    """Slots of device memory filled from pinned host memory on a side stream
    (graft_expert_stream_*)."""

    def __init__(self, slots, n_slots: int, blob: int):
        self._slots = slots
        self.n_slots, self.blob = n_slots, blob
        h = C.c_void_p()
        call("graft_expert_stream_create", _p(slots), n_slots, blob, C.byref(h))
        self._h = h

    def slot(self, s: int) -> int:
        return load().graft_expert_stream_slot(self._h, s)

    def fetch(self, s: int, host_blob) -> None:
        call("graft_expert_stream_fetch", self._h, s,
             host_blob if isinstance(host_blob, int) else _p(host_blob))

    def acquire(self, s: int, stream=None) -> None:
        call("graft_expert_stream_acquire", self._h, s, _s(stream))

    def release(self, s: int, stream=None) -> None:
        call("graft_expert_stream_release", self._h, s, _s(stream))

    def sync(self) -> None:
        call("graft_expert_stream_sync", self._h)

    def close(self) -> None:
        if self._h:
            call("graft_expert_stream_destroy", self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def vq_params(M: int, K: int, cb_size: int = 256) -> VQParams:
    return VQParams(M, K, K // 32, cb_size)


def gemv_vq_wide(IDX, Cb, S, x, y, P: VQParams, stream=None) -> None:
    call("graft_gemv_vq_wide", _p(IDX), _p(Cb), _p(S), _p(x), _p(y), C.byref(P), _s(stream))


def gemv_vq_ex(IDX, Cb, S, scale_group: int, x, y, P: VQParams, stream=None) -> None:
    import torch
    y_f16 = int(getattr(y, "dtype", None) == torch.float16)
    call("graft_gemv_vq_ex", _p(IDX), _p(Cb), _p(S), scale_group, _p(x), _p(y), y_f16,
         C.byref(P), _s(stream))


def vq_decode(IDX, Cb, out, n_idx: int, stream=None) -> None:
    call("graft_vq_decode", _p(IDX), _p(Cb), _p(out), n_idx, _s(stream))


def vq_quantize(W, iters: int = 25, sub: int = 200_000, seed: int = 0, stream=None):
    """The VQ quantiser (vq-gemv/quant/pq_quantize.py:50-75) on the GPU: W fp32
    [M, K] (device) -> (IDX uint8 [M, K/2], C fp16 [256, 2], S fp16 [M, K/32])."""
    import torch
    M, K = W.shape
    P = VQQuantParams(M, K, iters, sub, seed)
    nbytes = load().graft_vq_quantize_workspace(C.byref(P))
    if nbytes == 0:
        raise GraftError("graft_vq_quantize_workspace", 1,
                         f"bad parameters (M={M} K={K} sub={sub})")
    ws = torch.empty(nbytes, dtype=torch.uint8, device=W.device)
    IDX = torch.empty((M, K // 2), dtype=torch.uint8, device=W.device)
    Cb = torch.empty((256, 2), dtype=torch.float16, device=W.device)
    S = torch.empty((M, K // 32), dtype=torch.float16, device=W.device)
    call("graft_vq_quantize", _p(W), _p(IDX), _p(Cb), _p(S), C.byref(P), _p(ws), nbytes,
         _s(stream))
    return IDX, Cb, S


# -------------------------------------------------------------------- MoE --
def moe_params(hidden: int, inter: int, n_experts: int, top_k: int) -> MoEParams:
    P = MoEParams()
    call("graft_moe_params", hidden, inter, n_experts, top_k, C.byref(P))
    return P


def moe_format(scale_f16=False, has_bias_out=True, act_f16=False, y_f16=False,
               expert_lo=0, expert_hi=None, n_experts=None) -> MoEFormat:
    hi = expert_hi if expert_hi is not None else (n_experts if n_experts is not None else 256)
    return MoEFormat(int(scale_f16), int(has_bias_out), int(act_f16), int(y_f16),
                     expert_lo, hi)


def moe_router_topk(R, x, idx, wgt, P: MoEParams, xsh, xh, stream=None) -> None:
    call("graft_moe_router_topk", _p(R), _p(x), _p(idx), _p(wgt), C.byref(P), _p(xsh), _p(xh),
         _s(stream))


def moe_fused_gate_up_swiglu(pool, idx, xh, h, P: MoEParams, stream=None) -> None:
    call("graft_moe_fused_gate_up_swiglu", _p(pool), _p(idx), _p(xh), _p(h), C.byref(P),
         _s(stream))


def moe_fused_down_combine(pool, idx, wgt, h, y, P: MoEParams, stream=None) -> None:
    call("graft_moe_fused_down_combine", _p(pool), _p(idx), _p(wgt), _p(h), _p(y), C.byref(P),
         _s(stream))


def moe_fused_gate_up_swiglu_at(pool, idx, xh, h, P: MoEParams, xsh, stream=None) -> None:
    call("graft_moe_fused_gate_up_swiglu_at", _p(pool), _p(idx), _p(xh), _p(h), C.byref(P),
         _p(xsh), _s(stream))


def moe_fused_down_combine_at(pool, idx, wgt, h, y, P: MoEParams, xsh, stream=None) -> None:
    call("graft_moe_fused_down_combine_at", _p(pool), _p(idx), _p(wgt), _p(h), _p(y),
         C.byref(P), _p(xsh), _s(stream))


class MoEWorkspace:
    """One device buffer carved into the scratch the three MoE kernels share
    (selected experts, weights, resident-expert list, fp16 x, h, sum(h))."""

    def __init__(self, P: MoEParams, device=None):
        import torch
        n = load().graft_moe_scratch_bytes(C.byref(P))
        self.buffer = torch.empty(n + 256, dtype=torch.uint8, device=device or "cuda")
        base = (self.buffer.data_ptr() + 255) & ~255
        self.scratch = MoEScratch()
        call("graft_moe_scratch_carve", base, n, C.byref(P), C.byref(self.scratch))
        # the one-launch block's tagged words start from zero (on the current stream)
        call("graft_moe_scratch_init", C.byref(P), C.byref(self.scratch),
             _s(torch.cuda.current_stream()))
        self.P = P

    def tensor(self, name: str, dtype, numel: int):
        """A view of one scratch field (idx, wgt, local, xh, h, xsh) as a tensor."""
        import torch
        addr = getattr(self.scratch, name)
        off = addr - self.buffer.data_ptr()
        nbytes = numel * torch.empty((), dtype=dtype).element_size()
        return self.buffer[off:off + nbytes].view(dtype)


def moe_block(pool, R, x, y, P: MoEParams, ws: MoEWorkspace, stream=None) -> None:
    call("graft_moe_block", _p(pool), _p(R), _p(x), _p(y), C.byref(P), C.byref(ws.scratch),
         _s(stream))


def moe_block_ex(pool, R, x, y, P: MoEParams, fmt: MoEFormat | None, ws: MoEWorkspace,
                 stream=None) -> None:
    call("graft_moe_block_ex", _p(pool), _p(R), _p(x), _p(y), C.byref(P),
         C.byref(fmt) if fmt is not None else None, C.byref(ws.scratch), _s(stream))


def gemm_set_tcgen05(on: bool) -> bool:
    """Whether graft_gemm_int4_sb_f16 runs 9..16 tokens on the tcgen05 kernel
    or (the default) keeps every shape on the mma.sync tile engine; returns
    the previous setting."""
    return bool(load().graft_gemm_set_tcgen05(1 if on else 0))


def moe_set_down_pass(split: bool) -> bool:
    """The block's down pass on every SM without clusters (True) or as
    clusters of top_k CTAs (False, the default); returns the previous setting."""
    return bool(load().graft_moe_set_down_pass(1 if split else 0))


def moe_set_one_launch(on) -> int:
    """Where the MoE block runs as one launch instead of three: True/1 the
    whole block on one GPU, 2 a rank's share of an expert-parallel block, 3
    both, False/0 neither.  Returns the previous setting (the same bits)."""
    return int(load().graft_moe_set_one_launch(int(on)))


# ------------------------------------------ key/value cache and attention --
# (these calls take a few microseconds on the GPU in a decode step, so the host
# side keeps to what each call needs)
_DTYPES: dict = {}


def _dtype_code(dtype) -> int:
    if not _DTYPES:
        import torch
        _DTYPES.update({torch.float16: 0, torch.bfloat16: 1, torch.float32: 2})
    code = _DTYPES.get(dtype)
    if code is None:
        raise TypeError(f"unsupported element type {dtype}")
    return code


_RAW_STREAM: list = []


def _raw_stream(stream, dev: int) -> int:
    """_s() without a Stream object for the usual case, the current stream; the
    tensors' device must be the current one."""
    if dev < 0:
        raise ValueError("the tensors must be on a GPU")
    if not _RAW_STREAM:
        import torch
        torch.cuda.current_stream()      # (CUDA is initialised from here on)
        try:
            _RAW_STREAM.extend((torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice))
        except AttributeError:
            _RAW_STREAM.extend((lambda d: torch.cuda.current_stream(d).cuda_stream,
                                torch.cuda.current_device))
    now = _RAW_STREAM[1]()
    if now != dev:
        raise ValueError(f"the tensors are on cuda:{dev}, the current device is cuda:{now}")
    if stream is not None:
        return stream if isinstance(stream, int) else stream.cuda_stream
    return _RAW_STREAM[0](now)


def _ints(t, name: str):
    import torch
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32, not {t.dtype}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name} must be contiguous")
    return t


def _elsewhere(t, dev: int):
    raise ValueError(f"expected a tensor on {f'cuda:{dev}' if dev >= 0 else 'the CPU'}, "
                     f"not on {t.device}")


def _one_device(*tensors) -> int:
    """The GPU that all of them are on; -1 for the CPU (calls refuse it)."""
    dev = tensors[0].get_device()
    for t in tensors:
        if t.get_device() != dev:
            _elsewhere(t, dev)
    return dev


def _heads(t, heads: int, dim: int, dev: int) -> Heads:
    """A [tokens, heads, dim] tensor with any token and head strides."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 3 or shape[1] != heads or shape[2] != dim:
        raise ValueError(f"expected a [tokens, {heads}, {dim}] tensor, not {tuple(shape)}")
    if stride[2] != 1 and dim > 1:
        raise ValueError("the last dimension must be contiguous")
    code = _dtype_code(t.dtype)
    if t.get_device() != dev:
        _elsewhere(t, dev)
    # (the stride of a single token or head is any number)
    return Heads(t.data_ptr(), stride[0] if shape[0] > 1 else 0, stride[1] if heads > 1 else 0,
                 shape[0], code)


def _dense(t, dtype, shape, dev: int) -> int | None:
    """The address of a contiguous tensor of that type and shape; None for None."""
    if t is None:
        return None
    if t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"expected a contiguous {dtype} {tuple(shape)} tensor")
    if t.get_device() != dev:
        _elsewhere(t, dev)
    return t.data_ptr()


class KVCache:
    """A paged 8-bit key/value cache over the caller's tensors: k and v int8 or
    float8_e4m3fn [n_blocks, kv_heads, block_tokens, head_dim], k_scale and
    v_scale fp32 [n_blocks, kv_heads], all contiguous."""

    def __init__(self, k, v, k_scale, v_scale):
        import torch
        formats = {torch.int8: 0, torch.float8_e4m3fn: 1}
        if k.dtype not in formats or v.dtype != k.dtype:
            raise TypeError("k and v must both be int8 or both float8_e4m3fn")
        if k.dim() != 4 or v.shape != k.shape:
            raise ValueError("k and v must be [n_blocks, kv_heads, block_tokens, head_dim]")
        for s in (k_scale, v_scale):
            if s.dtype != torch.float32 or s.shape != k.shape[:2]:
                raise ValueError("scales must be fp32 [n_blocks, kv_heads]")
        if not all(t.is_contiguous() for t in (k, v, k_scale, v_scale)):
            raise ValueError("the cache's tensors must be contiguous")
        self.dev = _one_device(k, v, k_scale, v_scale)
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        n, h, bt, d = k.shape
        self.desc = KVCacheDesc(_p(k), _p(v), _p(k_scale), _p(v_scale), n, h, bt, d,
                                formats[k.dtype])
        self.ref, self.heads, self.dim, self.block_tokens = C.byref(self.desc), h, d, bt

    @classmethod
    def empty(cls, n_blocks: int, kv_heads: int, head_dim: int, block_tokens: int = 64,
              dtype=None, device="cuda"):
        """A new cache (dtype torch.int8, the default, or torch.float8_e4m3fn)."""
        import torch
        shape = (n_blocks, kv_heads, block_tokens, head_dim)
        k, v = (torch.zeros(shape, dtype=torch.int8, device=device).view(dtype or torch.int8)
                for _ in range(2))
        ks, vs = (torch.zeros(shape[:2], dtype=torch.float32, device=device) for _ in range(2))
        return cls(k, v, ks, vs)


class KVRange:
    """Consecutive tokens of each sequence (kv_range)."""

    def __init__(self, block_table, start, cu_tokens, max_tokens: int, max_len: int):
        if block_table.dim() != 2:
            raise ValueError("block_table must be [n_seqs, blocks]")
        n = block_table.shape[0]
        if tuple(start.shape) != (n,) or tuple(cu_tokens.shape) != (n + 1,):
            raise ValueError("start must be [n_seqs] and cu_tokens [n_seqs + 1]")
        self._keep = (_ints(block_table, "block_table"), _ints(start, "start"),
                      _ints(cu_tokens, "cu_tokens"))
        self.dev = _one_device(block_table, start, cu_tokens)
        stride = block_table.stride(0) if n > 1 else block_table.shape[1]
        self.desc = KVRangeDesc(_p(block_table), _p(start), _p(cu_tokens), n, stride, max_tokens,
                                max_len)
        # (a row may be a slice of a wider table: the library sees only its stride)
        self.blocks, self.max_len = block_table.shape[1] if n else 1 << 31, max_len
        self.ref = C.byref(self.desc)


def kv_range(block_table, start, cu_tokens, max_tokens: int, max_len: int) -> KVRange:
    """Tokens at positions start[b] .. of each sequence b: as many as cu_tokens
    (int32 [n_seqs + 1], running sums from 0) says, in the blocks that
    block_table (int32 [n_seqs, blocks]) names.  max_tokens and max_len bound a
    sequence's tokens in the range and its last position + 1."""
    return KVRange(block_table, start, cu_tokens, max_tokens, max_len)


def _bad_range(cache: KVCache, rng: KVRange):
    if rng.dev != cache.dev:
        raise ValueError("the cache and the range are on different devices")
    raise ValueError(f"a block table of {rng.blocks} blocks of {cache.block_tokens} tokens a "
                     f"sequence does not hold max_len {rng.max_len}")


def _kv_move(name: str, cache: KVCache, K, V, rng: KVRange, stream) -> None:
    h, d, dev = cache.heads, cache.dim, cache.dev
    K, V = _heads(K, h, d, dev), _heads(V, h, d, dev)
    if rng.dev != dev or rng.blocks * cache.block_tokens < rng.max_len:
        _bad_range(cache, rng)
    call(name, cache.ref, C.byref(K), C.byref(V), rng.ref, _raw_stream(stream, dev))


def kv_write(cache: KVCache, K, V, rng: KVRange, stream=None) -> None:
    """Quantises K and V [tokens, kv_heads, head_dim] into the cache (graft_kv_write)."""
    _kv_move("graft_kv_write", cache, K, V, rng, stream)


def kv_read(cache: KVCache, K, V, rng: KVRange, stream=None) -> None:
    """Reads the range back into K and V [tokens, kv_heads, head_dim] (graft_kv_read)."""
    _kv_move("graft_kv_read", cache, K, V, rng, stream)


def kv_device_errors(clear: bool = False) -> dict:
    """Findings of the cache and attention kernels (graft_kv_device_errors)."""
    b = C.c_uint32()
    call("graft_kv_device_errors", C.byref(b), int(clear))
    return {"block": bool(b.value & 1), "bounds": bool(b.value & 2), "wait": bool(b.value & 4)}


def attn_params(q_heads: int, dtype=None, scale: float = 1.0, window: int = 0) -> AttnParams:
    """dtype: the queries' type, torch.float16 or torch.bfloat16 (checked here;
    the call goes by the tensors)."""
    if dtype is not None and _dtype_code(dtype) > 1:
        raise TypeError("queries are fp16 or bf16")
    return AttnParams(q_heads, window, scale)


def _scratch(n: int, init: str, device):
    """A zeroed workspace of n bytes: buffer, 256-byte aligned address, device."""
    import torch
    buffer = torch.empty(n + 256, dtype=torch.uint8, device=device)
    addr, dev = (buffer.data_ptr() + 255) & ~255, buffer.get_device()
    call(init, addr, n, _raw_stream(None, dev))
    return buffer, addr, dev


class AttnWorkspace:
    """The scratch of attn_kv8 for a cache, a range's bounds and params."""

    def __init__(self, cache: KVCache, rng: KVRange, P: AttnParams, device=None):
        n = load().graft_attn_kv8_workspace(C.byref(cache.desc), C.byref(rng.desc), C.byref(P))
        if n == 0:
            raise GraftError("graft_attn_kv8_workspace", 1,
                             load().graft_last_error_string().decode())
        self.buffer, self.addr, self.dev = _scratch(n, "graft_attn_kv8_init", device or cache.k.device)
        self.nbytes = n


def attn_kv8(cache: KVCache, q, out, rng: KVRange, P: AttnParams, ws: AttnWorkspace, sinks=None,
             lse=None, stream=None) -> None:
    """Attention of the range's tokens (q and out [tokens, q_heads, head_dim])
    over the cache (graft_attn_kv8)."""
    d, hq, dev = cache.dim, P.q_heads, cache.dev
    if sinks is not None or lse is not None:
        from torch import float32
        sinks, lse = (_dense(sinks, float32, (hq,), dev),
                      _dense(lse, float32, (q.shape[0], hq), dev))
    q, out = _heads(q, hq, d, dev), _heads(out, hq, d, dev)
    if rng.dev != dev or rng.blocks * cache.block_tokens < rng.max_len:
        _bad_range(cache, rng)
    if ws.dev != dev:
        raise ValueError("the workspace is on another device than the tensors")
    call("graft_attn_kv8", cache.ref, C.byref(q), C.byref(out), rng.ref, sinks, lse, C.byref(P),
         ws.addr, ws.nbytes, _raw_stream(stream, dev))


# ------------------------------------------------------ log probabilities --
def logprob_params(rows: int, vocab: int, top_k: int, dtype, scale: float = 1.0) -> LogprobParams:
    return LogprobParams(rows, vocab, top_k, _dtype_code(dtype), vocab, scale)


class LogprobWorkspace:
    """The scratch of logprobs."""

    def __init__(self, P: LogprobParams, device=None):
        n = load().graft_logprobs_workspace(C.byref(P))
        if n == 0:
            raise GraftError("graft_logprobs_workspace", 1,
                             load().graft_last_error_string().decode())
        self.buffer, self.addr, self.dev = _scratch(n, "graft_logprobs_init", device or "cuda")
        self.nbytes = n


def logprobs(logits, targets, logprob, entropy, top_logprob, top_index, P: LogprobParams,
             ws: LogprobWorkspace, stream=None) -> None:
    """Log probability of targets, entropy and top alternatives of each row of
    logits [rows, vocab] (graft_logprobs); outputs that are None are left out."""
    from torch import float32, int32
    rows, vocab, k = P.rows, P.vocab, P.top_k
    if logits.shape != (rows, vocab) or _dtype_code(logits.dtype) != P.dtype:
        raise ValueError("logits do not match the params")
    stride = logits.stride()
    if stride[1] != 1 and vocab > 1:
        raise ValueError("a row of logits must be contiguous")
    dev = logits.get_device()
    args = (_dense(targets, int32, (rows,), dev), _dense(logprob, float32, (rows,), dev),
            _dense(entropy, float32, (rows,), dev), _dense(top_logprob, float32, (rows, k), dev),
            _dense(top_index, int32, (rows, k), dev))
    Q = LogprobParams(rows, vocab, k, P.dtype, stride[0] if rows > 1 else vocab, P.scale)
    raw = _raw_stream(stream, dev)
    if ws.dev != dev:
        raise ValueError("the workspace is on another device than the tensors")
    call("graft_logprobs", logits.data_ptr(), *args, C.byref(Q), ws.addr, ws.nbytes, raw)


# ----------------------------------------------------------- multi-GPU --
COMM_ID_BYTES = 128


def comm_unique_id() -> bytes:
    """A fresh communicator id (rank 0); hand the bytes to every rank."""
    buf = C.create_string_buffer(COMM_ID_BYTES)
    call("graft_comm_get_unique_id", C.addressof(buf))
    return buf.raw


class Comm:
    """The ranks' communicator (one per process and GPU, on the current device).
    Collective: every rank constructs it with the same id."""

    def __init__(self, uid: bytes, nranks: int, rank: int):
        assert len(uid) == COMM_ID_BYTES
        self._buf = C.create_string_buffer(uid, COMM_ID_BYTES)
        self.handle = C.c_void_p()
        call("graft_comm_init", C.byref(self.handle), C.addressof(self._buf), nranks, rank)
        self.rank, self.nranks = rank, nranks

    @property
    def fused(self) -> bool:
        """True when the ranks run the fused (peer-memory) forms."""
        return bool(load().graft_comm_fused(self.handle))

    def alloc(self, shape, dtype):
        """A zeroed symmetric buffer (collective) as a CUDA tensor: outputs of the
        multi-GPU calls placed in it are gathered by the computing kernel itself."""
        import math
        import torch
        n = math.prod(shape) * torch.empty((), dtype=dtype).element_size()
        ptr = C.c_void_p()
        call("graft_comm_alloc", self.handle, n, C.byref(ptr))
        typestr = {torch.float16: "<f2", torch.float32: "<f4", torch.uint8: "|u1"}[dtype]

        class _Buf:
            __cuda_array_interface__ = {"shape": tuple(shape), "typestr": typestr,
                                        "data": (ptr.value, False), "version": 2}
        t = torch.as_tensor(_Buf(), device="cuda")
        self._owned = getattr(self, "_owned", []) + [ptr.value]
        return t

    def status(self) -> None:
        """Raises GraftError (GRAFT_ETIMEDOUT) once a fused call's wait for a
        peer has given up; sticky until the communicator is re-created."""
        call("graft_comm_status", self.handle)

    def set_fused(self, on: bool) -> None:
        """Fused (peer-memory) forms on, or off so that every call runs its NCCL
        form; every rank must make the same setting."""
        call("graft_comm_set_fused", self.handle, int(bool(on)))

    def set_wait_limit(self, ns: int) -> None:
        """Time limit of every peer wait of the fused calls (ns; 4 s by default)."""
        call("graft_comm_set_wait_limit", self.handle, ns)

    def close(self) -> None:
        if self.handle:
            for p in getattr(self, "_owned", []):
                call("graft_comm_free", self.handle, p)
            self._owned = []
            call("graft_comm_destroy", self.handle)
            self.handle = C.c_void_p()


def shard_rows(M_total: int, nranks: int, rank: int) -> tuple[int, int]:
    """Row block [lo, hi) of rank `rank` in the row-sharded GEMV (equal blocks)."""
    if M_total % nranks:
        raise ValueError(f"M={M_total} does not split evenly over {nranks} ranks")
    m = M_total // nranks
    return rank * m, (rank + 1) * m


def expert_range(n_experts: int, nranks: int, rank: int) -> tuple[int, int]:
    """Experts [lo, hi) held by rank `rank` in the expert-parallel MoE block."""
    if n_experts % nranks:
        raise ValueError(f"{n_experts} experts do not split evenly over {nranks} ranks")
    e = n_experts // nranks
    return rank * e, (rank + 1) * e


def gemv_int4_sharded(comm: Comm, W, SB, x, y_full, P: GemvParams, stream=None) -> None:
    """This rank's row shard (P: its M rows) into y_full[rank*M:], then all-gather."""
    call("graft_gemv_int4_sharded", comm.handle, _p(W), _p(SB), _p(x), _p(y_full), C.byref(P),
         _s(stream))


def gemm_int4_sharded(comm: Comm, W, SB, X, Y_full, B: int, P: GemvParams, stream=None) -> None:
    """B tokens through this rank's row shard (P: its M rows), all-gathered so
    that Y_full [B, nranks*M] holds every token's whole output."""
    call("graft_gemm_int4_sharded", comm.handle, _p(W), _p(SB), _p(X), _p(Y_full), B,
         C.byref(P), _s(stream))


def moe_block_ep(comm: Comm, pool, R, x, y, P: MoEParams, fmt: MoEFormat | None,
                 ws: MoEWorkspace, stream=None) -> None:
    """Expert-parallel block: `pool` holds this rank's experts only; y = full output."""
    call("graft_moe_block_ep", comm.handle, _p(pool), _p(R), _p(x), _p(y), C.byref(P),
         C.byref(fmt) if fmt is not None else None, C.byref(ws.scratch), _s(stream))

