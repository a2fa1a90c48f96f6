/*
 * cuda_graft.h -- C ABI of libcuda-graft.so: the LLM-decode hot path of
 * agastya-choudhary123/kernels (int4 group-affine GEMV, VQ codebook GEMV, fused
 * MoE block) as sm_100a (B200) CUDA kernels.
 *
 * Each entry point replaces one Metal kernel of the reference and keeps its
 * argument order = the kernel's [[buffer(i)]] index order, its params struct
 * and its buffer layouts, so a host that bound the Metal kernel by index can
 * bind this function argument by argument.  Differences from Metal:
 *   - buffers are caller-owned DEVICE pointers (cudaMalloc), not MTLBuffers;
 *   - the params struct is a HOST pointer read at call time (Metal setBytes);
 *   - the last argument is the CUDA stream the work is enqueued on (0 = the
 *     legacy default stream); calls are asynchronous, never synchronise, never
 *     allocate, and may be captured into a CUDA graph;
 *   - the return value is a status code; graft_last_error_string() explains a
 *     non-zero code.  No entry point exits or aborts the process.
 * Unless stated otherwise, every pointer to a vector loaded as 16-byte words
 * (W, IDX, x, h) must be 16-byte aligned and every length a multiple of the
 * stated granule; violations return GRAFT_EINVAL before anything is launched.
 */
#ifndef CUDA_GRAFT_H
#define CUDA_GRAFT_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Same object as cudaStream_t / CUstream. */
typedef struct CUstream_st* graft_stream_t;

/* ------------------------------------------------------------------ status */
enum {
    GRAFT_OK = 0,
    GRAFT_EINVAL = 1,    /* bad shape, alignment or argument                 */
    GRAFT_ECUDA = 2,     /* a CUDA runtime call or kernel launch failed      */
    GRAFT_ENCCL = 3,     /* an NCCL call failed                              */
    GRAFT_ETIMEDOUT = 4, /* a bounded device-side wait gave up               */
    GRAFT_ENOTSUP = 5    /* not supported on this device / build             */
};

/* Message for the last non-zero status returned on this host thread. */
const char* graft_last_error_string(void);
/* Library version string, e.g. "cuda-graft 0.1 sm_100a". */
const char* graft_version(void);

/* ===================================================== int4 group-affine ===
 * Layout (int4-gemv/src/kernels.metal:3-8): W is [M][K/8] uint32, row-major;
 * code j of word w is k = 8w+j (low nibble = lowest k).  One fp16 scale and
 * one fp16 bias per group of G consecutive k:  w[m,k] = S[m,k/G]*q[m,k] + B[m,k/G].
 * Constraints: K % 32 == 0, G % 32 == 0, K % G == 0 (the reference harness
 * also demands K % 512 == 0, int4-gemv/src/main.mm:140; these kernels do not).
 */

/* GemvParams, int4-gemv/src/kernels.metal:42-49 (host copy int4-gemv/src/main.mm:26). */
typedef struct {
    uint32_t M;         /* rows / output length          */
    uint32_t K;         /* reduction length              */
    uint32_t G;         /* quant group size              */
    uint32_t words_pr;  /* uint32 words per row  = K/8   */
    uint32_t groups_pr; /* groups per row        = K/G   */
    uint32_t chunks_pg; /* 32-weight chunks per group = G/32 */
} GraftGemvParams;

/* Fills P from (M, K, G) the way int4-gemv/src/main.mm:143 does. */
int graft_gemv_params(uint32_t M, uint32_t K, uint32_t G, GraftGemvParams* P);

/* xsum32, int4-gemv/src/kernels.metal:54-65.  Buffers: 0 x (fp16[K]),
 * 1 xs (fp32[K/32], xs[j] = sum of x[32j..32j+31]), 2 P. */
int graft_xsum32(const void* x, float* xs, const GraftGemvParams* P, graft_stream_t stream);

/* gemv_int4_wide_unroll (v6, the reference's best), int4-gemv/src/kernels.metal:399-448;
 * also stands in for gemv_int4_fused (v4, :295-335) and gemv_int4_wide (v5, :354-392),
 * which compute the same y from the same buffers.
 * Buffers: 0 W, 1 SB (interleaved fp16 (scale,bias) pairs, [M][K/G][2]),
 * 2 unused (kept so the argument order equals the Metal buffer index),
 * 3 x (fp16[K]), 4 y (fp32[M]), 5 xs (fp32[K/32] from graft_xsum32), 6 P. */
int graft_gemv_int4_wide_unroll(const void* W, const void* SB, const void* unused,
                                const void* x, float* y, const float* xs,
                                const GraftGemvParams* P, graft_stream_t stream);

/* gemv_int4_simd (v1), int4-gemv/src/kernels.metal:104-136; also stands in for
 * gemv_int4_scalar (v0, :71-95) and gemv_int4_multirow[_tgx] (v2/v3, :149-250).
 * Buffers: 0 W, 1 S (fp16[M][K/G]), 2 B (fp16[M][K/G]), 3 x, 4 y (fp32[M]), 5 xs, 6 P. */
int graft_gemv_int4_simd(const void* W, const void* S, const void* B, const void* x,
                         float* y, const float* xs, const GraftGemvParams* P,
                         graft_stream_t stream);

/* The BASELINE decode form of the v6 kernel: same W/SB/x layout, fp16 y[M]
 * rounded once from an fp32 accumulation, and the per-32 sums of x computed
 * inside the kernel (no xsum32 prepass, no xs buffer). */
int graft_gemv_int4_sb_f16out(const void* W, const void* SB, const void* x, void* y_f16,
                              const GraftGemvParams* P, graft_stream_t stream);

/* ExpertParams, moe-pipeline/src/main.mm:53: {M, K, G, quads_pr = K/32 (16-byte
 * words per row), groups_pr = K/G, chunks_pg = G/32}. */
typedef struct {
    uint32_t M, K, G, quads_pr, groups_pr, chunks_pg;
} GraftExpertParams;

/* Fills P from (M, K, G); GRAFT_EINVAL unless K % 32 == 0 and G | K, 32 | G. */
int graft_expert_params(uint32_t M, uint32_t K, uint32_t G, GraftExpertParams* P);

/* xsum32 over fp32 x, moe-pipeline/src/kernels.metal:37-48: xs[j] = sum of
 * x[32j .. 32j+31] in the reference's order.  x 16-byte aligned. */
int graft_xsum32_f32(const float* x, float* xs, const GraftExpertParams* P,
                     graft_stream_t stream);

/* gemv_int4_bf16, moe-pipeline/src/kernels.metal:53-83 (one projection of a
 * gpt-oss expert as stored on disk): W [M][K/8] u32 codes, S, B bf16 [M][K/G],
 * BI bf16 [M] (per-row output bias), x fp32 [K], y fp32 [M], xs = xsum32 of x.
 *   y[m] = sum_g S[m,g]*(q . x)_g + B[m,g]*xs_g  +  BI[m]
 * Buffers 0..7 in the reference's order.  x is rounded to fp16 when staged (as
 * the MoE block's router pass does); accumulation is fp32. */
int graft_gemv_int4_bf16(const void* W, const void* S, const void* B, const void* BI,
                         const float* x, float* y, const float* xs, const GraftExpertParams* P,
                         graft_stream_t stream);

/* The interleaved-SB int4 GEMV for B = 1..16 tokens at once (no reference
 * counterpart: the reference decodes one token): X fp16 [B][K] row-major,
 * Y fp16 [B][M] row-major, Y[b] = W . X[b] with fp32 accumulation.  The
 * weights are read once per launch; a launch takes as many tokens as their
 * staged x leaves shared memory for (all 16 up to K = 4096, 5 at K = 14336),
 * larger B runs in chunks.  G = 32, 64 or 128; W and X 16-byte aligned. */
int graft_gemm_int4_sb_f16(const void* W, const void* SB, const void* X, void* Y, uint32_t B,
                           const GraftGemvParams* P, graft_stream_t stream);
/* on = 1: B = 9..16 with G = 64, K a multiple of 256 (up to about 5k) and
 * 16-byte aligned W/SB/X run on the tcgen05 tensor cores (weights decoded
 * into tensor memory, x in shared memory, fp32 accumulators in tensor
 * memory) instead of the mma.sync tile engine.  Off by default: measured
 * slower at 16 tokens (128 against 95 us on a 128256 x 4096 lm_head).
 * Returns the previous setting. */
int graft_gemm_set_tcgen05(int on);

/* stream_read, int4-gemv/src/kernels.metal:262-283: reads nquads 16-byte words
 * of src once, XOR-folds them and stores to sink[0] only if the fold is
 * 0xFFFFFFFF (never, for real data): the pure-read bandwidth ceiling. */
int graft_stream_read(const void* src, uint32_t* sink, uint64_t nquads,
                      graft_stream_t stream);

/* Engine of the dense GEMVs (int4 and VQ), process-wide:
 *   GRAFT_ENGINE_TENSOR     (default) tiles of 16 rows streamed by TMA into
 *                           shared memory, row dots on mma.sync (f16 x f16 ->
 *                           f32) -- the fast path on B200;
 *   GRAFT_ENGINE_CUDA_CORE  register-direct: 16-byte loads straight to
 *                           registers, fp32 FMAs of exact fp16 products, warp
 *                           shuffles; no tensor cores (the reference's own
 *                           batch-1 formulation).
 * Results agree within the fp32-accumulation tolerance; neither depends on
 * timing.  GRAFT_ENGINE=cuda-core in the environment sets the default.  The
 * fused all-gather of graft_gemv_int4_sharded needs the tensor engine; under
 * the CUDA-core engine it gathers with NCCL. */
/* Error bits the kernels set on the current device, instead of hanging or
 * faulting: byte 0 int4 GEMV, byte 1 VQ GEMV, byte 2 MoE block; in each, bit 0
 * = a wait for a shared-memory slot gave up after 2 s (the call's output is
 * wrong), and for the VQ GEMV bit 1 = its shared-memory layout check failed
 * (nothing was written).  In byte 0, bit 4 is the same give-up in the tcgen05
 * batched kernel and bit 5 in the batched tile kernel (which also runs the
 * batch-1 GEMV of tall matrices and of scale rows that are not 16-byte
 * strided).  Synchronises the device; clears the bits if `clear`. */
int graft_device_errors(uint32_t* bits, int clear);

#define GRAFT_ENGINE_TENSOR 0
#define GRAFT_ENGINE_CUDA_CORE 1
int graft_set_gemv_engine(int engine);
int graft_get_gemv_engine(void);

/* ============================================================ VQ (d = 2) ===
 * Layout (vq-gemv/src/kernels.metal:15-19): IDX [M][K/2] uint8, the codeword
 * index of weights (2i, 2i+1); C [256][2] fp16, one codebook per matrix;
 *   w[m, 2i+t] = S[m, (2i)/SG] * C[IDX[m,i]][t].
 * Constraint: K % 32 == 0.
 */

/* VQParams, vq-gemv/src/kernels.metal:32-37. */
typedef struct {
    uint32_t M;         /* rows                               */
    uint32_t K;         /* reduction length                   */
    uint32_t chunks_pr; /* 32-weight chunks per row = K/32    */
    uint32_t cb_size;   /* codebook entries (must be 256)     */
} GraftVQParams;

/* gemv_vq_wide (the reference's best), vq-gemv/src/kernels.metal:337-380; also
 * stands in for gemv_vq_scalar/_shared/_replicated/_device (:71-228).
 * Buffers: 0 IDX, 1 C, 2 S (fp16[M][K/32], SG = 32), 3 x (fp16[K]), 4 y (fp32[M]), 5 P. */
int graft_gemv_vq_wide(const void* IDX, const void* C, const void* S, const void* x,
                       float* y, const GraftVQParams* P, graft_stream_t stream);

/* General form: scale_group SG is 32 (reference, S [M][K/32]) or K (one scale
 * per row, S [M]; the BASELINE configuration); y is fp32 (y_f16 = 0) or fp16. */
int graft_gemv_vq_ex(const void* IDX, const void* C, const void* S, uint32_t scale_group,
                     const void* x, void* y, int y_f16, const GraftVQParams* P,
                     graft_stream_t stream);

/* Decodes codewords: out[2i+t] = C[IDX[i]][t] (fp16 bits), n_idx indices. */
int graft_vq_decode(const void* IDX, const void* C, void* out, uint64_t n_idx,
                    graft_stream_t stream);

/* The VQ quantiser, vq-gemv/quant/pq_quantize.py:50-75 (quantize_matrix, with
 * _kmeans :28-47): W fp32 [M][K] -> IDX [M][K/2], C fp16 [256][2] and
 * S fp16 [M][K/32] (max |w| of each 32), the layout graft_gemv_vq_ex reads
 * with scale_group 32; w ~ S[m][2i/32] * C[IDX[m][i]][t].  Lloyd's k-means
 * (iters passes, reference 25) on sub sampled normalised pairs (reference
 * 200000; all pairs if there are fewer).  The sample and the initial
 * centroids come from seeded splitmix64 draws, not the reference's MLX
 * generator; the result is deterministic and bit-identical run to run. */
typedef struct {
    uint32_t M, K;      /* W rows and columns, K % 32 == 0          */
    uint32_t iters;     /* Lloyd passes                             */
    uint32_t sub;       /* sample size, 1 .. 2^22                   */
    uint64_t seed;
} GraftVQQuantParams;
/* Device workspace bytes graft_vq_quantize needs (0 for bad params). */
uint64_t graft_vq_quantize_workspace(const GraftVQQuantParams* P);
int graft_vq_quantize(const float* W, void* IDX, void* C, void* S, const GraftVQQuantParams* P,
                      void* ws, uint64_t ws_bytes, graft_stream_t stream);

/* ============================================================ MoE block ===
 * One decode token through a gpt-oss-style MoE block: router + top-k + softmax,
 * gate/up + SwiGLU, down + weighted combine, in three kernels.
 * Expert weights live in one pool: expert e's blob starts at pool + e*blob
 * (with an expert range [expert_lo, expert_hi), at pool + (e-expert_lo)*blob);
 * projection p (gate/up/down) at off_p inside it, and inside a projection W
 * (uint32 [rows][K/8]) at sub_w, S and B ([rows][K/64]) at sub_s/sub_b and the
 * per-row output bias BI ([rows]) at sub_bi (moe-fused/src/main.mm:23-25).
 * The reference format has bf16 S/B/BI, an fp32 router R [n_experts][hidden]
 * and fp32 x; the BASELINE format (GraftMoEFormat) has fp16 S/B, no BI, an fp16
 * router and fp16 x.  SwiGLU is gpt-oss's:
 *   h = min(g,7) * sigmoid(1.702*min(g,7)) * (clamp(u,-7,7) + 1).
 * Constraints: hidden, inter multiples of 64; top_k <= 8; n_experts <= 256.
 */

/* MoEParams, moe-fused/src/kernels.metal:22-35 (host copy moe-fused/src/main.mm:27-31).
 * The 64-bit block starts at byte 40, as in the reference. */
typedef struct {
    uint32_t hidden, inter, n_experts, top_k;
    uint32_t quads_hid, quads_int;   /* hidden/32, inter/32 */
    uint32_t groups_hid, groups_int; /* hidden/64, inter/64 */
    uint32_t chunks_pg;              /* 64/32 = 2           */
    uint64_t blob, off_gate, off_up, off_down;
    uint64_t sub_w, sub_s, sub_b, sub_bi;
} GraftMoEParams;

/* Fills P with the expert blob layout of moe-fused/src/main.mm:23-25,
 * generalised to any hidden/inter: inside a projection of R rows and K columns
 * W (R*K/2 B) is followed by S and B (R*K/32 B each) and BI (2R B); projections
 * gate, up, down follow one another, each padded to 16 bytes, and the blob is
 * padded to 16 KiB.  For hidden = inter = 2880 this gives exactly the
 * reference's offsets (blob 14,024,704; up at 4,671,360; down at 9,342,720). */
int graft_moe_params(uint32_t hidden, uint32_t inter, uint32_t n_experts, uint32_t top_k,
                     GraftMoEParams* P);

/* Format of the expert pool and activations (BASELINE vs reference). */
typedef struct {
    uint32_t scale_f16;    /* 0: bf16 S/B/BI (reference)   1: fp16 S/B (BASELINE)  */
    uint32_t has_bias_out; /* 1: per-row output bias BI at sub_bi                   */
    uint32_t act_f16;      /* 0: fp32 R and x (reference)  1: fp16 R and x         */
    uint32_t y_f16;        /* 0: fp32 y                    1: fp16 y               */
    uint32_t expert_lo;    /* experts in [expert_lo, expert_hi) are resident (the  */
    uint32_t expert_hi;    /* pool holds just these, expert_lo first) and contribute
                              to y (expert parallelism); the others are skipped    */
} GraftMoEFormat;

/* router_topk, moe-fused/src/kernels.metal:121-163.  Buffers: 0 R (fp32
 * [n_experts][hidden]), 1 x (fp32[hidden]), 2 idx (u32[top_k]), 3 wgt
 * (fp32[top_k]), 4 P, 5 xsh (fp32[top_k*quads_int], zeroed), 6 xh (fp16[hidden]).
 * Top-k is repeated strict-'>' argmax (the lowest expert index wins a tie);
 * softmax is over the k selected logits. */
int graft_moe_router_topk(const float* R, const float* x, uint32_t* idx, float* wgt,
                          const GraftMoEParams* P, float* xsh, void* xh,
                          graft_stream_t stream);

/* fused_gate_up_swiglu, moe-fused/src/kernels.metal:177-215.  Buffers: 0 pool,
 * 1 idx, 2 xh (fp16[hidden]), 3 h (fp16[top_k][inter]), 4 P. */
int graft_moe_fused_gate_up_swiglu(const void* pool, const uint32_t* idx, const void* xh,
                                   void* h, const GraftMoEParams* P, graft_stream_t stream);

/* fused_down_combine, moe-fused/src/kernels.metal:224-265.  Buffers: 0 pool,
 * 1 idx, 2 wgt, 3 h, 4 y (fp32[hidden]), 5 P. */
int graft_moe_fused_down_combine(const void* pool, const uint32_t* idx, const float* wgt,
                                 const void* h, float* y, const GraftMoEParams* P,
                                 graft_stream_t stream);

/* Atomic variants, moe-fused/src/kernels.metal:410-487: pass 2 also adds each
 * h value into xsh[e*quads_int + m/32]; pass 3 takes the per-32 sums of h from
 * xsh.  xsh must have been zeroed by graft_moe_router_topk. */
int graft_moe_fused_gate_up_swiglu_at(const void* pool, const uint32_t* idx,
                                      const void* xh, void* h, const GraftMoEParams* P,
                                      float* xsh, graft_stream_t stream);
int graft_moe_fused_down_combine_at(const void* pool, const uint32_t* idx, const float* wgt,
                                    const void* h, float* y, const GraftMoEParams* P,
                                    const float* xsh, graft_stream_t stream);

/* Scratch the block's kernels pass between them, carved from one caller
 * buffer.  `sync` holds the one-launch block's tagged words (router partials,
 * split row sums, h): they carry the launch they belong to, so the region needs
 * no reset between calls, but the caller must not write it. */
typedef struct {
    uint32_t* idx;   /* [top_k] selected experts                           */
    float* wgt;      /* [top_k] softmax weights                            */
    uint32_t* local; /* [1 + 2*top_k] count, slots and pool indices of the
                        selected experts this rank holds                     */
    void* xh;        /* fp16 [hidden]                                      */
    void* h;         /* fp16 [top_k][inter]                                */
    float* xsh;      /* [top_k * inter/32]                                 */
    float* ypart;    /* fp32 [hidden]: a rank's partial y (expert parallel) */
    void* sync;      /* tagged words of the one-launch block               */
} GraftMoEScratch;

/* Bytes of scratch graft_moe_scratch_carve needs for P. */
size_t graft_moe_scratch_bytes(const GraftMoEParams* P);
/* Carves `base` (device memory, 256-byte aligned, graft_moe_scratch_bytes long).
 * Host arithmetic only: nothing is written to the buffer. */
int graft_moe_scratch_carve(void* base, size_t bytes, const GraftMoEParams* P,
                            GraftMoEScratch* out);
/* Zeroes the scratch's `sync` region on `stream` (before the first block call
 * with a new buffer, and again if the buffer was used for anything else).  A
 * block call that finds a region it has not seen zeroes it itself, except
 * inside a stream capture, where it runs the three-kernel block instead. */
int graft_moe_scratch_init(const GraftMoEParams* P, const GraftMoEScratch* scratch,
                           graft_stream_t stream);

/* The whole block in three launches (router_topk, gate_up_swiglu,
 * down_combine), as encodeFused does (moe-fused/src/main.mm:176-206), in the
 * reference format (bf16 S/B/BI, fp32 R/x/y). */
int graft_moe_block(const void* pool, const float* R, const float* x, float* y,
                    const GraftMoEParams* P, const GraftMoEScratch* scratch,
                    graft_stream_t stream);

/* The block in any GraftMoEFormat (NULL = the reference format).  With
 * expert_lo/expert_hi a sub-range, `pool` holds only experts expert_lo ..
 * expert_hi-1 and y is this rank's partial sum over the selected experts it
 * holds (zero if none); the caller sums partials across ranks. */
int graft_moe_block_ex(const void* pool, const void* R, const void* x, void* y,
                       const GraftMoEParams* P, const GraftMoEFormat* fmt,
                       const GraftMoEScratch* scratch, graft_stream_t stream);

/* graft_moe_block and graft_moe_block_ex run the block as ONE launch where the
 * shapes allow it (the tile engine's shapes; one CTA per SM whose CTAs hand
 * the router logits, split row sums and h to one another through the
 * scratch's `sync` region), else as the three launches above.  Bits of on:
 * 1 = the whole block on one GPU, 2 = a rank's share of an expert-parallel
 * block (graft_moe_block_ex on an expert sub-range, graft_moe_block_ep); the
 * default is 0 (three launches) unless set.  Returns the previous setting.
 * Process-wide, not thread-safe against concurrent block calls. */
int graft_moe_set_one_launch(int on);
/* The three-launch block's down + combine pass: split = 1 runs it on every SM
 * without thread-block clusters, its units split evenly and a tile split
 * between CTAs handed on through the scratch's `sync` region; split = 0 (the
 * default, measured faster) runs it as clusters of top_k CTAs combining
 * through distributed shared memory.  Returns the previous setting. */
int graft_moe_set_down_pass(int split);

/* graft_moe_block_ex without a caller-provided scratch buffer -- for callers
 * that cannot call cudaMalloc (hosts that own all device memory through their
 * own arena and give a library no allocator, hosts that must not allocate
 * after start-up).  No counterpart in the
 * reference: the Metal harness always allocated its scratch buffers itself.
 * The scratch lives in a fixed 256 KiB device array inside the library (per
 * device, held until exit); configurations needing more return GRAFT_EINVAL.
 * All calls on a device share that array, so calls that can overlap on the GPU
 * race; calls on one stream are safe.  The first call on a device looks up the
 * array's address and should come before any stream capture. */
int graft_moe_block_noalloc(const void* pool, const void* R, const void* x, void* y,
                            const GraftMoEParams* P, const GraftMoEFormat* fmt,
                            graft_stream_t stream);

/* ==================================================== expert streaming ===
 * moe-pipeline (moe-pipeline/src/main.mm): experts stream from pinned host
 * memory into device slots on a side stream while the GPU computes.  The
 * experts.bin blob layout is GraftMoEParams' (blob, off_gate/up/down,
 * sub_w/s/b/bi; bf16 S, B and a bf16 per-row output bias BI).
 *
 * A graft_expert_stream_t owns a non-blocking copy stream and two events per
 * slot; the slots themselves are caller-owned device memory (n_slots * blob
 * bytes, 16-byte aligned).  Per expert i with depth d (the reference's order,
 * refill before compute, moe-pipeline/src/main.mm:333-363):
 *     acquire(slot(i), compute)            compute waits for the slot's copy
 *     fetch(slot(i+d), host_blob(i+d))     copy waits until the slot is released
 *     graft_expert_forward(slot(i), ...)   on compute
 *     release(slot(i), compute)
 * with n_slots >= d + 1.  Nothing blocks the host; not graph-capturable. */
typedef struct GraftExpertStream* graft_expert_stream_t;

int graft_expert_stream_create(void* slots, uint32_t n_slots, uint64_t blob_bytes,
                               graft_expert_stream_t* out);
int graft_expert_stream_destroy(graft_expert_stream_t es);
/* Device address of a slot (null if out of range). */
void* graft_expert_stream_slot(graft_expert_stream_t es, uint32_t slot);
/* Enqueues the copy of one blob (pinned host memory) into a slot, after the
 * slot's last release; GRAFT_EINVAL if host_blob is not pinned. */
int graft_expert_stream_fetch(graft_expert_stream_t es, uint32_t slot, const void* host_blob);
int graft_expert_stream_acquire(graft_expert_stream_t es, uint32_t slot, graft_stream_t stream);
int graft_expert_stream_release(graft_expert_stream_t es, uint32_t slot, graft_stream_t stream);
/* Blocks until every enqueued copy has landed. */
int graft_expert_stream_sync(graft_expert_stream_t es);

/* Caller-owned fp32 scratch of graft_expert_forward: xs_x [hidden/32],
 * gate, up, h [inter] (16-byte aligned), xs_h [inter/32]. */
typedef struct {
    float* xs_x;
    float* gate;
    float* up;
    float* h;
    float* xs_h;
} GraftExpertScratch;

/* One expert, encode_expert (moe-pipeline/src/main.mm:201-239): xsum32(x),
 * gate = gemv_int4_bf16(gate), up = gemv_int4_bf16(up), h = SwiGLU(gate, up)
 * (moe-pipeline/src/kernels.metal:88-98), xsum32(h), y = gemv_int4_bf16(down, h).
 * blob: one expert (device memory, e.g. a slot); x fp32 [hidden]; y fp32 [hidden]. */
int graft_expert_forward(const void* blob, const float* x, float* y, const GraftMoEParams* P,
                         const GraftExpertScratch* scratch, graft_stream_t stream);

/* =========================================================== multi-GPU ===
 * One process (or host thread) per GPU; the ranks share an NCCL communicator
 * over NVLink/NVSwitch.  The multi-GPU forms of the path: the reference's
 * hetero CPU/GPU row split (hetero-gemv/src/main.mm:196-239) made a row split
 * across GPUs, and the MoE block split by expert: */
typedef struct GraftComm* graft_comm_t;
#define GRAFT_COMM_ID_BYTES 128

/* Rank 0 creates the id; the host hands the 128 bytes to every rank. */
int graft_comm_get_unique_id(void* id);
/* Joins the communicator on the current device (collective over all ranks). */
int graft_comm_init(graft_comm_t* comm, const void* id, int nranks, int rank);
int graft_comm_destroy(graft_comm_t comm);
int graft_comm_info(graft_comm_t comm, int* rank, int* nranks);
/* Symmetric buffer (collective): allocated on every rank and mapped into the
 * other ranks' address spaces (CUDA IPC over NVLink).  Outputs of the
 * multi-GPU calls placed in such a buffer are gathered by the computing kernel
 * itself, with no separate collective.  Zero-filled. */
int graft_comm_alloc(graft_comm_t comm, size_t bytes, void** ptr);
int graft_comm_free(graft_comm_t comm, void* ptr);
/* 1 if this communicator runs the fused (peer-memory) forms, else 0. */
int graft_comm_fused(graft_comm_t comm);
/* Turns the fused forms off (0) or back on (1, the default where peer mapping
 * works): off, every multi-GPU call runs its NCCL form.  Every rank must make
 * the same setting before the same calls. */
int graft_comm_set_fused(graft_comm_t comm, int on);
/* GRAFT_ETIMEDOUT once a fused call's wait for a peer has given up (a rank
 * did not reach the call): the reference's fail-fast status checks
 * (int4-gemv/src/main.mm:38-42, :109-113) as a status, never an exit.  The
 * condition is sticky: after it, the fused calls of this communicator make no
 * peer stores and wait for nothing (their outputs are invalid) until the
 * communicator is destroyed and re-created.  Synchronises the device. */
int graft_comm_status(graft_comm_t comm);
/* The time limit of every peer wait of the fused calls, in nanoseconds (4 s
 * by default); a wait that runs past it gives up as described above. */
int graft_comm_set_wait_limit(graft_comm_t comm, uint64_t ns);

/* Row-sharded int4 GEMV (interleaved SB layout, fp16 y): this rank holds rows
 * [rank*M, (rank+1)*M) of an (nranks*M) x K matrix, P describing its shard
 * (M rows).  It computes its slice into y_full + rank*M and all-gathers, so
 * every rank's y_full (fp16 [nranks*M]) holds the whole output.  With y_full
 * inside a buffer from graft_comm_alloc (at the same offset on every rank) the
 * gather is fused into the GEMV kernel (peer stores); otherwise it is an NCCL
 * all-gather after it. */
int graft_gemv_int4_sharded(graft_comm_t comm, const void* W, const void* SB, const void* x,
                            void* y_full, const GraftGemvParams* P, graft_stream_t stream);

/* The same for B = 1..16 tokens (graft_gemm_int4_sb_f16 on the shard): X fp16
 * [B][K]; Y_full fp16 [B][nranks*M], row b the whole output of token b.  The
 * rank's rows of every token land at Y_full + b*nranks*M + rank*M; fused
 * (peer stores in the kernel's epilogue) with Y_full from graft_comm_alloc,
 * else B in-place NCCL all-gathers in one group. */
int graft_gemm_int4_sharded(graft_comm_t comm, const void* W, const void* SB, const void* X,
                            void* Y_full, uint32_t B, const GraftGemvParams* P,
                            graft_stream_t stream);

/* Expert-parallel MoE block: the ranks split the n_experts experts into equal
 * contiguous ranges (rank r holds [r*E/n, (r+1)*E/n), `pool` holding just
 * those); the router runs on every rank, each rank computes its selected
 * local experts' weighted partial output, and the partials are summed across
 * ranks (fp32) so every rank's y holds the block output.  fmt's expert range
 * is ignored; fmt->y_f16 chooses fp16 or fp32 y. */
int graft_moe_block_ep(graft_comm_t comm, const void* pool, const void* R, const void* x,
                       void* y, const GraftMoEParams* P, const GraftMoEFormat* fmt,
                       const GraftMoEScratch* scratch, graft_stream_t stream);

/* ==================================================== 8-bit key/value cache ===
 * A paged cache of attention keys and values in 8 bits, with one fp32 scale
 * for each block of tokens and head (K and V apart):
 *   codes  [n_blocks][kv_heads][block_tokens][head_dim]  (one byte each)
 *   scales [n_blocks][kv_heads]                          value = code * scale
 * Codes are signed integers in [-127, 127] (GRAFT_KV_INT8) or 8-bit floats
 * with 4 exponent and 3 mantissa bits, largest value 448 (GRAFT_KV_E4M3);
 * scales are finite and not negative.  graft_kv_write stores none below 2^-64;
 * attention takes a smaller one of V for 2^-64.
 * Constraints: block_tokens 16, 32, 64 or 128; head_dim a multiple of 16, at
 * most 256; code pointers 16-byte aligned, scale pointers 4-byte aligned. */
enum { GRAFT_KV_INT8 = 0, GRAFT_KV_E4M3 = 1 };
/* Element types of 16- and 32-bit buffers. */
enum { GRAFT_F16 = 0, GRAFT_BF16 = 1, GRAFT_F32 = 2 };

typedef struct {
    void* k;                 /* codes                                         */
    void* v;
    float* k_scale;
    float* v_scale;
    uint32_t n_blocks, kv_heads, block_tokens, head_dim;
    uint32_t format;         /* GRAFT_KV_INT8 or GRAFT_KV_E4M3                */
} GraftKVCache;

/* Consecutive tokens of each of n_seqs sequences: sequence b's tokens lie at
 * positions start[b] .. start[b] + n_b - 1, n_b = cu_tokens[b+1] -
 * cu_tokens[b] >= 0 (0 allowed), and are rows cu_tokens[b] .. of a buffer
 * that holds all sequences' tokens one after the other (cu_tokens[0] = 0).
 * Position p is in block block_table[b*table_stride + p / block_tokens].
 * The arrays are in device memory and read when the kernels run; the host
 * gives two upper bounds: max_tokens >= every n_b and max_len >= every
 * start[b] + n_b.  Block numbers outside the cache and lengths beyond the
 * bounds are skipped by the kernels and reported (graft_kv_device_errors). */
typedef struct {
    const int32_t* block_table;  /* [n_seqs][table_stride]                    */
    const int32_t* start;        /* [n_seqs]                                  */
    const int32_t* cu_tokens;    /* [n_seqs + 1]                              */
    uint32_t n_seqs, table_stride;
    uint32_t max_tokens, max_len;
} GraftKVRange;

/* Rows of heads: element d of head h of token t is
 * data[t*token_stride + h*head_stride + d] (strides in elements; a slice of a
 * joint q/k/v buffer, or a transposed one).  data 16-byte aligned, strides in
 * bytes multiples of 16. */
typedef struct {
    void* data;
    uint64_t token_stride, head_stride;
    uint32_t tokens;             /* rows in the buffer                        */
    uint32_t dtype;              /* GRAFT_F16, GRAFT_BF16 or GRAFT_F32        */
} GraftHeads;

/* Quantises the range's keys and values into the cache.  In each block that a
 * sequence's new tokens touch, per head:
 *   scale = max(amax / qmax, 2^-64, the old scale if the block already holds
 *           earlier tokens of the sequence)         qmax = 127 or 448
 *   code  = x / scale, rounded to nearest even;
 * where the scale grew, the earlier tokens' codes are rounded again to it
 * (code * old scale / new scale).  A block's first tokens start its scale
 * afresh, whatever an earlier owner left.  amax is taken over finite values;
 * an infinity is stored as +-qmax and a NaN as 0, so a cache holds finite
 * numbers only.  No two sequences of a call may touch the same block. */
int graft_kv_write(const GraftKVCache* cache, const GraftHeads* K, const GraftHeads* V,
                   const GraftKVRange* range, graft_stream_t stream);

/* Reads the range back: code * scale, rounded once to the buffers' type. */
int graft_kv_read(const GraftKVCache* cache, const GraftHeads* K, const GraftHeads* V,
                  const GraftKVRange* range, graft_stream_t stream);

/* Device-side findings of the cache and attention kernels, or-ed together:
 * GRAFT_KV_EBLOCK: a block number outside the cache; GRAFT_KV_EBOUNDS: lengths
 * beyond max_tokens, max_len, the block table or a buffer; GRAFT_KV_EWAIT: a
 * bounded wait gave up.  Synchronises the device; clear != 0 resets them. */
enum { GRAFT_KV_EBLOCK = 1, GRAFT_KV_EBOUNDS = 2, GRAFT_KV_EWAIT = 4 };
int graft_kv_device_errors(uint32_t* bits, int clear);

/* ------------------------------------------------- attention over the cache */
typedef struct {
    uint32_t q_heads;   /* a multiple of kv_heads: q head h reads kv head h / (q_heads/kv_heads);
                           at most 256 times kv_heads (128 times above head_dim 128)  */
    uint32_t window;    /* keys a query sees, itself included; 0 = all        */
    float scale;        /* of the scores, e.g. 1/sqrt(head_dim); finite       */
} GraftAttnParams;

/* Attention of the range's tokens over the cache, which holds their own keys
 * and values already (graft_kv_write first).  Token i of a sequence, at
 * position p = start + i, sees keys j with p - window < j <= p:
 *   o = sum_j exp(scale q.k_j - lse) v_j,
 *   lse = log( sum_j exp(scale q.k_j)  [+ exp(sinks[h])] ).
 * Blocks wholly before the window of a sequence's first new token are not
 * read, nor are their entries in the block table.
 * Scores, maxima and sums are fp32; the weights of the second product are
 * rounded to fp16: with all its 11 bits down to 2^-13 of a row's largest at
 * least, and as 0 from 2^-25 on at the earliest (2^-24 and 2^-35 where few rows
 * are taken or head_dim is 65 to 128).  In lse and in the sum that the output is
 * divided by they count in full.
 * A value's scale counts as part of its weight here.  exp2, log2 and the last
 * division are the device's approximate ones (about 2^-22).
 * q and out: GRAFT_F16 or GRAFT_BF16, the same type.  sinks (fp32 [q_heads], a
 * score that takes weight but has no value) and lse (fp32 [tokens][q_heads])
 * may be null.  Few rows a key/value head (max_tokens * q_heads/kv_heads up to
 * 32, 16 or 8 for head_dim up to 64, 128 or 256) take one pass over the keys at
 * the rate of HBM; more take tcgen05 tiles of 256 rows.  ws:
 * graft_attn_kv8_workspace bytes, 256-byte aligned, zeroed once by
 * graft_attn_kv8_init; it serves any call that it is large enough for, one at a
 * time. */
size_t graft_attn_kv8_workspace(const GraftKVCache* cache, const GraftKVRange* range,
                                const GraftAttnParams* P);
int graft_attn_kv8_init(void* ws, size_t ws_bytes, graft_stream_t stream);
int graft_attn_kv8(const GraftKVCache* cache, const GraftHeads* q, const GraftHeads* out,
                   const GraftKVRange* range, const float* sinks, float* lse,
                   const GraftAttnParams* P, void* ws, size_t ws_bytes, graft_stream_t stream);

/* ======================================================== log probabilities ===
 * From rows of logits (the lm_head's output), with z = scale * logit:
 *   lse          = log sum_v exp(z_v)
 *   logprob[r]   = z[targets[r]] - lse       (NaN for a target outside 0..vocab-1)
 *   entropy[r]   = lse - sum_v p_v z_v
 *   top_logprob, top_index [r][top_k]: the largest logits, in falling order,
 *     equal ones by rising index.
 * A logit of -inf is a token that cannot come: it adds nothing, and is never
 * listed (index -1, log probability -inf fill up a row that has fewer than
 * top_k others).  A row without any possible token gives logprob -inf and
 * entropy 0; a row with a NaN or +inf gives NaN log probabilities and entropy. */
typedef struct {
    uint32_t rows, vocab;
    uint32_t top_k;      /* 0 .. 32                                           */
    uint32_t dtype;      /* of the logits: GRAFT_F16, GRAFT_BF16 or GRAFT_F32 */
    uint64_t row_stride; /* elements from row to row (>= vocab, any value)    */
    float scale;         /* 1/temperature, 2^-100 to 2^100                    */
} GraftLogprobParams;

/* logits aligned to its element; targets (int32 [rows]) and logprob may both be
 * null, entropy may be null, top_* may be null when top_k is 0.  ws as for
 * graft_attn_kv8: graft_logprobs_workspace bytes, 256-byte aligned, zeroed once by
 * graft_logprobs_init and kept for calls of one stream at a time. */
size_t graft_logprobs_workspace(const GraftLogprobParams* P);
int graft_logprobs_init(void* ws, size_t ws_bytes, graft_stream_t stream);
int graft_logprobs(const void* logits, const int32_t* targets, float* logprob, float* entropy,
                   float* top_logprob, int32_t* top_index, const GraftLogprobParams* P, void* ws,
                   size_t ws_bytes, graft_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* CUDA_GRAFT_H */
