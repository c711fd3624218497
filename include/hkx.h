/*
 * hkx.h -- the C ABI of libhkx.so: GEMM with a fused epilogue on MI355X (gfx950).
 *
 * C = epilogue(A . B^T accumulated in fp32), A (M, K) and B (N, K) K-contiguous
 * (F.linear's layout), bf16 x bf16 or fp8-e4m3 x fp8-e4m3, C (M, N) in bf16, fp16,
 * fp32, int8 or fp8-e4m3.
 *
 * Plain pointers and sizes only; no torch types. Every pointer is a device pointer
 * on the current HIP device; every launch goes on the stream passed in. The library
 * allocates nothing and never synchronizes: a caller that needs a workspace asks
 * hkx_gemm_workspace() for its size and passes it in (HkxGemmArgs.ws).
 *
 * What each entry point replaces in the reference (vivienfanghuagood/hk-dsl 0.9.24):
 *
 *   hkx_gemm            the launches hk.templates.gemm prepares for a plan, one
 *                       `kern(a, b, c, *extra, *ep_tensors, **consts)` per Step
 *                       (python/hk/templates/gemm.py:577-665, launch convention
 *                       python/hk/ops/_epilogue.py:28-43), which end in
 *                       hipModuleLaunchKernel on the caller's stream
 *                       (mlir/python/HKLaunch.c:1-25, python/hk/runtime/codeobj.py:265-276).
 *                       The kernels it runs replace gemm_cdna.gemm_kernel
 *                       (python/hk/ops/gemm_cdna.py:57-586), gemm_cdna_dp.gemm_kernel and
 *                       its split-K shares (python/hk/ops/gemm_cdna_dp.py:30-243),
 *                       reduce_epilogue_kernel (gemm_cdna_dp.py:295-324, 361-383) and
 *                       decode_gemm_kernel (python/hk/ops/decode_gemm.py:37-180).
 *   hkx_scaled_mm       hk.ops.gemm.scaled_mm's launch (python/hk/ops/gemm.py:884-975):
 *                       bf16 (A . B^T) * scale_a * scale_b (+ bias), fp8 operands.
 *   hkx_mx_gemm         hk.ops.mxfp8.gemm / gemm_pp's launch (python/hk/ops/mxfp8.py:64-110,
 *                       gemm_cdna.gemm_kernel with mx=True, python/hk/ops/gemm_cdna.py:82-94):
 *                       bf16 C = (sa . A)(sb . B)^T, fp8-e4m3 operands with OCP MX E8M0
 *                       scales, one byte a row and 32 K.
 *   hkx_mx_quant        hk.ops.mxfp8.quant's launch (python/hk/ops/mxfp8.py:605-660): bf16
 *                       rows to fp8-e4m3 with an E8M0 scale a 32-column block, AITER's
 *                       per_1x32 rule (python/hk/mx.py:17-31), the scales in the OCP
 *                       layout the MX GEMM reads.
 *   hkx_gemm_workspace  gemm_cdna_dp.scratch_for / decode_gemm.scratch_for
 *                       (gemm_cdna_dp.py:330-338, decode_gemm.py:283-298): the size of
 *                       the fp32 share buffer a plan needs (the caller allocates it).
 *   hkx_mx_gemm_workspace  the same for hkx_mx_gemm's split-K shares (this build splits
 *                       K across workgroups where the reference's MX kernel runs few tiles
 *                       unsplit, python/hk/ops/mxfp8.py:64-110).
 *   hkx_last_error      the message the reference raises in Python (ValueError /
 *                       TypeError texts of templates/gemm.py:770-803).
 */
#ifndef HKX_H_
#define HKX_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define HKX_ABI_VERSION 4

/* Status codes. */
#define HKX_OK 0
#define HKX_ERR_SHAPE 1       /* a shape / stride / alignment the kernels do not take */
#define HKX_ERR_DTYPE 2       /* an element type the kernels do not take */
#define HKX_ERR_WORKSPACE 3   /* ws missing or smaller than hkx_gemm_workspace() */
#define HKX_ERR_LAUNCH 4      /* hipLaunchKernel failed; hkx_last_error() has hipGetErrorString */
#define HKX_ERR_ARG 5         /* a malformed argument (epilogue program, operand, null pointer) */

/* Element types. */
#define HKX_BF16 0
#define HKX_FP16 1
#define HKX_FP32 2
#define HKX_FP8E4M3 3 /* OCP e4m3 (float8_e4m3fn): max 448, no inf */
#define HKX_INT8 4
/* fp8 operand pairs with e5m2 (OCP float8_e5m2: max 57344, inf and nan), as ab_dtype only;
 * they run on 256 x 256 ring tiles (the quadrant kernel's dequant forms, else the half-stage
 * ring kernel): */
#define HKX_FP8E5M2 5        /* A and B e5m2 */
#define HKX_FP8_E4M3_E5M2 6  /* A e4m3, B e5m2 (e.g. activations against a gradient) */
#define HKX_FP8_E5M2_E4M3 7  /* A e5m2, B e4m3 */
#define HKX_FP4E2M1 8 /* OCP e2m1, two a byte, the even column in the low bits: the MXFP4 calls only */

/* Epilogue operand kinds: what an operand is against C (M, N) -- templates/gemm.py:116-135. */
#define HKX_ROW 1  /* (N,) or (1, N): one value per column of C (a bias, a per-channel scale) */
#define HKX_COL 2  /* (M, 1): one value per row (a per-token scale); ld = its row stride */
#define HKX_TILE 3 /* (M, N): one per element (a residual); ld = its row stride */

/* Epilogue forms. */
#define HKX_EP_NONE 0     /* C = acc */
#define HKX_EP_FUSED 1    /* C = act(acc * col_scale[m] * row_scale[n] * cmul + row_add[n] + tile_add[m,n] + cadd) */
#define HKX_EP_PROGRAM 2  /* C = the register program below, run once per element on the fp32 sum */
#define HKX_EP_SILU_MUL 3 /* C[:, j] = silu(acc[:, j]) * acc[:, N + j]; B is (2N, K), gate rows then up rows */

/* Activations of the fused form. */
#define HKX_ACT_NONE 0
#define HKX_ACT_GELU_TANH 1
#define HKX_ACT_SILU 2
#define HKX_ACT_RELU 3

/* Program opcodes: dst <- f(a, b, c); registers are fp32, R0 starts as the accumulator. */
#define HKX_OP_MOV 0    /* dst = r[a] */
#define HKX_OP_LOAD 1   /* dst = operand a at this element (by its kind), as fp32 */
#define HKX_OP_CONST 2  /* dst = imm */
#define HKX_OP_ROW 3    /* dst = the element's row of C */
#define HKX_OP_COL 4    /* dst = the element's column of C, plus col0 */
#define HKX_OP_ADD 5
#define HKX_OP_SUB 6
#define HKX_OP_MUL 7
#define HKX_OP_DIV 8
#define HKX_OP_MAX 9
#define HKX_OP_MIN 10
#define HKX_OP_EXP 11
#define HKX_OP_EXP2 12
#define HKX_OP_LOG 13
#define HKX_OP_LOG2 14
#define HKX_OP_ABS 15
#define HKX_OP_RELU 16
#define HKX_OP_GELU 17  /* tanh approximation */
#define HKX_OP_SILU 18
#define HKX_OP_SQRT 19
#define HKX_OP_RSQRT 20
#define HKX_OP_NEG 21
#define HKX_OP_STEP 22  /* 1 where r[a] > 0, else 0 */
#define HKX_OP_SELLE 23 /* dst = r[a] <= 0 ? r[b] : r[c] */
#define HKX_OP_M 24     /* dst = M (C's rows) */
#define HKX_OP_TANH 25
#define HKX_OP_SIGMOID 26
#define HKX_OP_SQUARE 27 /* dst = r[a] * r[a] */
#define HKX_NUM_OPS 28

#define HKX_MAX_OPERANDS 8
#define HKX_MAX_INSTR 64
#define HKX_MAX_REGS 16

typedef struct HkxOperand {
  const void* ptr; /* device pointer */
  int32_t kind;    /* HKX_ROW / HKX_COL / HKX_TILE */
  int32_t dtype;   /* HKX_BF16 / HKX_FP16 / HKX_FP32 */
  int64_t ld;      /* COL, TILE: row stride in elements. ROW: 1 (a vector) or 0 (one value
                      broadcast to every column) */
} HkxOperand;

typedef struct HkxInstr {
  uint8_t op, dst, a, b, c, pad0, pad1, pad2;
  float imm;
} HkxInstr;

typedef struct HkxEpilogue {
  int32_t form; /* HKX_EP_* */
  /* HKX_EP_FUSED: operand indices into ops[] (-1 = absent), the activation, constants. */
  int32_t act;
  int32_t col_scale, row_scale, row_add, tile_add;
  float cmul, cadd;
  /* HKX_EP_PROGRAM */
  int32_t nins;
  int32_t out_reg;
  int32_t col0; /* added to HKX_OP_COL (a launch on a column slice of a larger C) */
  int32_t nops;
  HkxOperand ops[HKX_MAX_OPERANDS];
  HkxInstr ins[HKX_MAX_INSTR];
} HkxEpilogue;

/* Kernel families (HkxGemmArgs.kernel). */
#define HKX_KERNEL_AUTO 0
#define HKX_KERNEL_TILE 1   /* LDS-tiled MFMA GEMM, tile_m x tile_n blocks, optional split-K */
#define HKX_KERNEL_DECODE 2 /* skinny-M weight-streaming GEMM (M <= 32), optional split-K */

/* Tile kernel schedules (HkxGemmArgs.tile_schedule). */
#define HKX_TILE_AUTO 0
#define HKX_TILE_PINGPONG 1 /* 8 waves, two a SIMD taking turns at the MFMA; 256 x 256 only */
#define HKX_TILE_W4 2       /* 4 waves, one a SIMD (2 x 2, 32 x 32 MFMAs), up to four LDS
                               stages; 256, 128 or 64 x 256 and 128 or 64 x 128 */
#define HKX_TILE_W8 3       /* 8 waves, register-staged fills, 16 x 16 MFMAs; every tile
                               shape but 64 x 128 */
#define HKX_TILE_RING 4     /* 8 waves taking turns at the MFMA, one workgroup a CU walking its
                               tiles through one LDS ring, epilogue stored from registers;
                               256 x 256 only, C rows 16-byte aligned, N % 8 == 0 */

/* HKX_TILE_PINGPONG variant bits (HkxGemmArgs.variant; 0 = the default). */
#define HKX_PP_MFMA32 1   /* 32 x 32 MFMA fragments (the fp8 and paired forms always use them) */
#define HKX_PP_ONE_TILE 2 /* one tile a workgroup, instead of a grid of one workgroup a CU */

/* HKX_TILE_RING variant bits. */
#define HKX_RING_WAVESPLIT 4 /* the columns whose 256 x 256 tiles make whole waves of the CUs
                                on the ring kernel, the rest of N on the 4-wave kernel's
                                128 x 256 tiles (two launches; no split over K) -- the
                                reference's ppw candidate (gemm_cdna.py:834-835, 923-930) */
#define HKX_RING_STREAMK 8   /* the whole waves likewise on the ring kernel, the rest of N on
                                ring tiles split over K so that they fill the CUs (fp32 shares
                                in the workspace, then one pass that sums them in split order
                                and applies the epilogue) -- the reference's dp+sk stream-K
                                mode (gemm_cdna.py:421-496, 635-729) without its in-kernel
                                fix-up; hkx_gemm_workspace() sizes the shares */
#define HKX_RING_HALFSTAGE 16 /* every form on the half-stage ring kernel. Without it a call the
                                 quadrant kernel takes runs there (bf16 operands and C, no
                                 split, no epilogue or a bf16 bias and an activation): each
                                 wave's output spread over the tile's four 128 x 128 quadrants,
                                 whole 128-byte lines a fill -- the reference's pp schedule
                                 (gemm_cdna.py:57-586). Combines with the two bits above */

/* HKX_KERNEL_DECODE variant bits. */
#define HKX_DEC_STREAM 1  /* one workgroup a CU streaming W (M <= 16, or M <= 32 from K =
                             2048; K a multiple of 1024 up to 32768, no split): in
                             blocks of 16 rows, or, with no residual and no vector scale, in
                             chunks of whole rows -- 4 rows at K = 4096, M <= 4, N <= 32768
                             or at M <= 2 any N with W under 2 GiB (one or two chunks a short
                             workgroup at M <= 3, and at M = 4 up to N = 8192; else strided
                             over one workgroup a CU); 8 rows, one
                             a wave, at K = 1024 (M <= 3) and K = 2048 (M <= 2); other calls
                             take the blocked kernel */

typedef struct HkxGemmArgs {
  const void* a; /* (M, K), row stride lda elements */
  const void* b; /* (N, K) -- (2N, K) for HKX_EP_SILU_MUL -- row stride ldb elements */
  void* c;       /* (M, N), row stride ldc elements */
  int64_t lda, ldb, ldc;
  int32_t m, n, k;
  int32_t ab_dtype; /* HKX_BF16, HKX_FP8E4M3 (both operands), or an e5m2 pair code */
  int32_t c_dtype;  /* HKX_BF16 / HKX_FP16 / HKX_FP32 / HKX_INT8 / HKX_FP8E4M3 */
  int32_t kernel;   /* HKX_KERNEL_* */
  int32_t tile_m;   /* TILE: 64, 128 or 256 (256 x 128 on W8 only, 64 x 128 on W4 only) */
  int32_t tile_n;   /* TILE: 128 or 256 */
  int32_t splits;   /* >= 1; > 1 stores fp32 shares to ws and sums them in order */
  int32_t tile_schedule; /* TILE: HKX_TILE_*; AUTO = RING for 256 x 256 tiles it takes,
                            else PINGPONG for 256 x 256, else W4 where the tile takes it,
                            else W8 */
  int32_t variant;  /* TILE, PINGPONG: HKX_PP_* bits (for tuning); DECODE: HKX_DEC_* bits */
  int32_t decode_waves; /* DECODE: waves per workgroup (4, 8 or 16); 0 = default */
  int32_t decode_rows;  /* DECODE: W rows per workgroup (16 or 32); 0 = default */
  void* ws;         /* fp32 workspace, hkx_gemm_workspace() bytes */
  size_t ws_bytes;
  HkxEpilogue ep;
  /* A split over K finished in the kernel: int32 arrival counters, hkx_gemm_counters() of
     them, all zero before the first call. With them the blocked decode kernel (one counter
     a block of rows) and the 4-wave tile kernel (one a tile) finish the split themselves:
     each workgroup stores its fp32 share and arrives at its counter, and the last to arrive
     sums the shares in split order (as the second launch does, so the result is the same),
     applies the epilogue and sets the counter back to zero -- one launch. NULL: the shares
     are summed by a second launch. Measured on MI355X, the decode finish costs what the
     second launch does, the tile finish 4-10 us more a call at M = 16-128 (its last
     arrivers' chain of share stores, arrival and share loads is all tail); hk's Python
     layer passes counters for decode splits only. Calls that overlap in time on one GPU
     must not share counters. */
  int32_t* counters;
  int64_t counters_len;
} HkxGemmArgs;

/* Library identity. */
int hkx_abi_version(void);
/* sizeof(HkxOperand), sizeof(HkxInstr), sizeof(HkxEpilogue), sizeof(HkxGemmArgs) into
 * out[0..3]: lets a binding check its struct layouts against the library's. */
void hkx_abi_sizes(size_t out[4]);
/* The message of the last failed call on this thread ("" if none). */
const char* hkx_last_error(void);

/* Bytes of fp32 workspace hkx_gemm needs for these args (0 if none). Resolves
 * HKX_KERNEL_AUTO the way hkx_gemm does. Host-only, needs no GPU. */
size_t hkx_gemm_workspace(const HkxGemmArgs* args);

/* int32 arrival counters hkx_gemm uses for these args (0 if the plan has no in-kernel
 * arrival): the blocked decode kernel or the 4-wave tile kernel split over K, unpaired,
 * fused or no epilogue (the tile kernel: all the shares under 4 GiB). Replaces
 * the counter half of decode_gemm.scratch_for (python/hk/ops/decode_gemm.py:283-298), whose
 * kernel arrives at cnt[b] and whose last arriver sums, finishes and resets it (:155-170).
 * Host-only, needs no GPU. */
size_t hkx_gemm_counters(const HkxGemmArgs* args);

/* Checks args (HKX_OK or an error code, message in hkx_last_error) without launching.
 * Host-only, needs no GPU. */
int hkx_gemm_check(const HkxGemmArgs* args);

/* Launch the plan for args on stream (a hipStream_t; NULL = the null stream).
 * Returns HKX_OK or an error code; hkx_last_error() says why. */
int hkx_gemm(const HkxGemmArgs* args, void* stream);

/* hkx_gemm with no workspace argument and no allocation: the plan's fp32 workspace (split-K
 * shares, a register program's sum) is a static device array of the library,
 * HKX_NOALLOC_SCRATCH_BYTES on each GPU it runs on, held until the process ends. args->ws
 * and args->ws_bytes are ignored. A plan that needs more than that fails with
 * HKX_ERR_WORKSPACE (nothing launched). Calls no hipMalloc / hipFree; every kernel writes
 * each scratch byte it reads in the same call, so nothing needs clearing between calls.
 * Every call on one GPU shares that GPU's array: two calls that overlap in time on one GPU
 * (other streams, or graphs replayed concurrently) race on it -- serialise them.
 * No counterpart in the reference: it is for callers that cannot allocate (code under
 * HIP-graph capture, serving loops and harnesses that forbid hipMalloc). */
#define HKX_NOALLOC_SCRATCH_BYTES (64u << 20)
int hkx_gemm_noalloc(const HkxGemmArgs* args, void* stream);

/* bf16 C = (A . B^T) * scale_a * scale_b (+ bias), A (M, K) and B (N, K) fp8-e4m3,
 * scale_a fp32 with sa_ld 0 (one value for all rows: per-tensor) or its row
 * stride (per-token, (M, 1)); scale_b fp32, sb_per_channel 0 (one value) or 1
 * ((N,), per-channel); bias bf16 (N,) or NULL. Row strides in elements. */
int hkx_scaled_mm(const void* a, int64_t lda, const void* b, int64_t ldb,
                  const float* scale_a, int64_t sa_ld, const float* scale_b,
                  int32_t sb_per_channel, const void* bias, void* c, int64_t ldc,
                  int32_t m, int32_t n, int32_t k, void* ws, size_t ws_bytes,
                  void* stream);

/* bf16 C = (sa . A)(sb . B)^T: A (M, K) and B (N, K) fp8-e4m3, sa (M, K/32) and sb
 * (N, K/32) E8M0 bytes (scale 2^(s - 127) for its row and 32 K), row strides lda, ldb,
 * ldc in elements and sa_ld, sb_ld in bytes. K a multiple of 128, N of 8; sa and sb
 * 4-byte aligned with sa_ld, sb_ld multiples of 4 and >= K/32; C's rows 16-byte aligned.
 * M any. Up to M = 16, and up to 32 at a short K, the 8-bit decode kernel runs it in one
 * pass; elsewhere the plan of tiles, K splits and columns of least estimated time. A split's
 * fp32 shares go through ws
 * (hkx_mx_gemm_workspace() bytes where 256 x 256 tiles fill less than half the CUs and K is 2048
 * or more; HKX_ERR_WORKSPACE if smaller), summed in split order by a second pass. */
int hkx_mx_gemm(const void* a, int64_t lda, const void* b, int64_t ldb, const uint8_t* sa,
                int64_t sa_ld, const uint8_t* sb, int64_t sb_ld, void* c, int64_t ldc,
                int32_t m, int32_t n, int32_t k, void* ws, size_t ws_bytes, void* stream);

/* Bytes of fp32 workspace hkx_mx_gemm takes at M x N x K (0: none; its plan uses all of it or
 * less). */
size_t hkx_mx_gemm_workspace(int32_t m, int32_t n, int32_t k);

/* x bf16 (M, K) -> q fp8-e4m3 (M, K) and s (M, K/32) E8M0 bytes: per 32-column block,
 * e = ceil(log2(amax / 448)) with amax >= 2^-126, q = x / 2^e rounded to nearest even,
 * s = clamp(e + 127, 0, 254). K a multiple of 32; row strides in elements (bytes for
 * q and s). */
int hkx_mx_quant(const void* x, int64_t ldx, void* q, int64_t ldq, uint8_t* s, int64_t lds,
                 int32_t m, int32_t k, void* stream);

/* The same as hkx_block_norm quantizes y: for a block with an infinity or a NaN s = 255 (E8M0's NaN)
 * and codes 0 (hkx_mx_quant makes them +-448), and of a block below 2^-119 e is -127, which is what s
 * stands for (there e is less than the s it is clamped to). */
int hkx_mx_quant_nan(const void* x, int64_t ldx, void* q, int64_t ldq, uint8_t* s, int64_t lds,
                     int32_t m, int32_t k, void* stream);

/* ---------------------------------------------------------------- MXFP4, and the block norm */

/* x (M, K) of x_dtype (bf16, fp16, fp32) -> q (M, K/2 bytes) packed e2m1 and s (M, K/32) E8M0
 * bytes: per 32-column block e = ceil(log2(amax / 6)) at least -127, q = x / 2^e rounded to the
 * nearest, ties to the even code, s = e + 127; a block with an infinity or a NaN has s = 255
 * (E8M0's NaN) and codes 0. K a multiple of 32; x's rows 16-byte aligned, q's 4-byte; strides in
 * elements of x and bytes of q and s. */
int hkx_mx4_quant(const void* x, int64_t ldx, int32_t x_dtype, void* q, int64_t ldq, uint8_t* s,
                  int64_t lds, int32_t m, int32_t k, void* stream);

/* The numbers MX values stand for: q (M, K) packed e2m1 (HKX_FP4E2M1) or e4m3 (HKX_FP8E4M3) with s
 * (M, K/32) E8M0 bytes -> y (M, K) of y_dtype, rounded once; a block of scale 255 is NaN. y's rows
 * 16-byte aligned, q's 4-byte (8-byte for e4m3). */
int hkx_mx_dequant(const void* q, int64_t ldq, int32_t q_dtype, const uint8_t* s, int64_t lds,
                   void* y, int64_t ldy, int32_t y_dtype, int32_t m, int32_t k, void* stream);

/* bf16 C (M, N) = (sa . A)(sb . B)^T (+ bias): A (M, K) packed e2m1 or e4m3, B (N, K) packed e2m1,
 * sa (M, K/32) and sb (N, K/32) E8M0 bytes. silu_mul: B has 2N rows, Z = (sa . A)(sb . B)^T (+ bias
 * of 2N) and C = silu(Z[:, :N]) * Z[:, N:]. Sums in fp32, one rounding. Any M and N, K a multiple of
 * 32. Row strides lda, ldb, sa_ld, sb_ld in bytes, ldc in elements; A's and B's rows 16-byte, the
 * scales' anywhere (whole aligned dwords of them are read: up to 3 bytes before the first and past the
 * last). */
#define HKX_MX4_AUTO 0
#define HKX_MX4_TILE64 1  /* 64 x 128 tiles, 4 waves */
#define HKX_MX4_TILE128 2 /* 128 x 128 tiles, 4 waves */
#define HKX_MX4_QUAD 3    /* 256 x 256 tiles, 8 waves, persistent; C under 4 GiB */
#define HKX_MX4_SKINNY 4  /* the decode kernel, 64 rows of C a workgroup; no splits */
typedef struct {
  int32_t size; /* sizeof(HkxMx4GemmArgs): the library refuses another layout */
  int32_t a_dtype;
  const void* a;
  const void* b;
  const uint8_t* sa;
  const uint8_t* sb;
  const void* bias; /* NULL: none */
  void* c;
  int64_t lda, ldb, sa_ld, sb_ld, ldc;
  int32_t m, n, k;
  int32_t bias_dtype; /* HKX_BF16 / HKX_FP16 / HKX_FP32 */
  int32_t silu_mul;
  int32_t kernel; /* HKX_MX4_AUTO, or the kernel to run (tuning, tests) */
  int32_t splits; /* of K, where kernel is given (0: 1); no split is empty */
  int32_t reserved;
  void* ws; /* hkx_mx4_gemm_workspace() bytes, 16-byte aligned; NULL where that is 0 */
  size_t ws_bytes;
} HkxMx4GemmArgs;
int hkx_mx4_gemm(const HkxMx4GemmArgs* args, void* stream);
/* (goes by every size, stride and c's alignment, so these are set first) */
size_t hkx_mx4_gemm_workspace(const HkxMx4GemmArgs* args);

/* Between two blocks, a row at a time: u = x rsqrt(mean x^2 + eps) post (u = x without post), h =
 * residual_scale residual + branch_scale gate u, y = h rsqrt(mean h^2 + eps) pre (no y without pre).
 * x and y of x_dtype (bf16, fp16, fp32), residual and h of r_dtype (the same or fp32), post and pre
 * (d,) of w_dtype and gate of gate_dtype (x's or fp32). The gate's rows, d long (gate_col 1) or one
 * value (0), stand one after another, each for gate_rows rows of x. quant 1: y as MXFP8 (e4m3, ldy
 * bytes a row) with y_scales, 2: as MXFP4, 4: as e4m3 with one fp32 scale a row, as hkx_fp8_quant's
 * (y_scales: rows of float; ldys is not used); d then a multiple of 32 and every row 16-byte aligned (1 and 2).
 * rstd (rows, 2) fp32 keeps the two norms' factors for the backward pass (NULL: not kept). d at most
 * 16384, in the backward pass 8192. Strides in elements. */
typedef struct {
  int32_t size; /* sizeof(HkxBlockNormArgs) */
  int32_t x_dtype, r_dtype, w_dtype, gate_dtype;
  int32_t rows, d;
  int32_t gate_rows, gate_col;
  int32_t quant;
  float branch_scale, residual_scale, eps;
  int32_t reserved;
  const void* x;
  const void* residual;
  const void* post;
  const void* pre;
  const void* gate;
  void* h;
  void* y;
  uint8_t* y_scales;
  float* rstd;
  int64_t ldx, ldr, ldh, ldy, ldys;
} HkxBlockNormArgs;
int hkx_block_norm(const HkxBlockNormArgs* args, void* stream);

/* Its gradients from dh and dy (NULL: zero): dx (x's type), dresidual (its type), dpost and dpre
 * (w_dtype), dgate (the gate's shape and type, summed over the rows and columns it is broadcast
 * over); dpost, dpre and dgate may be NULL. f as in the forward call, with its rstd; f's h, y and
 * y_scales are not used. A run of rows is summed in fp32 and the runs in 64 bits, in a fixed
 * order: the same bits every call. */
typedef struct {
  int32_t size; /* sizeof(HkxBlockNormGradArgs) */
  int32_t reserved;
  HkxBlockNormArgs f;
  const void* dh;
  const void* dy;
  void* dx;
  void* dresidual;
  void* dpost;
  void* dpre;
  void* dgate;
  int64_t lddh, lddy, lddx, lddr;
  void* ws; /* hkx_block_norm_backward_workspace() bytes, 16-byte aligned */
  size_t ws_bytes;
} HkxBlockNormGradArgs;
int hkx_block_norm_backward(const HkxBlockNormGradArgs* args, void* stream);
size_t hkx_block_norm_backward_workspace(const HkxBlockNormGradArgs* args);

/* ---------------------------------------------------------------- experts: rows in groups
 *
 * R rows stand in the order of their experts: rows offsets[e] .. offsets[e + 1] are expert e's (offsets of
 * experts + 1 int32 on the GPU, from 0, at most rows), those behind offsets[experts] are nobody's. A host need not
 * know them: grids are sized for any. Offsets out of order or past the rows are clamped, an index out of range reads
 * zeros: nothing outside the operands is touched. At most 1024 experts and 2^31 - 256
 * rows. */

#define HKX_EXPERTS_NT 0 /* C[r] = A[r or index[r]] . B_e^T, B_e (n, k) */
#define HKX_EXPERTS_NN 1 /* C[r] = A[r] . B_e, B_e (k, n) */
#define HKX_EXPERTS_TN 2 /* C_e = sum of its rows A[r]^T B[r], (m, n) an expert */
typedef struct {
  int32_t size; /* sizeof(HkxExpertsGemmArgs) */
  int32_t op;
  int32_t ab_dtype; /* HKX_BF16; HKX_FP8E4M3 with scales (NT) */
  int32_t experts, rows;
  int32_t a_rows;    /* A's rows, where index names them */
  int32_t m, n, k;   /* n: C's columns; k: the contraction (not TN); m: C's rows an expert (TN) */
  int32_t silu_mul;  /* NT: B_e has n gate rows, then n up rows: C = silu(gate) * up */
  int32_t zero_rest; /* NT, NN: C's rows behind the last group are zeroed, otherwise left */
  int32_t bias_dtype, sa_ld, sb_col; /* sa_ld: 1 a scale a row of A, 0 one; sb_col: 1 a scale a row of B, 0 one an expert */
  int32_t kernel;                    /* HKX_EXPERTS_AUTO, or the kernel to run (tuning, tests) */
  int32_t c_dtype;                   /* HKX_BF16; NN: or HKX_FP32 */
  const void* a;
  const void* b;
  void* c;
  void* z; /* NT with silu_mul: the 2 n columns before it, bf16 (NULL: not kept) */
  const int32_t* offsets;
  const int32_t* index; /* NT: each row's row of A (NULL: its own) */
  const void* bias;     /* NT: (experts, n), 2 n with silu_mul (NULL: none) */
  const float* sa;
  const float* sb;
  int64_t lda, ldb, ldc, ldz;        /* row strides, elements */
  int64_t b_expert, c_expert;        /* strides of an expert, elements (NT, NN: B's; TN: C's) */
  int64_t bias_ld, sb_ld;            /* of the bias and the scales */
  void* ws;                          /* hkx_experts_gemm_workspace() bytes, 16-byte aligned */
  size_t ws_bytes;
} HkxExpertsGemmArgs;
#define HKX_EXPERTS_AUTO 0
#define HKX_EXPERTS_TILE16 1  /* tiles of 16, 64 or 128 rows */
#define HKX_EXPERTS_TILE64 2
#define HKX_EXPERTS_TILE128 3
#define HKX_EXPERTS_QUAD 4 /* 256 x 256 tiles, 8 waves, persistent; C, z and the bias in 16-byte aligned rows */
#define HKX_EXPERTS_SKINNY16 5 /* the decode kernel, 16 or 32 rows (NT; a gradient goes by its size) */
#define HKX_EXPERTS_SKINNY32 6
/* C from bf16 or fp8 operands, sums in fp32, rounded once to bf16 or, in NN with an fp32 C, kept. n and k multiples of 8 (m too; an fp8 k of 16), rows
 * and experts of A and B 16-byte aligned, of C and z 8-byte (an fp32 C 16-byte), of the bias and scales (a row of B
 * each) 16-byte. */
int hkx_experts_gemm(const HkxExpertsGemmArgs* args, void* stream);
/* (goes by every size, stride and address, so these are set first) */
size_t hkx_experts_gemm_workspace(const HkxExpertsGemmArgs* args);

/* dz from dy (rows, n) and z (rows, 2 n), bf16: the gradient of silu(z[:n]) * z[n:]. Rows behind
 * offsets[experts] are left. Rows 16-byte aligned, n a multiple of 8. */
int hkx_experts_silu_grad(const void* z, int64_t ldz, const void* dy, int64_t lddy, void* dz, int64_t lddz,
                          const int32_t* offsets, int32_t experts, int32_t rows, int32_t n, void* stream);

/* db[e] (experts, n) of db_dtype = the sum of its rows of dz (bf16), in 64 bits. */
int hkx_experts_bias_grad(const void* dz, int64_t lddz, const int32_t* offsets, void* db, int32_t db_dtype,
                          int32_t experts, int32_t rows, int32_t n, void* stream);

/* out[r] = x[index[r]] (a_rows rows of k bf16; zeros where index is out of range). */
int hkx_experts_gather(const void* x, int64_t ldx, const int32_t* index, void* out, int64_t ldo, int32_t rows,
                       int32_t a_rows, int32_t k, void* stream);

/* The gradient of x from that of its rows: dx[i] (bf16) = the sum over j of dr[slots[i, j]] (fp32; a slot outside dr's
 * `rows`: nothing), in fp32, in order of j, rounded once. */
int hkx_experts_gather_grad(const float* dr, int64_t lddr, const int32_t* slots, void* dx, int64_t lddx, int32_t t,
                            int32_t k, int32_t rows, int32_t d, void* stream);

/* The k largest of each token's logits (t, e), a tie to the lower expert, NaN above all, -inf never chosen:
 * chosen (t, k) int32 in falling order (-1: none left) and weights (t, k) fp32, their softmax over the token's
 * experts, or with renormalize over the chosen. And the rows of the chosen in order of (expert, token):
 * offsets (e + 1), rows (t k) each row's token (-1 behind the last), slots (t, k) each choice's row (-1: none).
 * e at most 1024, k at most 64 and e. */
typedef struct {
  int32_t size; /* sizeof(HkxExpertsRouteArgs) */
  int32_t dtype; /* the logits' */
  int32_t t, e, k, renormalize;
  const void* logits;
  int64_t ld;
  float* weights;
  int32_t* chosen;
  int32_t* offsets;
  int32_t* rows;
  int32_t* slots;
  void* ws; /* hkx_experts_route_workspace() bytes, 16-byte aligned */
  size_t ws_bytes;
} HkxExpertsRouteArgs;
int hkx_experts_route(const HkxExpertsRouteArgs* args, void* stream);
size_t hkx_experts_route_workspace(const HkxExpertsRouteArgs* args);

/* The logits' gradient (t, e) of `dtype` from dweights (t, k) fp32 and the forward call's chosen and weights. */
int hkx_experts_route_backward(const void* logits, int64_t ld, int32_t dtype, const float* weights,
                               const int32_t* chosen, const float* dweights, void* dlogits, int64_t lddl, int32_t t,
                               int32_t e, int32_t k, int32_t renormalize, void* stream);

/* out[i] = sum over j of weights[i, j] y[slots[i, j]] (weights NULL: ones; a slot outside y's `rows`: nothing), in fp32,
 * in order of j; out (t, d) and y of `dtype`. */
int hkx_experts_combine(const void* y, int64_t ldy, int32_t dtype, const int32_t* slots, const float* weights,
                        void* out, int64_t ldo, int32_t t, int32_t k, int32_t rows, int32_t d, void* stream);

/* dy[r] = the sum of weights[i, j] dout[i] over the slots[i, j] that name row r, in fp32 and in their order (zeros where none
 * does), and dweights[i, j] = <dout[i], y[slots[i, j]]>, 0 of no row. rows = t k. Either may be NULL: not wanted (without
 * dweights y may be NULL, without dy `ws`, 8 bytes of 4-byte aligned scratch memory a row). */
int hkx_experts_combine_backward(const void* y, int64_t ldy, const void* dout, int64_t lddo, int32_t dtype,
                                 const int32_t* slots, const float* weights, void* dy, int64_t lddy, float* dweights,
                                 void* ws, int32_t t, int32_t k, int32_t rows, int32_t d, void* stream);

/* x (m, k) of x_dtype -> q (m, k) e4m3 and s (m) fp32: s = max |x| / 448 of the row (at least 2^-126; 1 for a row of
 * zeros), q = x / s rounded to nearest even. A row with an infinity or a NaN has s = NaN and codes 0. Any k and
 * alignment of whole elements (16 bytes of x, 8 of q and k a multiple of 8: pieces of 8). */
int hkx_fp8_quant(const void* x, int64_t ldx, int32_t x_dtype, void* q, int64_t ldq, float* s, int32_t m, int32_t k,
                  void* stream);

#ifdef __cplusplus
}
#endif

#endif /* HKX_H_ */
