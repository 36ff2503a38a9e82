/*
 * gemmkit_cuda.h -- C ABI of the B200 (sm_100a) engine for gemmkit's quantized-inference
 * GEMM path.
 *
 * Every entry mirrors a gemmkit (Rust, v0.1.2) API function: same name after the `gk_`
 * prefix, same argument order and meaning (element strides as signed `ptrdiff_t`, `rs`/`cs`
 * views, `beta == 0` never reads C), plus a trailing CUDA stream. Pointers are DEVICE
 * pointers. Calls are asynchronous on `stream` (NULL = the legacy default stream); they
 * never unwind and return a status code. Where gemmkit panics with a `gemmkit:` message,
 * the entry returns GK_EINVAL and gk_last_error() returns the same message.
 *
 * Two tiers, as in gemmkit:
 *   - checked entries take gk_matref / gk_matmut views (a slice length plus rows, cols and
 *     strides, exactly MatRef / MatMut, gemmkit/src/api.rs:99-118) and run gemmkit's
 *     validation (gemmkit/src/api.rs:188-315, gemmkit/src/adapter.rs:190-280);
 *   - `_unchecked` entries take raw pointers and strides (negative strides allowed) and
 *     trust the caller, as gemmkit's `*_unchecked` functions do.
 *
 * Extensions beyond gemmkit (no counterpart there, see the notes on each): independent
 * bias / scale axes and ReLU in the requant descriptor, packed-B requant entries, i8
 * batched entries, and the f32-output bf16/f16 GEMM.
 */
#ifndef GEMMKIT_CUDA_H
#define GEMMKIT_CUDA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes. */
enum {
    GK_OK = 0,
    GK_EINVAL = 1,   /* argument rejected (the gemmkit panic cases) */
    GK_ENOMEM = 2,   /* device allocation failed */
    GK_ECUDA = 3,    /* a CUDA runtime/driver call failed */
    GK_ETIMEOUT = 4, /* a bounded device wait gave up (see gk_device_status) */
    GK_ENODEV = 5,   /* no sm_100 device, or the kernels are not loadable */
};

typedef void *gk_stream_t; /* a cudaStream_t */

/* gemmkit::Parallelism (gemmkit/src/parallel.rs:25-39). On the device the engine always
 * uses the whole GPU; the value is accepted for API parity and otherwise ignored. */
typedef enum { GK_PAR_SERIAL = 0, GK_PAR_RAYON = 1 } gk_par_kind;
typedef struct {
    int32_t kind;    /* gk_par_kind */
    int32_t threads; /* Rayon(n): n; 0 = all */
} gk_parallelism;

/* gemmkit::Workspace (gemmkit/src/workspace.rs:53-190): reusable device scratch for the
 * operand packs a call may need. NULL selects a per-thread, per-device default. */
typedef struct gk_workspace gk_workspace;

/* gemmkit::PackedRhs<i8> (gemmkit/src/api/packed.rs:34-41): B packed once on the device
 * into the engine's K-major tile layout, read-only, shareable across streams. */
typedef struct gk_packed_rhs gk_packed_rhs;

/* Checked views: element (i, j) at data[i*rs + j*cs]; `len` is the slice length in
 * elements (gemmkit MatRef / MatMut, gemmkit/src/api.rs:99-118). */
typedef struct {
    const void *data;
    size_t len;
    size_t rows, cols;
    ptrdiff_t rs, cs;
} gk_matref;
typedef struct {
    void *data;
    size_t len;
    size_t rows, cols;
    ptrdiff_t rs, cs;
} gk_matmut;

/* Requant axis of a bias or scale vector, in the user's (row, col) frame. */
typedef enum { GK_AXIS_NONE = 0, GK_AXIS_ROW = 1, GK_AXIS_COL = 2 } gk_axis;

/* Extended requant descriptor (extension of gemmkit::Requantize,
 * gemmkit/src/api/int8.rs:185-209): gemmkit ties bias and scales to the row axis; here each
 * has its own axis (per-row, per-column, or none / per-tensor), and `relu` raises the
 * lower clamp to clamp(zero_point), which equals requantizing max(acc + bias, 0). */
typedef struct {
    float scale;           /* per-tensor scale, used when scale_axis == GK_AXIS_NONE */
    const float *scales;   /* device vector, length m (ROW) or n (COL) */
    int32_t scale_axis;    /* gk_axis */
    int32_t zero_point;    /* [-128, 127] for i8 output, [0, 255] for u8 */
    const int32_t *bias;   /* device vector, length m (ROW) or n (COL); NULL = none */
    int32_t bias_axis;     /* gk_axis */
    int32_t relu;          /* nonzero: ReLU before requantization */
    size_t scales_len;     /* checked tier only: slice lengths of scales / bias */
    size_t bias_len;
} gk_requant;

/* ---- library -------------------------------------------------------------------------- */

const char *gk_version(void);
/* Thread-local text of the last error returned by an entry on this thread. */
const char *gk_last_error(void);
/* Read (and with clear != 0 reset) the device status word of `device`. GK_STATUS_OFFSETS means a
 * grouped call's offsets did not ascend inside its rows (the call ran on the offsets made safe,
 * see gk_gemm_half_grouped); any other bit that a bounded in-kernel wait gave up (GK_ETIMEOUT).
 * Synchronizes the device. */
#define GK_STATUS_OFFSETS (1u << 5)
int gk_device_status(int device, int clear, uint32_t *status);

int gk_workspace_create(gk_workspace **out);
void gk_workspace_free(gk_workspace *ws);

/* ---- i8 -> i32 ----------------------------------------------------------------------- */

/* gemm_i8_unchecked_with (gemmkit/src/api/int8.rs:136-178):
 * C(i32) <- alpha*A(i8)*B(i8) + beta*C, wrapping on overflow. */
int gk_gemm_i8_unchecked(gk_workspace *ws, size_t m, size_t k, size_t n, int32_t alpha,
                         const int8_t *a, ptrdiff_t rsa, ptrdiff_t csa, const int8_t *b,
                         ptrdiff_t rsb, ptrdiff_t csb, int32_t beta, int32_t *c, ptrdiff_t rsc,
                         ptrdiff_t csc, gk_parallelism par, gk_stream_t stream);

/* gemm_i8_with (gemmkit/src/api/int8.rs:38-84): validate_gemm_views, then the above. */
int gk_gemm_i8(gk_workspace *ws, int32_t alpha, gk_matref a, gk_matref b, int32_t beta,
               gk_matmut c, gk_parallelism par, gk_stream_t stream);

/* ---- i8 -> i8 / u8 requantized ------------------------------------------------------- */

/* gemm_i8_requant_unchecked_with (gemmkit/src/api/int8.rs:404-457):
 * C(i8) <- clamp(zp + round_ne(scale*(A*B + bias[i])), -128, 127), f64 scale step. */
int gk_gemm_i8_requant_unchecked(gk_workspace *ws, size_t m, size_t k, size_t n,
                                 const int8_t *a, ptrdiff_t rsa, ptrdiff_t csa, const int8_t *b,
                                 ptrdiff_t rsb, ptrdiff_t csb, float scale,
                                 const float *row_scales, int has_row_scales, int32_t zero_point,
                                 const int32_t *bias, int has_bias, int8_t *c, ptrdiff_t rsc,
                                 ptrdiff_t csc, gk_parallelism par, gk_stream_t stream);

/* gemm_i8_requant_u8_unchecked_with (gemmkit/src/api/int8.rs:619-672): u8 output [0, 255]. */
int gk_gemm_i8_requant_u8_unchecked(gk_workspace *ws, size_t m, size_t k, size_t n,
                                    const int8_t *a, ptrdiff_t rsa, ptrdiff_t csa,
                                    const int8_t *b, ptrdiff_t rsb, ptrdiff_t csb, float scale,
                                    const float *row_scales, int has_row_scales,
                                    int32_t zero_point, const int32_t *bias, int has_bias,
                                    uint8_t *c, ptrdiff_t rsc, ptrdiff_t csc, gk_parallelism par,
                                    gk_stream_t stream);

/* gemm_i8_requant_with / gemm_i8_requant_u8_with (gemmkit/src/api/int8.rs:280-338,
 * 495-552): the checked tier with gemmkit's validation and wording (per-row scales and bias
 * when the descriptor's axes are ROW; other axes are the extension). out_u8 selects the u8
 * entry. */
int gk_gemm_i8_requant(gk_workspace *ws, gk_matref a, gk_matref b, const gk_requant *req,
                       gk_matmut c, int out_u8, gk_parallelism par, gk_stream_t stream);

/* Extension: the raw tier with the extended descriptor (independent axes, ReLU). */
int gk_gemm_i8_requant_ex_unchecked(gk_workspace *ws, size_t m, size_t k, size_t n,
                                    const int8_t *a, ptrdiff_t rsa, ptrdiff_t csa,
                                    const int8_t *b, ptrdiff_t rsb, ptrdiff_t csb,
                                    const gk_requant *req, void *c, ptrdiff_t rsc, ptrdiff_t csc,
                                    int out_u8, gk_parallelism par, gk_stream_t stream);

/* ---- prepacked B ------------------------------------------------------------------------ */

/* prepack_rhs_i8_unchecked (gemmkit/src/api/packed.rs:386-453): pack a k x n device B once;
 * the pack runs on `stream`. */
int gk_prepack_rhs_i8_unchecked(const int8_t *b, ptrdiff_t rsb, ptrdiff_t csb, size_t k,
                                size_t n, gk_stream_t stream, gk_packed_rhs **out);
/* prepack_rhs_i8 (gemmkit/src/api/packed.rs:372-384): check_view on B, then the above. */
int gk_prepack_rhs_i8(gk_matref b, gk_stream_t stream, gk_packed_rhs **out);
void gk_packed_rhs_free(gk_packed_rhs *p);
size_t gk_packed_rhs_rows(const gk_packed_rhs *p); /* PackedRhs::rows (k) */
/* No counterpart in gemmkit (its PackedRhs lives only in memory): store a packed B and load it
 * back, so weights are packed once and later loaded device-ready. gk_packed_rhs_serialize
 * writes a 64-byte header (magic "GKPACK01", k, n, padded dimensions, layout tag) plus the
 * packed bytes into host memory `out` of `cap` bytes (out == NULL: only set *needed).
 * gk_packed_rhs_deserialize checks the header (magic, layout, dimensions, length) and returns
 * a new handle on the current device, complete when it returns. */
int gk_packed_rhs_serialize(const gk_packed_rhs *p, void *out, size_t cap, size_t *needed);
int gk_packed_rhs_deserialize(const void *in, size_t len, gk_stream_t stream,
                              gk_packed_rhs **out);
size_t gk_packed_rhs_cols(const gk_packed_rhs *p); /* PackedRhs::cols (n) */

/* gemm_i8_packed_b_unchecked_with (gemmkit/src/api/packed.rs:609-680): C(i32) <- alpha *
 * A * packedB + beta*C. Like gemmkit, rejects a C that is not column-major-ish
 * (|csc| < |rsc|) with gemmkit's message. */
int gk_gemm_i8_packed_b_unchecked(gk_workspace *ws, int32_t alpha, size_t m, const int8_t *a,
                                  ptrdiff_t rsa, ptrdiff_t csa, const gk_packed_rhs *packed,
                                  int32_t beta, int32_t *c, ptrdiff_t rsc, ptrdiff_t csc,
                                  gk_parallelism par, gk_stream_t stream);
/* gemm_i8_packed_b_with (gemmkit/src/api/packed.rs:493-571). */
int gk_gemm_i8_packed_b(gk_workspace *ws, int32_t alpha, gk_matref a,
                        const gk_packed_rhs *packed, int32_t beta, gk_matmut c,
                        gk_parallelism par, gk_stream_t stream);

/* Extension (gemmkit has no packed requant entry; dispatch/int.rs:5): requantized product
 * with a prepacked B, any C orientation. Bit-identical to gk_gemm_i8_requant_ex_unchecked
 * on the unpacked B. Small m takes the bandwidth-bound small-M kernel shape. */
int gk_gemm_i8_packed_b_requant_unchecked(gk_workspace *ws, size_t m, const int8_t *a,
                                          ptrdiff_t rsa, ptrdiff_t csa,
                                          const gk_packed_rhs *packed, const gk_requant *req,
                                          void *c, ptrdiff_t rsc, ptrdiff_t csc, int out_u8,
                                          gk_parallelism par, gk_stream_t stream);

/* The decode-step GEMV. gemmkit reaches its small-shape route only from inside dispatch
 * (special/small_mn.rs:834-1060, gated at dispatch.rs:438-482); this entry names it:
 * C = requant(A * packedB) for 1 <= m <= 64 activation rows. When the packed side is the
 * wider one (n > m) this runs on the bandwidth-bound small-M kernel that streams the
 * prepacked weights once from HBM (unless GEMMKIT_CUDA_GEMV=0); when n <= m both sides are
 * at most 64 wide and the product goes to the general tile kernel. Arguments and results as
 * gk_gemm_i8_packed_b_requant_unchecked; m outside [1, 64] is GK_EINVAL. */
int gk_gemv_i8_requant_unchecked(gk_workspace *ws, size_t m, const int8_t *a, ptrdiff_t rsa,
                                 ptrdiff_t csa, const gk_packed_rhs *packed,
                                 const gk_requant *req, void *c, ptrdiff_t rsc, ptrdiff_t csc,
                                 int out_u8, gk_stream_t stream);

/* ---- batched (extension: gemmkit's batched entries are float-only, api/batched.rs:188) -- */

/* Strided batch of independent requantized products, shaped as gemmkit's
 * gemm_batched_unchecked_with (gemmkit/src/api/batched.rs:649): element e uses
 * A + e*a_bs, B + e*b_bs, C + e*c_bs, and the bias / scales vectors at + e*bias_bs /
 * + e*scales_bs (0 = shared by every element). */
int gk_gemm_i8_requant_batched_unchecked(gk_workspace *ws, size_t batch, size_t m, size_t k,
                                         size_t n, const int8_t *a, ptrdiff_t rsa, ptrdiff_t csa,
                                         ptrdiff_t a_bs, const int8_t *b, ptrdiff_t rsb,
                                         ptrdiff_t csb, ptrdiff_t b_bs, const gk_requant *req,
                                         ptrdiff_t bias_bs, ptrdiff_t scales_bs, void *c,
                                         ptrdiff_t rsc, ptrdiff_t csc, ptrdiff_t c_bs, int out_u8,
                                         gk_parallelism par, gk_stream_t stream);

/* Pointer-array batch, shaped as gemm_batched_ptr_unchecked over GemmProblem
 * (gemmkit/src/api/batched.rs:711-760, gemmkit/src/dispatch.rs:135). */
typedef struct {
    size_t m, k, n;
    const int8_t *a;
    ptrdiff_t rsa, csa;
    const int8_t *b;
    ptrdiff_t rsb, csb;
    void *c;
    ptrdiff_t rsc, csc;
    gk_requant req;
} gk_i8_requant_problem;
int gk_gemm_i8_requant_batched_ptr_unchecked(gk_workspace *ws,
                                             const gk_i8_requant_problem *problems,
                                             size_t count, int out_u8, gk_parallelism par,
                                             gk_stream_t stream);

/* ---- half -> f32 (extension: gemmkit's gemm::<bf16> writes bf16, dispatch/mixed.rs:1395;
 * its f32-output family is the internal deep-k twin, dispatch/mixed.rs:97-221) ---------- */

/* C(f32) <- alpha*A*B + beta*C with bf16 (or f16) A and B, f32 accumulation; beta == 0
 * never reads C. Argument order as gemm_unchecked (gemmkit/src/api.rs:469). */
int gk_gemm_bf16_f32_unchecked(gk_workspace *ws, size_t m, size_t k, size_t n, float alpha,
                               const uint16_t *a, ptrdiff_t rsa, ptrdiff_t csa,
                               const uint16_t *b, ptrdiff_t rsb, ptrdiff_t csb, float beta,
                               float *c, ptrdiff_t rsc, ptrdiff_t csc, gk_parallelism par,
                               gk_stream_t stream);
int gk_gemm_f16_f32_unchecked(gk_workspace *ws, size_t m, size_t k, size_t n, float alpha,
                              const uint16_t *a, ptrdiff_t rsa, ptrdiff_t csa, const uint16_t *b,
                              ptrdiff_t rsb, ptrdiff_t csb, float beta, float *c, ptrdiff_t rsc,
                              ptrdiff_t csc, gk_parallelism par, gk_stream_t stream);
/* Checked tier (gemm_with, gemmkit/src/api.rs:400-466 validation). is_f16 selects f16. */
int gk_gemm_half_f32(gk_workspace *ws, int is_f16, float alpha, gk_matref a, gk_matref b,
                     float beta, gk_matmut c, gk_parallelism par, gk_stream_t stream);

/* Strided batch of half -> f32 products (gemm_batched_unchecked_with shape,
 * gemmkit/src/api/batched.rs:649). */
int gk_gemm_half_f32_batched_unchecked(gk_workspace *ws, int is_f16, size_t batch, size_t m,
                                       size_t k, size_t n, float alpha, const uint16_t *a,
                                       ptrdiff_t rsa, ptrdiff_t csa, ptrdiff_t a_bs,
                                       const uint16_t *b, ptrdiff_t rsb, ptrdiff_t csb,
                                       ptrdiff_t b_bs, float beta, float *c, ptrdiff_t rsc,
                                       ptrdiff_t csc, ptrdiff_t c_bs, gk_parallelism par,
                                       gk_stream_t stream);

/* ---- fused float epilogue on the half -> f32 GEMM ------------------------------------- */

/* gemmkit's gemm_fused (gemmkit/src/api/fused.rs:149-176) computes act(alpha*A*B + beta*C +
 * bias) for f32/f64 GEMMs: the bias per row (length m) or per column (length n), then ReLU or
 * LeakyReLU(slope) (gemmkit/src/kernel/epilogue.rs:258-330). These entries give the bf16 /
 * f16 -> f32 GEMM the same fused epilogue (gemmkit has none for half inputs): the unchecked
 * tier takes gemm_fused_unchecked's (bias, bias_dim, has_bias, act) selectors, the checked
 * tier validates the views like gk_gemm_half_f32 and the bias length like gemmkit. With k == 0
 * or alpha == 0, C <- act(beta*C + bias) (gemmkit/src/dispatch/float.rs:671-676). */
enum gk_act { GK_ACT_NONE = 0, GK_ACT_RELU = 1, GK_ACT_LEAKY_RELU = 2 };
int gk_gemm_half_f32_fused_unchecked(gk_workspace *ws, int is_f16, size_t m, size_t k, size_t n,
                                     float alpha, const uint16_t *a, ptrdiff_t rsa,
                                     ptrdiff_t csa, const uint16_t *b, ptrdiff_t rsb,
                                     ptrdiff_t csb, float beta, float *c, ptrdiff_t rsc,
                                     ptrdiff_t csc, const float *bias, int bias_dim,
                                     int has_bias, int act, float leak, gk_parallelism par,
                                     gk_stream_t stream);
int gk_gemm_half_f32_fused(gk_workspace *ws, int is_f16, float alpha, gk_matref a, gk_matref b,
                           float beta, gk_matmut c, const float *bias, size_t bias_len,
                           int bias_dim, int act, float leak, gk_parallelism par,
                           gk_stream_t stream);

/* ---- fused i32 epilogue on the i8 -> i32 GEMM ------------------------------------------ */

/* The integer counterpart of gk_gemm_half_f32_fused: C = act(alpha*A*B + beta*C + bias) with
 * i8 operands and i32 C, every step wrapping mod 2^32 as gemmkit's int32_epilogue does
 * (gemmkit/src/kernel/int.rs:36-120), the i32 bias per row (length m) or per column (length
 * n), then ReLU as max(v, 0) on the signed value. gemmkit's FusedEpi (gemmkit/src/kernel/
 * epilogue.rs:258-330) composes bias-then-activation for float GEMMs only; this entry applies
 * the same composition to gemm_i8 (gemmkit/src/api/int8.rs:136-178) inside the GEMM's
 * epilogue. act is GK_ACT_NONE or GK_ACT_RELU (GK_ACT_LEAKY_RELU is GK_EINVAL: its slope is a
 * float). With k == 0 or alpha == 0, C <- act(beta*C + bias). The checked tier validates the
 * views like gk_gemm_i8 and the bias length like gk_gemm_half_f32_fused. */
int gk_gemm_i8_fused_unchecked(gk_workspace *ws, size_t m, size_t k, size_t n, int32_t alpha,
                               const int8_t *a, ptrdiff_t rsa, ptrdiff_t csa, const int8_t *b,
                               ptrdiff_t rsb, ptrdiff_t csb, int32_t beta, int32_t *c,
                               ptrdiff_t rsc, ptrdiff_t csc, const int32_t *bias, int bias_dim,
                               int has_bias, int act, gk_parallelism par, gk_stream_t stream);
int gk_gemm_i8_fused(gk_workspace *ws, int32_t alpha, gk_matref a, gk_matref b, int32_t beta,
                     gk_matmut c, const int32_t *bias, size_t bias_len, int bias_dim, int act,
                     gk_parallelism par, gk_stream_t stream);

/* ---- products of rows grouped by expert (no counterpart in gemmkit) -------------------- */

/* Element types of the entries below. */
typedef enum { GK_F32 = 0, GK_F16 = 1, GK_BF16 = 2 } gk_dtype;

/* The experts' products of a mixture-of-experts layer: the rows of A and C are sorted by group
 * (expert), group g being the rows offsets[g] <= i < offsets[g + 1], and
 *   C[i, :] <- alpha * A[i, :] * B[g] + beta * C[i, :].
 * `offsets` is a DEVICE array of groups + 1 int32 (1 <= groups <= 1024) that the host never reads,
 * so a router may still be writing it on the same stream. It must ascend inside [0, A.rows];
 * the kernels use its running maximum clamped to that range, so no offset reaches outside the
 * buffers, and an array that had to be changed sets GK_STATUS_OFFSETS in the device status word.
 * A group may be empty; rows of C before the first and past the last offset are left as they are.
 * A (rows x k) and B (k x n, group g at + g * b_gs elements; b_gs == 0: one B for every group)
 * are bf16, or f16 with is_f16; C is f32 or the operands' type (out_type), computed in f32 and
 * rounded once. beta == 0 never reads C; k == 0 or alpha == 0 is C <- beta * C on the groups'
 * rows and reads neither A nor B. Any non-negative strides. An A with unit column stride and a B
 * with a unit row or column stride, 16-byte aligned and every other stride a multiple of 16 bytes,
 * are read in place (in the weight gradient A and B with unit column strides); other operands
 * are first copied to aligned scratch, stream-ordered memory of the operand's size (all groups of
 * B) from a pool of the engine's, which keeps at most 1/64 of the device's memory past the next
 * synchronisation (see gk_scratch_release). In a capture the scratch is the graph's own.
 * The gradient of A is the same call with C's gradient as A and B viewed transposed. Calls may
 * be captured and may run on several streams at once. */
int gk_gemm_half_grouped(int is_f16, size_t groups, const int32_t *offsets, float alpha,
                         gk_matref a, gk_matref b, ptrdiff_t b_gs, float beta, gk_matmut c,
                         int out_type, gk_parallelism par, gk_stream_t stream);
/* The weight gradient: C[g] <- alpha * A_g^T * B_g + beta * C[g] with A (rows x m) and B (rows x
 * n) grouped as above, A_g the rows of group g, and C[g] (m x n) at + g * c_gs elements. The
 * contraction runs over the group's rows; an empty group's C[g] becomes beta * C[g] (zeros when
 * beta == 0). Rows of A and B outside the groups are never used, whatever they hold. Each
 * group of C must end before the next begins. */
int gk_gemm_half_grouped_wgrad(int is_f16, size_t groups, const int32_t *offsets, float alpha,
                               gk_matref a, gk_matref b, float beta, gk_matmut c, ptrdiff_t c_gs,
                               int out_type, gk_parallelism par, gk_stream_t stream);
/* Gives the scratch that the two entries above keep on `device` back to it; synchronizes the
 * device when there is any. Not during a capture. */
int gk_scratch_release(int device);

/* ---- microscaled 4-bit floating point (no counterpart in gemmkit) ----------------------- */

/* Formats: e2m1 elements (0, 0.5, 1, 1.5, 2, 3, 4, 6 and negatives) in blocks of consecutive
 * elements of a row that share a scale.
 *   GK_FP4_MX  blocks of 32, scale 2^(floor(log2 amax) - 2) (e8m0);
 *   GK_FP4_NV  blocks of 16, scale e4m3(amax / (6 * s)) times a per-matrix f32 scale s.
 * An element is x / (block scale [* s]) rounded to the nearest e2m1 value, ties to even, saturating
 * at 6; decisions are exact (as if in infinite precision). A block that holds an infinity or a NaN
 * gets a NaN scale: its values, and every product with them, are NaN. */
typedef enum { GK_FP4_MX = 0, GK_FP4_NV = 1 } gk_fp4_format;

/* A rows x cols matrix in 4 bits, quantised along its columns (the contraction of a product), in
 * device memory that the caller owns: `data` holds the codes, `scales` the scales in the engine's
 * tile order (both 16-byte aligned; sizes from gk_fp4_data_bytes / gk_fp4_scale_bytes).
 * The rows form `groups` groups: equal ones (a stack of matrices, offsets == NULL; groups == 1 for
 * a plain matrix), or ragged ones given by a device array of groups + 1 offsets as in
 * gk_gemm_half_grouped. The scales are laid out per group, so a matrix must be read with the
 * groups it was written with. `scale` is the nv format's s (2^-100 .. 2^100); 1 for mx. */
typedef struct {
    int32_t fmt;            /* gk_fp4_format */
    float scale;
    size_t groups;
    const int32_t *offsets; /* device, groups + 1 entries, or NULL */
    size_t rows, cols;
    uint8_t *data;
    size_t data_len;        /* bytes */
    uint8_t *scales;
    size_t scales_len;      /* bytes */
} gk_fp4_matrix;

size_t gk_fp4_data_bytes(size_t rows, size_t cols);
/* ragged: nonzero when the rows are grouped by offsets. */
size_t gk_fp4_scale_bytes(int fmt, size_t groups, int ragged, size_t rows, size_t cols);

/* Quantize x (f32, f16 or bf16 by x_type, a gk_dtype; any non-negative strides) into dst. For a
 * stack x views group 0's rows and the groups lie x_gs elements apart; otherwise x_gs is
 * unused. Rows outside ragged groups are neither read nor written. */
int gk_quantize_fp4(gk_matref x, int x_type, ptrdiff_t x_gs, const gk_fp4_matrix *dst,
                    gk_stream_t stream);
/* The f32 values that q stands for (one rounding, by s, in the nv format). */
int gk_dequantize_fp4(const gk_fp4_matrix *q, gk_matmut out, gk_stream_t stream);
/* A 4-bit matrix from plain row-major parts, as checkpoints hold them: codes two a byte (the
 * first in the low nibble) at codes_ld bytes a row, one scale byte a block (e8m0, or e4m3 without
 * sign) at scales_ld bytes a row. */
int gk_fp4_import(const uint8_t *codes, size_t codes_len, size_t codes_ld, const uint8_t *scales,
                  size_t scales_len, size_t scales_ld, const gk_fp4_matrix *dst,
                  gk_stream_t stream);

/* C <- alpha * A * B^T + beta * C with A (rows x k) and B (n x k per group) in 4 bits and the same
 * format, on the block-scaled tensor cores with f32 accumulation; C (rows x n) is f32, f16 or bf16
 * (out_type, a gk_dtype), rounded once. With groups, row i of A's group g is multiplied by B's
 * g-th matrix: A's groups may be ragged (a device array, as in gk_gemm_half_grouped, with the same
 * rules for its contents and for rows outside the groups) or equal, B's are equal; both have the
 * same number. beta == 0 never reads C; k == 0 or alpha == 0 is C <- beta * C. The product of
 * alpha and the two matrix scales must be a normal f32 number (or alpha 0, infinite or NaN).
 * Needs no workspace, allocates nothing and may be captured. */
int gk_gemm_fp4(float alpha, const gk_fp4_matrix *a, const gk_fp4_matrix *b, float beta,
                gk_matmut c, int out_type, gk_parallelism par, gk_stream_t stream);

/* ---- producer step: f32 activations -> i8 (no counterpart in gemmkit) ---------------- */

/* Quantize a rows x cols f32 view (element (i, j) at x[i*rsx + j*csx]) into i8 (q[i*rsq +
 * j*csq]), the step that feeds the requantizing GEMMs: q = saturate_i8(zp +
 * round_half_even(f64(x) / f64(scale))) in f64, NaN -> zp. With row_scales == NULL one
 * per-tensor scale / zero_point (scale must be finite and > 0, zp in [-128, 127], as
 * gemmkit's requant checks them); otherwise each row gets scale_r = max |x_r| / 127 (1 for an
 * all-zero row), written to row_scales[i], with zero point 0 (symmetric, per token). */
int gk_quantize_f32_i8_unchecked(size_t rows, size_t cols, const float *x, ptrdiff_t rsx,
                                 ptrdiff_t csx, int8_t *q, ptrdiff_t rsq, ptrdiff_t csq,
                                 float scale, int32_t zero_point, float *row_scales,
                                 gk_stream_t stream);

/* ---- tuning (the gemmkit-tune profile mechanism, gemmkit/src/tuning.rs:592-621) ------- */

/* Force the tile width (N of the MMA: 16, 32, 64, 128, 192 or 256) for later calls on this
 * thread; 0 drops this thread's override, so the process-wide GEMMKIT_CUDA_BN knob applies
 * again (its default, 0, chooses the width per shape). */
int gk_set_tile_n(int bn);

/* The engine's knobs, the counterpart of gemmkit's tuning getters / setters
 * (gemmkit/src/tuning.rs:660-690): a compiled default, an environment override read once
 * (`export GEMMKIT_CUDA_...=v`, the form the tuner's profile uses) and a process-wide run-time
 * override. gk_knob_names lists them (comma-separated): GEMMKIT_CUDA_BN (0 = per shape, or 16,
 * 32, 64, 128, 192, 256), GEMMKIT_CUDA_PAIR, GEMMKIT_CUDA_GEMV, GEMMKIT_CUDA_PDL,
 * GEMMKIT_CUDA_STREAMK, GEMMKIT_CUDA_GEMV_SK, GEMMKIT_CUDA_EPI16, GEMMKIT_CUDA_MN_B,
 * GEMMKIT_CUDA_REQUANT_F32 (0 / 1),
 * GEMMKIT_CUDA_BN_SHORTK (as GEMMKIT_CUDA_BN), GEMMKIT_CUDA_STAGES (0 or 2 .. 12) and
 * GEMMKIT_CUDA_GEMV_SPLIT (0 .. 8). gk_knob_set with a negative value drops the run-time override;
 * an unknown name or an out-of-range value returns GK_EINVAL. */
const char *gk_knob_names(void);
int gk_knob_get(const char *name, int64_t *value);
int gk_knob_set(const char *name, int64_t value);

/* ---- i8 -> i32 without allocation ------------------------------------------------------ */

/* No counterpart in gemmkit. The i8 -> i32 product of gk_gemm_i8_unchecked (same arguments
 * minus the workspace and Parallelism, same result bytes) for callers that must not
 * allocate device memory: hosts that give the GPU a fixed budget through their own
 * allocator, or latency-critical loops where cudaMalloc / cudaFree could synchronise the
 * device. Operands that need packing (not K-contiguous or not 16-byte aligned) are packed
 * into one file-scope device array of GK_NOALLOC_SCRATCH_BYTES, which every GPU that loads
 * the library holds until exit; a call whose packs need more returns GK_EINVAL. The first
 * call on a device looks up that array's device address; make it before any stream capture.
 * All calls share the array: calls that overlap on the GPU race, so order them on one
 * stream. Never calls cudaMalloc, cudaFree or an allocating library routine. */
#define GK_NOALLOC_SCRATCH_BYTES (16u << 20)
int gk_gemm_i8_noalloc_unchecked(size_t m, size_t k, size_t n, int32_t alpha, const int8_t *a,
                                 ptrdiff_t rsa, ptrdiff_t csa, const int8_t *b, ptrdiff_t rsb,
                                 ptrdiff_t csb, int32_t beta, int32_t *c, ptrdiff_t rsc,
                                 ptrdiff_t csc, gk_stream_t stream);

/* ---- sharding across the GPUs of one node (no counterpart in gemmkit) ------------------ */

/* gemmkit runs in one process. For the sharded paths each GPU has its own process; a device
 * buffer of one process is exported as a CUDA IPC handle plus the pointer's offset inside its
 * allocation, and the other processes of the node map it (a plain peer mapping over NVLink).
 * gk_ipc_open reference-counts mappings of one allocation; gk_ipc_close releases one. */
typedef struct gk_ipc_handle {
    unsigned char bytes[64];
    uint64_t offset;
} gk_ipc_handle;
int gk_ipc_export(const void *dev_ptr, gk_ipc_handle *out);
int gk_ipc_open(const gk_ipc_handle *h, void **peer_ptr);
int gk_ipc_close(void *peer_ptr);

/* Mirrored outputs: the product of gk_gemm_bf16_f32_unchecked / gk_gemm_f16_f32_unchecked
 * (is_f16 selects), whose epilogue also stores every element of C at the same offset from
 * each of `mirrors[0 .. nmirror)` (nmirror <= 7; usually peer GPUs' copies of C mapped with
 * gk_ipc_open). This is the column-sharded wide GEMM with C replicated: each GPU computes
 * its block of columns and writes it into every GPU's C in the same kernel, tile by tile,
 * instead of a separate all-gather. beta reads only the local C. Needs k > 0 and
 * alpha != 0 (GK_EINVAL otherwise). The mirrors are complete once the kernel has finished
 * and the caller has synchronised with the other GPUs (for example an NCCL barrier on the
 * same stream). */
int gk_gemm_half_f32_mirrored_unchecked(gk_workspace *ws, int is_f16, size_t m, size_t k,
                                        size_t n, float alpha, const uint16_t *a, ptrdiff_t rsa,
                                        ptrdiff_t csa, const uint16_t *b, ptrdiff_t rsb,
                                        ptrdiff_t csb, float beta, float *c, ptrdiff_t rsc,
                                        ptrdiff_t csc, void *const *mirrors, int nmirror,
                                        gk_stream_t stream);
/* The same for the requantizing i8 product: gk_gemm_i8_requant_batched_unchecked's arguments
 * (batch >= 1; bias_bs / scales_bs the per-element strides of bias and scales), optionally
 * with a prepacked B instead of (b, rsb, csb, b_bs) (then batch must be 1), plus mirrors.
 * The batch-sharded path uses it to replicate each GPU's slice of a batch. */
int gk_gemm_i8_requant_mirrored_unchecked(gk_workspace *ws, size_t batch, size_t m, size_t k,
                                          size_t n, const int8_t *a, ptrdiff_t rsa,
                                          ptrdiff_t csa, ptrdiff_t a_bs, const int8_t *b,
                                          ptrdiff_t rsb, ptrdiff_t csb, ptrdiff_t b_bs,
                                          const gk_packed_rhs *packed, const gk_requant *req,
                                          ptrdiff_t bias_bs, ptrdiff_t scales_bs, void *c,
                                          ptrdiff_t rsc, ptrdiff_t csc, ptrdiff_t c_bs,
                                          int out_u8, void *const *mirrors, int nmirror,
                                          gk_stream_t stream);

/* ---- self test of the bounded-wait path ----------------------------------------------- */

/* Launch a kernel that waits on an mbarrier no one arrives on, with a `timeout_ns` bound,
 * and report the outcome: GK_ETIMEOUT (the expected result) once the wait gave up and the
 * kernel returned, leaving the context usable. */
int gk_selftest_wait_timeout(uint64_t timeout_ns, gk_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif
