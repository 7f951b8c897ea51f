/* zkml_gpu.h -- C ABI of the MI355X (gfx950) Groth16 prover core.
 *
 * Drop-in boundary for the data-parallel hot path of gdtsitlauri/cuda-zkml's
 * prover.  Every entry point names the reference interface it replaces
 * (paths relative to the reference root).  Plain pointers and sizes only.
 *
 * Data layouts are the reference's in-memory layouts:
 *   zk_fr, zk_fq      32 bytes: 4 x uint64 little endian, Montgomery form with
 *                     R = 2^256 (src/field/fp.cuh:28-31, 322-324).
 *   zk_g1_affine      64 bytes: x, y (zk_fq).  x = y = 0 encodes the point at
 *                     infinity (no finite curve point has x = y = 0).
 *   zk_g2_affine      128 bytes: x.c0, x.c1, y.c0, y.c1.
 *   reference structs G1Affine (72 bytes: x, y, bool infinity at byte 64) and
 *                     G2Affine (136 bytes, bool at byte 128) are accepted by the
 *                     *_host entry points (src/curve/g1.cuh:29-33, g2.cuh:25-29).
 *   zk_sparse_entry   40 bytes {int32 row; int32 col; zk_fr value}
 *                     (src/prover/circuit.cuh:32-36).
 *
 * Errors: every function returns ZK_OK (0) or a positive zk_status; the
 * reference instead exits the process on a device error (src/common.cuh:11-19).
 * zk_last_error() gives a message for the last failure on a context.
 *
 * Streams: `stream` arguments are hipStream_t values; NULL selects the
 * context's own stream.  Calls that return a host value synchronize.
 * A context is not re-entrant: one host thread per context at a time.
 * The NTT calls (zk_ntt, zk_coset_ntt, zk_quotient_h) of one context share
 * its pass-to-pass scratch buffer whatever stream they are given: two such
 * calls on different streams must not overlap (order the second stream after
 * the first with an event, or synchronize between them).  Twiddle and coset
 * tables are complete before a call returns, so they are safe on any stream.
 */
#ifndef ZKML_GPU_H
#define ZKML_GPU_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct zk_context zk_context;
typedef struct zk_r1cs zk_r1cs;
typedef struct zk_pk zk_pk;

enum zk_status {
  ZK_OK = 0,
  ZK_ERR_INVALID = 1,   /* bad argument */
  ZK_ERR_SIZE = 2,      /* size outside the supported range */
  ZK_ERR_OOM = 3,       /* device or host allocation failed */
  ZK_ERR_HIP = 4,       /* HIP runtime error */
  ZK_ERR_IO = 5,        /* file missing, truncated or malformed */
  ZK_ERR_WITNESS = 6,   /* witness does not satisfy the R1CS */
  ZK_ERR_MISMATCH = 7   /* witness / key / circuit sizes disagree */
};

typedef struct zk_sparse_entry {
  int32_t row;
  int32_t col;
  uint64_t value[4];
} zk_sparse_entry;

/* ---- context and device memory ---------------------------------------- */
int zk_create(int device, zk_context** out);
void zk_destroy(zk_context* ctx);
const char* zk_status_string(int status);
const char* zk_last_error(const zk_context* ctx);
int zk_synchronize(zk_context* ctx);
void* zk_get_stream(zk_context* ctx);
int zk_dev_alloc(zk_context* ctx, size_t bytes, void** d_ptr);
int zk_dev_free(zk_context* ctx, void* d_ptr);
int zk_memcpy_h2d(zk_context* ctx, void* d_dst, const void* h_src, size_t bytes);
int zk_memcpy_d2h(zk_context* ctx, void* h_dst, const void* d_src, size_t bytes);
int zk_memcpy_d2d(zk_context* ctx, void* d_dst, const void* d_src, size_t bytes);
/* Test hook, no counterpart in the reference: the nth device allocation
 * from now that the library makes for its own workspaces and NTT tables
 * (1 = the next one) fails with ZK_ERR_OOM, once; 0 disarms.  For tests of
 * the error paths only; affects every context of the process. */
int zk_debug_fail_device_alloc(int nth);
/* Test hook, no counterpart in the reference: the next `count` MSM jobs that
 * zk_prove would hand to the context's host worker threads are refused as if
 * no worker could be started, so the jobs run on the calling thread instead;
 * 0 disarms.  For tests of that fallback only; affects every context of the
 * process. */
int zk_debug_fail_thread_start(int count);

/* Per-kernel timing with HIP events recorded on the stream each kernel is
 * launched on (off by default).  Names: see zk_kernel_stats_names(). */
int zk_set_profiling(zk_context* ctx, int enable);
/* Time only the kernels of this name (NULL or "": all).  Each timed launch
 * adds two event records to its stream, so a throughput run times just the
 * kernel it reports. */
int zk_set_profiling_only(zk_context* ctx, const char* kernel);
int zk_kernel_stats(zk_context* ctx, const char* kernel, uint64_t* launches, double* total_ms);
int zk_reset_kernel_stats(zk_context* ctx);
const char* zk_kernel_stats_names(zk_context* ctx);

/* ---- NTT over Fr -------------------------------------------------------
 * Replaces bn254::ntt_gpu(Fr* d_out, const Fr* d_in, int log_n, bool inverse)
 * (src/ntt/ntt.cuh:49, src/ntt/ntt.cu:354-465) and ntt_gpu_inplace (:467).
 * out[j] = sum_i in[i] * w^(i*j), w = 5^((r-1)/2^28)^(2^(28-log_n)); the
 * inverse uses w^-1 and scales by n^-1.  Natural order in and out; d_out may
 * equal d_in.  1 <= log_n <= 24 (NTT_MAX_LOG, src/common.cuh:78); the reference
 * returns silently above that, this returns ZK_ERR_SIZE.  `batch` transforms
 * of n elements each are laid out back to back. */
int zk_ntt(zk_context* ctx, void* d_out, const void* d_in, int log_n, int inverse, int batch, void* stream);

/* No counterpart in the reference: zk_ntt for callers that cannot allocate
 * device memory (code under HIP graph capture, tight serving loops, harnesses
 * that forbid hipMalloc).  Same transform, layouts and stream argument as
 * zk_ntt, with 1 <= log_n <= 16 and batch * 2^log_n <= 2^18 elements; larger
 * sizes return ZK_ERR_SIZE.  Allocates nothing: its twiddle tables and
 * pass-to-pass buffer live in a fixed device array of the library (17 MB per
 * GPU, held from library load to process end) that every call on a GPU
 * shares.  Each log_n has its own table slot, filled by the first call of
 * that size; a call on a stream under graph capture records that fill into
 * the graph, so replays do not depend on the calls made between capture and
 * replay.  Calls that overlap on one GPU race on the pass-to-pass buffer:
 * order them on one stream or synchronize between them. */
int zk_ntt_noalloc(zk_context* ctx, void* d_out, const void* d_in, int log_n, int inverse, int batch, void* stream);

/* Coset NTT as used by Groth16Prover::compute_h (src/prover/groth16.cu:350-383):
 * forward: out = NTT(in[i] * g^i); inverse: out[i] = iNTT(in)[i] * g^-i.
 * g is a small plain integer (the prover uses 5; the coset tests also use 7). */
int zk_coset_ntt(zk_context* ctx, void* d_out, const void* d_in, int log_n, uint64_t g, int inverse, int batch,
                 void* stream);

/* ---- MSM ----------------------------------------------------------------
 * Replaces bn254::msm_g1 / msm_g2 (src/msm/msm.cuh:67-68, msm.cu:320-598):
 * result = sum_i scalars[i] * points[i].  Device-resident inputs (points in
 * zk_g1_affine / zk_g2_affine layout, scalars zk_fr), result written to host
 * memory as an affine point in the same layout (the reference returns a
 * Jacobian point whose callers convert it to affine).  n == 0 gives infinity;
 * n above 2^26 returns ZK_ERR_SIZE. */
int zk_msm_g1(zk_context* ctx, const void* d_points, const void* d_scalars, size_t n, void* h_result,
              void* stream);
int zk_msm_g2(zk_context* ctx, const void* d_points, const void* d_scalars, size_t n, void* h_result,
              void* stream);

/* MSMs over one base set, its conversion done once.  No counterpart in the
 * reference (bn254::msm_g1 / msm_g2 read affine points on every call); for
 * callers that run many MSMs over the same points.  zk_msm_prepare_points
 * writes the n points (zk_g1_affine, or zk_g2_affine when g2 != 0) as the
 * MSM's point records into d_recs, zk_msm_record_bytes(g2) bytes per point;
 * d_recs must not overlap d_points (ZK_ERR_INVALID).  zk_msm_g1_prepared /
 * zk_msm_g2_prepared then give the same result as zk_msm_g1 / zk_msm_g2 over
 * those points, without the per-call conversion; the records stay valid
 * while d_recs is unchanged. */
size_t zk_msm_record_bytes(int g2);
int zk_msm_prepare_points(zk_context* ctx, const void* d_points, size_t n, int g2, void* d_recs, void* stream);
int zk_msm_g1_prepared(zk_context* ctx, const void* d_recs, const void* d_scalars, size_t n, void* h_result,
                       void* stream);
int zk_msm_g2_prepared(zk_context* ctx, const void* d_recs, const void* d_scalars, size_t n, void* h_result,
                       void* stream);

/* Window configuration the MSM uses for n points (replaces
 * bn254::MSMConfig::for_size, src/msm/msm.cuh:40-64): window bits c (the
 * widest window) and the number of signed-digit windows.  CPU only. */
int zk_msm_config(size_t n, int g2, int* window_bits, int* windows);

/* KZG commitment over G1 (replaces KZGCommitment::commit / ::open,
 * src/prover/groth16.cuh:197-207, groth16.cu:393-438).  d_srs_g1: device
 * zk_g1_affine [tau^i]_1, i < degree; d_coeffs: device Fr (Montgomery), f_i
 * ascending, `degree` coefficients.  zk_kzg_commit writes sum f_i [tau^i]_1
 * (affine, as zk_msm_g1).  zk_kzg_open writes the opening proof
 * sum q_i [tau^i]_1 with q = (f - f(z)) / (x - z) (synthetic division on the
 * GPU; degree <= 1 gives infinity, as the reference) and, when f_z is not
 * NULL, f(z) (Montgomery Fr).  z: Montgomery Fr.  The verifier equation is
 * e(C - f(z) G1, G2) = e(proof, [tau]_2 - z G2). */
int zk_kzg_commit(zk_context* ctx, const void* d_srs_g1, const void* d_coeffs, size_t degree, void* h_commitment,
                  void* stream);
int zk_kzg_open(zk_context* ctx, const void* d_srs_g1, const void* d_coeffs, size_t degree, const uint64_t z[4],
                void* h_proof, uint64_t f_z[4], void* stream);

/* Host-pointer drop-ins with the reference's exact signature semantics:
 * h_points are reference G1Affine / G2Affine structs (72 / 136 bytes),
 * h_scalars are Fr, h_result receives a reference G1Jacobian / G2Jacobian
 * (96 / 192 bytes: x, y, z Montgomery; z = 1, or z = 0 for infinity). */
int zk_msm_g1_host(zk_context* ctx, const void* h_points, const void* h_scalars, int n, void* h_result_jacobian);
int zk_msm_g2_host(zk_context* ctx, const void* h_points, const void* h_scalars, int n, void* h_result_jacobian);

/* ---- fixed-base generation (setup and synthetic inputs) -----------------
 * d_out[i] = k[i] * G for the group generator G (G1 (1,2), G2 EIP-197:
 * src/curve/g1.cuh:40, g2.cuh:47-65); k in zk_fr layout (Montgomery). */
int zk_g1_generator_mul(zk_context* ctx, const void* d_scalars, size_t n, void* d_out, void* stream);
int zk_g2_generator_mul(zk_context* ctx, const void* d_scalars, size_t n, void* d_out, void* stream);

/* ---- R1CS and the quotient polynomial -----------------------------------
 * zk_r1cs_create uploads the reference's COO matrices (R1CS::A/B/C,
 * src/prover/circuit.cuh:39-50) once and keeps them on the device in CSR form.
 * zk_quotient_h replaces Groth16Prover::compute_h (groth16.cu:263-390):
 * h = (A.w * B.w - C.w) / (x^n - 1) via 3 iNTT, 3 coset NTT (shift 5, or 7
 * when 5^n = 1), a pointwise step and a coset iNTT, all resident on the
 * device.  d_h receives n = 2^ceil(log2(max(num_constraints, 4))) elements. */
int zk_r1cs_create(zk_context* ctx, int num_constraints, int num_variables, int num_public,
                   const zk_sparse_entry* A, size_t nA, const zk_sparse_entry* B, size_t nB,
                   const zk_sparse_entry* C, size_t nC, zk_r1cs** out);
void zk_r1cs_destroy(zk_r1cs* r1cs);
int zk_r1cs_domain(const zk_r1cs* r1cs, int* log_n);
int zk_quotient_h(zk_context* ctx, const zk_r1cs* r1cs, const void* d_witness, size_t m, void* d_h, void* stream);

/* ---- proving key, setup and prove ---------------------------------------
 * zk_pk_load replaces ProvingKey::load_streaming (groth16.cu:1190-1314): reads
 * a ZKMLPK3 file with the same checks and keeps all queries on the device.
 * For 2^14 .. 2^23 variables it also builds window tables of the queries (W
 * shifted copies of each, W = 13 to 20) that zk_prove's MSMs run on: device
 * memory grows by that factor (about 20 GB at 2^22) and the load takes longer
 * (1.5 s instead of 0.8 s at 2^22); proofs are the same bytes.
 * zk_setup replaces Groth16Prover::setup (groth16.cu:446-642) for a given
 * toxic-waste seed (the reference's deterministic seed is 0xDEADBEEF42) and
 * writes a ZKMLPK3 proving key and a verification key (verifier.cu:103-148).
 * zk_prove replaces Groth16Prover::prove (groth16.cu:655-920): r and s are the
 * first two nonzero Fr::from_uint(std::mt19937_64(blind_seed)()) draws (the
 * reference's deterministic seed is 0xCAFEBABE); the 256-byte proof is
 * A.x, A.y, B.x.c0, B.x.c1, B.y.c0, B.y.c1, C.x, C.y in standard form
 * (Groth16Proof::serialize, groth16.cu:1058-1074).  check_witness mirrors the
 * ZKML_SKIP_WITNESS_CHECK switch (groth16.cu:687-695).  The five MSMs run
 * concurrently on streams of the context (one host thread each).
 * timings_ms (optional, 8 doubles): total (host clock, from the witness
 * upload to the serialized proof), witness upload + quotient, then each
 * MSM's own duration (GPU events; they overlap): A, B(G2), L, H, B1, and the
 * host assembly after the last MSM. */
int zk_pk_load(zk_context* ctx, const char* path, zk_pk** out);
void zk_pk_destroy(zk_pk* pk);
int zk_pk_info(const zk_pk* pk, int* num_constraints, int* num_variables, int* num_public);
int zk_setup(zk_context* ctx, const zk_r1cs* r1cs, uint64_t toxic_seed, const char* pk_path, const char* vk_path);
int zk_prove(zk_context* ctx, const zk_pk* pk, const zk_r1cs* r1cs, const void* h_witness, size_t m,
             int num_public, uint64_t blind_seed, int check_witness, uint8_t proof_out[256], double* timings_ms);

/* ---- R1CS / witness files and the synthetic R1CS (host code) ------------
 * iden3 binary formats (circom / snarkjs): .r1cs version 1, .wtns version 2.
 * zk_iden3_r1cs_write replaces export_r1cs_iden3 and zk_wtns_write replaces
 * export_wtns_iden3 (src/prover/r1cs_export.cuh:41-92): same bytes for the
 * same R1CS (public wires as nPubOut, nPubIn = 0, identity label map).
 * Matrix values and witnesses are the reference's Montgomery Fr words; files
 * hold standard form.  Reading: zk_iden3_r1cs_info gives the sizes (public =
 * nPubOut + nPubIn), then zk_iden3_r1cs_read fills caller arrays of those
 * sizes; zk_wtns_info / zk_wtns_read likewise.
 * zk_synthetic_r1cs builds a large random R1CS (the shape of the 2^22-row
 * benchmark statement) from a seed: w[0] = 1, num_public + num_inputs uniform variables, then per row A and
 * B with 1-3 terms over earlier variables (uniform coefficients) and C = one
 * fresh variable set to (A.w)(B.w), so the witness satisfies every row.
 * Capacities: A, B 3 * num_constraints entries, C num_constraints, w_mont
 * 1 + num_public + num_inputs + num_constraints elements. */
int zk_iden3_r1cs_info(const char* path, int* num_constraints, int* num_variables, int* num_public,
                       int* num_private, size_t* nA, size_t* nB, size_t* nC);
int zk_iden3_r1cs_read(const char* path, zk_sparse_entry* A, zk_sparse_entry* B, zk_sparse_entry* C);
int zk_iden3_r1cs_write(const char* path, int num_constraints, int num_variables, int num_public, int num_private,
                        const zk_sparse_entry* A, size_t nA, const zk_sparse_entry* B, size_t nB,
                        const zk_sparse_entry* C, size_t nC);
int zk_wtns_info(const char* path, size_t* m);
int zk_wtns_read(const char* path, void* w_mont, size_t m);
int zk_wtns_write(const char* path, const void* w_mont, size_t m);
int zk_synthetic_r1cs(int num_constraints, int num_public, int num_inputs, uint64_t seed, zk_sparse_entry* A,
                      size_t* nA, zk_sparse_entry* B, size_t* nB, zk_sparse_entry* C, size_t* nC, void* w_mont);

/* ---- 8-bit integer layers -------------------------------------------------
 * No counterpart in the reference, whose GPU layers work on field elements
 * (src/nn/layers.cu:37-190).  The linear layer of a quantized model (LINEAR of
 * the statement producer below: weights n_out x n_in, row major) over whole
 * batches, in the integers a statement proves, and with the scales that tie
 * them to the real-valued model.
 *
 * zk_i8_matmul: acc[t][n] = sum_k x[t][k] w[n][k] (int8, exact in int32;
 * n_in <= 131071, n_out <= 2^26), then
 *   y_type ZK_I32: y = acc (no scales, no bias);
 *   else           y = (float(acc) * x_scale[t]) * w_scale[n] + bias[n],
 * each operation rounded to 32-bit floats in this order (float(acc) *
 * x_scale[t] without leaving their range above), then once to y_type; relu !=
 * 0 replaces what is below zero by zero (a NaN stays).  d_x_scale (rows), d_w_scale and d_bias (n_out)
 * may be NULL (1, 1 and 0).  ld_* are row strides in elements, at least the
 * row's length; rows of x and w may start at any byte (they may be read in
 * whole aligned 4-byte words, whose other bytes do not matter).
 * zk_i8_quantize: scale[t] = max_k |x[t][k]| / 127, q[t][k] = the integer
 * nearest to (127 x[t][k]) / max_k |x[t][k]| (ties to even), the product and
 * the quotient each rounded to 32-bit floats.  For f16 and bf16 rows this is
 * the integer nearest to the exact quotient; of an f32 row a quotient within
 * 2^-16 of a half may go to either side.  A row of zeros has scale 0 and
 * zeros; a row that holds an infinity or a NaN has scale NaN
 * and zeros, so that what is made of it is NaN.
 * zk_i8_linear: zk_i8_quantize of x's rows, then zk_i8_matmul with their
 * scales.  d_work: zk_i8_linear_work(rows, n_in) bytes (0: sizes out of
 * range), 16-byte aligned, free again when the call's work on the stream is
 * done.
 * zk_i8_matmul_experts: rows offsets[e] .. offsets[e+1] of y (see
 * zk_experts_sort) use expert e's weights, d_w + e * n_out * ld_w, w_scale and
 * bias + e * n_out; row p takes row order[p] / slots of x (tokens rows) and
 * its scale, or row p itself when d_order is NULL.  Rows that belong to no
 * expert, or whose order names no token, become zeros (no tokens: d_x may be
 * NULL).  offsets[0] is 0 and the offsets do not fall.  At most 2^22 rows; ZK_ERR_SIZE also where rows and
 * n_out make more than 2^22 tiles.
 * None of these allocates, waits or uses memory of the context, so calls on
 * different streams do not touch each other.  y may not overlap an input.
 * stream may be hipStreamLegacy (the default stream of a program that does
 * not name one). */
enum zk_type { ZK_F32 = 0, ZK_F16 = 1, ZK_BF16 = 2, ZK_I32 = 3 };
enum { ZK_MAX_EXPERTS = 1024, ZK_MAX_EXPERT_ROWS = 1 << 22 };

int zk_i8_matmul(zk_context* ctx, const int8_t* d_x, size_t ld_x, const float* d_x_scale, const int8_t* d_w,
                 size_t ld_w, const float* d_w_scale, const float* d_bias, size_t rows, size_t n_out, size_t n_in,
                 int relu, void* d_y, int y_type, size_t ld_y, void* stream);
int zk_i8_quantize(zk_context* ctx, const void* d_x, int x_type, size_t ld_x, size_t rows, size_t cols, int8_t* d_q,
                   size_t ld_q, float* d_scale, void* stream);
size_t zk_i8_linear_work(size_t rows, size_t n_in);
int zk_i8_linear(zk_context* ctx, const void* d_x, int x_type, size_t ld_x, const int8_t* d_w, size_t ld_w,
                 const float* d_w_scale, const float* d_bias, size_t rows, size_t n_out, size_t n_in, int relu,
                 void* d_y, int y_type, size_t ld_y, void* d_work, size_t work_bytes, void* stream);
int zk_i8_matmul_experts(zk_context* ctx, const int8_t* d_x, size_t ld_x, const float* d_x_scale, size_t tokens,
                         const int8_t* d_w, size_t ld_w, const float* d_w_scale, const float* d_bias,
                         const int32_t* d_offsets, int experts, const int32_t* d_order, int slots, size_t rows,
                         size_t n_out, size_t n_in, int relu, void* d_y, int y_type, size_t ld_y, void* stream);

/* Test hook: the name of the kernel that zk_i8_matmul takes for these sizes and
 * strides, x and w at addresses with the low bits of `address`; with experts > 0
 * that of zk_i8_matmul_experts.  NULL: sizes out of range.  Host only. */
const char* zk_debug_i8_kernel(size_t rows, size_t n_out, size_t n_in, size_t ld_x, size_t ld_w, size_t address,
                               int experts);

/* ---- layers with 4-bit weights ----------------------------------------------
 * No counterpart in the reference.  The 8-bit rows above (int8 with a scale
 * each) times weights of 4 bits, -8 to 7, with a scale for each group of `group`
 * (32, 64 or a multiple of 128) neighbouring weights of a channel, the last of
 * which may be shorter.
 * Layout: a channel's weights are zk_i4_row_bytes(n_in) = 64 ceil(n_in / 128)
 * bytes (0: n_in above 2^24); in each 64 of them, which are 128 weights, byte b
 * holds weight b in its low and weight 64 + b in its high four bits, two's
 * complement.  What lies behind a row's last weight does not matter.  Rows start
 * at multiples of 16 bytes (d_w and ld_w, in bytes).  The scale of group g of
 * channel n is d_w_scale[g * n_out + n], of type scale_type (ZK_F32, ZK_F16 or
 * ZK_BF16).
 *
 * zk_i4_quantize: a matrix of rows x cols to this layout.  scale = max |w| of the
 * group / 7, rounded to scale_type; q = the integer nearest to w / scale (ties to
 * even), between -8 and 7.  A group of zeros, or whose scale rounds to zero, has
 * scale 0 and zeros, one whose scale rounds to infinity that scale and zeros, one that
 * holds an infinity or a NaN scale NaN and zeros.  Padding becomes zero.
 * zk_i4_matmul: y[t][n] = x_scale[t] * sum_g w_scale[g][n] acc[t][n][g] + bias[n]
 * with acc[t][n][g] = sum_k x[t][k] q[n][k] over group g.  Sums within 128
 * weights are exact; the groups' terms, of a longer one those of each 128 weights, are
 * added in 32-bit floats, in an order that depends on the sizes, the strides and
 * x's address, never on the order of execution; the token's scale and the bias follow in one
 * fused operation, then one rounding to y_type (ZK_F32, ZK_F16, ZK_BF16).  relu,
 * strides, NULL scales and biases and rows of x at any byte as in zk_i8_matmul
 * (d_w_scale may not be NULL); at most 2^26 channels.  Scales of weights below
 * 2^-122 count to a multiple of 2^-145.
 * zk_i4_linear: zk_i8_quantize of x's rows, then zk_i4_matmul, few rows in an order of
 * sums of their own.  d_work: zk_i4_linear_work(rows, n_in) bytes (0: sizes out of
 * range), 16-byte aligned, free again when the call's work on the stream is done.
 * zk_i4_matmul_experts: as zk_i8_matmul_experts; expert e's weights begin at
 * d_w + e * n_out * ld_w bytes, its scales at d_w_scale[e * groups * n_out], its
 * biases at d_bias[e * n_out].
 * None of these allocates, waits or uses memory of the context.  Outputs may not
 * overlap an input. */
size_t zk_i4_row_bytes(size_t n_in);
int zk_i4_quantize(zk_context* ctx, const void* d_w, int w_type, size_t ld_w, size_t rows, size_t cols, int group,
                   void* d_q, size_t ld_q, void* d_scale, int scale_type, void* stream);
int zk_i4_matmul(zk_context* ctx, const int8_t* d_x, size_t ld_x, const float* d_x_scale, const void* d_w, size_t ld_w,
                 const void* d_w_scale, int scale_type, int group, const float* d_bias, size_t rows, size_t n_out,
                 size_t n_in, int relu, void* d_y, int y_type, size_t ld_y, void* stream);
size_t zk_i4_linear_work(size_t rows, size_t n_in);
int zk_i4_linear(zk_context* ctx, const void* d_x, int x_type, size_t ld_x, const void* d_w, size_t ld_w,
                 const void* d_w_scale, int scale_type, int group, const float* d_bias, size_t rows, size_t n_out,
                 size_t n_in, int relu, void* d_y, int y_type, size_t ld_y, void* d_work, size_t work_bytes,
                 void* stream);
int zk_i4_matmul_experts(zk_context* ctx, const int8_t* d_x, size_t ld_x, const float* d_x_scale, size_t tokens,
                         const void* d_w, size_t ld_w, const void* d_w_scale, int scale_type, int group,
                         const float* d_bias, const int32_t* d_offsets, int experts, const int32_t* d_order, int slots,
                         size_t rows, size_t n_out, size_t n_in, int relu, void* d_y, int y_type, size_t ld_y,
                         void* stream);

/* Test hook: the name of the kernel that zk_i4_matmul takes for these sizes, x at an
 * address with the low bits of `address`; with experts > 0 that of
 * zk_i4_matmul_experts.  NULL: sizes out of range.  Host only. */
const char* zk_debug_i4_kernel(size_t rows, size_t n_out, size_t n_in, size_t ld_x, size_t address, int group,
                               int experts);

/* ---- routed experts ---------------------------------------------------------
 * No counterpart in the reference, whose routing ends with each sample's class
 * and flag (src/prover/statement_v2.cuh:243-266).  Samples ("tokens") sorted by
 * the expert that a route names and put back with the routes' weights.  A pair
 * i = token * slots + j is a token's j-th route.
 *
 * zk_experts_sort: stable counting sort of the pairs by expert (1 to 1024
 * experts, at most 2^22 pairs).  offsets[e] (experts + 1 words) = pairs with an
 * expert below e; order[p] = the pair at position p; place[i] = the pair's
 * position.  A pair whose expert is outside [0, experts) is dropped: place[i] =
 * -1, and order[p] = -1 from offsets[experts] on.  d_work:
 * zk_experts_sort_work(pairs, experts) bytes (0: none needed, may be NULL).
 * zk_experts_gather: out[p] = x[order[p] / slots], zeros where order[p] is -1.
 * Its gradient is zk_experts_combine of the rows' gradients without weights.
 * zk_experts_combine: out[t] = sum_j weight[t][j] * y[place[t][j]] over the
 * pairs that have a place, summed in 32-bit floats in the order of j, rounded
 * once; d_weight NULL: 1.  Tokens with no place become zeros.
 * zk_experts_combine_grad: for the gradient g of that sum,
 *   grad_y[place[t][j]] = weight[t][j] * g[t], zeros where order is -1;
 *   grad_weight[t][j] = sum_c g[t][c] * y[place[t][j]][c], 0 for dropped pairs.
 * d_grad_weight may be NULL (then d_y may be, too).  place and order are those
 * of one zk_experts_sort, rows <= tokens * slots.
 * type: that of all rows (ZK_F32, ZK_F16, ZK_BF16); ld_* row strides in
 * elements.  Results do not depend on the order of execution.  Indexes outside
 * their range are taken as -1. */
size_t zk_experts_sort_work(size_t pairs, int experts);
int zk_experts_sort(zk_context* ctx, const int32_t* d_expert, size_t pairs, int experts, int32_t* d_offsets,
                    int32_t* d_order, int32_t* d_place, void* d_work, size_t work_bytes, void* stream);
int zk_experts_gather(zk_context* ctx, const void* d_x, int type, size_t ld_x, size_t cols, const int32_t* d_order,
                      size_t rows, size_t tokens, int slots, void* d_out, size_t ld_out, void* stream);
int zk_experts_combine(zk_context* ctx, const void* d_y, int type, size_t ld_y, size_t cols, const int32_t* d_place,
                       const float* d_weight, size_t rows, size_t tokens, int slots, void* d_out, size_t ld_out,
                       void* stream);
int zk_experts_combine_grad(zk_context* ctx, const void* d_grad, size_t ld_grad, const void* d_y, size_t ld_y,
                            int type, size_t cols, const int32_t* d_order, const int32_t* d_place,
                            const float* d_weight, size_t rows, size_t tokens, int slots, void* d_grad_y,
                            size_t ld_grad_y, float* d_grad_weight, void* stream);

/* ---- the experts' router ------------------------------------------------------
 * No counterpart in the reference.  Which experts a token's gate scores name, with
 * which weights, how evenly, and the gradients.  scores: tokens x experts, ZK_F32,
 * ZK_F16, ZK_BF16, or ZK_I32 (a gate's exact sums from zk_i8_matmul), rows at
 * stride ld.  p[t] = softmax over the experts of scale * scores[t] (scale positive
 * and finite), in 32-bit floats.  A score of minus infinity (ZK_I32: INT32_MIN) is
 * a masked expert: never chosen, probability 0.
 *
 * zk_experts_route: a token's `slots` experts (1 to 32) by falling score, of equal
 * scores the lower expert first, as zk_experts_sort takes them, and their weights:
 * p of the chosen, or with renormalize != 0 these divided by their sum.  A token
 * with fewer unmasked experts has expert -1 and weight 0 in the slots that are
 * left (all of them in a masked row: padding); one with a NaN or an infinity above
 * has experts -1 and weights NaN.
 * With d_count, d_prob and d_loss (all or none) also, over the n tokens that have
 * a score other than masked,
 *   count[e] = routes that name e (experts + 1 words; count[experts] = n),
 *   prob[e] = sum_t p[t][e] / n,
 *   loss = experts * sum_e count[e] / (n * slots) * prob[e]       (1 if all are even),
 * prob and loss 0 without such a token, NaN with a NaN or an infinity above.
 * d_work: zk_experts_route_work(tokens, experts) bytes (0: none needed, may be
 * NULL), 8-byte aligned, used only with these outputs.
 * zk_experts_balance: the same three for given routes (tokens x slots); a route
 * outside [0, experts) names none, nor does one of a masked row, whatever it holds.
 * zk_experts_route_grad: the gradient with regard to the scores of what depends
 * on the weights by grad_weight (tokens x slots; NULL: nothing does) and on the
 * loss by grad_loss[0] (d_count NULL: nothing does; else the counts of
 * zk_experts_route or zk_experts_balance, constants to the gradient).  expert,
 * scale and renormalize as in the forward call; the same expert twice counts
 * twice.  Masked scores get 0, a row with a NaN or an infinity above NaN.
 * At most 1024 experts and 2^22 pairs.  No result depends on the order of
 * execution.  None of these allocates, waits or uses memory of the context; calls
 * that overlap need a workspace each.  Outputs may not overlap an input. */
enum { ZK_MAX_SLOTS = 32 };
size_t zk_experts_route_work(size_t tokens, int experts);
int zk_experts_route(zk_context* ctx, const void* d_scores, int type, size_t ld, size_t tokens, int experts, int slots,
                     float scale, int renormalize, int32_t* d_expert, float* d_weight, int32_t* d_count,
                     float* d_prob, float* d_loss, void* d_work, size_t work_bytes, void* stream);
int zk_experts_balance(zk_context* ctx, const void* d_scores, int type, size_t ld, size_t tokens, int experts,
                       int slots, float scale, const int32_t* d_expert, int32_t* d_count, float* d_prob,
                       float* d_loss, void* d_work, size_t work_bytes, void* stream);
int zk_experts_route_grad(zk_context* ctx, const void* d_scores, int type, size_t ld, size_t tokens, int experts,
                          int slots, float scale, int renormalize, const int32_t* d_expert,
                          const float* d_grad_weight, const int32_t* d_count, const float* d_grad_loss,
                          void* d_grad_scores, size_t ld_grad, void* stream);

/* ---- pairing and verification (host code, no device needed) -------------
 * zk_pairing replaces bn254::pairing (src/curve/pairing.cuh:198-282): the
 * reduced optimal ate pairing e(P, Q).  P: 64 bytes x, y; Q: 128 bytes x.c0,
 * x.c1, y.c0, y.c1; both standard form little endian, all-zero = infinity.
 * out: the Fp12 value as 12 x 32 bytes standard form in the reference's order
 * (c0.c0.c0, c0.c0.c1, c0.c1.c0, ..., c1.c2.c1).
 * zk_verify replaces Groth16Verifier::verify (groth16.cu:967-1022): vk_bytes
 * is a verification-key file image (verifier.cu:103-148), proof256 a proof
 * file image, publics npub x 32-byte standard-form scalars.  *valid = 1 when
 * e(-A, B) e(alpha, beta) e(vk_x, gamma) e(C, delta) == 1; a public-input
 * count other than the key's rejects (valid = 0, status ZK_OK), as in the
 * reference.  A and C must be on the curve and B on the twist and in the
 * order-r subgroup (the reference does not check; it would reject such
 * points only by chance).
 * zk_verify_files replaces zkml-verify's loading (src/cli/verify.cu): the
 * public-input file is .bin (i32 count + 32-byte scalars) or .json (decimal
 * list). */
int zk_pairing(const void* p_std, const void* q_std, void* out_std);
int zk_verify(const void* vk_bytes, size_t vk_len, const void* proof256, const void* publics_std, int npub,
              int* valid);
int zk_verify_files(const char* vk_path, const char* proof_path, const char* publics_path, int* valid);

/* ---- Poseidon (host code) -------------------------------------------------
 * BN254 Fr, t = 3, x^5, R_F = 8, R_P = 57: the circomlib instance of the
 * reference (src/prover/gadgets.cuh:323-427, poseidon_constants.cuh).  Values
 * cross as 4 x u64 standard form (inputs >= r are reduced mod r).
 * zk_poseidon_permute replaces poseidon_permute_native (state: 3 elements, in
 * place); zk_poseidon_hash2 replaces poseidon_hash2_native (= circomlib
 * Poseidon([a, b])); zk_poseidon_commit replaces poseidon_commit_native (rate-2
 * sponge, capacity (n << 64) | domain, output state[1]; domains "MODEL" =
 * 0x4d4f44454c and "INPUT" = 0x494e505554).  zk_poseidon_constants writes the
 * 195 round constants and the 3 x 3 MDS matrix (row major), either may be
 * NULL. */
int zk_poseidon_permute(uint64_t state[12]);
int zk_poseidon_hash2(const uint64_t a[4], const uint64_t b[4], uint64_t out[4]);
int zk_poseidon_commit(const uint64_t* values, size_t n, uint64_t domain, uint64_t out[4]);
int zk_poseidon_constants(uint64_t* round_constants, uint64_t* mds);

/* ---- statement producer (host code) ---------------------------------------
 * zk_statement_v2_build replaces build_statement_v2
 * (src/prover/statement_v2.cuh:82-253) with the TracedBuilder gadgets
 * (gadgets.cuh:128-457): one R1CS + witness for `batch` samples of a quantized
 * model, term for term the reference's (same variables, rows and term order).
 * Layers mirror NNModel::Layer (src/nn/inference.cuh:95-147); type values are
 * the reference's LayerType (src/nn/layers.cuh:36-43).  Model values and
 * inputs are signed integers (v -> v mod r; |v| >= 2^62 -> 0, as the
 * reference's Fp -> int64 conversion).  LINEAR: weights out_size x in_size row
 * major, bias out_size.  CONV2D: CHW, weights [out_c][in_c][kh][kw], bias
 * out_c; in_size / out_size are derived from the conv fields.  RELU_EXACT:
 * relu_bits in [1, 252], relu_shift in [0, 62].  RELU_APPROX: y = scale (c0 +
 * c1 x + c2 x^2 + c3 x^3).  SOFTMAX_APPROX only as the last layer (outside the
 * statement); SELF_ATTENTION is rejected.  inputs: batch x n_in.
 * Options mirror StatementV2Options (statement_v2.cuh:31-42); an all-zero
 * struct (or NULL) is the reference's default, compare_bits 0 meaning 48.
 * Field values are 4 x u64 standard form; input_blinding holds batch of them.
 * Errors: ZK_ERR_INVALID with the reference's message in err (err_cap bytes).
 * Results: zk_statement_info (sizes), zk_statement_r1cs (COO, Montgomery
 * values, caller arrays of nA / nB / nC entries), zk_statement_witness
 * (num_variables Montgomery Fr), zk_statement_layout (public-input layout,
 * ZK_LAYOUT_* indices; -1 for absent groups), zk_statement_scores (batch x
 * n_out final scores), zk_statement_check (R1CS::verify_witness,
 * src/prover/circuit.cuh:92-124: ZK_OK or ZK_ERR_WITNESS),
 * zk_statement_write (iden3 .r1cs / .wtns; either path may be NULL) and
 * zk_statement_meta_json (statement_v2_meta_json, statement_v2.cuh:255-287;
 * *len = length without the terminator, ZK_ERR_SIZE if cap is too small). */
enum zk_layer_type {
  ZK_LAYER_LINEAR = 0,
  ZK_LAYER_RELU_APPROX = 1,
  ZK_LAYER_SOFTMAX_APPROX = 2,
  ZK_LAYER_SELF_ATTENTION = 3,
  ZK_LAYER_RELU_EXACT = 4,
  ZK_LAYER_CONV2D = 5
};

typedef struct zk_layer {
  int32_t type;
  int32_t in_size, out_size;
  int32_t conv_in_c, conv_in_h, conv_in_w, conv_out_c, conv_kh, conv_kw, conv_stride, conv_pad;
  int32_t relu_bits, relu_shift;
  int64_t relu_c[4];
  int64_t relu_scale;
  const int64_t* weights;
  const int64_t* bias;
} zk_layer;

typedef struct zk_statement_options {
  uint64_t model_tag[4];
  int32_t has_context;
  uint64_t context[4];
  int32_t private_input;
  const uint64_t* input_blinding;
  int32_t private_model;
  int32_t private_outputs;
  int32_t route;
  int64_t route_threshold;
  int32_t compare_bits;
} zk_statement_options;

enum zk_statement_layout_index {
  ZK_LAYOUT_BATCH = 0,
  ZK_LAYOUT_N_IN,
  ZK_LAYOUT_N_OUT,
  ZK_LAYOUT_OUTPUTS_START,
  ZK_LAYOUT_MODEL_TAG,
  ZK_LAYOUT_CONTEXT,
  ZK_LAYOUT_MODEL_COMMITMENT,
  ZK_LAYOUT_INPUTS_START,
  ZK_LAYOUT_INPUT_SLOT,
  ZK_LAYOUT_ROUTE_START,
  ZK_LAYOUT_NUM_PUBLIC,
  ZK_STATEMENT_LAYOUT_WORDS
};

typedef struct zk_statement zk_statement;
int zk_statement_v2_build(const zk_layer* layers, int num_layers, const int64_t* inputs, int batch, int n_in,
                          const zk_statement_options* options, zk_statement** out, char* err, size_t err_cap);
void zk_statement_destroy(zk_statement* st);
int zk_statement_info(const zk_statement* st, int* num_constraints, int* num_variables, int* num_public,
                      int* num_private, size_t* nA, size_t* nB, size_t* nC);
int zk_statement_layout(const zk_statement* st, int32_t layout[ZK_STATEMENT_LAYOUT_WORDS]);
int zk_statement_r1cs(const zk_statement* st, zk_sparse_entry* A, zk_sparse_entry* B, zk_sparse_entry* C);
int zk_statement_witness(const zk_statement* st, void* w_mont);
int zk_statement_scores(const zk_statement* st, int64_t* scores);
int zk_statement_check(const zk_statement* st);
int zk_statement_write(const zk_statement* st, const char* r1cs_path, const char* wtns_path);
int zk_statement_meta_json(const zk_statement* st, uint64_t model_tag64, char* buf, size_t cap, size_t* len);

#ifdef __cplusplus
}
#endif
#endif /* ZKML_GPU_H */
