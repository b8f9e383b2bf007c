/*
 * mvquant -- B200 (sm_100a) operators of a decode step with 4-bit weights.
 *
 * C ABI of libmvquant.so: products with 4-bit weights and group scales, the
 * weights written out, and the row operations that feed those products (the
 * residual's addition with RMSNorm, the gated activation) with an optional
 * output in 8 bits. Conventions are those of mvdecode.h: plain device
 * pointers, strides in elements, work enqueued on the caller's CUDA stream, an
 * MVQ_* status returned, the message of a failure from mvq_last_error()
 * (thread-local). Nothing here allocates, synchronises the device, reads
 * device memory from the host or keeps state between calls. Call with the
 * device that owns the pointers current.
 *
 * Every call takes one struct whose fields are 8 bytes wide, in this order,
 * with no padding (a binding that pays per marshalled argument fills it once).
 *
 * No reference counterpart: micro-vllm computes these layers with torch tensor
 * operations on unquantised weights (src/micro_vllm/model.py:25-41, 126-165).
 */
#ifndef MVQUANT_H_
#define MVQUANT_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#define MVQ_API __attribute__((visibility("default")))
#else
#define MVQ_API
#endif

#define MVQ_ABI_VERSION 1

/* Element types; the first three are mvdecode.h's. */
#define MVQ_DTYPE_F32 0
#define MVQ_DTYPE_F16 1
#define MVQ_DTYPE_BF16 2
#define MVQ_DTYPE_I8 3
#define MVQ_DTYPE_E4M3 4

/* Status codes (mvdecode.h's values). */
#define MVQ_OK 0
#define MVQ_ERR_INVALID_ARGUMENT 1
#define MVQ_ERR_UNSUPPORTED 2
#define MVQ_ERR_CUDA 4

/*
 * The weight's records. W is [n, k], W[r, c] = (code - zero) * scale with code
 * and zero in 0..15 and one scale (and zero) per row and per `group` columns
 * (32, 64 or 128). It is cut into tiles of 64 rows and chunks of 128 columns,
 * both padded; the record of tile i and chunk j starts at byte
 * (i * ceil(k / 128) + j) * record_bytes of `records` and holds
 *   4096 bytes of codes: [h 0..3][p 0..1][lane 0..31][word 0..3] 32-bit words.
 *     With g = lane / 4, t = lane % 4 and word = 2 q + e, the word holds the
 *     columns c = 32 h + 16 e + 4 t + s (s 0..3) of rows 32 p + 16 q + g (the low
 *     nibbles of bytes) and 32 p + 16 q + 8 + g (the high nibbles), s = 0, 2, 1, 3
 *     in bytes 0..3, each nibble the code with its highest bit inverted;
 *   128 bytes of scales for each group of the chunk: [g 0..7][p][q][half], fp16
 *     or bf16, of row 32 p + 16 q + 8 half + g;
 *   with zero points, 64 bytes for each group: zero - 8 as int8, in that order.
 * A record is a multiple of 64 bytes; `records` is aligned to 16.
 */
#define MVQ_TILE_ROWS 64
#define MVQ_CHUNK_COLUMNS 128

/*
 * y = (x W^T) * x_scale + bias + residual for m rows of x: sums in fp32 (in
 * 32-bit integers within a group for int8 x), one rounding to out_dtype.
 * x: [m, k] of x_dtype, feature stride 1; x_scale: [m] fp32, or NULL for 1.
 * bias [n] and residual [m, n]: of out_dtype, or NULL; residual may be out.
 */
typedef struct MvqLinearArgs {
    const void* x; int64_t x_stride_row; const void* x_scale;
    const void* records; int64_t n; int64_t k; int64_t group; int64_t has_zeros; int64_t scale_dtype;
    const void* bias; const void* residual; int64_t residual_stride_row;
    void* out; int64_t out_stride_row; int64_t m; int64_t x_dtype; int64_t out_dtype;
} MvqLinearArgs;
MVQ_API int mvq_w4_linear(const MvqLinearArgs* args, void* stream);

/* out[r, c] = (code - zero) * scale, rounded once to out_dtype (fp32, fp16 or bf16). */
typedef struct MvqDequantizeArgs {
    const void* records; int64_t n; int64_t k; int64_t group; int64_t has_zeros; int64_t scale_dtype;
    void* out; int64_t out_stride_row; int64_t out_dtype;
} MvqDequantizeArgs;
MVQ_API int mvq_w4_dequantize(const MvqDequantizeArgs* args, void* stream);

/*
 * For each row: s = to_dtype(x + residual), y = weight * s * rsqrt(mean(s^2) +
 * eps) in fp32. residual_out (if not NULL) gets s. residual NULL: s = x.
 * out_dtype == dtype: out gets y, rounded once. MVQ_DTYPE_I8 / MVQ_DTYPE_E4M3:
 * scales[row] = max|y| / top (top 127 / 448) and out = round(y / scale), ties to
 * even, zeros where the scale is zero; a row with a NaN or an infinite y gets a
 * NaN scale and zeros. residual_out may be x or residual; in dtype, out may be x
 * (an 8-bit out may not lie over an input).
 */
typedef struct MvqNormArgs {
    const void* x; int64_t x_stride_row; const void* residual; int64_t residual_stride_row;
    const void* weight; void* out; int64_t out_stride_row; void* scales;
    void* residual_out; int64_t residual_out_stride_row; int64_t rows; int64_t hidden; double eps;
    int64_t dtype; int64_t out_dtype;
} MvqNormArgs;
MVQ_API int mvq_add_rms_norm(const MvqNormArgs* args, void* stream);

/*
 * y = silu(g) * u in fp32 for rows [g | u] of 2 * width elements (zero for g below
 * -88.72, where exp(-g) passes fp32's range); out and scales as above (8 bits only).
 */
typedef struct MvqSiluArgs {
    const void* gate_up; int64_t stride_row; void* out; int64_t out_stride_row; void* scales;
    int64_t rows; int64_t width; int64_t dtype; int64_t out_dtype;
} MvqSiluArgs;
MVQ_API int mvq_silu_mul_quant(const MvqSiluArgs* args, void* stream);

/*
 * Sticky bit of this library's kernels on `device`: 1 if a bounded wait gave up
 * (its call's result is NaN). Reading synchronises with the device's legacy
 * stream, as mv_device_status does for libmvdecode.so.
 */
#define MVQ_DEVICE_STATUS_WAIT_TIMEOUT 1
MVQ_API int mvq_device_status(int32_t device, uint32_t* status);
MVQ_API int mvq_clear_device_status(int32_t device);

/*
 * Exercises that path, as mv_selftest_wait_timeout does for libmvdecode.so: one
 * warp on `stream` waits, as the kernels do, on a barrier that nothing completes,
 * for limit_ns (at most 100 ms), gives up, sets the bit and returns.
 */
MVQ_API int mvq_selftest_wait_timeout(uint64_t limit_ns, void* stream);

MVQ_API int mvq_abi_version(void);

/* Message for the last non-MVQ_OK status returned on this thread. */
MVQ_API const char* mvq_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* MVQUANT_H_ */
