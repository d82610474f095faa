// Low-precision operators on embeddings: codes of 8 and 4 bits with scales, made from float rows (alone or behind a
// root-mean-square norm), read back, and multiplied (see quantise.hip and mx_product.hip).
#pragma once
#include "common.h"

namespace ixa {

// Element types of float rows and of results.
enum ElementType : int { kTypeF32 = 0, kTypeF16 = 1, kTypeBF16 = 2 };

// Code formats.  The microscaled ones hold blocks of 32 consecutive elements of a row; a block's scale is a power of two,
// stored as its exponent + 127 in one byte (255: not a number).
enum CodeFormat : int {
    kFormatInt8 = 0,    // d bytes, one fp32 scale per row
    kFormatMxFp8 = 1,   // ceil(d / 32) blocks of 32 bytes (E4M3, largest number 448)
    kFormatMxFp4 = 2,   // ceil(d / 32) blocks of 16 bytes (E2M1, largest number 6; the lower half of a byte comes first)
};

constexpr int kMxBlock = 32;
constexpr int kMaxCodeDim = 16384;

inline int mx_blocks(int d) { return (d + kMxBlock - 1) / kMxBlock; }
// Bytes of one row's codes.
inline int64_t code_bytes(int format, int d)
{
    return format == kFormatInt8 ? d : (int64_t)mx_blocks(d) * (format == kFormatMxFp8 ? 32 : 16);
}

// Rows x[n][ld] of element type `type` become codes and scales; sqr_sum (may be null) takes the squared norms of what the
// codes stand for.  fixed_scale > 0 (int8 only): every row's scale.
void op_quantise(const void *x, int64_t ld, int type, int64_t n, int d, int format, float fixed_scale, uint8_t *codes,
                 void *scales, float *sqr_sum, hipStream_t s);

// The values that codes and scales stand for, rounded to element type `type`, in rows out[n][ld].
void op_dequantise(const uint8_t *codes, const void *scales, int format, int64_t n, int d, int type, void *out, int64_t ld,
                   hipStream_t s);

// h = x + residual (residual may be null), written to sum (may be null) rounded to the type; codes and scales of
// h / sqrt(mean(h^2) + eps) * weight (weight may be null: 1).
void op_rms_norm_quantise(const void *x, int64_t ld_x, const void *residual, int64_t ld_residual, const void *weight,
                          int type, int64_t n, int d, float eps, void *sum, int64_t ld_sum, int format, float fixed_scale,
                          uint8_t *codes, void *scales, float *sqr_sum, hipStream_t s);

// out[m][ld] = scores of rows a (MXFP4 or MXFP8) against rows b (MXFP4): inner products g, or (a_sqr + b_sqr) - 2 g.
void op_mx_product(const uint8_t *a_codes, const uint8_t *a_scales, int a_format, int64_t m, const uint8_t *b_codes,
                   const uint8_t *b_scales, int64_t n, int d, int metric, const float *a_sqr, const float *b_sqr,
                   int out_type, void *out, int64_t ld, hipStream_t s);

// An error the device (or its absence) answered with becomes this library's.
inline void check_answer(hipError_t e)
{
    if (e == hipSuccess) {
        return;
    }
    int count = 0;
    IXA_REQUIRE(hipGetDeviceCount(&count) == hipSuccess && count > 0, kErrIndexNotInit,
                "no HIP device available: this library has no CPU path");
    IXA_HIP(e);
}
// after a launch
inline void check_launch() { check_answer(hipGetLastError()); }

}  // namespace ixa
