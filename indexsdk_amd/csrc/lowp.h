// Low-precision operators on embeddings: codes of 8 and 4 bits with scales, made from float rows (alone or behind a
// root-mean-square norm), read back, and multiplied (see quantise.hip and mx_product.hip).
#pragma once
#include "common.h"

#include <algorithm>
#include <map>
#include <tuple>

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

// Rows of 4-bit codes with a scale, and where `zeros` is given a zero point, for each group of `group` (32, 64 or 128) elements:
// value = (code - zero) * scale.  The lower half of a byte comes first; rows take whole groups.
inline int group_count(int group, int d) { return (d + group - 1) / group; }
inline int64_t group_row_bytes(int group, int d) { return (int64_t)group_count(group, d) * (group / 2); }
void check_groups(const char *op, int group, int scale_type, int64_t n, int d, const uint8_t *codes, const void *scales);

// Rows x[n][ld] become codes, scales of scale_type [n][groups] and, unless null, zeros [n][groups].
void op_group_quantise(const void *x, int64_t ld, int type, int64_t n, int d, int group, int scale_type, uint8_t *codes,
                       void *scales, uint8_t *zeros, hipStream_t s);

// Their values, rounded to `type`, in rows out[n][ld].
void op_group_dequantise(const uint8_t *codes, const void *scales, const uint8_t *zeros, int group, int scale_type, int64_t n,
                         int d, int type, void *out, int64_t ld, hipStream_t s);

// out[m][ld] = alpha * (rows x . the values of rows of codes) + bias (may be null), rounded to out_type.  The workspace takes
// group_product_workspace bytes and holds x as the matrix cores want it where there are many rows or long ones.
constexpr int64_t kMaxProductRows = 1 << 23;
int64_t group_product_workspace(int type, int64_t m, int d);
void op_group_product(const void *x, int64_t ld_x, int type, int64_t m, const uint8_t *codes, const void *scales,
                      const uint8_t *zeros, int group, int scale_type, int64_t n, int d, float alpha, const float *bias,
                      int out_type, void *out, int64_t ld, void *workspace, int64_t workspace_bytes, hipStream_t s);

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

// Workgroups of a kernel that the current device runs at a time: devices and partitions differ in their CUs.
inline int64_t resident_workgroups(const void *kern, int threads, size_t lds)
{
    static std::mutex mu;
    static std::map<std::tuple<int, const void *, int, size_t>, int64_t> known;
    int device;
    IXA_HIP(hipGetDevice(&device));
    std::lock_guard<std::mutex> lock(mu);
    int64_t &count = known[std::make_tuple(device, kern, threads, lds)];
    if (count == 0) {
        int per_cu = 0, cus = 0;
        IXA_HIP(hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, kern, threads, lds));
        IXA_HIP(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device));
        count = (int64_t)std::max(1, per_cu) * std::max(1, cus);
    }
    return count;
}

}  // namespace ixa
