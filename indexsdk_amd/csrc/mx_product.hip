// Scores of query rows a against stored rows b in microscaled codes: g[i][j] = sum over k of a[i][k] b[j][k], or the squared
// distance (|a_i|^2 + |b_j|^2) - g - g in the library's expanded form.
//
// v_mfma_scale_f32_32x32x64_f8f6f4 multiplies 32 x 64 by 64 x 32 codes and applies the power-of-two scale of each row's
// block of 32 itself.  A lane (row l & 31, half h = l >> 5) gives it, in 4 bits, the 16 bytes of block h of its row; in 8
// bits, bytes 16 h .. 16 h + 15 of block 0 and the same of block 1; and in both the scale of block h.
//
// Two 4-bit numbers multiply and add up without any loss in the instruction.  Products of an 8-bit and a 4-bit number span
// more bits than it keeps (what lies under about 2^-14 of the largest product is dropped: 1e-4 of the sum of magnitudes
// was measured on random codes), so an 8-bit operand goes in twice: the codes of magnitude 2 and more, then the others.
// Within either half all products are multiples of the smallest that the instruction keeps (2^8.8 * 6 against 2^-2 * 0.5, and
// 2 * 6 against 2^-9 * 0.5), and the sums are those of 32 bits.
#include "lowp.h"

namespace ixa {

namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));

constexpr int kE4M3 = 0, kE2M1 = 4;   // operand formats of the instruction

struct ProductParams {
    const uint8_t *a_codes, *a_scales, *b_codes, *b_scales;
    const float *a_sqr, *b_sqr;
    int64_t m, n, ld;
    int blocks, metric;
    void *out;
};

// bytes of w whose magnitude is 2 or more (E4M3: exponent field 8 and up) as ones
__device__ __forceinline__ uint32_t large_bytes(uint32_t w)
{
    const uint32_t u = (w >> 6) & 0x01010101u;
    return (u << 8) - u;
}

template <int FA>
__device__ __forceinline__ v16f multiply(const uint4 (&a)[FA == kE2M1 ? 1 : 2], uint32_t a_scale, uint4 b, uint32_t b_scale,
                                         v16f c)
{
    const v8i bv = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
    if constexpr (FA == kE2M1) {
        const v8i av = {(int)a[0].x, (int)a[0].y, (int)a[0].z, (int)a[0].w, 0, 0, 0, 0};
        return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, c, kE2M1, kE2M1, 0, (int)a_scale, 0, (int)b_scale);
    } else {
        const uint32_t w[8] = {a[0].x, a[0].y, a[0].z, a[0].w, a[1].x, a[1].y, a[1].z, a[1].w};
        v8i lo, hi;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t mask = large_bytes(w[i]);
            lo[i] = (int)(w[i] & ~mask);
            hi[i] = (int)(w[i] & mask);
        }
        c = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(lo, bv, c, kE4M3, kE2M1, 0, (int)a_scale, 0, (int)b_scale);
        return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(hi, bv, c, kE4M3, kE2M1, 0, (int)a_scale, 0, (int)b_scale);
    }
}

// One wavefront per 32 x 32 scores, operands straight from memory.
template <int FA, typename T>
__global__ __launch_bounds__(256) void mx_product_kernel(ProductParams p)
{
    const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
    const int64_t col_tiles = (p.n + 31) / 32;
    const int64_t tile = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int64_t row0 = tile / col_tiles * 32, col0 = tile % col_tiles * 32;
    if (row0 >= p.m) {
        return;
    }
    const int64_t arow = min(row0 + r, p.m - 1), brow = min(col0 + r, p.n - 1);
    constexpr int kABytes = FA == kE2M1 ? 16 : 32;
    const uint8_t *ac = p.a_codes + arow * p.blocks * kABytes, *as = p.a_scales + arow * p.blocks;
    const uint8_t *bc = p.b_codes + brow * p.blocks * 16, *bs = p.b_scales + brow * p.blocks;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    v16f acc = {};
    for (int t = 0; t < p.blocks; t += 2) {
        const bool mine = t + h < p.blocks;   // the second block of the last step may not exist: zero codes, scale 1
        uint4 a[FA == kE2M1 ? 1 : 2];
        if constexpr (FA == kE2M1) {
            a[0] = mine ? *reinterpret_cast<const uint4 *>(ac + (t + h) * 16) : zero;
        } else {
            a[0] = *reinterpret_cast<const uint4 *>(ac + t * 32 + h * 16);
            a[1] = t + 1 < p.blocks ? *reinterpret_cast<const uint4 *>(ac + t * 32 + 32 + h * 16) : zero;
        }
        const uint4 b = mine ? *reinterpret_cast<const uint4 *>(bc + (t + h) * 16) : zero;
        acc = multiply<FA>(a, mine ? as[t + h] : 127, b, mine ? bs[t + h] : 127, acc);
    }
    const int64_t col = col0 + r;
    if (col >= p.n) {
        return;
    }
    const bool l2 = p.metric == kMetricL2;
    const float bq = l2 ? p.b_sqr[col] : 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int64_t row = row0 + 8 * (i / 4) + 4 * h + i % 4;
        if (row < p.m) {
            float v = acc[i];
            if (l2) {
                v = (p.a_sqr[row] + bq) - v - v;
            }
            static_cast<T *>(p.out)[row * p.ld + col] = (T)v;
        }
    }
}

template <int FA>
void launch(const ProductParams &p, int out_type, hipStream_t s)
{
    const int64_t tiles = ((p.m + 31) / 32) * ((p.n + 31) / 32);
    IXA_REQUIRE(tiles <= (int64_t)4 * 0x7fffffff, kErrInvalidParam, "mx_product: %ld x %ld scores in one call", (long)p.m,
                (long)p.n);
    const dim3 grid((unsigned)((tiles + 3) / 4));
    if (out_type == kTypeF32) {
        hipLaunchKernelGGL((mx_product_kernel<FA, float>), grid, dim3(256), 0, s, p);
    } else if (out_type == kTypeF16) {
        hipLaunchKernelGGL((mx_product_kernel<FA, _Float16>), grid, dim3(256), 0, s, p);
    } else {
        hipLaunchKernelGGL((mx_product_kernel<FA, __bf16>), grid, dim3(256), 0, s, p);
    }
    check_launch();
}

bool aligned(const void *p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

}  // namespace

void op_mx_product(const uint8_t *a_codes, const uint8_t *a_scales, int a_format, int64_t m, const uint8_t *b_codes,
                   const uint8_t *b_scales, int64_t n, int d, int metric, const float *a_sqr, const float *b_sqr,
                   int out_type, void *out, int64_t ld, hipStream_t s)
{
    IXA_REQUIRE(a_codes && a_scales && b_codes && b_scales && out, kErrInvalidParam, "operator buffers can not be nullptr.");
    IXA_REQUIRE(a_format == kFormatMxFp8 || a_format == kFormatMxFp4, kErrInvalidParam,
                "mx_product: unsupported code format %d", a_format);
    IXA_REQUIRE(out_type >= kTypeF32 && out_type <= kTypeBF16, kErrInvalidParam, "mx_product: unsupported element type %d",
                out_type);
    IXA_REQUIRE(m >= 0 && m <= 0x7fffffff && n >= 0 && n <= 0x7fffffff && d >= 1 && d <= kMaxCodeDim, kErrInvalidParam,
                "mx_product: rows %ld x %ld (< 2^31), dims %d (1 ... %d)", (long)m, (long)n, d, kMaxCodeDim);
    IXA_REQUIRE(ld >= n && ld <= (int64_t)1 << 40, kErrInvalidParam, "mx_product: rows of %ld scores in steps of %ld", (long)n,
                (long)ld);
    IXA_REQUIRE(metric == kMetricL2 || metric == kMetricInnerProduct, kErrInvalidParam, "Unsupported metric type");
    IXA_REQUIRE(metric != kMetricL2 || (a_sqr && b_sqr), kErrInvalidParam,
                "mx_product: squared distances need the squared norms of both sides");
    IXA_REQUIRE(aligned(a_codes, 16) && aligned(b_codes, 16) && aligned(out, out_type == kTypeF32 ? 4 : 2) &&
                    aligned(a_sqr, 4) && aligned(b_sqr, 4),
                kErrInvalidParam, "mx_product: codes have to start on 16 bytes, norms and scores on their elements");
    if (m == 0 || n == 0) {
        return;
    }
    const ProductParams p{a_codes, a_scales, b_codes, b_scales, a_sqr, b_sqr, m, n, ld, mx_blocks(d), metric, out};
    if (a_format == kFormatMxFp4) {
        launch<kE2M1>(p, out_type, s);
    } else {
        launch<kE4M3>(p, out_type, s);
    }
}

}  // namespace ixa
