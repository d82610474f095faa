// Float rows into 4-bit codes with a scale, and optionally a zero point, per group of 32, 64 or 128 elements, and back.
//
// Without zero points   scale = max|x| / 7,       zero = 8
// with them             scale = (high - low) / 15, zero = -low / scale rounded to the nearest integer,
//                       low = min(0, min x), high = max(0, max x)
// The quotient is rounded to fp32 and then to the scale's type, and ends at that type's largest number; with the scale as it is
// stored, code = x / scale rounded to the nearest integer (halfway to even), plus zero, clamped to 0 ... 15.  Where the scale is
// 0 all values are.  A group with an infinity or a NaN gets a NaN scale and codes that stand for zeros.
// Both directions move every byte once and are bound by memory: 1,000,003 x 200 fp32 rows in steps of 208 take 179 us into codes
// (5.1 TB/s) and 207 back (4.5), 131072 x 4096 462 (5.2) and 544 (4.5).  Two rows in flight per thread; four are no faster.
#include "row_access.h"

#include <algorithm>
#include <type_traits>

namespace ixa {

namespace {

constexpr int kThreads = 256;

struct GroupParams {
    const void *in;
    void *out;
    uint8_t *codes, *zeros;
    void *scales;
    int64_t n, ld, row0;                        // row0: the first row of this launch
    int d, groups, chunks, rows, scale_type;    // chunks of 8 elements per row, rows that a workgroup works on at a time
};

__device__ __forceinline__ float load_scale(const void *scales, int type, int64_t i)
{
    return type == kTypeF32 ? static_cast<const float *>(scales)[i]
           : type == kTypeF16 ? (float)static_cast<const _Float16 *>(scales)[i] : (float)static_cast<const __bf16 *>(scales)[i];
}

// Floats in an order of integers: NaN with a sign lie below -infinity, others above infinity.
__device__ __forceinline__ int ordered(float v)
{
    const int b = __float_as_int(v);
    return b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float unordered(int k) { return __int_as_float(k ^ ((k >> 31) & 0x7fffffff)); }

// a / 7 or a / 15 (a >= 0) rounded to fp32: the quotient in 64 bits by its reciprocal and one correction is right to the last
// bit, and no quotient by 7 or 15 lies close enough to a halfway point of 32 bits for two roundings to differ from one.
template <int D>
__device__ __forceinline__ float quotient(double a)
{
    const double r = 1.0 / D, q = a * r;
    return (float)fma(fma(-(double)D, q, a), r, q);
}

// The integer nearest to x / s: q = x * inv rounded is off by less than 2^-17 before it is, so only what lies that close to a
// halfway point has to be looked at, by a remainder that fp32 holds exactly.
constexpr float kNearHalf = 0.5f - 0x1p-16f;
__device__ __forceinline__ float settle(float x, float s, float q)
{
    const float rest = fmaf(-q, s, x), half = 0.5f * s;
    const bool odd = ((int)q & 1) != 0;
    return rest > half || (rest == half && odd) ? q + 1.f : rest < -half || (rest == -half && odd) ? q - 1.f : q;
}

// Eight elements per thread, a group in 4, 8 or 16 neighbouring threads, two rows in flight.
template <typename T, int G, bool ZEROS>
__global__ __launch_bounds__(kThreads) void group_quantise_kernel(GroupParams p)
{
    constexpr int kLanes = G / kEight, kRows = 2;
    const int across = min(p.chunks, kThreads / kLanes * kLanes), in = threadIdx.x / across;
    if (in >= p.rows) {
        return;   // whole groups of lanes: `across` and `chunks` are multiples of kLanes
    }
    const int64_t first = p.row0 + (int64_t)blockIdx.x * (p.rows * kRows) + in;
    for (int c = threadIdx.x - in * across; c < p.chunks; c += across) {
        Eight<T> raw[kRows];
        const int at = c * kEight, count = min(kEight, max(0, p.d - at));
#pragma unroll
        for (int k = 0; k < kRows; k++) {
            const int64_t row = min(first + k * p.rows, p.n - 1);
            raw[k].load(static_cast<const T *>(p.in) + row * p.ld + (count ? at : 0), count, (T)0.f);
        }
#pragma unroll
        for (int k = 0; k < kRows; k++) {
            const int64_t row = first + k * p.rows;
            float x[kEight];
#pragma unroll
            for (int i = 0; i < kEight; i++) {
                x[i] = (float)raw[k].v[i];
            }
            float scale;
            bool bad;
            double low = 0.0;
            if constexpr (ZEROS) {
                int least = 0, most = 0;    // the order of 0
#pragma unroll
                for (int i = 0; i < kEight; i++) {
                    least = min(least, ordered(x[i]));
                    most = max(most, ordered(x[i]));
                }
                least = over_lanes<kLanes>(least, [](int a, int b) { return min(a, b); });
                most = over_lanes<kLanes>(most, [](int a, int b) { return max(a, b); });
                const float inf = __builtin_inff();
                bad = most >= ordered(inf) || least <= ordered(-inf);
                low = bad ? 0.0 : (double)unordered(least);
                scale = quotient<15>(bad ? 0.0 : (double)unordered(most) - low);
            } else {
                int top = 0;
#pragma unroll
                for (int i = 0; i < kEight; i++) {
                    top = max(top, __float_as_int(x[i]) & 0x7fffffff);
                }
                top = over_lanes<kLanes>(top, [](int a, int b) { return max(a, b); });
                bad = top >= 0x7f800000;
                scale = quotient<7>(bad ? 0.0 : (double)__int_as_float(top));
            }
            _Float16 scale16 = (_Float16)fminf(scale, 65504.f);
            __bf16 scale_b = (__bf16)fminf(scale, 0x1.fep127f);
            scale = p.scale_type == kTypeF32 ? scale : p.scale_type == kTypeF16 ? (float)scale16 : (float)scale_b;
            // the reciprocal of a small scale would not be finite
            const float unit = scale < 0x1p-90f ? 0x1p64f : 1.f, s = scale * unit;
            const float inv = s > 0.f && !bad ? 1.0f / s : 0.f;
            float zero = 8.f;
            if constexpr (ZEROS) {
                const float y = (float)-low * unit;
                zero = s > 0.f ? fminf(settle(y, s, rintf(y * inv)), 15.f) : 0.f;
            }
            float q[kEight], nearest = 0.f;
#pragma unroll
            for (int i = 0; i < kEight; i++) {
                x[i] = bad ? 0.f : x[i] * unit;
                const float t = x[i] * inv;
                q[i] = rintf(t);
                nearest = fmaxf(nearest, fabsf(t - q[i]));
            }
            if (nearest > kNearHalf) {
#pragma unroll
                for (int i = 0; i < kEight; i++) {
                    q[i] = fabsf(q[i]) < 32.f ? settle(x[i], s, q[i]) : q[i];
                }
            }
            float half[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                half[h] = 0.f;
#pragma unroll
                for (int i = 3; i >= 0; i--) {
                    half[h] = fmaf(half[h], 16.f, __builtin_amdgcn_fmed3f(q[4 * h + i] + zero, 0.f, 15.f));
                }
            }
            if (row < p.n) {
                reinterpret_cast<uint32_t *>(p.codes)[row * p.chunks + c] = (uint32_t)half[0] | (uint32_t)half[1] << 16;
                if (c % kLanes == 0) {
                    const int64_t slot = row * p.groups + c / kLanes;
                    if (p.scale_type == kTypeF32) {
                        static_cast<float *>(p.scales)[slot] = bad ? __builtin_nanf("") : scale;
                    } else if (p.scale_type == kTypeF16) {
                        static_cast<_Float16 *>(p.scales)[slot] = bad ? (_Float16)__builtin_nanf("") : scale16;
                    } else {
                        static_cast<__bf16 *>(p.scales)[slot] = bad ? (__bf16)__builtin_nanf("") : scale_b;
                    }
                    if constexpr (ZEROS) {
                        p.zeros[slot] = (uint8_t)zero;
                    }
                }
            }
        }
    }
}

// Eight codes per thread, two rows in flight.
template <typename T, int G, bool PAST>
__global__ __launch_bounds__(kThreads) void group_read_kernel(GroupParams p)
{
    constexpr int kLanes = G / kEight, kRows = 2;
    const int across = min(p.chunks, kThreads), in = threadIdx.x / across;
    if (in >= p.rows) {
        return;
    }
    const int64_t first = p.row0 + (int64_t)blockIdx.x * (p.rows * kRows) + in;
    for (int c = threadIdx.x - in * across; c < p.chunks; c += kThreads) {
        uint32_t code[kRows];
        float scale[kRows], zero[kRows];
#pragma unroll
        for (int k = 0; k < kRows; k++) {
            const int64_t row = min(first + k * p.rows, p.n - 1), slot = row * p.groups + c / kLanes;
            code[k] = reinterpret_cast<const uint32_t *>(p.codes)[row * p.chunks + c];
            scale[k] = load_scale(p.scales, p.scale_type, slot);
            zero[k] = p.zeros ? (float)p.zeros[slot] : 8.f;
        }
#pragma unroll
        for (int k = 0; k < kRows; k++) {
            const int64_t row = first + k * p.rows;
            Eight<T> v;
#pragma unroll
            for (int i = 0; i < kEight; i++) {
                float product = ((float)(code[k] >> (4 * i) & 15u) - zero[k]) * scale[k];
                asm("" : "+v"(product));   // a product in fp32 it is: one instruction for it and fp16 would round only once
                v.v[i] = (T)product;
            }
            if (row < p.n) {
                const int at = c * kEight;
                v.template store<PAST>(static_cast<T *>(p.out) + row * p.ld + min(at, p.d), min(kEight, p.d - at));
            }
        }
    }
}

// A launch has less than 2^32 threads: more rows than half a million workgroups take go in several.
template <typename Launch>
void in_launches(GroupParams p, Launch launch)
{
    constexpr int64_t kGroups = 1 << 19;
    const int64_t rows = (int64_t)p.rows * 2;
    for (p.row0 = 0; p.row0 < p.n; p.row0 += kGroups * rows) {
        launch(p, dim3((unsigned)std::min(kGroups, (p.n - p.row0 + rows - 1) / rows)));
        check_launch();
    }
}

template <typename F>
void with_group(int group, F f)
{
    if (group == 32) {
        f(std::integral_constant<int, 32>());
    } else if (group == 64) {
        f(std::integral_constant<int, 64>());
    } else {
        f(std::integral_constant<int, 128>());
    }
}

GroupParams params(int64_t n, int d, int group, int scale_type)
{
    GroupParams p{};
    p.n = n;
    p.d = d;
    p.groups = group_count(group, d);
    p.chunks = p.groups * (group / kEight);
    p.rows = std::max(1, kThreads / p.chunks);
    p.scale_type = scale_type;
    return p;
}

}  // namespace

void check_groups(const char *op, int group, int scale_type, int64_t n, int d, const uint8_t *codes, const void *scales)
{
    IXA_REQUIRE(group == 32 || group == 64 || group == 128, kErrInvalidParam, "%s: groups of %d elements (32, 64 or 128)", op,
                group);
    check_type(op, scale_type);
    IXA_REQUIRE(n >= 0 && n <= 0x7fffffff && d >= 1 && d <= kMaxCodeDim, kErrInvalidParam,
                "%s: rows %ld (< 2^31), dims %d (1 ... %d)", op, (long)n, d, kMaxCodeDim);
    IXA_REQUIRE((codes && scales) || n == 0, kErrInvalidParam, "operator buffers can not be nullptr.");
    IXA_REQUIRE(on_bytes(codes, 16) && on_bytes(scales, element_bytes(scale_type)), kErrInvalidParam,
                "%s: codes have to start on 16 bytes, scales on their elements", op);
}

void op_group_quantise(const void *x, int64_t ld, int type, int64_t n, int d, int group, int scale_type, uint8_t *codes,
                       void *scales, uint8_t *zeros, hipStream_t s)
{
    check_type("group_quantise", type);
    check_groups("group_quantise", group, scale_type, n, d, codes, scales);
    check_row_buffer("group_quantise", x, ld, type, n, d);
    if (n == 0) {
        return;
    }
    GroupParams p = params(n, d, group, scale_type);
    p.in = x;
    p.ld = ld;
    p.codes = codes;
    p.scales = scales;
    p.zeros = zeros;
    with_type(type, [&](auto t) {
        with_group(group, [&](auto g) {
            in_launches(p, [&](const GroupParams &q, dim3 grid) {
                if (zeros) {
                    hipLaunchKernelGGL((group_quantise_kernel<decltype(t), decltype(g)::value, true>), grid, dim3(kThreads), 0, s, q);
                } else {
                    hipLaunchKernelGGL((group_quantise_kernel<decltype(t), decltype(g)::value, false>), grid, dim3(kThreads), 0, s, q);
                }
            });
        });
    });
}

void op_group_dequantise(const uint8_t *codes, const void *scales, const uint8_t *zeros, int group, int scale_type, int64_t n,
                         int d, int type, void *out, int64_t ld, hipStream_t s)
{
    check_type("group_dequantise", type);
    check_groups("group_dequantise", group, scale_type, n, d, codes, scales);
    check_row_buffer("group_dequantise", out, ld, type, n, d);
    if (n == 0) {
        return;
    }
    // Rows that do not fit into the last cache go past it: 1,000,003 x 200 fp32 222 -> 207 us, and a quantisation that follows has no lines to
    // write back, 216 -> 179; 131072 x 4096 615 -> 544 and 506 -> 462.  16384 x 768, which fit, 13.8 -> 19.5.
    const bool past = (double)n * (double)ld * (double)element_bytes(type) > 0x1p27;
    GroupParams p = params(n, d, group, scale_type);
    p.out = out;
    p.ld = ld;
    p.codes = const_cast<uint8_t *>(codes);
    p.scales = const_cast<void *>(scales);
    p.zeros = const_cast<uint8_t *>(zeros);
    with_type(type, [&](auto t) {
        with_group(group, [&](auto g) {
            in_launches(p, [&](const GroupParams &q, dim3 grid) {
                if (past) {
                    hipLaunchKernelGGL((group_read_kernel<decltype(t), decltype(g)::value, true>), grid, dim3(kThreads), 0, s, q);
                } else {
                    hipLaunchKernelGGL((group_read_kernel<decltype(t), decltype(g)::value, false>), grid, dim3(kThreads), 0, s, q);
                }
            });
        });
    });
}

}  // namespace ixa
