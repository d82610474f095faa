// Float rows into codes of 8 or 4 bits with scales, alone or behind a residual addition and a root-mean-square norm, and
// codes back into float rows.  All three move every byte once and compute little: they are bound by memory, a few rows by
// the latency of one load and of the sums over a row.
//
// Microscaled formats (blocks of 32 elements x_0..x_31 of a row; columns behind the last are zeros):
//   E = clamp(floor(log2 max|x_i|) - t + 127, 0, 254), t = 2 for E2M1 and 8 for E4M3 (their largest power of two); zeros: 0
//   code_i = x_i * 2^(127 - E) rounded to the nearest number of the format, halfway to even, beyond the largest to it
// A block that holds an infinity or a NaN gets E = 255, the scale that stands for NaN, and zero codes.
// int8: scale = max|x| / 127 over the row, code = x * (127 / max|x|) rounded to the nearest integer, halfway to even; a row
// that holds an infinity or a NaN gets a NaN scale and zero codes.  With a fixed scale, codes are clamped to +-127, NaN to 0.
#include "lowp.h"

#include <algorithm>
#include <type_traits>

namespace ixa {

namespace {

typedef float f2 __attribute__((ext_vector_type(2)));
typedef short s2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kVec = 8;                       // elements a lane handles at a time: four lanes hold one block
constexpr uint32_t kInfBits = 0x7f800000u;
constexpr uint32_t kNaNScale = 255;

template <typename T>
struct Vec8 {
    T v[kVec];
};

// Eight elements as they lie in memory.
template <typename T>
struct Raw8 {
    u4 w[kVec * sizeof(T) / 16];
    __device__ __forceinline__ void values(float (&v)[kVec]) const
    {
        const Vec8<T> t = __builtin_bit_cast(Vec8<T>, *this);
#pragma unroll
        for (int i = 0; i < kVec; i++) {
            v[i] = (float)t.v[i];
        }
    }
};

// `count` elements, zeros behind them.  FILL: none of them are loaded like eight, which p then points at, so that nothing
// diverges.
template <bool FILL, typename T>
__device__ __forceinline__ Raw8<T> load8(const T *__restrict__ p, int count, bool whole)
{
    if (whole && (count == kVec || (FILL && count == 0))) {
        Raw8<T> w;
#pragma unroll
        for (size_t i = 0; i < kVec * sizeof(T) / 16; i++) {
            w.w[i] = reinterpret_cast<const u4 *>(p)[i];
            w.w[i] = FILL && count == 0 ? u4{} : w.w[i];
        }
        return w;
    }
    Vec8<T> t;
#pragma unroll
    for (int i = 0; i < kVec; i++) {
        t.v[i] = i < count ? p[i] : (T)0.f;
    }
    return __builtin_bit_cast(Raw8<T>, t);
}

// PAST: past the caches (two kinds of store in one kernel would be merged into the ordinary one)
template <bool PAST, typename T>
__device__ __forceinline__ void store8(T *__restrict__ p, int count, bool whole, const float (&v)[kVec])
{
    if (whole && count == kVec) {
        constexpr int kWords = kVec * sizeof(T) / 16;
        struct Words {
            u4 w[kWords];
        };
        Vec8<T> t;
#pragma unroll
        for (int i = 0; i < kVec; i++) {
            t.v[i] = (T)v[i];
        }
        const Words w = __builtin_bit_cast(Words, t);
#pragma unroll
        for (int i = 0; i < kWords; i++) {
            if constexpr (PAST) {
                __builtin_nontemporal_store(w.w[i], reinterpret_cast<u4 *>(p) + i);
            } else {
                reinterpret_cast<u4 *>(p)[i] = w.w[i];
            }
        }
    } else if (count > 0) {
#pragma unroll
        for (int i = 0; i < kVec; i++) {
            if (i < count) {
                p[i] = (T)v[i];
            }
        }
    }
}

// lane exchanges inside four, eight and sixteen lanes without the LDS
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v)
{
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
constexpr int kQuadXor1 = 0xb1, kQuadXor2 = 0x4e, kHalfMirror = 0x141, kMirror = 0x140;

__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }

// the largest value of four lanes that hold one block
__device__ __forceinline__ uint32_t quad_max(uint32_t v)
{
    v = umax(v, dpp<kQuadXor1>(v));
    return umax(v, dpp<kQuadXor2>(v));
}

// v of another lane, 32 or 64 bits
template <int CTRL, typename V>
__device__ __forceinline__ V dpp_of(V v)
{
    if constexpr (sizeof(V) == 4) {
        return __builtin_bit_cast(V, dpp<CTRL>(__builtin_bit_cast(uint32_t, v)));
    } else {
        const uint2 w = __builtin_bit_cast(uint2, v);
        return __builtin_bit_cast(V, make_uint2(dpp<CTRL>(w.x), dpp<CTRL>(w.y)));
    }
}

// v of a lane and of the one 16 or 32 (HALVES) lanes from it, joined: swapping odd rows of 16 lanes (the upper half) of one
// register with even ones (the lower half) of its copy leaves one of the two in either register, without the LDS
template <bool HALVES, typename V, typename Op>
__device__ __forceinline__ V swapped(V v, Op op)
{
    struct Box {
        uint32_t w[sizeof(V) / 4];
    };
    Box a = __builtin_bit_cast(Box, v), b;
#pragma unroll
    for (size_t i = 0; i < sizeof(V) / 4; i++) {
        const auto t = HALVES ? __builtin_amdgcn_permlane32_swap(a.w[i], a.w[i], false, false)
                              : __builtin_amdgcn_permlane16_swap(a.w[i], a.w[i], false, false);
        a.w[i] = t[0];
        b.w[i] = t[1];
    }
    return op(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b));
}

// Reductions over the L lanes of a row; with L = 256 over the workgroup, through `box` (a barrier on either side).
template <int L, typename V, typename Op>
__device__ __forceinline__ V row_reduce(V v, double *box, Op op)
{
    v = op(v, dpp_of<kQuadXor1>(v));
    v = op(v, dpp_of<kQuadXor2>(v));
    v = op(v, dpp_of<kHalfMirror>(v));
    v = op(v, dpp_of<kMirror>(v));
    if constexpr (L >= 32) {
        v = swapped<false>(v, op);
    }
    if constexpr (L >= 64) {
        v = swapped<true>(v, op);
    }
    if constexpr (L == 256) {
        V *const of = reinterpret_cast<V *>(box);
        __syncthreads();   // the readers of the last reduction are done with the box
        if ((threadIdx.x & 63) == 0) {
            of[threadIdx.x >> 6] = v;
        }
        __syncthreads();
        v = op(op(of[0], of[1]), op(of[2], of[3]));
    }
    return v;
}
template <int L, typename V>
__device__ __forceinline__ V row_sum(V v, double *box)
{
    return row_reduce<L>(v, box, [](V a, V b) { return a + b; });
}
template <int L>
__device__ __forceinline__ uint32_t row_max(uint32_t v, double *box)
{
    return row_reduce<L>(v, box, umax);
}

struct RowParams {
    const void *x, *residual, *weight;
    int64_t ld_x, ld_residual, ld_sum, n, row0;   // row0: the first row of this launch
    int d, blocks;
    float eps, fixed_scale;
    double inv_d;
    void *sum;
    uint8_t *codes;
    void *scales;
    float *sqr_sum;
    int format;
    bool whole_x, whole_residual, whole_weight, whole_sum;   // rows start on 16 bytes: eight elements in wide loads
    bool past;                                               // sums pass the caches by (PAST)
};

// What eight elements become, and their share of the squared norm of what the codes stand for.  `biased`: the block's scale.
__device__ __forceinline__ float encode_fp4(const float (&y)[kVec], uint32_t biased, bool want_sqr, uint32_t &code)
{
    const float scale = biased ? __uint_as_float(biased << 23) : __uint_as_float(0x400000u);
    code = 0;
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, y[0], y[1], scale, 0);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, y[2], y[3], scale, 1);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, y[4], y[5], scale, 2);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, y[6], y[7], scale, 3);
    float ss = 0.f;
    if (want_sqr) {
        const f2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, scale, 0),
                         __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, scale, 1),
                         __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, scale, 2),
                         __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, scale, 3)};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            ss = fmaf(v[i].x, v[i].x, ss);
            ss = fmaf(v[i].y, v[i].y, ss);
        }
    }
    return ss;
}

__device__ __forceinline__ float encode_fp8(const float (&y)[kVec], uint32_t biased, bool want_sqr, uint32_t (&code)[2])
{
    const float scale = biased ? __uint_as_float(biased << 23) : __uint_as_float(0x400000u);
    const float top = 448.f * scale;   // the instruction makes a NaN of what lies beyond the largest number
    float ss = 0.f;
#pragma unroll
    for (int w = 0; w < 2; w++) {
        s2 c = {0, 0};
        c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, __builtin_amdgcn_fmed3f(y[4 * w], -top, top),
                                                     __builtin_amdgcn_fmed3f(y[4 * w + 1], -top, top), scale, false);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, __builtin_amdgcn_fmed3f(y[4 * w + 2], -top, top),
                                                     __builtin_amdgcn_fmed3f(y[4 * w + 3], -top, top), scale, true);
        code[w] = __builtin_bit_cast(uint32_t, c);
        if (want_sqr) {
            const f2 lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(code[w], scale, false);
            const f2 hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(code[w], scale, true);
            ss = fmaf(lo.x, lo.x, ss);
            ss = fmaf(lo.y, lo.y, ss);
            ss = fmaf(hi.x, hi.x, ss);
            ss = fmaf(hi.y, hi.y, ss);
        }
    }
    return ss;
}

// v + rest toward zero, its last bit set if anything was lost: rounding that once more, to a number of a few bits, gives what
// rounding the sum itself would, also next to a halfway point and to a power of two (4096 x 768 to 8 bits: one to four codes
// fall to the wrong side if a sum is rounded to nearest first).
__device__ __forceinline__ float round_to_odd(float v, float rest)
{
    const float sum = v + rest, lost = rest - (sum - v);
    const uint32_t bits = __float_as_uint(sum);
    return lost == 0.f ? sum : __uint_as_float((bits - ((__float_as_uint(lost) ^ bits) >> 31)) | 1u);
}

// One row per L lanes (16, 32, 64 or the workgroup's 256), held in registers: C times eight elements per lane, so that a
// row is read once whatever is computed from it: its largest values, its sum of squares, and with a residual its sum, which is
// written in between.  Bound by memory: 1.2M x 200 from fp32 to 4 bits 207 us, 5.5 TB/s; the norm of 131072 x 4096 bfloat16 with
// a residual to int8 620 us, 6.1 TB/s, with the vector units busy for three quarters of it; one row by the latency of its load and
// its sums, 4 to 5 us from call to call.  The longest rows take a bound on registers (norm of 30000 x 16384: one workgroup per
// CU 835 us, two 628).
template <typename T, int L, int C, bool NORM, bool PAST>
__global__ __launch_bounds__(kThreads, C >= 8 ? 2 : C >= 4 ? 4 : 1) void row_quantise_kernel(RowParams p)
{
    __shared__ double box[4];
    const int lane = threadIdx.x % L;
    const int64_t row = p.row0 + (int64_t)blockIdx.x * (kThreads / L) + threadIdx.x / L;
    if (L < 256 && row >= p.n) {
        return;   // whole groups of lanes that share no data with others (with L = 256 the grid is the number of rows)
    }
    // Up to 16 elements of a lane: the row, its residual and the weight are all on their way before the first is needed (1.2M x
    // 200 with a residual 357 -> 342 us); with more they would take the registers of other wavefronts.
    constexpr bool kTogether = NORM && C <= 2;
    auto part = [&](const T *row_of, int c, bool whole) {
        const int at = (c * L + lane) * kVec;
        const int count = min(kVec, max(0, p.d - at));
        return load8<kTogether>(row_of + (count ? at : 0), count, whole);
    };
    const T *const w = NORM ? static_cast<const T *>(p.weight) : nullptr;
    float y[C][kVec];
    Raw8<T> xv[kTogether ? C : 1], wv[kTogether ? C : 1], rv[kTogether ? C : 1];
    const T *x = static_cast<const T *>(p.x) + row * p.ld_x;
    const T *r = static_cast<const T *>(p.residual) + row * p.ld_residual;
    if constexpr (kTogether) {
#pragma unroll
        for (int c = 0; c < C; c++) {
            xv[c] = part(x, c, p.whole_x);
        }
        if (p.residual) {
#pragma unroll
            for (int c = 0; c < C; c++) {
                rv[c] = part(r, c, p.whole_residual);
            }
        }
        if (w) {
#pragma unroll
            for (int c = 0; c < C; c++) {
                wv[c] = part(w, c, p.whole_weight);
            }
        }
    }
#pragma unroll
    for (int c = 0; c < C; c++) {
        (kTogether ? xv[kTogether ? c : 0] : part(x, c, p.whole_x)).values(y[c]);
    }
    if constexpr (NORM) {
        if (p.residual) {
#pragma unroll
            for (int c = 0; c < C; c++) {
                float v[kVec];
                (kTogether ? rv[kTogether ? c : 0] : part(r, c, p.whole_residual)).values(v);
#pragma unroll
                for (int i = 0; i < kVec; i++) {
                    y[c][i] += v[i];
                }
            }
        }
        if (p.sum) {
            // the one rounding of the sum to the rows' type; the norm goes on with the unrounded sum
            T *o = static_cast<T *>(p.sum) + row * p.ld_sum;
#pragma unroll
            for (int c = 0; c < C; c++) {
                const int at = (c * L + lane) * kVec;
                const int count = min(kVec, max(0, p.d - at));
                store8<PAST>(o + (count ? at : 0), count, p.whole_sum, y[c]);
            }
        }
        // Eight squares are added in 32 bits, all else up to the root's reciprocal in 64.  Before microscaled codes that and the
        // products with it and the weight are held in two parts of 32 and rounded once: codes are as far apart as 2^-3 of a value,
        // and every rounding before them moves some to a neighbour.  int8 codes come of two more products in 32 bits by their
        // definition, and here of two before these, with a root rounded to 32 bits (in two parts 500000 x 384 takes 288 us
        // instead of 256, 131072 x 4096 642 instead of 623).
        auto sum_of_squares = [&]() {
            double sum = 0.0;
#pragma unroll
            for (int c = 0; c < C; c++) {
                float ss = 0.f;
#pragma unroll
                for (int i = 0; i < kVec; i++) {
                    ss = fmaf(y[c][i], y[c][i], ss);
                }
                sum += (double)ss;
            }
            return row_sum<L>(sum, box);
        };
        double mean = sum_of_squares() * p.inv_d + p.eps;
        // Finite elements whose squares pass the largest number of 32 bits, or lose bits below the smallest that count next to eps:
        // once more with elements 2^-80 or 2^80 times as large.  (Two branches: with the factor chosen ahead of one, rows that need
        // neither took 5 % longer, 1.2M x 200 with a residual to 4 bits 361 us instead of 345.)
        auto again = [&](float unit) {
#pragma unroll
            for (int c = 0; c < C; c++) {
#pragma unroll
                for (int i = 0; i < kVec; i++) {
                    y[c][i] *= unit;
                }
            }
            mean = sum_of_squares() * p.inv_d + (double)p.eps * unit * unit;
        };
        if (mean == __builtin_inf()) {
            again(0x1p-80f);
        } else if (mean < 0x1p-100) {
            again(0x1p80f);
        }
        double root = __builtin_amdgcn_rsq(mean);   // half of a double's bits at least, and a step of Newton's for the rest
        root = mean == __builtin_inf() ? 0.0 : root * fma(-0.5 * mean * root, root, 1.5);
        const float high = (float)root, low = (float)(root - (double)high);
        auto multiply = [&](auto in_parts) {
#pragma unroll
            for (int c = 0; c < C; c++) {
                float f[kVec];
                if (w) {
                    (kTogether ? wv[kTogether ? c : 0] : part(w, c, p.whole_weight)).values(f);
                }
#pragma unroll
                for (int i = 0; i < kVec; i++) {
                    float v = y[c][i] * high;
                    if constexpr (decltype(in_parts)::value) {
                        float rest = fmaf(y[c][i], low, fmaf(y[c][i], high, -v));
                        if (w) {
                            const float t = v * f[i];
                            rest = fmaf(rest, f[i], fmaf(v, f[i], -t));
                            v = t;
                        }
                        y[c][i] = round_to_odd(v, rest);
                    } else {
                        y[c][i] = w ? v * f[i] : v;
                    }
                }
            }
        };
        if (p.format == kFormatInt8) {
            multiply(std::false_type());
        } else {
            multiply(std::true_type());
        }
    }
    const bool want_sqr = p.sqr_sum != nullptr;
    float ss = 0.f;
    if (p.format == kFormatInt8) {
        float scale = p.fixed_scale, inv;
        bool bad = false;
        if (scale > 0.f) {
            inv = 1.0f / scale;
        } else {
            uint32_t top = 0;
#pragma unroll
            for (int c = 0; c < C; c++) {
#pragma unroll
                for (int i = 0; i < kVec; i++) {
                    top = umax(top, __float_as_uint(y[c][i]) & 0x7fffffffu);
                }
            }
            top = row_max<L>(top, box);
            bad = top >= kInfBits;
            float t = __uint_as_float(top);
            scale = bad ? __builtin_nanf("") : t / 127.0f;
            if (t < 0x1p-90f) {   // 127 / t would not be finite
                t *= 0x1p64f;
#pragma unroll
                for (int c = 0; c < C; c++) {
#pragma unroll
                    for (int i = 0; i < kVec; i++) {
                        y[c][i] *= 0x1p64f;
                    }
                }
            }
            inv = t > 0.f && !bad ? 127.0f / t : 0.f;
        }
        int sq = 0;
        uint8_t *o = p.codes + row * p.d;
        auto encode = [&](auto fixed) {
#pragma unroll
            for (int c = 0; c < C; c++) {
                const int at = (c * L + lane) * kVec;
                const int count = min(kVec, max(0, p.d - at));
                uint32_t q[kVec], w[2];
#pragma unroll
                for (int i = 0; i < kVec; i++) {
                    float v = y[c][i] * inv;
                    if constexpr (decltype(fixed)::value) {
                        v = v != v ? 0.f : __builtin_amdgcn_fmed3f(v, -127.f, 127.f);
                    }
                    q[i] = __float_as_uint(v + 0x1.8p23f);   // rounded to an integer, halfway to even: the lowest byte is the code
                }
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    w[k] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(q[4 * k + 3], q[4 * k + 2], 0x0c0c0400u),
                                                 __builtin_amdgcn_perm(q[4 * k + 1], q[4 * k], 0x0c0c0400u), 0x05040100u);
                    w[k] = bad ? 0u : w[k];
                    sq = __builtin_amdgcn_sdot4((int)w[k], (int)w[k], sq, false);
                }
                if (count == kVec && (p.d & 7) == 0) {
                    *reinterpret_cast<uint2 *>(o + at) = make_uint2(w[0], w[1]);
                } else {
#pragma unroll
                    for (int i = 0; i < kVec; i++) {
                        if (i < count) {
                            o[at + i] = (uint8_t)(w[i / 4] >> (8 * (i % 4)));
                        }
                    }
                }
            }
        };
        if (p.fixed_scale > 0.f) {
            encode(std::true_type());
        } else {
            encode(std::false_type());
        }
        if (lane == 0 && p.scales) {
            static_cast<float *>(p.scales)[row] = scale;
        }
        if (want_sqr) {
            ss = row_sum<L>((float)sq, box) * scale * scale;   // a lane's sum is at most C * 8 * 127^2: exact in 24 bits
        }
    } else {
        const bool four = p.format == kFormatMxFp4;
#pragma unroll
        for (int c = 0; c < C; c++) {
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < kVec; i++) {
                top = umax(top, __float_as_uint(y[c][i]) & 0x7fffffffu);
            }
            top = quad_max(top);
            const bool bad = top >= kInfBits;
            const int e = (int)(top >> 23) - (four ? 2 : 8);
            const uint32_t biased = (uint32_t)max(e, 0);
            const int at = (c * L + lane) * kVec, block = at / kMxBlock;
            if (block >= p.blocks) {
                continue;   // four lanes at a time
            }
            const int64_t slot = row * p.blocks + block;
            float part;
            if (four) {
                uint32_t code;
                part = encode_fp4(y[c], biased, want_sqr, code);
                reinterpret_cast<uint32_t *>(p.codes)[slot * 4 + (lane & 3)] = bad ? 0u : code;
            } else {
                uint32_t code[2];
                part = encode_fp8(y[c], biased, want_sqr, code);
                reinterpret_cast<uint2 *>(p.codes)[slot * 4 + (lane & 3)] = bad ? make_uint2(0, 0) : make_uint2(code[0], code[1]);
            }
            ss += bad ? __builtin_nanf("") : part;
            if ((lane & 3) == 0) {
                static_cast<uint8_t *>(p.scales)[slot] = (uint8_t)(bad ? kNaNScale : biased);
            }
        }
        if (want_sqr) {
            ss = row_sum<L>(ss, box);
        }
    }
    if (want_sqr && lane == 0) {
        p.sqr_sum[row] = ss;
    }
}

// A launch has less than 2^32 threads: more rows than half a million workgroups take go in several.
template <typename Params, typename Launch>
void in_launches(Params p, int rows_per_group, Launch launch)
{
    constexpr int64_t kGroups = 1 << 19;
    for (p.row0 = 0; p.row0 < p.n; p.row0 += kGroups * rows_per_group) {
        launch(p, (unsigned)std::min(kGroups, (p.n - p.row0 + rows_per_group - 1) / rows_per_group));
        check_launch();
    }
}

template <typename T, int L, int C, bool NORM>
void launch_rows_of(const RowParams &p, hipStream_t s)
{
    in_launches(p, kThreads / L, [&](const RowParams &q, unsigned grid) {
        if (NORM && p.past) {
            hipLaunchKernelGGL((row_quantise_kernel<T, L, C, NORM, NORM>), dim3(grid), dim3(kThreads), 0, s, q);
        } else {
            hipLaunchKernelGGL((row_quantise_kernel<T, L, C, NORM, false>), dim3(grid), dim3(kThreads), 0, s, q);
        }
    });
}

// Few lanes with two to four times eight elements each: sums over lanes cost more than sums in a lane (norms with a residual to
// int8 of 1M x 128: 16 lanes 162 us, 32 lanes 289; of 1.2M x 200: 16 lanes 327, 32 lanes 360; of 500000 x 384: 32 lanes 254, 64
// lanes 297; of 150000 x 1536: 64 lanes 278, the workgroup 322), up to what a wavefront's registers keep in flight (131072 x
// 4096: 64 lanes with eight times eight elements 665 us, the workgroup with two times 618).
template <typename T, bool NORM>
void launch_rows(const RowParams &p, hipStream_t s)
{
    const int d = p.d;
    if (d <= 128) {
        launch_rows_of<T, 16, 1, NORM>(p, s);
    } else if (d <= 256) {
        launch_rows_of<T, 16, 2, NORM>(p, s);
    } else if (d <= 512) {
        launch_rows_of<T, 32, 2, NORM>(p, s);
    } else if (d <= 1024) {
        launch_rows_of<T, 64, 2, NORM>(p, s);
    } else if (d <= 2048) {
        launch_rows_of<T, 64, 4, NORM>(p, s);
    } else if (d <= 4096) {
        launch_rows_of<T, 256, 2, NORM>(p, s);
    } else if (d <= 8192) {
        launch_rows_of<T, 256, 4, NORM>(p, s);
    } else {
        launch_rows_of<T, 256, 8, NORM>(p, s);
    }
}

template <bool NORM>
void launch_rows(const RowParams &p, int type, hipStream_t s)
{
    if (type == kTypeF32) {
        launch_rows<float, NORM>(p, s);
    } else if (type == kTypeF16) {
        launch_rows<_Float16, NORM>(p, s);
    } else {
        launch_rows<__bf16, NORM>(p, s);
    }
}

size_t type_bytes(int type) { return type == kTypeF32 ? 4 : 2; }
bool aligned(const void *p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
// Float rows that the last cache (256 MB) could not hold for whoever reads them next pass it by, which leaves it to what is
// still to be read: the norm of 131072 x 4096 650 -> 624 us, and in turns with reading codes back the quantisation of
// 1.2M x 200 243 -> 220.  Of fp32 rows a lane stores two pieces of 16 bytes 32 apart, which leave gaps past the caches: whole
// pages do not mind (131072 x 4096 read back from int8 630 -> 580 us), other rows do (1.2M x 200 from 4 bits 244 -> 370; the norm
// with its fp32 sum 588 -> 612, of 131072 x 4096 1230 -> 1243).
bool pass_caches(int64_t n, int64_t ld, int type) { return (double)n * (double)ld * (double)type_bytes(type) > 0x1p27; }
// rows of eight elements at least that all start on 16 bytes
bool whole_rows(const void *p, int64_t ld, int type, int d)
{
    return d >= kVec && aligned(p, 16) && (ld * (int64_t)type_bytes(type)) % 16 == 0;
}

// No rows need no buffers: the address of an empty array is null.
void check_rows(const char *op, const void *p, int64_t ld, int type, int64_t n, int d)
{
    IXA_REQUIRE(p || n == 0, kErrInvalidParam, "operator buffers can not be nullptr.");
    IXA_REQUIRE(aligned(p, type_bytes(type)), kErrInvalidParam, "%s: rows are not aligned to their elements", op);
    IXA_REQUIRE(ld >= d && ld <= (int64_t)1 << 40, kErrInvalidParam, "%s: rows of %d elements in steps of %ld", op, d, (long)ld);
}

// Rows are worked on side by side, in no order: a sum written over a row of an input that another workgroup (or another
// wavefront of the same row) has still to read would change what that one reads.  Each row of the sum lies on its own input
// row as a whole, where it is written behind its reads, or on none; the latter with the same stride (two column ranges of
// one buffer) or outright.
bool sum_collides(const void *sum, int64_t ld_sum, const void *in, int64_t ld_in, int type, int64_t n, int d)
{
    const __int128 size = (__int128)type_bytes(type), a = (__int128)reinterpret_cast<uintptr_t>(sum),
                   b = (__int128)reinterpret_cast<uintptr_t>(in), row = size * d;
    if (a + ((n - 1) * size * ld_sum + row) <= b || b + ((n - 1) * size * ld_in + row) <= a) {
        return false;
    }
    if (n == 1 || ld_sum != ld_in) {
        return n > 1 || a != b;
    }
    const __int128 step = size * ld_in, apart = (a > b ? a - b : b - a) % step;
    return a != b && (apart < row || apart > step - row);
}

void check_codes(const char *op, int type, int64_t n, int d, int format, const uint8_t *codes, const void *scales, bool fixed)
{
    IXA_REQUIRE(type >= kTypeF32 && type <= kTypeBF16, kErrInvalidParam, "%s: unsupported element type %d", op, type);
    IXA_REQUIRE(format >= kFormatInt8 && format <= kFormatMxFp4, kErrInvalidParam, "%s: unsupported code format %d", op, format);
    IXA_REQUIRE(n >= 0 && n <= 0x7fffffff && d >= 1 && d <= kMaxCodeDim, kErrInvalidParam,
                "%s: rows %ld (< 2^31), dims %d (1 ... %d)", op, (long)n, d, kMaxCodeDim);
    IXA_REQUIRE((codes && (scales || fixed)) || n == 0, kErrInvalidParam, "operator buffers can not be nullptr.");
    IXA_REQUIRE(aligned(codes, 16) && (format != kFormatInt8 || aligned(scales, 4)), kErrInvalidParam,
                "%s: codes have to start on 16 bytes and fp32 scales on 4", op);
}

void check_fixed(const char *op, int format, float fixed_scale)
{
    IXA_REQUIRE(fixed_scale == 0.f || (format == kFormatInt8 && fixed_scale >= 1e-30f && fixed_scale <= 1e30f),
                kErrInvalidParam, "%s: a fixed scale (%g) goes with int8 codes and lies in [1e-30, 1e30]", op,
                (double)fixed_scale);
}

// ----- codes back into rows ---------------------------------------------------------------------------------------------

constexpr int kReadRows = 2;

struct ReadParams {
    const uint8_t *codes;
    const void *scales;
    int64_t n, ld, row0;           // row0: the first row of this launch
    int d, blocks, chunks, rows;   // chunks of 8 elements per row, rows that a workgroup reads at a time
    void *out;
    bool whole;
};

// The eight values of chunk c of a row.
template <int FORMAT>
__device__ __forceinline__ void read_chunk(const ReadParams &p, int64_t row, int c, float (&v)[kVec])
{
    const int at = c * kVec;
    if constexpr (FORMAT == kFormatInt8) {
        const float scale = static_cast<const float *>(p.scales)[row];
        const uint8_t *q = p.codes + row * p.d + at;
        if ((p.d & 7) == 0) {
            const uint2 w = *reinterpret_cast<const uint2 *>(q);
            const uint32_t u[2] = {w.x, w.y};
#pragma unroll
            for (int i = 0; i < kVec; i++) {
                v[i] = (float)(int8_t)(u[i / 4] >> (8 * (i % 4))) * scale;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kVec; i++) {
                v[i] = at + i < p.d ? (float)(int8_t)q[i] * scale : 0.f;
            }
        }
    } else {
        const int64_t slot = row * p.blocks + at / kMxBlock;
        const uint32_t biased = static_cast<const uint8_t *>(p.scales)[slot];
        const float scale = biased ? __uint_as_float(biased << 23) : __uint_as_float(0x400000u);
        if constexpr (FORMAT == kFormatMxFp8) {
            const uint2 w = reinterpret_cast<const uint2 *>(p.codes)[slot * 4 + (c & 3)];
            const uint32_t u[2] = {w.x, w.y};
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const f2 lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(u[i], scale, false);
                const f2 hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(u[i], scale, true);
                v[4 * i] = lo.x;
                v[4 * i + 1] = lo.y;
                v[4 * i + 2] = hi.x;
                v[4 * i + 3] = hi.y;
            }
        } else {
            const uint32_t u = reinterpret_cast<const uint32_t *>(p.codes)[slot * 4 + (c & 3)];
            const f2 t[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, scale, 0),
                             __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, scale, 1),
                             __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, scale, 2),
                             __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, scale, 3)};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                v[2 * i] = t[i].x;
                v[2 * i + 1] = t[i].y;
            }
        }
#pragma unroll
        for (int i = 0; i < kVec; i++) {
            v[i] = biased == kNaNScale ? __builtin_nanf("") : v[i];
        }
    }
}

// Eight elements per thread: a quarter of a block, 16 bytes of 16-bit values, which neighbours store next to each other (with
// sixteen, stores that pass the caches by cover every second 16 bytes: 238 us for 1.2M x 200 from 4 bits).  Two rows per thread
// share its place in the row and are in flight together: 104 us, 6.2 TB/s (four rows 107, eight 115; and 131072 x 4096
// from int8 267, 294 and 341 us, 6.0 TB/s with two).
template <typename T, int FORMAT, bool PAST>
__global__ __launch_bounds__(kThreads) void read_codes_kernel(ReadParams p)
{
    const int across = min(p.chunks, kThreads), in = threadIdx.x / across;
    if (in >= p.rows) {
        return;
    }
    const int64_t first = p.row0 + (int64_t)blockIdx.x * (p.rows * kReadRows) + in;
    for (int c = threadIdx.x - in * across; c < p.chunks; c += kThreads) {
        float v[kReadRows][kVec];
#pragma unroll
        for (int k = 0; k < kReadRows; k++) {
            read_chunk<FORMAT>(p, min(first + k * p.rows, p.n - 1), c, v[k]);
        }
#pragma unroll
        for (int k = 0; k < kReadRows; k++) {
            const int64_t row = first + k * p.rows;
            if (row < p.n) {
                store8<PAST>(static_cast<T *>(p.out) + row * p.ld + c * kVec, min(kVec, p.d - c * kVec), p.whole, v[k]);
            }
        }
    }
}

template <typename T, int FORMAT>
void launch_read(const ReadParams &p, bool past, hipStream_t s)
{
    in_launches(p, p.rows * kReadRows, [&](const ReadParams &q, unsigned grid) {
        if (past) {
            hipLaunchKernelGGL((read_codes_kernel<T, FORMAT, true>), dim3(grid), dim3(kThreads), 0, s, q);
        } else {
            hipLaunchKernelGGL((read_codes_kernel<T, FORMAT, false>), dim3(grid), dim3(kThreads), 0, s, q);
        }
    });
}

template <typename T>
void launch_read(const ReadParams &p, int format, bool past, hipStream_t s)
{
    if (format == kFormatInt8) {
        launch_read<T, kFormatInt8>(p, past, s);
    } else if (format == kFormatMxFp8) {
        launch_read<T, kFormatMxFp8>(p, past, s);
    } else {
        launch_read<T, kFormatMxFp4>(p, past, s);
    }
}

}  // namespace

void op_quantise(const void *x, int64_t ld, int type, int64_t n, int d, int format, float fixed_scale, uint8_t *codes,
                 void *scales, float *sqr_sum, hipStream_t s)
{
    check_codes("quantise", type, n, d, format, codes, scales, fixed_scale > 0.f);
    check_rows("quantise", x, ld, type, n, d);
    check_fixed("quantise", format, fixed_scale);
    IXA_REQUIRE(aligned(sqr_sum, 4), kErrInvalidParam, "quantise: squared norms are not aligned to their elements");
    if (n == 0) {
        return;
    }
    RowParams p{};
    p.x = x;
    p.ld_x = ld;
    p.n = n;
    p.d = d;
    p.blocks = mx_blocks(d);
    p.fixed_scale = fixed_scale;
    p.codes = codes;
    p.scales = scales;
    p.sqr_sum = sqr_sum;
    p.format = format;
    p.whole_x = whole_rows(x, ld, type, d);
    launch_rows<false>(p, type, s);
}

void op_rms_norm_quantise(const void *x, int64_t ld_x, const void *residual, int64_t ld_residual, const void *weight,
                          int type, int64_t n, int d, float eps, void *sum, int64_t ld_sum, int format, float fixed_scale,
                          uint8_t *codes, void *scales, float *sqr_sum, hipStream_t s)
{
    check_codes("rms_norm_quantise", type, n, d, format, codes, scales, fixed_scale > 0.f);
    check_rows("rms_norm_quantise", x, ld_x, type, n, d);
    if (residual) {
        check_rows("rms_norm_quantise", residual, ld_residual, type, n, d);
    }
    if (sum) {
        check_rows("rms_norm_quantise", sum, ld_sum, type, n, d);
        IXA_REQUIRE(n == 0 || (!sum_collides(sum, ld_sum, x, ld_x, type, n, d) &&
                               !(residual && sum_collides(sum, ld_sum, residual, ld_residual, type, n, d))),
                    kErrInvalidParam, "rms_norm_quantise: rows of the sum have to be an input's own rows (same address and "
                    "stride) or share no element with it");
    }
    if (weight) {
        check_rows("rms_norm_quantise", weight, d, type, 1, d);
    }
    check_fixed("rms_norm_quantise", format, fixed_scale);
    IXA_REQUIRE(eps > 0.f && eps < __builtin_inff(), kErrInvalidParam, "rms_norm_quantise: eps %g has to be positive",
                (double)eps);
    IXA_REQUIRE(aligned(sqr_sum, 4), kErrInvalidParam, "rms_norm_quantise: squared norms are not aligned to their elements");
    if (n == 0) {
        return;
    }
    RowParams p{};
    p.x = x;
    p.residual = residual;
    p.weight = weight;
    p.ld_x = ld_x;
    p.ld_residual = ld_residual;
    p.ld_sum = ld_sum;
    p.n = n;
    p.d = d;
    p.blocks = mx_blocks(d);
    p.eps = eps;
    p.inv_d = 1.0 / d;
    p.fixed_scale = fixed_scale;
    p.sum = sum;
    p.codes = codes;
    p.scales = scales;
    p.sqr_sum = sqr_sum;
    p.format = format;
    p.whole_x = whole_rows(x, ld_x, type, d);
    p.whole_residual = whole_rows(residual, ld_residual, type, d);
    p.whole_weight = whole_rows(weight, 0, type, d);
    p.whole_sum = whole_rows(sum, ld_sum, type, d);
    p.past = sum && pass_caches(n, ld_sum, type);
    launch_rows<true>(p, type, s);
}

void op_dequantise(const uint8_t *codes, const void *scales, int format, int64_t n, int d, int type, void *out, int64_t ld,
                   hipStream_t s)
{
    check_codes("dequantise", type, n, d, format, codes, scales, false);
    check_rows("dequantise", out, ld, type, n, d);
    if (n == 0) {
        return;
    }
    ReadParams p{};
    p.codes = codes;
    p.scales = scales;
    p.n = n;
    p.ld = ld;
    p.d = d;
    p.blocks = mx_blocks(d);
    p.chunks = (d + kVec - 1) / kVec;
    p.rows = p.chunks >= kThreads ? 1 : kThreads / p.chunks;
    p.out = out;
    p.whole = whole_rows(out, ld, type, d);
    const bool past = pass_caches(n, ld, type);
    if (type == kTypeF32) {
        launch_read<float>(p, format, past, s);
    } else if (type == kTypeF16) {
        launch_read<_Float16>(p, format, past, s);
    } else {
        launch_read<__bf16>(p, format, past, s);
    }
}

}  // namespace ixa
