// Eight elements of a row at a time, at any alignment, and exchanges between neighbouring lanes.
#pragma once
#include "lowp.h"

#include <algorithm>

namespace ixa {

constexpr int kEight = 8;

// Eight elements as they lie in memory.  Global memory takes wide loads and stores at any address: one instruction for 16-bit
// elements and two for fp32, also where a row starts on an element only.
template <typename T>
struct Eight {
    typedef T Lane __attribute__((ext_vector_type(kEight)));
    typedef T Anywhere __attribute__((ext_vector_type(kEight), aligned(sizeof(T))));
    Lane v;
    // `count` elements, `fill` behind them
    __device__ __forceinline__ void load(const T *__restrict__ p, int count, T fill)
    {
        if (count >= kEight) {
            v = *reinterpret_cast<const Anywhere *>(p);
        } else {
#pragma unroll
            for (int i = 0; i < kEight; i++) {
                v[i] = i < count ? p[i] : fill;
            }
        }
    }
    // PAST: past the caches
    template <bool PAST = false>
    __device__ __forceinline__ void store(T *__restrict__ p, int count) const
    {
        if (count >= kEight) {
            if constexpr (PAST) {
                __builtin_nontemporal_store(v, reinterpret_cast<Anywhere *>(p));
            } else {
                *reinterpret_cast<Anywhere *>(p) = v;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kEight; i++) {
                if (i < count) {
                    p[i] = v[i];
                }
            }
        }
    }
};

// the value of the lane that CTRL names, within 16 lanes
template <int CTRL>
__device__ __forceinline__ int lane_of(int v)
{
    return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, true);
}
constexpr int kXor1 = 0xb1, kXor2 = 0x4e, kMirror8 = 0x141, kMirror16 = 0x140;

// Op over groups of LANES (4, 8 or 16) lanes; every one of them has the result.
template <int LANES, typename Op>
__device__ __forceinline__ int over_lanes(int v, Op op)
{
    v = op(v, lane_of<kXor1>(v));
    v = op(v, lane_of<kXor2>(v));
    if constexpr (LANES >= 8) {
        v = op(v, lane_of<kMirror8>(v));
    }
    if constexpr (LANES >= 16) {
        v = op(v, lane_of<kMirror16>(v));
    }
    return v;
}

// Op over the 64 lanes of a wavefront, 32 or 64 bits; every lane has the result.
template <int CTRL, typename V>
__device__ __forceinline__ V value_of_lane(V v)
{
    if constexpr (sizeof(V) == 4) {
        return __builtin_bit_cast(V, lane_of<CTRL>(__builtin_bit_cast(int, v)));
    } else {
        const int2 w = __builtin_bit_cast(int2, v);
        return __builtin_bit_cast(V, make_int2(lane_of<CTRL>(w.x), lane_of<CTRL>(w.y)));
    }
}
template <typename V, typename Op>
__device__ __forceinline__ V over_wave(V v, Op op)
{
    v = op(v, value_of_lane<kXor1>(v));
    v = op(v, value_of_lane<kXor2>(v));
    v = op(v, value_of_lane<kMirror8>(v));
    v = op(v, value_of_lane<kMirror16>(v));
    struct Box {
        uint32_t w[sizeof(V) / 4];
    };
    Box a = __builtin_bit_cast(Box, v), b;
#pragma unroll
    for (size_t i = 0; i < sizeof(V) / 4; i++) {
        const auto t = __builtin_amdgcn_permlane16_swap(a.w[i], a.w[i], false, false);
        a.w[i] = t[0];
        b.w[i] = t[1];
    }
    v = op(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b));
    a = __builtin_bit_cast(Box, v);
#pragma unroll
    for (size_t i = 0; i < sizeof(V) / 4; i++) {
        const auto t = __builtin_amdgcn_permlane32_swap(a.w[i], a.w[i], false, false);
        a.w[i] = t[0];
        b.w[i] = t[1];
    }
    return op(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b));
}

// ----- host -------------------------------------------------------------------------------------------------------------

inline size_t element_bytes(int type) { return type == kTypeF32 ? 4 : 2; }
inline bool on_bytes(const void *p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

inline void check_type(const char *op, int type)
{
    IXA_REQUIRE(type >= kTypeF32 && type <= kTypeBF16, kErrInvalidParam, "%s: unsupported element type %d", op, type);
}
// Rows of an operator: no rows need no buffer.
inline void check_row_buffer(const char *op, const void *p, int64_t ld, int type, int64_t n, int64_t d)
{
    IXA_REQUIRE(p || n == 0 || d == 0, kErrInvalidParam, "operator buffers can not be nullptr.");
    IXA_REQUIRE(on_bytes(p, element_bytes(type)), kErrInvalidParam, "%s: rows are not aligned to their elements", op);
    IXA_REQUIRE(ld >= d && ld <= (int64_t)1 << 40, kErrInvalidParam, "%s: rows of %ld elements in steps of %ld", op, (long)d,
                (long)ld);
}

// Whether rows of a result lie on rows of an input that others have still to read: each row has to be its own input row as a
// whole, or to share no element with any (two column ranges of one buffer, or apart outright).
inline bool rows_collide(const void *out, int64_t ld_out, const void *in, int64_t ld_in, int type, int64_t n, int64_t d)
{
    const __int128 size = (__int128)element_bytes(type), a = (__int128)reinterpret_cast<uintptr_t>(out),
                   b = (__int128)reinterpret_cast<uintptr_t>(in), row = size * d;
    if (a + ((n - 1) * size * ld_out + row) <= b || b + ((n - 1) * size * ld_in + row) <= a) {
        return false;
    }
    if (n == 1 || ld_out != ld_in) {
        return n > 1 || a != b;
    }
    const __int128 step = size * ld_in, apart = (a > b ? a - b : b - a) % step;
    return a != b && (apart < row || apart > step - row);
}

// A kernel for each element type.
template <typename F>
void with_type(int type, F f)
{
    if (type == kTypeF32) {
        f(float());
    } else if (type == kTypeF16) {
        f((_Float16)0.f);
    } else {
        f((__bf16)0.f);
    }
}

}  // namespace ixa
