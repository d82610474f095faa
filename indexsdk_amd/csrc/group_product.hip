// Float rows x against rows of 4-bit codes with a scale, and where there is one a zero point, per group of 32, 64 or 128 elements:
//   out[i][j] = alpha * sum over groups g of scale[j][g] * (sum over k in g of x[i][k] (code[j][k] - zero[j][g])) + bias[j]
//
// The differences are small integers, which fp16 holds exactly; v_mfma_f32_16x16x32_f16 adds a group's products in fp32, one
// multiply-add per group applies its scale.  fp16 rows go in as they are.  bfloat16 and fp32 rows are multiplied by the power
// of two that brings their largest finite element to 2^14 ... 2^15, and become one fp16 number each (bfloat16: exact but for
// what lies 2^-39 below that element) or two (fp32: to 2^-22 of an element or 2^-39 of the largest); the power is taken back in fp32.
//
// Eight codes of a register become fp16 in nine instructions: under an exponent of 2^10 the low bits of a half are the
// integer 1024 + code, under 2^6 bits 4 ... 7 are 64 + code; a packed addition takes 1024 + zero or 64 + zero away, without
// rounding.  The pairs come as elements (0, 4), (1, 5), (2, 6), (3, 7): x is stored in that order.
//
// A lane of the instruction (column r = l & 15, quarter q = l >> 4) wants codes 8 q ... 8 q + 7 of each 32 of its row and loads
// codes 32 q ... 32 q + 31 of each 128: four registers that two swaps of 32 and two of 16 lanes transpose.
//
// What bounds it: for few rows the codes, which are read once (one bfloat16 row against 1,000,000 x 768 in groups of 64 with zero
// points: 88 us, 4.9 TB/s; 64 rows against 1,000,000 x 200: 133 us, two thirds of them stores); for many the vector
// instructions that make integers of codes, which share a SIMD's issue with the products (2048 x 131,072 x 768 bfloat16 in groups of 128 to
// bfloat16: 615 us, 0.67 PFLOP/s, the vector unit busy for 57 % and the matrix cores for 28 % of the cycles; in groups of 32 with
// four times as many multiply-adds to fp32 818 us; fp32 rows, two pieces, 1442 us).
#include "row_access.h"

#include <algorithm>
#include <type_traits>

namespace ixa {

namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int kStep = 128;         // columns of a step: 64 bytes of codes
constexpr int kLoaded = 0x0f70;    // s_waitcnt: all loads are there, also those into LDS
// Pieces of this size, the powers of two and what four wavefronts hold of scales and zero points (groups of 32): two workgroups share a CU's.
constexpr size_t kHalfLds = 80 * 1024 - 256 - 4 * 64 * 4 * 8;

struct GroupProductParams {
    const void *x;
    const uint8_t *codes, *zeros;
    const void *scales;
    const float *bias;
    void *out;
    const uint8_t *pieces;       // rows of fp16 pieces [m][pieces][steps * 128], and their exponents [m]
    const int *exponents;
    int64_t m, n, ld_x, ld, scale_count;
    int type, scale_type, out_type, d, groups, row_bytes, steps;
    bool has_zeros;
    float alpha;
};

// eight elements of a row as fp32, zeros behind the last
__device__ __forceinline__ void load_eight(const void *row, int type, int at, int d, float (&v)[kEight])
{
    const int count = min(kEight, max(0, d - at));
    at = count ? at : 0;
    if (type == kTypeF32) {
        Eight<float> e;
        e.load(static_cast<const float *>(row) + at, count, 0.f);
#pragma unroll
        for (int i = 0; i < kEight; i++) {
            v[i] = e.v[i];
        }
    } else if (type == kTypeF16) {
        Eight<_Float16> e;
        e.load(static_cast<const _Float16 *>(row) + at, count, (_Float16)0.f);
#pragma unroll
        for (int i = 0; i < kEight; i++) {
            v[i] = (float)e.v[i];
        }
    } else {
        Eight<__bf16> e;
        e.load(static_cast<const __bf16 *>(row) + at, count, (__bf16)0.f);
#pragma unroll
        for (int i = 0; i < kEight; i++) {
            v[i] = (float)e.v[i];
        }
    }
}

// bits of the largest finite magnitude
__device__ __forceinline__ int finite_top(const float (&v)[kEight])
{
    int top = 0;
#pragma unroll
    for (int i = 0; i < kEight; i++) {
        const int b = __float_as_int(v[i]) & 0x7fffffff;
        top = max(top, b < 0x7f800000 ? b : 0);
    }
    return top;
}
// the power of two that brings a magnitude to 2^14 ... 2^15
__device__ __forceinline__ int power_for(int top)
{
    return top == 0 ? 0 : 15 - __builtin_amdgcn_frexp_expf(__int_as_float(top));
}

// fp16 pieces of eight elements, in the order in which codes come out of a register
template <int P>
__device__ __forceinline__ void split_eight(const float (&v)[kEight], int power, h8 (&piece)[P])
{
#pragma unroll
    for (int i = 0; i < kEight; i++) {
        constexpr int kPlace[kEight] = {0, 2, 4, 6, 1, 3, 5, 7};
        const float y = ldexpf(v[i], power);
        const _Float16 high = (_Float16)y;
        piece[0][kPlace[i]] = high;
        if constexpr (P == 2) {
            const float rest = y - (float)high;
            piece[1][kPlace[i]] = (_Float16)(fabsf(y) <= 0x1p15f ? rest : 0.f);   // not of an infinity or a NaN
        }
    }
}

__device__ __forceinline__ h2 minus_zero_point(float zero) { return h2{(_Float16)(-1024.f - zero), (_Float16)(-1024.f - zero)}; }

// (0, 4), (1, 5), (2, 6), (3, 7) of eight codes, less their zero point
__device__ __forceinline__ h8 integers(uint32_t w, h2 minus)
{
    const h2 minus_64 = minus + h2{(_Float16)960.f, (_Float16)960.f};
    const uint32_t up = w >> 8;
    const h2 a = __builtin_bit_cast(h2, (w & 0x000f000fu) | 0x64006400u) + minus;
    const h2 b = __builtin_bit_cast(h2, (w & 0x00f000f0u) | 0x54005400u) + minus_64;
    const h2 c = __builtin_bit_cast(h2, (up & 0x000f000fu) | 0x64006400u) + minus;
    const h2 e = __builtin_bit_cast(h2, (up & 0x00f000f0u) | 0x54005400u) + minus_64;
    return h8{a.x, a.y, b.x, b.y, c.x, c.y, e.x, e.y};
}

// 64 lanes' four registers: quarter q's register i becomes quarter i's register q
__device__ __forceinline__ u4 transpose(u4 d)
{
    const auto a = __builtin_amdgcn_permlane32_swap(d.x, d.z, false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(d.y, d.w, false, false);
    const auto lo = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    const auto hi = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    return u4{lo[0], lo[1], hi[0], hi[1]};
}

// The scales (WIDE: fp32) and zero points of SG groups from `g` on of one row, in two parts so that nothing waits for the load, which
// ends with the array at the latest (the array has SG scales at least).  No branch is around a load: behind one the compiler
// waits for it, and with it for all that is in flight.
template <int SG, bool WIDE>
struct GroupScales {
    static_assert(SG == 1 || SG == 2 || SG == 4, "");
    typedef std::conditional_t<WIDE, uint32_t, uint16_t> Raw;
    Raw raw[SG];
    uint32_t zero_raw;
    int over;               // scales of the run that lie before `g`
    __device__ __forceinline__ void load(const GroupProductParams &p, int64_t row, int g)
    {
        const int64_t at = row * p.groups + g, from = min(at, p.scale_count - SG);
        over = (int)(at - from);
        __builtin_memcpy(raw, static_cast<const Raw *>(p.scales) + from, sizeof(raw));
        zero_raw = 0;
        __builtin_memcpy(&zero_raw, p.zeros + from, SG);      // any bytes where there are no zero points
    }
    // groups behind the row's last one get scale 0: x has zeros there
    __device__ __forceinline__ void take(const GroupProductParams &p, int g, bool there, float (&scale)[SG], h2 (&minus)[SG])
    {
        uint32_t of[SG];
        if constexpr (SG == 1) {
            of[0] = raw[0];
        } else if constexpr (!WIDE) {
            typedef std::conditional_t<SG == 2, uint32_t, uint64_t> All;
            const All all = __builtin_bit_cast(All, raw) >> (16 * over);
#pragma unroll
            for (int t = 0; t < SG; t++) {
                of[t] = (uint32_t)(all >> (16 * t)) & 0xffffu;
            }
        } else if constexpr (SG == 2) {
            of[0] = over ? raw[1] : raw[0];
            of[1] = raw[1];
        } else {
            const uint32_t a = over & 2 ? raw[2] : raw[0], b = over & 2 ? raw[3] : raw[1];
            of[0] = over & 1 ? b : a;
            of[1] = over & 1 ? raw[2] : b;
            of[2] = over & 1 ? raw[3] : raw[2];
            of[3] = raw[3];
        }
        const uint32_t zero = p.has_zeros ? zero_raw >> (8 * over) : 0x08080808u;
        const bool half = p.scale_type == kTypeF16;
#pragma unroll
        for (int t = 0; t < SG; t++) {
            float s = __uint_as_float(WIDE ? of[t] : of[t] << 16);
            if constexpr (!WIDE) {
                s = half ? (float)__builtin_bit_cast(_Float16, (uint16_t)of[t]) : s;
            }
            scale[t] = there && g + t < p.groups ? s : 0.f;
            minus[t] = minus_zero_point((float)(zero >> (8 * t) & 255u));
        }
    }
};

// One lane's sums of a row become scores of columns col ... col + N - 1.
template <int N>
__device__ __forceinline__ void store_scores(const GroupProductParams &p, int64_t row, int power, int64_t col, const float (&sum)[N],
                                             const float (&bias)[N])
{
    if (row >= p.m || col >= p.n) {
        return;
    }
    float v[N];
#pragma unroll
    for (int j = 0; j < N; j++) {
        v[j] = fmaf(p.alpha, ldexpf(sum[j], -power), bias[j]);
    }
    const int64_t at = row * p.ld + col;
    const auto write = [&](auto *out) {
        typedef std::remove_pointer_t<decltype(out)> T;
        typedef T Scores __attribute__((ext_vector_type(N), aligned(sizeof(T))));
        Scores s;
#pragma unroll
        for (int j = 0; j < N; j++) {
            s[j] = (T)v[j];
        }
        if (col + N <= p.n) {
            // past the caches, which keep what is read again: 2048 x 131072 scores 733 -> 635 us, 64 x 1M 163 -> 132, few ones as fast
            __builtin_nontemporal_store(s, reinterpret_cast<Scores *>(out + at));
        } else {
#pragma unroll
            for (int j = 0; j < N; j++) {
                if (col + j < p.n) {
                    out[at + j] = s[j];
                }
            }
        }
    };
    if (p.out_type == kTypeF32) {
        write(static_cast<float *>(p.out));
    } else if (p.out_type == kTypeF16) {
        write(static_cast<_Float16 *>(p.out));
    } else {
        write(static_cast<__bf16 *>(p.out));
    }
}

template <int N>
__device__ __forceinline__ void load_bias(const GroupProductParams &p, int64_t col, float (&bias)[N])
{
#pragma unroll
    for (int j = 0; j < N; j++) {
        bias[j] = p.bias && col + j < p.n ? p.bias[col + j] : 0.f;
    }
}

// A fragment's 32 columns of up to 64 rows in LDS: 64 bytes per row, piece q of row r at place q ^ ((r >> 1) & 3).
__device__ __forceinline__ int piece_place(int r, int q) { return r * 64 + ((q ^ ((r >> 1) & 3)) * 16); }

// Few rows of x (MF fragments of 16): their fp16 pieces stay in LDS, while the wavefronts stream NF fragments of coded rows past
// them, U steps of 128 columns ahead.  KS wavefronts of the workgroup share a tile, a part of its steps each, where there are few
// tiles.  Row j of 16 is row 4 (j & 3) + (j >> 2) of its fragment, so that RI = 1, 2 or 4 registers of a lane's four hold all
// rows of up to 4, 8 or 16.
template <int P, int MF, int RI, int NF, int U, int KS, int SG, bool WIDE, int W>
__global__ __launch_bounds__(W * 64) void group_stream_kernel(GroupProductParams p, int64_t tiles)
{
    static_assert(NF * U == 4 && (MF == 1 || RI == 4), "a lane brings the scales of one row and step");
    extern __shared__ __align__(16) uint8_t smem[];
    const int rows = (int)p.m, block_bytes = rows * 64;       // of 32 columns of one piece
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int *const power = reinterpret_cast<int *>(smem + (size_t)p.steps * 4 * P * block_bytes);
    constexpr int kTurn = 64 * SG * 8;                       // scales and zero points of NF * 16 rows and U steps
    constexpr int kShare = KS > 1 ? MF * NF * RI * 256 : 0;   // a wavefront's sums, for the one that adds them up
    uint8_t *const turn = reinterpret_cast<uint8_t *>(power + 64) + wave * std::max(kTurn, kShare);
    // all threads, a half, a quarter ... of them bring a row
    constexpr int kLog = W == 4 ? 8 : 9;
    const int lg = rows > 1 ? kLog - (32 - __builtin_clz(rows - 1)) : kLog, per_row = 1 << lg;
    const int my_row = tid >> lg, e = tid & (per_row - 1);
    const size_t x_bytes = (size_t)(p.type == kTypeF32 ? 4 : 2) * (size_t)p.ld_x;
    const uint8_t *const x_row = static_cast<const uint8_t *>(p.x) + (size_t)min(my_row, rows - 1) * x_bytes;
    if (tid < 64) {
        power[tid] = 0;
    }
    __syncthreads();
    if (p.type != kTypeF16) {
        int top = 0;
        if (my_row < rows) {
            for (int c = e; c * kEight < p.d; c += per_row) {
                float v[kEight];
                load_eight(x_row, p.type, c * kEight, p.d, v);
                top = max(top, finite_top(v));
            }
            atomicMax(&power[my_row], top);
        }
        __syncthreads();
        top = tid < 64 ? power[tid] : 0;
        __syncthreads();
        if (tid < 64) {
            power[tid] = power_for(top);
        }
        __syncthreads();
    }
    if (my_row < rows) {
        for (int c = e; c < p.steps * (kStep / kEight); c += per_row) {
            float v[kEight];
            h8 piece[P];
            load_eight(x_row, p.type, c * kEight, p.d, v);
            split_eight<P>(v, power[my_row], piece);
#pragma unroll
            for (int k = 0; k < P; k++) {
                *reinterpret_cast<h8 *>(smem + (size_t)((c >> 2) * P + k) * block_bytes + piece_place(my_row, c & 3)) = piece[k];
            }
        }
    }
    int a_row[MF];
#pragma unroll
    for (int i = 0; i < MF; i++) {
        a_row[i] = min(i * 16 + (r >> 2) + (r & 3) * 4, rows - 1);
    }
    __syncthreads();
    const int part = wave % KS;
    // whole batches of U steps each
    const int share = KS > 1 ? ((p.steps + U * KS - 1) / (U * KS)) * U : p.steps;
    const int t0 = min(part * share, p.steps), t1 = min(t0 + share, p.steps);
    for (int64_t first = (int64_t)blockIdx.x * (W / KS); first < tiles; first += (int64_t)gridDim.x * (W / KS)) {
        const int64_t tile = first + wave / KS;
        if (KS == 1 && tile >= tiles) {
            break;
        }
        const bool mine = KS == 1 || tile < tiles;     // wavefronts that share tiles meet at barriers
        const int64_t col0 = tile * (NF * 16);
        const int last = mine ? (int)min<int64_t>(NF * 16, p.n - col0) - 1 : 0;   // rows behind the last one repeat it
        const uint8_t *const codes = p.codes + (mine ? col0 : 0) * p.row_bytes;
        uint32_t offset[NF];
#pragma unroll
        for (int j = 0; j < NF; j++) {
            offset[j] = (uint32_t)(min(r * NF + j, last) * p.row_bytes);
        }
        const int scale_row = lane % (NF * 16), scale_step = lane / (NF * 16);
        u4 next[U][NF];
        GroupScales<SG, WIDE> next_scales;
        auto fetch = [&](int t) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                const uint32_t byte = (uint32_t)min((t + u) * 64 + q * 16, p.row_bytes - 16);
#pragma unroll
                for (int j = 0; j < NF; j++) {
                    next[u][j] = *reinterpret_cast<const u4 *>(codes + (offset[j] + byte));
                }
            }
            next_scales.load(p, (mine ? col0 : 0) + min(scale_row, last), min((t + scale_step) * SG, p.groups - 1));
        };
        v4f acc[MF][NF] = {};
        if (t0 < t1) {
            fetch(t0);
        }
        for (int t = t0; t < t1; t += U) {
            {
                float scale[SG];
                h2 minus[SG];
                next_scales.take(p, min((t + scale_step) * SG, p.groups - 1), t + scale_step < p.steps, scale, minus);
                const int slot = (scale_step * NF + scale_row % NF) * 16 + scale_row / NF;
#pragma unroll
                for (int g = 0; g < SG; g++) {
                    reinterpret_cast<float *>(turn)[slot * SG + g] = scale[g];
                    reinterpret_cast<h2 *>(turn + kTurn / 2)[slot * SG + g] = minus[g];
                }
            }
            u4 now[U][NF];
#pragma unroll
            for (int u = 0; u < U; u++) {
#pragma unroll
                for (int j = 0; j < NF; j++) {
                    now[u][j] = transpose(next[u][j]);
                }
            }
            if (t + U < t1) {
                fetch(t + U);
            }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (u > 0 && t + u >= t1) {
                    break;
                }
                float scale[NF][SG];
                h2 minus[NF][SG];
#pragma unroll
                for (int j = 0; j < NF; j++) {
#pragma unroll
                    for (int g = 0; g < SG; g++) {
                        scale[j][g] = reinterpret_cast<const float *>(turn)[((u * NF + j) * 16 + r) * SG + g];
                        minus[j][g] = reinterpret_cast<const h2 *>(turn + kTurn / 2)[((u * NF + j) * 16 + r) * SG + g];
                    }
                }
                constexpr int kBlocks = 4 / SG;   // of 32 columns per group, 4 of a step
#pragma unroll
                for (int g = 0; g < SG; g++) {
                    // x has zeros there; where a branch would make registers spill they are multiplied
                    if (g > 0 && !(P == 2 && MF == 4 && W == 8) && (t + u) * SG + g >= p.groups) {
                        break;
                    }
                    v4f sum[MF][NF] = {};
#pragma unroll
                    for (int b = 0; b < kBlocks; b++) {
                        const int block = g * kBlocks + b;
                        h8 w[NF];
#pragma unroll
                        for (int j = 0; j < NF; j++) {
                            w[j] = integers(now[u][j][block], minus[j][g]);
                        }
#pragma unroll
                        for (int k = 0; k < P; k++) {
#pragma unroll
                            for (int i = 0; i < MF; i++) {
                                const h8 a = *reinterpret_cast<const h8 *>(
                                    smem + (size_t)(((t + u) * 4 + block) * P + k) * block_bytes + piece_place(a_row[i], q));
#pragma unroll
                                for (int j = 0; j < NF; j++) {
                                    sum[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, w[j], sum[i][j], 0, 0, 0);
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < MF; i++) {
#pragma unroll
                        for (int j = 0; j < NF; j++) {
#pragma unroll
                            for (int k = 0; k < RI; k++) {
                                acc[i][j][k] = fmaf(scale[j][g], sum[i][j][k], acc[i][j][k]);
                            }
                            asm volatile("" : "+v"(acc[i][j]));   // not left for later, which would keep the sums
                        }
                    }
                }
            }
            __builtin_amdgcn_wave_barrier();
        }
        if constexpr (KS > 1) {
            // the first of a tile's wavefronts adds the others' sums to its own, in their order
            float *const box = reinterpret_cast<float *>(turn);
            if (part > 0) {
#pragma unroll
                for (int i = 0; i < MF; i++) {
#pragma unroll
                    for (int j = 0; j < NF; j++) {
#pragma unroll
                        for (int k = 0; k < RI; k++) {
                            box[((i * NF + j) * RI + k) * 64 + lane] = acc[i][j][k];
                        }
                    }
                }
            }
            __syncthreads();
            if (part == 0) {
                for (int w = 1; w < KS; w++) {
                    const float *const other = reinterpret_cast<const float *>(turn + w * std::max(kTurn, kShare));
#pragma unroll
                    for (int i = 0; i < MF; i++) {
#pragma unroll
                        for (int j = 0; j < NF; j++) {
#pragma unroll
                            for (int k = 0; k < RI; k++) {
                                acc[i][j][k] += other[((i * NF + j) * RI + k) * 64 + lane];
                            }
                        }
                    }
                }
            }
            __syncthreads();
            if (part > 0 || !mine) {
                continue;
            }
        }
        const int64_t col = col0 + r * NF;
        float bias[NF];
        load_bias(p, col, bias);
#pragma unroll
        for (int i = 0; i < MF; i++) {
#pragma unroll
            for (int k = 0; k < RI; k++) {
                const int row = i * 16 + q + 4 * k;
                float sum[NF];
#pragma unroll
                for (int j = 0; j < NF; j++) {
                    sum[j] = acc[i][j][k];
                }
                store_scores(p, row, power[min(row, 63)], col, sum, bias);
            }
        }
    }
}

// Rows of x as fp16 pieces for the kernel below, zeros up to whole steps, and the power of two each was multiplied by.  A wavefront
// per row: 2048 rows of 768 take 6.8 us, 10.7 with a workgroup per row and its barriers.
template <int P>
__global__ __launch_bounds__(256) void group_pieces_kernel(GroupProductParams p, uint8_t *pieces, int *exponents)
{
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (row >= p.m) {
        return;
    }
    const uint8_t *const x_row = static_cast<const uint8_t *>(p.x) + (size_t)row * (size_t)p.ld_x * (p.type == kTypeF32 ? 4 : 2);
    int power = 0;
    if (p.type != kTypeF16) {
        int top = 0;
        for (int c = lane; c * kEight < p.d; c += 64) {
            float v[kEight];
            load_eight(x_row, p.type, c * kEight, p.d, v);
            top = max(top, finite_top(v));
        }
        power = power_for(over_wave(top, [](int a, int b) { return max(a, b); }));
    }
    if (lane == 0) {
        exponents[row] = power;
    }
    const int across = p.steps * (kStep / kEight);
    for (int c = lane; c < across; c += 64) {
        float v[kEight];
        h8 piece[P];
        load_eight(x_row, p.type, c * kEight, p.d, v);
        split_eight<P>(v, power, piece);
#pragma unroll
        for (int k = 0; k < P; k++) {
            reinterpret_cast<h8 *>(pieces)[(row * P + k) * across + c] = piece[k];
        }
    }
}

// Many rows: tiles of WM * 64 rows by WN * 64 coded rows, 64 x 64 per wavefront.  A step's 128 columns of x's pieces go straight
// into one of two LDS buffers while the other is multiplied; codes come to the registers of the wavefront that multiplies
// them, scales and zero points through LDS, all a step ahead.
template <int P, int WM, int WN, int SG, bool WIDE>
__global__ __launch_bounds__(256, 2) void group_tile_kernel(GroupProductParams p, int row_tiles, int col_tiles, int per_xcd)
{
    static_assert(WM * WN == 4, "");
    constexpr int kRows = WM * 64, kCols = WN * 64, kHalf = kRows * 128, kPiece = 2 * kHalf, kABytes = P * kPiece;
    constexpr int kScales = kCols * SG * 4, kBuffer = kABytes + 2 * kScales;
    extern __shared__ __align__(16) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / WN, wn = wave % WN;
    const int64_t id = (int64_t)(blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
    if (id >= (int64_t)row_tiles * col_tiles) {
        return;
    }
    // an XCD's workgroups in flight share columns: row tiles change fastest
    const int64_t row0 = id % row_tiles * kRows, col0 = id / row_tiles * kCols;
    const int last_row = (int)min<int64_t>(kRows, p.m - row0) - 1, last_col = (int)min<int64_t>(kCols, p.n - col0) - 1;
    const uint8_t *const codes = p.codes + col0 * p.row_bytes;
    const int64_t piece_row = (int64_t)p.steps * kStep * 2;    // bytes
    const uint8_t *const a_base = p.pieces + row0 * P * piece_row;
    uint32_t b_from[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        b_from[j] = (uint32_t)(min(wn * 64 + r * 4 + j, last_col) * p.row_bytes);
    }
    u4 next[4];
    GroupScales<SG, WIDE> next_scales;
    const int scale_col = tid % kCols;
    auto fetch = [&](int step, uint8_t *buffer) {
        // 8 rows of 128 bytes at a time; lane l brings the 16 bytes that belong at place l & 7 of row l >> 3
        const int at = lane & 7;
#pragma unroll
        for (int k = 0; k < P; k++) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
#pragma unroll
                for (int run = 0; run < kRows / 32; run++) {
                    const int row = (run * 4 + wave) * 8 + (lane >> 3);
                    const uint8_t *from = a_base + ((int64_t)min(row, last_row) * P + k) * piece_row + step * 256 + h * 128 +
                                          ((at ^ ((row >> 1) & 7)) * 16);
                    uint8_t *to = buffer + k * kPiece + h * kHalf + (run * 4 + wave) * 1024;
                    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from,
                                                     (__attribute__((address_space(3))) void *)to, 16, 0, 0);
                }
            }
        }
        const uint32_t byte = (uint32_t)min(step * 64 + q * 16, p.row_bytes - 16);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            next[j] = *reinterpret_cast<const u4 *>(codes + (b_from[j] + byte));
        }
        next_scales.load(p, col0 + min(scale_col, last_col), step * SG);
    };
    auto put_scales = [&](int step, uint8_t *buffer) {
        if (tid < kCols) {
            float scale[SG];
            h2 minus[SG];
            next_scales.take(p, step * SG, true, scale, minus);
#pragma unroll
            for (int g = 0; g < SG; g++) {
                reinterpret_cast<float *>(buffer + kABytes)[scale_col * SG + g] = scale[g];
                reinterpret_cast<h2 *>(buffer + kABytes + kScales)[scale_col * SG + g] = minus[g];
            }
        }
    };
    v4f acc[4][4] = {};
    fetch(0, smem);
    put_scales(0, smem);
    __builtin_amdgcn_s_waitcnt(kLoaded);
    __syncthreads();
    for (int step = 0; step < p.steps; step++) {
        const uint8_t *const here = smem + (step & 1) * kBuffer;
        uint8_t *const other = smem + (step & 1 ? 0 : kBuffer);
        u4 now[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            now[j] = transpose(next[j]);
        }
        if (step + 1 < p.steps) {
            fetch(step + 1, other);
        }
        constexpr int kBlocks = 4 / SG;
        auto rows_of = [&](int k, int block, int i) {
            const int row = wm * 64 + i * 16 + r;
            return *reinterpret_cast<const h8 *>(here + k * kPiece + (block >> 1) * kHalf + row * 128 +
                                                 ((((block & 1) * 4 + q) ^ ((row >> 1) & 7)) * 16));
        };
#pragma unroll
        for (int g = 0; g < SG; g++) {
            if (g > 0 && step * SG + g >= p.groups) {
                break;      // x has zeros there
            }
            h2 minus[4];
            float scale[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                scale[j] = reinterpret_cast<const float *>(here + kABytes)[(wn * 64 + r * 4 + j) * SG + g];
                minus[j] = reinterpret_cast<const h2 *>(here + kABytes + kScales)[(wn * 64 + r * 4 + j) * SG + g];
            }
            // one row of fragments at a time: no more sums than that at a time beside the results
            h8 w[kBlocks][4];
#pragma unroll
            for (int b = 0; b < kBlocks; b++) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    w[b][j] = integers(now[j][g * kBlocks + b], minus[j]);
                }
            }
            // The next row's are on their way from LDS while this one is multiplied, if registers hold both (128 x 32768 x 4096 in groups of 64
            // 82 -> 75 us, 2048 x 131072 x 768 in groups of 32 886 -> 832).
            constexpr int kHeld = P * kBlocks <= 4 ? 2 : 1;
            h8 a[kHeld][kBlocks][P];
            auto read = [&](int i) {
#pragma unroll
                for (int b = 0; b < kBlocks; b++) {
#pragma unroll
                    for (int k = 0; k < P; k++) {
                        a[i % kHeld][b][k] = rows_of(k, g * kBlocks + b, i);
                    }
                }
            };
            if (kHeld == 2) {
                read(0);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (kHeld == 1 || i < 3) {
                    read(i + kHeld - 1);
                }
                v4f sum[4] = {};
#pragma unroll
                for (int b = 0; b < kBlocks; b++) {
#pragma unroll
                    for (int k = 0; k < P; k++) {
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            sum[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i % kHeld][b][k], w[b][j], sum[j], 0, 0, 0);
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; j++) {
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        acc[i][j][k] = fmaf(scale[j], sum[j][k], acc[i][j][k]);
                    }
                }
                // multiply-adds left for later would keep all their sums in registers
                asm volatile("" : "+v"(acc[i][0]), "+v"(acc[i][1]), "+v"(acc[i][2]), "+v"(acc[i][3]));
            }
        }
        if (step + 1 < p.steps) {
            put_scales(step + 1, other);
        }
        __builtin_amdgcn_s_waitcnt(kLoaded);
        __syncthreads();
    }
    const int64_t col = col0 + wn * 64 + r * 4;
    float bias[4];
    load_bias(p, col, bias);
#pragma unroll
    for (int i = 0; i < 4; i++) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int64_t row = row0 + wm * 64 + i * 16 + q * 4 + k;
            const float sum[4] = {acc[i][0][k], acc[i][1][k], acc[i][2][k], acc[i][3][k]};
            store_scores(p, row, p.exponents[min(row, p.m - 1)], col, sum, bias);
        }
    }
}

// Fewer than four scales in all (up to three short rows of codes): a thread per score.  Sums before the scale are of x times its power of
// two here too, or they could pass the largest number where the score does not.
__global__ __launch_bounds__(256) void group_tiny_kernel(GroupProductParams p, int group)
{
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, row = id / p.n, col = id - row * p.n;
    if (row >= p.m) {
        return;
    }
    const uint8_t *const x_row = static_cast<const uint8_t *>(p.x) + (size_t)row * (size_t)p.ld_x * (p.type == kTypeF32 ? 4 : 2);
    int top = 0;
    for (int at = 0; p.type != kTypeF16 && at < p.d; at += kEight) {
        float v[kEight];
        load_eight(x_row, p.type, at, p.d, v);
        top = max(top, finite_top(v));
    }
    const int power = power_for(top);
    float sum = 0.f, of_group = 0.f;
    for (int at = 0; at < p.d; at += kEight) {
        const int64_t slot = col * p.groups + at / group;
        const float zero = p.has_zeros ? (float)p.zeros[slot] : 8.f;
        const uint32_t code = *reinterpret_cast<const uint32_t *>(p.codes + col * p.row_bytes + at / 2);
        float v[kEight];
        load_eight(x_row, p.type, at, p.d, v);
#pragma unroll
        for (int i = 0; i < kEight; i++) {
            of_group += at + i < p.d ? ldexpf(v[i], power) * ((float)(code >> (4 * i) & 15u) - zero) : 0.f;
        }
        if ((at + kEight) % group == 0 || at + kEight >= p.d) {
            const float scale = p.scale_type == kTypeF32   ? static_cast<const float *>(p.scales)[slot]
                                : p.scale_type == kTypeF16 ? (float)static_cast<const _Float16 *>(p.scales)[slot]
                                                           : (float)static_cast<const __bf16 *>(p.scales)[slot];
            sum = fmaf(scale, of_group, sum);
            of_group = 0.f;
        }
    }
    const float sums[1] = {sum};
    float bias[1];
    load_bias(p, col, bias);
    store_scores(p, row, power, col, sums, bias);
}

int pieces_of(int type) { return type == kTypeF32 ? 2 : 1; }
int steps_of(int d) { return (d + kStep - 1) / kStep; }
size_t row_lds(int type, int64_t m, int d) { return (size_t)steps_of(d) * 4 * pieces_of(type) * (size_t)m * 64; }
// Few rows whose pieces fit a CU's LDS stay there.
constexpr size_t kTurnLds = 8 * 64 * 4 * 8;
bool stays(int type, int64_t m, int d) { return m <= 64 && row_lds(type, m, d) + 256 + kTurnLds <= 160 * 1024; }

template <int P, int MF, int RI, int NF, int U, int KS, int SG, bool WIDE, int W>
void launch_stream(const GroupProductParams &p, hipStream_t s)
{
    constexpr size_t turn = W * std::max(64 * SG * 8, KS > 1 ? MF * NF * RI * 256 : 0);
    static_assert(turn <= kTurnLds, "");
    const size_t lds = row_lds(p.type, p.m, p.d) + 256 + turn;
    const int64_t tiles = (p.n + NF * 16 - 1) / (NF * 16);
    const auto kern = group_stream_kernel<P, MF, RI, NF, U, KS, SG, WIDE, W>;
    require_dynamic_lds(reinterpret_cast<const void *>(kern), lds);
    const int64_t most = resident_workgroups(reinterpret_cast<const void *>(kern), W * 64, lds);
    hipLaunchKernelGGL(kern, dim3((unsigned)std::min((tiles * KS + W - 1) / W, most)), dim3(W * 64), lds, s, p, tiles);
    check_launch();
}

template <int P, int SG, bool WIDE, int W>
void launch_stream(const GroupProductParams &p, hipStream_t s)
{
    // Fragments of 16 stored rows four steps ahead up to 32768 rows, more and wider ones beyond: a bfloat16 row of 768 in groups of 64 against
    // 16384 takes 5.5 us, 6.4 with wide ones, against 32768 6.5 with both, against 65536 9.6 and 8.4; 64 rows of 200 in groups of 32 11.6 and 13.9,
    // 13.2 and 14.2, 17.7 and 14.3.
    // Long rows' steps are shared: 16 bfloat16 rows of 2048 in groups of 64 against 4096 take 14.2 us, 17.8 if they are not, of 1024 9.4 and 10.6,
    // of 512 6.6 and 6.8 (against 16384 17.8 and 21.0, 12.7 and 10.8, 8.6 and 7.0).
    const bool narrow = p.n <= 32768, deep = narrow && p.steps >= 8;
    // up to 16 rows of fewer than eight steps need no eight wavefronts: they have 56 KB of pieces at most
    constexpr bool kShallow = W == 4;
    if (p.m <= 4) {
        if (deep) {
            launch_stream<P, 1, 1, 1, 4, 4, SG, WIDE, W>(p, s);
        } else if (!narrow) {
            launch_stream<P, 1, 1, 2, 2, 1, SG, WIDE, W>(p, s);
        } else if constexpr (kShallow) {
            launch_stream<P, 1, 1, 1, 4, 1, SG, WIDE, W>(p, s);
        }
    } else if (p.m <= 16) {
        if (deep) {
            launch_stream<P, 1, 4, 1, 4, 4, SG, WIDE, W>(p, s);
        } else if (!narrow) {
            launch_stream<P, 1, 4, 2, 2, 1, SG, WIDE, W>(p, s);
        } else if constexpr (kShallow) {
            launch_stream<P, 1, 4, 1, 4, 1, SG, WIDE, W>(p, s);
        }
    } else if (p.m <= 32) {
        narrow ? launch_stream<P, 2, 4, 1, 4, 1, SG, WIDE, W>(p, s) : launch_stream<P, 2, 4, 4, 1, 1, SG, WIDE, W>(p, s);
    } else {
        // with eight wavefronts, 256 registers each, four columns' worth of fragments would spill
        narrow ? launch_stream<P, 4, 4, 1, 4, 1, SG, WIDE, W>(p, s) : launch_stream<P, 4, 4, W == 8 ? 2 : 4, W == 8 ? 2 : 1, 1, SG, WIDE, W>(p, s);
    }
}

template <int P, int WM, int WN, int SG, bool WIDE>
void launch_tiles(const GroupProductParams &p, hipStream_t s)
{
    const int64_t row_tiles = (p.m + WM * 64 - 1) / (WM * 64), col_tiles = (p.n + WN * 64 - 1) / (WN * 64);
    const int64_t per_xcd = (row_tiles * col_tiles + 7) / 8;
    IXA_REQUIRE(per_xcd * 8 * 256 <= 0xffffffffll, kErrInvalidParam, "group_product: %ld x %ld scores in one call", (long)p.m,
                (long)p.n);
    // one buffer where there is one step: of two pieces two workgroups share a CU then
    const size_t lds = std::min(p.steps, 2) * ((size_t)P * WM * 64 * 256 + 2 * WN * 64 * SG * 4);
    const auto kern = group_tile_kernel<P, WM, WN, SG, WIDE>;
    require_dynamic_lds(reinterpret_cast<const void *>(kern), lds);
    hipLaunchKernelGGL(kern, dim3((unsigned)per_xcd * 8), dim3(256), lds, s, p, (int)row_tiles, (int)col_tiles, (int)per_xcd);
    check_launch();
}

template <int P, int SG, bool WIDE>
void launch(GroupProductParams &p, uint8_t *workspace, hipStream_t s)
{
    if (stays(p.type, p.m, p.d)) {
        // Four wavefronts where two such workgroups share a CU, eight where one has it to itself (48 bfloat16 rows of 768, 72 KB of pieces,
        // groups of 32, against 100,003 rows: 51 us with four, 36 with eight; 4096 rows: 22 and 18).
        row_lds(p.type, p.m, p.d) <= kHalfLds ? launch_stream<P, SG, WIDE, 4>(p, s) : launch_stream<P, SG, WIDE, 8>(p, s);
        return;
    }
    int *const exponents = reinterpret_cast<int *>(workspace);
    uint8_t *const pieces = workspace + round_up(p.m * 4, 256);
    hipLaunchKernelGGL((group_pieces_kernel<P>), dim3((unsigned)((p.m + 3) / 4)), dim3(256), 0, s, p, pieces, exponents);
    check_launch();
    p.pieces = pieces;
    p.exponents = exponents;
    if (p.m <= 64) {
        launch_tiles<P, 1, 4, SG, WIDE>(p, s);
    } else {
        launch_tiles<P, 2, 2, SG, WIDE>(p, s);
    }
}

}  // namespace

int64_t group_product_workspace(int type, int64_t m, int d)
{
    check_type("group_product", type);
    IXA_REQUIRE(m >= 0 && m <= kMaxProductRows && d >= 1 && d <= kMaxCodeDim, kErrInvalidParam,
                "group_product: rows %ld (0 ... %ld), dims %d (1 ... %d)", (long)m, (long)kMaxProductRows, d, kMaxCodeDim);
    return m == 0 || stays(type, m, d) ? 0 : round_up(m * 4, 256) + m * pieces_of(type) * steps_of(d) * kStep * 2;
}

void op_group_product(const void *x, int64_t ld_x, int type, int64_t m, const uint8_t *codes, const void *scales,
                      const uint8_t *zeros, int group, int scale_type, int64_t n, int d, float alpha, const float *bias,
                      int out_type, void *out, int64_t ld, void *workspace, int64_t workspace_bytes, hipStream_t s)
{
    const int64_t need = group_product_workspace(type, m, d);
    const bool none = m == 0 || n == 0;
    check_type("group_product", out_type);
    check_groups("group_product", group, scale_type, m == 0 ? 0 : n, d, codes, scales);
    check_row_buffer("group_product", x, ld_x, type, n == 0 ? 0 : m, d);
    check_row_buffer("group_product", out, ld, out_type, none ? 0 : m, n);
    IXA_REQUIRE(n >= 0 && n <= 0x7fffffff, kErrInvalidParam, "group_product: rows %ld (< 2^31)", (long)n);
    IXA_REQUIRE(alpha - alpha == 0.f, kErrInvalidParam, "group_product: alpha %g has to be finite", (double)alpha);
    IXA_REQUIRE(on_bytes(bias, 4), kErrInvalidParam, "group_product: biases are not aligned to their elements");
    if (none) {
        return;
    }
    IXA_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && on_bytes(workspace, 16)), kErrInvalidParam,
                "group_product: needs a workspace of %ld bytes on 16, has %ld", (long)need, (long)workspace_bytes);
    int device;
    check_answer(hipGetDevice(&device));   // what is asked of a kernel before its launch needs one
    GroupProductParams p{};
    p.x = x;
    p.codes = codes;
    p.has_zeros = zeros != nullptr;
    p.zeros = zeros ? zeros : codes;     // loads without use stay in an array
    p.scales = scales;
    p.bias = bias;
    p.out = out;
    p.m = m;
    p.n = n;
    p.ld_x = ld_x;
    p.ld = ld;
    p.type = type;
    p.scale_type = scale_type;
    p.out_type = out_type;
    p.d = d;
    p.groups = group_count(group, d);
    p.row_bytes = (int)group_row_bytes(group, d);
    p.steps = steps_of(d);
    p.scale_count = n * p.groups;
    p.alpha = alpha;
    if (p.scale_count < 4) {
        hipLaunchKernelGGL(group_tiny_kernel, dim3((unsigned)((m * n + 255) / 256)), dim3(256), 0, s, p, group);
        check_launch();
        return;
    }
    uint8_t *const work = static_cast<uint8_t *>(workspace);
    const auto of_group = [&](auto pieces, auto wide) {
        constexpr int P = decltype(pieces)::value;
        constexpr bool kWide = decltype(wide)::value;
        if (group == 32) {
            launch<P, 4, kWide>(p, work, s);
        } else if (group == 64) {
            launch<P, 2, kWide>(p, work, s);
        } else {
            launch<P, 1, kWide>(p, work, s);
        }
    };
    const auto of_type = [&](auto pieces) {
        if (scale_type == kTypeF32) {
            of_group(pieces, std::true_type());
        } else {
            of_group(pieces, std::false_type());
        }
    };
    if (type == kTypeF32) {
        of_type(std::integral_constant<int, 2>());
    } else {
        of_type(std::integral_constant<int, 1>());
    }
}

}  // namespace ixa
