// Scores of query rows a against stored rows b in microscaled codes: g[i][j] = sum over k of a[i][k] b[j][k], or the squared
// distance (|a_i|^2 + |b_j|^2) - 2 g, its last step one multiply-add.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 16 x 128 by 128 x 16 codes and applies the power-of-two scale of each row's
// block of 32 itself.  A lane (row r = l & 15, quarter g = l >> 4) gives it, in 4 bits, the 16 bytes of block g of its row;
// in 8 bits, bytes 16 g ... 16 g + 15 of the first and of the second 64; and in both the scale of block g.  A lane ends up with
// scores of queries 4 g ... 4 g + 3 and stored row r of the fragment; four fragments of stored rows are dealt so that row r of
// fragment j is row 4 r + j of 64, and the lane holds four scores next to each other: 16 lanes write 256 bytes in a row.
//
// Two 4-bit numbers multiply and add up without any loss in the instruction.  Products of an 8-bit and a 4-bit number span
// more bits than it keeps (what lies under about 2^-14 of the largest product is dropped: 1e-4 of the sum of magnitudes
// was measured on random codes), so an 8-bit operand goes in twice: the codes of magnitude 2 and more, then the others.
// Within either half all products are multiples of the smallest that the instruction keeps (2^8.8 * 6 against 2^-2 * 0.5,
// and 2 * 6 against 2^-9 * 0.5), and the sums are those of 32 bits.
#include "lowp.h"

#include <algorithm>
#include <type_traits>

namespace ixa {

namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));   // 16 bytes of codes

constexpr int kE4M3 = 0, kE2M1 = 4;   // operand formats of the instruction

struct ProductParams {
    const uint8_t *a_codes, *a_scales, *b_codes, *b_scales;
    const float *a_sqr, *b_sqr;
    int64_t m, n, ld;
    int blocks, metric;
    void *out;
    bool lines;   // rows of scores start on 64 bytes
};

__device__ __forceinline__ v8i wide(u4 lo) { return v8i{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, 0, 0, 0, 0}; }

// What a lane gives the instruction of one query fragment: 4-bit codes, or the two halves of 8-bit codes.
template <int FA>
struct AFragment;
template <>
struct AFragment<kE2M1> {
    v8i v;
    __device__ __forceinline__ void set(const u4 (&w)[1]) { v = wide(w[0]); }
    template <int BYTE = 0>   // which byte of the scales' registers
    __device__ __forceinline__ v4f multiply(int scale, const v8i &b, int b_scale, v4f c) const
    {
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(v, b, c, kE2M1, kE2M1, BYTE, scale, BYTE, b_scale);
    }
};
template <>
struct AFragment<kE4M3> {
    v8i small, large;
    __device__ __forceinline__ void set(const u4 (&w)[2])
    {
        const uint32_t u[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t two = u[i] & 0x40404040u;           // exponent field 8 and up: magnitude 2 and more
            const uint32_t mask = (two << 1) - (two >> 6);     // their seven bits below the sign
            small[i] = (int)(u[i] & ~mask);
            large[i] = (int)(u[i] & (mask | 0x80808080u));
        }
    }
    template <int BYTE = 0>
    __device__ __forceinline__ v4f multiply(int scale, const v8i &b, int b_scale, v4f c) const
    {
        c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(small, b, c, kE4M3, kE2M1, BYTE, scale, BYTE, b_scale);
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(large, b, c, kE4M3, kE2M1, BYTE, scale, BYTE, b_scale);
    }
};

// N values from `at` on of an array that ends at n: those behind its end repeat the last
template <int N>
__device__ __forceinline__ void load_run(const float *from, int64_t at, int64_t n, float (&v)[N])
{
    if (at + N <= n) {
        __builtin_memcpy(v, from + at, sizeof(v));
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) {
            v[i] = from[min(at + i, n - 1)];
        }
    }
}

// Scores are not read again here: where rows of scores start on 64 bytes they pass the caches by, which leaves these to the
// codes (2048 x 131072 x 768 to fp32: 360 -> 290 us); rows that start anywhere share lines, which the L2 has to join (1024 x
// 199999 x 128: 210 us, past the caches 330).  A wavefront's run is a line or more, but for 32 bytes where NF = 1 has 16-bit
// scores: few rows, whose scores are small.
// The scores of a lane: queries row ... row + 3 (element i of the accumulators) and columns col ... col + NF - 1 (fragment j).
template <typename T, int NF>
__device__ __forceinline__ void store_scores(const ProductParams &p, int64_t row, int64_t col, const v4f (&acc)[NF],
                                             const float (&b_sqr)[NF])
{
    if (row >= p.m || col >= p.n) {
        return;
    }
    const bool l2 = p.metric == kMetricL2;
    float a_sqr[4] = {};
    if (l2) {
        load_run(p.a_sqr, row, p.m, a_sqr);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (row + i < p.m) {
            typedef T Scores __attribute__((ext_vector_type(NF)));
            typedef T ScoresAnywhere __attribute__((ext_vector_type(NF), aligned(sizeof(T))));
            Scores v;
#pragma unroll
            for (int j = 0; j < NF; j++) {
                v[j] = (T)(l2 ? fmaf(acc[j][i], -2.f, a_sqr[i] + b_sqr[j]) : acc[j][i]);
            }
            T *o = static_cast<T *>(p.out) + (row + i) * p.ld + col;
            if (col + NF <= p.n) {
                if (p.lines) {
                    __builtin_nontemporal_store(v, reinterpret_cast<Scores *>(o));
                } else {
                    *reinterpret_cast<ScoresAnywhere *>(o) = v;
                }
            } else {
#pragma unroll
                for (int j = 0; j < NF; j++) {
                    if (col + j < p.n) {
                        o[j] = v[j];
                    }
                }
            }
        }
    }
}

// Fragments in LDS: 16 rows of 64 bytes are 1 KB, four 16-byte pieces per row, piece q of row r at place q ^ ((r >> 1) & 3):
// eight lanes in a row that read one piece of eight rows find them in all banks.
__device__ __forceinline__ int fragment_place(int r, int q) { return r * 64 + ((q ^ ((r >> 1) & 3)) * 16); }
// The same for NF fragments of stored rows dealt as above.  Neighbouring rows, which are written together, lie in fragments
// of their own: every second one swaps its rows in pairs to be in other banks.
template <int NF>
__device__ __forceinline__ int stored_place(int j, int r, int q)
{
    return j * 1024 + (NF > 1 ? r ^ (j & 1) : r) * 64 + ((q ^ ((r >> 1) & 3)) * 16);
}

// The scales of one row, four blocks at a time and in two parts so that nothing waits for the load: load_scales brings four
// bytes at `at` or, where those would end `over` bytes behind the array, its last four (`few`: the number of scales of an array
// that has less than four, else 0); take_scales shifts and masks them.  Blocks behind the last get scale 0, the smallest power
// of two: the queries' codes are zeros there.
__device__ __forceinline__ uint32_t load_scales(const uint8_t *base, int at, int over, int few)
{
    const uint8_t *from = base + (at - max(over, 0));
    uint32_t w = 0;
    if (few == 0) {
        __builtin_memcpy(&w, from, 4);
    } else {   // no loop: around one the compiler waits for every load in flight
        w = from[0] | (few > 1 ? (uint32_t)from[1] << 8 : 0u) | (few > 2 ? (uint32_t)from[2] << 16 : 0u);
    }
    return w;
}
__device__ __forceinline__ uint32_t take_scales(uint32_t w, int b, int over, int blocks)
{
    w >>= 8 * min(max(over, 0), 3);
    return blocks - b >= 4 ? w : w & ((1u << (8 * max(blocks - b, 0))) - 1u);
}
// `over` of a row's block 0 in an array of rows * blocks scales; of block b it is b more
__device__ __forceinline__ int scales_over(int64_t row, int64_t rows, int blocks)
{
    return (int)max(row * blocks - max(rows * blocks - 4, (int64_t)0), (int64_t)-0x40000000);
}
__device__ __forceinline__ int few_scales(int64_t rows, int blocks) { return rows * blocks < 4 ? (int)rows * blocks : 0; }

// Few queries (MF fragments of 16): their codes stay in LDS, all columns of them, while every wavefront streams NF fragments of
// stored rows past them, U steps of 128 columns ahead.  Bound by the stored rows and the scores, both moved once: 64 x 1M x
// 768 145 us, 4.6 TB/s; 1 x 1M x 1536 154 us, 5.3 TB/s; 1 x 1M x 128 15.5 us, 4.9 TB/s.  The stored rows come in whole pieces
// of 64 bytes, four lanes each, and change lanes in 1 KB of LDS per fragment and step that the wavefront has to itself: read
// the way the instruction wants them, 16 lanes would touch 16 rows at a time.  Only queries that exist take LDS, which is what
// limits the wavefronts of a CU in long rows (1 x 50000 x 4096: 50 -> 27 us).
template <int FA, int MF, int NF, int U, typename T>
__global__ __launch_bounds__(256) void mx_stream_kernel(ProductParams p, int steps, int64_t tiles)
{
    extern __shared__ __align__(16) uint8_t smem[];
    constexpr int kHalves = FA == kE2M1 ? 1 : 2;           // 64-byte halves of a row's step
    // the rows of fragments behind the last query read its codes, and their scores are not stored
    const int rows = (int)p.m, step_bytes = rows * 64 * kHalves;
    uint8_t *const scales = smem + (size_t)steps * step_bytes;   // [step][row][block of the step]
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint8_t *const turn = scales + (((size_t)steps * rows * 4 + 15) & ~(size_t)15) + wave * (NF * U * (1024 + 64));
    uint8_t *const turn_scales = turn + NF * U * 1024;
    static_assert(NF * U == 4, "a lane brings the scales of one row and step");
    const int a_row_bytes = p.blocks * 16 * kHalves, b_row_bytes = p.blocks * 16;
    // 256, 128 ... 4 threads bring a row; pieces behind its last block are zeros
    const int lg = rows > 1 ? 8 - (32 - __builtin_clz(rows - 1)) : 8, per_row = 1 << lg;
    if (const int row = (int)threadIdx.x >> lg, e = (int)threadIdx.x & (per_row - 1); row < rows) {
        const uint8_t *const from = p.a_scales + (int64_t)row * p.blocks;
        const int over = scales_over(row, p.m, p.blocks), few = few_scales(p.m, p.blocks);
        for (int step = e; step < steps; step += per_row) {
            reinterpret_cast<uint32_t *>(scales)[step * rows + row] = take_scales(
                load_scales(from, step * 4, over + step * 4, few), step * 4, over + step * 4, p.blocks);
        }
        for (int piece = e; piece < steps * 4 * kHalves; piece += per_row) {
            u4 v = u4{};
            if (piece * 16 < a_row_bytes) {
                v = *reinterpret_cast<const u4 *>(p.a_codes + (int64_t)row * a_row_bytes + piece * 16);
            }
            *reinterpret_cast<u4 *>(smem + (size_t)(piece >> 2) * rows * 64 + fragment_place(row, piece & 3)) = v;
        }
    }
    int a_row[MF];
#pragma unroll
    for (int i = 0; i < MF; i++) {
        a_row[i] = min(i * 16 + r, rows - 1);
    }
    __syncthreads();
    const int few = few_scales(p.n, p.blocks);
    const int64_t stride = (int64_t)gridDim.x * 4;
    for (int64_t tile = (int64_t)blockIdx.x * 4 + wave; tile < tiles; tile += stride) {
        const int64_t col0 = tile * (NF * 16);
        const int last = (int)min<int64_t>(NF * 16, p.n - col0) - 1;   // rows behind the last one repeat it
        const uint8_t *const codes = p.b_codes + col0 * b_row_bytes;
        uint32_t offset[NF];
#pragma unroll
        for (int k = 0; k < NF; k++) {
            offset[k] = (uint32_t)(min(k * 16 + (lane >> 2), last) * b_row_bytes);
        }
        const int scale_row = lane % (NF * 16), scale_step = lane / (NF * 16) % U;
        const uint8_t *const scale_from = p.b_scales + (col0 + min(scale_row, last)) * p.blocks;
        const int over = scales_over(col0 + min(scale_row, last), p.n, p.blocks);
        u4 next[U][NF];
        uint32_t next_scale = 0;
        // pieces behind the last block repeat it: the queries' codes are zeros there
        auto fetch = [&](int t) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                const uint32_t byte = (uint32_t)min((t + u) * 64 + (lane & 3) * 16, b_row_bytes - 16);
#pragma unroll
                for (int k = 0; k < NF; k++) {
                    next[u][k] = *reinterpret_cast<const u4 *>(codes + (offset[k] + byte));
                }
            }
            const int b_from = min(t + scale_step, steps - 1) * 4;
            next_scale = load_scales(scale_from, b_from, over + b_from, few);
        };
        fetch(0);
        v4f acc[MF][NF] = {};
        for (int t = 0; t < steps; t += U) {
#pragma unroll
            for (int u = 0; u < U; u++) {
#pragma unroll
                for (int k = 0; k < NF; k++) {
                    const int row = k * 16 + (lane >> 2);
                    *reinterpret_cast<u4 *>(turn + u * (NF * 1024) + stored_place<NF>(row % NF, row / NF, lane & 3)) = next[u][k];
                }
            }
            const int b_from = min(t + scale_step, steps - 1) * 4;
            reinterpret_cast<uint32_t *>(turn_scales)[scale_step * (NF * 16) + (scale_row % NF) * 16 + scale_row / NF] =
                take_scales(next_scale, b_from, over + b_from, p.blocks);
            if (t + U < steps) {
                fetch(t + U);
            }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (u > 0 && t + u >= steps) {
                    break;
                }
                v8i b[NF];
                int b_scale[NF];
#pragma unroll
                for (int j = 0; j < NF; j++) {
                    b[j] = wide(*reinterpret_cast<const u4 *>(turn + u * (NF * 1024) + stored_place<NF>(j, r, g)));
                    b_scale[j] = turn_scales[((u * NF + j) * 16 + r) * 4 + g];
                }
#pragma unroll
                for (int i = 0; i < MF; i++) {
                    u4 w[kHalves];
#pragma unroll
                    for (int k = 0; k < kHalves; k++) {
                        w[k] = *reinterpret_cast<const u4 *>(smem + (size_t)(t + u) * step_bytes + k * rows * 64 +
                                                                fragment_place(a_row[i], g));
                    }
                    const int a_scale = scales[((t + u) * rows + a_row[i]) * 4 + g];
                    AFragment<FA> a;
                    a.set(w);
#pragma unroll
                    for (int j = 0; j < NF; j++) {
                        acc[i][j] = a.multiply(a_scale, b[j], b_scale[j], acc[i][j]);
                    }
                }
            }
            __builtin_amdgcn_wave_barrier();
        }
        const int64_t col = col0 + r * NF;
        float b_sqr[NF] = {};
        if (p.metric == kMetricL2) {
            load_run(p.b_sqr, col, p.n, b_sqr);
        }
#pragma unroll
        for (int i = 0; i < MF; i++) {
            store_scores<T, NF>(p, i * 16 + g * 4, col, acc[i], b_sqr);
        }
    }
}

// Many queries: tiles of WM * MF * 16 queries by WN * 64 stored rows, one wavefront per MF * 16 x 64 of them (MF x 4 fragments).
// Codes and scales of both sides go through two LDS buffers of U steps (128 columns each); while one is multiplied, the next is
// written from registers and the one after it is on its way from memory.  Any sizes and strides.  Bound by the scores in short
// rows (2048 x 131072 x 200 to fp32: 235 us, 4.6 TB/s), in long ones by what the wavefronts read from LDS between products: 2048 x
// 100001 x 768 288 us, 1.1 PFLOP/s with 3 TB/s of scores; 1024 x 60001 x 2016 124 us, 2 PFLOP/s.
template <int FA, int WM, int WN, int MF, int U, typename T>
__global__ __launch_bounds__(WM * WN * 64, MF == 8 || FA == kE4M3 ? 2 : 3)
void mx_tile_kernel(ProductParams p, int row_tiles, int col_tiles, int per_xcd)
{
    constexpr int kHalves = FA == kE2M1 ? 1 : 2, NF = 4, kThreads = WM * WN * 64;
    constexpr int kRows = WM * MF * 16, kCols = WN * 64;
    constexpr int kABytes = kRows * 64 * kHalves * U, kBBytes = kCols * 64 * U;
    constexpr int kAPieces = kABytes / 16 / kThreads, kBPieces = kBBytes / 16 / kThreads;   // per thread
    constexpr int kScaleRows = (kRows + kCols + kThreads - 1) / kThreads;
    constexpr int kBuffer = kABytes + kBBytes + (kRows + kCols) * 4 * U;
    static_assert(U == 1 || U == 2, "the scales of a row's block in a buffer are one read");
    __shared__ __align__(16) uint8_t smem[2 * kBuffer];
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / WN, wn = wave % WN;
    const int64_t id = (int64_t)(blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
    if (id >= (int64_t)row_tiles * col_tiles) {
        return;
    }
    const int64_t band = id / (8 * (int64_t)col_tiles);
    const int high = min(8, row_tiles - (int)band * 8);
    const int64_t in = id - band * 8 * col_tiles;
    const int64_t row0 = (band * 8 + in % high) * kRows, col0 = in / high * kCols;
    const int steps = (p.blocks + 3) / 4, stages = (steps + U - 1) / U;
    const int a_row_bytes = p.blocks * 16 * kHalves, b_row_bytes = p.blocks * 16;

    const uint8_t *const a_base = p.a_codes + row0 * a_row_bytes, *const b_base = p.b_codes + col0 * b_row_bytes;
    const int last_row = (int)min<int64_t>(kRows, p.m - row0) - 1, last_col = (int)min<int64_t>(kCols, p.n - col0) - 1;
    u4 a_piece[kAPieces], b_piece[kBPieces];
    uint32_t scale[kScaleRows][U];
    // the rows whose scales a thread brings
    static_assert(kRows % 64 == 0, "a wavefront's scales are all of one side");
    const uint8_t *scale_base[kScaleRows];
    int scale_offset[kScaleRows], over[kScaleRows];
    const int few = few_scales(p.n, p.blocks);   // a tile's queries have more than four scales: they are many, or long
#pragma unroll
    for (int k = 0; k < kScaleRows; k++) {
        const bool query = wave * 64 + k * kThreads < kRows;
        const int row = tid + k * kThreads, in = query ? min(row, last_row) : min(row - kRows, last_col);
        const int64_t first = query ? row0 : col0;
        scale_base[k] = (query ? p.a_scales : p.b_scales) + first * p.blocks;
        scale_offset[k] = in * p.blocks;
        over[k] = scales_over(first + in, query ? p.m : p.n, p.blocks);
    }
    auto bring = [&](int stage) {   // from memory into registers
#pragma unroll
        for (int k = 0; k < kScaleRows; k++) {
            if (const int row = wave * 64 + k * kThreads; row < kRows + kCols) {
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int b = (stage * U + u) * 4;
                    scale[k][u] = load_scales(scale_base[k], scale_offset[k] + b, over[k] + b, row < kRows ? 0 : few);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < kAPieces; k++) {
            const int e = tid + k * kThreads, row = min((e >> 2) % kRows, last_row);
            const int byte = (stage * U * kHalves + (e >> 2) / kRows) * 64 + (e & 3) * 16;
            a_piece[k] = *reinterpret_cast<const u4 *>(a_base + (uint32_t)(row * a_row_bytes + min(byte, a_row_bytes - 16)));
        }
#pragma unroll
        for (int k = 0; k < kBPieces; k++) {
            const int e = tid + k * kThreads, row = min((e >> 2) % kCols, last_col);
            const int byte = (stage * U + (e >> 2) / kCols) * 64 + (e & 3) * 16;
            b_piece[k] = *reinterpret_cast<const u4 *>(b_base + (uint32_t)(row * b_row_bytes + min(byte, b_row_bytes - 16)));
        }
    };
    auto put = [&](int stage) {     // from registers into LDS; queries' codes behind the last block are zeros
        uint8_t *const to = smem + (stage & 1) * kBuffer;
#pragma unroll
        for (int k = 0; k < kAPieces; k++) {
            const int e = tid + k * kThreads, row = (e >> 2) % kRows;
            const int byte = (stage * U * kHalves + (e >> 2) / kRows) * 64 + (e & 3) * 16;
            *reinterpret_cast<u4 *>(to + (e >> 2) / kRows * (kRows * 64) + (row >> 4) * 1024 + fragment_place(row & 15, e & 3)) =
                byte < a_row_bytes ? a_piece[k] : u4{};
        }
#pragma unroll
        for (int k = 0; k < kBPieces; k++) {
            const int e = tid + k * kThreads, row = (e >> 2) % kCols;
            *reinterpret_cast<u4 *>(to + kABytes + (e >> 2) / kCols * (kCols * 64) + (row >> 6) * 4096 +
                                       stored_place<NF>(row & 3, (row & 63) >> 2, e & 3)) = b_piece[k];
        }
#pragma unroll
        for (int k = 0; k < kScaleRows; k++) {
            const int row = tid + k * kThreads;
            if (row < kRows + kCols) {
                const int place = row < kRows ? row : (row & ~63) | ((row & 3) * 16 + ((row & 63) >> 2));
                uint8_t *const o = to + kABytes + kBBytes + place * 4 * U;
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int b = (stage * U + u) * 4;
                    scale[k][u] = take_scales(scale[k][u], b, over[k] + b, p.blocks);
                }
                if constexpr (U == 2) {   // block g of either step next to each other
                    *reinterpret_cast<uint2 *>(o) = make_uint2(__builtin_amdgcn_perm(scale[k][1], scale[k][0], 0x05010400u),
                                                               __builtin_amdgcn_perm(scale[k][1], scale[k][0], 0x07030602u));
                } else {
                    *reinterpret_cast<uint32_t *>(o) = scale[k][0];
                }
            }
        }
    };
    using Scales = std::conditional_t<U == 2, uint16_t, uint8_t>;

    v4f acc[MF][NF] = {};
    bring(0);
    put(0);
    if (stages > 1) {
        bring(1);
    }
    __syncthreads();
    for (int stage = 0; stage < stages; stage++) {
        const uint8_t *const from = smem + (stage & 1) * kBuffer;
        if (stage + 1 < stages) {
            put(stage + 1);
        }
        if (stage + 2 < stages) {
            bring(stage + 2);
        }
        const Scales *const sc = reinterpret_cast<const Scales *>(from + kABytes + kBBytes);
        int a_scale[MF], b_scale[NF];
#pragma unroll
        for (int i = 0; i < MF; i++) {
            a_scale[i] = sc[((wm * MF + i) * 16 + r) * 4 + g];
        }
#pragma unroll
        for (int j = 0; j < NF; j++) {
            b_scale[j] = sc[(kRows + wn * 64 + j * 16 + r) * 4 + g];
        }
        auto step = [&](auto which) {
            constexpr int u = decltype(which)::value;
            v8i b[NF];
#pragma unroll
            for (int j = 0; j < NF; j++) {
                b[j] = wide(*reinterpret_cast<const u4 *>(from + kABytes + u * (kCols * 64) + wn * 4096 +
                                                             stored_place<NF>(j, r, g)));
            }
#pragma unroll
            for (int i = 0; i < MF; i++) {
                u4 w[kHalves];
#pragma unroll
                for (int k = 0; k < kHalves; k++) {
                    w[k] = *reinterpret_cast<const u4 *>(from + (u * kHalves + k) * (kRows * 64) + (wm * MF + i) * 1024 +
                                                            fragment_place(r, g));
                }
                AFragment<FA> a;
                a.set(w);
#pragma unroll
                for (int j = 0; j < NF; j++) {
                    acc[i][j] = a.template multiply<u>(a_scale[i], b[j], b_scale[j], acc[i][j]);
                }
            }
        };
        step(std::integral_constant<int, 0>());
        if constexpr (U == 2) {
            if (stage * 2 + 1 < steps) {
                step(std::integral_constant<int, 1>());
            }
        }
        __syncthreads();
    }
    const int64_t col = col0 + wn * 64 + r * 4;
    float b_sqr[NF] = {};
    if (p.metric == kMetricL2 && col < p.n) {
        load_run(p.b_sqr, col, p.n, b_sqr);
    }
#pragma unroll
    for (int i = 0; i < MF; i++) {
        store_scores<T, NF>(p, row0 + (wm * MF + i) * 16 + g * 4, col, acc[i], b_sqr);
    }
}

typedef float v16f __attribute__((ext_vector_type(16)));

// v_mfma_scale_f32_32x32x64_f8f6f4: 32 x 64 by 64 x 32 codes, lane = row l & 31, half h = l >> 5.  In 4 bits the lane holds the
// 16 bytes of block h; in 8 bits bytes 16 h ... of block 0 and of block 1; its scores are of stored row l & 31 and queries
// 8 (i / 4) + 4 h + i mod 4.  It issues at 7.5 PFLOP/s of 4-bit products where the 16 x 16 one stops at 5.8.
template <int FA, int BYTE>
__device__ __forceinline__ v16f multiply32(const AFragment<FA> &a, int a_scale, const v8i &b, int b_scale, v16f c)
{
    if constexpr (FA == kE2M1) {
        return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a.v, b, c, kE2M1, kE2M1, BYTE, a_scale, BYTE, b_scale);
    } else {
        c = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a.small, b, c, kE4M3, kE2M1, BYTE, a_scale, BYTE, b_scale);
        return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a.large, b, c, kE4M3, kE2M1, BYTE, a_scale, BYTE, b_scale);
    }
}

// A 16-byte piece of row r of 32 rows of 64 bytes in LDS.  The 32 lanes of a half read one piece of 32 rows; of these, rows
// 0-3, 12-15, 20-23 and 24-27 go together, and the other sixteen: with this swap they are in all banks.
__device__ __forceinline__ int wide_place(int r, int q) { return r * 64 + ((q ^ ((r >> 2) & 3)) * 16); }

// Many queries and many columns: tiles of 256 queries by 256 stored rows, four wavefronts of 128 x 128 (4 x 4 fragments of
// 32 rows), one to a SIMD with 512 registers: twice the products per byte read from LDS of the kernel above.  Codes go
// from memory straight into a ring of R LDS buffers, one step of 128 columns each, scales four steps at a time (4 bytes of a
// row at a time touch its line in every step: 4096 x 32768 x 4096 365 us instead of 325).  A half-step of 64 columns reads the
// next one's fragments of stored rows while it multiplies its own, so that no wavefront meets a barrier without products to
// do; the last steps of a tile load the next one's first codes, which are on their way while scores leave.
// Long rows are bound by the products (4096 x 32768 x 4096: 325 us, 3.4 PFLOP/s; the instruction alone reaches 7.5 at the clock
// of a short loop, and the power of this one holds it near 1.7 GHz), short ones by the scores (2048 x 131072 x 768 to fp32:
// 235 us, 4.8 TB/s); 8-bit queries take every product twice (748 us, 2.9 PFLOP/s of both halves).
// Four steps and more, multiples of four stored rows, rows of scores that start on 64 bytes and have at most 2^23 of them, and
// scales that start on 4 bytes only.
template <int FA, int R, bool L2, typename T>
__global__ __launch_bounds__(256, 1) void mx_wide_kernel(ProductParams p, int row_tiles, int col_tiles, int per_xcd)
{
    constexpr int kHalves = FA == kE2M1 ? 1 : 2, kTile = 256, F = 4;
    constexpr int kABytes = kTile * 64 * kHalves, kBBytes = kTile * 64, kBuffer = kABytes + kBBytes;
    constexpr int kScaleBytes = 2 * kTile * 16;                       // of both sides, four steps
    constexpr int kLoads = 4 * kHalves + 4;                           // of codes, 1 KB each, per wavefront and step
    extern __shared__ __align__(16) uint8_t smem[];
    uint8_t *const scale_lds = smem + R * kBuffer;
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave >> 1, wn = wave & 1;
    const int steps = p.blocks >> 2;
    const int a_row_bytes = p.blocks * 16 * kHalves, b_row_bytes = p.blocks * 16;
    // Workgroup b runs on XCD b mod 8: each gets a contiguous run of tiles, eight query tiles high, and its workgroups take
    // them in turn, so that those at work at a time lie next to each other.
    const int end = min((int)(blockIdx.x & 7) * per_xcd + per_xcd, row_tiles * col_tiles);
    int id = (int)(blockIdx.x & 7) * per_xcd + (int)(blockIdx.x >> 3);
    if (id >= end) {
        return;
    }

    // LDS holds 16 rows of 64 bytes in 1 KB (wide_place); a wavefront loads runs wave, wave + 4, ... of either side, lane l
    // the piece that belongs at place l & 3 of row l >> 2.  Stored row 4 r + j of each 128 is row r of fragment j, so that
    // a lane ends up with four scores in a row; rows behind the last one repeat it.
    int64_t row0, col0;   // of the tile whose codes are loaded
    const uint8_t *a_base, *b_base, *a_scale_from, *b_scale_from;
    uint32_t a_from[4], b_from[4];
    auto set_tile = [&]() {
        int l = lane;
        asm volatile("" : "+v"(l));   // what follows from the lane alone is not kept in registers for the next tile
        const int fr = l >> 2, fq = (l & 3) ^ ((fr >> 2) & 3);
        const int band = id / (8 * col_tiles), in = id - band * 8 * col_tiles, high = min(8, row_tiles - band * 8);
        row0 = (int64_t)(band * 8 + in % high) * kTile;
        col0 = (int64_t)(in / high) * kTile;
        a_base = p.a_codes + row0 * a_row_bytes;
        b_base = p.b_codes + col0 * b_row_bytes;
        const int last_row = (int)min<int64_t>(kTile, p.m - row0) - 1, last_col = (int)min<int64_t>(kTile, p.n - col0) - 1;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            a_from[k] = (uint32_t)(min((wave + 4 * k) * 16 + fr, last_row) * a_row_bytes + fq * 16);
            const int run = wave + 4 * k;   // of 128 rows run >> 3, fragment (run >> 1) & 3, rows 16 (run & 1) ...
            const int row = (run >> 3) * 128 + ((run & 1) * 16 + fr) * 4 + ((run >> 1) & 3);
            b_from[k] = (uint32_t)(min(row, last_col) * b_row_bytes + fq * 16);
        }
        // rows of scales, 16 bytes each, in the order of the fragments' rows
        const int scale_run = wave * 2 + (l >> 5);   // 32 rows: of 128 rows scale_run >> 2, fragment scale_run & 3
        a_scale_from = p.a_scales + (row0 + min(wave * 64 + l, last_row)) * p.blocks;
        b_scale_from = p.b_scales + (col0 + min((scale_run >> 2) * 128 + (l & 31) * 4 + (scale_run & 3), last_col)) * p.blocks;
    };
    auto load_lds = [&](const uint8_t *from, uint8_t *to) {
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from,
                                         (__attribute__((address_space(3))) void *)to, 16, 0, 0);
    };
    // The first of the four steps whose scales come together; the last four of a row may overlap those before.
    auto first_of = [&](int step) { return min(step & ~3, steps - 4); };
    int loaded = 0, used = 0;   // place of the scales among the R - 1 that R - 1 steps in a row may need
    auto issue = [&](int step, uint8_t *ring, int k) {   // a quarter of the codes of a step, and four steps' scales
        if (k == 0 && (step & 3) == 0) {
            uint8_t *const to = scale_lds + loaded * kScaleBytes + wave * 1024;
            loaded = loaded == R - 2 ? 0 : loaded + 1;
            load_lds(a_scale_from + first_of(step) * 4, to);
            load_lds(b_scale_from + first_of(step) * 4, to + kTile * 16);
        }
        uint8_t *const to = ring + wave * 1024 + k * 4096;
#pragma unroll
        for (int half = 0; half < kHalves; half++) {
            load_lds(a_base + (step * kHalves + half) * 64 + a_from[k], to + half * (kTile * 64));
        }
        load_lds(b_base + step * 64 + b_from[k], to + kABytes);
    };

    v16f acc[F][F] = {};
    u4 a[2][2][kHalves], b[2][F];   // of two blocks of two query fragments; of two half-steps
    auto read_b = [&](const uint8_t *ring, int half, int j) {
        return *reinterpret_cast<const u4 *>(ring + kABytes + (wn * 4 + j) * 2048 + wide_place(r, half * 2 + h));
    };
    auto read_a = [&](const uint8_t *ring, int half, int i, u4 (&v)[kHalves]) {
        const uint8_t *const from = ring + (wm * 4 + i) * 2048;
        if constexpr (FA == kE2M1) {
            v[0] = *reinterpret_cast<const u4 *>(from + wide_place(r, half * 2 + h));
        } else {
            v[0] = *reinterpret_cast<const u4 *>(from + half * (kTile * 64) + wide_place(r, h));
            v[1] = *reinterpret_cast<const u4 *>(from + half * (kTile * 64) + wide_place(r, 2 + h));
        }
    };
    // scales of row r of a fragment: those of blocks h and 2 + h in bytes 0 and 2
    auto read_scales = [&](const uint8_t *of_step, int row) {
        return *reinterpret_cast<const uint32_t *>(of_step + (row + r) * 16);
    };
    int a_scale[F], b_scale[F];
    const int a_row = wm * 128, b_row = kTile + wn * 128;

    bool more = true, stores = false;
    int place = 0;   // in the ring
    auto one = [&](int step) {
        const uint8_t *const here = smem + place * kBuffer;
        uint8_t *const free = smem + (place == 0 ? R - 1 : place - 1) * kBuffer;
        place = place == R - 1 ? 0 : place + 1;
        const uint8_t *const after = smem + place * kBuffer;   // behind the last step: the first one of the next tile
        const int step_after = step + 1 == steps ? 0 : step + 1;
        if ((step_after & 3) == 0) {
            used = used == R - 2 ? 0 : used + 1;
        }
        const uint8_t *const scales_after = scale_lds + used * kScaleBytes + (step_after - first_of(step_after)) * 4;
        if (step + R - 1 == steps) {   // from here on the next tile's codes are loaded
            id += gridDim.x >> 3;
            more = id < end;
            if (more) {
                set_tile();
            }
        }
        const bool loads = step + R - 1 < steps || more;
        const int ahead = step + R - 1 < steps ? step + R - 1 : step + R - 1 - steps;
        // every wavefront is done with the step before: its place in the ring is free
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        auto half_step = [&](auto which_half) {
            constexpr int half = decltype(which_half)::value;
            const uint8_t *const next = half == 0 ? here : after;
            uint32_t w[2 * F];   // the next step's scales
#pragma unroll
            for (int i = 0; i < F; i += 2) {   // eight products at a time
                AFragment<FA> f;
                f.set(a[i >> 1][0]);
                acc[i][0] = multiply32<FA, half * 2>(f, a_scale[i], wide(b[half][0]), b_scale[0], acc[i][0]);
                // the reads for the next eight start behind the first of these, whose operands were waited for with all
                // others in flight, and have the time of the other seven
                asm volatile("" : "+a"(acc[i][0]) : : "memory");
                __builtin_amdgcn_sched_barrier(0);
                if (loads) {
                    issue(ahead, free, half * 2 + (i >> 1));
                }
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    read_a(i == 0 ? here : next, i == 0 ? half : half ^ 1, i == 0 ? 2 + k : k, a[(i >> 1) ^ 1][k]);
                    b[half ^ 1][i + k] = read_b(next, half ^ 1, i + k);
                }
                if constexpr (half == 1) {
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        w[i + k] = read_scales(scales_after, a_row + (i + k) * 32);
                        w[F + i + k] = read_scales(scales_after, b_row + (i + k) * 32);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    if (k == 1) {
                        f.set(a[i >> 1][1]);
                    }
#pragma unroll
                    for (int j = 1 - k; j < F; j++) {
                        acc[i + k][j] = multiply32<FA, half * 2>(f, a_scale[i + k], wide(b[half][j]), b_scale[j], acc[i + k][j]);
                    }
                }
                asm volatile(""
                             : "+a"(acc[i][1]), "+a"(acc[i][2]), "+a"(acc[i][3]), "+a"(acc[i + 1][0]), "+a"(acc[i + 1][1]),
                               "+a"(acc[i + 1][2]), "+a"(acc[i + 1][3])
                             :
                             : "memory");
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (half == 1) {
#pragma unroll
                for (int i = 0; i < F; i++) {
                    a_scale[i] = (int)(w[i] >> (8 * h));
                    b_scale[i] = (int)(w[F + i] >> (8 * h));
                }
            }
        };
        half_step(std::integral_constant<int, 0>());
        // the other half reads ahead from the next step: its codes have to be there, what was issued later (half of a step's
        // loads and R - 3 steps' before) may be on its way
        constexpr int kLater = (R - 3) * kLoads + kLoads / 2;
        if (loads && step < R - 2 && stores) {
            // behind these loads 64 stores of the last tile's scores and kLater loads were issued: at most 63 are left
            __builtin_amdgcn_s_waitcnt(0xcf7f);
        } else if (loads) {
            __builtin_amdgcn_s_waitcnt(0x0f70 | (kLater & 15) | (kLater >> 4) << 14);
        } else {
            __builtin_amdgcn_s_waitcnt(0x0f70);
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        half_step(std::integral_constant<int, 1>());
    };
    set_tile();
#pragma unroll
    for (int k = 0; k < R - 1; k++) {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            issue(k, smem + k * kBuffer, q);
        }
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int j = 0; j < F; j++) {
        b[0][j] = read_b(smem, 0, j);
        a_scale[j] = (int)(read_scales(scale_lds, a_row + j * 32) >> (8 * h));
        b_scale[j] = (int)(read_scales(scale_lds, b_row + j * 32) >> (8 * h));
    }
    read_a(smem, 0, 0, a[0][0]);
    read_a(smem, 0, 1, a[0][1]);
    for (;;) {
        const int64_t tile_row = row0, tile_col = col0;
#pragma unroll 1
        for (int step = 0; step < steps; step++) {
            one(step);
        }
        // the next tile's first codes are on their way while this one's scores leave
        const int64_t col = tile_col + wn * 128 + r * 4;
        stores = true;   // 64 of them, dropped ones among them
        // The norms of the wavefront's 128 queries, one a lane: a load among the stores would wait for those before it.
        float b_sqr[4] = {};
        int norms[2] = {};
        if constexpr (L2) {
            if (col < p.n) {
                load_run(p.b_sqr, col, p.n, b_sqr);
            }
            norms[0] = __float_as_int(p.a_sqr[min(tile_row + wm * 128 + lane, p.m - 1)]);
            norms[1] = __float_as_int(p.a_sqr[min(tile_row + wm * 128 + 64 + lane, p.m - 1)]);
        }
        // Stores with bounds of their own: what lies behind the last query or the last stored row is dropped, and no lane
        // is masked out (v_readlane takes norms from all of them).  Rows of at most 2^23 bytes keep offsets in 32 bits.
        const int64_t first = tile_row + wm * 128;
        const uint32_t up = (uint32_t)p.ld * (uint32_t)sizeof(T), rows = (uint32_t)max((int64_t)0, min((int64_t)128, p.m - first));
        const __amdgpu_buffer_rsrc_t out = __builtin_amdgcn_make_buffer_rsrc(
            static_cast<uint8_t *>(p.out) + min(first, p.m - 1) * up, 0, (int)(rows * up), 0x00027000);
        const uint32_t offset = col < p.n ? h * 4 * up + (uint32_t)col * (uint32_t)sizeof(T) : 0x80000000u;
        typedef T Scores __attribute__((ext_vector_type(4)));
        typedef uint32_t Words __attribute__((ext_vector_type(sizeof(T))));
#pragma unroll
        for (int i = 0; i < F; i++) {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                // one group of stores after the other: all scores at a time would not fit the registers that take them from
                // the accumulators, and what they displace would be waited for, with all codes on their way, in every step
                asm volatile(""
                             : "+a"(acc[i][0]), "+a"(acc[i][1]), "+a"(acc[i][2]), "+a"(acc[i][3]), "+v"(norms[0]), "+v"(norms[1])
                             :
                             : "memory");
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int at = i % 2 * 32 + k * 8 + e;
                    float a_sqr = 0.f;
                    if constexpr (L2) {
                        const int low = __builtin_amdgcn_readlane(norms[i / 2], at);
                        const int high = __builtin_amdgcn_readlane(norms[i / 2], at + 4);
                        a_sqr = __int_as_float(h ? high : low);
                    }
                    Scores v;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float g = acc[i][j][4 * k + e];
                        v[j] = (T)(L2 ? fmaf(g, -2.f, a_sqr + b_sqr[j]) : g);
                    }
                    const uint32_t to = offset + (uint32_t)(i * 32 + k * 8 + e) * up;
                    constexpr int kNonTemporal = 2;
                    if constexpr (sizeof(T) == 4) {
                        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(Words, v), out, to, 0, kNonTemporal);
                    } else {
                        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(Words, v), out, to, 0, kNonTemporal);
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < F; i++) {
#pragma unroll
            for (int j = 0; j < F; j++) {
                acc[i][j] = v16f{};
            }
        }
        if (!more) {
            return;
        }
    }
}

bool aligned(const void *p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

template <int FA>
size_t stream_lds(int64_t m, int pieces, int steps)
{
    return (size_t)steps * m * (FA == kE2M1 ? 64 : 128) + (((size_t)steps * m * 4 + 15) & ~(size_t)15) + 4 * pieces * (1024 + 64);
}

template <int FA, int MF, int NF, int U, typename T>
void launch_stream(const ProductParams &p, hipStream_t s)
{
    const int steps = (p.blocks + 3) / 4;
    const size_t lds = stream_lds<FA>(p.m, NF * U, steps);
    const int64_t tiles = (p.n + NF * 16 - 1) / (NF * 16);
    const void *kern = reinterpret_cast<const void *>(mx_stream_kernel<FA, MF, NF, U, T>);
    require_dynamic_lds(kern, lds);
    const dim3 grid((unsigned)std::min((tiles + 3) / 4, resident_workgroups(kern, 256, lds)));
    hipLaunchKernelGGL((mx_stream_kernel<FA, MF, NF, U, T>), grid, dim3(256), lds, s, p, steps, tiles);
    check_launch();
}

template <int FA, int WM, int WN, int MF, int U, typename T>
void launch_tiles(const ProductParams &p, hipStream_t s)
{
    const int64_t row_tiles = (p.m + WM * MF * 16 - 1) / (WM * MF * 16), col_tiles = (p.n + WN * 64 - 1) / (WN * 64);
    const int64_t per_xcd = (row_tiles * col_tiles + 7) / 8;
    IXA_REQUIRE(per_xcd * 8 * (WM * WN * 64) <= 0xffffffffll, kErrInvalidParam, "mx_product: %ld x %ld scores in one call", (long)p.m,
                (long)p.n);
    hipLaunchKernelGGL((mx_tile_kernel<FA, WM, WN, MF, U, T>), dim3((unsigned)per_xcd * 8), dim3(WM * WN * 64), 0, s, p,
                       (int)row_tiles, (int)col_tiles, (int)per_xcd);
    check_launch();
}

template <int FA, bool L2, typename T>
void launch_wide(const ProductParams &p, hipStream_t s)
{
    constexpr int R = FA == kE2M1 ? 4 : 3;
    constexpr size_t lds = R * (256 * 64 * (FA == kE2M1 ? 2 : 3)) + (R - 1) * 512 * 16;
    const int64_t row_tiles = (p.m + 255) / 256, col_tiles = (p.n + 255) / 256;
    const int64_t per_xcd = (row_tiles * col_tiles + 7) / 8;
    const void *kern = reinterpret_cast<const void *>(mx_wide_kernel<FA, R, L2, T>);
    require_dynamic_lds(kern, lds);
    IXA_REQUIRE(per_xcd <= 0x0fffffff, kErrInvalidParam, "mx_product: %ld x %ld scores in one call", (long)p.m, (long)p.n);
    // a multiple of 8: the workgroups of an XCD share its run of tiles
    const int64_t grid = std::min(per_xcd, std::max<int64_t>(1, resident_workgroups(kern, 256, lds) / 8)) * 8;
    hipLaunchKernelGGL((mx_wide_kernel<FA, R, L2, T>), dim3((unsigned)grid), dim3(256), lds, s, p, (int)row_tiles, (int)col_tiles,
                       (int)per_xcd);
    check_launch();
}

template <int FA, typename T>
void launch_type(const ProductParams &p, hipStream_t s)
{
    const int steps = (p.blocks + 3) / 4;
    const int mf = p.m <= 16 ? 1 : p.m <= 32 ? 2 : 4;
    // Half a CU's LDS, so that two workgroups share it, is the line; it is right for 33 ... 64 queries in part only and for fewer
    // not at all.  8-bit queries, the whole LDS and the tiles below: 64 x 20000 x 1024 18.5 us and 15.7, 64 x 500000 x 1024 121 and 143,
    // 16 x 30000 x 4096 23.5 and 46, 16 x 200000 x 4096 111 and 226, 8 x 100000 x 8192 128 and 230; in 4 bits 64 x 200000 x 4096 163
    // and 155.
    if (p.m <= 64 && stream_lds<FA>(p.m, 4, steps) <= 80 * 1024) {
        // Up to 2048 tiles of 16 stored rows (eight wavefronts per CU) such tiles, four steps at a time; else tiles of 64 rows,
        // or, for up to 16 queries with more than one step, of 32 rows and 128 bytes of each at a time: with 64 bytes, and the
        // many wavefronts that few queries leave room for, the two visits to a line of memory are too far apart.
        // 1 x 20000 x 4096: 16 rows 9.9 us, 32 rows 12.5, 64 rows 20.6; 1 x 1M x 1536: 150, 154, 199; 64 x 1M x 768: 253, 171,
        // 145; 32 x 1M x 512: 96, 76, 72; 1 x 1M x 128: 26.8, 17.8, 15.5.  Around the line, 16 rows and the other: 32 x 30000 x 512
        // 6.9 and 7.7, 60000 10.3 and 8.5; 64 x 30000 x 768 14.0 and 13.9, 60000 22.0 and 15.4; 64 x 30000 x 128 6.6 and 7.1, 100000
        // 13.5 and 8.6; 1 x 30000 x 1536 8.3 and 8.0, 60000 12.6 and 10.9, 100000 17.3 and 18.2.
        const bool narrow = p.n <= 16 * 2048;
        if (mf == 1) {
            if (narrow) {
                launch_stream<FA, 1, 1, 4, T>(p, s);
            } else if (steps == 1) {
                launch_stream<FA, 1, 4, 1, T>(p, s);
            } else {
                launch_stream<FA, 1, 2, 2, T>(p, s);
            }
        } else if (mf == 2) {
            narrow ? launch_stream<FA, 2, 1, 4, T>(p, s) : launch_stream<FA, 2, 4, 1, T>(p, s);
        } else {
            narrow ? launch_stream<FA, 4, 1, 4, T>(p, s) : launch_stream<FA, 4, 4, 1, T>(p, s);
        }
        return;
    }
    // Wide tiles where at most a fifth of their queries do not exist and either every CU gets one (2048 x 131072 x 768: 235 us,
    // the tiles below 277; 1024 x 32768 x 768: 42 and 48; with 256 of them, 1024 x 16384 x 768, both 24) or there are many
    // columns (2048 x 4096 x 4096: 39 us against 48; with few columns and 128 tiles the others are ahead, 1024 x 8192 x 1024: 20
    // against 18).
    const int64_t wide_rows = (p.m + 255) / 256, wide_tiles = wide_rows * ((p.n + 255) / 256);
    if (p.blocks % 4 == 0 && p.blocks >= 16 && p.n % 4 == 0 && p.lines && p.ld <= (1 << 23) / (int)sizeof(T) &&
        aligned(p.a_scales, 4) && aligned(p.b_scales, 4) && wide_rows * 256 * 4 <= p.m * 5 &&
        wide_tiles >= (p.blocks >= 64 ? 128 : 256)) {
        p.metric == kMetricL2 ? launch_wide<FA, true, T>(p, s) : launch_wide<FA, false, T>(p, s);
        return;
    }
    const int64_t tiles = ((p.m + 127) / 128) * ((p.n + 255) / 256);
    // Tiles of 128 x 256, of 64 x 256 where that would be less than three for two CUs (300 x 20000 x 1030: 25 us, 128 x 256 31;
    // 1024 x 8192 x 1024: 26 and 34; with 391 of them, 100 x 100003 x 200, 14.8 and 12.9), and of 256 x 256 and two steps at
    // a time for 4-bit queries with two such tiles and more per CU in rows of 512 columns and more (1024 x 60001 x 2016: 124 us,
    // 128 x 256 154; 2048 x 100001 x 768: 288 and 312; shorter rows 2048 x 131072 x 200: 282 and 234; fewer tiles
    // 1000 x 20001 x 4096: 100 and 97; with 8-bit queries 4096 x 32768 x 2080: 513 and 498).  Half of a tile of 128 and more has
    // no queries where there are 64: with 8-bit ones 64 x 256 would be ahead (64 x 500000 x 1024 100 us against 143, 16 x 200000 x
    // 4096 151 and 226, 32 x 100000 x 16384 295 and 451), with 4-bit ones not (64 x 200000 x 4096 200 and 155).
    if (tiles < 384) {
        launch_tiles<FA, 1, 4, 4, 1, T>(p, s);
        return;
    }
    if constexpr (FA == kE2M1) {
        if (p.blocks >= 16 && wide_rows * 256 * 4 <= p.m * 5 && wide_tiles >= 512) {
            launch_tiles<FA, 2, 4, 8, 2, T>(p, s);
            return;
        }
    }
    launch_tiles<FA, 1, 4, 8, 1, T>(p, s);
}

template <int FA>
void launch(const ProductParams &p, int out_type, hipStream_t s)
{
    if (out_type == kTypeF32) {
        launch_type<FA, float>(p, s);
    } else if (out_type == kTypeF16) {
        launch_type<FA, _Float16>(p, s);
    } else {
        launch_type<FA, __bf16>(p, s);
    }
}

}  // namespace

void op_mx_product(const uint8_t *a_codes, const uint8_t *a_scales, int a_format, int64_t m, const uint8_t *b_codes,
                   const uint8_t *b_scales, int64_t n, int d, int metric, const float *a_sqr, const float *b_sqr,
                   int out_type, void *out, int64_t ld, hipStream_t s)
{
    const bool none = m == 0 || n == 0;   // needs no buffers: the address of an empty array is null
    IXA_REQUIRE((a_codes && a_scales && b_codes && b_scales && out) || none, kErrInvalidParam,
                "operator buffers can not be nullptr.");
    IXA_REQUIRE(a_format == kFormatMxFp8 || a_format == kFormatMxFp4, kErrInvalidParam,
                "mx_product: unsupported code format %d", a_format);
    IXA_REQUIRE(out_type >= kTypeF32 && out_type <= kTypeBF16, kErrInvalidParam, "mx_product: unsupported element type %d",
                out_type);
    IXA_REQUIRE(m >= 0 && m <= 0x7fffffff && n >= 0 && n <= 0x7fffffff && d >= 1 && d <= kMaxCodeDim, kErrInvalidParam,
                "mx_product: rows %ld x %ld (< 2^31), dims %d (1 ... %d)", (long)m, (long)n, d, kMaxCodeDim);
    IXA_REQUIRE(ld >= n && ld <= (int64_t)1 << 40, kErrInvalidParam, "mx_product: rows of %ld scores in steps of %ld", (long)n,
                (long)ld);
    IXA_REQUIRE(metric == kMetricL2 || metric == kMetricInnerProduct, kErrInvalidParam, "Unsupported metric type");
    IXA_REQUIRE(metric != kMetricL2 || (a_sqr && b_sqr) || none, kErrInvalidParam,
                "mx_product: squared distances need the squared norms of both sides");
    IXA_REQUIRE(aligned(a_codes, 16) && aligned(b_codes, 16) && aligned(out, out_type == kTypeF32 ? 4 : 2) &&
                    aligned(a_sqr, 4) && aligned(b_sqr, 4),
                kErrInvalidParam, "mx_product: codes have to start on 16 bytes, norms and scores on their elements");
    if (none) {
        return;
    }
    int device;
    check_answer(hipGetDevice(&device));   // what is asked of a kernel before its launch needs one
    const ProductParams p{a_codes, a_scales, b_codes, b_scales, a_sqr, b_sqr, m, n, ld, mx_blocks(d), metric, out,
                          aligned(out, 64) && ld * (out_type == kTypeF32 ? 4 : 2) % 64 == 0};
    if (a_format == kFormatMxFp4) {
        launch<kE2M1>(p, out_type, s);
    } else {
        launch<kE4M3>(p, out_type, s);
    }
}

}  // namespace ixa
