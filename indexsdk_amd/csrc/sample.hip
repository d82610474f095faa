// Columns drawn from rows of scores.  For a row x_0 ... x_(n-1) with temperature T, top-k k, top-p p and min-p m:
//   w_i = exp((x_i - max x) / T);  T <= 0: only the best column counts
//   the columns in the order of falling scores, equal ones in the order of columns, are cut to the first k, then to the fewest
//   whose weights reach p of those of all that are left, then to those with w_i >= m
//   a draw with the random number u is the first column, in the order of columns, at which the running sum of the weights that are
//   left passes u times their total
// Scores of -infinity and NaN are columns that are not there; beside +infinity everything else is.
//
// Weights below 2^-960 count as 0.  Every decision is one about sums of weights next to a border, so weights and sums are held in 64
// bits: an exponential is 13 instructions of the same rate as in 32.
//
// One workgroup per row reads it once (a few, each a part, where there are few rows).  The largest scores of some of its columns
// give a bound that a few hundred scores of the row reach; these go to a list in LDS, and while k or p or m keep no more than what
// is in the list, all else happens there: sorted by score, cut, and drawn from.  Rows without filters are drawn from by the sums
// of their segments.  Everything else (flat rows whose p keeps thousands, large k) reads the row twice again: a histogram of counts
// finds the bins around the cut, whose columns go through the list while the weights above them are added up; where these are more than it
// holds, sums over parts of their range of scores find the part with the cut, which is divided again.
//
// What bounds it: one read of the scores where k cuts (1024 rows of 100003 bf16, four draws each: 74 us, 2.8 TB/s), the exponentials in 64 bits where
// all of a row's are needed (without filters 105 us, with top-p 134 us, with settings that leave every fifth row flat 190 us), and
// for a few rows the steps of one workgroup that wait for each other (a row of 32768 fp32 under all filters: 13 us).
#include "power_of_two.h"
#include "row_access.h"
#include "scores.h"

#include <algorithm>
#include <type_traits>

namespace ixa {

namespace {

constexpr int kList = 2048;         // candidates of a row
constexpr int kPartList = 1024;     // and of a part of one
constexpr int kBins = 4096;         // of a histogram of counts
constexpr int kDigits = 1024, kAround = 32, kMoves = 3;
constexpr int kSegments = 512;      // at most: parts of a row whose sums are kept
constexpr int kBlock = 512;         // columns that a wavefront reads at a time
constexpr int kTurns = 4;           // such blocks in flight
constexpr int kSample = 2;          // blocks of each wavefront that the bound comes from
constexpr int kSmall = 64;          // entries that are sorted by exchanges, or by counting
constexpr int kReach = 350;         // candidates that p is hoped to be content with
constexpr int kFew = 256;           // candidates that every wavefront holds in registers, four per lane
constexpr int kOneWave = 32;        // draws up to which one wavefront makes them all
constexpr int kMaxParts = 16, kPartThreads = 512;
constexpr double kNothing = -960.0;    // logarithms of weights that count as 0; in sums over whole rows as 2^-960

// What a workgroup finds out about its part of a row.
struct PartHead {
    uint32_t top, low, reference, bound;     // low: the lowest of the columns that the bound comes from
    uint32_t listed, fine;
    uint32_t high, unused;                   // high: a bound that about kFew / 2 scores reach
};

struct SampleParams {
    const void *scores;
    const float *temperature, *top_p, *min_p, *uniform;
    const int32_t *top_k;
    int64_t *labels;
    float *probs;
    int64_t ld, n;
    int draws, parts;
    PartHead *heads;         // [rows][parts]
    uint64_t *lists;         // [rows][parts][kPartList]
    double *segments;        // [rows][kSegments]
};

// Scores in an order of integers; 0: a column that is not there.
__device__ __forceinline__ uint32_t key_of(float x)
{
    const uint32_t b = __float_as_uint(x + 0.f);     // -0 is 0
    const uint32_t k = (int)b < 0 ? ~b : b | 0x80000000u;
    return x > -__builtin_inff() ? k : 0u;
}
__device__ __forceinline__ float score_of(uint32_t k) { return __uint_as_float((int)k < 0 ? k & 0x7fffffffu : ~k); }

// The lane's that CTRL names within the rows of ROWS, 0 where there is none.
template <int CTRL, int ROWS>
__device__ __forceinline__ double shifted(double v)
{
    const int2 w = __builtin_bit_cast(int2, v);
    return __builtin_bit_cast(double, make_int2(__builtin_amdgcn_update_dpp(0, w.x, CTRL, ROWS, 0xf, false),
                                                __builtin_amdgcn_update_dpp(0, w.y, CTRL, ROWS, 0xf, false)));
}
// Running sums over the wavefront, inclusive: within 16 lanes, then the last of a row to the next, and of two to the next two.
__device__ __forceinline__ double wave_scan(double v)
{
    v += shifted<0x111, 0xf>(v);
    v += shifted<0x112, 0xf>(v);
    v += shifted<0x114, 0xf>(v);
    v += shifted<0x118, 0xf>(v);
    v += shifted<0x142, 0xa>(v);
    v += shifted<0x143, 0xc>(v);
    return v;
}

__device__ __forceinline__ uint64_t larger(uint64_t a, uint64_t b) { return a > b ? a : b; }

struct SampleShared {
    uint64_t list[kList];           // score's key above the column's complement
    union {
        double sum[kList];          // of the list's weights; a histogram is of no more use by then
        unsigned long long tally[2 * kDigits];
        uint32_t count[kBins];
        struct {
            uint64_t sorted[kFew];
            uint32_t rank[kFew];
        };
    };
    double segment[kSegments];
    uint64_t best[kFew];            // the highest of a longer list
    uint32_t places[kDigits];       // of parts of the list
    double box[2][16];
    uint32_t tops[64];
    uint32_t ubox[16], lows[16];
    uint32_t lengths[16];           // of the wavefronts' lists
    uint32_t listed, found, found_best;
    double before;
};

// The workgroup's; by this name everywhere, so that the compiler sees LDS in every access.
__shared__ SampleShared lds;

// What is drawn from: columns of at least `least` (an order of score and column as in the list) with weights of at least min_p.
struct Row {
    double scale;      // log2(e) / T
    float top;         // the largest score, or another that weights are relative to
    double from;       // the same in 64 bits, where infinity is a number that all others are far below
    double min_p;
    uint64_t least;
    __device__ __forceinline__ Row(double s, float t, double m) : scale(s), top(t), from(t), min_p(m), least(0)
    {
        if (t == __builtin_inff()) {
            from = 1e300;
            scale = fmax(s, 1.0);
        }
    }
    __device__ __forceinline__ double logarithm(float x) const { return (fmin((double)x, 1e300) - from) * scale; }
    // of a score that is there; what counts as 0 is 0, or in a sum of many 2^-960
    __device__ __forceinline__ double weight(float x) const
    {
        const double t = logarithm(x);
        return t > kNothing ? power_of_two(t) : 0.0;
    }
    __device__ __forceinline__ double addend(float x) const { return power_of_two(fmax(logarithm(x), kNothing)); }
    __device__ __forceinline__ uint64_t place(uint32_t key, uint32_t column) const { return (uint64_t)key << 32 | ~column; }
    // of a column: 0 where it is cut off
    __device__ __forceinline__ double kept(float x, uint32_t column) const
    {
        const uint32_t key = key_of(x);
        if (key == 0 || place(key, column) < least) {
            return 0.0;
        }
        const double w = weight(x);
        return w >= min_p ? w : 0.0;
    }
};

template <typename T, int NT>
struct Sampler {
    static constexpr int kWaves = NT / 64;
    const T *row;
    const int64_t n;
    const int tid, lane, wave;

    __device__ __forceinline__ Eight<T> load(int64_t block) const
    {
        const int64_t at = block * kBlock + lane * kEight;
        Eight<T> e;
        const int count = (int)min((int64_t)kEight, max((int64_t)0, n - at));
        e.load(row + (count ? at : 0), count, (T)-__builtin_inff());
        return e;
    }
    __device__ __forceinline__ int64_t blocks() const { return (n + kBlock - 1) / kBlock; }
    __device__ __forceinline__ uint32_t column(int64_t block, int i) const { return (uint32_t)(block * kBlock + lane * kEight + i); }

    // f(block, scores) over blocks from ... to - 1, TURNS of them in flight
    template <int TURNS, typename F>
    __device__ __forceinline__ void run(int64_t from, int64_t to, F f) const
    {
        for (int64_t b = from; b < to; b += TURNS) {
            Eight<T> e[TURNS];
#pragma unroll
            for (int u = 0; u < TURNS; u++) {
                e[u] = load(min(b + u, to - 1));
            }
#pragma unroll
            for (int u = 0; u < TURNS; u++) {
                if (u == 0 || b + u < to) {
                    float x[kEight];
#pragma unroll
                    for (int i = 0; i < kEight; i++) {
                        x[i] = (float)e[u].v[i];
                    }
                    f(b + u, x);
                }
            }
        }
    }
    // over those of a wavefront's part of the row
    template <typename F>
    __device__ __forceinline__ void each(F f) const
    {
        run<2>(blocks() * wave / kWaves, blocks() * (wave + 1) / kWaves, f);
    }

    __device__ __forceinline__ double block_sum(double v) const
    {
        v = over_wave(v, [](double a, double b) { return a + b; });
        __syncthreads();
        if (lane == 0) {
            lds.box[0][wave] = v;
        }
        __syncthreads();
        v = 0.0;
        for (int w = 0; w < kWaves; w++) {
            v += lds.box[0][w];
        }
        return v;
    }
    __device__ __forceinline__ uint32_t block_max(uint32_t v) const
    {
        v = over_wave(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
        __syncthreads();
        if (lane == 0) {
            lds.ubox[wave] = v;
        }
        __syncthreads();
        v = 0;
        for (int w = 0; w < kWaves; w++) {
            v = max(v, lds.ubox[w]);
        }
        return v;
    }

    // Running sums (inclusive) of a[0 ... m), in place.
    __device__ __forceinline__ void scan(double *a, int m) const
    {
        const int per = (m + NT - 1) / NT, from = tid * per;
        double sum = 0.0;
        for (int i = from; i < min(from + per, m); i++) {
            sum += a[i];
        }
        const double upto = wave_scan(sum);
        __syncthreads();
        if (lane == 63) {
            lds.box[1][wave] = upto;
        }
        __syncthreads();
        const double before_me = __shfl_up(upto, 1);
        double run = lane == 0 ? 0.0 : before_me;
        for (int w = 0; w < wave; w++) {
            run += lds.box[1][w];
        }
        for (int i = from; i < min(from + per, m); i++) {
            run += a[i];
            a[i] = run;
        }
        __syncthreads();
    }

    // list[0 ... m) in falling order (m <= kList): by 1024 parts of the range of the keys' upper halves, and in each part by counting
    // the larger ones.
    __device__ __forceinline__ void sort(int m) const
    {
        constexpr int kOwn = (kList + NT - 1) / NT, kPer = kDigits / NT > 0 ? kDigits / NT : 1;
        if (m <= kSmall) {
            return sort_by_exchange(m);
        }
        uint64_t e[kOwn];
        uint32_t top = 0, low = 0;
#pragma unroll
        for (int u = 0; u < kOwn; u++) {
            const int i = u * NT + tid;
            e[u] = i < m ? lds.list[i] : 0;
            top = max(top, (uint32_t)(e[u] >> 32));
            low = max(low, i < m ? ~(uint32_t)(e[u] >> 32) : 0u);
        }
        top = block_max(top);
        low = ~block_max(low);
        const int shift = max(0, 32 - __builtin_clz((top - low) | 1u) - 10);
        auto part_of = [&](uint64_t v) { return (top - (uint32_t)(v >> 32)) >> shift; };
        for (int i = tid; i < kDigits; i += NT) {
            lds.places[i] = 0;
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kOwn; u++) {
            if (u * NT + tid < m) {
                atomicAdd(&lds.places[part_of(e[u])], 1u);
            }
        }
        __syncthreads();
        uint32_t n_of[kPer], sum = 0, most = 0;
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            n_of[i] = tid * kPer + i < kDigits ? lds.places[tid * kPer + i] : 0u;
            sum += n_of[i];
            most = max(most, n_of[i]);
        }
        if (block_max(most) > (uint32_t)kSmall) {
            return sort_by_exchange(m);      // many equal ones, or few far from the others
        }
        const double upto = wave_scan((double)sum);
        if (lane == 63) {
            lds.box[1][wave] = upto;
        }
        __syncthreads();
        uint32_t start = (uint32_t)upto - sum;
        for (int w = 0; w < wave; w++) {
            start += (uint32_t)lds.box[1][w];
        }
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            if (tid * kPer + i < kDigits) {
                lds.places[tid * kPer + i] = start;
            }
            start += n_of[i];
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kOwn; u++) {
            if (u * NT + tid < m) {
                lds.list[atomicAdd(&lds.places[part_of(e[u])], 1u)] = e[u];     // now where the next part starts
            }
        }
        __syncthreads();
        uint32_t to[kOwn];
#pragma unroll
        for (int u = 0; u < kOwn; u++) {
            const uint32_t part = part_of(e[u]);
            const bool there = u * NT + tid < m;
            const int from = there && part > 0 ? (int)lds.places[part - 1] : 0, end = there ? (int)lds.places[part] : 0;
            to[u] = (uint32_t)from;
            for (int i = from; i < end; i++) {
                to[u] += lds.list[i] > e[u] ? 1u : 0u;
            }
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kOwn; u++) {
            if (u * NT + tid < m) {
                lds.list[to[u]] = e[u];
            }
        }
        __syncthreads();
    }
    __device__ __forceinline__ void sort_by_exchange(int m) const
    {
        int size = 2;
        while (size < m) {
            size <<= 1;
        }
        for (int i = m + tid; i < size; i += NT) {
            lds.list[i] = 0;
        }
        // Exchanges over up to 64 entries stay among the 128 that one wavefront has, whose accesses to LDS happen in their order.
        __syncthreads();
        for (int k = 2; k <= size; k <<= 1) {
            for (int j = k >> 1; j > 0; j >>= 1) {
                for (int t = tid; t < size / 2; t += NT) {
                    const int a = (t & ~(j - 1)) * 2 + (t & (j - 1)), b = a + j;
                    const uint64_t x = lds.list[a], y = lds.list[b];
                    if ((x < y) == ((a & k) == 0)) {
                        lds.list[a] = y;
                        lds.list[b] = x;
                    }
                }
                if (j >= 128 || (j == 1 && k >= 128)) {
                    __syncthreads();
                } else {
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    __builtin_amdgcn_wave_barrier();
                }
            }
        }
        __syncthreads();
    }

    // How many of the list's m entries, in their order, it takes for their running sums (in `sum`) to reach `target`; m + 1: all are
    // less.
    __device__ __forceinline__ int reach(double target, int m) const
    {
        int lo = 0, hi = m;    // the first that is not less
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (lds.sum[mid] < target) {
                lo = mid + 1;
            } else {
                hi = mid;
            }
        }
        return lo + 1;
    }

    // sums of `value(x, column)` over segments of `per` blocks
    template <typename F>
    __device__ __forceinline__ double segment_sums(int64_t per, F value) const
    {
        const int segments = (int)((blocks() + per - 1) / per);
        for (int g = wave; g < segments; g += kWaves) {
            double v = 0.0;
            run<2>(g * per, min(blocks(), (g + 1) * per), [&](int64_t b, const float(&x)[kEight]) {
#pragma unroll
                for (int i = 0; i < kEight; i++) {
                    v += value(x[i], column(b, i));
                }
            });
            v = over_wave(v, [](double a, double b) { return a + b; });
            if (lane == 0) {
                lds.segment[g] = v;
            }
        }
        return segment_total(segments);
    }
    __device__ __forceinline__ double segment_total(int segments) const
    {
        __syncthreads();
        double v = 0.0;
        for (int g = tid; g < segments; g += NT) {
            v += lds.segment[g];
        }
        return block_sum(v);
    }
    // A wavefront's search: the first column at which the running sum of `value` passes `target`, and its value; the last one with
    // a value if rounding hides it.
    template <typename F>
    __device__ __forceinline__ void locate(int64_t per, double target, F value, int64_t &at, double &what) const
    {
        const int segments = (int)((blocks() + per - 1) / per);
        double before = 0.0;
        // the first segment that passes the target, or the last with a value: a run of them per lane
        double sum = 0.0, run = 0.0;
        const int each_lane = (segments + 63) / 64, from = lane * each_lane, to = min(from + each_lane, segments);
        for (int i = from; i < to; i++) {
            sum += lds.segment[i];
        }
        const double upto_lane = wave_scan(sum);
        const uint64_t passes = __ballot(upto_lane > target && sum > 0.0), some = __ballot(sum > 0.0);
        const int l = passes ? __builtin_ctzll(passes) : some ? 63 - __builtin_clzll(some) : 0;
        const double before_lane = __shfl_up(upto_lane, 1);
        run = l == 0 ? 0.0 : __shfl(before_lane, l);
        int g = l * each_lane;
        for (int i = g; i < min((l + 1) * each_lane, segments); i++) {      // the same in every lane
            const double v = lds.segment[i];
            if (v > 0.0) {
                g = i;
                before = run;
                if (run + v > target) {
                    break;
                }
            }
            run += v;
        }
        run = before;
        at = -1;
        what = 0.0;
        bool done = false;
        // a segment whose sum is of nothing but weights that count as 0 is passed over
#pragma unroll 1
        for (; at < 0 && g < segments; g++) {
            this->template run<2>(g * per, min(blocks(), (g + 1) * per), [&](int64_t b, const float(&x)[kEight]) {
                if (done) {
                    return;
                }
                double v[kEight], sum = 0.0;
#pragma unroll
                for (int i = 0; i < kEight; i++) {
                    v[i] = value(x[i], column(b, i));
                    sum += v[i];
                }
                const double upto = wave_scan(sum), before_me = __shfl_up(upto, 1);
                double mine = run + (lane == 0 ? 0.0 : before_me);
                int hit = -1, last = -1;
                double hit_v = 0.0, last_v = 0.0;
#pragma unroll
                for (int i = 0; i < kEight; i++) {
                    mine += v[i];
                    if (v[i] > 0.0) {
                        if (hit < 0 && mine > target) {
                            hit = i;
                            hit_v = v[i];
                        }
                        last = i;
                        last_v = v[i];
                    }
                }
                const uint64_t hits = __ballot(hit >= 0), lasts = __ballot(last >= 0);
                if (hits) {
                    const int l = __builtin_ctzll(hits);
                    at = b * kBlock + l * kEight + __shfl(hit, l);
                    what = __shfl(hit_v, l);
                    done = true;
                } else if (lasts) {
                    const int l = 63 - __builtin_clzll(lasts);
                    at = b * kBlock + l * kEight + __shfl(last, l);
                    what = __shfl(last_v, l);
                }
                run += __shfl(upto, 63);
            });
        }
    }

    // Columns with scores in [low, high] go to the list, the sums of the weights above to the segments; their total, and the
    // number of columns above.
    __device__ __forceinline__ double collect(int64_t per, const Row &r, float low, float high, double &above) const
    {
        if (tid == 0) {
            lds.listed = 0;
        }
        __syncthreads();
        int mine = 0;
        const double total = segment_sums(per, [&](float x, uint32_t c) {
            const double w = r.addend(x);
            if (x >= low && x <= high) {
                const uint32_t at = atomicAdd(&lds.listed, 1u);
                if (at < kList) {
                    lds.list[at] = (uint64_t)key_of(x) << 32 | ~c;
                }
            }
            mine += x > high ? 1 : 0;
            return x > high ? w : 0.0;
        });
        above = block_sum((double)mine);
        return total;
    }

    // The first of BINS bins at which the running sum of value(bin), with `before` in front of the first, reaches `goal`, or the last
    // with a value; `before` becomes the sum in front of it.
    template <int BINS, typename F>
    __device__ __forceinline__ int cross(F value, double goal, double &before)
    {
        constexpr int kPer = (BINS + NT - 1) / NT;
        __syncthreads();
        double v[kPer], sum = 0.0;
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            v[i] = tid * kPer + i < BINS ? value(tid * kPer + i) : 0.0;
            sum += v[i];
        }
        const double upto = wave_scan(sum);
        if (lane == 63) {
            lds.box[1][wave] = upto;
        }
        if (tid == 0) {
            lds.found = 0;
            lds.before = before;
        }
        __syncthreads();
        double run = before;
        for (int w = 0; w < wave; w++) {
            run += lds.box[1][w];
        }
        const double before_me = __shfl_up(upto, 1);
        run += lane == 0 ? 0.0 : before_me;
        int at = -1, last = -1;
        double in_front = 0.0, in_front_of_last = 0.0;
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            if (v[i] > 0.0) {
                if (at < 0 && run + v[i] >= goal) {
                    at = tid * kPer + i;
                    in_front = run;
                }
                last = tid * kPer + i;
                in_front_of_last = run;
            }
            run += v[i];
        }
        // the lowest bin that reaches it, else the highest with a value
        const uint32_t mine = at >= 0 ? 0x80000000u | (uint32_t)(BINS - at) : last >= 0 ? (uint32_t)last + 1u : 0u;
        const uint32_t best = block_max(mine);
        if (best && mine == best) {
            lds.found = (uint32_t)(at >= 0 ? at : last);
            lds.before = at >= 0 ? in_front : in_front_of_last;
        }
        __syncthreads();
        before = lds.before;
        const int found = (int)lds.found;
        __syncthreads();
        return found;
    }

    // The place (score and column) of the last column kept: the count or (by_mass) the sum of weights up to it reaches `goal`.  Where
    // `summed`, the sums of segments of what is kept, min_p apart, are in lds.segment afterwards, their total in `total`.
    __device__ __forceinline__ uint64_t find_cut(const Row &r, float low, double goal, bool by_mass, double whole, bool &summed, double &total)
    {
        // Counts in bins of equal width in the scores, for sums down to weights of 2^-64; a bin's weights are its count times that of
        // its middle.  That is only where to look: sums in 64 bits decide.
        const float width = r.top - low, range = by_mass ? fminf(width, (float)(64.0 / r.scale)) : width;
        const float unit = range > 0.f && range < __builtin_inff() ? (float)kBins / range : 0.f;
        auto bin_of = [&](float x) {
            const float d = (r.top - x) * unit;
            return d < (float)(kBins - 1) ? (int)d : kBins - 1;     // also where 0 meets infinity
        };
        const int64_t per = segment_size();
        __syncthreads();
        for (int i = tid; i < kBins; i += NT) {
            lds.count[i] = 0;
        }
        __syncthreads();
        each([&](int64_t, const float(&x)[kEight]) {
#pragma unroll
            for (int i = 0; i < kEight; i++) {
                if (x[i] > -__builtin_inff()) {
                    atomicAdd(&lds.count[bin_of(x[i])], 1u);
                }
            }
        });
        double before = 0.0;
        const float step_down = unit > 0.f ? (float)r.scale / unit : 0.f;
        auto about = [&](int b) {
            const double c = (double)lds.count[b];
            return by_mass ? c * (double)__builtin_amdgcn_exp2f(((float)b + 0.5f) * -step_down) : c;
        };
        __syncthreads();
        // What these are off by comes from the few columns with large weights: as much is added to the goal as all are off by.
        double off = 0.0;
        if (whole > 0.0) {
            for (int b = tid; b < kBins; b += NT) {
                off += about(b);
            }
            off = block_sum(off) - whole;
        }
        int bin = cross<kBins>(about, goal + off, before);
        // The bin and its neighbours, as long as the list is likely to hold them: where the counts were off by little, the cut still
        // is among these.  That scores next to a threshold may fall to either side of the bins' edge does not matter.
        int first = bin, last = bin;
        const uint32_t likely = whole > 0.0 || !by_mass ? kFew : kList / 2;
        uint32_t room = lds.count[bin] < likely ? likely - lds.count[bin] : 0u;
        for (int i = 1; i <= kAround; i++) {
            const uint32_t up = bin - i >= 0 ? lds.count[bin - i] : 0u, down = bin + i < kBins ? lds.count[bin + i] : 0u;
            if (up + down > room) {
                break;
            }
            room -= up + down;
            first = max(bin - i, 0);
            last = min(bin + i, kBins - 1);
        }
        __syncthreads();
        const float inf = __builtin_inff(), least = -3.402823466e+38f, wide = unit > 0.f ? kAround / unit : inf;
        float high = first == 0 || !(unit > 0.f) ? inf : r.top - (float)first / unit;
        float bottom = last >= kBins - 1 || !(unit > 0.f) ? least : r.top - (float)(last + 1) / unit;
        int m, way = 0;
        bool lost = false;
        for (int moves = 0;; moves++) {
            double above;
            total = collect(per, r, bottom, high, above);
            before = by_mass ? total : above;
            m = (int)min(lds.listed, (uint32_t)kList + 1u);
            double upto = __builtin_inf();     // of more than the list holds: not known, and not needed
            if (m <= kList) {
                sort(m);
                for (int i = tid; i < m; i += NT) {
                    lds.sum[i] = r.weight(score_of((uint32_t)(lds.list[i] >> 32)));
                }
                __syncthreads();
                if (by_mass) {
                    scan(lds.sum, m);
                }
                upto = before + (m == 0 ? 0.0 : by_mass ? lds.sum[m - 1] : (double)m);
            }
            const bool under = before >= goal && high < inf && way <= 0, over = upto < goal && bottom > least && way >= 0;
            __syncthreads();
            if (!under && !over) {
                break;
            }
            if (moves == kMoves) {      // scores so far off, or so near to each other, that bins say little: all of them
                lost = true;
                bottom = least;
                high = inf;
                before = 0.0;
                break;
            }
            if (under) {
                way = -1;
                bottom = score_of(key_of(high) + 1);
                high = fmaxf(fminf(high + wide, inf), bottom);
            } else {
                way = 1;
                high = score_of(key_of(bottom) - 1);
                bottom = fminf(fmaxf(bottom - wide, least), high);
            }
        }
        if (lost || m > kList) {
            summed = false;
            return find_tie(r, bottom, high, before, goal, by_mass);
        }
        const double left = goal - before;
        int take = by_mass ? reach(left, m) : left < (double)m ? (int)left : m;
        take = min(take, m);
        take = max(take, min(1, m));
        // an empty list: everything above it is kept, or everything that is there
        const uint64_t place = m > 0 ? lds.list[take - 1] : before >= goal ? (uint64_t)(key_of(high) + 1) << 32 : 0;
        // to the segments, as integers: their sums do not depend on an order.  Up to kList weights of at most the first one's size.
        const int64_t columns = per * kBlock;
        const int segments = (int)((blocks() + per - 1) / per);
        const double largest = m > 0 ? r.weight(score_of((uint32_t)(lds.list[0] >> 32))) : 0.0;
        const double fixed = largest > 0.0 ? 0x1p51 / largest : 0.0;
        __syncthreads();       // the list's sums have been read: the tallies take their place
        for (int g = tid; g < segments; g += NT) {
            lds.tally[g] = 0;
        }
        __syncthreads();
        for (int i = tid; i < take; i += NT) {
            const uint64_t e = lds.list[i];
            atomicAdd(&lds.tally[(int64_t)(~(uint32_t)e) / columns],
                      (unsigned long long)__builtin_rint(r.weight(score_of((uint32_t)(e >> 32))) * fixed));
        }
        __syncthreads();
        for (int g = tid; g < segments; g += NT) {
            lds.segment[g] += (double)lds.tally[g] * (largest * 0x1p-51);
        }
        total = segment_total(segments);
        summed = true;
        return place;
    }

    // The same where [low, high] holds too many for the list, `before` above it: in up to kDigits parts, of which the one with the cut is
    // looked at again, until it is one key; among equal scores by column.  Where the cut is not among these, all up to `high` are gone through.
    // Sums of parts are integers, which do not depend on an order: weights relative to the part's highest, in units of 2^-62 and two
    // words.  So that none is small next to that, a range of weights wider than 2^8 goes by their logarithms first; then by keys.
    __device__ __forceinline__ uint64_t find_tie(const Row &r, float low, float high, double before, double goal, bool by_mass)
    {
        const int64_t per = segment_size();
        const float inf = __builtin_inff(), least = -3.402823466e+38f;
        uint32_t *const ends = reinterpret_cast<uint32_t *>(lds.list);     // each part's highest key, and the complements of the lowest ones
        uint32_t top, bottom;
        double run, w, ties;
        auto tie = [&](float v, uint32_t) { return key_of(v) == top ? 1.0 : 0.0; };
#pragma unroll 1
        for (bool again = true; again;) {
            again = false;
            uint32_t most = 0, fewest = 0;
            each([&](int64_t, const float(&x)[kEight]) {
#pragma unroll
                for (int i = 0; i < kEight; i++) {
                    const uint32_t key = x[i] >= low && x[i] <= high ? key_of(x[i]) : 0u;
                    most = max(most, key);
                    fewest = max(fewest, key ? ~key : 0u);
                }
            });
            top = block_max(most);
            bottom = ~block_max(fewest);
            run = before;
            if (top == 0 || (by_mass && r.logarithm(score_of(top)) <= kNothing)) {      // nothing here, or of no weight
                return high < inf ? (uint64_t)(key_of(high) + 1) << 32 : 0;
            }
            bool first = low > least;
#pragma unroll 1
            while (top > bottom) {
                const double from = by_mass ? r.logarithm(score_of(top)) : 0.0;
                const double range = by_mass ? from - fmax(r.logarithm(score_of(bottom)), kNothing) : 0.0;
                const bool by_size = range > 8.0;      // once: a part of them is narrower than 1
                const double width = range / kDigits, unit = by_size ? kDigits / range : 0.0;
                const int shift = max(0, 32 - __builtin_clz(top - bottom) - 10);
                auto highest = [&](int part) { return by_size ? from - part * width : from; };
                __syncthreads();
                for (int i = tid; i < kDigits; i += NT) {
                    lds.tally[i] = lds.tally[kDigits + i] = 0;
                    ends[i] = ends[kDigits + i] = 0;
                }
                __syncthreads();
                each([&](int64_t, const float(&x)[kEight]) {
#pragma unroll
                    for (int i = 0; i < kEight; i++) {
                        const uint32_t key = key_of(x[i]);
                        if (key < bottom || key > top) {
                            continue;
                        }
                        if (!by_mass) {
                            atomicAdd(&lds.tally[(top - key) >> shift], 1ull);
                            continue;
                        }
                        const double t = r.logarithm(x[i]);
                        if (t <= kNothing) {
                            continue;
                        }
                        const int part = by_size ? min(kDigits - 1, (int)((from - t) * unit)) : (int)((top - key) >> shift);
                        const double v = power_of_two(t - highest(part)) * 0x1p31;
                        const uint32_t whole = (uint32_t)v;
                        atomicAdd(&lds.tally[part], (unsigned long long)whole);
                        atomicAdd(&lds.tally[kDigits + part], (unsigned long long)(uint32_t)((v - whole) * 0x1p31));
                        if (by_size) {
                            atomicMax(&ends[part], key);
                            atomicMax(&ends[kDigits + part], ~key);
                        }
                    }
                });
                auto sum = [&](int part) {
                    return by_mass ? ((double)lds.tally[part] * 0x1p-31 + (double)lds.tally[kDigits + part] * 0x1p-62) *
                                         power_of_two(highest(part))
                                   : (double)lds.tally[part];
                };
                const int part = cross<kDigits>(sum, goal, run);
                if (first && run + sum(part) < goal) {
                    again = true;
                    break;
                }
                first = false;
                if (by_size) {
                    top = ends[part];
                    bottom = ~ends[kDigits + part];
                } else {
                    const uint32_t size = (1u << shift) - 1u;
                    top -= (uint32_t)part << shift;
                    bottom = top - bottom > size ? top - size : bottom;
                }
            }
            if (!again) {
                w = by_mass ? r.weight(score_of(top)) : 1.0;
                ties = segment_sums(per, tie);
                again = first && run + ties * w < goal;
            }
            low = least;
        }
        const double take = fmax(1.0, fmin(ties, w > 0.0 ? ceil((goal - run) / w) : ties));
        int64_t at;
        double one;
        locate(per, take - 0.5, tie, at, one);
        __syncthreads();
        return r.place(top, (uint32_t)at);
    }

    __device__ __forceinline__ int64_t segment_size() const
    {
        // four blocks where every wavefront gets that many; a row of no columns has no segment, but what is divided by is not 0
        return max(max((int64_t)1, min((int64_t)kTurns, (blocks() + kWaves - 1) / kWaves)), (blocks() + kSegments - 1) / kSegments);
    }
};

// A row's settings, and what follows from them.
struct Settings {
    double scale, top_p, min_p;
    int64_t count;
    bool by_count, by_mass, filtered, need_mass;
    __device__ __forceinline__ Settings(const SampleParams &p, int64_t row)
    {
        float temperature = p.temperature ? p.temperature[row] : 1.f;
        count = p.top_k ? p.top_k[row] : 0;
        top_p = p.top_p ? (double)p.top_p[row] : 1.0;
        min_p = p.min_p ? (double)p.min_p[row] : 0.0;
        count = count <= 0 ? p.n : min(p.n, count);
        if (!(temperature > 0.f)) {
            temperature = 1.f;
            count = 1;
        }
        scale = 1.44269504088896340735992468 / (double)temperature;
        by_count = count < p.n;
        by_mass = top_p < 1.0;     // not a number: no
        min_p = min_p > 0.0 ? fmin(min_p, 1.0) : 0.0;
        filtered = by_count || by_mass || min_p > 0.0;
        need_mass = !by_count;
    }
};

// A part of a row, once: its largest score, the sums of weights relative to a reference (`total`, and segment by segment), and the
// list.
template <typename T, int NT>
__device__ __forceinline__ PartHead scan_part(const Sampler<T, NT> &k, const Settings &set, int part, int parts, double &total)
{
    constexpr int kWaves = NT / 64, kOwn = kEight * kSample;
    SampleShared &s = lds;
    const int lane = k.lane, wave = k.wave;
    const int64_t per = k.segment_size(), all = (k.blocks() + per - 1) / per;
    const int g0 = (int)(all * part / parts), g1 = (int)(all * (part + 1) / parts);
    const int64_t b0 = g0 * per, b1 = min(k.blocks(), g1 * per), mine = b1 - b0, columns = min(k.n - b0 * kBlock, mine * kBlock);
    const float inf = __builtin_inff();

    // The largest of 64 groups of lanes in some of the columns: sixteen per lane, or all there are.
    constexpr int kLanes = kWaves;
    float lane_top = -inf, lane_low = inf;
    const int each = (int)min((int64_t)kOwn, (columns + NT - 1) / NT);
    // of columns that many of the sampled ones of which are wanted fewer are sampled: every group would have one
    const int seen = set.by_count ? kOwn : (int)min((int64_t)each, 1 + columns * 100 / ((int64_t)kReach / parts * NT));
    auto see = [&](float x, bool counts) {
        lane_top = counts ? fmaxf(lane_top, x) : lane_top;
        lane_low = x > -inf ? fminf(lane_low, x) : lane_low;
    };
    if (columns > NT * kOwn) {
        const int64_t first = b0 + mine * wave / kWaves;
#pragma unroll
        for (int u = 0; u < kSample; u++) {
            const Eight<T> e = k.load(first + u);
#pragma unroll
            for (int i = 0; i < kEight; i++) {
                see((float)e.v[i], u * kEight + i < seen);
            }
        }
    } else if (columns > 0) {
#pragma unroll
        for (int i = 0; i < kOwn; i++) {
            see((float)k.row[b0 * kBlock + min((int64_t)k.tid * each + min(i, each - 1), columns - 1)], i < seen);
        }
    }
    const int flip = (int)0x80000000;
    const int group_top = over_lanes<kLanes>((int)key_of(lane_top) ^ flip, [](int a, int b) { return max(a, b); });
    if (lane % kLanes == 0) {
        s.tops[wave * (64 / kLanes) + lane / kLanes] = (uint32_t)(group_top ^ flip);
    }
    __syncthreads();
    const uint32_t tops = s.tops[lane];
    const uint32_t sample_top = over_wave(tops, [](uint32_t a, uint32_t b) { return max(a, b); });
    const float reference = score_of(sample_top);
    // A bound that so many of the sampled columns reach that all of them have what is kept, but for one time in thousands: as
    // many more than expected as three deviations.
    PartHead h{0, 0, sample_top, 0xffffffffu, 0, 1, 0xffffffffu, 0};
    if (set.filtered && sample_top) {
        const float share = columns > NT * kOwn ? (float)(NT * min(seen, kOwn)) / (float)columns : fminf(1.f, (float)seen / (float)each);
        // the highest bound that one of so many of 64 groups of the sampled columns reaches as hold one of `reach` columns at least
        auto bound_for = [&](float reach) {
            const int groups = (int)fminf(60.f, 64.f * (1.f - __expf(-reach / 64.f)) + 1.5f);
            uint32_t b = 0;
#pragma unroll 1
            for (int bit = 31; bit >= 16; bit--) {
                const uint32_t at = b | 1u << bit;
                b = __popcll(__ballot(tops >= at)) >= groups ? at : b;
            }
            return max(b, 1u);
        };
        if (columns <= kFew) {
            h.bound = 1;      // everything that is there
        } else if (set.by_count) {
            const float wanted = (float)min(set.count, (int64_t)kList) / (float)parts * share;
            const float reach = wanted + 3.f * __builtin_amdgcn_sqrtf(wanted) + 4.f;
            h.bound = reach <= 130.f ? bound_for(reach) : h.bound;
        } else {
            // what a sum takes is not known ahead: a few hundred, and the highest of them first
            h.bound = bound_for(fminf((float)kReach / (float)parts * share + 4.f, 130.f));
            h.high = bound_for(fminf(140.f / (float)parts * share + 1.f, 100.f));
        }
    }
    const float bound = h.bound == 0xffffffffu ? __builtin_nanf("") : h.bound == 1 ? -3.402823466e+38f : score_of(h.bound);
    const bool sums = set.need_mass;
    constexpr int kOwnList = kList / kWaves;      // every wavefront has a list of its own
    uint64_t *const list = s.list + wave * kOwnList;
    int listed = 0;
    float top = -inf;
    double sum = 0.0;
    for (int g = g0 + wave; g < g1; g += kWaves) {
        double v = 0.0;
        k.template run<kTurns>(g * per, min(b1, (g + 1) * per), [&](int64_t b, const float(&x)[kEight]) {
            float most = x[0];
#pragma unroll
            for (int i = 1; i < kEight; i++) {
                most = fmaxf(most, x[i]);
            }
            top = fmaxf(top, most);
            if (sums) {
#pragma unroll
                for (int i = 0; i < kEight; i++) {
                    v += power_of_two(fmax(((double)x[i] - (double)reference) * set.scale, kNothing));
                }
            }
            if (__ballot(most >= bound)) {
#pragma unroll
                for (int i = 0; i < kEight; i++) {
                    const uint64_t hits = __ballot(x[i] >= bound);
                    if (hits) {
                        const int at = listed + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(hits >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)hits, 0));
                        if (x[i] >= bound && at < kOwnList) {
                            list[at] = (uint64_t)key_of(x[i]) << 32 | ~k.column(b, i);
                        }
                        listed += __popcll(hits);
                    }
                }
            }
        });
        if (sums) {
            v = over_wave(v, [](double a, double b) { return a + b; });
            sum += v;
            if (lane == 0) {
                s.segment[g] = v;
            }
        }
    }
    const uint32_t wave_top = over_wave(key_of(top), [](uint32_t a, uint32_t b) { return max(a, b); });
    const uint32_t wave_low = over_wave(key_of(-lane_low), [](uint32_t a, uint32_t b) { return max(a, b); });
    if (lane == 0) {
        s.box[0][wave] = sum;
        s.ubox[wave] = wave_top;
        s.lows[wave] = wave_low;
        s.lengths[wave] = (uint32_t)listed;
    }
    __syncthreads();
    total = 0.0;
    uint32_t together = 0, mine_from = 0;
    bool fits = true;
#pragma unroll 4
    for (int w = 0; w < kWaves; w++) {
        total += s.box[0][w];
        h.top = max(h.top, s.ubox[w]);
        h.low = max(h.low, s.lows[w]);
        mine_from += w < wave ? s.lengths[w] : 0u;
        together += s.lengths[w];
        fits = fits && s.lengths[w] <= (uint32_t)kOwnList;
    }
    h.listed = h.bound == 0xffffffffu || !fits || (parts > 1 && together > (uint32_t)kPartList) ? 0xffffffffu : together;
    if (h.listed != 0xffffffffu) {
        // one list of all
        uint64_t mine_of[(kOwnList + 63) / 64];
#pragma unroll
        for (int i = 0; i < (kOwnList + 63) / 64; i++) {
            mine_of[i] = i * 64 + lane < listed ? list[i * 64 + lane] : 0;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < (kOwnList + 63) / 64; i++) {
            if (i * 64 + lane < listed) {
                s.list[mine_from + i * 64 + lane] = mine_of[i];
            }
        }
    }
    __syncthreads();
    return h;
}

// The draws from a row whose candidates, at most kFew, are in the list, if these hold all that is kept: they are put in the order of
// their scores and, those that are kept, in that of their columns, by how many come before each; cuts and draws are ballots over what
// every wavefront holds in registers.
template <typename T, int NT, typename U>
__device__ __forceinline__ bool finish_few(const Sampler<T, NT> &k, const SampleParams &p, const Settings &set, const Row &r,
                                           const uint64_t *list, int m, bool complete, double total, int64_t *labels, float *probs, U draw_number)
{
    constexpr int kWaves = NT / 64, kParts = NT / kFew, kOf = kFew / 64;
    SampleShared &s = lds;
    const int tid = k.tid, lane = k.lane, wave = k.wave, own = tid % kFew, part = tid / kFew;
    if (tid < kFew) {
        s.rank[tid] = 0;
    }
    __syncthreads();
    if (own < m) {
        const uint64_t mine = list[own];
        int before = 0;
#pragma unroll 4
        for (int i = part; i < m; i += kParts) {
            before += list[i] > mine ? 1 : 0;
        }
        if (kParts > 1) {
            atomicAdd(&s.rank[own], (uint32_t)before);
        } else {
            s.rank[own] = (uint32_t)before;
        }
    }
    __syncthreads();
    if (tid < m) {
        s.sorted[s.rank[tid]] = list[tid];
    }
    __syncthreads();
    // One wavefront goes on (all of them at the same would take turns); the others wait for its word, and for many draws of theirs.
    double w[kOf], upto[kOf], run = 0.0, all = 0.0;
    int take = m;
    if (wave == 0) {
#pragma unroll
        for (int c = 0; c < kOf; c++) {
            const int e = c * 64 + lane;
            w[c] = upto[c] = 0.0;
            if (c * 64 < m) {
                w[c] = e < m ? r.weight(score_of((uint32_t)(s.sorted[e] >> 32))) : 0.0;
                upto[c] = run + wave_scan(w[c]);
                run = __shfl(upto[c], 63);
            }
        }
        auto how_many = [&](int size, auto is) {
            int count = 0;
#pragma unroll
            for (int c = 0; c < kOf; c++) {
                count += __popcll(__ballot(c * 64 + lane < size && is(c)));
            }
            return count;
        };
        auto sum_upto = [&](int size) {     // of the first `size` entries
            double v = 0.0;
#pragma unroll
            for (int c = 0; c < kOf; c++) {
                v = (size - 1) / 64 == c ? __shfl(upto[c], (size - 1) % 64) : v;
            }
            return v;
        };
        bool cut = complete;               // whether the list holds all that is kept
        if (set.by_count) {
            cut = cut || m >= set.count;
            take = (int)min((int64_t)m, set.count);
        }
        if (set.by_mass && (cut || !set.by_count)) {
            // of the sum of all that is left, which the list has or the whole row
            const double goal = set.top_p * (cut ? sum_upto(take) : total);
            const int need = how_many(take, [&](int c) { return upto[c] < goal; }) + 1;
            cut = cut || need <= take;
            take = min(take, need);
        }
        if (set.min_p > 0.0 && !(set.by_count && !cut)) {
            const int above = how_many(m, [&](int c) { return w[c] >= set.min_p; });
            cut = cut || above < m;
            take = min(take, above);
        }
        take = max(take, 1);
        if (cut) {
            all = sum_upto(take);
            // by column: how many of those that are kept come before each
#pragma unroll
            for (int c = 0; c < kOf; c++) {
                const int e = c * 64 + lane;
                if (c * 64 < take) {
                    const uint64_t mine = s.sorted[min(e, kFew - 1)];
                    int before = 0;
#pragma unroll 4
                    for (int i = 0; i < take; i++) {
                        before += (uint32_t)s.sorted[i] > (uint32_t)mine ? 1 : 0;
                    }
                    if (e < take) {
                        s.list[before] = mine;
                        s.segment[before] = w[c];
                    }
                }
            }
        }
        if (lane == 0) {
            s.found = cut ? (uint32_t)take : 0u;
            s.before = all;
        }
    }
    __syncthreads();
    take = (int)s.found;
    if (take == 0) {
        return false;
    }
    if (wave > 0 && p.draws <= kOneWave) {
        return true;
    }
    all = s.before;
    run = 0.0;
#pragma unroll
    for (int c = 0; c < kOf; c++) {
        const int e = c * 64 + lane;
        w[c] = upto[c] = 0.0;
        if (c * 64 < take) {
            w[c] = e < take ? s.segment[e] : 0.0;
            upto[c] = run + wave_scan(w[c]);
            run = __shfl(upto[c], 63);
        }
    }
    const int step = p.draws <= kOneWave ? 1 : kWaves;
    for (int d = wave; d < p.draws; d += step) {
        const double target = draw_number(d) * all;
        int at = 0;       // the first that passes it, or the last with a weight if rounding hides that
#pragma unroll
        for (int c = kOf - 1; c >= 0; c--) {
            const uint64_t some = __ballot(w[c] > 0.0);
            at = at == 0 && some ? c * 64 + 63 - __builtin_clzll(some) : at;
        }
#pragma unroll
        for (int c = kOf - 1; c >= 0; c--) {
            const uint64_t passes = __ballot(w[c] > 0.0 && upto[c] > target);
            at = passes ? c * 64 + __builtin_ctzll(passes) : at;
        }
        if (lane == 0) {
            labels[d] = (int64_t)(~(uint32_t)s.list[at]);
            if (probs) {
                probs[d] = (float)(s.segment[at] / all);
            }
        }
    }
    return true;
}

// The draws from a row whose list and sums are in LDS; `total`: of the row's weights relative to its largest score, or without filters
// to the reference.
template <typename T, int NT>
__device__ __forceinline__ void finish_row(Sampler<T, NT> &k, const SampleParams &p, const Settings &set, int64_t row,
                                           const PartHead &h, double total)
{
    constexpr int kWaves = NT / 64;
    SampleShared &s = lds;
    const int tid = k.tid, lane = k.lane, wave = k.wave;
    int64_t *const labels = p.labels + row * p.draws;
    float *const probs = p.probs ? p.probs + row * p.draws : nullptr;
    const float *const uniform = p.uniform + row * p.draws;
    if (h.top == 0) {
        for (int d = tid; d < p.draws; d += NT) {
            labels[d] = -1;
            if (probs) {
                probs[d] = 0.f;
            }
        }
        return;
    }
    const int64_t per = k.segment_size(), count = set.count;
    Row r(set.scale, score_of(set.filtered || !h.fine ? h.top : h.reference), set.min_p);
    if (!set.filtered && h.fine) {
        // weights count as 0 by what they are next to those of the best, not of the reference: scores of at most `border` are cut off
        const double border = (double)score_of(h.top) + kNothing / set.scale;
        const float nearest = (float)border;
        r.least = (uint64_t)min(key_of(nearest) + ((double)nearest > border ? 0u : 1u), h.top) << 32;
    }
    if (set.need_mass && !h.fine) {
        total = k.segment_sums(per, [&](float x, uint32_t) { return key_of(x) ? r.weight(x) : 0.0; });
    }
    auto draw_number = [&](int d) {
        const float u = uniform[d];
        return (double)(u > 0.f ? fminf(u, 0x1.fffffep-1f) : 0.f);
    };
    if (set.filtered) {
        const bool complete = h.bound == 1;      // every column that is there is in the list
        const int m = h.listed <= kList ? (int)h.listed : 0;
        bool hopeless = false;      // the whole list is short of what p takes
        if (m > kFew && set.by_mass && !set.by_count && !complete && set.min_p == 0.0) {
            double sum = 0.0;
            for (int i = tid; i < m; i += NT) {
                sum += r.weight(score_of((uint32_t)(s.list[i] >> 32)));
            }
            hopeless = k.block_sum(sum) < 0.999 * set.top_p * total;
        }
        // All candidates, or the highest of them, if they are few.
        int high = m;
        if (m > kFew && !hopeless && h.high != 0xffffffffu) {
            if (tid == 0) {
                s.found_best = 0;
            }
            __syncthreads();
            for (int i = tid; i < m; i += NT) {
                if ((uint32_t)(s.list[i] >> 32) >= h.high) {
                    const uint32_t at = atomicAdd(&s.found_best, 1u);      // in any order: they are put in theirs
                    if (at < kFew) {
                        s.best[at] = s.list[i];
                    }
                }
            }
            __syncthreads();
            high = (int)s.found_best;
        }
        if (!hopeless && high > 0 && high <= kFew &&
            finish_few(k, p, set, r, high < m ? s.best : s.list, high, complete && high == m, total, labels, probs, draw_number)) {
            return;
        }
        if (m > kFew && !hopeless) {
            int take = m;
            k.sort(m);
            for (int i = tid; i < m; i += NT) {
                s.sum[i] = r.weight(score_of((uint32_t)(s.list[i] >> 32)));
            }
            __syncthreads();
            k.scan(s.sum, m);
            bool cut = complete;
            if (set.by_count) {
                cut = cut || m >= count;
                take = (int)min((int64_t)m, count);
            }
            if (set.by_mass && (cut || !set.by_count)) {
                const int need = k.reach(set.top_p * (cut ? s.sum[take - 1] : total), take);
                cut = cut || need <= take;
                take = min(take, need);
            }
            if (set.min_p > 0.0 && !(set.by_count && !cut)) {
                int above = 0, below = m;      // weights fall along the list
                while (above < below) {
                    const int mid = (above + below) >> 1;
                    if (r.weight(score_of((uint32_t)(s.list[mid] >> 32))) >= set.min_p) {
                        above = mid + 1;
                    } else {
                        below = mid;
                    }
                }
                cut = cut || above < m;
                take = min(take, above);
            }
            take = max(take, 1);
            __syncthreads();
            if (cut) {
                // by columns: the complement falls as they rise
                for (int i = tid; i < take; i += NT) {
                    const uint64_t e = s.list[i];
                    s.list[i] = e << 32 | e >> 32;
                }
                __syncthreads();
                k.sort(take);
                for (int i = tid; i < take; i += NT) {
                    s.sum[i] = r.weight(score_of((uint32_t)s.list[i]));
                }
                __syncthreads();
                k.scan(s.sum, take);
                const double whole = s.sum[take - 1];
                for (int d = tid; d < p.draws; d += NT) {
                    const double target = draw_number(d) * whole;
                    int lo = 0, hi = take - 1;      // the first that passes it
                    while (lo < hi) {
                        const int mid = (lo + hi) >> 1;
                        if (s.sum[mid] > target) {
                            hi = mid;
                        } else {
                            lo = mid + 1;
                        }
                    }
                    labels[d] = (int64_t)(~(uint32_t)(s.list[lo] >> 32));
                    if (probs) {
                        probs[d] = (float)(r.weight(score_of((uint32_t)s.list[lo])) / whole);
                    }
                }
                return;
            }
        }
        __syncthreads();
        // the row again
        const float low = -score_of(h.low);
        double sum = total;
        bool summed = false;
#pragma unroll 1
        for (int mass = 0; mass < 2; mass++) {
            if (mass == 0 ? !set.by_count : !set.by_mass) {
                continue;
            }
            if (mass && set.by_count && !summed) {
                // the sum up to the cut by its columns
                sum = k.segment_sums(per, [&](float x, uint32_t c) { return key_of(x) && r.place(key_of(x), c) >= r.least ? r.weight(x) : 0.0; });
            }
            const uint64_t least = k.find_cut(r, low, mass ? set.top_p * sum : (double)count, mass, mass && !set.by_count ? total : 0.0, summed,
                                             sum);
            summed = summed && least >= r.least;
            r.least = larger(r.least, least);
        }
        // where min_p cuts more than the others the sums are not those of what is kept
        if (summed && (set.min_p == 0.0 || (r.least >> 32 && r.weight(score_of((uint32_t)(r.least >> 32))) >= set.min_p))) {
            total = sum;
        } else {
            total = k.segment_sums(per, [&](float x, uint32_t c) { return r.kept(x, c); });
        }
    }
    // by the sums of segments
    auto value = [&](float x, uint32_t c) { return r.kept(x, c); };
    for (int d = wave; d < p.draws; d += kWaves) {
        int64_t at;
        double w;
        k.locate(per, draw_number(d) * total, value, at, w);
        if (lane == 0) {
            labels[d] = at;
            if (probs) {
                probs[d] = (float)(w / total);
            }
        }
    }
}

template <typename T, int NT>
__device__ __forceinline__ Sampler<T, NT> sampler(const SampleParams &p, int64_t row)
{
    return Sampler<T, NT>{static_cast<const T *>(p.scores) + row * p.ld, p.n, (int)threadIdx.x, (int)threadIdx.x & 63,
                          __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6)};
}

// What a sum relative to `reference` is multiplied by to be one relative to `top`; 0: it can not be, exponentials were out of range.
__device__ __forceinline__ double unit_of(float reference, float top, double scale)
{
    const double t = ((double)reference - (double)top) * scale;
    return reference == top && top < __builtin_inff() ? 1.0 : t > kNothing ? power_of_two(t) : 0.0;
}

// Two workgroups of 512 threads share a CU, with 128 registers each and about 20 spilled, behind the loop over the row: 1024 rows of 100003
// bf16 with settings of their own take 207 us, 258 with 158 registers, none spilled and one workgroup per CU.
template <typename T, int NT>
__global__ __launch_bounds__(NT, NT == 256 ? 3 : 4) void sample_kernel(SampleParams p)
{
    const int64_t row = blockIdx.x;
    Sampler<T, NT> k = sampler<T, NT>(p, row);
    const Settings set(p, row);
    double total;
    PartHead h = scan_part(k, set, 0, 1, total);
    if (set.need_mass) {
        const double unit = h.reference ? unit_of(score_of(h.reference), score_of(h.top), set.scale) : 0.0;
        h.fine = unit > 0.0;
        total *= set.filtered ? unit : 1.0;
    }
    finish_row(k, p, set, row, h, total);
}

// A part of a row per workgroup, and what it found out.
template <typename T>
__global__ __launch_bounds__(kPartThreads, 4) void sample_part_kernel(SampleParams p)
{
    SampleShared &s = lds;
    const int64_t row = blockIdx.x / p.parts;
    const int part = (int)(blockIdx.x - row * p.parts);
    const Sampler<T, kPartThreads> k = sampler<T, kPartThreads>(p, row);
    const Settings set(p, row);
    double total;
    const PartHead h = scan_part(k, set, part, p.parts, total);
    if (k.tid == 0) {
        p.heads[blockIdx.x] = h;
    }
    if (h.listed <= kPartList) {
        for (int i = k.tid; i < (int)h.listed; i += kPartThreads) {
            p.lists[(int64_t)blockIdx.x * kPartList + i] = s.list[i];
        }
    }
    if (set.need_mass) {
        const int64_t per = k.segment_size(), all = (k.blocks() + per - 1) / per;
        for (int g = (int)(all * part / p.parts) + k.tid; g < (int)(all * (part + 1) / p.parts); g += kPartThreads) {
            p.segments[row * kSegments + g] = s.segment[g];
        }
    }
}

// The parts of a row, joined: the highest of their bounds is one that all lists go down to.
template <typename T>
__global__ __launch_bounds__(kPartThreads, 4) void sample_join_kernel(SampleParams p)
{
    SampleShared &s = lds;
    const int64_t row = blockIdx.x;
    Sampler<T, kPartThreads> k = sampler<T, kPartThreads>(p, row);
    const Settings set(p, row);
    PartHead all{0, 0, 0, 0, 0, 1, 0, 0};
    bool listed = true;
    for (int i = 0; i < p.parts; i++) {
        const PartHead h = p.heads[row * p.parts + i];
        if (h.top) {
            all.top = max(all.top, h.top);
            all.low = max(all.low, h.low);
            all.bound = max(all.bound, h.bound);
            all.high = max(all.high, h.high);
            listed = listed && h.listed <= kPartList;
        }
    }
    all.bound = max(all.bound, 1u);
    all.reference = all.top;
    if (k.tid == 0) {
        s.listed = 0;
    }
    __syncthreads();
    const float top = score_of(all.top);
    const int64_t per = k.segment_size(), segments = (k.blocks() + per - 1) / per;
    for (int i = 0; i < p.parts; i++) {
        const PartHead h = p.heads[row * p.parts + i];
        if (listed && h.top) {
            for (int e = k.tid; e < (int)h.listed; e += kPartThreads) {
                const uint64_t v = p.lists[(row * p.parts + i) * kPartList + e];
                if ((uint32_t)(v >> 32) >= all.bound) {
                    const uint32_t at = atomicAdd(&s.listed, 1u);
                    if (at < kList) {
                        s.list[at] = v;
                    }
                }
            }
        }
        if (set.need_mass) {
            const double unit = !h.top ? 1.0 : h.reference ? unit_of(score_of(h.reference), top, set.scale) : 0.0;
            for (int g = (int)(segments * i / p.parts) + k.tid; g < (int)(segments * (i + 1) / p.parts); g += kPartThreads) {
                const double v = h.top ? p.segments[row * kSegments + g] : 0.0;
                // what does not come out as a sum is found out again
                s.segment[g] = unit > 0.0 ? v * unit : __builtin_nan("");
            }
        }
    }
    __syncthreads();
    all.listed = listed ? s.listed : 0xffffffffu;
    double total = 0.0;
    if (set.need_mass && all.top) {
        total = k.segment_total((int)segments);
        all.fine = total == total;
    }
    finish_row(k, p, set, row, all, total);
}

// Parts of each row where there are few rows: as many as give every CU two workgroups, of 16384 columns at least.  Rows of 131072 fp32
// scores under top-p: one takes 26 us, 40 as a whole; 64 take 46 us, 60 as whole rows; 256 would take 64 us, 61 as whole rows.
int parts_of(int64_t rows, int64_t n)
{
    if (rows == 0 || rows > 128 || n < 65536) {
        return 1;
    }
    return (int)std::min<int64_t>({kMaxParts, std::max<int64_t>(2, 512 / rows), n / 16384});
}

}  // namespace

int64_t sample_workspace(int64_t rows, int64_t n)
{
    check_scores("sample", rows, n);
    const int64_t parts = parts_of(rows, n);
    return parts > 1 ? rows * (parts * (int64_t)(sizeof(PartHead) + kPartList * 8) + kSegments * 8) : 0;
}

void op_sample(const void *scores, int64_t ld, int type, int64_t rows, int64_t n, const float *temperature, const int32_t *top_k,
               const float *top_p, const float *min_p, const float *uniform, int draws, int64_t *labels, float *probs,
               void *workspace, int64_t workspace_bytes, hipStream_t s)
{
    check_type("sample", type);
    const int64_t need = sample_workspace(rows, n);
    check_row_buffer("sample", scores, ld, type, rows, n);
    IXA_REQUIRE(draws >= 0 && draws <= 1 << 20, kErrInvalidParam, "sample: %d draws (0 ... 2^20)", draws);
    const bool none = rows == 0 || draws == 0;
    IXA_REQUIRE((uniform && labels) || none, kErrInvalidParam, "operator buffers can not be nullptr.");
    IXA_REQUIRE(on_bytes(temperature, 4) && on_bytes(top_k, 4) && on_bytes(top_p, 4) && on_bytes(min_p, 4) && on_bytes(uniform, 4) &&
                    on_bytes(labels, 8) && on_bytes(probs, 4),
                kErrInvalidParam, "sample: settings, random numbers and results are not aligned to their elements");
    if (none) {
        return;
    }
    check_workspace("sample", workspace, workspace_bytes, need);
    SampleParams p{scores, temperature, top_p, min_p, uniform, top_k, labels, probs, ld, n, draws, parts_of(rows, n), nullptr, nullptr, nullptr};
    if (p.parts > 1) {
        uint8_t *const work = static_cast<uint8_t *>(workspace);
        p.lists = reinterpret_cast<uint64_t *>(work);
        p.segments = reinterpret_cast<double *>(work + rows * p.parts * (kPartList * 8));
        p.heads = reinterpret_cast<PartHead *>(work + rows * p.parts * (kPartList * 8) + rows * (kSegments * 8));
    }
    // Threads of a workgroup, by fp32 rows under top-p: 1024 rows of 4096 take 45 us with 256 and 55 with 512, 64 rows 31 and 25 (of 8192 48
    // and 59, 28 and 26).  A row per CU at most, 256 rows of 131072: 60 us with 1024 and 65 with 512, 38 and 36 of 32768; 300 rows of 131072: 99
    // and 89.
    with_type(type, [&](auto t) {
        typedef decltype(t) T;
        if (p.parts > 1) {
            hipLaunchKernelGGL((sample_part_kernel<T>), dim3((unsigned)(rows * p.parts)), dim3(kPartThreads), 0, s, p);
            check_launch();
            hipLaunchKernelGGL((sample_join_kernel<T>), dim3((unsigned)rows), dim3(kPartThreads), 0, s, p);
        } else if (n <= 4096) {
            hipLaunchKernelGGL((sample_kernel<T, 256>), dim3((unsigned)rows), dim3(256), 0, s, p);
        } else if (rows <= 256 && n >= 32768) {
            hipLaunchKernelGGL((sample_kernel<T, 1024>), dim3((unsigned)rows), dim3(1024), 0, s, p);
        } else {
            hipLaunchKernelGGL((sample_kernel<T, 512>), dim3((unsigned)rows), dim3(512), 0, s, p);
        }
    });
    check_launch();
}

}  // namespace ixa
