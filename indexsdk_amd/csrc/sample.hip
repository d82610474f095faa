// Columns drawn from rows of scores.  For a row x_0 ... x_(n-1) with temperature T, top-k k, top-p p and min-p m:
//   w_i = exp((x_i - max x) / T);  T <= 0: only the best column counts
//   the columns in the order of falling scores, equal ones in the order of columns, are cut to the first k, then to the fewest
//   whose weights reach p of those of all that are left, then to those with w_i >= m
//   a draw with the random number u is the first column, in the order of columns, at which the running sum of the weights that are
//   left passes u times their total
// Scores of -infinity and NaN are columns that are not there; beside +infinity everything else is.
//
// Every decision is one about sums of weights next to a border, so weights and sums are held in 64 bits: an exponential is 17
// instructions of the same rate as in 32.
//
// One workgroup per row reads it once (a few, each a part, where there are few rows).  The largest scores of some of its columns
// give a bound that about a hundred scores of the row reach; these go to a list in LDS, and while k or p or m keep no more than what
// is in the list, all else happens there: sorted by score, cut, and drawn from.  Rows without filters are drawn from by the sums
// of their segments.  Everything else (flat rows whose p keeps thousands, large k) reads the row again: a histogram of counts and
// weights finds the bin in which the cut lies, whose columns go through the list.
#include "row_access.h"
#include "scores.h"

#include <algorithm>
#include <type_traits>

namespace ixa {

namespace {

constexpr int kList = 2048;         // candidates of a row
constexpr int kPartList = 1024;     // and of a part of one
constexpr int kBins = 1024;
constexpr int kSegments = 512;      // at most: parts of a row whose sums are kept
constexpr int kBlock = 512;         // columns that a wavefront reads at a time
constexpr int kTurns = 4;           // such blocks in flight
constexpr int kSample = 2;          // blocks of each wavefront that the bound comes from
constexpr int kFew = 128;           // entries that are drawn from without being sorted by column
constexpr int kMaxParts = 16, kPartThreads = 512;
constexpr double kNothing = -1100.0;   // logarithms of weights that are 0 in 64 bits

// What a workgroup finds out about its part of a row.
struct PartHead {
    uint32_t top, reference, bound, listed;
    uint32_t fine, unused[3];
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

// 2^t for t <= 0 (and a little above): the polynomial of exp to the eleventh power, 6e-15
__device__ __forceinline__ double power_of_two(double t)
{
    const double whole = __builtin_rint(t), r = (t - whole) * 0.693147180559945309417232;
    double v = 1.0 / 39916800;
    v = fma(v, r, 1.0 / 3628800);
    v = fma(v, r, 1.0 / 362880);
    v = fma(v, r, 1.0 / 40320);
    v = fma(v, r, 1.0 / 5040);
    v = fma(v, r, 1.0 / 720);
    v = fma(v, r, 1.0 / 120);
    v = fma(v, r, 1.0 / 24);
    v = fma(v, r, 1.0 / 6);
    v = fma(v, r, 0.5);
    v = fma(v, r, 1.0);
    v = fma(v, r, 1.0);
    return __builtin_ldexp(v, (int)whole);
}

template <typename V>
__device__ __forceinline__ V wave_scan(V v)   // inclusive
{
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const V up = __shfl_up(v, o);
        v += lane >= o ? up : (V)0;
    }
    return v;
}

__device__ __forceinline__ uint64_t larger(uint64_t a, uint64_t b) { return a > b ? a : b; }

struct SampleShared {
    uint64_t list[kList];           // score's key above the column's complement
    union {
        double sum[kList];          // of the list's weights; a histogram is of no more use by then
        struct {
            unsigned long long mass[kBins];
            uint32_t count[kBins];
        };
    };
    union {
        double segment[kSegments];
        double few[2][kFew];        // running sums by column, and weights
    };
    double box[16];
    uint32_t tops[64];
    uint32_t ubox[16];
    uint32_t listed, found;
    uint64_t cut, before;
};

// What is drawn from: columns of at least `least` (an order of score and column as in the list) with weights of at least min_p.
struct Row {
    double scale;      // log2(e) / T
    float top;         // the largest score
    double min_p;
    uint64_t least;
    __device__ __forceinline__ double weight(float x) const
    {
        const double t = ((double)x - (double)top) * scale;
        return x == top ? 1.0 : t > kNothing ? power_of_two(t) : 0.0;
    }
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
    SampleShared &s;
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

    // f(block, scores) over blocks from ... to - 1, kTurns of them in flight
    template <typename F>
    __device__ __forceinline__ void run(int64_t from, int64_t to, F f) const
    {
        for (int64_t b = from; b < to; b += kTurns) {
            Eight<T> e[kTurns];
#pragma unroll
            for (int u = 0; u < kTurns; u++) {
                e[u] = load(min(b + u, to - 1));
            }
#pragma unroll
            for (int u = 0; u < kTurns; u++) {
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
        run(blocks() * wave / kWaves, blocks() * (wave + 1) / kWaves, f);
    }

    __device__ __forceinline__ double block_sum(double v) const
    {
        v = over_wave(v, [](double a, double b) { return a + b; });
        __syncthreads();
        if (lane == 0) {
            s.box[wave] = v;
        }
        __syncthreads();
        v = 0.0;
        for (int w = 0; w < kWaves; w++) {
            v += s.box[w];
        }
        return v;
    }
    __device__ __forceinline__ uint32_t block_max(uint32_t v) const
    {
        v = over_wave(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
        __syncthreads();
        if (lane == 0) {
            s.ubox[wave] = v;
        }
        __syncthreads();
        v = 0;
        for (int w = 0; w < kWaves; w++) {
            v = max(v, s.ubox[w]);
        }
        return v;
    }

    // Running sums (inclusive) of a[0 ... m), in place.
    __device__ void scan(double *a, int m) const
    {
        const int per = (m + NT - 1) / NT, from = tid * per;
        double sum = 0.0;
        for (int i = from; i < min(from + per, m); i++) {
            sum += a[i];
        }
        const double upto = wave_scan(sum);
        __syncthreads();
        if (lane == 63) {
            s.box[wave] = upto;
        }
        __syncthreads();
        const double before_me = __shfl_up(upto, 1);
        double run = lane == 0 ? 0.0 : before_me;
        for (int w = 0; w < wave; w++) {
            run += s.box[w];
        }
        for (int i = from; i < min(from + per, m); i++) {
            run += a[i];
            a[i] = run;
        }
        __syncthreads();
    }

    // list[0 ... m) in falling order (m <= kList)
    __device__ void sort(int m) const
    {
        int size = 2;
        while (size < m) {
            size <<= 1;
        }
        for (int i = m + tid; i < size; i += NT) {
            s.list[i] = 0;
        }
        // Exchanges over up to 64 entries stay among the 128 that one wavefront has, whose accesses to LDS happen in their order.
        __syncthreads();
        for (int k = 2; k <= size; k <<= 1) {
            for (int j = k >> 1; j > 0; j >>= 1) {
                for (int t = tid; t < size / 2; t += NT) {
                    const int a = (t & ~(j - 1)) * 2 + (t & (j - 1)), b = a + j;
                    const uint64_t x = s.list[a], y = s.list[b];
                    if ((x < y) == ((a & k) == 0)) {
                        s.list[a] = y;
                        s.list[b] = x;
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
            if (s.sum[mid] < target) {
                lo = mid + 1;
            } else {
                hi = mid;
            }
        }
        return lo + 1;
    }

    // sums of `value(x, column)` over segments of `per` blocks
    template <typename F>
    __device__ double segment_sums(int64_t per, F value) const
    {
        const int segments = (int)((blocks() + per - 1) / per);
        for (int g = wave; g < segments; g += kWaves) {
            double v = 0.0;
            run(g * per, min(blocks(), (g + 1) * per), [&](int64_t b, const float(&x)[kEight]) {
#pragma unroll
                for (int i = 0; i < kEight; i++) {
                    v += value(x[i], column(b, i));
                }
            });
            v = over_wave(v, [](double a, double b) { return a + b; });
            if (lane == 0) {
                s.segment[g] = v;
            }
        }
        return segment_total(segments);
    }
    __device__ double segment_total(int segments) const
    {
        __syncthreads();
        double v = 0.0;
        for (int g = tid; g < segments; g += NT) {
            v += s.segment[g];
        }
        return block_sum(v);
    }
    // A wavefront's search: the first column at which the running sum of `value` passes `target`, and its value; the last one with
    // a value if rounding hides it.
    template <typename F>
    __device__ void locate(int64_t per, double target, F value, int64_t &at, double &what) const
    {
        const int segments = (int)((blocks() + per - 1) / per);
        double before = 0.0;
        // the first segment that passes the target, or the last with a value: a run of them per lane
        double sum = 0.0, run = 0.0;
        const int each_lane = (segments + 63) / 64, from = lane * each_lane, to = min(from + each_lane, segments);
        for (int i = from; i < to; i++) {
            sum += s.segment[i];
        }
        const double upto_lane = wave_scan(sum);
        const uint64_t passes = __ballot(upto_lane > target && sum > 0.0), some = __ballot(sum > 0.0);
        const int l = passes ? __builtin_ctzll(passes) : some ? 63 - __builtin_clzll(some) : 0;
        const double before_lane = __shfl_up(upto_lane, 1);
        run = l == 0 ? 0.0 : __shfl(before_lane, l);
        int g = l * each_lane;
        for (int i = g; i < min((l + 1) * each_lane, segments); i++) {      // the same in every lane
            const double v = s.segment[i];
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
        const int64_t end = min(blocks(), (g + 1) * per);
        for (int64_t b = g * per; b < end; b++) {
            const Eight<T> e = load(b);
            double v[kEight], sum = 0.0;
#pragma unroll
            for (int i = 0; i < kEight; i++) {
                v[i] = value((float)e.v[i], column(b, i));
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
                return;
            }
            if (lasts) {
                const int l = 63 - __builtin_clzll(lasts);
                at = b * kBlock + l * kEight + __shfl(last, l);
                what = __shfl(last_v, l);
            }
            run += __shfl(upto, 63);
        }
    }

    // Columns for which pick(x, key, column) go to the list; false if they are too many.
    template <typename F>
    __device__ bool collect(F pick) const
    {
        if (tid == 0) {
            s.listed = 0;
        }
        __syncthreads();
        each([&](int64_t b, const float(&x)[kEight]) {
#pragma unroll
            for (int i = 0; i < kEight; i++) {
                const uint32_t key = key_of(x[i]), c = column(b, i);
                if (key && pick(x[i], key, c)) {
                    const uint32_t at = atomicAdd(&s.listed, 1u);
                    if (at < kList) {
                        s.list[at] = (uint64_t)key << 32 | ~c;
                    }
                }
            }
        });
        __syncthreads();
        return s.listed <= kList;
    }

    struct Limits {
        int64_t count;     // columns that may be kept
        double mass;       // and the sum that they have to reach (HUGE_VAL: none)
    };

    // The place (score and column) of the last column kept under either limit, among all columns that are there; the sum of the
    // weights up to and with it goes to `sum`.
    __device__ uint64_t find_cut(const Row &r, Limits limit, double &sum)
    {
        // bins of equal width in the scores, down to weights of 2^-64 for sums, and to the lowest score for counts
        float range = (float)(64.0 / r.scale);
        if (limit.mass == __builtin_huge_val()) {
            float lowest = __builtin_inff();
            each([&](int64_t, const float(&x)[kEight]) {
#pragma unroll
                for (int i = 0; i < kEight; i++) {
                    lowest = key_of(x[i]) ? fminf(lowest, x[i]) : lowest;
                }
            });
            range = r.top + score_of(block_max(key_of(-lowest)));
        }
        const float unit = range > 0.f && range < __builtin_inff() ? (float)kBins / range : 0.f;
        auto bin_of = [&](float x) {
            const float d = (r.top - x) * unit;
            return d < (float)(kBins - 1) ? (int)d : kBins - 1;     // also where 0 meets infinity
        };
        const double fixed = __builtin_ldexp(1.0, 62 - (64 - __builtin_clzll((unsigned long long)n)));
        auto add = [&](int b, float x) {
            atomicAdd(&s.count[b], 1u);
            if (limit.mass < __builtin_huge_val()) {
                atomicAdd(&s.mass[b], (unsigned long long)__builtin_rint(r.weight(x) * fixed));    // in any order
            }
        };
        uint64_t before_count = 0, before_mass = 0;
        // the first of m bins within a limit's reach
        auto cross = [&](int m) {
            __syncthreads();
            if (wave == 0) {
                const int per = (m + 63) / 64, from = lane * per, to = min(from + per, m);
                uint64_t c = 0, w = 0;
                for (int i = from; i < to; i++) {
                    c += s.count[i];
                    w += s.mass[i];
                }
                const uint64_t c_upto = before_count + wave_scan(c), w_upto = before_mass + wave_scan(w);
                auto over = [&](uint64_t a, uint64_t b) { return a >= (uint64_t)limit.count || (double)b / fixed >= limit.mass; };
                const uint64_t overs = __ballot(over(c_upto, w_upto) && c > 0), some = __ballot(c > 0);
                const int l = overs ? __builtin_ctzll(overs) : some ? 63 - __builtin_clzll(some) : 0;
                if (lane == l) {
                    uint64_t c_run = c_upto - c, w_run = w_upto - w;
                    int at = from;
                    s.cut = c_run;
                    s.before = w_run;
                    for (int i = from; i < to; i++) {
                        if (s.count[i]) {
                            at = i;
                            s.cut = c_run;
                            s.before = w_run;
                            if (over(c_run + s.count[i], w_run + s.mass[i])) {
                                break;
                            }
                        }
                        c_run += s.count[i];
                        w_run += s.mass[i];
                    }
                    s.found = (uint32_t)at;
                }
            }
            __syncthreads();
            const int at = (int)s.found;
            before_count = s.cut;
            before_mass = s.before;
            __syncthreads();
            return at;
        };
        auto clear = [&]() {
            __syncthreads();
            for (int i = tid; i < kBins; i += NT) {
                s.count[i] = 0;
                s.mass[i] = 0;
            }
            __syncthreads();
        };
        clear();
        each([&](int64_t, const float(&x)[kEight]) {
#pragma unroll
            for (int i = 0; i < kEight; i++) {
                if (key_of(x[i])) {
                    add(bin_of(x[i]), x[i]);
                }
            }
        });
        const int bin = cross(kBins);
        // a bin with too many for the list: by the bits of their keys, ten at a time
        uint32_t prefix = 0, known = 0;
        for (int shift = 32;;) {
            if (collect([&](float x, uint32_t key, uint32_t) { return bin_of(x) == bin && (key & known) == prefix; }) || shift == 0) {
                break;
            }
            const int bits = min(10, shift), to = shift - bits;
            const uint32_t mask = (1u << bits) - 1u;
            clear();
            each([&](int64_t, const float(&x)[kEight]) {
#pragma unroll
                for (int i = 0; i < kEight; i++) {
                    const uint32_t key = key_of(x[i]);
                    if (key && bin_of(x[i]) == bin && (key & known) == prefix) {
                        add(~(key >> to) & mask, x[i]);      // the largest first
                    }
                }
            });
            prefix |= (~(uint32_t)cross(1 << bits) & mask) << to;
            known |= mask << to;
            shift = to;
        }
        const double before = (double)before_mass / fixed;
        if (s.listed > kList) {
            // equal scores: as many of them as the limits allow, by their columns
            const float x = score_of(prefix);
            const double w = r.weight(x), ties = (double)s.listed;
            double take = (double)(limit.count - (int64_t)before_count);
            if (limit.mass < __builtin_huge_val()) {
                take = fmin(take, w > 0.0 ? ceil((limit.mass - before) / w) : ties);
            }
            take = fmax(1.0, fmin(take, ties));
            const int64_t per = segment_size();
            auto tie = [&](float v, uint32_t) { return key_of(v) == prefix ? 1.0 : 0.0; };
            segment_sums(per, tie);
            int64_t at;
            double one;
            locate(per, take - 0.5, tie, at, one);
            sum = before + take * w;
            __syncthreads();
            return r.place(prefix, (uint32_t)at);
        }
        const int m = (int)s.listed;
        sort(m);
        for (int i = tid; i < m; i += NT) {
            s.sum[i] = r.weight(score_of((uint32_t)(s.list[i] >> 32)));
        }
        __syncthreads();
        scan(s.sum, m);
        int take = (int)min((int64_t)m, limit.count - (int64_t)before_count);
        if (limit.mass < __builtin_huge_val()) {
            take = min(take, reach(limit.mass - before, m));
        }
        take = max(1, min(take, m));
        sum = before + s.sum[take - 1];
        const uint64_t place = s.list[take - 1];
        __syncthreads();
        return place;
    }

    __device__ __forceinline__ int64_t segment_size() const
    {
        // four blocks where every wavefront gets that many
        return max(min((int64_t)kTurns, (blocks() + kWaves - 1) / kWaves), (blocks() + kSegments - 1) / kSegments);
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

// A part of a row, once: its largest score, the sums of weights relative to a reference, segment by segment, and the list.
template <typename T, int NT>
__device__ __forceinline__ PartHead scan_part(const Sampler<T, NT> &k, const Settings &set, int part, int parts)
{
    constexpr int kWaves = NT / 64;
    SampleShared &s = k.s;
    const int lane = k.lane, wave = k.wave;
    const int64_t per = k.segment_size(), all = (k.blocks() + per - 1) / per;
    const int g0 = (int)(all * part / parts), g1 = (int)(all * (part + 1) / parts);
    const int64_t b0 = g0 * per, b1 = min(k.blocks(), g1 * per), mine = b1 - b0;

    // The largest of 64 groups of lanes in some of the columns.
    constexpr int kLanes = kWaves;
    const int64_t first = b0 + mine * wave / kWaves, end = b0 + mine * (wave + 1) / kWaves;
    float lane_top = -__builtin_inff();
#pragma unroll
    for (int u = 0; u < kSample; u++) {
        if (first + u < end) {
            const Eight<T> e = k.load(first + u);
#pragma unroll
            for (int i = 0; i < kEight; i++) {
                lane_top = fmaxf(lane_top, (float)e.v[i]);
            }
        }
    }
    const int flip = (int)0x80000000;
    const int group_top = over_lanes<kLanes>((int)key_of(lane_top) ^ flip, [](int a, int b) { return max(a, b); });
    if (lane % kLanes == 0) {
        s.tops[wave * (64 / kLanes) + lane / kLanes] = (uint32_t)(group_top ^ flip);
    }
    if (k.tid == 0) {
        s.listed = 0;
    }
    __syncthreads();
    const uint32_t tops = s.tops[lane];
    const uint32_t sample_top = over_wave(tops, [](uint32_t a, uint32_t b) { return max(a, b); });
    const float reference = score_of(sample_top);
    // A bound that so many of the sampled columns reach that all of them have what is kept, but for one time in thousands: as
    // many more than expected as three deviations.
    PartHead h{0, sample_top, 0xffffffffu, 0, 1, {}};
    const int64_t columns = min(k.n - b0 * kBlock, mine * kBlock);
    if (set.filtered && sample_top && columns > 0) {
        const float share = (float)min(columns, (int64_t)NT * kEight * kSample) / (float)columns;
        // what is wanted of all parts: k, or for sums a few hundred
        const float wanted = (set.by_count ? (float)min(set.count, (int64_t)kList) : 256.f) / (float)parts * share;
        const float reach = wanted + 3.f * __builtin_amdgcn_sqrtf(wanted) + 4.f;
        if (columns <= 4 * kFew) {
            h.bound = 1;      // everything that is there
        } else if (reach <= 130.f || !set.by_count) {
            // of 64 groups those that hold one of `reach` columns at least
            const int groups = (int)fminf(56.f, 64.f * (1.f - __expf(-reach / 64.f)) + 0.5f);
            uint32_t b = 0;
#pragma unroll
            for (int bit = 31; bit >= 16; bit--) {
                const uint32_t at = b | 1u << bit;
                b = __popcll(__ballot(tops >= at)) >= groups ? at : b;
            }
            h.bound = max(b, 1u);
        }
    }
    const float bound = h.bound == 0xffffffffu ? __builtin_nanf("") : h.bound == 1 ? -3.402823466e+38f : score_of(h.bound);
    const bool sums = set.need_mass;
    float top = -__builtin_inff();
    const int limit = parts > 1 ? kPartList : kList;
    for (int g = g0 + wave; g < g1; g += kWaves) {
        double v = 0.0;
        k.run(g * per, min(b1, (g + 1) * per), [&](int64_t b, const float(&x)[kEight]) {
            float most = x[0];
#pragma unroll
            for (int i = 1; i < kEight; i++) {
                most = fmaxf(most, x[i]);
            }
            top = fmaxf(top, most);
            if (sums) {
#pragma unroll
                for (int i = 0; i < kEight; i++) {
                    v += power_of_two(fmax(((double)x[i] - (double)reference) * set.scale, kNothing));   // NaN and -infinity: 0
                }
            }
            if (most >= bound) {
#pragma unroll
                for (int i = 0; i < kEight; i++) {
                    if (x[i] >= bound) {
                        const uint32_t at = atomicAdd(&s.listed, 1u);
                        if (at < (uint32_t)limit) {
                            s.list[at] = (uint64_t)key_of(x[i]) << 32 | ~k.column(b, i);
                        }
                    }
                }
            }
        });
        if (sums) {
            v = over_wave(v, [](double a, double b) { return a + b; });
            if (lane == 0) {
                s.segment[g] = v;
            }
        }
    }
    h.top = k.block_max(key_of(top));
    h.listed = h.bound == 0xffffffffu ? 0xffffffffu : s.listed;
    return h;
}

// The draws from a row whose list and sums are in LDS.
template <typename T, int NT>
__device__ __forceinline__ void finish_row(Sampler<T, NT> &k, const SampleParams &p, const Settings &set, int64_t row,
                                           const PartHead &h, double total)
{
    constexpr int kWaves = NT / 64;
    SampleShared &s = k.s;
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
    Row r{set.scale, score_of(h.top), set.min_p, 0};
    if (set.need_mass && !h.fine) {
        total = k.segment_sums(per, [&](float x, uint32_t) { return key_of(x) ? r.weight(x) : 0.0; });
    }
    auto draw_number = [&](int d) {
        const float u = uniform[d];
        return (double)(u > 0.f ? fminf(u, 0x1.fffffep-1f) : 0.f);
    };
    if (set.filtered) {
        const bool complete = h.bound == 1;      // every column that is there is in the list
        int m = h.listed <= kList ? (int)h.listed : 0, take = m;
        if (m > 0) {
            k.sort(m);
            for (int i = tid; i < m; i += NT) {
                s.sum[i] = r.weight(score_of((uint32_t)(s.list[i] >> 32)));
            }
            __syncthreads();
            k.scan(s.sum, m);
            bool cut = complete;               // whether the list holds all that is kept
            if (set.by_count) {
                cut = cut || m >= count;
                take = (int)min((int64_t)m, count);
            }
            if (set.by_mass && (cut || !set.by_count)) {
                // of the sum of all that is left, which the list has or the whole row
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
            const double all = s.sum[take - 1];
            __syncthreads();
            if (cut && take <= kFew) {
                // each entry's running sum by column, from all others in the order of the list
                if (tid < take) {
                    s.few[1][tid] = r.weight(score_of((uint32_t)(s.list[tid] >> 32)));
                }
                __syncthreads();
                if (tid < take) {
                    const uint32_t mine = (uint32_t)s.list[tid];       // the complement of the column
                    double v = 0.0;
                    for (int i = 0; i < take; i++) {
                        v += (uint32_t)s.list[i] >= mine ? s.few[1][i] : 0.0;
                    }
                    s.few[0][tid] = v;
                }
                __syncthreads();
                for (int d = wave; d < p.draws; d += kWaves) {
                    const double target = draw_number(d) * all;
                    // the lowest column that passes it, or the last with a weight if rounding hides that
                    uint64_t best = 0;
#pragma unroll
                    for (int c = 0; c < kFew / 64; c++) {
                        const int i = c * 64 + lane;
                        if (i < take && s.few[1][i] > 0.0) {
                            const uint32_t place = (uint32_t)s.list[i];
                            best = larger(best, s.few[0][i] > target ? 1ull << 63 | (uint64_t)place << 8 | (uint64_t)i
                                                                     : (uint64_t)(uint32_t)~place << 8 | (uint64_t)i);
                        }
                    }
                    best = over_wave(best, larger);
                    if (lane == 0) {
                        const int i = (int)(best & 127u);
                        labels[d] = (int64_t)(~(uint32_t)s.list[i]);
                        if (probs) {
                            probs[d] = (float)(s.few[1][i] / all);
                        }
                    }
                }
                return;
            }
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
        double sum = total;
        if (set.by_count) {
            r.least = k.find_cut(r, {count, __builtin_huge_val()}, sum);
            if (set.by_mass) {
                // the sum up to the cut by its columns
                auto value = [&](float x, uint32_t c) { return key_of(x) && r.place(key_of(x), c) >= r.least ? r.weight(x) : 0.0; };
                sum = k.segment_sums(per, value);
            }
        }
        if (set.by_mass) {
            r.least = larger(r.least, k.find_cut(r, {k.n + 1, set.top_p * sum}, sum));
        }
        total = k.segment_sums(per, [&](float x, uint32_t c) { return r.kept(x, c); });
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
__device__ __forceinline__ Sampler<T, NT> sampler(SampleShared &s, const SampleParams &p, int64_t row)
{
    return Sampler<T, NT>{s, static_cast<const T *>(p.scores) + row * p.ld, p.n, (int)threadIdx.x, (int)threadIdx.x & 63,
                          __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6)};
}

// What a sum relative to `reference` is multiplied by to be one relative to `top`; 0: it can not be.
__device__ __forceinline__ double unit_of(float reference, float top, double scale)
{
    const double t = ((double)reference - (double)top) * scale;
    return reference == top && top < __builtin_inff() ? 1.0 : t > -1000.0 ? power_of_two(t) : 0.0;
}

template <typename T, int NT>
__global__ __launch_bounds__(NT) void sample_kernel(SampleParams p)
{
    __shared__ SampleShared s;
    const int64_t row = blockIdx.x;
    Sampler<T, NT> k = sampler<T, NT>(s, p, row);
    const Settings set(p, row);
    PartHead h = scan_part(k, set, 0, 1);
    double total = 0.0;
    if (set.need_mass && h.top && h.fine) {
        const int64_t per = k.segment_size();
        const int segments = (int)((k.blocks() + per - 1) / per);
        const double unit = unit_of(score_of(h.reference), score_of(h.top), set.scale);
        total = k.segment_total(segments);
        h.fine = total < 0x1p1000 && unit > 0.0;
        total *= unit;
        if (!set.filtered) {
            for (int g = k.tid; g < segments; g += NT) {
                s.segment[g] *= unit;
            }
            __syncthreads();
        }
    }
    finish_row(k, p, set, row, h, total);
}

// A part of a row per workgroup, and what it found out.
template <typename T>
__global__ __launch_bounds__(kPartThreads) void sample_part_kernel(SampleParams p)
{
    __shared__ SampleShared s;
    const int64_t row = blockIdx.x / p.parts;
    const int part = (int)(blockIdx.x - row * p.parts);
    const Sampler<T, kPartThreads> k = sampler<T, kPartThreads>(s, p, row);
    const Settings set(p, row);
    const PartHead h = scan_part(k, set, part, p.parts);
    if (k.tid == 0) {
        p.heads[blockIdx.x] = h;
    }
    if (h.listed <= kPartList) {
        for (int i = k.tid; i < (int)h.listed; i += kPartThreads) {
            p.lists[(int64_t)blockIdx.x * kPartList + i] = s.list[i];
        }
    }
    if (set.need_mass && h.fine) {
        const int64_t per = k.segment_size(), all = (k.blocks() + per - 1) / per;
        for (int g = (int)(all * part / p.parts) + k.tid; g < (int)(all * (part + 1) / p.parts); g += kPartThreads) {
            p.segments[row * kSegments + g] = s.segment[g];
        }
    }
}

// The parts of a row, joined: the highest of their bounds is one that all lists go down to.
template <typename T>
__global__ __launch_bounds__(kPartThreads) void sample_join_kernel(SampleParams p)
{
    __shared__ SampleShared s;
    const int64_t row = blockIdx.x;
    Sampler<T, kPartThreads> k = sampler<T, kPartThreads>(s, p, row);
    const Settings set(p, row);
    PartHead all{0, 0, 0, 0, 1, {}};
    bool listed = true;
    for (int i = 0; i < p.parts; i++) {
        const PartHead h = p.heads[row * p.parts + i];
        if (h.top) {
            all.top = max(all.top, h.top);
            all.bound = max(all.bound, h.bound);
            listed = listed && h.listed <= kPartList;
            all.fine &= h.fine;
        }
    }
    all.bound = max(all.bound, 1u);
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
        if (set.need_mass && all.fine) {
            const double unit = h.top ? unit_of(score_of(h.reference), top, set.scale) : 0.0;
            for (int g = (int)(segments * i / p.parts) + k.tid; g < (int)(segments * (i + 1) / p.parts); g += kPartThreads) {
                const double v = h.top ? p.segments[row * kSegments + g] : 0.0;
                // what does not come out as a sum is found out again
                s.segment[g] = h.top && !(unit > 0.0) ? __builtin_nan("") : v * unit;
            }
        }
    }
    __syncthreads();
    all.listed = listed ? s.listed : 0xffffffffu;
    double total = 0.0;
    if (set.need_mass && all.top && all.fine) {
        total = k.segment_total((int)segments);
        all.fine = total < 0x1p1000;      // also not of what is no number
    }
    finish_row(k, p, set, row, all, total);
}

// Parts of each row where there are few rows: as many as give every second CU a workgroup, of 16384 columns at least (64 rows of
// 131072 under top-p: SAMPLE_PARTS).
int parts_of(int64_t rows, int64_t n)
{
    if (rows == 0 || rows > 128 || n < 65536) {
        return 1;
    }
    return (int)std::min<int64_t>({kMaxParts, 256 / rows, n / 16384});
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
