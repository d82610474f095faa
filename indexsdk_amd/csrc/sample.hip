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
// One workgroup per row reads it once.  The largest scores of its first columns (of each wavefront's part) give a bound that
// some hundred scores of the row reach; these go to a list in LDS, and while k or p or m keep no more than what is in the list, all else
// happens there: sorted by score and cut, sorted by column and drawn from.  Rows without filters are drawn from by the sums of
// their segments.  Everything else (flat rows whose p keeps thousands, large k) reads the row again: a histogram of counts
// and weights finds the bin in which the cut lies, whose columns go through the list.
#include "row_access.h"
#include "scores.h"

#include <algorithm>
#include <type_traits>

namespace ixa {

namespace {

constexpr int kList = 2048;         // candidates of a row
constexpr int kBins = 1024;
constexpr int kSegments = 1024;     // at most: parts of a row whose sums are kept
constexpr int kBlock = 512;         // columns that a wavefront reads at a time
constexpr int kSample = 2;          // such blocks of each wavefront that the bound comes from

struct SampleParams {
    const void *scores;
    const float *temperature, *top_p, *min_p, *uniform;
    const int32_t *top_k;
    int64_t *labels;
    float *probs;
    int64_t ld, n;
    int draws;
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

template <typename V, typename Op>
__device__ __forceinline__ V wave_reduce(V v, Op op)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        v = op(v, __shfl_xor(v, o));
    }
    return v;
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

struct SampleShared {
    uint64_t list[kList];           // score's key above the column's complement
    double sum[kList];
    double segment[kSegments];
    unsigned long long mass[kBins];
    uint32_t count[kBins];
    double box[16];
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
        return x == top ? 1.0 : t > -1080.0 ? power_of_two(t) : 0.0;
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

    __device__ __forceinline__ void load(int64_t block, float (&x)[kEight]) const
    {
        const int64_t at = block * kBlock + lane * kEight;
        Eight<T> e;
        const int count = (int)min((int64_t)kEight, max((int64_t)0, n - at));
        e.load(row + (count ? at : 0), count, (T)-__builtin_inff());
#pragma unroll
        for (int i = 0; i < kEight; i++) {
            x[i] = (float)e.v[i];
        }
    }
    __device__ __forceinline__ int64_t blocks() const { return (n + kBlock - 1) / kBlock; }
    __device__ __forceinline__ uint32_t column(int64_t block, int i) const { return (uint32_t)(block * kBlock + lane * kEight + i); }

    // f(block, scores) over the blocks of a wavefront's part of the row
    template <typename F>
    __device__ __forceinline__ void each(F f) const
    {
        const int64_t end = blocks() * (wave + 1) / kWaves;
        for (int64_t b = blocks() * wave / kWaves; b < end; b++) {
            float x[kEight];
            load(b, x);
            f(b, x);
        }
    }

    __device__ __forceinline__ double block_sum(double v) const
    {
        v = wave_reduce(v, [](double a, double b) { return a + b; });
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
        v = wave_reduce(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
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
                __syncthreads();
            }
        }
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
            const int64_t end = min(blocks(), (g + 1) * per);
            for (int64_t b = g * per; b < end; b++) {
                float x[kEight];
                load(b, x);
#pragma unroll
                for (int i = 0; i < kEight; i++) {
                    v += value(x[i], column(b, i));
                }
            }
            v = wave_reduce(v, [](double a, double b) { return a + b; });
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
        // the first segment that passes the target, or the last with a value: 16 of them per lane
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
            float x[kEight];
            load(b, x);
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
    __device__ uint64_t find_cut(const Row &r, float lowest, Limits limit, double &sum)
    {
        const float width = r.top - lowest;
        // bins of equal width in the scores, those of weights below 2^-64 in the last if sums are looked for
        float range = width;
        if (limit.mass < __builtin_huge_val() && limit.count >= n) {
            range = fminf(range, (float)(64.0 / r.scale));
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
        return max((int64_t)4, (blocks() + kSegments - 1) / kSegments);
    }
};

template <typename T, int NT>
__global__ __launch_bounds__(NT) void sample_kernel(SampleParams p)
{
    __shared__ SampleShared s;
    const int64_t row = blockIdx.x;
    typedef Sampler<T, NT> Work;
    Work k{s, static_cast<const T *>(p.scores) + row * p.ld, p.n, (int)threadIdx.x, (int)threadIdx.x & 63,
           __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6)};
    const int tid = k.tid, lane = k.lane, wave = k.wave;
    constexpr int kWaves = Work::kWaves;
    const int64_t n = p.n;
    float temperature = p.temperature ? p.temperature[row] : 1.f;
    int64_t count = p.top_k ? p.top_k[row] : 0;
    double top_p = p.top_p ? (double)p.top_p[row] : 1.0;
    double min_p = p.min_p ? (double)p.min_p[row] : 0.0;
    count = count <= 0 ? n : min(n, count);
    if (!(temperature > 0.f)) {
        temperature = 1.f;
        count = 1;
    }
    const bool by_count = count < n, by_mass = top_p < 1.0;     // not a number: no
    min_p = min_p > 0.0 ? fmin(min_p, 1.0) : 0.0;
    const bool filtered = by_count || by_mass || min_p > 0.0, need_mass = !by_count;
    Row r;
    r.scale = 1.44269504088896340735992468 / (double)temperature;
    r.min_p = min_p;
    r.least = 0;

    // The bound that some hundred scores reach: from the largest of each lane's first columns.
    const int64_t first = k.blocks() * wave / kWaves, end = k.blocks() * (wave + 1) / kWaves;
    float lane_top = -__builtin_inff();
    for (int64_t b = first; b < min(first + kSample, end); b++) {
        float x[kEight];
        k.load(b, x);
#pragma unroll
        for (int i = 0; i < kEight; i++) {
            lane_top = fmaxf(lane_top, x[i]);
        }
    }
    const uint32_t sample_top = k.block_max(key_of(lane_top));
    const float reference = score_of(sample_top);
    uint32_t bound = 0xffffffffu;    // nothing is listed
    const int wanted = by_count ? max(256, 2 * (int)min(count, (int64_t)kList)) : 768;
    if (filtered && wanted <= kList / 2 && sample_top) {
        uint32_t *const tops = s.count;
        tops[tid] = key_of(lane_top);
        if (tid == 0) {
            s.listed = 0;
        }
        __syncthreads();
        const double share = (double)min(n, (int64_t)NT * kEight * kSample) / (double)n;
        const int rank = (int)fmin(0.75 * NT, fmax(4.0, wanted * share));
        if (wave == 0) {
            uint32_t mine[kWaves];
#pragma unroll
            for (int i = 0; i < kWaves; i++) {
                mine[i] = tops[i * 64 + lane];
            }
            // the largest number of sixteen bits that `rank` of them reach
            uint32_t b = 0;
            for (int bit = 31; bit >= 16; bit--) {
                const uint32_t at = b | 1u << bit;
                int reached = 0;
#pragma unroll
                for (int i = 0; i < kWaves; i++) {
                    reached += __popcll(__ballot(mine[i] >= at));
                }
                b = reached >= rank ? at : b;
            }
            if (lane == 0) {
                s.found = max(b, 1u);
            }
        }
        __syncthreads();
        bound = s.found;
    }

    // The row, once: its largest and lowest score, the sum of weights relative to `reference`, segment by segment, and the list.
    const int64_t per = k.segment_size();
    const int segments = (int)((k.blocks() + per - 1) / per);
    uint32_t top_key = 0;
    float lowest = __builtin_inff();
    for (int g = wave; g < segments; g += kWaves) {
        double v = 0.0;
        const int64_t last = min(k.blocks(), (g + 1) * per);
        for (int64_t b = g * per; b < last; b++) {
            float x[kEight];
            k.load(b, x);
#pragma unroll
            for (int i = 0; i < kEight; i++) {
                const uint32_t key = key_of(x[i]);
                top_key = max(top_key, key);
                lowest = key ? fminf(lowest, x[i]) : lowest;
                if (need_mass) {
                    const double t = ((double)x[i] - (double)reference) * r.scale;
                    v += key && t > -1080.0 ? power_of_two(t) : 0.0;
                }
                if (key >= bound) {
                    const uint32_t at = atomicAdd(&s.listed, 1u);
                    if (at < kList) {
                        s.list[at] = r.place(key, k.column(b, i));
                    }
                }
            }
        }
        if (need_mass) {
            v = wave_reduce(v, [](double a, double b) { return a + b; });
            if (lane == 0) {
                s.segment[g] = v;
            }
        }
    }
    top_key = k.block_max(top_key);
    int64_t *const labels = p.labels + row * p.draws;
    float *const probs = p.probs ? p.probs + row * p.draws : nullptr;
    const float *const uniform = p.uniform + row * p.draws;
    if (top_key == 0) {
        for (int d = tid; d < p.draws; d += NT) {
            labels[d] = -1;
            if (probs) {
                probs[d] = 0.f;
            }
        }
        return;
    }
    r.top = score_of(top_key);
    double total = 0.0;
    if (need_mass) {
        // from the reference to the largest score
        const double t = ((double)reference - (double)r.top) * r.scale, unit = r.top == reference ? 1.0 : t > -1000.0 ? power_of_two(t) : 0.0;
        total = k.segment_total(segments);
        const bool fine = total < 0x1p1000 && unit > 0.0 && r.top < __builtin_inff();
        if (fine) {
            total *= unit;
            for (int g = tid; g < segments; g += NT) {
                s.segment[g] *= unit;
            }
            __syncthreads();
        } else {
            total = k.segment_sums(per, [&](float x, uint32_t) { return key_of(x) ? r.weight(x) : 0.0; });
        }
    }
    auto draw_number = [&](int d) {
        const float u = uniform[d];
        return (double)(u > 0.f ? fminf(u, 0x1.fffffep-1f) : 0.f);
    };

    if (filtered) {
        const bool complete = bound <= 1;      // every column that is there is in the list
        int m = bound != 0xffffffffu && s.listed <= kList ? (int)s.listed : 0, take = m;
        if (m > 0) {
            k.sort(m);
            for (int i = tid; i < m; i += NT) {
                s.sum[i] = r.weight(score_of((uint32_t)(s.list[i] >> 32)));
            }
            __syncthreads();
            k.scan(s.sum, m);
            bool cut = complete;               // whether the list holds all that is kept
            if (by_count) {
                cut = cut || m >= count;
                take = (int)min((int64_t)m, count);
            }
            if (by_mass && (cut || !by_count)) {
                // of the sum of all that is left, which the list has or the whole row
                const int need = k.reach(top_p * (cut ? s.sum[take - 1] : total), take);
                cut = cut || need <= take;
                take = min(take, need);
            }
            if (min_p > 0.0 && !(by_count && !cut)) {
                int above = 0, below = m;      // weights fall along the list
                while (above < below) {
                    const int mid = (above + below) >> 1;
                    if (r.weight(score_of((uint32_t)(s.list[mid] >> 32))) >= min_p) {
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
                const double all = s.sum[take - 1];
                for (int d = tid; d < p.draws; d += NT) {
                    const double target = draw_number(d) * all;
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
                        probs[d] = (float)(r.weight(score_of((uint32_t)s.list[lo])) / all);
                    }
                }
                return;
            }
        }
        __syncthreads();
        // the row again
        lowest = -score_of(k.block_max(key_of(-lowest)));
        double sum = total;
        if (by_count) {
            r.least = k.find_cut(r, lowest, {count, __builtin_huge_val()}, sum);
            if (by_mass) {
                // the sum up to the cut by its columns
                auto value = [&](float x, uint32_t c) { return key_of(x) && r.place(key_of(x), c) >= r.least ? r.weight(x) : 0.0; };
                sum = k.segment_sums(per, value);
            }
        }
        if (by_mass) {
            r.least = max(r.least, k.find_cut(r, lowest, {n + 1, top_p * sum}, sum));
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

}  // namespace

int64_t sample_workspace(int64_t rows, int64_t n)
{
    check_scores("sample", rows, n);
    return 0;
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
    const SampleParams p{scores, temperature, top_p, min_p, uniform, top_k, labels, probs, ld, n, draws};
    with_type(type, [&](auto t) {
        typedef decltype(t) T;
        if (rows <= 256) {
            hipLaunchKernelGGL((sample_kernel<T, 1024>), dim3((unsigned)rows), dim3(1024), 0, s, p);
        } else {
            hipLaunchKernelGGL((sample_kernel<T, 512>), dim3((unsigned)rows), dim3(512), 0, s, p);
        }
    });
    check_launch();
}

}  // namespace ixa
