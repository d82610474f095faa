// The loss of rows of scores against a teacher's top entries, and its gradient.  For a row of scores s_0 ... s_(n-1) and a teacher's
// k entries (label l_j, score t_j), with one temperature T:
//   p_j = exp(t_j / T - L), L = log sum_j exp(t_j / T) over the entries that are there, or given (the teacher's over all columns)
//   q_i = exp(s_i / T) / sum_i exp(s_i / T),   P = sum_j p_j
//   loss = T^2 sum_j p_j (log p_j - log q_(l_j)),   d loss / d s_i = T (P q_i - sum of p_j with l_j = i)
// Entries with a label outside 0 ... n - 1 are not there.  Rows without an entry or without a score above -infinity have loss and
// gradient 0.
//
// All of it is bound by memory.  A row that fits into a workgroup's registers is read once, while the gradient of the row before it is
// written: 4096 rows of 131072 bf16 take 435 us, 4.95 TB/s of the 5.2 at which memory is copied.  Longer rows are read twice, by a
// kernel for the sums (5.4 TB/s) and one for the gradient (5.6), or where only one of the two is asked for.  Reading a row again
// soon, from the cache behind the L2, is no faster than from memory: both come through the same 5.8 TB/s.
//
// Exponentials of fp32 scores take 2^t of both parts of the product with log2(e) / T, those of 16-bit scores the rounded product; 32 of
// them are added in 32 bits, all else in 64, also what the teacher's entries need: the loss is a small difference of large logarithms.
#include "power_of_two.h"
#include "row_access.h"
#include "scores.h"

#include <algorithm>
#include <type_traits>

namespace ixa {

namespace {

constexpr int kThreads = 256;
constexpr int kTurns = 4;                         // times eight scores of a thread in flight
constexpr int kPart = kThreads * kEight * kTurns;   // scores that such a workgroup reads at a time
constexpr int kAlone = 256;                       // entries that one wavefront sees to
constexpr double kLog2e = 1.44269504088896340735992468, kLn2 = 0.693147180559945309417232;

struct DistilParams {
    const void *scores;
    int64_t ld, n, rows;
    const int64_t *labels;
    const float *teacher, *whole;
    int k, parts, slots, buffers;       // parts of a row; places of the table of labels; rows of entries in LDS
    double temperature, scale;  // scale: log2(e) / T
    float high, low;            // the same in two parts
    int64_t part;               // scores per part
    float *loss, *stats;
    double *partial;            // [rows][parts][2]
    const float *given_stats, *row_weight;
    void *gradient;
    int64_t ld_gradient;
};

// exp((x - top) / T)
template <typename T>
__device__ __forceinline__ float exponential(float x, float top, const DistilParams &p)
{
    const float d = x - top, t = d * p.high;
    if constexpr (sizeof(T) == 4) {
        const float rest = fmaf(d, p.low, fmaf(d, p.high, -t));
        const float e = __builtin_amdgcn_exp2f(t);
        // beyond any number's reach the rest is no number
        return t > -200.f ? fmaf(e, rest * (float)kLn2, e) : e;
    } else {
        return __builtin_amdgcn_exp2f(t);
    }
}

// exp((x - top) / T) where many scores share one `top`: 2^(h x - c) of 16-bit scores is one instruction less, and its product is
// rounded once, together with the difference.  c is rounded too, by a factor that is the same for all of them.
template <typename T>
struct Exponent {
    float reference, h, c;
    __device__ __forceinline__ Exponent(float top, const DistilParams &p)
    {
        reference = top == -__builtin_inff() ? 0.f : top;
        h = p.high;
        if (fabsf(reference * h) > 0x1p21f && reference < __builtin_inff()) {
            // scores that differ from the largest one, by a 2048th of it at least, are e^-700 of it and less: also with a smaller h,
            // with which h x - c is exact for x = top
            h = __builtin_ldexpf(1.f, 21 - __builtin_amdgcn_frexp_expf(reference));
        }
        c = reference * h;
    }
    __device__ __forceinline__ float operator()(float x, const DistilParams &p) const
    {
        if constexpr (sizeof(T) == 4) {
            return exponential<T>(x, reference, p);
        } else {
            return __builtin_amdgcn_exp2f(fmaf(x, h, -c));
        }
    }
    // what these are to be multiplied by
    __device__ __forceinline__ double factor() const
    {
        return sizeof(T) == 4 || !(reference < __builtin_inff()) ? 1.0 : any_power_of_two((double)c - (double)reference * (double)h);
    }
};

// A largest score and the sum of exponentials relative to it (to 0 where there is none).
struct Sum {
    float top;
    double sum;
    __device__ __forceinline__ float reference() const { return top == -__builtin_inff() ? 0.f : top; }
    __device__ __forceinline__ void join(float other_top, double other_sum, const DistilParams &p)
    {
        const float both = fmaxf(top, other_top), r = both == -__builtin_inff() ? 0.f : both;
        // sums of nothing are 0 or no number
        const double mine = top == -__builtin_inff() ? 1.0 : any_power_of_two(((double)top - r) * p.scale);
        const double others = other_top == -__builtin_inff() ? 1.0 : any_power_of_two(((double)other_top - r) * p.scale);
        sum = sum * mine + other_sum * others;
        top = both;
    }
};

// Op over groups of LANES (1, 2, 4, 8 or 16) lanes, of 32 or 64 bits
template <int LANES, typename V, typename Op>
__device__ __forceinline__ V over_lanes_of(V v, Op op)
{
    if constexpr (LANES >= 2) {
        v = op(v, value_of_lane<kXor1>(v));
    }
    if constexpr (LANES >= 4) {
        v = op(v, value_of_lane<kXor2>(v));
    }
    if constexpr (LANES >= 8) {
        v = op(v, value_of_lane<kMirror8>(v));
    }
    if constexpr (LANES >= 16) {
        v = op(v, value_of_lane<kMirror16>(v));
    }
    return v;
}

// The threads' sums together.  box [NT / 64] is no other joint's until the workgroup's next barrier.
template <int NT>
__device__ __forceinline__ Sum joined(Sum mine, const DistilParams &p, Sum *box)
{
    auto both = [&](Sum a, float top) {
        const float r = top == -__builtin_inff() ? 0.f : top;
        return a.top == -__builtin_inff() ? a.sum : a.sum * any_power_of_two(((double)a.top - r) * p.scale);
    };
    auto larger = [](float a, float b) { return fmaxf(a, b); };
    auto add = [](double a, double b) { return a + b; };
    float top = over_wave(mine.top, larger);
    const double sum = over_wave(both(mine, top), add);
    if ((threadIdx.x & 63) == 0) {
        box[threadIdx.x >> 6] = {top, sum};
    }
    __syncthreads();
    Sum all = box[threadIdx.x & (NT / 64 - 1)];
    top = over_lanes_of<NT / 64>(all.top, larger);
    return {top, over_lanes_of<NT / 64>(both(all, top), add)};
}

// The sum over scores from ... to - 1 of a row, by the workgroup.
template <typename T, int NT>
__device__ Sum sum_of(const DistilParams &p, const T *row, int64_t from, int64_t to, Sum *box)
{
    Sum mine{-__builtin_inff(), 0.0};
    for (int64_t at = from; at < to; at += NT * kEight * kTurns) {
        Eight<T> v[kTurns];
#pragma unroll
        for (int u = 0; u < kTurns; u++) {
            const int64_t i = at + (u * NT + (int)threadIdx.x) * kEight;
            const int count = (int)min((int64_t)kEight, max((int64_t)0, to - i));
            v[u].load(row + (count ? i : from), count, (T)-__builtin_inff());
        }
        float top = mine.top;
#pragma unroll
        for (int u = 0; u < kTurns; u++) {
#pragma unroll
            for (int i = 0; i < kEight; i++) {
                top = fmaxf(top, (float)v[u].v[i]);
            }
        }
        const float r = top == -__builtin_inff() ? 0.f : top;
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < kTurns; u++) {
#pragma unroll
            for (int i = 0; i < kEight; i++) {
                sum += exponential<T>((float)v[u].v[i], r, p);
            }
        }
        // what was there becomes relative to the larger one
        mine.sum = mine.sum * (mine.top == -__builtin_inff() ? 1.0 : (double)exponential<float>(mine.top, r, p)) + (double)sum;
        mine.top = top;
    }
    return joined<NT>(mine, p, box);
}

// v as 32 bits that are rounded to T next: for 16-bit types toward zero with the last bit set if anything was lost, which gives what rounding
// v itself would.
template <typename T>
__device__ __forceinline__ float before_rounding(double v)
{
    const float f = (float)v;
    if constexpr (sizeof(T) == 4) {
        return f;
    } else {
        const double lost = v - (double)f;
        const uint32_t bits = __float_as_uint(f);
        return fabs(lost) > 0.0 ? __uint_as_float((bits - ((lost < 0.0) != ((int)bits < 0) ? 1u : 0u)) | 1u) : f;
    }
}

// The teacher's entries of rows, in LDS.  A crew works on them: the first wavefront, without a barrier, while the others go on; or
// where there are many the whole workgroup.  Its thread j has entries j, j + threads() ...
template <int NT>
struct Entries {
    struct Buffer {
        double *log_p;      // to the base of 2; later p
        int *column;        // -1: not there
        float *value;       // the score at the column, later the gradient
    };
    uint8_t *buffers;
    uint32_t *key, *first, *count;      // a table of the columns in the gradient's part
    double *box;
    int k, slots;
    bool alone;

    __device__ __forceinline__ Entries(const DistilParams &p, uint8_t *smem, double *box)
        : buffers(smem), key(reinterpret_cast<uint32_t *>(smem + p.buffers * buffer_bytes(p.k))), first(key + p.slots),
          count(first + p.slots), box(box), k(p.k), slots(p.slots), alone(p.k <= kAlone)
    {
    }
    static __host__ __device__ __forceinline__ uint32_t buffer_bytes(int k) { return (uint32_t)(k + (k & 1)) * 16; }
    __device__ __forceinline__ Buffer buffer(int which) const
    {
        double *const log_p = reinterpret_cast<double *>(buffers + which * buffer_bytes(k));
        int *const column = reinterpret_cast<int *>(log_p + k);
        return {log_p, column, reinterpret_cast<float *>(column + k)};
    }
    __device__ __forceinline__ bool crew() const { return !alone || __builtin_amdgcn_readfirstlane(threadIdx.x) < 64; }
    __device__ __forceinline__ int threads() const { return alone ? 64 : NT; }
    __device__ __forceinline__ int self() const
    {
        int j = threadIdx.x;
        asm volatile("" : "+v"(j));      // addresses are computed for each row: kept for all, they would not fit into registers
        return j;
    }
    __device__ __forceinline__ void sync() const
    {
        if (alone) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        } else {
            __syncthreads();
        }
    }
    template <typename Op>
    __device__ __forceinline__ double over(double v, Op op) const
    {
        v = over_wave(v, op);
        if (!alone) {
            __syncthreads();
            if ((threadIdx.x & 63) == 0) {
                box[threadIdx.x >> 6] = v;
            }
            __syncthreads();
            v = over_lanes_of<NT / 64>(box[threadIdx.x & (NT / 64 - 1)], op);
        }
        return v;
    }
    static __device__ __forceinline__ bool in_part(int column, int64_t from, int64_t to) { return column >= from && column < to; }

    // A row's labels, log p, and the scores at those in from ... to - 1; returns P.
    template <typename T>
    __device__ __forceinline__ double load(const Buffer &b, const DistilParams &p, int64_t row, int64_t from, int64_t to) const
    {
        const T *const scores = static_cast<const T *>(p.scores) + row * p.ld;
        const int64_t *const labels = p.labels + row * k;
        const float *const teacher = p.teacher + row * k;
        const int me = self();
        double top = -__builtin_inf();
#pragma unroll 2
        for (int j = me; j < k; j += threads()) {
            const int64_t l = labels[j];
            const double t = (double)teacher[j] * p.scale;
            const bool there = l >= 0 && l < p.n;
            b.column[j] = there ? (int)l : -1;
            b.log_p[j] = there ? t : -__builtin_inf();
            b.value[j] = there && l >= from && l < to ? (float)scores[l] : 0.f;
            top = there ? fmax(top, t) : top;
        }
        double lse;
        if (p.whole) {
            lse = (double)p.whole[row] * kLog2e;
        } else {
            top = over(top, [](double x, double y) { return fmax(x, y); });
            const double r = top == -__builtin_inf() ? 0.0 : top;
            double sum = 0.0;
            for (int j = me; j < k; j += threads()) {
                sum += b.column[j] >= 0 ? any_power_of_two(b.log_p[j] - r) : 0.0;
            }
            sum = over(sum, [](double x, double y) { return x + y; });
            lse = sum == 0.0 ? 0.0 : r + log2_of(sum);      // no entry above -infinity: p is 0
        }
        double total = 0.0;
        for (int j = me; j < k; j += threads()) {
            if (b.column[j] >= 0) {
                const double log_p = b.log_p[j] - lse;
                b.log_p[j] = log_p;
                total += any_power_of_two(log_p);
            }
        }
        return over(total, [](double x, double y) { return x + y; });
    }

    __device__ __forceinline__ void write_loss(const Buffer &b, const DistilParams &p, int64_t row, const Sum &all) const
    {
        const double log_sum = log2_of(all.sum);
        double loss = 0.0;
        for (int j = self(); j < k; j += threads()) {
            const double log_p = b.log_p[j], prob = any_power_of_two(log_p);      // 0 times infinity is nothing
            if (b.column[j] >= 0 && prob != 0.0) {
                loss += prob * (log_p - (((double)b.value[j] - (double)all.reference()) * p.scale - log_sum));
            }
        }
        loss = over(loss, [](double x, double y) { return x + y; });
        if (threadIdx.x == 0) {
            if (p.loss) {
                p.loss[row] = all.sum == 0.0 ? 0.f : (float)(loss * kLn2 * p.temperature * p.temperature);
            }
            if (p.stats) {
                p.stats[row * 2] = all.top;
                p.stats[row * 2 + 1] = (float)all.sum;
            }
        }
    }

    __device__ __forceinline__ int place(uint32_t of, bool insert) const
    {
        uint32_t at = (of * 2654435761u) & (uint32_t)(slots - 1);
        for (;;) {
            const uint32_t have = insert ? atomicCAS(&key[at], 0xffffffffu, of) : key[at];
            if (have == of || have == 0xffffffffu) {
                return (int)at;     // the table has twice as many places as there are labels
            }
            at = (at + 1) & (uint32_t)(slots - 1);
        }
    }
    __device__ __forceinline__ bool is_first(int j, int column) const { return first[place((uint32_t)column, false)] == (uint32_t)j; }

    // The gradient at the labels in from ... to - 1: unit (P q - sum of p)
    template <typename T>
    __device__ __forceinline__ void differentiate(const Buffer &b, const DistilParams &p, int64_t from, int64_t to, float reference,
                                                  float sum, double whole, double unit) const
    {
        const int me = self();
        for (int i = me; i < slots; i += threads()) {
            key[i] = first[i] = 0xffffffffu;
            count[i] = 0;
        }
        sync();
        for (int j = me; j < k; j += threads()) {
            const int column = b.column[j];
            b.log_p[j] = any_power_of_two(b.log_p[j]);
            if (in_part(column, from, to)) {
                const int at = place((uint32_t)column, true);
                atomicMin(&first[at], (uint32_t)j);
                atomicAdd(&count[at], 1u);
            }
        }
        sync();
        const double share = whole / (double)sum;
        for (int j = me; j < k; j += threads()) {
            const int column = b.column[j];
            if (in_part(column, from, to) && is_first(j, column)) {
                double prob = b.log_p[j];
                if (count[place((uint32_t)column, false)] > 1) {      // the same label again: added in the entries' order
                    for (int i = j + 1; i < k; i++) {
                        prob += b.column[i] == column ? b.log_p[i] : 0.0;
                    }
                }
                const double q = any_power_of_two(((double)b.value[j] - (double)reference) * p.scale) * share;
                b.value[j] = before_rounding<T>(unit * (q - prob));
            }
        }
    }
    // Columns with labels, behind all others.
    template <typename T>
    __device__ __forceinline__ void write(const Buffer &b, T *gradient, int64_t from, int64_t to) const
    {
        for (int j = self(); j < k; j += threads()) {
            const int column = b.column[j];
            if (in_part(column, from, to) && is_first(j, column)) {
                gradient[column] = (T)b.value[j];
            }
        }
    }
};

// One workgroup per row or per part of a row.
template <typename T>
__global__ __launch_bounds__(kThreads) void distil_sum_kernel(DistilParams p)
{
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ double box[kThreads / 64];
    __shared__ Sum sums[kThreads / 64];
    const int64_t row = blockIdx.x / p.parts, part = blockIdx.x - row * p.parts;
    const T *const scores = static_cast<const T *>(p.scores) + row * p.ld;
    const Sum all = sum_of<T, kThreads>(p, scores, part * p.part, min(p.n, (part + 1) * p.part), sums);
    if (p.parts == 1) {
        const Entries<kThreads> entries(p, smem, box);
        if (entries.crew()) {
            entries.template load<T>(entries.buffer(0), p, row, 0, p.n);
            entries.write_loss(entries.buffer(0), p, row, all);
        }
    } else if (threadIdx.x == 0) {
        p.partial[blockIdx.x * 2] = all.top;
        p.partial[blockIdx.x * 2 + 1] = all.sum;
    }
}

// The parts of a row, joined in their order.
template <typename T>
__global__ __launch_bounds__(kThreads) void distil_join_kernel(DistilParams p)
{
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ double box[kThreads / 64];
    const int64_t row = blockIdx.x;
    const Entries<kThreads> entries(p, smem, box);
    if (entries.crew()) {
        const double *const of = p.partial + row * p.parts * 2;
        Sum all{-__builtin_inff(), 0.0};
        for (int i = 0; i < p.parts; i++) {
            all.join((float)of[i * 2], of[i * 2 + 1], p);
        }
        entries.template load<T>(entries.buffer(0), p, row, 0, p.n);
        entries.write_loss(entries.buffer(0), p, row, all);
    }
}

// What is computed from v is computed again behind this, rather than kept.
template <typename T>
__device__ __forceinline__ void forget(Eight<T> &v)
{
    typedef uint32_t Words __attribute__((ext_vector_type(sizeof(v.v) / 4)));
    Words w = __builtin_bit_cast(Words, v.v);
    asm volatile("" : "+v"(w));
    v.v = __builtin_bit_cast(typename Eight<T>::Lane, w);
}

// What a row's gradient is made of.
template <typename T>
struct Gradient {
    Exponent<T> exponent;
    double unit;
    float sum, factor;
    bool nothing;
    __device__ __forceinline__ Gradient(const DistilParams &p, int64_t row, float top, float sum, double whole)
        : exponent(top, p), unit((p.row_weight ? (double)p.row_weight[row] : 1.0) * p.temperature), sum(sum),
          factor((float)(unit * whole * exponent.factor() / (double)sum)),
          nothing(__builtin_amdgcn_readfirstlane(sum == 0.f || whole == 0.0))      // the same in all lanes
    {
    }
    // eight scores
    __device__ __forceinline__ void of(Eight<T> &v, const DistilParams &p) const
    {
        if (nothing) {
            v.v = (T)0.f;
            return;
        }
        typedef float Floats __attribute__((ext_vector_type(kEight)));
        Floats g;
#pragma unroll
        for (int c = 0; c < kEight; c++) {
            g[c] = exponent((float)v.v[c], p) * factor;
        }
        v.v = __builtin_convertvector(g, typename Eight<T>::Lane);
    }
};

// One workgroup per part of a row.
template <typename T>
__global__ __launch_bounds__(kThreads) void distil_gradient_kernel(DistilParams p)
{
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ double box[kThreads / 64], whole;
    const int64_t row = blockIdx.x / p.parts, from = (blockIdx.x - row * p.parts) * p.part, to = min(p.n, from + p.part);
    const T *const scores = static_cast<const T *>(p.scores) + row * p.ld;
    T *const gradient = static_cast<T *>(p.gradient) + row * p.ld_gradient;
    Eight<T> v[kTurns];
    auto load = [&](int64_t at) {
#pragma unroll
        for (int u = 0; u < kTurns; u++) {
            const int64_t i = at + (u * kThreads + (int)threadIdx.x) * kEight;
            const int count = (int)min((int64_t)kEight, max((int64_t)0, to - i));
            v[u].load(scores + (count ? i : from), count, (T)-__builtin_inff());
        }
    };
    load(from);
    const Entries<kThreads> entries(p, smem, box);
    if (entries.crew()) {
        const double sum = entries.template load<T>(entries.buffer(0), p, row, from, to);
        if (threadIdx.x == 0) {
            whole = sum;
        }
    }
    __syncthreads();       // the scores at labels have been read: the gradient may take their place
    const Gradient<T> all(p, row, p.given_stats[row * 2], p.given_stats[row * 2 + 1], whole);
    if (entries.crew() && !all.nothing) {
        entries.template differentiate<T>(entries.buffer(0), p, from, to, all.exponent.reference, all.sum, whole, all.unit);
    }
    for (int64_t at = from; at < to; at += kPart) {
#pragma unroll
        for (int u = 0; u < kTurns; u++) {
            const int64_t i = at + (u * kThreads + (int)threadIdx.x) * kEight;
            all.of(v[u], p);
            v[u].template store<true>(gradient + min(i, to), (int)min((int64_t)kEight, to - i));
        }
        if (at + kPart < to) {
            load(at + kPart);
        }
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);     // vmcnt(0): a column's first value is in memory before its second is sent
    __syncthreads();
    if (entries.crew() && !all.nothing) {
        entries.write(entries.buffer(0), gradient, from, to);
    }
}

// Workgroups with rows of their own, which stay in registers, EIGHTS times eight scores of a thread's: loss and gradient.  A row is
// read while the gradient of the one before it is written.
template <typename T, int NT, int EIGHTS>
__global__ __launch_bounds__(NT, 4) void distil_row_kernel(DistilParams p)
{
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ double box[NT / 64], whole_of[2];
    __shared__ Sum sums[2][NT / 64];
    const int whole = (int)p.n & ~(kEight - 1), left = (int)p.n - whole;     // the last scores are single ones
    Eight<T> v[EIGHTS];
    T last;
    // Eight scores of a thread (a row has eight at least), the first of the row's in place of those past its end.  No branch around it, or the scores would be waited for
    // where the branch ends.
    auto load = [&](int u, const T *scores, int end, uint32_t at) {
        const int from = u * NT * kEight;
        at = from + (int)at < end ? at : 0u;
        v[u].load(reinterpret_cast<const T *>(reinterpret_cast<const char *>(scores + (from < end ? from : 0)) + at * sizeof(T)),
                  kEight, (T)0.f);
    };
    auto load_last = [&](const T *scores) {
        last = (int)threadIdx.x < left ? scores[whole + (int)threadIdx.x] : (T)-__builtin_inff();
    };
    {
        int end = whole;
        uint32_t at = threadIdx.x * kEight;
        asm volatile("" : "+s"(end), "+v"(at));
#pragma unroll
        for (int u = 0; u < EIGHTS; u++) {
            load(u, static_cast<const T *>(p.scores) + blockIdx.x * p.ld, end, at);
        }
    }
    load_last(static_cast<const T *>(p.scores) + blockIdx.x * p.ld);
    const Entries<NT> entries(p, smem, box);
    auto load_entries = [&](int64_t row, int which) {
        const double sum = entries.template load<T>(entries.buffer(which), p, row, 0, p.n);
        if (threadIdx.x == 0) {
            whole_of[which] = sum;
        }
    };
    if (entries.crew()) {
        load_entries(blockIdx.x, 0);
    }
    T *before = nullptr;       // a gradient whose columns with labels are not written yet
    int which = 0;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, which ^= 1) {
        // what follows from these is computed for each row: kept for all of them it would not fit into the registers
        int end = whole;
        uint32_t at = threadIdx.x * kEight;
        asm volatile("" : "+s"(end), "+v"(at));
        float top = (float)last;
#pragma unroll
        for (int u = 0; u < EIGHTS; u++) {
            if ((u + 1) * NT * kEight > end) {
                if (u * NT * kEight + (int)at >= end) {
                    v[u].v = (T)-__builtin_inff();
                }
            }
#pragma unroll
            for (int c = 0; c < kEight; c++) {
                top = fmaxf(top, (float)v[u].v[c]);
            }
        }
        const Exponent<T> mine(top, p);
        float part = 0.f;
        double sum = (double)mine((float)last, p);
        asm volatile("" : "+s"(end), "+v"(at));
#pragma unroll
        for (int u = 0; u < EIGHTS; u++) {
            if (u * NT * kEight < end) {
                forget(v[u]);
#pragma unroll
                for (int c = 0; c < kEight; c++) {
                    part += mine((float)v[u].v[c], p);
                }
            }
            if (u % 4 == 3) {
                sum += (double)part;
                part = 0.f;
            }
        }
        const int64_t next = row + gridDim.x;
        __builtin_amdgcn_s_waitcnt(0x0f70);     // vmcnt(0): what is before has been written
        const Sum all = joined<NT>({top, sum * mine.factor()}, p, sums[which]);
        const double mass = whole_of[which];
        const Gradient<T> g(p, row, all.top, (float)all.sum, mass);
        if (entries.crew()) {
            if (before) {
                entries.write(entries.buffer(which ^ 1), before, 0, p.n);
            }
            const auto buffer = entries.buffer(which);
            entries.write_loss(buffer, p, row, all);
            if (!g.nothing) {
                entries.template differentiate<T>(buffer, p, 0, p.n, g.exponent.reference, g.sum, mass, g.unit);
            }
            if (next < p.rows) {
                load_entries(next, which ^ 1);
            }
        }
        T *const gradient = static_cast<T *>(p.gradient) + row * p.ld_gradient;
        const T *const scores = static_cast<const T *>(p.scores) + (next < p.rows ? next : row) * p.ld;
        asm volatile("" : "+s"(end), "+v"(at));
#pragma unroll
        for (int u = 0; u < EIGHTS; u++) {
            const int from = u * NT * kEight;
            if (from < end) {
                forget(v[u]);
                g.of(v[u], p);
                if (from + (int)at < end) {
                    v[u].template store<true>(
                        reinterpret_cast<T *>(reinterpret_cast<char *>(gradient + from) + at * sizeof(T)), kEight);
                }
            }
            load(u, scores, next < p.rows ? end : 0, at);
        }
        if ((int)threadIdx.x < left) {
            Eight<T> one;
            one.v = last;
            g.of(one, p);
            gradient[whole + (int)threadIdx.x] = one.v[0];
        }
        load_last(scores);
        before = g.nothing ? nullptr : gradient;
    }
    if (before) {
        __builtin_amdgcn_s_waitcnt(0x0f70);
        __syncthreads();
        if (entries.crew()) {
            entries.write(entries.buffer(which ^ 1), before, 0, p.n);
        }
    }
}

// Parts of a row so that about `groups` workgroups share the work, of at least `least` scores each.
int parts_for(int64_t rows, int64_t n, int64_t groups, int64_t least)
{
    const int64_t most = std::max<int64_t>(1, (n + least - 1) / least);
    return (int)std::min(most, std::max<int64_t>(1, groups / std::max<int64_t>(rows, 1)));
}
int sum_parts(int64_t rows, int64_t n) { return parts_for(rows, n, 2048, kPart); }

DistilParams params_of(const DistilTask &t)
{
    DistilParams p{};
    p.scores = t.scores;
    p.ld = t.ld;
    p.n = t.n;
    p.rows = t.rows;
    p.labels = t.labels;
    p.teacher = t.teacher;
    p.whole = t.whole;
    p.k = t.k;
    p.buffers = 1;
    p.temperature = t.temperature;
    p.scale = kLog2e / (double)t.temperature;
    p.high = (float)p.scale;
    p.low = (float)(p.scale - (double)p.high);
    return p;
}
void set_parts(DistilParams &p, int parts)
{
    // whole turns of a workgroup
    p.part = std::max<int64_t>(kPart, round_up((p.n + parts - 1) / parts, kPart));
    p.parts = (int)std::max<int64_t>(1, (p.n + p.part - 1) / p.part);
}

void check_task(const char *op, const DistilTask &t)
{
    check_type(op, t.type);
    check_scores(op, t.rows, t.n);
    check_row_buffer(op, t.scores, t.ld, t.type, t.rows, t.n);
    IXA_REQUIRE(t.k >= 0 && t.k <= kMaxTeacher, kErrInvalidParam, "%s: %d entries per row (0 ... %d)", op, t.k, kMaxTeacher);
    IXA_REQUIRE((t.labels && t.teacher) || t.rows == 0 || t.k == 0, kErrInvalidParam, "operator buffers can not be nullptr.");
    IXA_REQUIRE(on_bytes(t.labels, 8) && on_bytes(t.teacher, 4) && on_bytes(t.whole, 4), kErrInvalidParam,
                "%s: the teacher's entries are not aligned to their elements", op);
    IXA_REQUIRE(t.temperature >= 1e-6f && t.temperature <= 1e6f, kErrInvalidParam, "%s: temperature %g (1e-6 ... 1e6)", op,
                (double)t.temperature);
}

int slots_for(int k) { return std::max(64, pow2_ceil(2 * k)); }
size_t entry_bytes(const DistilParams &p)
{
    return (size_t)p.buffers * Entries<kThreads>::buffer_bytes(p.k) + (size_t)p.slots * 12;
}

void launch(void (*kernel)(DistilParams), int64_t groups, int threads, size_t lds, const DistilParams &p, hipStream_t s)
{
    require_dynamic_lds(reinterpret_cast<const void *>(kernel), lds);
    hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(threads), lds, s, p);
    check_launch();
}

void run_loss(const DistilTask &t, float *loss, float *stats, double *partial, hipStream_t s)
{
    DistilParams p = params_of(t);
    p.loss = loss;
    p.stats = stats;
    p.partial = partial;
    set_parts(p, sum_parts(t.rows, t.n));
    with_type(t.type, [&](auto e) {
        typedef decltype(e) T;
        launch(distil_sum_kernel<T>, t.rows * p.parts, kThreads, p.parts == 1 ? entry_bytes(p) : 0, p, s);
        if (p.parts > 1) {
            launch(distil_join_kernel<T>, t.rows, kThreads, entry_bytes(p), p, s);
        }
    });
}

void run_gradient(const DistilTask &t, const float *stats, const float *row_weight, void *gradient, int64_t ld_gradient,
                  hipStream_t s)
{
    DistilParams p = params_of(t);
    p.given_stats = stats;
    p.row_weight = row_weight;
    p.gradient = gradient;
    p.ld_gradient = ld_gradient;
    p.slots = slots_for(t.k);
    // parts of 32 KB of scores, or less where there are few (4096 rows of 131072 bf16: 381 us, 404 with 16 KB and 410 with 64 KB;
    // 999 of 100003 fp32: 162 us, 175 with 64 KB)
    set_parts(p, std::max(parts_for(t.rows, t.n, 2048, kPart), parts_for(1, t.n, 1 << 20, (t.type == kTypeF32 ? 1 : 2) * kPart)));
    with_type(t.type, [&](auto e) { launch(distil_gradient_kernel<decltype(e)>, t.rows * p.parts, kThreads, entry_bytes(p), p, s); });
}

template <int NT, int EIGHTS>
void run_rows(const DistilTask &t, const float *row_weight, float *loss, void *gradient, int64_t ld_gradient, hipStream_t s)
{
    DistilParams p = params_of(t);
    p.row_weight = row_weight;
    p.loss = loss;
    p.gradient = gradient;
    p.ld_gradient = ld_gradient;
    p.slots = slots_for(t.k);
    p.buffers = 2;
    with_type(t.type, [&](auto e) {
        typedef decltype(e) T;
        // as many workgroups as are resident at once
        const auto kernel = distil_row_kernel<T, NT, std::max(EIGHTS / (sizeof(T) == 4 ? 2 : 1), 4)>;
        require_dynamic_lds(reinterpret_cast<const void *>(kernel), entry_bytes(p));
        const int64_t groups = resident_workgroups(reinterpret_cast<const void *>(kernel), NT, entry_bytes(p));
        launch(kernel, std::min(t.rows, groups), NT, entry_bytes(p), p, s);
    });
}

// Rows that fit into a workgroup's registers, 256 bytes of each thread's, are read once.  From 2048 rows on a wavefront or two of
// them take a row (4096 rows of 8192 bf16: 38.5 us, 47.2 with 256 threads; 1024 rows: 20.0 and 17.6), but not where there is more to do
// about the labels.  Fewer than 128 rows of more than 8192 go in parts, as longer ones do (32 rows of 131072 bf16: 18.2 us, 20.8 in registers, 64 rows
// 20.5 and 20.4, 128 rows 30.8 and 20.3; 96 rows of 32768 fp32 16.4 and 17.6, 160 rows 19.6 and 16.6; but 64 rows of 9000 fp32 19.8 and 14.2).
bool in_rows(const DistilTask &t, const float *row_weight, float *loss, void *gradient, int64_t ld_gradient, hipStream_t s)
{
    const int64_t threads = (t.n + 127) / 128 * (int64_t)(element_bytes(t.type) / 2);
    if (t.n < kEight || threads > 1024) {
        return false;
    }
    if (t.rows >= 2048 && t.k <= kAlone && threads <= (t.n <= 256 * 4 * kEight ? 64 : 128)) {
        threads <= 64 ? run_rows<64, 16>(t, row_weight, loss, gradient, ld_gradient, s)
                      : run_rows<128, 16>(t, row_weight, loss, gradient, ld_gradient, s);
    } else if (t.n <= 256 * 4 * kEight) {
        run_rows<256, 4>(t, row_weight, loss, gradient, ld_gradient, s);
    } else if (t.rows < 128) {
        return false;
    } else if (threads <= 256) {
        run_rows<256, 16>(t, row_weight, loss, gradient, ld_gradient, s);
    } else if (threads <= 512) {
        run_rows<512, 16>(t, row_weight, loss, gradient, ld_gradient, s);
    } else {
        run_rows<1024, 16>(t, row_weight, loss, gradient, ld_gradient, s);
    }
    return true;
}

void check_gradient(const char *op, const DistilTask &t, const float *row_weight, const void *gradient, int64_t ld_gradient)
{
    check_row_buffer(op, gradient, ld_gradient, t.type, t.rows, t.n);
    IXA_REQUIRE(on_bytes(row_weight, 4), kErrInvalidParam, "%s: weights of rows are not aligned to their elements", op);
    IXA_REQUIRE(t.rows == 0 || t.n == 0 || !rows_collide(gradient, ld_gradient, t.scores, t.ld, t.type, t.rows, t.n), kErrInvalidParam,
                "%s: the gradient's rows have to be the scores' own (same address and stride) or share no element with them", op);
}

}  // namespace

int64_t distil_workspace(int64_t rows, int64_t n)
{
    check_scores("distil", rows, n);
    // sums of the parts and, for a step, two numbers per row
    return rows == 0 ? 0 : round_up(rows * sum_parts(rows, n) * 16, 256) + round_up(rows * 8, 256);
}

void op_distil_loss(const DistilTask &t, float *loss, float *stats, void *workspace, int64_t workspace_bytes, hipStream_t s)
{
    check_task("distil_loss", t);
    IXA_REQUIRE(loss || t.rows == 0, kErrInvalidParam, "operator buffers can not be nullptr.");
    IXA_REQUIRE(on_bytes(loss, 4) && on_bytes(stats, 4), kErrInvalidParam, "distil_loss: results are not aligned to their elements");
    if (t.rows == 0) {
        return;
    }
    check_workspace("distil_loss", workspace, workspace_bytes, distil_workspace(t.rows, t.n));
    int device;
    check_answer(hipGetDevice(&device));
    run_loss(t, loss, stats, static_cast<double *>(workspace), s);
}

void op_distil_gradient(const DistilTask &t, const float *stats, const float *row_weight, void *gradient, int64_t ld_gradient,
                        hipStream_t s)
{
    check_task("distil_gradient", t);
    check_gradient("distil_gradient", t, row_weight, gradient, ld_gradient);
    IXA_REQUIRE(stats || t.rows == 0, kErrInvalidParam, "operator buffers can not be nullptr.");
    IXA_REQUIRE(on_bytes(stats, 4), kErrInvalidParam, "distil_gradient: statistics are not aligned to their elements");
    if (t.rows == 0 || t.n == 0) {
        return;
    }
    int device;
    check_answer(hipGetDevice(&device));
    run_gradient(t, stats, row_weight, gradient, ld_gradient, s);
}

void op_distil_step(const DistilTask &t, const float *row_weight, float *loss, void *gradient, int64_t ld_gradient,
                    void *workspace, int64_t workspace_bytes, hipStream_t s)
{
    check_task("distil_step", t);
    check_gradient("distil_step", t, row_weight, gradient, ld_gradient);
    IXA_REQUIRE(loss || t.rows == 0, kErrInvalidParam, "operator buffers can not be nullptr.");
    IXA_REQUIRE(on_bytes(loss, 4), kErrInvalidParam, "distil_step: results are not aligned to their elements");
    if (t.rows == 0) {
        return;
    }
    check_workspace("distil_step", workspace, workspace_bytes, distil_workspace(t.rows, t.n));
    int device;
    check_answer(hipGetDevice(&device));
    if (in_rows(t, row_weight, loss, gradient, ld_gradient, s)) {
        return;
    }
    double *const partial = static_cast<double *>(workspace);
    float *const stats = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) +
                                                   round_up(t.rows * sum_parts(t.rows, t.n) * 16, 256));
    run_loss(t, loss, stats, partial, s);
    if (t.n > 0) {
        run_gradient(t, stats, row_weight, gradient, ld_gradient, s);
    }
}

}  // namespace ixa
