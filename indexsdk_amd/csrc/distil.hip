// The loss of rows of scores against a teacher's top entries, and its gradient.  For a row of scores s_0 ... s_(n-1) and a teacher's
// k entries (label l_j, score t_j), with one temperature T:
//   p_j = exp(t_j / T - L), L = log sum_j exp(t_j / T) over the entries that are there, or given (the teacher's over all columns)
//   q_i = exp(s_i / T) / sum_i exp(s_i / T),   P = sum_j p_j
//   loss = T^2 sum_j p_j (log p_j - log q_(l_j)),   d loss / d s_i = T (P q_i - sum of p_j with l_j = i)
// Entries with a label outside 0 ... n - 1 are not there.  Rows without an entry or without a score above -infinity have loss and
// gradient 0.
//
// All of it is bound by memory: the scores are read once for their largest and their sum of exponentials, and once more to
// write the gradient.  Exponentials of fp32 scores take 2^t of both parts of the product with log2(e) / T, those of 16-bit
// scores the rounded product; 32 of them are added in 32 bits, all else in 64, also what the teacher's entries need: the loss
// is a small difference of large logarithms.
#include "row_access.h"
#include "scores.h"

#include <algorithm>
#include <type_traits>

namespace ixa {

namespace {

constexpr int kThreads = 256;
constexpr int kTurns = 4;                         // times eight scores of a thread in flight
constexpr int kPart = kThreads * kEight * kTurns;   // scores that a workgroup reads at a time
constexpr int kEntries = kMaxTeacher / kThreads;  // a thread's
constexpr double kLog2e = 1.44269504088896340735992468, kLn2 = 0.693147180559945309417232;

struct DistilParams {
    const void *scores;
    int64_t ld, n, rows;
    const int64_t *labels;
    const float *teacher, *whole;
    int k, parts, slots;        // parts of a row; places of the table of labels
    double temperature;
    float high, low;            // log2(e) / T in two parts
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

// A largest score and the sum of exponentials relative to it (to 0 where there is none).
struct Sum {
    float top;
    double sum;
    __device__ __forceinline__ float reference() const { return top == -__builtin_inff() ? 0.f : top; }
    __device__ __forceinline__ void join(float other_top, double other_sum, const DistilParams &p)
    {
        const float both = fmaxf(top, other_top), r = both == -__builtin_inff() ? 0.f : both;
        // sums of nothing are 0 or no number
        const double mine = top == -__builtin_inff() ? 1.0 : exp2(((double)top - r) * kLog2e / p.temperature);
        const double others = other_top == -__builtin_inff() ? 1.0 : exp2(((double)other_top - r) * kLog2e / p.temperature);
        sum = sum * mine + other_sum * others;
        top = both;
    }
};

template <typename V, typename Op>
__device__ __forceinline__ V over_block(V v, V *box, Op op)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        v = op(v, __shfl_xor(v, o));
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        box[threadIdx.x >> 6] = v;
    }
    __syncthreads();
    v = box[0];
#pragma unroll
    for (int w = 1; w < kThreads / 64; w++) {
        v = op(v, box[w]);
    }
    return v;
}

// The sum over scores from ... to - 1 of a row, by the workgroup.
template <typename T>
__device__ Sum sum_of(const DistilParams &p, const T *row, int64_t from, int64_t to, double *box)
{
    Sum mine{-__builtin_inff(), 0.0};
    for (int64_t at = from; at < to; at += kPart) {
        Eight<T> v[kTurns];
#pragma unroll
        for (int u = 0; u < kTurns; u++) {
            const int64_t i = at + (u * kThreads + (int)threadIdx.x) * kEight;
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
    Sum all{over_block(mine.top, reinterpret_cast<float *>(box), [](float a, float b) { return fmaxf(a, b); }), 0.0};
    const float r = all.reference();
    const double part = mine.top == -__builtin_inff() ? mine.sum : mine.sum * exp2(((double)mine.top - r) * kLog2e / p.temperature);
    all.sum = over_block(part, box, [](double a, double b) { return a + b; });
    return all;
}

// A thread's entries of the teacher's: columns (-1: not there), log p and p; returns P, the same in every thread.
__device__ double entries_of(const DistilParams &p, int64_t row, int (&column)[kEntries], double (&log_p)[kEntries], double *box)
{
    double top = -__builtin_inf();
#pragma unroll
    for (int e = 0; e < kEntries; e++) {
        const int j = e * kThreads + (int)threadIdx.x;
        column[e] = -1;
        log_p[e] = -__builtin_inf();
        if (e * kThreads < p.k && j < p.k) {
            const int64_t l = p.labels[row * p.k + j];
            const double t = (double)p.teacher[row * p.k + j] / p.temperature;
            if (l >= 0 && l < p.n) {
                column[e] = (int)l;
                log_p[e] = t;
                top = fmax(top, t);
            }
        }
    }
    double lse;
    if (p.whole) {
        lse = p.whole[row];
    } else {
        top = over_block(top, box, [](double a, double b) { return fmax(a, b); });
        const double r = top == -__builtin_inf() ? 0.0 : top;
        double sum = 0.0;
#pragma unroll
        for (int e = 0; e < kEntries; e++) {
            sum += e * kThreads < p.k && column[e] >= 0 ? exp(log_p[e] - r) : 0.0;
        }
        sum = over_block(sum, box, [](double a, double b) { return a + b; });
        lse = sum == 0.0 ? 0.0 : r + log(sum);      // no entry above -infinity: p is 0
    }
    double total = 0.0;
#pragma unroll
    for (int e = 0; e < kEntries; e++) {
        if (e * kThreads < p.k && column[e] >= 0) {
            log_p[e] -= lse;
            total += exp(log_p[e]);
        }
    }
    return over_block(total, box, [](double a, double b) { return a + b; });
}

template <typename T>
__device__ void finish_loss(const DistilParams &p, int64_t row, const Sum &all, double *box)
{
    int column[kEntries];
    double log_p[kEntries];
    entries_of(p, row, column, log_p, box);
    const T *const scores = static_cast<const T *>(p.scores) + row * p.ld;
    const double log_sum = log(all.sum);
    double loss = 0.0;
#pragma unroll
    for (int e = 0; e < kEntries; e++) {
        const double prob = exp(log_p[e]);      // 0 times infinity is nothing
        if (e * kThreads < p.k && column[e] >= 0 && prob != 0.0) {
            const double log_q = ((double)(float)scores[column[e]] - (double)all.reference()) / p.temperature - log_sum;
            loss += prob * (log_p[e] - log_q);
        }
    }
    loss = over_block(loss, box, [](double a, double b) { return a + b; });
    if (threadIdx.x == 0) {
        if (p.loss) {
            p.loss[row] = all.sum == 0.0 ? 0.f : (float)(loss * p.temperature * p.temperature);
        }
        if (p.stats) {
            p.stats[row * 2] = all.top;
            p.stats[row * 2 + 1] = (float)all.sum;
        }
    }
}

// One workgroup per row or per part of a row.
template <typename T>
__global__ __launch_bounds__(kThreads) void distil_sum_kernel(DistilParams p)
{
    __shared__ double box[4];
    const int64_t row = blockIdx.x / p.parts, part = blockIdx.x - row * p.parts;
    const T *const scores = static_cast<const T *>(p.scores) + row * p.ld;
    const Sum all = sum_of(p, scores, part * p.part, min(p.n, (part + 1) * p.part), box);
    if (p.parts == 1) {
        finish_loss<T>(p, row, all, box);
    } else if (threadIdx.x == 0) {
        p.partial[blockIdx.x * 2] = all.top;
        p.partial[blockIdx.x * 2 + 1] = all.sum;
    }
}

// The parts of a row, joined in their order.
template <typename T>
__global__ __launch_bounds__(kThreads) void distil_join_kernel(DistilParams p)
{
    __shared__ double box[4];
    const int64_t row = blockIdx.x;
    const double *const of = p.partial + row * p.parts * 2;
    Sum all{-__builtin_inff(), 0.0};
    for (int i = 0; i < p.parts; i++) {
        all.join((float)of[i * 2], of[i * 2 + 1], p);
    }
    finish_loss<T>(p, row, all, box);
}

// The labels of a row that lie in one part of it, each once, in a table in LDS.
struct Labels {
    uint32_t *key, *first, *count;
    int slots;
    float *prob;
    int *column;
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
};

// The gradient of one part of a row.  Columns with labels are written once more behind the others.
template <typename T>
__global__ __launch_bounds__(kThreads) void distil_gradient_kernel(DistilParams p)
{
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ double box[4];
    const int64_t row = blockIdx.x / p.parts, from = (blockIdx.x - row * p.parts) * p.part, to = min(p.n, from + p.part);
    const T *const scores = static_cast<const T *>(p.scores) + row * p.ld;
    T *const gradient = static_cast<T *>(p.gradient) + row * p.ld_gradient;
    uint32_t *const table = reinterpret_cast<uint32_t *>(smem);
    const Labels labels{table, table + p.slots, table + 2 * p.slots, p.slots, reinterpret_cast<float *>(table + 3 * p.slots),
                        reinterpret_cast<int *>(table + 3 * p.slots) + p.k};
    for (int i = threadIdx.x; i < p.slots; i += kThreads) {
        labels.key[i] = 0xffffffffu;
        labels.first[i] = 0xffffffffu;
        labels.count[i] = 0;
    }
    int column[kEntries];
    double log_p[kEntries];
    const double whole = entries_of(p, row, column, log_p, box);
    const float top = p.given_stats[row * 2], sum = p.given_stats[row * 2 + 1];
    const float reference = top == -__builtin_inff() ? 0.f : top;
    const double unit = (p.row_weight ? (double)p.row_weight[row] : 1.0) * p.temperature;
    const bool nothing = sum == 0.f || whole == 0.0;
    const float factor = nothing ? 0.f : (float)(unit * whole / (double)sum);
    auto mine = [&](int e) { return e * kThreads < p.k && column[e] >= from && column[e] < to && !nothing; };
#pragma unroll
    for (int e = 0; e < kEntries; e++) {
        const int j = e * kThreads + (int)threadIdx.x;
        if (e * kThreads < p.k && j < p.k) {
            labels.prob[j] = (float)exp(log_p[e]);
            labels.column[j] = column[e];
        }
        if (mine(e)) {
            const int at = labels.place((uint32_t)column[e], true);
            atomicMin(&labels.first[at], (uint32_t)j);
            atomicAdd(&labels.count[at], 1u);
        }
    }
    __syncthreads();
    T value[kEntries];
#pragma unroll
    for (int e = 0; e < kEntries; e++) {
        const int j = e * kThreads + (int)threadIdx.x;
        value[e] = (T)0.f;
        if (mine(e)) {
            const int at = labels.place((uint32_t)column[e], false);
            if (labels.first[at] != (uint32_t)j) {
                column[e] = -1;
                continue;
            }
            double prob = exp(log_p[e]);
            if (labels.count[at] > 1) {      // the same label again: added in the entries' order
                for (int i = j + 1; i < p.k; i++) {
                    prob += labels.column[i] == column[e] ? (double)labels.prob[i] : 0.0;
                }
            }
            const double q = exp(((double)(float)scores[column[e]] - (double)reference) / p.temperature) / (double)sum;
            value[e] = (T)(float)(unit * (whole * q - prob));
        }
    }
    __syncthreads();       // the scores at labels have been read: the gradient may take their place
    for (int64_t at = from; at < to; at += kPart) {
        Eight<T> v[kTurns];
#pragma unroll
        for (int u = 0; u < kTurns; u++) {
            const int64_t i = at + (u * kThreads + (int)threadIdx.x) * kEight;
            const int count = (int)min((int64_t)kEight, max((int64_t)0, to - i));
            v[u].load(scores + (count ? i : from), count, (T)-__builtin_inff());
        }
#pragma unroll
        for (int u = 0; u < kTurns; u++) {
            const int64_t i = at + (u * kThreads + (int)threadIdx.x) * kEight;
#pragma unroll
            for (int c = 0; c < kEight; c++) {
                const float g = exponential<T>((float)v[u].v[c], reference, p) * factor;
                v[u].v[c] = (T)(nothing ? 0.f : g);
            }
            v[u].store(gradient + min(i, to), (int)min((int64_t)kEight, to - i));
        }
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);     // vmcnt(0): a column's first value is in memory before its second is sent
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kEntries; e++) {
        if (mine(e)) {
            gradient[column[e]] = value[e];
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
    p.temperature = t.temperature;
    const double scale = kLog2e / (double)t.temperature;
    p.high = (float)scale;
    p.low = (float)(scale - (double)p.high);
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

void run_loss(const DistilTask &t, float *loss, float *stats, double *partial, hipStream_t s)
{
    DistilParams p = params_of(t);
    p.loss = loss;
    p.stats = stats;
    p.partial = partial;
    set_parts(p, sum_parts(t.rows, t.n));
    with_type(t.type, [&](auto e) {
        typedef decltype(e) T;
        hipLaunchKernelGGL((distil_sum_kernel<T>), dim3((unsigned)(t.rows * p.parts)), dim3(kThreads), 0, s, p);
        check_launch();
        if (p.parts > 1) {
            hipLaunchKernelGGL((distil_join_kernel<T>), dim3((unsigned)t.rows), dim3(kThreads), 0, s, p);
            check_launch();
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
    p.slots = std::max(64, pow2_ceil(2 * t.k));
    set_parts(p, std::max(parts_for(t.rows, t.n, 2048, kPart), parts_for(1, t.n, 1 << 20, 2 * kPart)));
    const size_t lds = (size_t)p.slots * 12 + (size_t)t.k * 8;
    with_type(t.type, [&](auto e) {
        const auto kern = distil_gradient_kernel<decltype(e)>;
        require_dynamic_lds(reinterpret_cast<const void *>(kern), lds);
        hipLaunchKernelGGL(kern, dim3((unsigned)(t.rows * p.parts)), dim3(kThreads), lds, s, p);
        check_launch();
    });
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
    double *const partial = static_cast<double *>(workspace);
    float *const stats = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) +
                                                   round_up(t.rows * sum_parts(t.rows, t.n) * 16, 256));
    run_loss(t, loss, stats, partial, s);
    if (t.n > 0) {
        run_gradient(t, stats, row_weight, gradient, ld_gradient, s);
    }
}

}  // namespace ixa
