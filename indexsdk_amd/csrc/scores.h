// Operators on rows of scores: columns drawn from them, and their loss against a teacher's top entries (see sample.hip and
// distil.hip).
#pragma once
#include "lowp.h"

namespace ixa {

constexpr int64_t kMaxScoreRows = 1 << 22, kMaxScoreColumns = 0x7fffffff;
constexpr int kMaxTeacher = 2048;     // entries per row, the most that a top-k selection returns

inline void check_scores(const char *op, int64_t rows, int64_t n)
{
    IXA_REQUIRE(rows >= 0 && rows <= kMaxScoreRows && n >= 0 && n <= kMaxScoreColumns, kErrInvalidParam,
                "%s: rows %ld (0 ... %ld), columns %ld (< 2^31)", op, (long)rows, (long)kMaxScoreRows, (long)n);
}
inline void check_workspace(const char *op, const void *workspace, int64_t have, int64_t need)
{
    IXA_REQUIRE(need == 0 || (workspace && have >= need && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0), kErrInvalidParam,
                "%s: needs a workspace of %ld bytes on 16, has %ld", op, (long)need, (long)have);
}

// `draws` columns of each row of scores[rows][ld], see sample.hip.  temperature, top_k, top_p, min_p [rows] may be null.
int64_t sample_workspace(int64_t rows, int64_t n);
void op_sample(const void *scores, int64_t ld, int type, int64_t rows, int64_t n, const float *temperature, const int32_t *top_k,
               const float *top_p, const float *min_p, const float *uniform, int draws, int64_t *labels, float *probs,
               void *workspace, int64_t workspace_bytes, hipStream_t s);

// What a teacher says about rows of scores, and the loss against it, see distil.hip.
struct DistilTask {
    const void *scores;
    int64_t ld;
    int type;
    int64_t rows, n;
    const int64_t *labels;     // [rows][k]
    const float *teacher;      // [rows][k]
    int k;
    const float *whole;        // [rows] or null
    float temperature;
};
int64_t distil_workspace(int64_t rows, int64_t n);
void op_distil_loss(const DistilTask &task, float *loss, float *stats, void *workspace, int64_t workspace_bytes, hipStream_t s);
void op_distil_gradient(const DistilTask &task, const float *stats, const float *row_weight, void *gradient, int64_t ld_gradient,
                        hipStream_t s);
void op_distil_step(const DistilTask &task, const float *row_weight, float *loss, void *gradient, int64_t ld_gradient,
                    void *workspace, int64_t workspace_bytes, hipStream_t s);

}  // namespace ixa
