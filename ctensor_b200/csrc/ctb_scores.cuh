// Host-visible interface of the attention-score kernels (ctb_scores.cu).
#pragma once
#include "ctb_common.cuh"

namespace ctb {

// An operand [batch, heads, queries, keys] with unit stride along the keys.
struct ScoreRows {
    const float* p;
    int64_t sb, sh, sq;
    int64_t even;                       // distance of consecutive rows in (batch, head, query) order, -1: none; set by the launchers
};
// An Int32 rule table with a stride per dim; p == NULL: the rule is absent.
struct ScoreTable {
    const int32_t* p;
    int64_t sb, si;
};

struct ScoreGeom {
    int64_t batch, heads, queries, keys;
    float scale, cap, over_cap;         // over_cap = scale / cap where cap > 0
    int32_t causal;
    ScoreTable query_start, key_lengths, prefix, query_docs, key_docs;
    const float* slopes;
    int64_t slope_stride;
};

int launch_score_softmax(const ScoreGeom& g, ScoreRows scores, float* out, cudaStream_t stream);
// grad_slopes may be NULL; `partials` (one double per row) is used with it.
int launch_score_softmax_backward(const ScoreGeom& g, ScoreRows grad, ScoreRows probs, ScoreRows scores, float* grad_scores,
                                  float* grad_slopes, double* partials, cudaStream_t stream);

}  // namespace ctb
