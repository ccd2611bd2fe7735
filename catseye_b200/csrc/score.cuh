// score.cuh — log probabilities of given tokens, with each row's entropy and
// its likeliest tokens.
#pragma once
#include "kv.cuh"

namespace cats {

constexpr int SCORE_MAX_K = 32;

struct ScoreArgs {
    const void *logits;      // [rows][ld], the first `vocab` of a row
    const int *targets;      // [rows], < 0: none (may be null)
    float *logprob;          // [rows] (may be null)
    float *entropy;          // [rows] (may be null)
    int *top_ids;            // [rows][k]
    float *top_logprob;      // [rows][k]
    long long ld;
    int rows, vocab, k;
    int *err;
};

cudaError_t launch_logprobs(const ScoreArgs &a, int type, cudaStream_t st);

} // namespace cats
