// Orthogonalisation of matrices of few columns, as the gate weights of logic layers are: gram_steps.cu.
#pragma once

#include "common.cuh"

namespace dl {

constexpr int kGramColumns = 16;
constexpr int kMostSteps = 64;

struct GramMatrix {
    const void *g;
    float *momentum;   // null: g as it is
    void *out;         // the result, or the weights that are updated
    int64_t rows;
    float rate;
};
struct GramJob {
    static constexpr int kMost = 32;
    GramMatrix matrix[kMost];
    int count;
    int64_t batch;     // of matrices behind each other at entry 0, where there is one entry
    int cols, type;
    bool update;
    float keep, nesterov, decay;   // 1 - momentum; the momentum, or 1: the update is the momentum itself; of the weights
};

int64_t gram_workspace_bytes(int64_t matrices, int64_t rows, int sms);
int launch_gram_steps(const GramJob &job, int steps, const float *coefficients, double eps, double *workspace, int sms, cudaStream_t st,
                      const char *what);

}  // namespace dl
