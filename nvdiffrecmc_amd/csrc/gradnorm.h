// gradnorm.h -- what the clipped Adam step (optim.hip) shares with the gradient norm (gradnorm.hip).
#pragma once

#include "common.h"

// The counters of an Adam optimizer in device memory (nvdr_hip.h nvdr_adam_step): steps taken, a spare word, beta1^t, beta2^t as doubles.
// What one step needs of them, in the same arithmetic wherever it is computed:
struct AdamStep {
    float factor;               // of clipping
    float step_size;            // lr / (1 - beta1^t)
    float bc2_sqrt;             // sqrt(1 - beta2^t)
    int step;                   // t
};

__device__ __forceinline__ AdamStep adam_begin(const int *state, double lr, double beta1, double beta2)
{
    const double *pw = (const double *)(state + 2);
    AdamStep s;
    s.factor = 1.0f;
    s.step = state[0] + 1;
    const double b1p = (s.step == 1 ? 1.0 : pw[0]) * beta1, b2p = (s.step == 1 ? 1.0 : pw[1]) * beta2;
    s.step_size = (float)(lr / (1.0 - b1p));
    s.bc2_sqrt = (float)sqrt(1.0 - b2p);
    return s;
}

__device__ __forceinline__ void adam_advance(int *state, double beta1, double beta2)
{
    const int step = state[0] + 1;
    double *pw = (double *)(state + 2);
    pw[0] = (step == 1 ? 1.0 : pw[0]) * beta1;
    pw[1] = (step == 1 ? 1.0 : pw[1]) * beta2;
    state[0] = step;
}

struct AdamBegin {
    int *state;
    double lr, beta1, beta2;
    AdamStep *step;             // receives what the update reads
};

// The norm of the gradients of the tensors that are not frozen, times their grad_scale, into *norm, and the beginning of the step into *adam.step
int nvdr_adam_norm(const nvdr_adam_tensor *tensors, int n_tensors, int norm_type, double max_norm, double *workspace, int64_t workspace_len, float *norm,
                   const AdamBegin &adam, hipStream_t stream);
