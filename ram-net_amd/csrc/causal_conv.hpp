// The short causal convolution: jobs of its launches.
//
//     s[t, d] = bias[d] + sum_j weight[d, j] x[t - (W - 1) + j, d];   y = s or silu(s)
//
// Inputs before a sequence's first token are the rows of its state (zeros without one).
#pragma once

#include "sequences.hpp"

namespace ramnet {

enum : int { kConvMaxWidth = 8 };

struct ConvJob {
    SequenceJob seq;
    const void *x;             // (B, T, D), strides x_at of batch row and token
    const void *weight, *bias; // (D, W); (D) or null
    const void *init;          // (N, W - 1, D), or null: zeros
    void *y, *state;           // (B, T, D) dense; (N, W - 1, D), may be init
    int dtype, D, W, silu;
    int64_t x_at[2];
    int step;                  // tokens of a piece, at least kConvMaxWidth
};

// Gradients, in the inputs' types, dense.
struct ConvGrads {
    const void *dy;      // (B, T, D), strides dy_at
    const void *dstate;  // (N, W - 1, D), or null: zeros
    void *dx, *dinit;    // dinit may be null
    void *dweight, *dbias;  // dbias may be null
    float *partial;      // [piece][W + 1][D] sums of dweight and dbias
    int64_t dy_at[2];
};

// Tokens of a piece, and bytes of the workspace of a call.
int conv_step(const ConvJob &job, bool backward);
int64_t conv_layout(ConvJob &job, bool backward, char *base, ConvGrads *grads);
hipError_t launch_conv(const ConvJob &job, hipStream_t stream, const char **why);
hipError_t launch_conv_backward(const ConvJob &job, const ConvGrads &grads, hipStream_t stream, const char **why);

}  // namespace ramnet
