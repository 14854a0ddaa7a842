// The gated delta rule: jobs of its launches and device helpers they share.
//
// One matrix S (Dk x Dv, fp32) per sequence and value head, per token:
//     S <- e^g S;   u = beta (v - S^T k);   S <- S + k u^T;   o = scale S^T q
#pragma once

#include "ramnet_device.hpp"

namespace ramnet {

enum : int { kDeltaMaxDk = 256, kDeltaChunk = 64, kDeltaReach = 1 << 30 };

// Tensors of one call; strides in elements, of batch row, token and head (the
// last dimension is dense). Value head h reads key head h / (Hv / Hk).
struct DeltaJob {
    const void *q, *k, *v;      // (B, T, Hk, Dk) twice, (B, T, Hv, Dv)
    const void *g, *beta;       // (B, T, Hv)
    const float *init;          // (N, Hv, Dk, Dv), or null: zeros
    float *state;               // (N, Hv, Dk, Dv); may be init
    void *o;                    // (B, T, Hv, Dv), dense
    const int32_t *cu;          // (N + 1) bounds of packed sequences (B == 1), or null: N == B
    const int32_t *lengths;     // (B) tokens that count, or null: all
    int dtype, g_dtype, beta_dtype;
    int B, T, N, Hk, Hv, Dk, Dv;
    float scale;
    int64_t q_at[3], k_at[3], v_at[3], g_at[3], beta_at[3];
};

// Workspace of a call in chunks of 64 tokens (one record per chunk and value
// head, record = chunk * Hv + head), and what a training forward keeps.
struct DeltaWork {
    int32_t *offsets;  // (N + 1) first chunk of each packed sequence; null where sequences are rows
    int32_t *order;    // (N) packed sequences, longest first; null likewise
    double *gamma;     // [record][64] running sums of the decays within the chunk, in powers of 2
    float *vec;        // [record][8][64] scales and decays of the tokens (delta_split.hpp)
    uint32_t *y;       // [record][2][6][64][4] N^-1 as matrix operands of fp16 parts (backward: transposed)
    uint32_t *p_frags; // the same of scale lower(Q K^T . L) diag(beta) (backward: transposed, without beta)
    float *p;          // [record][64][64] scale lower(Q K^T . L)    (backward)
    float *bl;         // [record][64][64] strictlower(K K^T . L)   (backward)
    // rows of Dv values, zeros up to a multiple of 8 (delta_row):
    float *x;          // [record][64][..] gradient of the values    (backward)
    float *dstate;     // [record][Dk][..] gradient after the chunk  (backward)
    float *e;          // [record][64][..] v - S^T k of each token   (kept)
    float *states;     // [record][Dk][..] state before the chunk    (kept)
    // where the time axis of a row is cut into segments that run side by side (parts > 1),
    // per row, value head and segment:
    float *ends;       // [Dk][Dv] state after the segment: first from zeros (the first from init), then in full;
                       //   in the last place the row's init
    float *maps;       // [wide][wide] what the segment makes of the state before it (kept)
    int parts, part_chunks, uncut;  // (at most; chunks of one; the most chunks that a row is not cut at)
    int per_row;       // chunks of a row where sequences are rows
    int chunks;        // records / Hv
};

// Gradients; those of the inputs have their types, strides dense.
struct DeltaGrads {
    const void *d_o;       // (B, T, Hv, Dv), strides d_o_at
    const float *d_state;  // (N, Hv, Dk, Dv), or null: zeros
    void *dq, *dk, *dv, *dg, *dbeta;
    float *dinit;          // or null
    int64_t d_o_at[3];
};

__device__ __forceinline__ float load_code(const void *p, int code, int64_t at) {
    if (code == 0)
        return static_cast<const float *>(p)[at];
    if (code == 1)
        return static_cast<float>(static_cast<const _Float16 *>(p)[at]);
    return load_f32(static_cast<const bf16_t *>(p) + at);
}

// A value that all lanes share, in a scalar register.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Tokens of one sequence: `len` from token t0 of batch row b. Bounds that are
// out of order or out of range give fewer tokens, never ones outside [0, T).
struct DeltaSpan {
    int b, t0, len;
};

__device__ __forceinline__ DeltaSpan delta_span(const DeltaJob &job, int n) {
    if (job.cu) {
        const int lo = min(max(job.cu[n], 0), job.T), hi = min(max(job.cu[n + 1], lo), job.T);
        return {0, lo, hi - lo};
    }
    return {n, 0, job.lengths ? min(max(job.lengths[n], 0), job.T) : job.T};
}

// Dk as the chunked kernels are built for it.
inline int delta_padded(int Dk) {
    return Dk <= 32 ? 32 : Dk <= 64 ? 64 : Dk <= 96 ? 96 : Dk <= 128 ? 128 : Dk <= 160 ? 160 : 256;
}

// Length of a row of Dv values in the workspace.
__host__ __device__ inline int delta_row(int Dv) { return (Dv + 7) / 8 * 8; }

// Whether a head's matrix in the workspace, its rows padded, ends within the reach of
// the chunked kernels' 32-bit offsets (delta_split.hpp: kNowhere lies past every window).
inline bool delta_within_reach(const DeltaJob &job) {
    return static_cast<int64_t>(delta_padded(job.Dk)) * delta_row(job.Dv) * 4 <= kDeltaReach;
}

// A decay of one step. e^-200 is 0 in fp32 as e^-inf is; held there, sums of
// decays stay finite and differences of them free of inf - inf. (A NaN stays.)
__device__ __forceinline__ float delta_decay(float g) { return g < -200.f ? -200.f : g; }

}  // namespace ramnet
