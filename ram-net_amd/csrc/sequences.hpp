// Sequences of a call and the pieces of time they are cut into, for operators
// that walk time: a piece is at most `step` consecutive tokens of one sequence.
//
// Sequences are the rows of a batch (of T tokens, or of `lengths`), or packed
// one after the other into a batch of one between the bounds `cu`. Bounds are
// read on the device: one below its forerunner or outside [0, T] is held to
// these, so that sequences never overlap and no token lies outside the tensors.
// Tokens of no sequence (behind a row's length, before the first bound, behind
// the last) are in pieces of their own, of sequence -1.
#pragma once

#include "ramnet_device.hpp"

namespace ramnet {

struct SequenceJob {
    const int32_t *cu;       // (N + 1), or null: N == B rows
    const int32_t *lengths;  // (B), or null: T
    int B, T, N;
    // of packed sequences, from launch_sequences: (N + 1) each
    int32_t *bounds;         // cu as it is used
    int32_t *first;          // first piece of each sequence; in the last place how many there are
};

// One piece; tokens count from the start of the row.
struct TimePiece {
    int seq, row;    // (seq -1: tokens of no sequence)
    int t0, len;     // its tokens
    int lo, hi;      // its sequence's
    int at, count;   // its place among its sequence's pieces, and how many these are
    int rest;        // tokens of no sequence directly behind it (rows of a length below T)
};

__host__ __device__ inline int pieces_of(int tokens, int step) { return tokens > 0 ? (tokens + step - 1) / step : 1; }

// How many pieces a call has at most. Every sequence has one at least, also an empty one.
__host__ __device__ inline int64_t most_pieces(const SequenceJob &job, int step) {
    if (job.cu)
        return static_cast<int64_t>(job.T) / step + job.N + 2;
    return static_cast<int64_t>(job.B) * pieces_of(job.T, step);
}

__device__ __forceinline__ int clamped(int x, int lo, int hi) { return min(max(x, lo), hi); }

// Piece p; false where there is none of that number.
__device__ inline bool time_piece(const SequenceJob &job, int step, int p, TimePiece &out) {
    if (!job.cu) {
        const int per_row = pieces_of(job.T, step), row = p / per_row, at = p - row * per_row;
        const int n = job.lengths ? clamped(job.lengths[row], 0, job.T) : job.T;
        const int t0 = at * step, t1 = min(t0 + step, job.T);
        out = {row, row, t0, clamped(n - t0, 0, t1 - t0), 0, n, at, pieces_of(n, step), 0};
        out.rest = t1 - t0 - out.len;
        return true;
    }
    const int N = job.N, total = job.first[N];
    if (p >= total) {  // before the first bound, then behind the last
        const int head = job.bounds[0], tail = job.bounds[N], heads = (head + step - 1) / step;
        const int at = p - total, t0 = at < heads ? at * step : tail + (at - heads) * step;
        const int end = at < heads ? head : job.T;
        out = {-1, 0, t0, 0, 0, 0, 0, 0, clamped(end - t0, 0, step)};
        return t0 < end;
    }
    int lo = 0, hi = N;  // first[lo] <= p < first[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (job.first[mid] <= p)
            lo = mid;
        else
            hi = mid;
    }
    const int begin = job.bounds[lo], end = job.bounds[lo + 1], at = p - job.first[lo];
    const int t0 = begin + at * step;
    out = {lo, 0, t0, min(step, end - t0), begin, end, at, pieces_of(end - begin, step), 0};
    return true;
}

// bounds and first of packed sequences cut into pieces of `step` tokens.
hipError_t launch_sequences(const SequenceJob &job, int step, hipStream_t stream);

}  // namespace ramnet
