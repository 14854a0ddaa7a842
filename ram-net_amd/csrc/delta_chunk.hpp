// Chunked form of the gated delta rule: helpers of its kernels.
//
// Within a chunk of 64 tokens, gamma_i the sum of the decays up to token i and
// L_ij = e^(gamma_i - gamma_j) for i >= j:
//     Bl = strictlower(K K^T . L),  N = I + Bl diag(beta),  Y = N^-1
//     E = Y (V - e^gamma . K S)           (E_i = v_i - S_i^T k_i, decayed S_i)
//     O = scale e^gamma . (Q S) + P diag(beta) E,   P = scale lower(Q K^T . L)
//     S <- e^gamma_C S + K^T diag(e^(gamma_C - gamma) beta) E
#pragma once

#include "delta_rule.hpp"

#include <type_traits>

namespace ramnet {

constexpr double kLog2e = 1.4426950408889634;

// e^x for x in powers of 2: the difference of two sums of decays, rounded once.
__device__ __forceinline__ float decay_of(double x) { return __builtin_amdgcn_exp2f(static_cast<float>(x)); }

typedef float f32x4 __attribute__((ext_vector_type(4)));

// One 16x16 tile += A (16 x 4 steps) B: lane l gives A[l % 16][4 (l / 16) + r]
// and B[4 (l / 16) + r][l % 16] for the four steps r, and holds rows
// 4 (l / 16) + r of column l % 16: a result tile is a B operand as it lies.
__device__ __forceinline__ f32x4 mfma4(f32x4 a, f32x4 b, f32x4 c) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], b[r], c, 0, 0, 0);
    return c;
}

__device__ __forceinline__ f32x4 load4(const float *p) { return *reinterpret_cast<const f32x4 *>(p); }
// Four rows of a column.
__device__ __forceinline__ f32x4 load4(const float *p, int64_t step) {
    return f32x4{p[0], p[step], p[2 * step], p[3 * step]};
}

// A chunk: record-level place, its tokens t0 .. t0 + len of row b (len 0: none).
struct DeltaPlace {
    int n, b, t0, len;
};

__device__ __forceinline__ DeltaPlace delta_place(const DeltaJob &job, const DeltaWork &work, int chunk) {
    int n, first;
    if (work.offsets) {
        if (chunk >= work.offsets[job.N])
            return {-1, 0, 0, 0};
        int lo = 0, hi = job.N;  // offsets[lo] <= chunk < offsets[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (work.offsets[mid] <= chunk)
                lo = mid;
            else
                hi = mid;
        }
        n = lo;
        first = work.offsets[n];
    } else {
        n = chunk / work.per_row;
        first = n * work.per_row;
    }
    const DeltaSpan span = delta_span(job, n);
    const int from = (chunk - first) * kDeltaChunk;
    return {n, span.b, span.t0 + from, max(0, min(kDeltaChunk, span.len - from))};
}

// Tokens of no packed sequence lie before the first one and after the last. Chunks that
// no sequence has share them (there is one for every 64 of these tokens): f(from, to)
// for chunk `at`'s tokens (one block for all of them: 2.6 ms where 100 of 32768 count).
template<typename F>
__device__ __forceinline__ void delta_outside(const DeltaJob &job, const DeltaWork &work, int at, F f) {
    const int used = work.offsets[job.N], shares = work.chunks - used, share = at - used;
    const int before = delta_span(job, 0).t0;
    const DeltaSpan last = delta_span(job, job.N - 1);
    const int after = max(before, last.t0 + last.len);
    const int64_t tokens = before + (job.T - after);
    const int from = static_cast<int>(tokens * share / shares), to = static_cast<int>(tokens * (share + 1) / shares);
    f(min(from, before), min(to, before));
    f(max(from, before) - before + after, max(to, before) - before + after);
}

// The sequence whose states a chain's block walks.
__device__ __forceinline__ int delta_line(const DeltaWork &work, int at) { return work.order ? work.order[at] : at; }

// First chunk and number of chunks of a sequence.
__device__ __forceinline__ void delta_chunks(const DeltaJob &job, const DeltaWork &work, int n, const DeltaSpan &span,
                                             int &first, int &count) {
    count = (span.len + kDeltaChunk - 1) / kDeltaChunk;
    if (work.offsets) {
        first = work.offsets[n];
        count = min(count, work.offsets[n + 1] - first);  // (fewer only where the bounds are out of order)
    } else {
        first = n * work.per_row;
    }
}

// Which of `items` (and which of its `groups` column groups) block `at` has: an
// item's groups read the same keys and queries (and write parts of the same cache
// lines), so they go to one of the eight compute dies, which take blocks in turn, at
// one time.
__device__ __forceinline__ void split_block(int at, int groups, int items, int &group, int &item) {
    const int even = items / 8 * 8 * groups;
    if (at < even) {
        group = at / 8 % groups;
        item = at / 8 / groups * 8 + at % 8;
    } else {
        group = (at - even) % groups;
        item = items / 8 * 8 + (at - even) / groups;
    }
}

// Segments of a row of `count` chunks.
__device__ __forceinline__ int delta_segments(const DeltaWork &work, int count) {
    return count > work.uncut ? (count + work.part_chunks - 1) / work.part_chunks : 1;
}

constexpr int kLdsBytes = 160 * 1024;

// Whether rows of q and k are whole pieces of 16 bytes at 16-byte addresses.
template<typename Scalar>
__host__ __device__ inline bool rows_whole(const DeltaJob &job) {
    constexpr int V = 16 / static_cast<int>(sizeof(Scalar));
    const int64_t steps = job.q_at[0] | job.q_at[1] | job.q_at[2] | job.k_at[0] | job.k_at[1] | job.k_at[2];
    const uintptr_t starts = reinterpret_cast<uintptr_t>(job.q) | reinterpret_cast<uintptr_t>(job.k);
    return job.Dk % 8 == 0 && steps % V == 0 && starts % 16 == 0;
}

}  // namespace ramnet
