// The pieces of packed sequences: their bounds in order, and a running count of pieces.
#include "sequences.hpp"

namespace ramnet {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / kWave;

// One block, 1024 sequences a turn: a running maximum of the bounds, then a running sum of
// the pieces, each by shuffles within a wave and over the waves' results in LDS. Latency
// alone: 4 us for up to 1024 sequences.
__global__ __launch_bounds__(kThreads) void sequences_kernel(const SequenceJob job, int step) {
    __shared__ int tops[kWaves], sums[kWaves];
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave, wave = tid / kWave, N = job.N;
    int top = 0, total = 0;  // of the turns before
    for (int base = 0; base <= N; base += kThreads) {
        const int n = base + tid;
        int lo = clamped(job.cu[min(n, N)], 0, job.T);
#pragma unroll
        for (int m = 1; m < kWave; m <<= 1)
            lo = max(lo, __shfl_up(lo, m));
        if (lane == kWave - 1)
            tops[wave] = lo;
        __syncthreads();
        int before = top;
        for (int w = 0; w < kWaves; ++w) {
            before = w < wave ? max(before, tops[w]) : before;
            top = max(top, tops[w]);
        }
        lo = max(lo, before);
        const int hi = max(lo, clamped(job.cu[min(n + 1, N)], 0, job.T));
        const int mine = n < N ? pieces_of(hi - lo, step) : 0;
        int run = mine;
#pragma unroll
        for (int m = 1; m < kWave; m <<= 1) {
            const int x = __shfl_up(run, m);
            run += lane >= m ? x : 0;
        }
        if (lane == kWave - 1)
            sums[wave] = run;
        __syncthreads();
        int start = total;
        for (int w = 0; w < kWaves; ++w) {
            start += w < wave ? sums[w] : 0;
            total += sums[w];
        }
        if (n <= N) {
            job.bounds[n] = lo;
            job.first[n] = start + run - mine;
        }
        __syncthreads();
    }
}

}  // namespace

hipError_t launch_sequences(const SequenceJob &job, int step, hipStream_t stream) {
    hipLaunchKernelGGL(sequences_kernel, dim3(1), dim3(kThreads), 0, stream, job, step);
    return hipGetLastError();
}

}  // namespace ramnet
