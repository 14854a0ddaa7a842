// Verification of drafted tokens. Draft s of a row stays if all before it did
// and accept_s q(x_s) < p(x_s) (q = 1 where the drafts have no probabilities).
// With n drafts kept, one more token is drawn from the target's place n:
// after a refused draft from max(p - q, 0) (p without x_n where there are no
// probabilities; p itself where nothing is left), else from p. It is the
// first index whose running sum passes sample * total, among those with a
// weight above 0.
//
// Bound by reading one target row and one draft row of V; small batches by the
// latency of what depends on what (tokens, their probabilities, the rows). One
// block a row of the batch: each of its 16 waves sums one stretch of the
// vocabulary, then the block walks the one stretch in which the threshold falls
// (it comes from the L2) with a running sum in order. All sums in 64 bits, in a
// fixed order: a draw next to a border of the running sum would go by the
// rounding of 32. What waves find is put together by ballots: LDS atomics on one
// word go lane by lane (20 us of a call). 192 rows of 128257 in fp32 (197 MB): 45 us,
// 4.4 TB/s; one row of 32000: 9 us of latency.
#include "ramnet_device.hpp"
#include "ramnet_kernels.hpp"

namespace ramnet {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / kWave;

template<typename Scalar>
struct Piece {
    static constexpr int kN = 16 / sizeof(Scalar);
    uint32_t w[4];
    __device__ __forceinline__ float operator[](int e) const {
        if constexpr (sizeof(Scalar) == 4)
            return __uint_as_float(w[e]);
        else
            return bits_f32<Scalar>((w[e / 2] >> (e % 2 * 16)) & 0xFFFFu);
    }
};

// 16 bytes at an element's alignment (a row of odd length begins anywhere).
template<typename Scalar>
__device__ __forceinline__ Piece<Scalar> load_piece(const Scalar *p) {
    struct __attribute__((packed, aligned(sizeof(Scalar)))) Raw {
        uint32_t w[4];
    };
    const Raw r = *reinterpret_cast<const Raw *>(p);
    return {{r.w[0], r.w[1], r.w[2], r.w[3]}};
}

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1)
        x += __shfl_xor(x, m);
    return x;
}

template<typename Scalar>
__global__ __launch_bounds__(kThreads) void verify_kernel(const VerifyJob job) {
    __shared__ double sums[kWaves], scan[kWaves];
    __shared__ int refused_s[kWaves], found_s[kWaves], last_s[kWaves];
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int64_t b = blockIdx.x;
    const int V = job.V, S = job.S;
    const int64_t *tokens = job.tokens + b * S;
    const Scalar *target = static_cast<const Scalar *>(job.target) + b * job.target_at[0];
    const Scalar *draft = job.draft ? static_cast<const Scalar *>(job.draft) + b * job.draft_at[0] : nullptr;
    // the first place that is refused
    const int len = job.lens ? min(max(job.lens[b], 0), S) : S;
    int first = S;
    for (int s0 = wave * kWave; s0 < S; s0 += kThreads) {
        const int s = s0 + lane;
        bool stays = s >= S;
        if (s < S) {
            const int64_t x = tokens[s];
            const double accept = job.accept[b * S + s];
            if (s < len && x >= 0 && x < V) {
                const double p = load_f32(target + s * job.target_at[1] + x);
                const double q = draft ? static_cast<double>(load_f32(draft + s * job.draft_at[1] + x)) : 1.0;
                stays = accept * q < p;
            }
        }
        const uint64_t out = __ballot(!stays);
        if (out) {
            first = s0 + __ffsll(static_cast<unsigned long long>(out)) - 1;
            break;
        }
    }
    if (lane == 0)
        refused_s[wave] = first;
    __syncthreads();
    int n = S;
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
        n = min(n, refused_s[w]);
    const bool refused = n < len;
    const Scalar *p = target + n * job.target_at[1];
    const Scalar *q = refused && draft ? draft + n * job.draft_at[1] : nullptr;
    const int64_t ruled = refused && !draft ? tokens[n] : -1;
    const int without = ruled >= 0 && ruled < V ? static_cast<int>(ruled) : -1;

    // (comparisons keep a NaN, as a maximum of torch does; fmax would drop it)
    auto left = [&](float pv, float qv, int at) {
        const double d = static_cast<double>(pv) - (q ? static_cast<double>(qv) : 0.0);
        return at == without || d < 0.0 ? 0.0 : d;
    };

    // the sums of each wave's stretch: whole pieces, and for the last wave the row's
    // last few elements, one a lane
    constexpr int N = Piece<Scalar>::kN, kDeep = 4;
    const int part = (V + kWaves * N - 1) / (kWaves * N) * N, full = V / N * N;
    const int lo = min(wave * part, full), hi = min(lo + part, full);
    const bool tail = wave == kWaves - 1 && full + lane < V;
    auto stretch = [&](auto weight) {
        double sum = tail ? weight(load_f32(p + full + lane), q ? load_f32(q + full + lane) : 0.f, full + lane) : 0.0;
        for (int at = lo + lane * N; at < hi; at += kDeep * kWave * N) {
            Piece<Scalar> x[kDeep], y[kDeep];
#pragma unroll
            for (int i = 0; i < kDeep; ++i) {
                const int from = at + i * kWave * N;
                x[i] = from < hi ? load_piece(p + from) : Piece<Scalar>{};
                y[i] = q && from < hi ? load_piece(q + from) : Piece<Scalar>{};
            }
#pragma unroll
            for (int i = 0; i < kDeep; ++i)
#pragma unroll
                for (int e = 0; e < N; ++e)
                    sum += weight(x[i][e], y[i][e], at + i * kWave * N + e);
        }
        sum = wave_sum(sum);
        if (lane == 0)
            sums[wave] = sum;
        __syncthreads();
        double total = 0.0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
            total += sums[w];
        return total;
    };
    double total = stretch(left);
    const bool own = refused && !(total > 0.0);  // nothing is left (or a NaN): the target's own weights
    if (own) {
        __syncthreads();
        total = stretch([](float pv, float, int) { return static_cast<double>(pv); });
    }
    const double border = static_cast<double>(job.sample[b]) * total;
    double seen = 0.0, before = 0.0;  // the sums before the next stretch, and before at_wave's
    int at_wave = -1;
    for (int w = 0; w < kWaves; ++w) {
        if (sums[w] > 0.0) {
            at_wave = w, before = seen;  // (stays at the last one with a weight where rounding lets none pass)
            if (seen + sums[w] > border)
                break;
        }
        seen += sums[w];
    }
    int found = V, last = -1;
    if (at_wave >= 0) {
        const int from = min(at_wave * part, full), to = at_wave == kWaves - 1 ? V : min(from + part, full);
        const int each = (to - from + kThreads - 1) / kThreads;
        const int begin = min(from + tid * each, to), end = min(begin + each, to);
        auto weight = [&](int i) {
            const float pv = load_f32(p + i);
            return own ? static_cast<double>(pv) : left(pv, q ? load_f32(q + i) : 0.f, i);
        };
        double mine = 0.0;
        for (int i = begin; i < end; ++i)
            mine += weight(i);
        double run = mine;
#pragma unroll
        for (int m = 1; m < kWave; m <<= 1) {
            const double x = __shfl_up(run, m);
            run += lane >= m ? x : 0.0;
        }
        if (lane == kWave - 1)
            scan[wave] = run;
        __syncthreads();
        for (int w = 0; w < wave; ++w)
            before += scan[w];
        run = before + (run - mine);
        for (int i = begin; i < end && found == V; ++i) {
            const double x = weight(i);
            run += x;
            if (x > 0.0) {
                last = i;
                found = run > border ? i : V;
            }
        }
    }
    // threads have the vocabulary in order: the first that found, the last with a weight
    const uint64_t finds = __ballot(found < V), any = __ballot(last >= 0);
    if (finds)
        found = __shfl(found, __ffsll(static_cast<unsigned long long>(finds)) - 1);
    if (any)
        last = __shfl(last, kWave - 1 - __clzll(static_cast<long long>(any)));
    if (lane == 0)
        found_s[wave] = finds ? found : V, last_s[wave] = any ? last : -1;
    __syncthreads();
    int64_t *out = job.out + b * (S + 1);
    int chosen = V, highest = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
        chosen = min(chosen, found_s[w]), highest = max(highest, last_s[w]);
    // (none passes by rounding, or with a sample of 1: the last one with a weight; a NaN gives 0)
    if (chosen == V)
        chosen = border == border ? highest : 0;
    for (int s = tid; s <= S; s += kThreads)
        out[s] = s < n ? tokens[s] : s == n ? chosen : -1;
    if (tid == 0)
        job.taken[b] = n;
}

}  // namespace

hipError_t launch_verify_drafts(const VerifyJob &job, hipStream_t stream, const char **why) {
    const dim3 grid(static_cast<unsigned>(job.B)), block(kThreads);
    switch (job.dtype) {
        case kF32: hipLaunchKernelGGL(verify_kernel<float>, grid, block, 0, stream, job); break;
        case kF16: hipLaunchKernelGGL(verify_kernel<_Float16>, grid, block, 0, stream, job); break;
        case kBF16: hipLaunchKernelGGL(verify_kernel<bf16_t>, grid, block, 0, stream, job); break;
        default: *why = "verify_drafts: unsupported dtype"; return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace ramnet
