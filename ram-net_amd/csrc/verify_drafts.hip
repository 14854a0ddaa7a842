// Verification of drafted tokens. Draft s of a row stays if all before it did
// and accept_s q(x_s) < p(x_s) (q = 1 where the drafts have no probabilities).
// With n drafts kept, one more token is drawn from the target's place n:
// after a refused draft from max(p - q, 0) (p without x_n where there are no
// probabilities; p itself where nothing is left), else from p. It is the
// first index whose running sum passes sample * total, among those with a
// weight above 0.
//
// Bound by reading one target row and one draft row of V. One block a row of
// the batch: each of its 16 waves sums one stretch of the vocabulary, then the
// block walks the one stretch in which the threshold falls (it comes from the
// L2) with a running sum in order. All sums in 64 bits, in a fixed order: a
// draw next to a border of the running sum would go by the rounding of 32.
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
    __shared__ double sums[kWaves][2];
    __shared__ double scan[kWaves];
    __shared__ int taken_s, found_s, last_s;
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave, wave = tid / kWave;
    const int64_t b = blockIdx.x;
    const int V = job.V, S = job.S;
    const int64_t *tokens = job.tokens + b * S;
    const Scalar *target = static_cast<const Scalar *>(job.target) + b * job.target_at[0];
    const Scalar *draft = job.draft ? static_cast<const Scalar *>(job.draft) + b * job.draft_at[0] : nullptr;
    const int len = job.lens ? min(max(job.lens[b], 0), S) : S;

    if (tid == 0)
        taken_s = len, found_s = V, last_s = -1;
    __syncthreads();
    for (int s = tid; s < len; s += kThreads) {
        const int64_t x = tokens[s];
        bool stays = false;
        if (x >= 0 && x < V) {
            const double p = load_f32(target + s * job.target_at[1] + x);
            const double q = draft ? static_cast<double>(load_f32(draft + s * job.draft_at[1] + x)) : 1.0;
            stays = static_cast<double>(job.accept[b * S + s]) * q < p;
        }
        if (!stays)
            atomicMin(&taken_s, s);
    }
    __syncthreads();
    const int n = taken_s;
    const bool refused = n < len;
    const Scalar *p = target + n * job.target_at[1];
    const Scalar *q = refused && draft ? draft + n * job.draft_at[1] : nullptr;
    const int64_t without = refused && !draft ? tokens[n] : -1;

    // (comparisons keep a NaN, as a maximum of torch does; fmax would drop it)
    auto left = [&](float pv, float qv, int at) {
        const double d = static_cast<double>(pv) - (q ? static_cast<double>(qv) : 0.0);
        return at == without || d < 0.0 ? 0.0 : d;
    };

    // the sums of each wave's stretch
    constexpr int N = Piece<Scalar>::kN;
    const int part = (V + kWaves * N - 1) / (kWaves * N) * N;
    const int lo = min(wave * part, V), hi = min(lo + part, V);
    double rest = 0.0, whole = 0.0;
    constexpr int kDeep = 4;
    int at = lo + lane * N;
    for (; at + (kDeep - 1) * kWave * N + N <= hi; at += kDeep * kWave * N) {
        Piece<Scalar> a[kDeep], c[kDeep];
#pragma unroll
        for (int i = 0; i < kDeep; ++i) {
            a[i] = load_piece(p + at + i * kWave * N);
            c[i] = q ? load_piece(q + at + i * kWave * N) : Piece<Scalar>{};
        }
#pragma unroll
        for (int i = 0; i < kDeep; ++i)
#pragma unroll
            for (int e = 0; e < N; ++e) {
                rest += left(a[i][e], c[i][e], at + i * kWave * N + e);
                whole += static_cast<double>(a[i][e]);
            }
    }
    for (; at < hi; at += kWave * N) {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (at + e < hi) {
                const float pv = load_f32(p + at + e);
                rest += left(pv, q ? load_f32(q + at + e) : 0.f, at + e);
                whole += static_cast<double>(pv);
            }
    }
    rest = wave_sum(rest), whole = wave_sum(whole);
    if (lane == 0)
        sums[wave][0] = rest, sums[wave][1] = whole;
    __syncthreads();
    double total[2] = {0.0, 0.0};
    for (int w = 0; w < kWaves; ++w)
        total[0] += sums[w][0], total[1] += sums[w][1];
    const int kind = total[0] > 0.0 ? 0 : 1;  // (a NaN goes to the target's own weights)
    const double border = static_cast<double>(job.sample[b]) * total[kind];
    double seen = 0.0, before = 0.0;  // the sums before the next stretch, and before at_wave's
    int at_wave = -1;
    for (int w = 0; w < kWaves; ++w) {
        if (sums[w][kind] > 0.0) {
            at_wave = w, before = seen;  // (stays at the last one with a weight where rounding lets none pass)
            if (seen + sums[w][kind] > border)
                break;
        }
        seen += sums[w][kind];
    }
    if (at_wave >= 0) {
        seen = before;
        const int from = min(at_wave * part, V), to = min(from + part, V);
        const int each = (to - from + kThreads - 1) / kThreads;
        const int first = min(from + tid * each, to), end = min(first + each, to);
        auto weight = [&](int i) {
            const float pv = load_f32(p + i);
            return kind ? static_cast<double>(pv) : left(pv, q ? load_f32(q + i) : 0.f, i);
        };
        double mine = 0.0;
        for (int i = first; i < end; ++i)
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
            seen += scan[w];
        run = seen + (run - mine);
        for (int i = first; i < end; ++i) {
            const double x = weight(i);
            run += x;
            if (x > 0.0) {
                atomicMax(&last_s, i);
                if (run > border) {
                    atomicMin(&found_s, i);
                    break;
                }
            }
        }
    }
    __syncthreads();
    int64_t *out = job.out + b * (S + 1);
    // (none passes by rounding, or with a sample of 1: the last one with a weight; a NaN gives 0)
    const int chosen = found_s < V ? found_s : border == border ? max(last_s, 0) : 0;
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
