// One token a row from a uniform number, and the probabilities it is drawn with.
//
// Weights are w_i = e^((l_i - max) / temperature) (a NaN counts as -inf, +inf as far above the rest).
// Tokens are ordered by descending logit, equal ones by index; each filter keeps a prefix of that order:
// the first top_k; of these, those whose sum of weights before them is below top_p times the sum of all; those of
// w >= min_p. The token is the lowest index of a kept one whose running sum (by index) passes random * sum.
//
// Weights are computed in 64 bits and added up as whole numbers of 2^-F: sums do not depend on their order,
// and a token next to a border does not go by the rounding of 32 bits.
//
// One block a row. The end of the prefix is found by counts and sums of the weights in 2048 bins, even in the
// logit; in the bin where it lies, by comparing all its tokens with each other.
#include "ramnet_kernels.hpp"
#include "vector16.hpp"

namespace ramnet {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / kWave, kBins = 2048, kList = 2048;

// A token's place in the order as one number, greater for earlier ones.
__device__ __forceinline__ uint64_t order_of(float l, int index) {
    const uint32_t bits = __float_as_uint(l);
    const uint32_t key = bits ^ (static_cast<uint32_t>(static_cast<int32_t>(bits) >> 31) | 0x80000000u);
    return static_cast<uint64_t>(key) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(index));
}
__device__ __forceinline__ float logit_of(uint64_t order) {
    const uint32_t key = static_cast<uint32_t>(order >> 32);
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

template<typename T, typename Op>
__device__ __forceinline__ T wave_reduce(T x, Op op) {
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1)
        x = op(x, __shfl_xor(x, m));
    return x;
}

struct Shared {
    uint32_t counts[kBins];
    uint64_t sums[kBins];
    uint64_t list[kList], weights[kList];
    uint64_t scan[2][kWaves];
    float tops[kWaves], lows[kWaves];
    uint64_t before, through;  // results that one thread finds
    int count_before, bin, listed;
    uint64_t order;
};

template<typename Scalar>
struct Sampler {
    const Scalar *row;
    int V, tid, lane, wave;
    Shared &s;
    float top, low;         // the greatest logit, the smallest finite one
    float scale;            // bins per unit of the logit
    double rate, unit;      // 1 / temperature, 2^F
    double least;           // min_p
    uint64_t border;        // order of the last token kept

    __device__ __forceinline__ float clean(float l) const { return l != l ? -INFINITY : l + 0.f; }

    // f(logit, index) for all tokens, 16 bytes a thread, all threads of the block side by side.
    template<typename F>
    __device__ __forceinline__ void sweep(F f) const {
        constexpr int N = 16 / sizeof(Scalar), kDeep = 4;
        const int full = V / N * N;
        for (int at = tid * N; at < full; at += kDeep * kThreads * N) {
            Vec<Scalar, N> x[kDeep];
#pragma unroll
            for (int i = 0; i < kDeep; ++i) {
                const int from = at + i * kThreads * N;
                x[i] = from < full ? load_vec<Scalar, N>(row + from) : Vec<Scalar, N>{};
            }
#pragma unroll
            for (int i = 0; i < kDeep; ++i) {
                const int from = at + i * kThreads * N;
                if (from < full) {
#pragma unroll
                    for (int e = 0; e < N; ++e)
                        f(clean(x[i][e]), from + e);
                }
            }
        }
        if (full + tid < V)
            f(clean(load_f32(row + full + tid)), full + tid);
    }

    __device__ __forceinline__ double weight(float l) const {
        if (l == top)
            return 1.0;
        return l == -INFINITY || top == INFINITY ? 0.0 : exp((static_cast<double>(l) - static_cast<double>(top)) * rate);
    }
    __device__ __forceinline__ uint64_t whole(double w) const { return static_cast<uint64_t>(w * unit + 0.5); }
    __device__ __forceinline__ int bin(float l) const {
        if (l == top)
            return 0;
        const float at = (top - l) * scale;  // (descending with l, whatever it rounds to)
        return at < static_cast<float>(kBins - 1) ? static_cast<int>(at) : kBins - 1;
    }
    // Whether a token is drawn from.
    __device__ __forceinline__ bool kept(float l, int index, double &w) const {
        if (order_of(l, index) < border)
            return false;
        w = weight(l);
        return w >= least && l > -INFINITY;
    }

    // The sums of x over the threads before, and over all.
    __device__ __forceinline__ uint64_t block_scan(uint64_t x, uint64_t &total, int which) {
        uint64_t run = x;
#pragma unroll
        for (int m = 1; m < kWave; m <<= 1) {
            const uint64_t y = __shfl_up(run, m);
            run += lane >= m ? y : 0;
        }
        __syncthreads();
        if (lane == kWave - 1)
            s.scan[which][wave] = run;
        __syncthreads();
        uint64_t before = 0;
        total = 0;
        for (int w = 0; w < kWaves; ++w) {
            before += w < wave ? s.scan[which][w] : 0;
            total += s.scan[which][w];
        }
        return before + run - x;
    }

    __device__ __forceinline__ void clear_bins() {
        __syncthreads();
        for (int i = tid; i < kBins; i += kThreads)
            s.counts[i] = 0, s.sums[i] = 0;
        __syncthreads();
    }

    // The first bin where tokens, or their weights, reach what is asked for: k tokens (target 0), or a sum of
    // `target` beyond `base`. False (in all threads) if none does.
    __device__ bool find_bin(uint64_t k, double target, uint64_t base, int first_count) {
        static_assert(kBins == 2 * kThreads, "two bins a thread");
        if (tid == 0)
            s.bin = -1;
        const uint64_t c0 = s.counts[2 * tid], c1 = s.counts[2 * tid + 1], w0 = s.sums[2 * tid], w1 = s.sums[2 * tid + 1];
        uint64_t all_c, all_w;
        uint64_t c = block_scan(c0 + c1, all_c, 0) + static_cast<uint64_t>(first_count), w = block_scan(w0 + w1, all_w, 1) + base;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint64_t ci = i ? c1 : c0, wi = i ? w1 : w0;
            const bool here = ci > 0 && (target > 0.0 ? static_cast<double>(w) < target && static_cast<double>(w + wi) >= target
                                                      : c < k && c + ci >= k);
            if (here)
                s.bin = 2 * tid + i, s.before = w, s.count_before = static_cast<int>(c);
            c += ci, w += wi;
        }
        __syncthreads();
        return s.bin >= 0;
    }

    // The order of the k-th token, or of the last one with less than `target` before it; `through`: the weights
    // up to it. The bins hold what find_bin needs.
    __device__ bool find_border(uint64_t k, double target, uint64_t &order, uint64_t &through) {
        if (!find_bin(k, target, 0, 0))
            return false;
        const int level = s.bin;
        uint64_t base = s.before, lo = 0, hi = ~0ull;
        int count_before = s.count_before, members = static_cast<int>(s.counts[level]);
        bool narrowed = false;
        auto member = [&](float l, uint64_t o) { return narrowed ? o >= lo && o <= hi : bin(l) == level; };
        while (members > kList) {
            if (!narrowed) {
                uint64_t least_o = ~0ull, most_o = 0;
                sweep([&](float l, int i) {
                    if (bin(l) == level) {
                        const uint64_t o = order_of(l, i);
                        least_o = min(least_o, o), most_o = max(most_o, o);
                    }
                });
                auto smaller = [](uint64_t a, uint64_t b) { return a < b ? a : b; };
                auto greater = [](uint64_t a, uint64_t b) { return a > b ? a : b; };
                least_o = wave_reduce(least_o, smaller), most_o = wave_reduce(most_o, greater);
                __syncthreads();
                if (lane == 0)
                    s.scan[0][wave] = least_o, s.scan[1][wave] = most_o;
                __syncthreads();
                lo = ~0ull, hi = 0;
                for (int w = 0; w < kWaves; ++w)
                    lo = smaller(lo, s.scan[0][w]), hi = greater(hi, s.scan[1][w]);
                narrowed = true;
            }
            // bins of equal width in the order, the greatest first
            int shift = 0;
            while (((hi - lo) >> shift) >= kBins)
                ++shift;
            clear_bins();
            sweep([&](float l, int i) {
                const uint64_t o = order_of(l, i);
                if (o >= lo && o <= hi) {
                    const int b = static_cast<int>((hi - o) >> shift);
                    atomicAdd(&s.counts[b], 1u);
                    atomicAdd(reinterpret_cast<unsigned long long *>(&s.sums[b]), whole(weight(l)));
                }
            });
            __syncthreads();
            if (!find_bin(k, target, base, count_before))
                return false;
            base = s.before, count_before = s.count_before;
            const int at = s.bin;
            members = static_cast<int>(s.counts[at]);
            const uint64_t most = hi - (static_cast<uint64_t>(at) << shift);
            const uint64_t width = (1ull << shift) - 1;
            lo = most - lo > width ? most - width : lo;
            hi = most;
        }
        __syncthreads();
        if (tid == 0)
            s.listed = 0;
        __syncthreads();
        sweep([&](float l, int i) {
            const uint64_t o = order_of(l, i);
            if (member(l, o)) {
                const int at = atomicAdd(&s.listed, 1);
                s.list[at] = o, s.weights[at] = whole(weight(l));
            }
        });
        __syncthreads();
        for (int i = tid; i < members; i += kThreads) {
            const uint64_t o = s.list[i], w = s.weights[i];
            uint64_t before = base;
            int rank = 0;
            for (int j = 0; j < members; ++j) {
                const bool ahead = s.list[j] > o;
                rank += ahead, before += ahead ? s.weights[j] : 0;
            }
            const bool last = target > 0.0 ? static_cast<double>(before) < target &&
                                                 (static_cast<double>(before + w) >= target || rank == members - 1)
                                           : static_cast<uint64_t>(count_before + rank + 1) == k;
            if (last)
                s.order = o, s.through = before + w;
        }
        __syncthreads();
        order = s.order, through = s.through;
        return true;
    }
};

__device__ __forceinline__ double setting(const float *of_rows, double of_all, int64_t row) {
    return of_rows ? static_cast<double>(of_rows[row]) : of_all;
}

template<typename Scalar>
__global__ __launch_bounds__(kThreads) void sample_kernel(const SampleJob job) {
    __shared__ Shared shared;
    const int64_t r = blockIdx.x;
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave, wave = tid / kWave, V = job.V;
    Sampler<Scalar> me{static_cast<const Scalar *>(job.logits) + r * job.row_at, V, tid, lane, wave, shared};
    float *probs = job.probs ? job.probs + r * V : nullptr;

    me.top = -INFINITY, me.low = INFINITY;
    me.sweep([&](float l, int) {
        me.top = l > me.top ? l : me.top;
        me.low = l > -INFINITY && l < me.low ? l : me.low;
    });
    me.top = wave_reduce(me.top, [](float a, float b) { return a > b ? a : b; });
    me.low = wave_reduce(me.low, [](float a, float b) { return a < b ? a : b; });
    if (lane == 0)
        shared.tops[wave] = me.top, shared.lows[wave] = me.low;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) {
        me.top = fmaxf(me.top, shared.tops[w]);
        me.low = fminf(me.low, shared.lows[w]);
    }
    if (me.top == -INFINITY) {  // nothing to draw from
        if (tid == 0 && job.tokens)
            job.tokens[r] = 0;
        for (int i = tid; probs && i < V; i += kThreads)
            probs[i] = 0.f;
        return;
    }
    const double temperature = setting(job.temperature, job.temperature_of_all, r);
    int64_t k = job.top_k ? job.top_k[r] : job.top_k_of_all;
    const double p = setting(job.top_p, job.top_p_of_all, r);
    me.rate = 1.0 / temperature;
    if (!(temperature > 0.0))  // the greatest alone
        k = 1, me.rate = 1.0;
    const double least = setting(job.min_p, job.min_p_of_all, r);
    me.least = least > 0.0 ? (least < 1.0 ? least : 1.0) : 0.0;
    me.unit = job.unit;
    const float range = me.top - me.low;
    me.scale = range > 0.f && range < INFINITY ? static_cast<float>(kBins - 1) / range : 0.f;
    me.border = 0;
    const bool by_count = k > 0 && k < V, by_sum = p < 1.0;
    if (by_count || by_sum) {
        me.clear_bins();
        uint64_t total = 0;
        me.sweep([&](float l, int) {
            const int b = me.bin(l);
            atomicAdd(&shared.counts[b], 1u);
            if (by_sum) {
                const uint64_t w = me.whole(me.weight(l));
                atomicAdd(reinterpret_cast<unsigned long long *>(&shared.sums[b]), w);
                total += w;
            }
        });
        uint64_t all = 0;
        me.block_scan(total, all, 0);
        uint64_t order = 0, through = 0;
        if (by_count && me.find_border(static_cast<uint64_t>(k), 0.0, order, through))
            me.border = order, all = through;
        if (by_sum) {
            // (a narrowed search by count has used the bins for its own)
            if (by_count) {
                me.clear_bins();
                me.sweep([&](float l, int i) {
                    if (order_of(l, i) >= me.border) {
                        const int b = me.bin(l);
                        atomicAdd(&shared.counts[b], 1u);
                        atomicAdd(reinterpret_cast<unsigned long long *>(&shared.sums[b]), me.whole(me.weight(l)));
                    }
                });
                __syncthreads();
            }
            const double target = p > 0.0 ? p * static_cast<double>(all) : 0.0;
            if (!(target > 0.0)) {
                if (me.find_border(1, 0.0, order, through))
                    me.border = order > me.border ? order : me.border;
            } else if (me.find_border(0, target, order, through)) {
                me.border = order > me.border ? order : me.border;
            }
        }
    }
    // The kept weights by stretches of the vocabulary, a wave each, in order of the index.
    const int part = (V + kWaves - 1) / kWaves, lo = min(wave * part, V), hi = min(lo + part, V);
    uint64_t sum = 0;
    for (int i = lo + lane; i < hi; i += kWave) {
        double w;
        sum += me.kept(me.clean(load_f32(me.row + i)), i, w) ? me.whole(w) : 0;
    }
    sum = wave_reduce(sum, [](uint64_t a, uint64_t b) { return a + b; });
    __syncthreads();
    if (lane == 0)
        shared.scan[0][wave] = sum;
    __syncthreads();
    uint64_t total = 0;
    for (int w = 0; w < kWaves; ++w)
        total += shared.scan[0][w];
    if (job.tokens) {
        const double threshold = static_cast<double>(job.random[r]) * static_cast<double>(total);
        uint64_t seen = 0, before = 0;
        int at = 0;
        for (int w = 0; w < kWaves; ++w) {
            const uint64_t next = seen + shared.scan[0][w];
            if (shared.scan[0][w] > 0) {
                at = w, before = seen;  // (stays at the last one with a weight where none passes)
                if (static_cast<double>(next) > threshold)
                    break;
            }
            seen = next;
        }
        const int from = min(at * part, V), to = min(from + part, V);
        const int each = (to - from + kThreads - 1) / kThreads, begin = min(from + tid * each, to), end = min(begin + each, to);
        uint64_t mine = 0;
        for (int i = begin; i < end; ++i) {
            double w;
            mine += me.kept(me.clean(load_f32(me.row + i)), i, w) ? me.whole(w) : 0;
        }
        uint64_t all;
        uint64_t run = before + me.block_scan(mine, all, 1);
        int found = V, last = -1;
        for (int i = begin; i < end && found == V; ++i) {
            double w;
            const uint64_t x = me.kept(me.clean(load_f32(me.row + i)), i, w) ? me.whole(w) : 0;
            run += x;
            if (x > 0) {
                last = i;
                found = static_cast<double>(run) > threshold ? i : V;
            }
        }
        found = wave_reduce(found, [](int a, int b) { return a < b ? a : b; });
        last = wave_reduce(last, [](int a, int b) { return a > b ? a : b; });
        __syncthreads();
        if (lane == 0)
            shared.counts[wave] = found, shared.counts[kWaves + wave] = last;
        __syncthreads();
        if (tid == 0) {
            for (int w = 0; w < kWaves; ++w) {
                found = min(found, static_cast<int>(shared.counts[w]));
                last = max(last, static_cast<int>(shared.counts[kWaves + w]));
            }
            job.tokens[r] = found < V ? found : last;
        }
    }
    if (probs) {
        const double inv = me.unit / static_cast<double>(total);
        for (int i = tid; i < V; i += kThreads) {
            double w;
            probs[i] = me.kept(me.clean(load_f32(me.row + i)), i, w) ? static_cast<float>(w * inv) : 0.f;
        }
    }
}

}  // namespace

hipError_t launch_sample_tokens(const SampleJob &job, hipStream_t stream, const char **why) {
    const dim3 grid(static_cast<unsigned>(job.R)), block(kThreads);
    switch (job.dtype) {
        case kF32: hipLaunchKernelGGL(sample_kernel<float>, grid, block, 0, stream, job); break;
        case kF16: hipLaunchKernelGGL(sample_kernel<_Float16>, grid, block, 0, stream, job); break;
        case kBF16: hipLaunchKernelGGL(sample_kernel<bf16_t>, grid, block, 0, stream, job); break;
        default: *why = "sample_tokens: unsupported dtype"; return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace ramnet
