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
// One block a row, which it reads from memory once and from the caches after that. Where few tokens are kept they
// are gathered in LDS together with some more, by a limit that each wave's greatest logits give, and compared
// with each other. Otherwise the end of the prefix is found by counts and sums of the weights in 2048 bins, even
// in the logit, and in the bin where it lies as before; then a pass adds up what is kept by stretches of the index.
#include "ramnet_kernels.hpp"
#include "vector16.hpp"

namespace ramnet {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / kWave, kBins = 2048, kList = kThreads;
// The most tokens that top_k keeps on the way by lists: a limit that 16 lanes of each wave reach lets in some 400
// of a language model's.
constexpr int kListCount = 256;

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

// The block's LDS, by one name: through a pointer it would be read as memory of any kind.
__device__ __forceinline__ Shared &lds() {
    __shared__ Shared shared;
    return shared;
}

struct Least {
    template<typename T> __device__ T operator()(T a, T b) const { return a < b ? a : b; }
};
struct Most {
    template<typename T> __device__ T operator()(T a, T b) const { return a > b ? a : b; }
};
struct Sum {
    template<typename T> __device__ T operator()(T a, T b) const { return a + b; }
};

// 2^x for x <= 0, to 1e-14: the series of e^(f ln 2) for the fraction f of x, in [-1/2, 1/2], to its 11th power.
__device__ __forceinline__ double power_of_2(double x) {
    const double whole = __builtin_rint(x), f = (x - whole) * 0.693147180559945309417;
    double sum = 1.0 / 39916800.0;
    constexpr double kTerms[] = {1.0 / 3628800.0, 1.0 / 362880.0, 1.0 / 40320.0, 1.0 / 5040.0, 1.0 / 720.0, 1.0 / 120.0,
                                 1.0 / 24.0,      1.0 / 6.0,      0.5,           1.0,          1.0};
#pragma unroll
    for (double term : kTerms)
        sum = fma(sum, f, term);
    return __builtin_amdgcn_ldexp(sum, static_cast<int>(whole));
}

template<typename Scalar>
struct Sampler {
    const Scalar *row;
    int V, tid, lane, wave;
    float top, low;         // the greatest logit, the smallest finite one
    float scale;            // bins per unit of the logit
    double rate, unit;      // log2(e) / temperature, 2^F
    double least;           // min_p
    uint64_t border;        // order of the last token kept

    __device__ __forceinline__ float clean(float l) const { return l != l ? -INFINITY : l + 0.f; }

    // f(logit, index) for all tokens, 16 bytes a thread, all threads of the block side by side.
    template<int kDeep = 2, typename F>
    __device__ __forceinline__ void sweep(F f) const {
        constexpr int N = 16 / sizeof(Scalar);
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

    // (a difference of -inf, or of nothing times 0, is held to where the weight is 0)
    __device__ __forceinline__ double weight(float l) const {
        const double x = (static_cast<double>(l) - static_cast<double>(top)) * rate;
        return l == top ? 1.0 : power_of_2(x > -2000.0 ? x : -2000.0);
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
        return w >= least && l > -INFINITY;  // (order_of(-inf) is greater than that of no token)
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
            lds().scan[which][wave] = run;
        __syncthreads();
        uint64_t before = 0;
        total = 0;
        for (int w = 0; w < kWaves; ++w) {
            before += w < wave ? lds().scan[which][w] : 0;
            total += lds().scan[which][w];
        }
        return before + run - x;
    }

    template<typename T, typename Op>
    __device__ __forceinline__ T block_reduce(T x, Op op) {
        auto put = [&](T v) {
            if constexpr (sizeof(T) == 8)
                lds().scan[0][wave] = __builtin_bit_cast(uint64_t, v);
            else
                lds().scan[0][wave] = __builtin_bit_cast(uint32_t, v);
        };
        auto get = [&](int w) {
            if constexpr (sizeof(T) == 8)
                return __builtin_bit_cast(T, lds().scan[0][w]);
            else
                return __builtin_bit_cast(T, static_cast<uint32_t>(lds().scan[0][w]));
        };
        x = wave_reduce(x, op);
        __syncthreads();
        if (lane == 0)
            put(x);
        __syncthreads();
        x = get(0);
        for (int w = 1; w < kWaves; ++w)
            x = op(x, get(w));
        return x;
    }

    // A limit that at least `count` logits reach, from the greatest one of each lane: the waves whose lanes have
    // logits all give their share of it.
    __device__ __forceinline__ float limit_of(float mine, int count) {
        const int waves = min(V / static_cast<int>(16 / sizeof(Scalar)) / kWave, kWaves), each = (count + waves - 1) / max(waves, 1);
        if (waves == 0 || each > kWave)
            return -INFINITY;
        int ahead = 0;
#pragma unroll
        for (int i = 0; i < kWave; ++i) {
            const float other = readlane_f(mine, i);
            ahead += other > mine || (other == mine && i < lane) ? 1 : 0;
        }
        const int at = __ffsll(static_cast<unsigned long long>(__ballot(ahead == each - 1))) - 1;
        return block_reduce(wave < waves ? readlane_f(mine, at) : INFINITY, Least{});
    }

    // The tokens that reach `limit`, and their weights, in the list, in any order; more than kList in `found` if
    // they are too many. `sum`: the weights of all tokens, where they are wanted.
    __device__ __forceinline__ void gather(float limit, bool wanted, int &found, uint64_t &sum) {
        __syncthreads();
        if (tid == 0)
            lds().listed = 0;
        __syncthreads();
        uint64_t total = 0;
        sweep([&](float l, int i) {
            if (wanted)
                total += whole(weight(l));
            if (l >= limit) {
                const int at = atomicAdd(&lds().listed, 1);
                if (at < kList)
                    lds().list[at] = order_of(l, i);
            }
        });
        sum = wanted ? block_reduce(total, Sum{}) : 0;
        __syncthreads();
        found = lds().listed;
        if (tid < min(found, kList))
            lds().weights[tid] = whole(weight(logit_of(lds().list[tid])));
        __syncthreads();
    }

    // The rest of the way where the list has all tokens that can be kept. `all`: the sum that top_p is a share of,
    // where it is not that of the first k. False if the list ends before that share does.
    __device__ __forceinline__ bool finish(int members, uint64_t k, bool by_sum, double p, uint64_t all, double u, int64_t *token, float *probs) {
        const bool mine = tid < members;
        const uint64_t order = mine ? lds().list[tid] : 0;
        uint64_t weights = mine ? lds().weights[tid] : 0, before = 0;
        int rank = 0;
        if (mine) {
            for (int j = 0; j < members; ++j) {
                const bool ahead = lds().list[j] > order;
                rank += ahead, before += ahead ? lds().weights[j] : 0;
            }
        }
        if (by_sum) {
            if (k < static_cast<uint64_t>(V))
                all = block_reduce(static_cast<uint64_t>(rank) < k ? weights : 0, Sum{});
            else if (static_cast<double>(block_reduce(weights, Sum{})) < p * static_cast<double>(all) && members < V)
                return false;
        }
        const double target = by_sum ? p * static_cast<double>(all) : INFINITY;
        const float l = logit_of(order);
        const double exact = mine ? weight(l) : 0.0;
        const bool stays = mine && l > -INFINITY &&
                           (rank == 0 || (static_cast<uint64_t>(rank) < k && static_cast<double>(before) < target && exact >= least));
        weights = stays ? weights : 0;
        const uint64_t total = block_reduce(weights, Sum{});  // (nobody reads the list's weights any more)
        const double threshold = u * static_cast<double>(total);
        const int index = static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(order));
        if (probs && stays)
            probs[index] = static_cast<float>(exact * unit / static_cast<double>(total));
        if (token) {
            if (mine)
                lds().weights[tid] = weights;
            __syncthreads();
            int first = V, last = -1;
            if (weights > 0) {
                uint64_t run = 0;
                for (int j = 0; j < members; ++j)
                    run += static_cast<uint32_t>(lds().list[j]) >= static_cast<uint32_t>(order) ? lds().weights[j] : 0;
                first = static_cast<double>(run) > threshold ? index : V, last = index;
            }
            first = block_reduce(first, Least{}), last = block_reduce(last, Most{});
            if (tid == 0)
                *token = first < V ? first : last;
        }
        return true;
    }

    __device__ __forceinline__ void clear_bins() {
        __syncthreads();
        for (int i = tid; i < kBins; i += kThreads)
            lds().counts[i] = 0, lds().sums[i] = 0;
        __syncthreads();
    }

    // The first bin where tokens, or their weights, reach what is asked for: k tokens (target 0), or a sum of
    // `target` beyond `base`. False (in all threads) if none does.
    __device__ __forceinline__ bool find_bin(uint64_t k, double target, uint64_t base, int first_count) {
        static_assert(kBins == 2 * kThreads, "two bins a thread");
        if (tid == 0)
            lds().bin = -1;
        const uint64_t c0 = lds().counts[2 * tid], c1 = lds().counts[2 * tid + 1], w0 = lds().sums[2 * tid], w1 = lds().sums[2 * tid + 1];
        uint64_t all_c, all_w;
        uint64_t c = block_scan(c0 + c1, all_c, 0) + static_cast<uint64_t>(first_count), w = block_scan(w0 + w1, all_w, 1) + base;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint64_t ci = i ? c1 : c0, wi = i ? w1 : w0;
            const bool here = ci > 0 && (target > 0.0 ? static_cast<double>(w) < target && static_cast<double>(w + wi) >= target
                                                      : c < k && c + ci >= k);
            if (here)
                lds().bin = 2 * tid + i, lds().before = w, lds().count_before = static_cast<int>(c);
            c += ci, w += wi;
        }
        __syncthreads();
        return lds().bin >= 0;
    }

    // The order of the k-th token, or of the last one with less than `target` before it; `through`: the weights
    // up to it. The bins hold what find_bin needs.
    __device__ __forceinline__ bool find_border(uint64_t k, double target, uint64_t &order, uint64_t &through) {
        if (!find_bin(k, target, 0, 0))
            return false;
        const int level = lds().bin;
        uint64_t base = lds().before, lo = 0, hi = ~0ull;
        int count_before = lds().count_before, members = static_cast<int>(lds().counts[level]);
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
                least_o = wave_reduce(least_o, Least{}), most_o = wave_reduce(most_o, Most{});
                __syncthreads();
                if (lane == 0)
                    lds().scan[0][wave] = least_o, lds().scan[1][wave] = most_o;
                __syncthreads();
                lo = ~0ull, hi = 0;
                for (int w = 0; w < kWaves; ++w)
                    lo = min(lo, lds().scan[0][w]), hi = max(hi, lds().scan[1][w]);
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
                    atomicAdd(&lds().counts[b], 1u);
                    atomicAdd(reinterpret_cast<unsigned long long *>(&lds().sums[b]), whole(weight(l)));
                }
            });
            __syncthreads();
            if (!find_bin(k, target, base, count_before))
                return false;
            base = lds().before, count_before = lds().count_before;
            const int at = lds().bin;
            members = static_cast<int>(lds().counts[at]);
            const uint64_t most = hi - (static_cast<uint64_t>(at) << shift);
            const uint64_t width = (1ull << shift) - 1;
            lo = most - lo > width ? most - width : lo;
            hi = most;
        }
        __syncthreads();
        if (tid == 0)
            lds().listed = 0;
        __syncthreads();
        sweep([&](float l, int i) {
            const uint64_t o = order_of(l, i);
            if (member(l, o)) {
                const int at = atomicAdd(&lds().listed, 1);
                lds().list[at] = o, lds().weights[at] = whole(weight(l));
            }
        });
        __syncthreads();
        if (tid < members) {
            const uint64_t o = lds().list[tid], w = lds().weights[tid];
            uint64_t before = base;
            int rank = 0;
            for (int j = 0; j < members; ++j) {
                const bool ahead = lds().list[j] > o;
                rank += ahead, before += ahead ? lds().weights[j] : 0;
            }
            const bool last = target > 0.0 ? static_cast<double>(before) < target &&
                                                 (static_cast<double>(before + w) >= target || rank == members - 1)
                                           : static_cast<uint64_t>(count_before + rank + 1) == k;
            if (last)
                lds().order = o, lds().through = before + w;
        }
        __syncthreads();
        order = lds().order, through = lds().through;
        return true;
    }
};

__device__ __forceinline__ double setting(const float *of_rows, double of_all, int64_t row) {
    return of_rows ? static_cast<double>(of_rows[row]) : of_all;
}

template<typename Scalar>
__global__ __launch_bounds__(kThreads) void sample_kernel(const SampleJob job) {
    const int64_t r = blockIdx.x;
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave, wave = tid / kWave, V = job.V;
    Sampler<Scalar> me{static_cast<const Scalar *>(job.logits) + r * job.row_at, V, tid, lane, wave};
    float *probs = job.probs ? job.probs + r * V : nullptr;

    me.top = -INFINITY, me.low = INFINITY;
    me.template sweep<4>([&](float l, int) {
        me.top = l > me.top ? l : me.top;
        me.low = l > -INFINITY && l < me.low ? l : me.low;
    });
    const float mine = me.top;
    me.low = wave_reduce(me.low, Least{});
    const float top = wave_reduce(mine, Most{});
    if (lane == 0)
        lds().tops[wave] = top, lds().lows[wave] = me.low;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) {
        me.top = w ? fmaxf(me.top, lds().tops[w]) : lds().tops[0];
        me.low = fminf(me.low, lds().lows[w]);
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
    me.rate = 1.4426950408889634074 / temperature;
    if (!(temperature > 0.0))  // the greatest alone
        k = 1, me.rate = 1.0;
    const double least = setting(job.min_p, job.min_p_of_all, r);
    me.least = least > 0.0 ? (least < 1.0 ? least : 1.0) : 0.0;
    me.unit = job.unit;
    const float range = me.top - me.low;
    me.scale = range > 0.f && range < INFINITY ? static_cast<float>(kBins - 1) / range : 0.f;
    me.border = 0;
    const bool by_count = k > 0 && k < V, by_sum = p < 1.0;
    const double u = job.tokens ? static_cast<double>(job.random[r]) : 0.0;
    if (by_count ? k <= kListCount : by_sum || me.least > 0.0) {
        float limit;
        if (by_count || by_sum) {
            // (for a share, some more than a language model's usually has)
            limit = me.limit_of(mine, by_count ? static_cast<int>(k) : 256);
        } else {
            // below the logit of weight min_p by more than the roundings on the way
            const double cut = static_cast<double>(me.top) + log2(me.least) / me.rate;
            limit = static_cast<float>(cut - (fabs(cut) + fabs(static_cast<double>(me.top))) * 1e-6 - 1e-37);
            limit = limit < me.top ? limit : -INFINITY;
        }
        int members;
        uint64_t all;
        me.gather(limit, !by_count && by_sum, members, all);
        if (members <= kList) {
            if (probs) {
                constexpr int N = 4;
                for (int i = tid * N; i < V / N * N; i += kThreads * N)
                    store_vec<float, N>(probs + i, {});
                if (V / N * N + tid < V)
                    probs[V / N * N + tid] = 0.f;
                __syncthreads();
            }
            if (me.finish(members, by_count ? static_cast<uint64_t>(k) : static_cast<uint64_t>(V), by_sum, p > 0.0 ? p : 0.0, all, u,
                          job.tokens ? job.tokens + r : nullptr, probs))
                return;
        }
    }
    if (by_count || by_sum) {
        me.clear_bins();
        uint64_t total = 0;
        me.sweep([&](float l, int) {
            const int b = me.bin(l);
            atomicAdd(&lds().counts[b], 1u);
            if (by_sum) {
                const uint64_t w = me.whole(me.weight(l));
                atomicAdd(reinterpret_cast<unsigned long long *>(&lds().sums[b]), w);
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
                        atomicAdd(&lds().counts[b], 1u);
                        atomicAdd(reinterpret_cast<unsigned long long *>(&lds().sums[b]), me.whole(me.weight(l)));
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
    // The kept weights by stretches of the vocabulary, a wave each, in order of the index: whole pieces of 16 bytes,
    // and for the last wave the row's last few elements
    constexpr int N = 16 / sizeof(Scalar), kDeep = 2;
    const int full = V / N * N, part = (V + kWaves * N - 1) / (kWaves * N) * N;
    const int lo = min(wave * part, full), hi = min(lo + part, full);
    uint64_t sum = 0;
    for (int at = lo + lane * N; at < hi; at += kDeep * kWave * N) {
        Vec<Scalar, N> x[kDeep];
#pragma unroll
        for (int i = 0; i < kDeep; ++i)
            x[i] = at + i * kWave * N < hi ? load_vec<Scalar, N>(me.row + at + i * kWave * N) : Vec<Scalar, N>{};
#pragma unroll
        for (int i = 0; i < kDeep; ++i) {
            if (at + i * kWave * N < hi) {
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    double w;
                    sum += me.kept(me.clean(x[i][e]), at + i * kWave * N + e, w) ? me.whole(w) : 0;
                }
            }
        }
    }
    if (wave == kWaves - 1 && full + lane < V) {
        double w;
        sum += me.kept(me.clean(load_f32(me.row + full + lane)), full + lane, w) ? me.whole(w) : 0;
    }
    sum = wave_reduce(sum, Sum{});
    __syncthreads();
    if (lane == 0)
        lds().scan[0][wave] = sum;
    __syncthreads();
    uint64_t total = 0;
    for (int w = 0; w < kWaves; ++w)
        total += lds().scan[0][w];
    if (job.tokens) {
        const double threshold = u * static_cast<double>(total);
        uint64_t seen = 0, before = 0;
        int at = 0;
        for (int w = 0; w < kWaves; ++w) {
            const uint64_t next = seen + lds().scan[0][w];
            if (lds().scan[0][w] > 0) {
                at = w, before = seen;  // (stays at the last one with a weight where none passes)
                if (static_cast<double>(next) > threshold)
                    break;
            }
            seen = next;
        }
        const int from = min(at * part, full), to = at == kWaves - 1 ? V : min(from + part, full);
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
        found = me.block_reduce(found, Least{}), last = me.block_reduce(last, Most{});
        if (tid == 0)
            job.tokens[r] = found < V ? found : last;
    }
    if (probs) {
        const double inv = me.unit / static_cast<double>(total);
        auto value = [&](float l, int i) {
            double w;
            return me.kept(me.clean(l), i, w) ? static_cast<float>(w * inv) : 0.f;
        };
        for (int at = tid * N; at < full; at += kThreads * N) {
            const Vec<Scalar, N> x = load_vec<Scalar, N>(me.row + at);
#pragma unroll
            for (int e = 0; e < N; e += 4) {
                const float out[4] = {value(x[e], at + e), value(x[e + 1], at + e + 1), value(x[e + 2], at + e + 2),
                                      value(x[e + 3], at + e + 3)};
                store_vec<float, 4>(probs + at + e, round_vec<float, 4>(out));
            }
        }
        if (full + tid < V)
            probs[full + tid] = value(load_f32(me.row + full + tid), full + tid);
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
