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
// are gathered in LDS and compared with each other: with some more, by a limit that each wave's greatest logits
// give, or with the bin where the prefix ends, which counts (by top_k) or sums of the weights (by top_p) in 2048
// bins tell. Otherwise the end is found within that bin, and a pass adds up what is kept by stretches of the index.
//
// 192 rows of 128257 bf16, a block on three of four compute units: greedy 27 us, top_k of 50 30 (49 MB read, 2 TB/s), no
// filter 46, top_p of 0.9 at temperature 1.5 110, of which two passes of weights take 25 each, bound by their
// instructions (some 35 a token, 12 of 64 bits), and the search 22. One row of 32000, fp32: 12 to 17 us, the latency of
// its passes and barriers. Masked rows take no longer: with 20 tokens left and a top_k of 50 28 us and 12.6.
#include "ramnet_kernels.hpp"
#include "vector16.hpp"

namespace ramnet {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / kWave, kBins = 2 * kThreads, kList = kThreads;
// The most tokens of top_k that are gathered by a limit: one that 16 lanes of each wave reach lets in some 400
// of a language model's.
constexpr int kListCount = 256;
// Bins of a sum for each halving of the weight: what lies past 2^-32 is in the last bin.
constexpr float kBinsAHalving = 64.f;
// The least logit of a token that can be drawn: one of -inf is in no list and no count.
constexpr float kLeastLogit = -__FLT_MAX__;

// A token's place in the order as one number, greater for earlier ones; its upper half goes by the logit alone.
__device__ __forceinline__ uint32_t key_of(float l) {
    const uint32_t bits = __float_as_uint(l);
    return bits ^ (static_cast<uint32_t>(static_cast<int32_t>(bits) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float logit_of_key(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
__device__ __forceinline__ uint64_t order_of(float l, int index) {
    return static_cast<uint64_t>(key_of(l)) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(index));
}
__device__ __forceinline__ float logit_of(uint64_t order) { return logit_of_key(static_cast<uint32_t>(order >> 32)); }
__device__ __forceinline__ int index_of(uint64_t order) {
    return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(order));
}

struct Shared {
    uint32_t counts[kBins];
    uint64_t sums[kBins];
    uint64_t list[kList];
    uint64_t scan[2][kWaves];
    double powers[32];       // 2^(i / 32)
    uint64_t before, order;  // results that one thread finds
    int count_before, count_through, bin, listed;
};

// The block's LDS, by one name: through a pointer it would be read as memory of any kind.
__device__ __forceinline__ Shared &lds() {
    __shared__ Shared shared;
    return shared;
}
__device__ __forceinline__ void add(uint64_t &to, uint64_t x) {
    atomicAdd(reinterpret_cast<unsigned long long *>(&to), static_cast<unsigned long long>(x));
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

// The value of the lane whose number differs in one bit.
template<int XOR>
__device__ __forceinline__ uint32_t lane_xor(uint32_t x) {
    if constexpr (XOR == 1) {
        return __builtin_amdgcn_mov_dpp(x, 0xB1, 0xF, 0xF, true);  // quad_perm 1 0 3 2
    } else if constexpr (XOR == 2) {
        return __builtin_amdgcn_mov_dpp(x, 0x4E, 0xF, 0xF, true);  // quad_perm 2 3 0 1
    } else if constexpr (XOR == 4) {
        const uint32_t up = __builtin_amdgcn_update_dpp(0u, x, 0x104, 0xF, 0x5, false);  // row_shl:4, lanes without bit 2
        return __builtin_amdgcn_update_dpp(up, x, 0x114, 0xF, 0xA, false);               // row_shr:4, lanes with it
    } else if constexpr (XOR == 8) {
        return __builtin_amdgcn_mov_dpp(x, 0x128, 0xF, 0xF, true);  // row_ror:8
    } else {
        const auto r = XOR == 16 ? __builtin_amdgcn_permlane16_swap(x, x, false, false)
                                 : __builtin_amdgcn_permlane32_swap(x, x, false, false);
        return __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)) & XOR ? r[0] : r[1];
    }
}

template<int XOR, typename T>
__device__ __forceinline__ T lane_xor_of(T x) {
    if constexpr (sizeof(T) == 8) {
        const uint64_t bits = __builtin_bit_cast(uint64_t, x);
        return __builtin_bit_cast(T, static_cast<uint64_t>(lane_xor<XOR>(static_cast<uint32_t>(bits >> 32))) << 32 |
                                         lane_xor<XOR>(static_cast<uint32_t>(bits)));
    } else {
        return __builtin_bit_cast(T, lane_xor<XOR>(__builtin_bit_cast(uint32_t, x)));
    }
}

template<typename T, typename Op>
__device__ __forceinline__ T wave_reduce(T x, Op op) {
    x = op(x, lane_xor_of<1>(x)), x = op(x, lane_xor_of<2>(x)), x = op(x, lane_xor_of<4>(x));
    x = op(x, lane_xor_of<8>(x)), x = op(x, lane_xor_of<16>(x));
    return op(x, lane_xor_of<32>(x));
}

// x and the values of the lanes before it, added up: within rows of 16 by shifts, then row by row.
template<int CONTROL, int ROWS>
__device__ __forceinline__ uint64_t shifted(uint64_t x) {
    const uint32_t low = __builtin_amdgcn_update_dpp(0u, static_cast<uint32_t>(x), CONTROL, ROWS, 0xF, false);
    const uint32_t high = __builtin_amdgcn_update_dpp(0u, static_cast<uint32_t>(x >> 32), CONTROL, ROWS, 0xF, false);
    return static_cast<uint64_t>(high) << 32 | low;
}
__device__ __forceinline__ uint64_t wave_scan(uint64_t x) {
    x += shifted<0x111, 0xF>(x), x += shifted<0x112, 0xF>(x);  // row_shr:1, 2, 4, 8
    x += shifted<0x114, 0xF>(x), x += shifted<0x118, 0xF>(x);
    x += shifted<0x142, 0xA>(x);                               // row_bcast:15, to rows 1 and 3
    return x + shifted<0x143, 0xC>(x);                         // row_bcast:31, to rows 2 and 3
}

// 2^x for x in [-1000, 0], to 2e-15: of x in parts of 1/32, which adding 3 2^46 leaves in the lowest bits of the
// sum, the last five bits by a table (whose 32 values lie in as many pairs of LDS banks), those above into the
// exponent, and what is left, up to 1/64, by the series of e^(f ln 2) to its 5th power.
constexpr int kParts = 32;
__device__ __forceinline__ double power_of_2(double x) {
    constexpr double kRound = 3.0 * 70368744177664.0, kLn2 = 0.693147180559945309417;
    const double shifted = x + kRound, f = x - (shifted - kRound);
    double terms[] = {kLn2 * kLn2 * kLn2 * kLn2 * kLn2 / 120.0, kLn2 * kLn2 * kLn2 * kLn2 / 24.0, kLn2 * kLn2 * kLn2 / 6.0,
                      kLn2 * kLn2 / 2.0, kLn2};
    const int part = static_cast<int>(__builtin_bit_cast(uint64_t, shifted));
    double sum = terms[0];
#pragma unroll
    for (int i = 1; i < 5; ++i) {
        asm("" : "+s"(terms[i]));  // (in scalar registers: from vector registers each would be copied first)
        sum = fma(sum, f, terms[i]);
    }
    const double of_part = lds().powers[part & (kParts - 1)];
    sum = fma(sum * f, of_part, of_part);
    return __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, sum) +
                                          (static_cast<uint64_t>(static_cast<uint32_t>(part >> 5)) << 52));
}

template<typename Scalar>
struct Sampler {
    const Scalar *row;
    int V, tid, lane, wave;
    float top;              // the greatest logit
    float scale;            // bins per unit of the logit
    double rate, unit;      // log2(e) / temperature, 2^F
    double least;           // min_p
    float last_logit;       // the last token kept: of its logit those up to its index, of greater ones all
    int last_index;

    __device__ __forceinline__ float clean(float l) const { return l != l ? -INFINITY : l + 0.f; }

    // f(logit, index) for all tokens, 16 bytes a thread, all threads of the block side by side. (kRaw: of logits as
    // they are stored, for an f that passes over a NaN by itself.)
    template<bool kRaw = false, typename F>
    __device__ __forceinline__ void sweep(F f) const {
        constexpr int N = 16 / sizeof(Scalar), kDeep = 4;
        auto value = [&](float l) { return kRaw ? l : clean(l); };
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
                        f(value(x[i][e]), from + e);
                }
            }
        }
        if (full + tid < V)
            f(value(load_f32(row + full + tid)), full + tid);
    }

    // The same with one piece ahead, for an f that takes longer than the read.
    template<typename F>
    __device__ __forceinline__ void sweep_ahead(F f) const {
        constexpr int N = 16 / sizeof(Scalar), kStep = kThreads * N;
        const int full = V / N * N;
        Vec<Scalar, N> next{};
        if (tid * N < full)
            next = load_vec<Scalar, N>(row + tid * N);
        for (int at = tid * N; at < full; at += kStep) {
            const Vec<Scalar, N> x = next;
            if (at + kStep < full)
                next = load_vec<Scalar, N>(row + at + kStep);
#pragma unroll
            for (int e = 0; e < N; ++e)
                f(x[e], at + e);
        }
        if (full + tid < V)
            f(load_f32(row + full + tid), full + tid);
    }

    // (what is no number, as a difference of -inf or nothing times 0, is held to where no part of the sum is left)
    __device__ __forceinline__ double weight(float l) const {
        const double x = fma(static_cast<double>(l), rate, -static_cast<double>(top) * rate);
        return power_of_2(l == top ? 0.0 : __builtin_fmax(x, -1000.0));
    }
    // A weight in whole parts of 1 / unit, below 2^52: they are the last bits of its sum with 2^52.
    __device__ __forceinline__ uint64_t whole(double w) const {
        return __builtin_bit_cast(uint64_t, fma(w, unit, 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;
    }
    __device__ __forceinline__ int bin(float l) const {
        const float at = l == top ? 0.f : (top - l) * scale;  // (descending with l, whatever it rounds to; a NaN last)
        return static_cast<int>(__builtin_fminf(at, static_cast<float>(kBins - 1)));
    }
    // Whether a token is in the prefix kept. A NaN is not, nor is -inf, also where the prefix has no end yet.
    __device__ __forceinline__ bool within(float l, int index) const {
        return l > last_logit || (l == last_logit && index <= last_index);
    }
    __device__ __forceinline__ void end_with(uint64_t order) { last_logit = logit_of(order), last_index = index_of(order); }
    // Whether a token is drawn from. (A branch around the weight: without it rows that keep few took up to 15 us
    // more, those that keep most no less.)
    __device__ __forceinline__ bool kept(float l, int index, double &w) const {
        if (!within(l, index))
            return false;
        w = weight(l);
        return w >= least;
    }

    // What op makes of the 16 waves' values, from a value a lane that goes by the lane's place in its row of 16.
    template<typename T, typename Op>
    __device__ __forceinline__ static T row_reduce(T x, Op op) {
        static_assert(kWaves == 16, "a row of lanes");
        x = op(x, lane_xor_of<1>(x)), x = op(x, lane_xor_of<2>(x)), x = op(x, lane_xor_of<4>(x));
        return op(x, lane_xor_of<8>(x));
    }

    // The sum of x over the threads before.
    __device__ __forceinline__ uint64_t block_scan(uint64_t x, int which) {
        const uint64_t run = wave_scan(x);
        __syncthreads();
        if (lane == kWave - 1)
            lds().scan[which][wave] = run;
        __syncthreads();
        const uint64_t of_wave = lds().scan[which][lane % kWaves];
        return row_reduce(lane % kWaves < wave ? of_wave : 0, Sum{}) + run - x;
    }

    template<typename T>
    __device__ __forceinline__ static uint64_t as_word(T x) {
        if constexpr (sizeof(T) == 8)
            return __builtin_bit_cast(uint64_t, x);
        else
            return __builtin_bit_cast(uint32_t, x);
    }
    template<typename T>
    __device__ __forceinline__ static T of_word(uint64_t x) {
        if constexpr (sizeof(T) == 8)
            return __builtin_bit_cast(T, x);
        else
            return __builtin_bit_cast(T, static_cast<uint32_t>(x));
    }

    // Over the block; of two values at once.
    template<typename T, typename Op>
    __device__ __forceinline__ T block_reduce(T x, Op op) {
        x = wave_reduce(x, op);
        __syncthreads();
        if (lane == 0)
            lds().scan[0][wave] = as_word(x);
        __syncthreads();
        return row_reduce(of_word<T>(lds().scan[0][lane % kWaves]), op);
    }
    template<typename T, typename OpT, typename U, typename OpU>
    __device__ __forceinline__ void block_reduce(T &x, OpT op_x, U &y, OpU op_y) {
        x = wave_reduce(x, op_x), y = wave_reduce(y, op_y);
        __syncthreads();
        if (lane == 0)
            lds().scan[0][wave] = as_word(x), lds().scan[1][wave] = as_word(y);
        __syncthreads();
        x = row_reduce(of_word<T>(lds().scan[0][lane % kWaves]), op_x);
        y = row_reduce(of_word<U>(lds().scan[1][lane % kWaves]), op_y);
    }

    // A limit that at least `count` logits reach, from the greatest one of each lane: the waves whose lanes have
    // logits all give their share of it, each to the 16 upper bits. Where that would be -inf (many tokens are masked)
    // the least finite number, which all tokens reach that can be drawn.
    __device__ __forceinline__ float limit_of(float mine, int count) {
        const int waves = min(V / static_cast<int>(16 / sizeof(Scalar)) / kWave, kWaves), each = (count + waves - 1) / max(waves, 1);
        if (waves == 0 || each > kWave)
            return kLeastLogit;
        const uint32_t key = key_of(mine);
        uint32_t reached = 0;
#pragma unroll
        for (uint32_t bit = 1u << 31; bit >= 1u << 16; bit >>= 1)
            reached |= __popcll(__ballot(key >= (reached | bit))) >= each ? bit : 0;
        reached = block_reduce(wave < waves ? reached : ~0u, Least{});
        return reached > key_of(-INFINITY) ? logit_of_key(reached) : kLeastLogit;
    }

    // The tokens of which `wanted` is true in the list, in any order. How many they are: where
    // more than kList the list has some of them.
    template<bool kRaw = false, typename F>
    __device__ __forceinline__ int gather(F wanted) {
        __syncthreads();
        if (tid == 0)
            lds().listed = 0;
        __syncthreads();
        sweep<kRaw>([&](float l, int i) {
            if (wanted(l, i)) {
                const int at = atomicAdd(&lds().listed, 1);
                if (at < kList)
                    lds().list[at] = order_of(kRaw ? clean(l) : l, i);
            }
        });
        __syncthreads();
        return lds().listed;
    }

    // One step of a bitonic sort within a wave.
    template<int STRIDE>
    __device__ __forceinline__ uint64_t step(uint64_t x, int size) const {
        const uint32_t low = lane_xor<STRIDE>(static_cast<uint32_t>(x)), high = lane_xor<STRIDE>(static_cast<uint32_t>(x >> 32));
        const uint64_t other = static_cast<uint64_t>(high) << 32 | low;
        const bool greater = ((tid & STRIDE) == 0) == ((tid & size) == 0);
        return (other > x) == greater ? other : x;
    }
    template<int STRIDE>
    __device__ __forceinline__ uint64_t steps(uint64_t x, int size) const {
        x = step<STRIDE>(x, size);
        if constexpr (STRIDE > 1)
            return steps<STRIDE / 2>(x, size);
        return x;
    }

    // The numbers of the first `count` threads, one each, the greatest to the first thread, zeros behind them: a
    // bitonic sort, by lane swaps within a wave and through LDS across waves.
    __device__ __forceinline__ uint64_t sorted(uint64_t x, int count) const {
        x = steps<1>(x, 2), x = steps<2>(x, 4), x = steps<4>(x, 8);
        x = steps<8>(x, 16), x = steps<16>(x, 32), x = steps<32>(x, 64);
        for (int size = 2 * kWave; size < 2 * count; size *= 2) {
            for (int stride = size / 2; stride >= kWave; stride /= 2) {
                __syncthreads();
                lds().sums[tid] = x;
                __syncthreads();
                const uint64_t other = lds().sums[tid ^ stride];
                const bool greater = ((tid & stride) == 0) == ((tid & size) == 0);
                x = (other > x) == greater ? other : x;
            }
            x = steps<32>(x, size);
        }
        return x;
    }

    // The rest of the way where the list has all tokens that can be kept: of these the first k, and those with less
    // than the share p of `all` before them (0: of the first k).
    __device__ __forceinline__ void finish(int members, uint64_t k, bool by_sum, double p, uint64_t all, double u, int64_t *token,
                                           float *probs) {
        if (probs) {
            constexpr int N = 4;
            for (int i = tid * N; i < V / N * N; i += kThreads * N)
                store_vec<float, N>(probs + i, {});
            if (V / N * N + tid < V)
                probs[V / N * N + tid] = 0.f;
        }
        const uint64_t order = sorted(tid < members ? lds().list[tid] : 0, members);
        const bool mine = tid < members;
        const float l = logit_of(order);
        const double exact = mine ? weight(l) : 0.0;
        uint64_t part = mine ? whole(exact) : 0;
        const uint64_t before = block_scan(part, 0);
        if (by_sum && all == 0)
            all = block_reduce(static_cast<uint64_t>(tid) < k ? part : 0, Sum{});
        const double target = by_sum ? p * static_cast<double>(all) : INFINITY;
        const bool stays = mine && within(l, index_of(order)) &&
                           (tid == 0 || (static_cast<uint64_t>(tid) < k && static_cast<double>(before) < target && exact >= least));
        part = stays ? part : 0;
        int drawn = part > 0 ? tid + 1 : 0;  // (those with a weight are a prefix)
        uint64_t parts = part;
        block_reduce(parts, Sum{}, drawn, Most{});
        const double total = static_cast<double>(parts);
        if (probs && stays)  // (the zeros are behind the barriers of that sum)
            probs[index_of(order)] = static_cast<float>(exact * unit / total);
        if (token) {
            // by index, each with its place among the weights
            lds().list[tid] = part;
            const uint64_t at = sorted(part > 0 ? order << 32 | static_cast<uint32_t>(tid) : 0, drawn);
            __syncthreads();
            const uint64_t own = tid < drawn ? lds().list[static_cast<uint32_t>(at)] : 0;
            const uint64_t run = block_scan(own, 0);
            const double threshold = u * total;
            // (the first that passes or, where by rounding none does, the last)
            if (tid < drawn && !(static_cast<double>(run) > threshold) &&
                (static_cast<double>(run + own) > threshold || tid == drawn - 1))
                *token = index_of(at >> 32);
        }
    }

    __device__ __forceinline__ void clear_bins() {
        __syncthreads();
        for (int i = tid; i < kBins; i += kThreads)
            lds().counts[i] = 0, lds().sums[i] = 0;
        __syncthreads();
    }

    // The first bin where the tokens reach k of them or, where there is a target, the weights reach it; the counts
    // and sums of the bins before it come on top of `count` and `sum`.
    __device__ __forceinline__ bool find_bin(uint64_t k, double target, uint64_t sum, int count) {
        if (tid == 0)
            lds().bin = -1;
        const bool by_sum = target > 0.0;
        uint64_t of[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
            of[i] = by_sum ? lds().sums[2 * tid + i] : lds().counts[2 * tid + i];
        uint64_t before = block_scan(of[0] + of[1], 0) + (by_sum ? sum : static_cast<uint64_t>(count));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint64_t through = before + of[i];
            if (by_sum ? static_cast<double>(before) < target && static_cast<double>(through) >= target : before < k && through >= k) {
                lds().bin = 2 * tid + i, lds().before = before;
                lds().count_before = static_cast<int>(before), lds().count_through = static_cast<int>(through);
            }
            before = through;
        }
        __syncthreads();
        return lds().bin >= 0;
    }

    // The order of the k-th token, or of the last one with less than `target` before it, in the bin that find_bin
    // has found (of tokens that `within` holds, as all searches count them): as long as it holds more tokens than the
    // list, it is cut into 2048 parts again, now by the order. Where no token is met, an end that keeps all.
    // `through`: with a target the weights up to that one, it among them (0: not known).
    __device__ __forceinline__ uint64_t find_border(uint64_t k, double target, uint64_t &through) {
        through = 0;
        const int level = lds().bin;
        if (tid == 0)  // (behind barriers before a thread that meets its token writes)
            lds().order = order_of(-INFINITY, -1);
        const bool by_sum = target > 0.0;
        uint64_t base = by_sum ? lds().before : 0, lo = 0, hi = ~0ull;
        int count = by_sum ? 0 : lds().count_before;
        // (two comparisons tell most tokens from those of the bin, which lie between these by more than the roundings)
        const float slack = fabsf(top) * 1e-6f + static_cast<float>(level + 1) / scale * 1e-6f;
        const bool narrow = scale > 0.f && slack < INFINITY;
        const float high = narrow ? top - static_cast<float>(level) / scale + slack : INFINITY;
        const float low = narrow && level < kBins - 1 ? top - static_cast<float>(level + 1) / scale - slack : -INFINITY;
        int members = gather([&](float l, int i) { return l >= low && l <= high && bin(l) == level && within(l, i); });
        if (members > kList) {
            uint64_t least_o = ~0ull, most_o = 0;
            sweep([&](float l, int i) {
                const uint64_t o = order_of(l, i);
                if (bin(l) == level && within(l, i))
                    least_o = min(least_o, o), most_o = max(most_o, o);
            });
            block_reduce(least_o, Least{}, most_o, Most{});
            lo = least_o, hi = most_o;
        }
        while (members > kList) {
            int shift = 0;
            while (((hi - lo) >> shift) >= kBins)
                ++shift;
            clear_bins();
            sweep_ahead([&](float raw, int i) {
                const float l = clean(raw);
                const uint64_t o = order_of(l, i);
                if (o >= lo && o <= hi) {
                    const int b = static_cast<int>((hi - o) >> shift);
                    if (by_sum)
                        add(lds().sums[b], whole(weight(l)));
                    else
                        atomicAdd(&lds().counts[b], 1u);
                }
            });
            __syncthreads();
            if (!find_bin(k, target, base, count))
                return lo;  // (not met: the parts' sums are the bin's)
            base = by_sum ? lds().before : 0, count = by_sum ? 0 : lds().count_before;
            hi -= static_cast<uint64_t>(lds().bin) << shift;
            const uint64_t width = (1ull << shift) - 1;
            lo = hi - lo > width ? hi - width : lo;
            members = gather([&](float l, int i) {
                const uint64_t o = order_of(l, i);
                return o >= lo && o <= hi;
            });
        }
        const uint64_t own = sorted(tid < members ? lds().list[tid] : 0, members);
        const uint64_t part = tid < members ? whole(weight(logit_of(own))) : 0;
        const uint64_t before = base + block_scan(part, 0);
        if (tid < members) {
            const double from = static_cast<double>(before), to = static_cast<double>(before + part);
            if (by_sum ? from < target && (to >= target || tid == members - 1) : static_cast<uint64_t>(count + tid + 1) == k)
                lds().order = own, lds().before = before + part;
        }
        __syncthreads();
        const uint64_t order = lds().order;
        through = by_sum && index_of(order) >= 0 ? lds().before : 0;
        return order;
    }
};

__device__ __forceinline__ double setting(const float *of_rows, double of_all, int64_t row) {
    return of_rows ? static_cast<double>(of_rows[row]) : of_all;
}

template<typename Scalar>
__global__ __launch_bounds__(kThreads) void sample_kernel(const SampleJob job) {
    const int64_t r = blockIdx.x;
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave, V = job.V;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    Sampler<Scalar> me{static_cast<const Scalar *>(job.logits) + r * job.row_at, V, tid, lane, wave};
    float *probs = job.probs ? job.probs + r * V : nullptr;
    int64_t *token = job.tokens ? job.tokens + r : nullptr;

    if (tid < kParts)
        lds().powers[tid] = exp2(tid * (1.0 / kParts));
    float mine = -INFINITY, low = INFINITY;
    me.sweep([&](float l, int) {
        mine = l > mine ? l : mine;
        low = l > -INFINITY && l < low ? l : low;
    });
    me.top = me.block_reduce(mine, Most{});
    if (me.top == -INFINITY) {  // nothing to draw from
        if (tid == 0 && token)
            *token = 0;
        for (int i = tid; probs && i < V; i += kThreads)
            probs[i] = 0.f;
        return;
    }
    const double temperature = setting(job.temperature, job.temperature_of_all, r);
    const double p = setting(job.top_p, job.top_p_of_all, r), least = setting(job.min_p, job.min_p_of_all, r);
    int64_t k = job.top_k ? job.top_k[r] : job.top_k_of_all;
    me.rate = 1.4426950408889634074 / temperature;
    if (!(temperature > 0.0))
        me.rate = 1.0;
    if (!(temperature > 0.0) || p <= 0.0)  // the greatest alone
        k = 1;
    const bool by_count = k > 0 && k < V, by_sum = p < 1.0 && k != 1;
    const uint64_t first = by_count ? static_cast<uint64_t>(k) : static_cast<uint64_t>(V);
    me.least = least > 0.0 ? (least < 1.0 ? least : 1.0) : 0.0;
    me.unit = job.unit, me.last_logit = -INFINITY, me.last_index = -1;
    // (below 0 draws as 0 does; from 1 on, or no number, the last kept token)
    const float random = token ? job.random[r] : 0.f;
    const double u = random < 0.f ? 0.0 : static_cast<double>(random);
    // A list of those that top_k or min_p may keep
    const bool few = by_count && k <= kListCount;
    if (few || (me.least > 0.0 && !by_sum)) {
        float limit = me.top;
        if (few && k > 1) {
            limit = me.limit_of(mine, static_cast<int>(k));
        } else if (!few) {
            // below the logit of weight min_p by more than the roundings on the way
            const double cut = static_cast<double>(me.top) + log2(me.least) / me.rate;
            limit = static_cast<float>(cut - (fabs(cut) + fabs(static_cast<double>(me.top))) * 1e-6 - 1e-37);
            limit = limit < me.top && limit > kLeastLogit ? limit : kLeastLogit;
        }
        const int members = me.gather([&](float l, int) { return l >= limit; });
        if (members <= kList) {
            me.finish(members, first, by_sum, p, 0, u, token, probs);
            return;
        }
    }
    uint64_t kept_sum = 0;  // of the kept weights, where the search for the last one gives it
    if (by_count) {
        const float range = me.top - me.block_reduce(low, Least{});
        me.scale = range > 0.f && range < INFINITY ? static_cast<float>(kBins - 1) / range : 0.f;
        me.clear_bins();
        me.template sweep<true>([&](float l, int) {
            if (l > -INFINITY)
                atomicAdd(&lds().counts[me.bin(l)], 1u);
        });
        __syncthreads();
        // (not found: fewer tokens than top_k can be drawn, and it keeps them all)
        const bool found = me.find_bin(first, 0.0, 0, 0);
        const int level = found ? lds().bin : kBins - 1;
        if (!found || lds().count_through <= kList) {
            const int members = me.template gather<true>([&](float l, int) { return l > -INFINITY && me.bin(l) <= level; });
            if (members <= kList) {
                me.finish(members, first, by_sum, p, 0, u, token, probs);
                return;
            }
        }
        if (found)
            me.end_with(me.find_border(first, 0.0, kept_sum));
    }
    if (by_sum) {
        me.scale = static_cast<float>(me.rate) * kBinsAHalving;
        me.clear_bins();
        uint64_t all = 0, last = 0;
        auto count = [&](float l) {
            const uint64_t w = me.whole(me.weight(l));
            const int b = me.bin(l);
            all += w;
            if (b < kBins - 1)
                add(lds().sums[b], w);
            else
                last += w;
        };
        if (by_count)
            me.sweep_ahead([&](float l, int i) {
                if (me.within(l, i))
                    count(l);
            });
        else  // (a NaN has neither weight nor bin as it is)
            me.sweep_ahead([&](float l, int) { count(l); });
        me.block_reduce(all, Sum{}, last, Sum{});
        if (tid == 0)
            lds().sums[kBins - 1] = last;
        __syncthreads();
        const double target = p * static_cast<double>(all);
        if (me.find_bin(0, target, 0, 0)) {
            // min_p ends in bin `cut` or one beside it, by the roundings of a token's bin
            const int cut = me.least > 0.0 ? static_cast<int>(__builtin_fmin(-log2(me.least) * kBinsAHalving, kBins)) : kBins;
            const bool by_least = cut + 1 < lds().bin;  // before top_p does
            const int level = by_least ? cut + 1 : lds().bin;
            // No weight is above its bin's first: a sum takes so many tokens at least. Where these fit the list, so
            // may all of them.
            double tokens = 0.0;
            uint64_t over = 0;  // of those that min_p keeps for sure
            for (int i = tid; i <= level; i += kThreads) {
                tokens += static_cast<double>(lds().sums[i]) * exp2(i / static_cast<double>(kBinsAHalving));
                over += i < cut - 1 ? lds().sums[i] : 0;
            }
            me.block_reduce(tokens, Sum{}, over, Sum{});
            if (tokens < kList * me.unit) {
                const int members = me.gather([&](float l, int i) { return me.bin(l) <= level && me.within(l, i); });
                if (members <= kList) {
                    me.finish(members, static_cast<uint64_t>(V), true, p, all, u, token, probs);
                    return;
                }
            }
            if (!by_least)
                me.end_with(me.find_border(0, target, kept_sum));
            if (by_least || me.weight(me.last_logit) < me.least) {
                uint64_t more = 0;
                me.sweep([&](float l, int i) {
                    const int b = me.bin(l);
                    double w;
                    if (b >= cut - 1 && b <= cut + 1 && me.kept(l, i, w))
                        more += me.whole(w);
                });
                kept_sum = over + me.block_reduce(more, Sum{});
            }
        }
    }
    // The kept weights by stretches of the vocabulary, a wave each, in order of the index: whole pieces of 16 bytes,
    // and for the last wave the row's last few elements
    constexpr int N = 16 / sizeof(Scalar);
    const int full = V / N * N, part = (V + kWaves * N - 1) / (kWaves * N) * N;
    const int lo = min(wave * part, full), hi = min(lo + part, full);
    auto share = [&](float l, int i) -> uint64_t {
        double w;
        return me.kept(l, i, w) ? me.whole(w) : 0;
    };
    auto value = [&](float l, int i, double inv) {
        double w;
        return me.kept(l, i, w) ? static_cast<float>(w * inv) : 0.f;
    };
    auto put = [&](int at, const float (&out)[N]) {
#pragma unroll
        for (int e = 0; e < N; e += 4) {
            const float four[4] = {out[e], out[e + 1], out[e + 2], out[e + 3]};
            store_vec<float, 4>(probs + at + e, round_vec<float, 4>(four));
        }
    };
    uint64_t sum = wave == kWaves - 1 && full + lane < V ? share(load_f32(me.row + full + lane), full + lane) : 0;
    auto stretch = [&](auto of, auto then) {
        Vec<Scalar, N> next{};
        if (lo + lane * N < hi)
            next = load_vec<Scalar, N>(me.row + lo + lane * N);
        for (int at = lo + lane * N; at < hi; at += kWave * N) {
            const Vec<Scalar, N> x = next;
            if (at + kWave * N < hi)
                next = load_vec<Scalar, N>(me.row + at + kWave * N);
            float out[N];
#pragma unroll
            for (int e = 0; e < N; ++e)
                sum += of(x[e], at + e, out[e]);
            then(at, out);
        }
    };
    // Where their sum is known the probabilities go out in the same pass (rows of 128257, top_p of 0.9: 115 us for 149).
    const auto nothing = [](int, const float(&)[N]) {};
    if (probs && kept_sum) {
        const double inv = me.unit / static_cast<double>(kept_sum);
        stretch(
            [&](float l, int i, float &out) -> uint64_t {
                double w;
                out = 0.f;
                if (!me.kept(l, i, w))
                    return 0;
                out = static_cast<float>(w * inv);
                return me.whole(w);
            },
            put);
    } else if (!by_count && !by_sum && me.least == 0.0) {
        stretch([&](float l, int, float &) { return me.whole(me.weight(l)); }, nothing);
    } else {
        stretch([&](float l, int i, float &) { return share(l, i); }, nothing);
    }
    sum = wave_reduce(sum, Sum{});
    __syncthreads();
    if (lane == 0)
        lds().scan[0][wave] = sum;
    __syncthreads();
    uint64_t parts = 0;
    for (int w = 0; w < kWaves; ++w)
        parts += lds().scan[0][w];
    const double total = static_cast<double>(parts);
    if (token) {
        const double threshold = u * total;
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
        // The stretch in turns of N tokens a thread, until the sum passes; where it never does, its last with a weight
        int found = V, last = -1;
        for (int base = from; base < to && found == V; base += kThreads * N) {
            const int begin = base + tid * N;
            Vec<Scalar, N> x{};
            if (begin + N <= V)
                x = load_vec<Scalar, N>(me.row + begin);
            uint64_t parts_of[N], own = 0;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int i = begin + e;
                const float l = begin + N <= V ? x[e] : i < V ? load_f32(me.row + i) : 0.f;
                parts_of[e] = share(l, i);
                parts_of[e] = i < to ? parts_of[e] : 0;
                own += parts_of[e];
            }
            uint64_t run = before + me.block_scan(own, 1);
            int here = V, latest = -1;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                run += parts_of[e];
                const bool on = parts_of[e] > 0;
                latest = on ? begin + e : latest;
                here = on && here == V && static_cast<double>(run) > threshold ? begin + e : here;
            }
            before += me.block_reduce(own, Sum{});
            me.block_reduce(here, Least{}, latest, Most{});
            found = here, last = max(last, latest);
        }
        if (tid == 0)
            *token = found < V ? found : last;
    }
    if (probs) {
        const double inv = me.unit / total;
        for (int at = tid * N; at < full && !kept_sum; at += kThreads * N) {
            const Vec<Scalar, N> x = load_vec<Scalar, N>(me.row + at);
            float out[N];
#pragma unroll
            for (int e = 0; e < N; ++e)
                out[e] = value(x[e], at + e, inv);
            put(at, out);
        }
        if (full + tid < V)
            probs[full + tid] = value(load_f32(me.row + full + tid), full + tid, inv);
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
