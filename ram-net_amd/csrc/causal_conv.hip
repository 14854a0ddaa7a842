// Short causal convolution of each channel over its last W <= 8 tokens, and its gradients.
//
// The forward is bound by memory: x is read once and y written once, 2 W operations an element. A
// thread takes 16 bytes of adjacent channels and walks a piece of time with the last W - 1 inputs in
// registers; what a piece reads of its forerunner comes from the L2. So is the backward in fp32 (x and dy
// read, dx written; 4.7 TB/s). In 16 bits it is not: its instructions a channel are the same for half the bytes, and at
// two waves a SIMD loads of four tokens and the work on them take turns (vector units 67% busy, 3.3 TB/s).
// Rows are read and written at any alignment: the last channels of a row whose length is no
// multiple of 16 bytes are taken with some of those before them, which two threads then compute alike.
//
// 8 x 4096 x 2048, W 4, bf16: 54.6 us, 4.9 TB/s, what a large copy reaches (fp32 112 us, 4.8 TB/s). 64 rows of one token x
// 4096: 6 us. The backward of 4 x 2048 x 2048, bf16: 38.6 us and 4 for the sums, the forward 17.9; 8003 packed tokens x
// 1001, W 3, fp32: 25 and 5, the forward 16.
#include "causal_conv.hpp"
#include "ramnet_kernels.hpp"
#include "vector16.hpp"

#include <type_traits>

namespace ramnet {

namespace {

constexpr int kThreads = 256, kAhead = 8;

// A thread's piece and channels: threads take pieces in order, all channels of a piece side by side.
template<int VEC>
struct ConvPlace {
    int piece, c0;  // (c0: its first channel)
    int others;     // how many of its channels, from the first on, the thread before has too

    __device__ __forceinline__ bool find(const ConvJob &job, int64_t pieces) {
        const int per_row = (job.D + VEC - 1) / VEC;
        const int64_t begin = static_cast<int64_t>(blockIdx.x) * kThreads;
        const int64_t p0 = begin / per_row;
        const int r = static_cast<int>(begin - p0 * per_row) + static_cast<int>(threadIdx.x);
        const int lane = r % per_row;
        const int64_t p = p0 + r / per_row;
        piece = static_cast<int>(p);
        c0 = min(lane * VEC, job.D - VEC);
        others = lane * VEC - c0;
        return p < pieces;
    }
};

// Stores all but the first `skip` elements.
template<typename Scalar, int VEC>
__device__ __forceinline__ void store_from(Scalar *p, const Vec<Scalar, VEC> &v, int skip) {
    if (VEC == 1 || skip == 0) {
        store_vec<Scalar, VEC>(p, v);
    } else {
#pragma unroll
        for (int e = 1; e < VEC; ++e)
            if (e >= skip)
                store_vec<Scalar, 1>(p + e, {{sizeof(Scalar) == 4 ? v.w[e % Vec<Scalar, VEC>::kWords]
                                                                  : v.w[e / 2] >> (e % 2 * 16)}});
    }
}

template<typename Scalar, int W, int VEC>
struct ConvTaps {
    float weight[W][VEC], bias[VEC];

    __device__ __forceinline__ ConvTaps(const ConvJob &job, int c0) {
        const Scalar *w = static_cast<const Scalar *>(job.weight) + static_cast<int64_t>(c0) * W;
        Vec<Scalar, VEC> rows[W];  // (adjacent in memory: all W taps of one channel, then the next one's)
#pragma unroll
        for (int j = 0; j < W; ++j)
            rows[j] = load_vec<Scalar, VEC>(w + j * VEC);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
#pragma unroll
            for (int j = 0; j < W; ++j)
                weight[j][e] = rows[(e * W + j) / VEC][(e * W + j) % VEC];
            bias[e] = job.bias ? load_f32(static_cast<const Scalar *>(job.bias) + c0 + e) : 0.f;
        }
    }
};

// The input of a sequence at `place` of it; before its first token a row of its state.
template<typename Scalar, int W, int VEC>
__device__ __forceinline__ Vec<Scalar, VEC> conv_input(const ConvJob &job, const TimePiece &piece, int c0, int place) {
    if (place >= 0)
        return load_vec<Scalar, VEC>(static_cast<const Scalar *>(job.x) + piece.row * job.x_at[0] +
                                     (piece.lo + place) * job.x_at[1] + c0);
    if (job.init)
        return load_vec<Scalar, VEC>(static_cast<const Scalar *>(job.init) +
                                     (static_cast<int64_t>(piece.seq) * (W - 1) + place + W - 1) * job.D + c0);
    return {};
}

template<typename Scalar, int W, int VEC>
__global__ __launch_bounds__(kThreads) void conv_kernel(const ConvJob job, int64_t pieces) {
    ConvPlace<VEC> at;
    TimePiece piece;
    if (!at.find(job, pieces) || !time_piece(job.seq, job.step, at.piece, piece))
        return;
    const int D = job.D, c0 = at.c0;
    // Channels of two threads have the same results from both. In place that is not so (one may read
    // the state that the other has written): then the thread before has them alone.
    const int skip = job.init && job.init == job.state ? at.others : 0;
    const int64_t row = static_cast<int64_t>(piece.row) * job.seq.T;
    Scalar *y = static_cast<Scalar *>(job.y) + c0;
    if (piece.seq >= 0 && (piece.len > 0 || piece.at == 0)) {
        const ConvTaps<Scalar, W, VEC> taps(job, c0);
        float win[W][VEC];  // the inputs of W tokens, the latest last
        const int place = piece.t0 - piece.lo;
#pragma unroll
        for (int j = 0; j + 1 < W; ++j) {
            const Vec<Scalar, VEC> v = conv_input<Scalar, W, VEC>(job, piece, c0, place - (W - 1) + j);
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                win[j + 1][e] = v[e];
        }
        // The state: by the one thread that also reads it, so that it may be updated in place.
        if (W > 1 && piece.at == 0) {
            Vec<Scalar, VEC> rows[W];
#pragma unroll
            for (int i = 0; i + 1 < W; ++i)
                rows[i] = conv_input<Scalar, W, VEC>(job, piece, c0, piece.hi - piece.lo - (W - 1) + i);
#pragma unroll
            for (int i = 0; i + 1 < W; ++i)
                store_from<Scalar, VEC>(static_cast<Scalar *>(job.state) +
                                            (static_cast<int64_t>(piece.seq) * (W - 1) + i) * D + c0,
                                        rows[i], skip);
        }
        const Scalar *x = static_cast<const Scalar *>(job.x) + piece.row * job.x_at[0] + piece.t0 * job.x_at[1] + c0;
        for (int t0 = 0; t0 < piece.len; t0 += kAhead) {
            Vec<Scalar, VEC> next[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
                next[i] = t0 + i < piece.len ? load_vec<Scalar, VEC>(x + (t0 + i) * job.x_at[1]) : Vec<Scalar, VEC>{};
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                float out[VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
#pragma unroll
                    for (int j = 0; j + 1 < W; ++j)
                        win[j][e] = win[j + 1][e];
                    win[W - 1][e] = next[i][e];
                    float s = taps.bias[e];
#pragma unroll
                    for (int j = 0; j < W; ++j)
                        s = fmaf(taps.weight[j][e], win[j][e], s);
                    out[e] = job.silu ? s * sigmoid(s) : s;
                }
                if (t0 + i < piece.len)
                    store_from<Scalar, VEC>(y + (row + piece.t0 + t0 + i) * D, round_vec<Scalar, VEC>(out), skip);
            }
        }
    }
    for (int i = 0; i < piece.rest; ++i)
        store_vec<Scalar, VEC>(y + (row + piece.t0 + piece.len + i) * D, Vec<Scalar, VEC>{});
}

// Gradients of a piece's inputs, and its sums of dweight and dbias. The inputs' convolution is made again; a gradient
// is whole W - 1 tokens later, also where these lie in the next piece.
template<typename Scalar, int W, int VEC>
__global__ __launch_bounds__(kThreads, W <= 4 && sizeof(Scalar) == 2 ? 4 : 2) void conv_backward_kernel(
    const ConvJob job, const ConvGrads grads, int64_t pieces) {
    ConvPlace<VEC> at;
    TimePiece piece;
    if (!at.find(job, pieces))
        return;
    const int D = job.D, c0 = at.c0;
    float dtap[W][VEC], dbias[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        dbias[e] = 0.f;
#pragma unroll
        for (int j = 0; j < W; ++j)
            dtap[j][e] = 0.f;
    }
    const bool any = time_piece(job.seq, job.step, at.piece, piece);
    if (any) {
        const int64_t row = static_cast<int64_t>(piece.row) * job.seq.T;
        Scalar *dx = static_cast<Scalar *>(grads.dx) + c0;
        if (piece.seq >= 0 && piece.at < piece.count) {
            const ConvTaps<Scalar, W, VEC> taps(job, c0);
            const int n = piece.hi - piece.lo, begin = piece.t0 - piece.lo, end = begin + piece.len;
            const int stop = min(end + W - 1, n);  // (tokens up to there reach back into the piece)
            float win[W][VEC], pend[W][VEC];       // pend[j]: gradient of the input at t - (W - 1) + j so far
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const Vec<Scalar, VEC> v = j > 0 ? conv_input<Scalar, W, VEC>(job, piece, c0, begin - W + j)
                                                 : Vec<Scalar, VEC>{};
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    win[j][e] = v[e], pend[j][e] = 0.f;
            }
            // The gradient of the input at `place` is whole: the new state's with it, it goes out.
            auto emit = [&](int place, const float (&sum)[VEC]) {
                if (place >= end || (begin > 0 && place < begin))
                    return;
                float out[VEC];
                Vec<Scalar, VEC> kept{};
                const int i = place - (n - (W - 1));
                if (grads.dstate && i >= 0)
                    kept = load_vec<Scalar, VEC>(static_cast<const Scalar *>(grads.dstate) +
                                                 (static_cast<int64_t>(piece.seq) * (W - 1) + i) * D + c0);
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    out[e] = sum[e] + kept[e];
                const Vec<Scalar, VEC> v = round_vec<Scalar, VEC>(out);
                if (place >= 0)
                    store_vec<Scalar, VEC>(dx + (row + piece.lo + place) * D, v);
                else if (grads.dinit)
                    store_vec<Scalar, VEC>(static_cast<Scalar *>(grads.dinit) +
                                               (static_cast<int64_t>(piece.seq) * (W - 1) + place + W - 1) * D + c0, v);
            };
            const Scalar *x = static_cast<const Scalar *>(job.x) + piece.row * job.x_at[0] + piece.lo * job.x_at[1] + c0;
            const Scalar *dy = static_cast<const Scalar *>(grads.dy) + piece.row * grads.dy_at[0] +
                               piece.lo * grads.dy_at[1] + c0;
            auto token = [&](int t, const Vec<Scalar, VEC> &xt, const Vec<Scalar, VEC> &dt, auto own) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
#pragma unroll
                    for (int j = 0; j + 1 < W; ++j)
                        win[j][e] = win[j + 1][e], pend[j][e] = pend[j + 1][e];
                    win[W - 1][e] = xt[e], pend[W - 1][e] = 0.f;
                    float d = dt[e];
                    if (job.silu) {
                        float s = taps.bias[e];
#pragma unroll
                        for (int j = 0; j < W; ++j)
                            s = fmaf(taps.weight[j][e], win[j][e], s);
                        const float g = sigmoid(s);
                        d *= g * (1.f + s * (1.f - g));
                    }
#pragma unroll
                    for (int j = 0; j < W; ++j) {
                        pend[j][e] = fmaf(taps.weight[j][e], d, pend[j][e]);
                        if constexpr (decltype(own)::value)
                            dtap[j][e] = fmaf(d, win[j][e], dtap[j][e]);
                    }
                    if constexpr (decltype(own)::value)
                        dbias[e] += d;
                }
                emit(t - (W - 1), pend[0]);
            };
            constexpr int kDeep = 4;
            for (int t0 = begin; t0 < end; t0 += kDeep) {
                Vec<Scalar, VEC> xs[kDeep], ds[kDeep];
#pragma unroll
                for (int i = 0; i < kDeep; ++i) {
                    xs[i] = t0 + i < end ? load_vec<Scalar, VEC>(x + (t0 + i) * job.x_at[1]) : Vec<Scalar, VEC>{};
                    ds[i] = t0 + i < end ? load_vec<Scalar, VEC>(dy + (t0 + i) * grads.dy_at[1]) : Vec<Scalar, VEC>{};
                }
#pragma unroll
                for (int i = 0; i < kDeep; ++i) {
                    if (t0 + i >= end)
                        break;
                    token(t0 + i, xs[i], ds[i], std::true_type{});
                }
            }
            for (int t = end; t < stop; ++t)  // (tokens behind the piece count for its inputs alone)
                token(t, load_vec<Scalar, VEC>(x + t * job.x_at[1]), load_vec<Scalar, VEC>(dy + t * grads.dy_at[1]),
                      std::false_type{});
            // (behind a sequence's last token: what is still pending)
#pragma unroll
            for (int j = 1; j < W; ++j)
                emit(stop - W + j, pend[j]);
        }
        for (int i = 0; i < piece.rest; ++i)
            store_vec<Scalar, VEC>(dx + (row + piece.t0 + piece.len + i) * D, Vec<Scalar, VEC>{});
    }
    // Rows of sums, one a piece: added up in order by conv_sum_kernel.
    float *to = grads.partial + static_cast<int64_t>(at.piece) * (W + 1) * D + c0;
#pragma unroll
    for (int e = 0; e < VEC; ++e)
        if (e >= at.others) {
#pragma unroll
            for (int j = 0; j < W; ++j)
                to[static_cast<int64_t>(j) * D + e] = dtap[j][e];
            to[static_cast<int64_t>(W) * D + e] = dbias[e];
        }
}

// dweight and dbias from the pieces' sums, in one order: a block takes 64 columns of (W + 1) D,
// its 16 waves every 16th piece each.
template<typename Scalar>
__global__ __launch_bounds__(1024) void conv_sum_kernel(const ConvJob job, const ConvGrads grads, int pieces) {
    __shared__ float sums[16][kWave];
    const int lane = static_cast<int>(threadIdx.x) % kWave, wave = static_cast<int>(threadIdx.x) / kWave;
    const int64_t columns = static_cast<int64_t>(job.W + 1) * job.D, column = static_cast<int64_t>(blockIdx.x) * kWave + lane;
    float sum = 0.f;
    if (column < columns) {
#pragma unroll 8
        for (int p = wave; p < pieces; p += 16)
            sum += grads.partial[p * columns + column];
    }
    sums[wave][lane] = sum;
    __syncthreads();
    if (wave > 0 || column >= columns)
        return;
    for (int w = 1; w < 16; ++w)
        sum += sums[w][lane];
    const int j = static_cast<int>(column / job.D), d = static_cast<int>(column - static_cast<int64_t>(j) * job.D);
    if (j < job.W)
        store_f32(static_cast<Scalar *>(grads.dweight) + static_cast<int64_t>(d) * job.W + j, sum);
    else if (grads.dbias)
        store_f32(static_cast<Scalar *>(grads.dbias) + d, sum);
}

template<typename Scalar, int W, int VEC>
hipError_t launch_of(const ConvJob &job, const ConvGrads *grads, int64_t pieces, hipStream_t stream) {
    const int64_t threads = pieces * ((job.D + VEC - 1) / VEC);
    const dim3 grid(static_cast<unsigned>((threads + kThreads - 1) / kThreads)), block(kThreads);
    if constexpr (VEC <= 4) {
        if (grads) {
            hipLaunchKernelGGL((conv_backward_kernel<Scalar, W, VEC>), grid, block, 0, stream, job, *grads, pieces);
            return hipGetLastError();
        }
    }
    hipLaunchKernelGGL((conv_kernel<Scalar, W, VEC>), grid, block, 0, stream, job, pieces);
    return hipGetLastError();
}

template<typename Scalar, int W>
hipError_t launch_width(const ConvJob &job, const ConvGrads *grads, int64_t pieces, hipStream_t stream) {
    // (the backward holds four rows of W a channel: with 16 bytes of 16-bit channels they leave two waves a SIMD, 53 us
    // of 4 x 2048 x 2048 for 36)
    constexpr int kWide = 16 / sizeof(Scalar), kNarrow = 4;
    if (grads)
        return job.D >= kNarrow ? launch_of<Scalar, W, kNarrow>(job, grads, pieces, stream)
                                : launch_of<Scalar, W, 1>(job, grads, pieces, stream);
    return job.D >= kWide ? launch_of<Scalar, W, kWide>(job, grads, pieces, stream)
                          : launch_of<Scalar, W, 1>(job, grads, pieces, stream);
}

template<typename Scalar>
hipError_t launch_type(const ConvJob &job, const ConvGrads *grads, int64_t pieces, hipStream_t stream) {
    switch (job.W) {
        case 1: return launch_width<Scalar, 1>(job, grads, pieces, stream);
        case 2: return launch_width<Scalar, 2>(job, grads, pieces, stream);
        case 3: return launch_width<Scalar, 3>(job, grads, pieces, stream);
        case 4: return launch_width<Scalar, 4>(job, grads, pieces, stream);
        case 5: return launch_width<Scalar, 5>(job, grads, pieces, stream);
        case 6: return launch_width<Scalar, 6>(job, grads, pieces, stream);
        case 7: return launch_width<Scalar, 7>(job, grads, pieces, stream);
        default: return launch_width<Scalar, 8>(job, grads, pieces, stream);
    }
}

hipError_t launch_any(const ConvJob &job, const ConvGrads *grads, hipStream_t stream, const char **why) {
    const int64_t pieces = most_pieces(job.seq, job.step);
    if (job.seq.cu) {
        const hipError_t err = launch_sequences(job.seq, job.step, stream);
        if (err != hipSuccess)
            return err;
    }
    switch (job.dtype) {
        case kF32: return launch_type<float>(job, grads, pieces, stream);
        case kF16: return launch_type<_Float16>(job, grads, pieces, stream);
        case kBF16: return launch_type<bf16_t>(job, grads, pieces, stream);
        default: *why = "causal_conv: unsupported dtype"; return hipErrorInvalidValue;
    }
}

}  // namespace

// Pieces of 16 tokens re-read W - 1 of theirs from the cache. The backward leaves W + 1 rows of sums a piece: a quarter
// of what it reads with 16 bits and W 4, an eighth with pieces of 32, which it takes where there are enough of them
// (4 x 2048 x 2048 channels, with the sums: pieces of 16 and of 32 43 us, of 64 56; 16000 x 4096 with 16 138, with 32 136).
int conv_step(const ConvJob &job, bool backward) {
    const int64_t rows = static_cast<int64_t>(job.seq.B) * job.seq.T * ((job.D + 3) / 4);
    return backward && rows >= (1 << 21) ? 32 : 16;
}

int64_t conv_layout(ConvJob &job, bool backward, char *base, ConvGrads *grads) {
    job.step = conv_step(job, backward);
    int64_t size = 0;
    auto region = [&](int64_t bytes) {
        char *at = base ? base + size : nullptr;
        size += (bytes + 255) / 256 * 256;
        return at;
    };
    if (job.seq.cu) {
        job.seq.bounds = reinterpret_cast<int32_t *>(region((job.seq.N + 1) * 4LL));
        job.seq.first = reinterpret_cast<int32_t *>(region((job.seq.N + 1) * 4LL));
    }
    if (backward) {
        float *partial = reinterpret_cast<float *>(region(most_pieces(job.seq, job.step) * (job.W + 1) * job.D * 4));
        if (grads)
            grads->partial = partial;
    }
    return size;
}

hipError_t launch_conv(const ConvJob &job, hipStream_t stream, const char **why) {
    return launch_any(job, nullptr, stream, why);
}

hipError_t launch_conv_backward(const ConvJob &job, const ConvGrads &grads, hipStream_t stream, const char **why) {
    const hipError_t err = launch_any(job, &grads, stream, why);
    if (err != hipSuccess)
        return err;
    const int pieces = static_cast<int>(most_pieces(job.seq, job.step));
    const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(job.W + 1) * job.D + kWave - 1) / kWave)), block(1024);
    switch (job.dtype) {
        case kF32: hipLaunchKernelGGL(conv_sum_kernel<float>, grid, block, 0, stream, job, grads, pieces); break;
        case kF16: hipLaunchKernelGGL(conv_sum_kernel<_Float16>, grid, block, 0, stream, job, grads, pieces); break;
        default: hipLaunchKernelGGL(conv_sum_kernel<bf16_t>, grid, block, 0, stream, job, grads, pieces); break;
    }
    return hipGetLastError();
}

}  // namespace ramnet
