// The selective scan: jobs of its launches and device helpers they share.
//
// S numbers h of state (fp32) per sequence and channel, per token and channel d of group g:
//     dt = softplus(raw + dt_bias)          (or raw + dt_bias)
//     h_n <- e^(dt A_dn) h_n + dt x B_gn;   s = sum_n C_gn h_n + skip x;   y = s silu(gate)   (or s)
//
// Four adjacent lanes hold a channel, NR = S / 4 (rounded up to 1, 2, 3, 4, 6, 8, 12 or 16) states each; a wave
// holds 16 channels. Tokens are taken four at a time: what a token needs once (its softplus, its gate)
// is done by one of the four lanes, and given to the others within vector instructions.
#pragma once

#include "buffer_window.hpp"
#include "sequences.hpp"
#include "vector16.hpp"

#include <type_traits>

namespace ramnet {

enum : int { kScanMaxStates = 64, kScanKept = 16, kScanStepTokens = 8, kScanStride = 1 << 22 };

struct ScanJob {
    SequenceJob seq;
    const void *x, *dt, *gate;  // (B, T, D), strides of batch row and token; gate may be null
    const void *B, *C;          // (B, T, G, S), strides of batch row, token and group
    const float *A;             // (D, S)
    const float *skip, *bias;   // (D), or null
    const float *init;          // (N, D, S), or null: zeros
    void *y;                    // (B, T, D) dense
    float *state;               // (N, D, S); may be init
    int dtype, softplus, D, S, G;
    int64_t x_at[2], dt_at[2], gate_at[2], B_at[3], C_at[3];  // (of tokens below kScanStride)
    int step;                   // tokens of a piece, a multiple of kScanKept
    // workspace, [piece][D][4 NR] and [piece][D]
    float *ends;                // state after each piece from zeros
    double *spans;              // sum of a piece's dt
    // of a training call: the state before every kScanKept tokens of a sequence, [slot][D][4 NR]
    float *kept;
};

// Gradients: of x, dt, gate, B and C in their types, of the others fp32; dense.
struct ScanGrads {
    const void *dy;       // (B, T, D), strides dy_at
    const float *dstate;  // (N, D, S), or null: zeros
    void *dx, *ddt, *dgate, *dB, *dC;
    float *dA, *dskip, *dbias, *dinit;  // (dskip, dbias and dinit may be null)
    int64_t dy_at[2];
    // workspace
    float *backs;    // [piece][D][4 NR] gradient of the state before each piece, from its own outputs
    float *groups;   // [channel block][B T][2][4 NR] sums of dB and dC over the block's channels
    float *sums;     // [piece][D][4 NR + 2] sums of dA, dskip and dbias over the piece's tokens
};

// NR of S states.
__host__ __device__ inline int scan_lane_states(int S) {
    for (const int states : {1, 2, 3, 4, 6, 8, 12})
        if (S <= 4 * states)
            return states;
    return 16;
}

// The place of a sequence's kept states: sequence `seq` from token lo on, one for every kScanKept tokens.
__host__ __device__ inline int64_t scan_slot(const SequenceJob &job, int seq, int lo) {
    return job.cu ? static_cast<int64_t>(lo / kScanKept) + seq
                  : static_cast<int64_t>(seq) * ((job.T + kScanKept - 1) / kScanKept);
}
__host__ __device__ inline int64_t scan_slots(const SequenceJob &job) {
    return job.cu ? static_cast<int64_t>(job.T) / kScanKept + job.N + 1
                  : static_cast<int64_t>(job.B) * ((job.T + kScanKept - 1) / kScanKept);
}

// Value of lane K of each four.
template<int K>
__device__ __forceinline__ float quad_lane(float x) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), K * 0x55, 0xF, 0xF, true));
}
template<int XOR>
__device__ __forceinline__ float quad_swap(float x) {
    constexpr int kControl = XOR == 1 ? 0xB1 : 0x4E;  // lanes 1 0 3 2, 2 3 0 1
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), kControl, 0xF, 0xF, true));
}

// Of four values a lane, each summed over the four lanes: lane i has the sum of v[i].
__device__ __forceinline__ float quad_sums(const float (&v)[4], int lane) {
    const bool odd = lane & 1, high = lane & 2;
    const float a = (odd ? v[1] : v[0]) + quad_swap<1>(odd ? v[0] : v[1]);
    const float b = (odd ? v[3] : v[2]) + quad_swap<1>(odd ? v[2] : v[3]);
    return (high ? b : a) + quad_swap<2>(high ? a : b);
}

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// log(1 + e^x) = max(x, 0) + log(1 + e), e = e^-|x| in (0, 1], the latter as 2 atanh(s), s = e / (2 + e): atanh(s) / s on
// (0, 1/3] by the polynomial in s^2 whose greatest relative error is least, 8e-9. `e` comes out for the derivative.
__device__ __forceinline__ float softplus(float x, float &e) {
    e = __builtin_amdgcn_exp2f(-fabsf(x) * kLog2e);
    const float s = e * __builtin_amdgcn_rcpf(2.f + e), q = s * s;
    const float sum = fmaf(fmaf(fmaf(fmaf(0.140891677f, q, 0.139803015f), q, 0.200124551f), q, 0.333331573f), q, 1.f);
    const float above = __int_as_float(max(__float_as_int(x), 0));  // (max(x, 0): of floats it is two instructions)
    return fmaf(2.f * s, sum, above);
}

// Writes of some lanes of a wave to LDS before reads of others.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

enum : int { kScanThreads = 256, kScanChannels = kScanThreads / 4 };

// Which channel a lane holds a quarter of; where there is none, the group's last one, which it does not write.
struct ScanPlace {
    int piece, group, channel, sub, block;  // (block: which 64 channels of the group)
    bool valid;

    __device__ __forceinline__ ScanPlace(const ScanJob &job) {
        const int wide = job.D / job.G, per_group = (wide + kScanChannels - 1) / kScanChannels;
        const int id = static_cast<int>(blockIdx.x), per_piece = per_group * job.G;
        piece = id / per_piece;
        const int at = id - piece * per_piece;
        group = at / per_group;
        block = at - group * per_group;
        const int c = block * kScanChannels + static_cast<int>(threadIdx.x) / 4;
        valid = c < wide;
        channel = group * wide + min(c, wide - 1);
        sub = static_cast<int>(threadIdx.x) % 4;
    }
};

// x as a value that the compiler cannot make from others again: offsets are made once, or (in load) for each load.
__device__ __forceinline__ int anew(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// The windows over a tensor's rows, one tile after the other: a tile's tokens that are there (none: it is empty). Steps
// from tile to tile are kept, as addresses made anew are some 25 scalar instructions a tensor and tile.
template<typename Scalar, int kSign = 1>
struct ScanCursor {
    const char *p;
    int step, rest;  // bytes from token to token; of the last token's row less a step

    __device__ __forceinline__ ScanCursor(const void *base, int64_t from, int64_t stride, int width)
        : p(reinterpret_cast<const char *>(static_cast<const Scalar *>(base) + from)),
          step(static_cast<int>(stride) * static_cast<int>(sizeof(Scalar))), rest(width * static_cast<int>(sizeof(Scalar)) - step) {}
    // `left`: tokens from this tile's first to the last.
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t next(int left) {
        const char *at = p;
        p += kSign * kScanKept * static_cast<int64_t>(step);
        return window(at, left > 0 ? min(left, kScanKept) * step + rest : 0);
    }
};

// One value of a lane's channel for each four tokens of a tile, through a window over it.
template<typename Scalar>
struct ScanRows {
    int at, step;  // bytes: the lane's place in the first four tokens; four tokens on

    __device__ __forceinline__ ScanRows(const ScanPlace &place, int64_t stride, bool on) {
        step = 4 * static_cast<int>(stride) * static_cast<int>(sizeof(Scalar));
        at = anew(on ? (place.sub * static_cast<int>(stride) + place.channel) * static_cast<int>(sizeof(Scalar)) : kNowhere);
    }
    // (kAnew: offsets are made for each load; kept over a loop they fill registers)
    template<bool kAnew = false>
    __device__ __forceinline__ void load(uint32_t (&to)[kScanKept / 4], __amdgpu_buffer_rsrc_t rows) const {
        const int from = kAnew ? anew(at) : at;
#pragma unroll
        for (int g = 0; g < kScanKept / 4; ++g)
            to[g] = buffer_bits<Scalar>(rows, from + g * step);
    }
};

// A wave's share of B or C of a tile, which it keeps in LDS as fp32, [token][4 NR], those past S zero.
template<typename Scalar, int NR>
struct ScanGroups {
    static constexpr int kRow = 4 * NR, kFloats = kScanKept * kRow;
    // tokens that a load of the wave spans (lanes past them have no part), and loads of a tile
    static constexpr int kSpan = kWave / kRow >= 4 ? kWave / kRow / 4 * 4 : kWave / kRow >= 2 ? 2 : 1, kLoads = kScanKept / kSpan;
    static_assert(kLoads * kSpan == kScanKept, "whole loads");
    int at, step, to;

    __device__ __forceinline__ ScanGroups(int lane, int64_t stride, int S) {
        const bool on = lane / kRow < kSpan;
        step = kSpan * static_cast<int>(stride) * static_cast<int>(sizeof(Scalar));
        at = anew(on && lane % kRow < S ? (lane / kRow * static_cast<int>(stride) + lane % kRow) * static_cast<int>(sizeof(Scalar))
                                        : kNowhere);
        to = on ? lane : -1;
    }
    template<bool kAnew = false>
    __device__ __forceinline__ void load(uint32_t (&to)[kLoads], __amdgpu_buffer_rsrc_t rows) const {
        const int from = kAnew ? anew(at) : at;
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
            to[i] = buffer_bits<Scalar>(rows, from + i * step);
    }
    __device__ __forceinline__ void store(float *tile, const uint32_t (&from)[kLoads]) const {
        if (kSpan * kRow == kWave || to >= 0) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                tile[i * kSpan * kRow + to] = bits_f32<Scalar>(from[i]);
        }
    }
};

// NR states of a channel, those past S zero. `p`: state n0 of it.
template<int NR>
__device__ __forceinline__ void load_states(float (&h)[NR], const float *p, int count) {
    if (count >= NR) {
#pragma unroll
        for (int j = 0; j < NR; ++j)
            h[j] = p[j];
    } else {
#pragma unroll
        for (int j = 0; j < NR; ++j)
            h[j] = j < count ? p[j] : 0.f;
    }
}
template<int NR>
__device__ __forceinline__ void store_states(float *p, const float (&h)[NR], int count) {
    if (count >= NR) {
#pragma unroll
        for (int j = 0; j < NR; ++j)
            p[j] = h[j];
    } else {
#pragma unroll
        for (int j = 0; j < NR; ++j)
            if (j < count)
                p[j] = h[j];
    }
}

// Whether a call walks its few tokens without staging (it then needs no workspace).
bool scan_is_step(const ScanJob &job);
// Places the buffers of a call in `base`, or sizes them (null base); chooses its pieces.
int64_t scan_layout(ScanJob &job, bool backward, char *base, ScanGrads *grads);
int64_t scan_kept_bytes(const ScanJob &job);
hipError_t launch_scan(const ScanJob &job, hipStream_t stream, const char **why);
hipError_t launch_scan_backward(const ScanJob &job, const ScanGrads &grads, hipStream_t stream, const char **why);

}  // namespace ramnet
