// Selective scan, gradients. With G_t the gradient of the state after token t,
//
//     G_t = C_t ds_t + a_{t+1} G_{t+1},   a_t = e^(dt_t A)
//     dC_t = ds_t h_t,   dB_t = dt_t x_t G_t          (both summed over a group's channels)
//     d(dt x)_t = B_t . G_t,   d(dt_t) = x_t d(dt x)_t + sum_n A G_t a_t h_{t-1},   dA = sum_t dt_t G_t a_t h_{t-1}
//
// The states are walked again from those kept every 16 tokens; a_t and a_t h_{t-1} of a tile stay in
// registers for the way back.
#include "ramnet_kernels.hpp"
#include "selective_scan.hpp"

namespace ramnet {

namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave, kChannels = kThreads / 4, kTile = kScanKept;

template<int CONTROL, int BANKS>
__device__ __forceinline__ float row_move(float old, float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(old), __float_as_int(x), CONTROL, 0xF, BANKS, false));
}

// Of 16 values a lane, each summed over the 16 lanes of the same place in their four: those of four q have value q.
__device__ __forceinline__ float channel_sums(float (&v)[16], int lane) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i + 8]), false, false);
        v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]), __float_as_uint(v[i + 4]), false, false);
        v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    const bool eight = lane & 8, four = lane & 4;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float keep = eight ? v[i + 2] : v[i], give = eight ? v[i] : v[i + 2];
        v[i] = keep + row_move<0x128, 0xF>(0.f, give);  // row_ror:8
    }
    const float keep = four ? v[1] : v[0], give = four ? v[0] : v[1];
    const float up = row_move<0x104, 0x5>(0.f, give);       // row_shl:4, lanes without bit 2
    return keep + row_move<0x114, 0xA>(up, give);           // row_shr:4, lanes with it
}

// Which channel a lane holds a quarter of; where there is none, the group's last one, which it does not write.
struct BackPlace {
    int piece, group, channel, sub, block;
    bool valid;

    __device__ __forceinline__ BackPlace(const ScanJob &job) {
        const int wide = job.D / job.G, per_group = (wide + kChannels - 1) / kChannels;
        const int id = static_cast<int>(blockIdx.x), per_piece = per_group * job.G;
        piece = id / per_piece;
        const int at = id - piece * per_piece;
        group = at / per_group;
        block = at - group * per_group;
        const int c = block * kChannels + static_cast<int>(threadIdx.x) / 4;
        valid = c < wide;
        channel = group * wide + min(c, wide - 1);
        sub = static_cast<int>(threadIdx.x) % 4;
    }
};

// What a lane reads of a tile: its channel's values of one token of each four, and its share of B and C.
template<typename Scalar, int NR>
struct BackTile {
    static constexpr int kRow = 8 * NR, kFloats = kTile * kRow, kLoads = kFloats / kWave;
    uint32_t x[kTile / 4], dt[kTile / 4], gate[kTile / 4], dy[kTile / 4], groups[kLoads];

    __device__ __forceinline__ void load(const ScanJob &job, const ScanGrads &grads, const TimePiece &piece,
                                         const BackPlace &at, int t, int lane, bool with_b) {
        const int64_t row = piece.row;
#pragma unroll
        for (int g = 0; g < kTile / 4; ++g) {
            const int64_t token = piece.t0 + min(t + 4 * g + at.sub, piece.len - 1);
            auto value = [&](const void *p, const int64_t *stride) {
                return load_bits(static_cast<const Scalar *>(p) + row * stride[0] + token * stride[1] + at.channel);
            };
            x[g] = with_b ? value(job.x, job.x_at) : 0u;
            dt[g] = value(job.dt, job.dt_at);
            gate[g] = job.gate ? value(job.gate, job.gate_at) : 0u;
            dy[g] = value(grads.dy, grads.dy_at);
        }
        const Scalar *B = static_cast<const Scalar *>(job.B) + row * job.B_at[0] + at.group * job.B_at[2];
        const Scalar *C = static_cast<const Scalar *>(job.C) + row * job.C_at[0] + at.group * job.C_at[2];
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int e = i * kWave + lane, n = e % (4 * NR);
            const int64_t token = piece.t0 + min(t + e / kRow, piece.len - 1);
            const bool second = e % kRow >= 4 * NR;
            groups[i] = n < job.S && (second || with_b)
                            ? load_bits(second ? C + token * job.C_at[1] + n : B + token * job.B_at[1] + n) : 0u;
        }
    }
    __device__ __forceinline__ void store_groups(float *to, int lane) const {
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
            to[i * kWave + lane] = bits_f32<Scalar>(groups[i]);
    }
};

// A decay of -inf is held to a finite one: times a dt of 0 (of a token that does not count) it gives 1.
template<int NR>
__device__ __forceinline__ void load_decays(float (&A2)[NR], const ScanJob &job, int channel, int n0) {
    load_states<NR>(A2, job.A + static_cast<int64_t>(channel) * job.S + n0, job.S - n0);
#pragma unroll
    for (int j = 0; j < NR; ++j) {
        const float a = A2[j] * kLog2e;
        A2[j] = a < -3e38f ? -3e38f : a;
    }
}

// The gradient of the state before each piece but a sequence's first, from the piece's own outputs, and the sum of
// its dt.
template<typename Scalar, int NR>
__global__ __launch_bounds__(kThreads) void scan_backs_kernel(const ScanJob job, const ScanGrads grads) {
    using Tile = BackTile<Scalar, NR>;
    __shared__ __align__(16) float lds[kWaves][2][Tile::kFloats];
    const BackPlace at(job);
    TimePiece piece;
    if (!time_piece(job.seq, job.step, at.piece, piece) || piece.seq < 0 || piece.at == 0 || piece.len == 0)
        return;
    const int lane = static_cast<int>(threadIdx.x) % kWave, sub = at.sub, n0 = sub * NR;
    float(*tile)[Tile::kFloats] = lds[threadIdx.x / kWave];
    float A2[NR], carry[NR];
    load_decays<NR>(A2, job, at.channel, n0);
#pragma unroll
    for (int j = 0; j < NR; ++j)
        carry[j] = 0.f;
    const float bias = job.bias ? job.bias[at.channel] : 0.f;
    double span = 0.0;
    Tile next;
    int t = (piece.len - 1) / kTile * kTile;
    next.load(job, grads, piece, at, t, lane, false);
    for (int turn = 0; t >= 0; t -= kTile, turn ^= 1) {
        float dv[kTile / 4], ds[kTile / 4];
#pragma unroll
        for (int g = 0; g < kTile / 4; ++g) {
            const bool live = t + 4 * g + sub < piece.len;
            const float raw = bits_f32<Scalar>(next.dt[g]) + bias, z = bits_f32<Scalar>(next.gate[g]);
            float e;
            dv[g] = live ? (job.softplus ? softplus(raw, e) : raw) : 0.f;
            ds[g] = bits_f32<Scalar>(next.dy[g]) * (job.gate ? z * sigmoid(z) : 1.f);
            ds[g] = live ? ds[g] : 0.f;
            span += static_cast<double>(dv[g]);
        }
        next.store_groups(tile[turn], lane);
        wave_sync();
        if (t > 0)
            next.load(job, grads, piece, at, t - kTile, lane, false);
#pragma unroll
        for (int g = kTile / 4 - 1; g >= 0; --g) {
            auto token = [&](auto k_) {
                constexpr int k = decltype(k_)::value;
                const float d = quad_lane<k>(dv[g]), s = quad_lane<k>(ds[g]);
                const float *c = tile[turn] + (4 * g + k) * Tile::kRow + 4 * NR + n0;
#pragma unroll
                for (int j = 0; j < NR; ++j)
                    carry[j] = __builtin_amdgcn_exp2f(d * A2[j]) * fmaf(c[j], s, carry[j]);
            };
            token(std::integral_constant<int, 3>{});
            token(std::integral_constant<int, 2>{});
            token(std::integral_constant<int, 1>{});
            token(std::integral_constant<int, 0>{});
        }
    }
    span += __shfl_xor(span, 1);
    span += __shfl_xor(span, 2);
    if (at.valid) {
        store_states<NR>(grads.backs + (static_cast<int64_t>(at.piece) * job.D + at.channel) * 4 * NR + n0, carry, NR);
        if (sub == 0)
            job.spans[static_cast<int64_t>(at.piece) * job.D + at.channel] = span;
    }
}

template<typename Scalar, int NR>
__global__ __launch_bounds__(kThreads) void scan_backward_kernel(const ScanJob job, const ScanGrads grads) {
    using Tile = BackTile<Scalar, NR>;
    // Tokens whose decays fit the registers; a tile is walked in so many parts.
    constexpr int kPart = NR <= 4 ? kTile : 4 * kTile / NR, kParts = kTile / kPart;
    __shared__ __align__(16) float lds[kWaves][Tile::kFloats], out[kWaves][Tile::kFloats];
    const BackPlace at(job);
    TimePiece piece;
    if (!time_piece(job.seq, job.step, at.piece, piece))
        return;
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave, wave = tid / kWave, sub = at.sub, n0 = sub * NR;
    const int channel = at.channel, D = job.D;
    const int64_t wide = static_cast<int64_t>(D) * 4 * NR, mine = static_cast<int64_t>(channel) * 4 * NR + n0;
    const int64_t row = static_cast<int64_t>(piece.row) * job.seq.T + piece.t0;
    Scalar *dx = static_cast<Scalar *>(grads.dx) + row * D + channel;
    Scalar *ddt = static_cast<Scalar *>(grads.ddt) + row * D + channel;
    Scalar *dgate = job.gate ? static_cast<Scalar *>(grads.dgate) + row * D + channel : nullptr;
    const int64_t tokens = static_cast<int64_t>(job.seq.B) * job.seq.T;
    float *groups = grads.groups + ((at.block * tokens + row) * job.G + at.group) * Tile::kRow;
    float dA[NR], dskip = 0.f, dbias = 0.f;
#pragma unroll
    for (int j = 0; j < NR; ++j)
        dA[j] = 0.f;
    if (piece.seq >= 0 && piece.at < piece.count) {
        float A2[NR], carry[NR], h[NR], h_next[NR];
        load_decays<NR>(A2, job, channel, n0);
#pragma unroll
        for (int j = 0; j < NR; ++j)
            carry[j] = 0.f;
        const int64_t state = (static_cast<int64_t>(piece.seq) * D + channel) * job.S + n0;
        if (grads.dstate)
            load_states<NR>(carry, grads.dstate + state, job.S - n0);
        for (int k = piece.count - 1; k > piece.at; --k) {
            const int64_t p = at.piece - piece.at + k;
            float back[NR];
            load_states<NR>(back, grads.backs + p * wide + mine, NR);
            const double span = job.spans[p * D + channel];
#pragma unroll
            for (int j = 0; j < NR; ++j)
                carry[j] = fmaf(__builtin_amdgcn_exp2f(static_cast<float>(A2[j] * span)), carry[j], back[j]);
        }
        const float bias = job.bias ? job.bias[channel] : 0.f, skip = job.skip ? job.skip[channel] : 0.f;
        const float *kept = job.kept + (scan_slot(job.seq, piece.seq, piece.lo) + (piece.t0 - piece.lo) / kScanKept) * wide + mine;
        Tile next;
        int t = (piece.len - 1) / kTile * kTile;
        if (piece.len > 0) {
            next.load(job, grads, piece, at, t, lane, true);
            load_states<NR>(h_next, kept + t / kTile * wide, NR);
        }
        for (; piece.len > 0 && t >= 0; t -= kTile) {
            float xv[kTile / 4], dv[kTile / 4], ev[kTile / 4], rv[kTile / 4], zv[kTile / 4], gv[kTile / 4], sv[kTile / 4];
#pragma unroll
            for (int g = 0; g < kTile / 4; ++g) {
                const bool live = t + 4 * g + sub < piece.len;
                const float raw = bits_f32<Scalar>(next.dt[g]) + bias;
                float e = 0.f;
                const float d = job.softplus ? softplus(raw, e) : raw;
                xv[g] = live ? bits_f32<Scalar>(next.x[g]) : 0.f;
                dv[g] = live ? d : 0.f, ev[g] = e, rv[g] = raw;
                zv[g] = bits_f32<Scalar>(next.gate[g]);
                gv[g] = live ? bits_f32<Scalar>(next.dy[g]) : 0.f;            // gradient of y
                sv[g] = job.gate ? gv[g] * zv[g] * sigmoid(zv[g]) : gv[g];    // of s
                sv[g] = live ? sv[g] : 0.f;
            }
#pragma unroll
            for (int j = 0; j < NR; ++j)
                h[j] = h_next[j];
            next.store_groups(lds[wave], lane);
            wave_sync();
            if (t > 0) {
                next.load(job, grads, piece, at, t - kTile, lane, true);
                load_states<NR>(h_next, kept + (t / kTile - 1) * wide, NR);
            }
            // the states before each part of the tile
            float from[kParts][NR];
#pragma unroll
            for (int part = 0; part < kParts; ++part) {
#pragma unroll
                for (int j = 0; j < NR; ++j)
                    from[part][j] = h[j];
                if (part + 1 < kParts) {
#pragma unroll
                    for (int g = part * kPart / 4; g < (part + 1) * kPart / 4; ++g) {
                        const float ux = dv[g] * xv[g];
                        auto token = [&](auto k_) {
                            constexpr int k = decltype(k_)::value;
                            const float d = quad_lane<k>(dv[g]), u = quad_lane<k>(ux);
                            const float *b = lds[wave] + (4 * g + k) * Tile::kRow + n0;
#pragma unroll
                            for (int j = 0; j < NR; ++j)
                                h[j] = fmaf(__builtin_amdgcn_exp2f(d * A2[j]), h[j], u * b[j]);
                        };
                        token(std::integral_constant<int, 0>{});
                        token(std::integral_constant<int, 1>{});
                        token(std::integral_constant<int, 2>{});
                        token(std::integral_constant<int, 3>{});
                    }
                }
            }
#pragma unroll
            for (int part = kParts - 1; part >= 0; --part) {
                float a[kPart][NR], ah[kPart][NR], ys[kPart / 4];
#pragma unroll
                for (int j = 0; j < NR; ++j)
                    h[j] = from[part][j];
#pragma unroll
                for (int i = 0; i < kPart / 4; ++i) {
                    const int g = part * kPart / 4 + i;
                    const float ux = dv[g] * xv[g];
                    float sums[4];
                    auto token = [&](auto k_) {
                        constexpr int k = decltype(k_)::value;
                        const float d = quad_lane<k>(dv[g]), u = quad_lane<k>(ux);
                        const float *b = lds[wave] + (4 * g + k) * Tile::kRow + n0, *c = b + 4 * NR;
                        sums[k] = 0.f;
#pragma unroll
                        for (int j = 0; j < NR; ++j) {
                            a[4 * i + k][j] = __builtin_amdgcn_exp2f(d * A2[j]);
                            ah[4 * i + k][j] = a[4 * i + k][j] * h[j];
                            h[j] = fmaf(u, b[j], ah[4 * i + k][j]);
                            sums[k] = fmaf(c[j], h[j], sums[k]);
                        }
                    };
                    token(std::integral_constant<int, 0>{});
                    token(std::integral_constant<int, 1>{});
                    token(std::integral_constant<int, 2>{});
                    token(std::integral_constant<int, 3>{});
                    ys[i] = quad_sums(sums, sub);
                }
                float sums[16] = {};  // of dB and dC, as many tokens of a group as it holds
#pragma unroll
                for (int i = kPart / 4 - 1; i >= 0; --i) {
                    const int g = part * kPart / 4 + i;
                    const float ux = dv[g] * xv[g];
                    float dus[4], das[4];
                    auto token = [&](auto k_) {
                        constexpr int k = decltype(k_)::value;
                        const float d = quad_lane<k>(dv[g]), u = quad_lane<k>(ux), s = quad_lane<k>(sv[g]);
                        const float *b = lds[wave] + (4 * g + k) * Tile::kRow + n0, *c = b + 4 * NR;
                        constexpr int kFill = NR == 1 ? 4 : NR <= 8 ? 8 / NR : 1;
                        constexpr int place = k % kFill * 2 * NR;
                        dus[k] = 0.f, das[k] = 0.f;
                        float db[NR], dc[NR];
#pragma unroll
                        for (int j = 0; j < NR; ++j) {
                            const float kept_h = ah[4 * i + k][j];
                            dc[j] = s * fmaf(u, b[j], kept_h);
                            const float G = fmaf(c[j], s, carry[j]);
                            db[j] = u * G;
                            dus[k] = fmaf(b[j], G, dus[k]);
                            const float through = G * kept_h;
                            das[k] = fmaf(through, A2[j], das[k]);
                            dA[j] = fmaf(through, d, dA[j]);
                            carry[j] = G * a[4 * i + k][j];
                        }
                        if constexpr (NR <= 8) {
                            // (lanes of channels that are not there hold copies of another's)
#pragma unroll
                            for (int j = 0; j < NR; ++j)
                                sums[place + j] = at.valid ? db[j] : 0.f, sums[place + NR + j] = at.valid ? dc[j] : 0.f;
                            if constexpr (k % kFill == 0) {
                                const float v = channel_sums(sums, lane);
                                const int q = lane / 4, which = q % (2 * NR) / NR, j = q % NR;
                                if (q < kFill * 2 * NR)
                                    out[wave][(4 * g + k + q / (2 * NR)) * Tile::kRow + which * 4 * NR + n0 + j] = v;
                            }
                        } else {
#pragma unroll
                            for (int which = 0; which < 2; ++which) {
#pragma unroll
                                for (int j = 0; j < NR; ++j)
                                    sums[j] = at.valid ? (which ? dc[j] : db[j]) : 0.f;
                                out[wave][(4 * g + k) * Tile::kRow + which * 4 * NR + n0 + lane / 4] = channel_sums(sums, lane);
                            }
                        }
                    };
                    token(std::integral_constant<int, 3>{});
                    token(std::integral_constant<int, 2>{});
                    token(std::integral_constant<int, 1>{});
                    token(std::integral_constant<int, 0>{});
                    const float du = quad_sums(dus, sub), da = quad_sums(das, sub) * kLn2;
                    float draw = fmaf(xv[g], du, da);
                    if (job.softplus) {
                        const float inv = __builtin_amdgcn_rcpf(1.f + ev[g]);
                        draw *= rv[g] >= 0.f ? inv : ev[g] * inv;
                    }
                    const int token_at = t + 4 * g + sub;
                    if (token_at < piece.len) {
                        dskip = fmaf(sv[g], xv[g], dskip);
                        dbias += draw;
                        const int64_t where = static_cast<int64_t>(token_at) * D;
                        if (at.valid) {
                            store_vec<Scalar, 1>(dx + where, {{round_bits<Scalar>(fmaf(dv[g], du, skip * sv[g]))}});
                            store_vec<Scalar, 1>(ddt + where, {{round_bits<Scalar>(draw)}});
                            if (dgate) {
                                const float sig = sigmoid(zv[g]), y = fmaf(skip, xv[g], ys[i]);
                                store_vec<Scalar, 1>(dgate + where, {{round_bits<Scalar>(
                                                                        gv[g] * y * sig * (1.f + zv[g] * (1.f - sig)))}});
                            }
                        }
                    }
                }
            }
            // dB and dC over the block's channels
            __syncthreads();
            for (int i = tid; i < Tile::kFloats; i += kThreads) {
                const int token_at = t + i / Tile::kRow;
                float sum = 0.f;
#pragma unroll
                for (int w = 0; w < kWaves; ++w)
                    sum += out[w][i];
                if (token_at < piece.len)
                    groups[static_cast<int64_t>(token_at) * job.G * Tile::kRow + i % Tile::kRow] = sum;
            }
            __syncthreads();
        }
        if (piece.at == 0 && grads.dinit && at.valid)
            store_states<NR>(grads.dinit + state, carry, job.S - n0);
    }
    for (int i = sub; i < piece.rest; i += 4) {
        const int64_t where = static_cast<int64_t>(piece.len + i) * D;
        if (at.valid) {
            store_vec<Scalar, 1>(dx + where, {{0u}});
            store_vec<Scalar, 1>(ddt + where, {{0u}});
            if (dgate)
                store_vec<Scalar, 1>(dgate + where, {{0u}});
        }
    }
    for (int i = tid; i < piece.rest * Tile::kRow; i += kThreads)
        groups[static_cast<int64_t>(piece.len + i / Tile::kRow) * job.G * Tile::kRow + i % Tile::kRow] = 0.f;
    dskip += quad_swap<1>(dskip), dbias += quad_swap<1>(dbias);
    dskip += quad_swap<2>(dskip), dbias += quad_swap<2>(dbias);
    if (at.valid) {
        float *to = grads.sums + (static_cast<int64_t>(at.piece) * D + channel) * (4 * NR + 2);
        store_states<NR>(to + n0, dA, NR);
        if (sub == 0)
            to[4 * NR] = dskip, to[4 * NR + 1] = dbias;
    }
}

// dB and dC: a thread adds up one value over the channel blocks of its group, in order.
template<typename Scalar>
__global__ __launch_bounds__(kThreads) void scan_groups_kernel(const ScanJob job, const ScanGrads grads, int blocks, int row) {
    const int64_t rows = static_cast<int64_t>(job.seq.B) * job.seq.T * job.G;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    if (i >= rows * row)
        return;
    float sum = 0.f;
    for (int b = 0; b < blocks; ++b)
        sum += grads.groups[b * rows * row + i];
    const int64_t at = i / row;
    const int e = static_cast<int>(i - at * row), which = e / (row / 2), n = e % (row / 2);
    if (n < job.S)
        store_f32(static_cast<Scalar *>(which ? grads.dC : grads.dB) + at * job.S + n, sum);
}

// dA, dskip and dbias: likewise over the pieces (fewer where packed sequences have fewer).
__global__ __launch_bounds__(1024) void scan_sums_kernel(const ScanJob job, const ScanGrads grads, int64_t pieces, int row) {
    __shared__ float sums[16][kWave];
    const int lane = static_cast<int>(threadIdx.x) % kWave, wave = static_cast<int>(threadIdx.x) / kWave;
    const int64_t columns = static_cast<int64_t>(job.D) * row, column = static_cast<int64_t>(blockIdx.x) * kWave + lane;
    TimePiece piece;
    float sum = 0.f;
    if (column < columns)
        for (int64_t p = wave; p < pieces; p += 16)
            if (!job.seq.cu || p < job.seq.first[job.seq.N])
                sum += grads.sums[p * columns + column];
    sums[wave][lane] = sum;
    __syncthreads();
    if (wave > 0 || column >= columns)
        return;
    for (int w = 1; w < 16; ++w)
        sum += sums[w][lane];
    const int64_t d = column / row;
    const int e = static_cast<int>(column - d * row);
    if (e < job.S)
        grads.dA[d * job.S + e] = sum;
    else if (e == row - 2 && grads.dskip)
        grads.dskip[d] = sum;
    else if (e == row - 1 && grads.dbias)
        grads.dbias[d] = sum;
}

template<typename Scalar, int NR>
hipError_t launch_states(const ScanJob &job, const ScanGrads &grads, hipStream_t stream) {
    const int64_t pieces = most_pieces(job.seq, job.step);
    const int blocks = (job.D / job.G + kChannels - 1) / kChannels;
    const dim3 grid(static_cast<unsigned>(pieces * job.G * blocks)), block(kThreads);
    if (job.seq.T > job.step)
        hipLaunchKernelGGL((scan_backs_kernel<Scalar, NR>), grid, block, 0, stream, job, grads);
    hipLaunchKernelGGL((scan_backward_kernel<Scalar, NR>), grid, block, 0, stream, job, grads);
    const int64_t values = static_cast<int64_t>(job.seq.B) * job.seq.T * job.G * 8 * NR;
    hipLaunchKernelGGL(scan_groups_kernel<Scalar>, dim3(static_cast<unsigned>((values + kThreads - 1) / kThreads)), block, 0,
                       stream, job, grads, blocks, 8 * NR);
    const int row = 4 * NR + 2;
    const int64_t columns = static_cast<int64_t>(job.D) * row;
    hipLaunchKernelGGL(scan_sums_kernel, dim3(static_cast<unsigned>((columns + kWave - 1) / kWave)), dim3(1024), 0, stream,
                       job, grads, pieces, row);
    return hipGetLastError();
}

template<typename Scalar>
hipError_t launch_type(const ScanJob &job, const ScanGrads &grads, hipStream_t stream) {
    switch (scan_lane_states(job.S)) {
        case 1: return launch_states<Scalar, 1>(job, grads, stream);
        case 2: return launch_states<Scalar, 2>(job, grads, stream);
        case 4: return launch_states<Scalar, 4>(job, grads, stream);
        case 8: return launch_states<Scalar, 8>(job, grads, stream);
        default: return launch_states<Scalar, 16>(job, grads, stream);
    }
}

}  // namespace

hipError_t launch_scan_backward(const ScanJob &job, const ScanGrads &grads, hipStream_t stream, const char **why) {
    if (job.seq.cu) {
        const hipError_t err = launch_sequences(job.seq, job.step, stream);
        if (err != hipSuccess)
            return err;
    }
    switch (job.dtype) {
        case kF32: return launch_type<float>(job, grads, stream);
        case kF16: return launch_type<_Float16>(job, grads, stream);
        case kBF16: return launch_type<bf16_t>(job, grads, stream);
        default: *why = "selective_scan: unsupported dtype"; return hipErrorInvalidValue;
    }
}

}  // namespace ramnet
