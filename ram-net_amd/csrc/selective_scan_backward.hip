// Selective scan, gradients. With G_t the gradient of the state after token t,
//
//     G_t = C_t ds_t + a_{t+1} G_{t+1},   a_t = e^(dt_t A)
//     dC_t = ds_t h_t,   dB_t = dt_t x_t G_t          (both summed over a group's channels)
//     d(dt x)_t = B_t . G_t,   d(dt_t) = x_t d(dt x)_t + sum_n A G_t a_t h_{t-1},   dA = sum_t dt_t G_t a_t h_{t-1}
//
// The states are walked again from those kept every 16 tokens; a_t and a_t h_{t-1} of a part of the tile stay in
// registers for the way back. Pieces are joined as in the forward, from the last to the first.
//
// Bound by vector instructions, 113 a token and wave with 16 states, 20 of them for the sums of dB and dC over a wave's
// channels: 4 x 2048 x 2048, gated, bf16: 280 us, 87% of the time issuing (bytes: 48 us), the pieces' ends 75, the sums 20.
// Sums over channels and tokens go through memory in one order: results do not change from call to call.
#include "ramnet_kernels.hpp"
#include "selective_scan.hpp"

#include <algorithm>

namespace ramnet {

namespace {

constexpr int kThreads = kScanThreads, kWaves = kThreads / kWave, kTile = kScanKept, kQuads = kTile / 4;

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
    using Groups = ScanGroups<Scalar, NR>;
    __shared__ __align__(16) float lds[kWaves][2][Groups::kFloats];
    const ScanPlace at(job);
    TimePiece piece;
    if (!time_piece(job.seq, job.step, at.piece, piece) || piece.seq < 0 || piece.at == 0 || piece.len == 0)
        return;
    const int lane = static_cast<int>(threadIdx.x) % kWave, sub = at.sub, n0 = sub * NR;
    float(*tile)[Groups::kFloats] = lds[threadIdx.x / kWave];
    float A2[NR], carry[NR];
    load_decays<NR>(A2, job, at.channel, n0);
#pragma unroll
    for (int j = 0; j < NR; ++j)
        carry[j] = 0.f;
    const float bias = job.bias ? job.bias[at.channel] : 0.f;
    double span = 0.0;
    int t = (piece.len - 1) / kTile * kTile;
    const int64_t token = piece.t0 + t, first_row = piece.row;
    ScanCursor<Scalar, -1> dt_at(job.dt, first_row * job.dt_at[0] + token * job.dt_at[1], job.dt_at[1], job.D),
        gate_at(job.gate, first_row * job.gate_at[0] + token * job.gate_at[1], job.gate_at[1], job.D),
        dy_at(grads.dy, first_row * grads.dy_at[0] + token * grads.dy_at[1], grads.dy_at[1], job.D),
        C_at(job.C, first_row * job.C_at[0] + at.group * job.C_at[2] + token * job.C_at[1], job.C_at[1], job.S);
    const ScanRows<Scalar> dt_rows(at, job.dt_at[1], true), gate_rows(at, job.gate_at[1], true), dy_rows(at, grads.dy_at[1], true);
    const Groups C_rows(lane, job.C_at[1], job.S);
    uint32_t dts[kQuads], gates[kQuads], dys[kQuads], Cs[Groups::kLoads];
    auto load = [&](int t) {
        const int left = piece.len - t;
        dt_rows.load(dts, dt_at.next(left));
        dy_rows.load(dys, dy_at.next(left));
        if (job.gate)
            gate_rows.load(gates, gate_at.next(left));
        C_rows.load(Cs, C_at.next(left));
    };
    load(t);
    for (int turn = 0; t >= 0; t -= kTile, turn ^= 1) {
        float dv[kQuads], sv[kQuads];
#pragma unroll
        for (int g = 0; g < kQuads; ++g) {
            dv[g] = bits_f32<Scalar>(dts[g]) + bias, sv[g] = bits_f32<Scalar>(dys[g]);
            if (job.softplus) {
                float e;
                dv[g] = softplus(dv[g], e);
            }
            if (job.gate) {
                const float z = bits_f32<Scalar>(gates[g]);
                sv[g] *= z * sigmoid(z);
            }
            const bool live = t + 4 * g + sub < piece.len;  // (rows may lie on each other: what is past the end may be read)
            dv[g] = live ? dv[g] : 0.f, sv[g] = live ? sv[g] : 0.f;
            span += static_cast<double>(dv[g]);
        }
        C_rows.store(tile[turn], Cs);
        wave_sync();
        if (t > 0)
            load(t - kTile);
        float c[2][4][NR];
        auto fetch = [&](int g) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int j = 0; j < NR; ++j)
                    c[g & 1][k][j] = tile[turn][(4 * g + k) * Groups::kRow + n0 + j];
        };
        fetch(kQuads - 1);
#pragma unroll
        for (int g = kQuads - 1; g >= 0; --g) {
            if (g > 0)
                fetch(g - 1);
            __builtin_amdgcn_sched_barrier(0);
            auto token = [&](auto k_) {
                constexpr int k = decltype(k_)::value;
                const float d = quad_lane<k>(dv[g]), s = quad_lane<k>(sv[g]);
#pragma unroll
                for (int j = 0; j < NR; ++j)
                    carry[j] = __builtin_amdgcn_exp2f(d * A2[j]) * fmaf(c[g & 1][k][j], s, carry[j]);
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

// What is read from LDS before is not kept in registers for after: B and C of a whole tile would fill them.
__device__ __forceinline__ void reread() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// Tokens whose decays fit the registers beside the rest: a tile is walked in parts of so many, and but for the last
// one twice. (16 states, 4 x 2048 x 2048 channels: parts of 16 spill, 545 us; of 8 283, of 4 280.)
template<int NR>
constexpr int scan_part() { return NR <= 2 ? kTile : NR <= 4 ? kTile / 2 : kTile / 4; }

// Waves a SIMD, and by that registers: 256 a lane spill from 24 states on (4 x 2048 x 2048 channels; 24 states 744 us
// with two waves, 779 with one; 32 states 979 and 784; 48 states 3004 and 1310; of 64 the LDS holds one block anyway).
template<int NR>
constexpr int scan_waves() { return NR >= 8 ? 1 : 2; }

template<typename Scalar, int NR, bool kGate>
__global__ __launch_bounds__(kThreads, scan_waves<NR>()) void scan_backward_kernel(const ScanJob job, const ScanGrads grads) {
    using Groups = ScanGroups<Scalar, NR>;
    constexpr int kPart = scan_part<NR>(), kParts = kTile / kPart, kRow = Groups::kRow, kFloats = Groups::kFloats;
    constexpr int kSpread = 2 * kRow;  // dB and dC of a token
    __shared__ __align__(16) float lds[kWaves][2 * kFloats], out[2][kWaves][2 * kFloats];
    const ScanPlace at(job);
    TimePiece piece;
    if (!time_piece(job.seq, job.step, at.piece, piece))
        return;
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave, sub = at.sub, n0 = sub * NR;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int channel = at.channel, D = job.D;
    const int64_t wide = static_cast<int64_t>(D) * kRow, mine = static_cast<int64_t>(channel) * kRow + n0;
    const int64_t row = static_cast<int64_t>(piece.row) * job.seq.T + piece.t0;
    const int64_t tokens = static_cast<int64_t>(job.seq.B) * job.seq.T;
    float *groups = grads.groups + ((at.block * tokens + row) * job.G + at.group) * kSpread;
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
        // (windows are made from the job for each tile: kept from one to the next they spill scalar registers, for the same time)
        auto rows_at = [&](const void *p, int64_t from, int64_t stride, int width, int left) {
            return window(static_cast<const Scalar *>(p) + from,
                          ((min(left, kTile) - 1) * stride + width) * static_cast<int>(sizeof(Scalar)));
        };
        const int64_t token = piece.t0, xr = piece.row * job.x_at[0], dr = piece.row * job.dt_at[0],
                      gr = piece.row * job.gate_at[0], yr = piece.row * grads.dy_at[0],
                      Br = piece.row * job.B_at[0] + at.group * job.B_at[2], Cr = piece.row * job.C_at[0] + at.group * job.C_at[2];
        // (lanes without a channel read zeros, and so add nothing to the sums over channels)
        const ScanRows<Scalar> x_rows(at, job.x_at[1], at.valid), dt_rows(at, job.dt_at[1], at.valid),
            gate_rows(at, job.gate_at[1], at.valid), dy_rows(at, grads.dy_at[1], at.valid), d_rows(at, D, at.valid);
        const Groups B_rows(lane, job.B_at[1], job.S), C_rows(lane, job.C_at[1], job.S);
        uint32_t xs[kQuads], dts[kQuads], gates[kQuads], dys[kQuads], Bs[Groups::kLoads], Cs[Groups::kLoads];
        auto load = [&](int t) {
            const int left = piece.len - t;
            dt_rows.template load<true>(dts, rows_at(job.dt, dr + (token + t) * job.dt_at[1], job.dt_at[1], D, left));
            x_rows.template load<true>(xs, rows_at(job.x, xr + (token + t) * job.x_at[1], job.x_at[1], D, left));
            dy_rows.template load<true>(dys, rows_at(grads.dy, yr + (token + t) * grads.dy_at[1], grads.dy_at[1], D, left));
            if constexpr (kGate)
                gate_rows.template load<true>(gates, rows_at(job.gate, gr + (token + t) * job.gate_at[1], job.gate_at[1], D, left));
            B_rows.template load<true>(Bs, rows_at(job.B, Br + (token + t) * job.B_at[1], job.B_at[1], job.S, left));
            C_rows.template load<true>(Cs, rows_at(job.C, Cr + (token + t) * job.C_at[1], job.C_at[1], job.S, left));
            load_states<NR>(h_next, kept + t / kTile * wide, NR);
        };
        int t = (piece.len - 1) / kTile * kTile;
        if (piece.len > 0)
            load(t);
        for (int turn = 0; piece.len > 0 && t >= 0; t -= kTile, turn ^= 1) {
            float xv[kQuads], dv[kQuads], ev[kQuads], rv[kQuads], zv[kQuads], gv[kQuads], sv[kQuads];
#pragma unroll
            for (int g = 0; g < kQuads; ++g) {
                const bool live = t + 4 * g + sub < piece.len;
                rv[g] = bits_f32<Scalar>(dts[g]) + bias, ev[g] = 0.f;
                const float d = job.softplus ? softplus(rv[g], ev[g]) : rv[g];
                dv[g] = live ? d : 0.f;
                xv[g] = live ? bits_f32<Scalar>(xs[g]) : 0.f;
                gv[g] = live ? bits_f32<Scalar>(dys[g]) : 0.f;  // gradient of y
                sv[g] = gv[g];                                  // of s
                if constexpr (kGate) {
                    zv[g] = bits_f32<Scalar>(gates[g]);
                    sv[g] = live ? gv[g] * zv[g] * sigmoid(zv[g]) : 0.f;
                }
            }
#pragma unroll
            for (int j = 0; j < NR; ++j)
                h[j] = h_next[j];
            B_rows.store(lds[wave], Bs);
            C_rows.store(lds[wave] + kFloats, Cs);
            wave_sync();
            if (t > 0)
                load(t - kTile);
            const int left = piece.len - t;
            const int64_t first = (row + t) * D;
            const auto dx_rows = rows_at(grads.dx, first, D, D, left), ddt_rows = rows_at(grads.ddt, first, D, D, left);
            const auto dgate_rows = rows_at(kGate ? grads.dgate : grads.dx, first, D, D, left);
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
                        reread();
                        const float ux = dv[g] * xv[g];
                        auto token = [&](auto k_) {
                            constexpr int k = decltype(k_)::value;
                            const float d = quad_lane<k>(dv[g]), u = quad_lane<k>(ux);
                            const float *b = lds[wave] + (4 * g + k) * kRow + n0;
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
#pragma unroll
                for (int j = 0; j < NR; ++j)  // (nor are the decays of the parts to come)
                    asm volatile("" : "+v"(A2[j]));
                float a[kPart][NR], ah[kPart][NR], ys[kPart / 4];
#pragma unroll
                for (int j = 0; j < NR; ++j)
                    h[j] = from[part][j];
#pragma unroll
                for (int i = 0; i < kPart / 4; ++i) {
                    reread();
                    const int g = part * kPart / 4 + i;
                    const float ux = dv[g] * xv[g];
                    float sums[4];
                    auto token = [&](auto k_) {
                        constexpr int k = decltype(k_)::value;
                        const float d = quad_lane<k>(dv[g]), u = quad_lane<k>(ux);
                        const float *b = lds[wave] + (4 * g + k) * kRow + n0, *c = b + kFloats;
                        sums[k] = 0.f;
#pragma unroll
                        for (int j = 0; j < NR; ++j) {
                            a[4 * i + k][j] = __builtin_amdgcn_exp2f(d * A2[j]);
                            ah[4 * i + k][j] = a[4 * i + k][j] * h[j];
                            h[j] = fmaf(u, b[j], ah[4 * i + k][j]);
                            if constexpr (kGate)
                                sums[k] = j ? fmaf(c[j], h[j], sums[k]) : c[j] * h[j];
                        }
                    };
                    token(std::integral_constant<int, 0>{});
                    token(std::integral_constant<int, 1>{});
                    token(std::integral_constant<int, 2>{});
                    token(std::integral_constant<int, 3>{});
                    if constexpr (kGate)
                        ys[i] = quad_sums(sums, sub);
                }
                float sums[16] = {};  // of dB and dC, as many tokens of a group as it holds
#pragma unroll
                for (int i = kPart / 4 - 1; i >= 0; --i) {
                    reread();
                    const int g = part * kPart / 4 + i;
                    const float ux = dv[g] * xv[g];
                    float dus[4], das[4];
                    auto token = [&](auto k_) {
                        constexpr int k = decltype(k_)::value;
                        const float d = quad_lane<k>(dv[g]), u = quad_lane<k>(ux), s = quad_lane<k>(sv[g]);
                        const float *b = lds[wave] + (4 * g + k) * kRow + n0, *c = b + kFloats;
                        constexpr int kFill = NR <= 2 ? 4 : NR <= 4 ? 2 : 1;
                        constexpr int place = k % kFill * 2 * NR;
                        if constexpr (NR > 4)
                            reread();
                        float db[NR], dc[NR];
#pragma unroll
                        for (int j = 0; j < NR; ++j) {
                            const float kept_h = ah[4 * i + k][j];
                            dc[j] = s * fmaf(u, b[j], kept_h);
                            const float G = fmaf(c[j], s, carry[j]);
                            db[j] = u * G;
                            const float through = G * kept_h;
                            dus[k] = j ? fmaf(b[j], G, dus[k]) : b[j] * G;
                            das[k] = j ? fmaf(through, A2[j], das[k]) : through * A2[j];
                            dA[j] = fmaf(through, d, dA[j]);
                            carry[j] = G * a[4 * i + k][j];
                        }
                        if constexpr (NR <= 8) {
#pragma unroll
                            for (int j = 0; j < NR; ++j)
                                sums[place + j] = db[j], sums[place + NR + j] = dc[j];
                            if constexpr (k % kFill == 0) {
                                const float v = channel_sums(sums, lane);
                                const int q = lane / 4, which = q % (2 * NR) / NR, j = q % NR;
                                if (kFill * 2 * NR == 16 || q < kFill * 2 * NR)
                                    out[turn][wave][(4 * g + k + q / (2 * NR)) * kSpread + which * kRow + n0 + j] = v;
                            }
                        } else {
#pragma unroll
                            for (int which = 0; which < 2; ++which) {
#pragma unroll
                                for (int j = 0; j < NR; ++j)
                                    sums[j] = which ? dc[j] : db[j];
                                const float v = channel_sums(sums, lane);
                                if (NR == 16 || lane / 4 < NR)
                                    out[turn][wave][(4 * g + k) * kSpread + which * kRow + n0 + lane / 4] = v;
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
                    draw = t + 4 * g + sub < piece.len ? draw : 0.f;
                    dskip = fmaf(sv[g], xv[g], dskip);
                    dbias += draw;
                    const int where = anew(d_rows.at) + g * d_rows.step;
                    buffer_store<Scalar>(fmaf(dv[g], du, skip * sv[g]), dx_rows, where);
                    buffer_store<Scalar>(draw, ddt_rows, where);
                    if constexpr (kGate) {
                        const float sig = sigmoid(zv[g]), y = fmaf(skip, xv[g], ys[i]);
                        buffer_store<Scalar>(gv[g] * y * sig * (1.f + zv[g] * (1.f - sig)), dgate_rows, where);
                    }
                }
            }
            // dB and dC over the block's channels; the next tile's are put beside them
            __syncthreads();
            for (int i = tid; i < 2 * kFloats; i += kThreads) {
                const int token_at = t + i / kSpread;
                float sum = 0.f;
#pragma unroll
                for (int w = 0; w < kWaves; ++w)
                    sum += out[turn][w][i];
                if (token_at < piece.len)
                    groups[static_cast<int64_t>(token_at) * job.G * kSpread + i % kSpread] = sum;
            }
        }
        if (piece.at == 0 && grads.dinit && at.valid)
            store_states<NR>(grads.dinit + state, carry, job.S - n0);
    }
    for (int i = sub; i < piece.rest; i += 4) {
        const int64_t where = (row + piece.len + i) * D + channel;
        if (at.valid) {
            store_vec<Scalar, 1>(static_cast<Scalar *>(grads.dx) + where, {{0u}});
            store_vec<Scalar, 1>(static_cast<Scalar *>(grads.ddt) + where, {{0u}});
            if (kGate)
                store_vec<Scalar, 1>(static_cast<Scalar *>(grads.dgate) + where, {{0u}});
        }
    }
    for (int i = tid; i < piece.rest * kSpread; i += kThreads)
        groups[static_cast<int64_t>(piece.len + i / kSpread) * job.G * kSpread + i % kSpread] = 0.f;
    dskip += quad_swap<1>(dskip), dbias += quad_swap<1>(dbias);
    dskip += quad_swap<2>(dskip), dbias += quad_swap<2>(dbias);
    if (at.valid) {
        float *to = grads.sums + (static_cast<int64_t>(at.piece) * D + channel) * (kRow + 2);
        store_states<NR>(to + n0, dA, NR);
        if (sub == 0)
            to[kRow] = dskip, to[kRow + 1] = dbias;
    }
}

// dB and dC: a thread adds up one value over the channel blocks of its group, in order.
template<typename Scalar>
__global__ __launch_bounds__(kThreads) void scan_groups_kernel(const ScanJob job, const ScanGrads grads, int blocks, int row) {
    const int64_t rows = static_cast<int64_t>(job.seq.B) * job.seq.T * job.G;
    const int64_t threads = static_cast<int64_t>(gridDim.x) * kThreads;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < rows * row; i += threads) {
        float sum = 0.f;
        for (int b = 0; b < blocks; ++b)
            sum += grads.groups[b * rows * row + i];
        const int64_t at = i / row;
        const int e = static_cast<int>(i - at * row), which = e / (row / 2), n = e % (row / 2);
        if (n < job.S)
            store_f32(static_cast<Scalar *>(which ? grads.dC : grads.dB) + at * job.S + n, sum);
    }
}

// dA, dskip and dbias: likewise over the pieces (fewer where packed sequences have fewer).
__global__ __launch_bounds__(1024) void scan_sums_kernel(const ScanJob job, const ScanGrads grads, int64_t pieces, int row) {
    __shared__ float sums[16][kWave];
    const int lane = static_cast<int>(threadIdx.x) % kWave, wave = static_cast<int>(threadIdx.x) / kWave;
    const int64_t columns = static_cast<int64_t>(job.D) * row, column = static_cast<int64_t>(blockIdx.x) * kWave + lane;
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
    const int blocks = (job.D / job.G + kScanChannels - 1) / kScanChannels;
    const dim3 grid(static_cast<unsigned>(pieces * job.G * blocks)), block(kThreads);
    if (job.seq.T > job.step)
        hipLaunchKernelGGL((scan_backs_kernel<Scalar, NR>), grid, block, 0, stream, job, grads);
    if (job.gate)
        hipLaunchKernelGGL((scan_backward_kernel<Scalar, NR, true>), grid, block, 0, stream, job, grads);
    else
        hipLaunchKernelGGL((scan_backward_kernel<Scalar, NR, false>), grid, block, 0, stream, job, grads);
    const int64_t values = static_cast<int64_t>(job.seq.B) * job.seq.T * job.G * 8 * NR;
    const int64_t value_blocks = std::min<int64_t>((values + kThreads - 1) / kThreads, 1 << 22);
    hipLaunchKernelGGL(scan_groups_kernel<Scalar>, dim3(static_cast<unsigned>(value_blocks)), block, 0, stream, job, grads,
                       blocks, 8 * NR);
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
        case 3: return launch_states<Scalar, 3>(job, grads, stream);
        case 4: return launch_states<Scalar, 4>(job, grads, stream);
        case 6: return launch_states<Scalar, 6>(job, grads, stream);
        case 8: return launch_states<Scalar, 8>(job, grads, stream);
        case 12: return launch_states<Scalar, 12>(job, grads, stream);
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
