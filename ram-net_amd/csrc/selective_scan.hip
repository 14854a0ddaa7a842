// Selective scan, forward: whole and packed prompts, decode steps, and what a training call keeps.
//
// Bound by vector instructions: every channel and state has a decay of its own, so no matrix product stands in for the
// recurrence. A token of 16 channels with 16 states is 20 of a wave for its states (two products, an exponential, which
// takes two's time, and two fused products each) and 11 around them. Pieces of a row are joined by linearity: with h_k
// the state after piece k from zeros and D_k the sum of its dt, the state before piece k + 1 is
// h_k + e^(A D_k) (the one before piece k). D_k is in 64 bits, as A D_k may be large where a decay ends.
// B and C of 16 tokens are in LDS for the wave that reads them (no barriers), the next 16 tokens' rows on their way.
//
// 8 x 4096 x 2048, 16 states, gated, bf16: 372 us (257 by its instructions, 109 by its bytes), one wave a SIMD, 69% of the
// time issuing. 1 x 32768 x 1024: 111 and 145, 90 to 95%. Decode, 64 rows x 2048: 8.0 us, 2048 rows: 126, 4.3 TB/s.
#include "ramnet_kernels.hpp"
#include "selective_scan.hpp"

#include <algorithm>
#include <cmath>

namespace ramnet {

namespace {

constexpr int kThreads = kScanThreads, kTile = kScanKept, kQuads = kTile / 4;

enum : int { kEnds, kWhole };

// kEnds: the state after each piece but a sequence's last, from zeros, and the sum of its dt.
// kWhole: y, and the state after the sequence.
template<typename Scalar, int NR, int kMode, bool kGate>
__global__ __launch_bounds__(kThreads) void scan_kernel(const ScanJob job) {
    using Groups = ScanGroups<Scalar, NR>;
    __shared__ __align__(16) float lds[kThreads / kWave][2][2 * Groups::kFloats];
    const ScanPlace at(job);
    TimePiece piece;
    if (!time_piece(job.seq, job.step, at.piece, piece))
        return;
    const int lane = static_cast<int>(threadIdx.x) % kWave, sub = at.sub, channel = at.channel, n0 = sub * NR;
    float(*tile)[2 * Groups::kFloats] = lds[threadIdx.x / kWave];
    const int count = job.S - n0;
    const int64_t wide = static_cast<int64_t>(job.D) * 4 * NR;  // floats of a workspace row
    const int64_t mine = static_cast<int64_t>(channel) * 4 * NR + n0;
    const int64_t row = static_cast<int64_t>(piece.row) * job.seq.T + piece.t0;
    Scalar *y = static_cast<Scalar *>(job.y) + row * job.D + channel;
    if (piece.seq >= 0 && piece.at < piece.count) {
        float h[NR], A2[NR];
        load_states<NR>(A2, job.A + static_cast<int64_t>(channel) * job.S + n0, count);
#pragma unroll
        for (int j = 0; j < NR; ++j)
            h[j] = 0.f, A2[j] *= kLog2e;
        const float *init = job.init ? job.init + (static_cast<int64_t>(piece.seq) * job.D + channel) * job.S + n0 : nullptr;
        if constexpr (kMode == kEnds) {
            if (piece.at == piece.count - 1) {
                // The sequence's state, for its first piece: the last one writes over it in place.
                if (piece.count > 1 && job.init && at.valid) {
                    load_states<NR>(h, init, count);
                    store_states<NR>(job.ends + at.piece * wide + mine, h, NR);
                }
                return;
            }
        } else {
            const int64_t first = at.piece - piece.at;
            if (job.init && piece.count == 1)
                load_states<NR>(h, init, count);
            else if (job.init)
                load_states<NR>(h, job.ends + (first + piece.count - 1) * wide + mine, NR);
            for (int k = 0; k < piece.at; ++k) {
                float end[NR];
                load_states<NR>(end, job.ends + (first + k) * wide + mine, NR);
                const double span = job.spans[(first + k) * job.D + channel];
#pragma unroll
                for (int j = 0; j < NR; ++j)
                    h[j] = fmaf(__builtin_amdgcn_exp2f(static_cast<float>(A2[j] * span)), h[j], end[j]);
            }
        }
        const float bias = job.bias ? job.bias[channel] : 0.f, skip = job.skip ? job.skip[channel] : 0.f;
        double span = 0.0;
        // Windows over the 16 tokens of a tile: tokens that are not there read 0 and are not written
        const int64_t token = piece.t0, first_row = piece.row;
        ScanCursor<Scalar> x_at(job.x, first_row * job.x_at[0] + token * job.x_at[1], job.x_at[1], job.D),
            dt_at(job.dt, first_row * job.dt_at[0] + token * job.dt_at[1], job.dt_at[1], job.D),
            gate_at(job.gate, first_row * job.gate_at[0] + token * job.gate_at[1], job.gate_at[1], job.D),
            B_at(job.B, first_row * job.B_at[0] + at.group * job.B_at[2] + token * job.B_at[1], job.B_at[1], job.S),
            C_at(job.C, first_row * job.C_at[0] + at.group * job.C_at[2] + token * job.C_at[1], job.C_at[1], job.S),
            y_at(job.y, row * job.D, job.D, job.D);
        const ScanRows<Scalar> x_rows(at, job.x_at[1], true), dt_rows(at, job.dt_at[1], true), gate_rows(at, job.gate_at[1], true),
            y_rows(at, job.D, at.valid);
        const Groups B_rows(lane, job.B_at[1], job.S), C_rows(lane, job.C_at[1], job.S);
        uint32_t xs[kQuads], ds[kQuads], gs[kQuads], Bs[Groups::kLoads], Cs[Groups::kLoads];
        auto load = [&](int t) {
            const int left = piece.len - t;
            dt_rows.load(ds, dt_at.next(left));
            x_rows.load(xs, x_at.next(left));
            B_rows.load(Bs, B_at.next(left));
            if constexpr (kMode == kWhole) {
                C_rows.load(Cs, C_at.next(left));
                if constexpr (kGate)
                    gate_rows.load(gs, gate_at.next(left));
            }
        };
        auto walk = [&](int t, const float *bc, auto whole) {
            float xv[kQuads], dv[kQuads], gv[kQuads];
#pragma unroll
            for (int g = 0; g < kQuads; ++g) {
                xv[g] = bits_f32<Scalar>(xs[g]), dv[g] = bits_f32<Scalar>(ds[g]) + bias;
                if constexpr (kGate && kMode == kWhole)
                    gv[g] = bits_f32<Scalar>(gs[g]);
            }
            if (job.softplus) {
                float e;
#pragma unroll
                for (int g = 0; g < kQuads; ++g)
                    dv[g] = softplus(dv[g], e);
            }
            load(t + kTile);  // (past the piece windows are empty: a branch would cost copies of all it may leave as it was)
            const __amdgpu_buffer_rsrc_t out = y_at.next(piece.len - t);
            // B and C of four tokens at a time, read from LDS while the four before are walked
            float b[2][4][NR], c[2][4][NR];
            auto fetch = [&](int g) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float *from = bc + (4 * g + k) * Groups::kRow + n0;
#pragma unroll
                    for (int j = 0; j < NR; ++j) {
                        b[g & 1][k][j] = from[j];
                        if constexpr (kMode == kWhole)
                            c[g & 1][k][j] = from[Groups::kFloats + j];
                    }
                }
            };
            fetch(0);
#pragma unroll
            for (int g = 0; g < kQuads; ++g) {
                if (g + 1 < kQuads)
                    fetch(g + 1);
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (kMode == kEnds)
                    span += decltype(whole)::value || t + 4 * g + sub < piece.len ? static_cast<double>(dv[g]) : 0.0;
                const float ux = dv[g] * xv[g];
                float sums[4];
                auto token = [&](auto k_) {
                    constexpr int k = decltype(k_)::value;
                    sums[k] = 0.f;
                    if (!decltype(whole)::value && t + 4 * g + k >= piece.len)
                        return;
                    const float d = quad_lane<k>(dv[g]), u = quad_lane<k>(ux);
#pragma unroll
                    for (int j = 0; j < NR; ++j) {
                        h[j] = fmaf(__builtin_amdgcn_exp2f(d * A2[j]), h[j], u * b[g & 1][k][j]);
                        if constexpr (kMode == kWhole)
                            sums[k] = j ? fmaf(c[g & 1][k][j], h[j], sums[k]) : c[g & 1][k][j] * h[j];
                    }
                };
                token(std::integral_constant<int, 0>{});
                token(std::integral_constant<int, 1>{});
                token(std::integral_constant<int, 2>{});
                token(std::integral_constant<int, 3>{});
                if constexpr (kMode == kWhole) {
                    float s = fmaf(skip, xv[g], quad_sums(sums, sub));
                    if constexpr (kGate)
                        s *= gv[g] * sigmoid(gv[g]);
                    buffer_store<Scalar>(s, out, y_rows.at + g * y_rows.step);
                }
            }
        };
        float *kept = nullptr;
        if (kMode == kWhole && job.kept)
            kept = job.kept + (scan_slot(job.seq, piece.seq, piece.lo) + (piece.t0 - piece.lo) / kScanKept) * wide + mine;
        if (piece.len > 0)
            load(0);
        for (int t = 0, turn = 0; t < piece.len; t += kTile, turn ^= 1) {
            B_rows.store(tile[turn], Bs);
            if constexpr (kMode == kWhole)
                C_rows.store(tile[turn] + Groups::kFloats, Cs);
            wave_sync();
            if (kMode == kWhole && job.kept && at.valid) {
                store_states<NR>(kept, h, NR);
                kept += wide;
            }
            if (t + kTile <= piece.len)
                walk(t, tile[turn], std::true_type{});
            else
                walk(t, tile[turn], std::false_type{});
        }
        if constexpr (kMode == kEnds) {
            span += __shfl_xor(span, 1);
            span += __shfl_xor(span, 2);
            if (at.valid) {
                store_states<NR>(job.ends + at.piece * wide + mine, h, NR);
                if (sub == 0)
                    job.spans[static_cast<int64_t>(at.piece) * job.D + channel] = span;
            }
        } else if (piece.at == piece.count - 1 && at.valid) {
            store_states<NR>(job.state + (static_cast<int64_t>(piece.seq) * job.D + channel) * job.S + n0, h, count);
        }
    }
    if (kMode == kWhole && at.valid)
        for (int i = sub; i < piece.rest; i += 4)
            store_vec<Scalar, 1>(y + static_cast<int64_t>(piece.len + i) * job.D, {{0u}});
}

// NR values of a token's B or C, those past S zero.
template<typename Scalar, int NR>
__device__ __forceinline__ void load_group(float (&to)[NR], const Scalar *p, int count) {
    if constexpr (NR * sizeof(Scalar) % 4 == 0) {
        if (count >= NR) {
            const Vec<Scalar, NR> v = load_vec<Scalar, NR>(p);
#pragma unroll
            for (int j = 0; j < NR; ++j)
                to[j] = v[j];
            return;
        }
    }
#pragma unroll
    for (int j = 0; j < NR; ++j)
        to[j] = j < count ? load_f32(p + j) : 0.f;
}

// Decode steps of up to kScanStepTokens tokens, bound by reading and writing the states: no staging, one wave
// 16 channels of a sequence, and of others where the grid has fewer rows than the batch (its rates are read once).
// kOne: of one token, which all lanes of a channel prepare alike; otherwise each prepares one of four.
template<typename Scalar, int NR, bool kOne>
__global__ __launch_bounds__(kThreads) void scan_step_kernel(const ScanJob job, int rows) {
    const ScanPlace at(job);
    const int sub = at.sub, channel = at.channel, n0 = sub * NR, count = job.S - n0, T = kOne ? 1 : job.seq.T;
    float A2[NR];
    load_states<NR>(A2, job.A + static_cast<int64_t>(channel) * job.S + n0, count);
#pragma unroll
    for (int j = 0; j < NR; ++j)
        A2[j] *= kLog2e;
    const float bias = job.bias ? job.bias[channel] : 0.f, skip = job.skip ? job.skip[channel] : 0.f;
    for (int b = at.piece; b < job.seq.B; b += rows) {
        const int len = job.seq.lengths ? clamped(job.seq.lengths[b], 0, T) : T, last = max(len - 1, 0);
        float h[NR];
        const int64_t where = (static_cast<int64_t>(b) * job.D + channel) * job.S + n0;
        if (job.init) {
            load_states<NR>(h, job.init + where, count);
        } else {
#pragma unroll
            for (int j = 0; j < NR; ++j)
                h[j] = 0.f;
        }
        const Scalar *x = static_cast<const Scalar *>(job.x) + b * job.x_at[0] + channel;
        const Scalar *dt = static_cast<const Scalar *>(job.dt) + b * job.dt_at[0] + channel;
        const Scalar *gate = static_cast<const Scalar *>(job.gate) + b * job.gate_at[0] + channel;
        const Scalar *B = static_cast<const Scalar *>(job.B) + b * job.B_at[0] + at.group * job.B_at[2] + n0;
        const Scalar *C = static_cast<const Scalar *>(job.C) + b * job.C_at[0] + at.group * job.C_at[2] + n0;
        Scalar *y = static_cast<Scalar *>(job.y) + static_cast<int64_t>(b) * T * job.D + channel;
        constexpr int kTokens = kOne ? 1 : 4, kDeep = kOne ? 1 : NR <= 4 ? 4 : NR <= 8 ? 2 : 1;
        for (int t0 = 0; t0 < T; t0 += kTokens) {
            const int t = kOne ? 0 : t0 + sub, from = min(t, last);  // (what is read of no token that counts goes nowhere)
            const float xv = load_f32(x + from * job.x_at[1]);
            const float raw = load_f32(dt + from * job.dt_at[1]) + bias;
            const float gv = job.gate ? load_f32(gate + from * job.gate_at[1]) : 0.f;
            float sums[4] = {}, d = raw, e, b_of[kDeep][NR], c_of[kDeep][NR];
            auto fetch = [&](int k0) {
#pragma unroll
                for (int k = 0; k < kDeep; ++k) {
                    const int at_token = min(t0 + k0 + k, last);
                    load_group<Scalar, NR>(b_of[k], B + at_token * job.B_at[1], count);
                    load_group<Scalar, NR>(c_of[k], C + at_token * job.C_at[1], count);
                }
            };
            fetch(0);
            if (job.softplus)
                d = softplus(raw, e);
            const float u = d * xv;
            auto token = [&](auto k_) {
                constexpr int k = decltype(k_)::value;
                if constexpr (k > 0 && k % kDeep == 0)
                    fetch(k);
                if (t0 + k >= len)
                    return;
                const float dk = kOne ? d : quad_lane<k>(d), uk = kOne ? u : quad_lane<k>(u);
#pragma unroll
                for (int j = 0; j < NR; ++j) {
                    h[j] = fmaf(__builtin_amdgcn_exp2f(dk * A2[j]), h[j], uk * b_of[k % kDeep][j]);
                    sums[k] = fmaf(c_of[k % kDeep][j], h[j], sums[k]);
                }
            };
            token(std::integral_constant<int, 0>{});
            if constexpr (!kOne) {
                token(std::integral_constant<int, 1>{});
                token(std::integral_constant<int, 2>{});
                token(std::integral_constant<int, 3>{});
            }
            float s = sums[0];
            if constexpr (kOne) {
                s += quad_swap<1>(s);
                s += quad_swap<2>(s);
            } else {
                s = quad_sums(sums, sub);
            }
            float out = fmaf(skip, xv, s);
            if (job.gate)
                out *= gv * sigmoid(gv);
            if (at.valid && t < T && (!kOne || sub == 0))
                store_vec<Scalar, 1>(y + static_cast<int64_t>(t) * job.D, {{round_bits<Scalar>(t < len ? out : 0.f)}});
        }
        if (at.valid)
            store_states<NR>(job.state + where, h, count);
    }
}

// Blocks of a decode step, past which they take several rows (2048 channels of 16 states, one token: 256 rows 18.6 us,
// a row a block 22.3; 2048 rows 126 for 155; blocks of 8192 22.4 and 128).
constexpr unsigned kStepBlocks = 4096;

// Blocks of a launch over `pieces` pieces.
unsigned blocks_of(const ScanJob &job, int64_t pieces) {
    return static_cast<unsigned>(pieces * job.G * ((job.D / job.G + kScanChannels - 1) / kScanChannels));
}

template<typename Scalar, int NR>
hipError_t launch_states(const ScanJob &job, hipStream_t stream) {
    const dim3 block(kThreads);
    if (scan_is_step(job)) {
        const unsigned per_row = blocks_of(job, 1);
        const int rows = std::min(job.seq.B, static_cast<int>((kStepBlocks + per_row - 1) / per_row));
        if (job.seq.T == 1)
            hipLaunchKernelGGL((scan_step_kernel<Scalar, NR, true>), dim3(rows * per_row), block, 0, stream, job, rows);
        else
            hipLaunchKernelGGL((scan_step_kernel<Scalar, NR, false>), dim3(rows * per_row), block, 0, stream, job, rows);
        return hipGetLastError();
    }
    const dim3 grid(blocks_of(job, most_pieces(job.seq, job.step)));
    if (job.seq.T > job.step)
        hipLaunchKernelGGL((scan_kernel<Scalar, NR, kEnds, false>), grid, block, 0, stream, job);
    if (job.gate)
        hipLaunchKernelGGL((scan_kernel<Scalar, NR, kWhole, true>), grid, block, 0, stream, job);
    else
        hipLaunchKernelGGL((scan_kernel<Scalar, NR, kWhole, false>), grid, block, 0, stream, job);
    return hipGetLastError();
}

template<typename Scalar>
hipError_t launch_type(const ScanJob &job, hipStream_t stream) {
    switch (scan_lane_states(job.S)) {
        case 1: return launch_states<Scalar, 1>(job, stream);
        case 2: return launch_states<Scalar, 2>(job, stream);
        case 3: return launch_states<Scalar, 3>(job, stream);
        case 4: return launch_states<Scalar, 4>(job, stream);
        case 6: return launch_states<Scalar, 6>(job, stream);
        case 8: return launch_states<Scalar, 8>(job, stream);
        case 12: return launch_states<Scalar, 12>(job, stream);
        default: return launch_states<Scalar, 16>(job, stream);
    }
}

}  // namespace

bool scan_is_step(const ScanJob &job) { return !job.seq.cu && !job.kept && job.seq.T <= kScanStepTokens; }

// Rows are cut into pieces where their channels alone leave compute units idle. The state after each piece from zeros
// is a pass of its own that costs two thirds of the other, so a row in many pieces takes as long as 1.35 in one do
// where the waves of either fill the machine: 4096 tokens of 1024 waves took 395 us in one piece, 550 in two
// (336 + 230) and 515 in four. From 768 waves on, three quarters of what runs at once, rows stay whole. Below that
// 4096 waves (four a SIMD) hide each other's latencies: 32768 tokens of 64 waves take 277 us in 32 pieces, 266 in 64.
// The backward has registers for two waves a SIMD, and keeps to 2048. A piece joins the ends of those before it one by
// one, so a row of few channels is cut into three quarters of the root of its tokens at most: 16 channels take 2438 us
// for 262144 tokens in 4096 pieces, 234 in 256 and 251 in 512; for 16384 tokens 87 in 256, 64 in 64 or 128.
int scan_step_tokens(const ScanJob &job, bool backward) {
    const int64_t rows = job.seq.B > 0 ? job.seq.B : 1;
    const int64_t waves = rows * job.G * ((job.D / job.G + 15) / 16), most = backward ? 2048 : 4096;
    const int64_t joined = std::max<int64_t>(1, static_cast<int64_t>(0.75 * std::sqrt(static_cast<double>(job.seq.T))));
    const int64_t parts = waves >= 768 ? 1 : std::min((most + waves - 1) / waves, joined);
    const int64_t tokens = (job.seq.T + parts - 1) / parts;
    const int64_t step = (tokens + kScanKept - 1) / kScanKept * kScanKept;
    return static_cast<int>(step < 64 ? 64 : step);
}

int64_t scan_layout(ScanJob &job, bool backward, char *base, ScanGrads *grads) {
    int64_t size = 0;
    auto region = [&](int64_t bytes) {
        char *at = base ? base + size : nullptr;
        size += (bytes + 255) / 256 * 256;
        return at;
    };
    if (!backward && scan_is_step(job))
        return 0;
    job.step = scan_step_tokens(job, backward);
    const int64_t pieces = most_pieces(job.seq, job.step), wide = 4LL * scan_lane_states(job.S);
    if (job.seq.cu) {
        job.seq.bounds = reinterpret_cast<int32_t *>(region((job.seq.N + 1) * 4LL));
        job.seq.first = reinterpret_cast<int32_t *>(region((job.seq.N + 1) * 4LL));
    }
    const bool cut = job.seq.T > job.step;
    if (cut) {
        job.spans = reinterpret_cast<double *>(region(pieces * job.D * 8));
        float *ends = reinterpret_cast<float *>(region(pieces * job.D * wide * 4));
        if (backward && grads)
            grads->backs = ends;
        else
            job.ends = ends;
    }
    if (backward) {
        const int64_t blocks = blocks_of(job, 1) / job.G;  // of a group
        float *groups = reinterpret_cast<float *>(region(blocks * job.seq.B * job.seq.T * job.G * 2 * wide * 4));
        float *sums = reinterpret_cast<float *>(region(pieces * job.D * (wide + 2) * 4));
        if (grads)
            grads->groups = groups, grads->sums = sums;
    }
    return size;
}

int64_t scan_kept_bytes(const ScanJob &job) { return scan_slots(job.seq) * job.D * 16 * scan_lane_states(job.S); }

hipError_t launch_scan(const ScanJob &job, hipStream_t stream, const char **why) {
    if (job.seq.cu) {
        const hipError_t err = launch_sequences(job.seq, job.step, stream);
        if (err != hipSuccess)
            return err;
    }
    switch (job.dtype) {
        case kF32: return launch_type<float>(job, stream);
        case kF16: return launch_type<_Float16>(job, stream);
        case kBF16: return launch_type<bf16_t>(job, stream);
        default: *why = "selective_scan: unsupported dtype"; return hipErrorInvalidValue;
    }
}

}  // namespace ramnet
