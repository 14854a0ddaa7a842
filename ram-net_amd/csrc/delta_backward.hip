// Gradients of the gated delta rule in chunks of 64 tokens. With the forward's
// names (delta_chunk.hpp), dO the output's gradient and D the state's after
// the chunk, E and S as the forward kept them:
//     X = Y^T (beta . (P^T dO + e^(gamma_C - gamma) . K D))        (= dV)
//     D <- e^gamma_C D + Q^T (scale e^gamma . dO) - K^T (e^gamma . X)
// runs from the last chunk to the first (chain); then, all chunks at once, with
// R1 = dO E^T and R2 = -X E^T:
//     dA = scale lower(R1 . L) beta_j,   dB = strictlower(R2 . L) beta_j
//     dQ = dA K + scale e^gamma . (dO S^T)
//     dK = dA^T Q + (dB + dB^T) K - e^gamma . (X S^T) + e^(gamma_C - gamma) beta . (E D^T)
//     dbeta_j = sum_i (P . R1 + Bl . R2)_ij + e^(gamma_C - gamma_j) K_j . (E D^T)_j
//     dgamma_i: the row sums less the column sums of (P . R1 + Bl . R2) beta_j, and what
//               e^gamma_i, e^(gamma_C - gamma_i) and e^gamma_C multiply;  dg: its sums from the end
#include "delta_split.hpp"
#include "ramnet_kernels.hpp"

namespace ramnet {

namespace {

// The states' gradient from the last chunk to the first; waves as in the
// forward's chain. The state's gradient and dv are fp32 results of fp32 values:
// every product takes both parts of both sides (dO's own 16 bits are one part).
// Rows in segments as in the forward's chain, the last one first (PART: the
// gradients at their starts from zeros at their ends; their maps are the
// forward's, transposed).
template<typename Scalar, int DT, int PIECES, int BUFS, bool PART>
__global__ __launch_bounds__(512, 2) void chain_back_kernel(const DeltaJob job, const DeltaWork work,
                                                            const DeltaGrads grads, int groups) {
    extern __shared__ __align__(16) float lds_base[];
    using Lds = ChunkLds<DT, PIECES, true>;
    constexpr int C = kDeltaChunk, BT = DT / 2;
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave, wave = uniform(tid / kWave);
    const int row = lane & 15, grp = lane >> 4;
    const int parts = PART ? work.parts - 1 : work.parts;
    int group, item;
    split_block(static_cast<int>(blockIdx.x), groups, job.N * job.Hv * parts, group, item);
    const int part = item % parts, line = item / parts;  // from the end
    const int head = line % job.Hv, n = delta_line(work, line / job.Hv);
    const int kh = head / (job.Hv / job.Hk);
    DeltaSpan span = delta_span(job, n);
    const int row_end = span.len;
    int first, count;
    delta_chunks(job, work, n, span, first, count);
    int skipped = 0;
    const int segments = delta_segments(work, count);
    if (part >= segments || (PART && part + 1 == segments))
        return;
    if (segments > 1) {
        const int to = count;
        skipped = (segments - 1 - part) * work.part_chunks;
        first += skipped;
        count = min(to - skipped, work.part_chunks);
        span.t0 += skipped * C, span.len = min(span.len - skipped * C, count * C);
    }
    auto buffer = [&](int i) {
        return Lds{reinterpret_cast<uint16_t *>(reinterpret_cast<char *>(lds_base) + (BUFS == 2 ? (i & 1) * Lds::kBytes : 0))};
    };

    if (wave >= 4) {
        const int at = tid - 256;
        const Scalar *k = static_cast<const Scalar *>(job.k) + span.b * job.k_at[0] + kh * job.k_at[2];
        const Scalar *q = static_cast<const Scalar *>(job.q) + span.b * job.q_at[0] + kh * job.q_at[2];
        Stager<Scalar, DT, PIECES, true> stager;
        auto bring = [&](auto wide) {
            auto load = [&](int i) {
                const int64_t t0 = span.t0 + i * C;
                stager.template load<decltype(wide)::value, true>(
                    k + t0 * job.k_at[1], job.k_at[1], q + t0 * job.q_at[1], job.q_at[1], min(C, span.len - i * C), job.Dk,
                    work.vec + (static_cast<int64_t>(first + i) * job.Hv + head) * kVecs * C, at);
            };
            if (count > 0) {
                load(count - 1);
                stager.template store<true>(buffer(count - 1), at);
            }
            __syncthreads();
            for (int i = count - 1; i >= 0; --i) {
                load(max(i - 1, 0));
                if constexpr (BUFS == 1)
                    __syncthreads();  // chunk i is done with
                stager.template store<true>(buffer(i - 1), at);
                __syncthreads();
            }
        };
        if (rows_whole<Scalar>(job))
            bring(std::true_type{});
        else
            bring(std::false_type{});
        return;
    }

    const int c = (group * 4 + wave) * 16 + row;
    const int64_t matrix = (static_cast<int64_t>(n) * job.Hv + head) * job.Dk * job.Dv;
    const int64_t piece = static_cast<int64_t>(line) * work.parts + part;  // of the segments' ends
    const Columns<float> state(job.Dv, job.Dv, grp, c), kept(delta_row(job.Dv), delta_row(job.Dv), grp, c);
    f32x4 s[DT];
    {
        const float *after = part == 0 ? grads.d_state ? grads.d_state + matrix : nullptr
                             : PART    ? nullptr
                                       : work.ends + (piece - 1) * job.Dk * job.Dv;
        const auto from = state.rows(after, after ? job.Dk : 0);
        state.each<DT>([&](int t, int r, int at) { s[t][r] = __uint_as_float(buffer_bits<float>(from, at)); });
    }
    const Scalar *d_o = static_cast<const Scalar *>(grads.d_o) + span.b * grads.d_o_at[0] + head * grads.d_o_at[2] +
                        span.t0 * grads.d_o_at[1];
    const int64_t dv_step = static_cast<int64_t>(job.Hv) * job.Dv;
    Scalar *dv = static_cast<Scalar *>(grads.dv) + (static_cast<int64_t>(span.b) * job.T + span.t0) * dv_step +
                 static_cast<int64_t>(head) * job.Dv;
    const Columns<Scalar> o_cols(grads.d_o_at[1], job.Dv, grp, c), v_cols(dv_step, job.Dv, grp, c);
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    uint32_t o_bits[16];
    auto load_o = [&](int i) {
        const auto from = o_cols.rows(d_o + static_cast<int64_t>(i) * C * grads.d_o_at[1], min(C, span.len - i * C));
        o_cols.template each<4>([&](int m, int r, int at) { o_bits[4 * m + r] = buffer_bits<Scalar>(from, at); });
    };
    // the next chunk's operands are asked for as soon as this one's have been used
    u32x4 y_hi[kFrags], y_lo[kFrags], p_hi[kFrags], p_lo[kFrags];
    auto load_frags = [&](const uint32_t *from, int i, u32x4 (&hi)[kFrags], u32x4 (&lo)[kFrags]) {
        const int64_t record = static_cast<int64_t>(first + i) * job.Hv + head;
        const u32x4 *at = reinterpret_cast<const u32x4 *>(from + record * 2 * kFragWords);
#pragma unroll
        for (int f = 0; f < kFrags; ++f)
            hi[f] = at[f * kWave + lane], lo[f] = at[(kFrags + f) * kWave + lane];
    };
    if (count > 0) {
        load_o(count - 1);
        load_frags(work.p_frags, count - 1, p_hi, p_lo);
        load_frags(work.y, count - 1, y_hi, y_lo);
        arrived(o_bits);
        arrived(p_hi);
        arrived(p_lo);
        arrived(y_hi);
        arrived(y_lo);
    }
    arrived(s);
    __syncthreads();

    for (int i = count - 1; i >= 0; --i) {
        const int64_t record = static_cast<int64_t>(first + i) * job.Hv + head;
        const Lds lds = buffer(i);
        const float *vec = lds.vec();
        const float total = vec[kVecTotal * C];
        if constexpr (!PART) {
            const auto to = kept.rows(work.dstate + record * job.Dk * delta_row(job.Dv), job.Dk);
            kept.each<DT>([&](int t, int r, int at) { buffer_store<float>(s[t][r], to, at); });
        }
        f32x4 out[4], du[4], x[4];
        float x_inverse;
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                out[m][r] = bits_f32<Scalar>(o_bits[4 * m + r]);
        const int then = max(i - 1, 0);  // (the first chunk's once more rather than a branch)
        load_o(then);
        {
            Operand<4> oo;
            oo.set(out);
#pragma unroll
            for (int m = 0; m < 4; ++m)
                x[m] = zero;
            // (dO's second part is 0 for bf16 but far below a column's largest)
            triangle<true, !__is_same(Scalar, bf16_t)>(p_hi, p_lo, oo.hi, oo.lo, x);
            x_inverse = vec[kVecInv * C + 1] * oo.inverse;
            load_frags(work.p_frags, then, p_hi, p_lo);
        }
        {
            Operand<DT> so;
            so.set(s);
#pragma unroll
            for (int m = 0; m < 4; ++m)
                du[m] = zero;
#pragma unroll
            for (int b = 0; b < BT; ++b)
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    const u32x4 kf = lds.row_frag(lds.k(0), m, b, lane);
                    du[m] = mfma16(kf, so.hi[b], du[m]);
                    du[m] = mfma16(kf, so.lo[b], du[m]);
                    if constexpr (PIECES == 2)
                        du[m] = mfma16(lds.row_frag(lds.k(1), m, b, lane), so.hi[b], du[m]);
                }
#pragma unroll
            for (int m = 0; m < 4; ++m)
                du[m] = (x[m] * x_inverse + du[m] * (load4(vec + kVecLeftK * C + 16 * m + 4 * grp) * so.inverse)) *
                        load4(vec + kVecBeta * C + 16 * m + 4 * grp);
        }
        {
            Operand<4> uo;
            uo.set(du);
#pragma unroll
            for (int m = 0; m < 4; ++m)
                x[m] = zero;
            triangle<true>(y_hi, y_lo, uo.hi, uo.lo, x);
            x_inverse = vec[kVecInv * C] * uo.inverse;
#pragma unroll
            for (int m = 0; m < 4; ++m)
                x[m] = x[m] * x_inverse;
            load_frags(work.y, then, y_hi, y_lo);
        }
        if constexpr (!PART) {
            const auto to = kept.rows(work.x + record * C * delta_row(job.Dv), C);
            kept.each<4>([&](int m, int r, int at) { buffer_store<float>(x[m][r], to, at); });
            const auto out_to = v_cols.rows(dv + static_cast<int64_t>(i) * C * dv_step, min(C, span.len - i * C));
            v_cols.template each<4>([&](int m, int r, int at) { buffer_store<Scalar>(x[m][r], out_to, at); });
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            x[m] = -(load4(vec + kVecGrowK * C + 16 * m + 4 * grp) * x[m]);
            out[m] = out[m] * load4(vec + kVecGrowQ * C + 16 * m + 4 * grp);
        }
        Operand<4> xo, oo;
        xo.set(x);
        oo.set(out);
        // (operands read ahead as in the forward's chain do not fit the registers here)
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            f32x4 a = zero, z = zero;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const u32x4 kf = lds.col_frag(lds.kt(0), t, b, lane), qf = lds.col_frag(lds.qt(0), t, b, lane);
                a = mfma16(kf, xo.hi[b], a);
                z = mfma16(qf, oo.hi[b], z);
                a = mfma16(kf, xo.lo[b], a);
                z = mfma16(qf, oo.lo[b], z);
                if constexpr (PIECES == 2) {
                    a = mfma16(lds.col_frag(lds.kt(1), t, b, lane), xo.hi[b], a);
                    z = mfma16(lds.col_frag(lds.qt(1), t, b, lane), oo.hi[b], z);
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r)
                s[t][r] = fmaf(a[r], xo.inverse, fmaf(z[r], oo.inverse, total * s[t][r]));
        }
        __syncthreads();
        if constexpr (BUFS == 1)
            __syncthreads();  // chunk i - 1 is there
    }
    float *const before = PART ? work.ends + piece * job.Dk * job.Dv
                          : part + 1 < segments || !grads.dinit ? nullptr
                                                                   : grads.dinit + matrix;
    if (before) {
        const auto to = state.rows(before, job.Dk);
        state.each<DT>([&](int t, int r, int at) { buffer_store<float>(s[t][r], to, at); });
    }
    if (!PART && part == 0 && !job.cu && c < job.Dv)  // tokens that do not count
        for (int64_t t = row_end + grp; t < job.T; t += 4)
            store_f32(dv + (t - skipped * C) * dv_step + c, 0.f);
}

// Sum over the 16 lanes of a row group (rotations within it).
template<int ROR>
__device__ __forceinline__ float rotated(float x) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x120 + ROR, 0xF, 0xF, true));
}
__device__ __forceinline__ float row_sum(float x) {
    x += rotated<8>(x);
    x += rotated<4>(x);
    x += rotated<2>(x);
    return x + rotated<1>(x);
}

__device__ __forceinline__ void store_code(void *p, int code, int64_t at, float v) {
    if (code == 0)
        static_cast<float *>(p)[at] = v;
    else if (code == 1)
        store_f32(static_cast<_Float16 *>(p) + at, v);
    else
        store_f32(static_cast<bf16_t *>(p) + at, v);
}

// Eight values of a row as they are in memory.
template<typename Scalar>
struct Eight {
    static constexpr int kWords = 2 * static_cast<int>(sizeof(Scalar));
    uint32_t w[kWords];

    // from column v of the row that begins at byte `at` of the window on, zeros from
    // `wide` on; EVEN: rows begin at multiples of 16 bytes and are whole pieces of them
    template<bool EVEN>
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t from, int at, int v, int wide) {
        constexpr int size = static_cast<int>(sizeof(Scalar)), each = 16 / size;
        at += v * size;
        if constexpr (EVEN) {
#pragma unroll
            for (int i = 0; i < kWords; i += 4) {
                const int e = i / 4 * each;
                const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(from, v + e < wide ? at + 4 * i : kNowhere, 0, 0);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    w[i + k] = x[k];
            }
        } else {
            uint32_t x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                x[e] = buffer_bits<Scalar>(from, v + e < wide ? at + e * size : kNowhere);
#pragma unroll
            for (int i = 0; i < kWords; ++i)
                w[i] = size == 4 ? x[i] : x[(2 * i) % 8] | x[(2 * i + 1) % 8] << 16;
        }
    }
    __device__ __forceinline__ float operator[](int e) const {
        return bits_f32<Scalar>(sizeof(Scalar) == 4 ? w[e % kWords] : (w[e / 2 % kWords] >> (e % 2 * 16)) & 0xFFFFu);
    }
    __device__ __forceinline__ float largest(float m) const {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            m = fmaxf(m, fabsf((*this)[e]));
        return m;
    }
};

// The fp16 parts of eight values.
template<typename Scalar>
__device__ __forceinline__ void split8(const Eight<Scalar> &x, float scale, u32x4 &hi, u32x4 &lo) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        uint32_t h, l;
        split2(x[2 * w], x[2 * w + 1], scale, h, l);
        hi[w] = h, lo[w] = l;
    }
}

// LDS of inputs_back_kernel, in halves: K and Q by element, then 64 columns of
// dO, X and E by token; where the products of these are done with, the token by
// token matrices of the second stage take their place.
template<int DT, int PIECES>
struct BackLds {
    static constexpr int kSlab = 64, kPitch = kSlab + 8, kPart = kDeltaChunk * kPitch;
    static constexpr int kCols = 16 * DT * (kDeltaChunk + 8);  // of K or Q, a part
    static constexpr int kKeys = 2 * PIECES * kCols;
    static constexpr int kParts = PIECES + 4, kSquares = 3 * 2;
    static constexpr int kBytes = 2 * (kKeys + kPart * (kParts > kSquares ? kParts : kSquares));
};

// The other gradients of one chunk and key head; its value heads one after the
// other, so that a shared head's sums have one order. Products over Dv with S
// and D: a wave has every eighth (or fourth) tile of Dk and all tokens, S and D come from
// memory straight into its registers, dO, X and E through LDS; what comes from
// memory is asked for one step ahead of its use.
// WIDE: q, k and d_o are read in pieces of 16 bytes. WAVES: 8, so that one's
// loads hide behind another's products (bf16, 4 rows of 2048 tokens, 8 heads of
// 128 x 128: 115 us of a training step's 377, 25 more with 4), or 4 of twice the registers
// where 8 spill (fp32, 3001 tokens, 6 heads of 72 x 96: 58 us, 116 with 8).
template<typename Scalar, int DT, int PIECES, bool WIDE, int WAVES>
__global__ __launch_bounds__(kWave *WAVES, WAVES / 4) void inputs_back_kernel(const DeltaJob job, const DeltaWork work,
                                                          const DeltaGrads grads) {
    extern __shared__ __align__(16) float lds_base[];
    using Lds = BackLds<DT, PIECES>;
    constexpr int C = kDeltaChunk, kPitchT = C + 8, kThreads = kWave * WAVES;
    constexpr int TW = (DT + WAVES - 1) / WAVES, NR = (10 + WAVES - 1) / WAVES, NI = 512 / kThreads;
    uint16_t *const halves = reinterpret_cast<uint16_t *>(lds_base);
    uint16_t *const kt = halves, *const qt = halves + PIECES * Lds::kCols, *const parts = halves + Lds::kKeys;
    __shared__ double gam[C];
    __shared__ float beta_s[C], grow[C], left[C], inv_k[C], inv_q[C];
    __shared__ float inv_o[C], inv_x[C], inv_e[C];              // of a slab's rows
    __shared__ float dots[3][WAVES][C];                             // [q, x, e][wave]
    __shared__ float rows[4][C], cols[4][C], diag[C], state_dot[WAVES], largest[3][WAVES];
    const int tid = static_cast<int>(threadIdx.x), wave = uniform(tid / kWave);
    int lane = tid % kWave, row = lane & 15, grp = lane >> 4;
    const int chunk = blockIdx.x, kh = blockIdx.y, shared = job.Hv / job.Hk;
    const DeltaPlace at = delta_place(job, work, chunk);
    const int Dk = job.Dk, Dv = job.Dv, row_v = delta_row(Dv);
    const int64_t dk_step = static_cast<int64_t>(job.Hk) * Dk;
    Scalar *dq = static_cast<Scalar *>(grads.dq) + static_cast<int64_t>(kh) * Dk;
    Scalar *dk = static_cast<Scalar *>(grads.dk) + static_cast<int64_t>(kh) * Dk;
    // tokens of no sequence or past a row's length
    auto clear = [&](int64_t from, int64_t to) {
        for (int64_t t = from + wave; t < to; t += WAVES) {
            for (int d = lane; d < Dk; d += kWave) {
                store_f32(dq + t * dk_step + d, 0.f);
                store_f32(dk + t * dk_step + d, 0.f);
            }
            for (int h = lane; h < shared; h += kWave) {
                store_code(grads.dg, job.g_dtype, t * job.Hv + kh * shared + h, 0.f);
                store_code(grads.dbeta, job.beta_dtype, t * job.Hv + kh * shared + h, 0.f);
            }
            if (job.cu)
                for (int i = lane; i < shared * Dv; i += kWave)
                    store_f32(static_cast<Scalar *>(grads.dv) + (t * job.Hv + kh * shared) * Dv + i, 0.f);
        }
    };
    if (job.cu) {
        if (at.n < 0) {
            delta_outside(job, work, chunk, clear);
            return;
        }
    } else if (at.len < C) {
        const int64_t base = static_cast<int64_t>(at.b) * job.T;
        clear(base + at.t0 + at.len, base + min(at.t0 + C, job.T));
    }
    if (at.len == 0)
        return;

    // K, and Q: by four waves each
    {
        using Keys = Stager<Scalar, DT, PIECES, true>;
        Keys keys;
        const Scalar *k = static_cast<const Scalar *>(job.k) + at.b * job.k_at[0] + at.t0 * job.k_at[1] + kh * job.k_at[2];
        const Scalar *q = static_cast<const Scalar *>(job.q) + at.b * job.q_at[0] + at.t0 * job.q_at[1] + kh * job.q_at[2];
        const float *scales = work.vec + (static_cast<int64_t>(chunk) * job.Hv + kh * shared) * kVecs * C + tid % 16 * 4;
        const bool is_q = wave >= 4;
        keys.template load_one<WIDE>(is_q ? q : k, is_q ? job.q_at[1] : job.k_at[1], at.len, Dk, tid % 256, keys.raw[0]);
        if constexpr (WAVES == 4)
            keys.template load_one<WIDE>(q, job.q_at[1], at.len, Dk, tid, keys.raw[1]);
        Keys::store_one(keys.raw[0], load4(scales + (is_q ? kVecSq : kVecSk) * C), tid % 256, nullptr, is_q ? qt : kt);
        if constexpr (WAVES == 4)
            Keys::store_one(keys.raw[1], load4(scales + kVecSq * C), tid, nullptr, qt);
    }
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    f32x4 sum_q[TW][4], sum_k[TW][4];
#pragma unroll
    for (int t = 0; t < TW; ++t)
#pragma unroll
        for (int m = 0; m < 4; ++m)
            sum_q[t][m] = sum_k[t][m] = zero;
    const int64_t token0 = static_cast<int64_t>(at.b) * job.T + at.t0;

    for (int h = 0; h < shared; ++h) {
        const int head = kh * shared + h;
        // (addresses made here are not kept over the loop: they would fill the registers)
        asm volatile("" : "+v"(lane));
        row = lane & 15, grp = lane >> 4;
        const int64_t record = static_cast<int64_t>(chunk) * job.Hv + head;
        const float *vec = work.vec + record * kVecs * C;
        const float *e = work.e + record * C * row_v, *x = work.x + record * C * row_v;
        const float *s = work.states + record * Dk * row_v, *d = work.dstate + record * Dk * row_v;
        const Scalar *d_o = static_cast<const Scalar *>(grads.d_o) + at.b * grads.d_o_at[0] +
                            at.t0 * grads.d_o_at[1] + head * grads.d_o_at[2];
        // a slab of dO, X and E: eight columns of a token a thread
        Eight<Scalar> xo[NI];
        Eight<float> xx[NI], xe[NI], sv[2], dv[2];
        const int slab_t = tid / 8, slab_c = tid % 8 * 8;
        const auto o_rows = window(d_o, (at.len - 1) * grads.d_o_at[1] * static_cast<int64_t>(sizeof(Scalar)) + Dv * sizeof(Scalar));
        const auto x_rows = window(x, static_cast<int64_t>(C) * row_v * 4), e_rows = window(e, static_cast<int64_t>(C) * row_v * 4);
        const auto s_rows = window(s, static_cast<int64_t>(Dk) * row_v * 4), d_rows = window(d, static_cast<int64_t>(Dk) * row_v * 4);
        auto load_slab = [&](int v0) {
#pragma unroll
            for (int n = 0; n < NI; ++n) {
                const int t = slab_t + n * (kThreads / 8);
                xo[n].template load<WIDE>(o_rows, t * static_cast<int>(grads.d_o_at[1] * sizeof(Scalar)), v0 + slab_c, Dv);
                xx[n].template load<true>(x_rows, t * row_v * 4, v0 + slab_c, row_v);
                xe[n].template load<true>(e_rows, t * row_v * 4, v0 + slab_c, row_v);
            }
        };
        auto load_states = [&](int v0, int t) {
            const int at_row = (16 * t + row) * row_v * 4;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                sv[b].template load<true>(s_rows, at_row, v0 + 32 * b + 8 * grp, row_v);
                dv[b].template load<true>(d_rows, at_row, v0 + 32 * b + 8 * grp, row_v);
            }
        };
        load_slab(0);
        if (wave < DT)
            load_states(0, wave);
        __syncthreads();
        if (wave == 0) {
            const double own = work.gamma[record * C + lane], end = work.gamma[record * C + C - 1];
            gam[lane] = own;
            grow[lane] = decay_of(own);
            left[lane] = decay_of(end - own);
        } else if (wave == 1) {
            beta_s[lane] = vec[kVecBeta * C + lane];
            inv_k[lane] = 1.f / vec[kVecSk * C + lane];
            inv_q[lane] = 1.f / vec[kVecSq * C + lane];
        }

        // dO S^T, X S^T, E D^T (this wave's tiles of Dk) and R1, R2 (every fourth lower tile)
        f32x4 os[TW][4], xs[TW][4], ed[TW][4], r1[NR], r2[NR];
#pragma unroll
        for (int t = 0; t < TW; ++t)
#pragma unroll
            for (int m = 0; m < 4; ++m)
                os[t][m] = xs[t][m] = ed[t][m] = zero;
#pragma unroll
        for (int n = 0; n < NR; ++n)
            r1[n] = r2[n] = zero;
        float both = 0.f;
        for (int v0 = 0; v0 < Dv; v0 += Lds::kSlab) {
            asm volatile("" : "+v"(lane));
            row = lane & 15, grp = lane >> 4;
            if (v0 > 0)
                __syncthreads();
#pragma unroll
            for (int n = 0; n < NI; ++n) {
                const int t = slab_t + n * (kThreads / 8);
                float mo = xo[n].largest(0.f), mx = xx[n].largest(0.f), me = xe[n].largest(0.f);
#pragma unroll
                for (int k = 1; k < 8; k <<= 1) {
                    mo = fmaxf(mo, __shfl_xor(mo, k));
                    mx = fmaxf(mx, __shfl_xor(mx, k));
                    me = fmaxf(me, __shfl_xor(me, k));
                }
                float io, ix, ie;
                const float so = scale_of(mo, io), sx = scale_of(mx, ix), se = scale_of(me, ie);
                if (tid % 8 == 0)
                    inv_o[t] = io, inv_x[t] = ix, inv_e[t] = ie;
                u32x4 hi, lo;
                auto put = [&](int part, u32x4 w) {
                    *reinterpret_cast<u32x4 *>(parts + part * Lds::kPart + t * Lds::kPitch + slab_c) = w;
                };
                split8(xx[n], sx, hi, lo);
                put(0, hi), put(1, lo);
                split8(xe[n], se, hi, lo);
                put(2, hi), put(3, lo);
                split8(xo[n], so, hi, lo);
                put(4, hi);
                if constexpr (PIECES == 2)
                    put(5, lo);
            }
            __syncthreads();
            const int v1 = v0 + Lds::kSlab;
            if (v1 < Dv)
                load_slab(v1);
            auto frag = [&](int part, int tile, int b) {
                return *reinterpret_cast<const u32x4 *>(parts + part * Lds::kPart + (16 * tile + row) * Lds::kPitch + 32 * b +
                                                        8 * grp);
            };
#pragma unroll
            for (int tw = 0; tw < TW; ++tw) {
                const int t = wave + WAVES * tw;
                if (t >= DT)
                    continue;
                float s_max = 0.f, d_max = 0.f;
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    s_max = sv[b].largest(s_max), d_max = dv[b].largest(d_max);
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        both = fmaf(sv[b][k], dv[b][k], both);
                }
                float s_inv, d_inv;
                const float s_scale = scale_of(column_max(s_max), s_inv), d_scale = scale_of(column_max(d_max), d_inv);
                u32x4 s_hi[2], s_lo[2], d_hi[2], d_lo[2];
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    split8(sv[b], s_scale, s_hi[b], s_lo[b]);
                    split8(dv[b], d_scale, d_hi[b], d_lo[b]);
                }
                if (t + WAVES < DT)
                    load_states(v0, t + WAVES);
                else if (v1 < Dv)
                    load_states(v1, wave);
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    __builtin_amdgcn_sched_barrier(0);  // (one tile's operands at a time: registers)
                    f32x4 a = zero, z = zero, w = zero;
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        if constexpr (PIECES == 2)
                            __builtin_amdgcn_sched_barrier(0);
                        const u32x4 fo = frag(4, m, b), fx = frag(0, m, b), fxl = frag(1, m, b), fe = frag(2, m, b),
                                    fel = frag(3, m, b);
                        a = mfma16(fo, s_hi[b], a);
                        z = mfma16(fx, s_hi[b], z);
                        w = mfma16(fe, d_hi[b], w);
                        a = mfma16(fo, s_lo[b], a);
                        z = mfma16(fx, s_lo[b], z);
                        w = mfma16(fe, d_lo[b], w);
                        if constexpr (PIECES == 2)
                            a = mfma16(frag(5, m, b), s_hi[b], a);
                        z = mfma16(fxl, s_hi[b], z);
                        w = mfma16(fel, d_hi[b], w);
                    }
                    const int i = 16 * m + 4 * grp;
                    os[tw][m] += a * (load4(inv_o + i) * s_inv);
                    xs[tw][m] += z * (load4(inv_x + i) * s_inv);
                    ed[tw][m] += w * (load4(inv_e + i) * d_inv);
                }
            }
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                const int tile = wave + WAVES * n;  // (0,0) (1,0) (1,1) (2,0) ...
                if (tile >= 10)
                    continue;
                const int ti = tile >= 6 ? 3 : tile >= 3 ? 2 : tile >= 1 ? 1 : 0, tj = tile - ti * (ti + 1) / 2;
                f32x4 a = zero, z = zero;
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const u32x4 fo = frag(4, ti, b), fx = frag(0, ti, b), fe = frag(2, tj, b), fel = frag(3, tj, b);
                    a = mfma16(fo, fe, a);
                    z = mfma16(fx, fe, z);
                    a = mfma16(fo, fel, a);
                    z = mfma16(fx, fel, z);
                    if constexpr (PIECES == 2)
                        a = mfma16(frag(5, ti, b), fe, a);
                    z = mfma16(frag(1, ti, b), fe, z);
                }
                const float ie = inv_e[16 * tj + row];
                r1[n] += a * (load4(inv_o + 16 * ti + 4 * grp) * ie);
                r2[n] += z * (load4(inv_x + 16 * ti + 4 * grp) * ie);
            }
        }
        asm volatile("" : "+v"(lane));
        row = lane & 15, grp = lane >> 4;
        const float *p = work.p + record * C * C, *bl = work.bl + record * C * C;
        float p_ij[NR][4], bl_ij[NR][4];
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            const int tile = min(wave + WAVES * n, 9);
            const int ti = tile >= 6 ? 3 : tile >= 3 ? 2 : tile >= 1 ? 1 : 0, tj = tile - ti * (ti + 1) / 2;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int place = (16 * ti + 4 * grp + r) * C + 16 * tj + row;
                p_ij[n][r] = p[place], bl_ij[n][r] = bl[place];
            }
        }
        both = row_sum(both);
        both += __shfl_xor(both, 16);
        both += __shfl_xor(both, 32);
        if (lane == 0)
            state_dot[wave] = both;

        // with the rows of Q and K: what e^gamma and e^(gamma_C - gamma) multiply
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            __builtin_amdgcn_sched_barrier(0);
            const int i = 16 * m + 4 * grp;
            const f32x4 gr = load4(grow + i), le = load4(left + i) * load4(beta_s + i);
            const f32x4 ik = load4(inv_k + i), iq = load4(inv_q + i);
            f32x4 q_dot = zero, x_dot = zero, e_dot = zero;
#pragma unroll
            for (int tw = 0; tw < TW; ++tw) {
                const int t = wave + WAVES * tw;
                if (t >= DT)
                    continue;
                const int place = (16 * t + row) * kPitchT + operand_at(i);
                f32x4 qv = zero, kv = zero;
#pragma unroll
                for (int p = 0; p < PIECES; ++p)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        kv[r] += static_cast<float>(__builtin_bit_cast(_Float16, kt[p * Lds::kCols + place + r]));
                        qv[r] += static_cast<float>(__builtin_bit_cast(_Float16, qt[p * Lds::kCols + place + r]));
                    }
                q_dot += qv * os[tw][m];
                x_dot += kv * xs[tw][m];
                e_dot += kv * ed[tw][m];
                sum_q[tw][m] += (job.scale * gr) * os[tw][m];
                sum_k[tw][m] += le * ed[tw][m] - gr * xs[tw][m];
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float a = row_sum(q_dot[r] * iq[r]), b = row_sum(x_dot[r] * ik[r]), w = row_sum(e_dot[r] * ik[r]);
                if (row == 0)
                    dots[0][wave][i + r] = a, dots[1][wave][i + r] = b, dots[2][wave][i + r] = w;
            }
        }

        // R1 and R2 with L: dA, dB, and their sums
        float a_max = 0.f, t_max = 0.f, b_max = 0.f;
        // from here on r1 is dA and r2 dB, without the scales of K and Q
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            const int tile = wave + WAVES * n;
            if (tile >= 10)
                continue;
            const int ti = tile >= 6 ? 3 : tile >= 3 ? 2 : tile >= 1 ? 1 : 0, tj = tile - ti * (ti + 1) / 2;
            const int j = 16 * tj + row;
            float of_cols = 0.f;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * ti + 4 * grp + r;
                float a = 0.f, b = 0.f, both_ij = 0.f;
                if (i >= j) {
                    const float decay = decay_of(gam[i] - gam[j]) * beta_s[j];
                    a = job.scale * decay * r1[n][r];
                    b = i > j ? -decay * r2[n][r] : 0.f;
                    both_ij = p_ij[n][r] * r1[n][r] - bl_ij[n][r] * r2[n][r];
                    if (i == j)
                        diag[i] = both_ij, both_ij = 0.f;
                }
                of_cols += both_ij;
                const float of_rows = row_sum(both_ij * beta_s[j]);
                if (row == 0)
                    rows[tj][i] = of_rows;
                r1[n][r] = a, r2[n][r] = b;
                a_max = fmaxf(a_max, fabsf(a * inv_k[j]));
                t_max = fmaxf(t_max, fabsf(a * inv_q[i]));
                b_max = fmaxf(b_max, fmaxf(fabsf(b * inv_k[j]), fabsf(b * inv_k[i])));
            }
            of_cols += __shfl_xor(of_cols, 16);
            of_cols += __shfl_xor(of_cols, 32);
            if (grp == 0)
                cols[ti][j] = of_cols;
        }
#pragma unroll
        for (int k = 1; k < 16; k <<= 1) {
            a_max = fmaxf(a_max, __shfl_xor(a_max, k));
            t_max = fmaxf(t_max, __shfl_xor(t_max, k));
            b_max = fmaxf(b_max, __shfl_xor(b_max, k));
        }
        a_max = column_max(a_max), t_max = column_max(t_max), b_max = column_max(b_max);
        if (lane == 0)
            largest[0][wave] = a_max, largest[1][wave] = t_max, largest[2][wave] = b_max;
        __syncthreads();
        if (wave == 0) {
            float strict = 0.f, of_rows = 0.f;
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                strict += m >= lane / 16 ? cols[m][lane] : 0.f;
                of_rows += m <= lane / 16 ? rows[m][lane] : 0.f;
            }
            float q_dot = 0.f, x_dot = 0.f, e_dot = 0.f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w)
                q_dot += dots[0][w][lane], x_dot += dots[1][w][lane], e_dot += dots[2][w][lane];
            const float beta = beta_s[lane], last = left[lane] * e_dot, held = beta * last;
            const float own = grow[lane] * (job.scale * q_dot - x_dot);
            // decays' sums from the end: 64 bits, their terms cancel
            double part = static_cast<double>(own) + static_cast<double>(of_rows) - static_cast<double>(beta * strict) -
                          static_cast<double>(held);
            double all = held;
#pragma unroll
            for (int m = 1; m < kWave; m <<= 1) {
                const double y = __shfl_down(part, m);
                part += lane + m < kWave ? y : 0.0;
                all += __shfl_xor(all, m);
            }
            double both_all = 0.0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w)
                both_all += static_cast<double>(state_dot[w]);
            all += static_cast<double>(grow[C - 1]) * both_all;
            if (lane < at.len) {
                const int64_t out = (token0 + lane) * job.Hv + head;
                store_code(grads.dg, job.g_dtype, out, static_cast<float>(part + all));
                store_code(grads.dbeta, job.beta_dtype, out, strict + diag[lane] + last);
            }
        }
        // dA, dA^T and dB + dB^T as operands, K's and Q's scales taken out of their columns
        float a_inv, t_inv, b_inv;
        auto all_max = [&](int k) {
            float m = largest[k][0];
#pragma unroll
            for (int w = 1; w < WAVES; ++w)
                m = fmaxf(m, largest[k][w]);
            return m;
        };
        const float a_scale = scale_of(all_max(0), a_inv), t_scale = scale_of(all_max(1), t_inv),
                    b_scale = scale_of(all_max(2), b_inv);
        auto put = [&](int matrix, int i, int j, float v, float scale) {
            const _Float16 hi = static_cast<_Float16>(v * scale);
            uint16_t *to = parts + matrix * Lds::kPart + i * Lds::kPitch + j;
            *to = __builtin_bit_cast(uint16_t, hi);
            to[3 * Lds::kPart] = __builtin_bit_cast(uint16_t, static_cast<_Float16>(fmaf(v, scale, -static_cast<float>(hi))));
        };
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            const int tile = wave + WAVES * n;
            if (tile >= 10)
                continue;
            const int ti = tile >= 6 ? 3 : tile >= 3 ? 2 : tile >= 1 ? 1 : 0, tj = tile - ti * (ti + 1) / 2;
            const int j = 16 * tj + row;
            // places of row i, and of column i in row j: positions of operands
            const int at_j = operand_at(j), at_i = operand_at(16 * ti + 4 * grp);
            const float kj = inv_k[j];
            const f32x4 ki = load4(inv_k + 16 * ti + 4 * grp), qi = load4(inv_q + 16 * ti + 4 * grp);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * ti + 4 * grp + r;
                const float a = r1[n][r], b = r2[n][r];
                put(0, i, at_j, a * kj, a_scale);
                put(1, j, at_i + r, a * qi[r], t_scale);
                // (on the diagonal the upper half is the lower's mirror: what is not below goes to a row's padding)
                put(2, i, ti != tj || i >= j ? at_j : C, b * kj, b_scale);
                put(2, j, ti != tj || i > j ? at_i + r : C, b * ki[r], b_scale);
                if (ti != tj) {
                    put(0, j, at_i + r, 0.f, 0.f);
                    put(1, i, at_j, 0.f, 0.f);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        __syncthreads();
        auto square = [&](int matrix, int tile, int b) {
            return *reinterpret_cast<const u32x4 *>(parts + matrix * Lds::kPart + (16 * tile + row) * Lds::kPitch + 32 * b +
                                                    8 * grp);
        };
#pragma unroll
        for (int tw = 0; tw < TW; ++tw) {
            const int t = wave + WAVES * tw;
            if (t >= DT)
                continue;
            u32x4 kf[PIECES][2], qf[PIECES][2];
#pragma unroll
            for (int n = 0; n < PIECES; ++n)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const int place = n * Lds::kCols + (16 * t + row) * kPitchT + 32 * b + 8 * grp;
                    kf[n][b] = *reinterpret_cast<const u32x4 *>(kt + place);
                    qf[n][b] = *reinterpret_cast<const u32x4 *>(qt + place);
                }
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                __builtin_amdgcn_sched_barrier(0);
                f32x4 a = zero, z = zero, w = zero;
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    auto product = [&](int matrix, const u32x4 (&f)[PIECES][2], f32x4 acc) {
                        const u32x4 hi = square(matrix, m, b);
                        acc = mfma16(hi, f[0][b], acc);
                        acc = mfma16(square(matrix + 3, m, b), f[0][b], acc);
                        if constexpr (PIECES == 2)
                            acc = mfma16(hi, f[PIECES - 1][b], acc);
                        return acc;
                    };
                    if (b <= m / 2)
                        a = product(0, kf, a);
                    if (b >= m / 2)
                        z = product(1, qf, z);
                    w = product(2, kf, w);
                }
                sum_q[tw][m] += a * a_inv;
                sum_k[tw][m] += z * t_inv + w * b_inv;
            }
        }
    }
#pragma unroll
    for (int tw = 0; tw < TW; ++tw) {
        const int t = wave + WAVES * tw;
        if (t >= DT)
            continue;
        const Columns<Scalar> to(dk_step, Dk, grp, 16 * t + row);
        const auto q_rows = to.rows(dq + token0 * dk_step, at.len), k_rows = to.rows(dk + token0 * dk_step, at.len);
        to.template each<4>([&](int m, int r, int place) {
            buffer_store<Scalar>(sum_q[tw][m][r], q_rows, place);
            buffer_store<Scalar>(sum_k[tw][m][r], k_rows, place);
        });
    }
}

// Whether a chunk's operands and the gradients' products fit the LDS.
template<int DT, int PIECES>
constexpr bool kTrains = ChunkLds<DT, PIECES, true>::kBytes <= kLdsBytes &&
                              BackLds<DT, PIECES>::kBytes + 12288 <= kLdsBytes;
static_assert(kTrains<16, 1> && kTrains<10, 2> && !kTrains<16, 2>);  // as delta_trains has it

template<typename Scalar>
hipError_t backward_typed(const DeltaJob &job, const DeltaWork &work, const DeltaGrads &grads, hipStream_t stream,
                          const char **why) {
    const int wide = delta_padded(job.Dk);
    const int tiles = (job.Dv + 15) / 16, groups = (tiles + 3) / 4;
    const int64_t lines = static_cast<int64_t>(job.N) * job.Hv;
    if (lines * work.parts * groups > 0x7fffffff || lines * tiles > 0x7fffffff) {
        *why = "delta rule: too many state columns for one launch";
        return hipErrorInvalidValue;
    }
    const dim3 part_grid(static_cast<unsigned>(lines * (work.parts - 1) * groups));
    const dim3 grid(static_cast<unsigned>(lines * work.parts * groups));
    constexpr int PIECES = sizeof(Scalar) == 4 ? 2 : 1;
    constexpr int V = 16 / static_cast<int>(sizeof(Scalar));
    const bool pieces = rows_whole<Scalar>(job) && job.Dv % V == 0 && reinterpret_cast<uintptr_t>(grads.d_o) % 16 == 0 &&
                        (grads.d_o_at[0] | grads.d_o_at[1] | grads.d_o_at[2]) % V == 0;
#define RAMNET_BACK(DT)                                                                                                         \
    if constexpr (kTrains<DT, PIECES>) {                                                                                        \
        if (wide == 16 * DT) {                                                                                                  \
            constexpr int each = ChunkLds<DT, PIECES, true>::kBytes, bufs = 2 * each <= kLdsBytes ? 2 : 1;                      \
            constexpr int back = BackLds<DT, PIECES>::kBytes;                                                                   \
            if (work.parts > 1) {                                                                                               \
                hipLaunchKernelGGL((chain_back_kernel<Scalar, DT, PIECES, bufs, true>), part_grid, dim3(512), bufs * each,      \
                                   stream, job, work, grads, groups);                                                           \
                if (const hipError_t err = launch_delta_join(job, work, true, stream))                                          \
                    return err;                                                                                                 \
            }                                                                                                                   \
            hipLaunchKernelGGL((chain_back_kernel<Scalar, DT, PIECES, bufs, false>), grid, dim3(512), bufs * each, stream,      \
                               job, work, grads, groups);                                                                       \
            if (const hipError_t err = hipGetLastError())                                                                       \
                return err;                                                                                                     \
            constexpr int waves = DT == 2 || (DT <= 8 && PIECES == 1) ? 8 : 4;                                                  \
            const dim3 in_grid(work.chunks, job.Hk), in_block(kWave * waves);                                                   \
            if (pieces)                                                                                                         \
                hipLaunchKernelGGL((inputs_back_kernel<Scalar, DT, PIECES, true, waves>), in_grid, in_block, back, stream,      \
                                   job, work, grads);                                                                           \
            else                                                                                                                \
                hipLaunchKernelGGL((inputs_back_kernel<Scalar, DT, PIECES, false, waves>), in_grid, in_block, back, stream,     \
                                   job, work, grads);                                                                           \
        }                                                                                                                       \
    }
    RAMNET_BACK(2)
    RAMNET_BACK(4)
    RAMNET_BACK(6)
    RAMNET_BACK(8)
    RAMNET_BACK(10)
    RAMNET_BACK(16)
#undef RAMNET_BACK
    return hipGetLastError();
}

}  // namespace

hipError_t launch_delta_backward(const DeltaJob &job, const DeltaWork &work, const DeltaGrads &grads, hipStream_t stream,
                                 const char **why) {
    switch (job.dtype) {
        case kF32: return backward_typed<float>(job, work, grads, stream, why);
        case kF16: return backward_typed<_Float16>(job, work, grads, stream, why);
        case kBF16: return backward_typed<bf16_t>(job, work, grads, stream, why);
        default: *why = "delta rule: unsupported dtype"; return hipErrorInvalidValue;
    }
}

}  // namespace ramnet
