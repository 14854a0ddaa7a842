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
template<typename Scalar, int DT, int PIECES, int BUFS>
__global__ __launch_bounds__(512, 2) void chain_back_kernel(const DeltaJob job, const DeltaWork work,
                                                            const DeltaGrads grads, int groups) {
    extern __shared__ __align__(16) float lds_base[];
    using Lds = ChunkLds<DT, PIECES, true>;
    constexpr int C = kDeltaChunk, BT = DT / 2;
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave, wave = tid / kWave;
    const int row = lane & 15, grp = lane >> 4;
    const int group = static_cast<int>(blockIdx.x) % groups;
    const int head = static_cast<int>(blockIdx.x) / groups % job.Hv;
    const int n = static_cast<int>(blockIdx.x) / groups / job.Hv;
    const int kh = head / (job.Hv / job.Hk);
    const DeltaSpan span = delta_span(job, n);
    int first, count;
    delta_chunks(job, work, n, span, first, count);
    auto buffer = [&](int i) {
        return Lds{reinterpret_cast<uint16_t *>(reinterpret_cast<char *>(lds_base) + (BUFS == 2 ? (i & 1) * Lds::kBytes : 0))};
    };

    if (wave >= 4) {
        const int at = tid - 256;
        const bool whole = rows_whole<Scalar>(job);
        const Scalar *k = static_cast<const Scalar *>(job.k) + span.b * job.k_at[0] + kh * job.k_at[2];
        const Scalar *q = static_cast<const Scalar *>(job.q) + span.b * job.q_at[0] + kh * job.q_at[2];
        Stager<Scalar, DT, PIECES, true> stager;
        auto load = [&](int i) {
            const int64_t t0 = span.t0 + i * C;
            stager.load(k + t0 * job.k_at[1], job.k_at[1], q + t0 * job.q_at[1], job.q_at[1], min(C, span.len - i * C),
                        job.Dk, whole, work.vec + (static_cast<int64_t>(first + i) * job.Hv + head) * kVecs * C, at);
        };
        if (count > 0) {
            load(count - 1);
            stager.store(buffer(count - 1), at);
        }
        __syncthreads();
        for (int i = count - 1; i >= 0; --i) {
            if (i > 0)
                load(i - 1);
            if constexpr (BUFS == 1)
                __syncthreads();  // chunk i is done with
            if (i > 0)
                stager.store(buffer(i - 1), at);
            __syncthreads();
        }
        return;
    }

    const int c = (group * 4 + wave) * 16 + row;
    const int64_t matrix = (static_cast<int64_t>(n) * job.Hv + head) * job.Dk * job.Dv;
    const Columns<float> state(job.Dv, job.Dv, grp, c);
    f32x4 s[DT];
    {
        const auto from = state.rows(grads.d_state + matrix, grads.d_state ? job.Dk : 0);
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
    }
    __syncthreads();

    for (int i = count - 1; i >= 0; --i) {
        const int64_t record = static_cast<int64_t>(first + i) * job.Hv + head;
        const Lds lds = buffer(i);
        const float *vec = lds.vec();
        const float total = vec[kVecGrowK * C + C - 1] * vec[kVecSk * C + C - 1];  // (a power of two: e^gamma_C)
        {
            const auto to = state.rows(work.dstate + record * job.Dk * job.Dv, job.Dk);
            state.each<DT>([&](int t, int r, int at) { buffer_store<float>(s[t][r], to, at); });
        }
        f32x4 out[4], du[4], x[4];
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                out[m][r] = bits_f32<Scalar>(o_bits[4 * m + r]);
        if (i > 0)
            load_o(i - 1);
        {
            Operand<4, true> oo;
            oo.set(out);
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                x[m] = zero;
#pragma unroll
                for (int b = m / 2; b < 2; ++b) {
                    const int f = m < 2 ? m * 2 + b : m + 2;
                    x[m] = mfma16(p_hi[f], oo.hi[b], x[m]);
                    x[m] = mfma16(p_lo[f], oo.hi[b], x[m]);
                    if constexpr (!__is_same(Scalar, bf16_t))
                        x[m] = mfma16(p_hi[f], oo.lo[b], x[m]);  // (0 for bf16 but far below a column's largest)
                }
                x[m] = x[m] * (load4(vec + kVecInvP * C + 16 * m + 4 * grp) * oo.inverse);
            }
            if (i > 0)
                load_frags(work.p_frags, i - 1, p_hi, p_lo);
        }
        {
            Operand<DT, true> so;
            so.set(s);
#pragma unroll
            for (int m = 0; m < 4; ++m)
                du[m] = zero;
#pragma unroll
            for (int b = 0; b < BT; ++b) {
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    const u32x4 kf = lds.row_frag(lds.k(0), m, b, lane);
                    du[m] = mfma16(kf, so.hi[b], du[m]);
                    du[m] = mfma16(kf, so.lo[b], du[m]);
                    if constexpr (PIECES == 2)
                        du[m] = mfma16(lds.row_frag(lds.k(1), m, b, lane), so.hi[b], du[m]);
                }
            }
#pragma unroll
            for (int m = 0; m < 4; ++m)
                du[m] = (x[m] + du[m] * (load4(vec + kVecLeftK * C + 16 * m + 4 * grp) * so.inverse)) *
                        load4(vec + kVecBeta * C + 16 * m + 4 * grp);
        }
        {
            Operand<4, true> uo;
            uo.set(du);
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                x[m] = zero;
#pragma unroll
                for (int b = m / 2; b < 2; ++b) {
                    const int f = m < 2 ? m * 2 + b : m + 2;
                    x[m] = mfma16(y_hi[f], uo.hi[b], x[m]);
                    x[m] = mfma16(y_hi[f], uo.lo[b], x[m]);
                    x[m] = mfma16(y_lo[f], uo.hi[b], x[m]);
                }
                x[m] = x[m] * (load4(vec + kVecInvY * C + 16 * m + 4 * grp) * uo.inverse);
            }
            if (i > 0)
                load_frags(work.y, i - 1, y_hi, y_lo);
        }
        {
            const auto to = state.rows(work.x + record * C * job.Dv, C);
            state.each<4>([&](int m, int r, int at) { buffer_store<float>(x[m][r], to, at); });
            const auto out_to = v_cols.rows(dv + static_cast<int64_t>(i) * C * dv_step, min(C, span.len - i * C));
            v_cols.template each<4>([&](int m, int r, int at) { buffer_store<Scalar>(x[m][r], out_to, at); });
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            x[m] = -(load4(vec + kVecGrowK * C + 16 * m + 4 * grp) * x[m]);
            out[m] = out[m] * load4(vec + kVecGrowQ * C + 16 * m + 4 * grp);
        }
        Operand<4, true> xo, oo;
        xo.set(x);
        oo.set(out);
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
    if (grads.dinit) {
        const auto to = state.rows(grads.dinit + matrix, job.Dk);
        state.each<DT>([&](int t, int r, int at) { buffer_store<float>(s[t][r], to, at); });
    }
    if (!job.cu && c < job.Dv)  // tokens that do not count
        for (int64_t t = span.len + grp; t < job.T; t += 4)
            store_f32(dv + t * dv_step + c, 0.f);
}

// Sum over the 16 lanes of a row group.
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
    for (int m = 1; m < 16; m <<= 1)
        x += __shfl_xor(x, m);
    return x;
}

__device__ __forceinline__ void store_code(void *p, int code, int64_t at, float v) {
    if (code == 0)
        static_cast<float *>(p)[at] = v;
    else if (code == 1)
        store_f32(static_cast<_Float16 *>(p) + at, v);
    else
        store_f32(static_cast<bf16_t *>(p) + at, v);
}

// The other gradients of one chunk and key head; its value heads one after the
// other, so that a shared head's sums have one order. Wave w has the tokens of
// tile w.
template<typename Scalar, int DT>
__global__ __launch_bounds__(256) void inputs_back_kernel(const DeltaJob job, const DeltaWork work,
                                                          const DeltaGrads grads) {
    extern __shared__ __align__(16) float lds[];
    constexpr int C = kDeltaChunk, wide = 16 * DT, pitch = wide + 4, NP = C + 4;
    float *ks = lds, *qs = ks + C * pitch, *da = qs + C * pitch, *db = da + C * NP;
    __shared__ double gam[C];
    __shared__ float beta_s[C], grow[C], left[C], rows[C], cols[4][C], diag[C], dots[C], state_dot[4];
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave, wave = tid / kWave;
    const int row = lane & 15, grp = lane >> 4;
    const int chunk = blockIdx.x, kh = blockIdx.y, shared = job.Hv / job.Hk;
    const DeltaPlace at = delta_place(job, work, chunk);
    const int Dk = job.Dk, Dv = job.Dv;
    const int64_t dk_step = static_cast<int64_t>(job.Hk) * Dk;
    Scalar *dq = static_cast<Scalar *>(grads.dq) + static_cast<int64_t>(kh) * Dk;
    Scalar *dk = static_cast<Scalar *>(grads.dk) + static_cast<int64_t>(kh) * Dk;
    // tokens of no sequence or past a row's length
    auto clear = [&](int64_t from, int64_t to) {
        for (int64_t t = from; t < to; ++t) {
            for (int d = tid; d < Dk; d += 256) {
                store_f32(dq + t * dk_step + d, 0.f);
                store_f32(dk + t * dk_step + d, 0.f);
            }
            for (int h = tid; h < shared; h += 256) {
                store_code(grads.dg, job.g_dtype, t * job.Hv + kh * shared + h, 0.f);
                store_code(grads.dbeta, job.beta_dtype, t * job.Hv + kh * shared + h, 0.f);
            }
            if (job.cu)
                for (int i = tid; i < shared * Dv; i += 256)
                    store_f32(static_cast<Scalar *>(grads.dv) + (t * job.Hv + kh * shared) * Dv + i, 0.f);
        }
    };
    if (job.cu) {
        if (at.n < 0) {
            if (chunk == work.offsets[job.N]) {
                const int start = delta_span(job, 0).t0;
                const DeltaSpan last = delta_span(job, job.N - 1);
                clear(0, start);
                clear(max(start, last.t0 + last.len), job.T);
            }
            return;
        }
    } else if (at.len < C) {
        const int64_t base = static_cast<int64_t>(at.b) * job.T;
        clear(base + at.t0 + at.len, base + min(at.t0 + C, job.T));
    }
    if (at.len == 0)
        return;

    stage_rows(static_cast<const Scalar *>(job.k) + at.b * job.k_at[0] + at.t0 * job.k_at[1] + kh * job.k_at[2],
               job.k_at[1], at.len, Dk, wide, ks, pitch);
    stage_rows(static_cast<const Scalar *>(job.q) + at.b * job.q_at[0] + at.t0 * job.q_at[1] + kh * job.q_at[2],
               job.q_at[1], at.len, Dk, wide, qs, pitch);
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    f32x4 sum_q[DT], sum_k[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
        sum_q[t] = sum_k[t] = zero;
    const int64_t token0 = static_cast<int64_t>(at.b) * job.T + at.t0;

    for (int h = 0; h < shared; ++h) {
        const int head = kh * shared + h;
        const int64_t record = static_cast<int64_t>(chunk) * job.Hv + head;
        __syncthreads();
        if (wave == 0) {
            const double own = work.gamma[record * C + lane], end = work.gamma[record * C + C - 1];
            gam[lane] = own;
            grow[lane] = expf(static_cast<float>(own));
            left[lane] = expf(static_cast<float>(end - own));
            beta_s[lane] = lane < at.len ? load_code(job.beta, job.beta_dtype, at.b * job.beta_at[0] +
                                                     static_cast<int64_t>(at.t0 + lane) * job.beta_at[1] +
                                                     head * job.beta_at[2]) : 0.f;
        }
        __syncthreads();
        const float *e = work.e + record * C * Dv, *x = work.x + record * C * Dv;
        const float *s = work.states + record * Dk * Dv, *d = work.dstate + record * Dk * Dv;
        const Scalar *d_o = static_cast<const Scalar *>(grads.d_o) + at.b * grads.d_o_at[0] +
                            at.t0 * grads.d_o_at[1] + head * grads.d_o_at[2];

        // dO S^T, X S^T, E D^T (rows: this wave's tokens) and R1, R2, over Dv
        const int tok = 16 * wave + row;
        auto of_row = [&](const float *src, int at_row, int rows_there, int v) {
            f32x4 f = zero;
            if (at_row < rows_there) {
                const float *from = src + static_cast<int64_t>(at_row) * Dv + v;
                if (v + 4 <= Dv && Dv % 4 == 0)
                    f = load4(from);
                else
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        f[r] = v + r < Dv ? from[r] : 0.f;
            }
            return f;
        };
        f32x4 os[DT], xs[DT], ed[DT], r1[4], r2[4];
#pragma unroll
        for (int t = 0; t < DT; ++t)
            os[t] = xs[t] = ed[t] = zero;
#pragma unroll
        for (int m = 0; m < 4; ++m)
            r1[m] = r2[m] = zero;
        float both = 0.f;
        for (int v = 4 * grp; v < (Dv + 15) / 16 * 16; v += 16) {
            f32x4 ao = zero;
            if (tok < at.len)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    ao[r] = v + r < Dv ? load_f32(d_o + tok * grads.d_o_at[1] + v + r) : 0.f;
            const f32x4 ax = of_row(x, tok, C, v), ae = of_row(e, tok, C, v);
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                const f32x4 bs = of_row(s, 16 * t + row, Dk, v), bd = of_row(d, 16 * t + row, Dk, v);
                os[t] = mfma4(ao, bs, os[t]);
                xs[t] = mfma4(ax, bs, xs[t]);
                ed[t] = mfma4(ae, bd, ed[t]);
                if (t % 4 == wave)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        both = fmaf(bs[r], bd[r], both);
            }
#pragma unroll
            for (int m = 0; m < 4; ++m)
                if (m <= wave) {
                    const f32x4 be = of_row(e, 16 * m + row, C, v);
                    r1[m] = mfma4(ao, be, r1[m]);
                    r2[m] = mfma4(ax, be, r2[m]);
                }
        }
        both = row_sum(both);
        both += __shfl_xor(both, 16);
        both += __shfl_xor(both, 32);
        if (lane == 0)
            state_dot[wave] = both;

        // with the rows of Q and K: what e^gamma and e^(gamma_C - gamma) multiply
        const f32x4 gr = load4(grow + 16 * wave + 4 * grp), le = load4(left + 16 * wave + 4 * grp);
        const f32x4 be = load4(beta_s + 16 * wave + 4 * grp);
        f32x4 q_dot = zero, x_dot = zero, e_dot = zero;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float kv = ks[(16 * wave + 4 * grp + r) * pitch + 16 * t + row];
                const float qv = qs[(16 * wave + 4 * grp + r) * pitch + 16 * t + row];
                q_dot[r] = fmaf(qv, os[t][r], q_dot[r]);
                x_dot[r] = fmaf(kv, xs[t][r], x_dot[r]);
                e_dot[r] = fmaf(kv, ed[t][r], e_dot[r]);
                sum_q[t][r] = fmaf(job.scale * gr[r], os[t][r], sum_q[t][r]);
                sum_k[t][r] += le[r] * be[r] * ed[t][r] - gr[r] * xs[t][r];
            }
        f32x4 own = zero, last = zero;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            own[r] = gr[r] * (job.scale * row_sum(q_dot[r]) - row_sum(x_dot[r]));
            last[r] = le[r] * row_sum(e_dot[r]);
        }

        // R1 and R2 with L: dA, dB, and their sums
        const float *p = work.p + record * C * C, *bl = work.bl + record * C * C;
        f32x4 of_rows = zero;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            float of_cols = 0.f;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * wave + 4 * grp + r, j = 16 * m + row;
                float a = 0.f, b = 0.f, both_ij = 0.f;
                if (i >= j) {
                    const float decay = expf(static_cast<float>(gam[i] - gam[j])) * beta_s[j];
                    a = job.scale * decay * r1[m][r];
                    b = i > j ? -decay * r2[m][r] : 0.f;
                    both_ij = p[i * C + j] * r1[m][r] - bl[i * C + j] * r2[m][r];
                    if (i == j)
                        diag[i] = both_ij;
                    else
                        of_cols += both_ij;
                }
                da[i * NP + j] = a;
                db[i * NP + j] = b;
                of_rows[r] += i > j ? both_ij * beta_s[j] : 0.f;
            }
            of_cols += __shfl_xor(of_cols, 16);
            of_cols += __shfl_xor(of_cols, 32);
            if (grp == 0)
                cols[wave][16 * m + row] = of_cols;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float sum = row_sum(of_rows[r]);
            if (row == 0) {
                rows[16 * wave + 4 * grp + r] = own[r] + sum;
                dots[16 * wave + 4 * grp + r] = last[r];
            }
        }
        __syncthreads();
        if (wave == 0) {
            const float strict = cols[0][lane] + cols[1][lane] + cols[2][lane] + cols[3][lane];
            const float beta = beta_s[lane];
            const float h = beta * dots[lane];
            // decays' sums from the end: 64 bits, their terms cancel
            double part = static_cast<double>(rows[lane]) - static_cast<double>(beta * strict) - static_cast<double>(h);
            double all = h;
#pragma unroll
            for (int m = 1; m < kWave; m <<= 1) {
                const double y = __shfl_down(part, m);
                part += lane + m < kWave ? y : 0.0;
                all += __shfl_xor(all, m);
            }
            all += static_cast<double>(grow[C - 1]) *
                   (static_cast<double>(state_dot[0]) + state_dot[1] + state_dot[2] + state_dot[3]);
            if (lane < at.len) {
                const int64_t out = (token0 + lane) * job.Hv + head;
                store_code(grads.dg, job.g_dtype, out, static_cast<float>(part + all));
                store_code(grads.dbeta, job.beta_dtype, out, strict + diag[lane] + dots[lane]);
            }
        }
        // dA K, dA^T Q, (dB + dB^T) K
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const f32x4 qa = load4(da + (16 * wave + row) * NP + 16 * j + 4 * grp);
            const f32x4 ka = load4(db + (16 * wave + row) * NP + 16 * j + 4 * grp);
            const f32x4 qt = load4(da + (16 * j + 4 * grp) * NP + 16 * wave + row, NP);
            const f32x4 kt = ka + load4(db + (16 * j + 4 * grp) * NP + 16 * wave + row, NP);
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                const f32x4 kb = load4(ks + (16 * j + 4 * grp) * pitch + 16 * t + row, pitch);
                sum_q[t] = mfma4(qa, kb, sum_q[t]);
                sum_k[t] = mfma4(kt, kb, sum_k[t]);
                sum_k[t] = mfma4(qt, load4(qs + (16 * j + 4 * grp) * pitch + 16 * t + row, pitch), sum_k[t]);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = 16 * wave + 4 * grp + r, d = 16 * t + row;
            if (i < at.len && d < Dk) {
                store_f32(dq + (token0 + i) * dk_step + d, sum_q[t][r]);
                store_f32(dk + (token0 + i) * dk_step + d, sum_k[t][r]);
            }
        }
}

template<typename Scalar>
hipError_t backward_typed(const DeltaJob &job, const DeltaWork &work, const DeltaGrads &grads, hipStream_t stream,
                          const char **why) {
    constexpr int C = kDeltaChunk;
    const int wide = job.Dk <= 32 ? 32 : job.Dk <= 64 ? 64 : job.Dk <= 96 ? 96 : job.Dk <= 128 ? 128
                     : job.Dk <= 160 ? 160 : 256;
    const int groups = (job.Dv + 63) / 64;
    const int64_t blocks = static_cast<int64_t>(job.N) * job.Hv * groups;
    if (blocks > 0x7fffffff) {
        *why = "delta rule: too many state columns for one launch";
        return hipErrorInvalidValue;
    }
    constexpr int PIECES = sizeof(Scalar) == 4 ? 2 : 1;
    const size_t bytes = (2 * C * (wide + 4) + 2 * C * (C + 4)) * sizeof(float);
#define RAMNET_BACK(DT)                                                                                              \
    if (wide == 16 * DT) {                                                                                           \
        constexpr int each = ChunkLds<DT, PIECES, true>::kBytes, bufs = 2 * each <= kLdsBytes ? 2 : 1;               \
        static_assert(each <= kLdsBytes);                                                                            \
        hipLaunchKernelGGL((chain_back_kernel<Scalar, DT, PIECES, bufs>), dim3(static_cast<unsigned>(blocks)),       \
                           dim3(512), bufs * each, stream, job, work, grads, groups);                                \
        if (const hipError_t err = hipGetLastError())                                                                \
            return err;                                                                                              \
        hipLaunchKernelGGL((inputs_back_kernel<Scalar, DT>), dim3(work.chunks, job.Hk), dim3(256), bytes, stream,    \
                           job, work, grads);                                                                        \
    }
    RAMNET_BACK(2)
    RAMNET_BACK(4)
    RAMNET_BACK(6)
    RAMNET_BACK(8)
    RAMNET_BACK(10)
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
