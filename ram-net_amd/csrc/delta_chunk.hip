// Gated delta rule in chunks of 64 tokens: what the chunks' own tokens give
// (prepare), then the states from chunk to chunk (chain).
#include "delta_chunk.hpp"
#include "ramnet_kernels.hpp"

namespace ramnet {

namespace {

// First chunk of each packed sequence, one block. The sum of the lengths is at
// most T where the bounds are in order; elsewhere it is held to the records
// there are.
__global__ __launch_bounds__(1024) void offsets_kernel(const DeltaJob job, const DeltaWork work) {
    __shared__ int wave_sum[16];
    __shared__ int carry;
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave, wave = tid / kWave;
    if (tid == 0)
        carry = 0, work.offsets[0] = 0;
    __syncthreads();
    for (int base = 0; base < job.N; base += 1024) {
        const int n = base + tid;
        int x = n < job.N ? (delta_span(job, n).len + kDeltaChunk - 1) / kDeltaChunk : 0;
#pragma unroll
        for (int m = 1; m < kWave; m <<= 1) {
            const int y = __shfl_up(x, m);
            x += lane >= m ? y : 0;
        }
        if (lane == kWave - 1)
            wave_sum[wave] = x;
        __syncthreads();
        int sum = carry;
        for (int w = 0; w < wave; ++w)
            sum = min(sum + wave_sum[w], work.chunks);
        sum = min(sum + x, work.chunks);
        if (n < job.N)
            work.offsets[n + 1] = sum;
        __syncthreads();
        if (tid == 1023)
            carry = sum;
        __syncthreads();
    }
}

// Y, P and gamma of one chunk and value head. Four waves.
template<typename Scalar>
__global__ __launch_bounds__(256) void prepare_kernel(const DeltaJob job, const DeltaWork work, int wide, bool backward) {
    extern __shared__ __align__(16) float lds[];
    constexpr int C = kDeltaChunk, NP = C + 4;
    const int pitch = wide + 4;
    float *ks = lds, *qs = ks + C * pitch, *nm = qs + C * pitch;
    float *ys = lds;  // (once the keys are done with)
    __shared__ double gam[C];
    __shared__ float beta_s[C];
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave, wave = tid / kWave;
    const int chunk = blockIdx.x, head = blockIdx.y, kh = head / (job.Hv / job.Hk);
    const DeltaPlace at = delta_place(job, work, chunk);
    if (at.len == 0) {
        // a record of no sequence: the tokens that no sequence covers have output 0
        if (at.n < 0 && chunk == work.offsets[job.N] && !backward) {
            const int first = delta_span(job, 0).t0;
            const DeltaSpan last = delta_span(job, job.N - 1);
            Scalar *o = static_cast<Scalar *>(job.o) + static_cast<int64_t>(head) * job.Dv;
            auto clear = [&](int from, int to) {
                for (int64_t t = from; t < to; ++t)
                    for (int c = tid; c < job.Dv; c += blockDim.x)
                        store_f32(o + t * job.Hv * job.Dv + c, 0.f);
            };
            clear(0, first);
            clear(max(first, last.t0 + last.len), job.T);
        }
        return;
    }
    stage_rows(static_cast<const Scalar *>(job.k) + at.b * job.k_at[0] + at.t0 * job.k_at[1] + kh * job.k_at[2],
               job.k_at[1], at.len, job.Dk, wide, ks, pitch);
    stage_rows(static_cast<const Scalar *>(job.q) + at.b * job.q_at[0] + at.t0 * job.q_at[1] + kh * job.q_at[2],
               job.q_at[1], at.len, job.Dk, wide, qs, pitch);
    if (wave == 0) {
        const int64_t t = at.t0 + lane;
        const bool have = lane < at.len;
        double x = have ? delta_decay(load_code(job.g, job.g_dtype, at.b * job.g_at[0] + t * job.g_at[1] + head * job.g_at[2])) : 0.f;
#pragma unroll
        for (int m = 1; m < kWave; m <<= 1) {
            const double y = __shfl_up(x, m);
            x += lane >= m ? y : 0.0;
        }
        gam[lane] = x;
        beta_s[lane] = have ? load_code(job.beta, job.beta_dtype,
                                        at.b * job.beta_at[0] + t * job.beta_at[1] + head * job.beta_at[2]) : 0.f;
        work.gamma[(static_cast<int64_t>(chunk) * job.Hv + head) * C + lane] = x;
    }
    __syncthreads();

    // K K^T and Q K^T, lower tiles; tile pairs go round the waves
    const int row = lane & 15, grp = lane >> 4;
    const int64_t record = static_cast<int64_t>(chunk) * job.Hv + head;
    float *y_out = work.y + record * C * C, *p_out = work.p + record * C * C;
    float *bl_out = backward ? work.bl + record * C * C : nullptr;
    for (int tile = wave; tile < 32; tile += 4) {
        const bool is_p = tile >= 16;
        const int ti = (tile & 15) >> 2, tj = tile & 3;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        if (tj <= ti) {
            const float *a = (is_p ? qs : ks) + (16 * ti + row) * pitch + 4 * grp;
            const float *b = ks + (16 * tj + row) * pitch + 4 * grp;
            for (int d = 0; d < wide; d += 16)
                acc = mfma4(load4(a + d), load4(b + d), acc);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = 16 * ti + 4 * grp + r, j = 16 * tj + row;
            const float decay = i >= j ? expf(static_cast<float>(gam[i] - gam[j])) : 0.f;
            if (is_p) {
                p_out[i * C + j] = i >= j ? job.scale * acc[r] * decay : 0.f;
            } else {
                const float x = i > j ? acc[r] * decay : 0.f;
                nm[i * NP + j] = x * beta_s[j];
                if (bl_out)
                    bl_out[i * C + j] = x;
            }
        }
    }
    __syncthreads();
    for (int i = tid; i < C * NP; i += 256)
        ys[i] = 0.f;
    __syncthreads();

    // inverse of the unit lower triangular N: 16-blocks by substitution (lane = column),
    // then pairs of blocks: low part -Yb Nba Ya
    {
        float x[16];
        const int o = 16 * wave;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float sum = i == row ? 1.f : 0.f;
#pragma unroll
            for (int j = 0; j < i; ++j)
                sum = fmaf(-nm[(o + i) * NP + o + j], x[j], sum);
            x[i] = sum;
        }
        if (grp == 0)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                ys[(o + i) * NP + o + row] = x[i];
    }
    __syncthreads();
    if (wave < 2) {
        const int a = 32 * wave, b = a + 16;
        f32x4 t = mfma4(load4(nm + (b + row) * NP + a + 4 * grp), load4(ys + (a + 4 * grp) * NP + a + row, NP),
                        f32x4{0.f, 0.f, 0.f, 0.f});
        t = mfma4(load4(ys + (b + row) * NP + b + 4 * grp), t, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
        for (int r = 0; r < 4; ++r)
            ys[(b + 4 * grp + r) * NP + a + row] = -t[r];
    }
    __syncthreads();
    f32x4 low[2];
    if (wave < 2) {
        const int c = 16 * wave;
        f32x4 t[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            t[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int m = 0; m < 2; ++m)
                t[i] = mfma4(load4(nm + (32 + 16 * i + row) * NP + 16 * m + 4 * grp),
                             load4(ys + (16 * m + 4 * grp) * NP + c + row, NP), t[i]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            low[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int m = 0; m < 2; ++m)
                low[i] = mfma4(load4(ys + (32 + 16 * i + row) * NP + 32 + 16 * m + 4 * grp), t[m], low[i]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                ys[(32 + 16 * i + 4 * grp + r) * NP + c + row] = -low[i][r];
    }
    __syncthreads();
    for (int i = tid; i < C * C; i += 256)
        y_out[i] = ys[i / C * NP + i % C];
}

// The states, 16 columns a wave: they do not meet, so a wave keeps its part of
// S in registers and needs no other wave's results. DT: Dk in tiles of 16.
template<typename Scalar, int DT>
__global__ __launch_bounds__(256) void chain_kernel(const DeltaJob job, const DeltaWork work, int groups) {
    extern __shared__ __align__(16) float lds[];
    constexpr int C = kDeltaChunk, wide = 16 * DT, pitch = wide + 4;
    float *ks = lds, *qs = ks + C * pitch;
    __shared__ float grow[C], left[C], beta_s[C];
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave, wave = tid / kWave;
    const int row = lane & 15, grp = lane >> 4;
    const int group = static_cast<int>(blockIdx.x) % groups;
    const int head = static_cast<int>(blockIdx.x) / groups % job.Hv;
    const int n = static_cast<int>(blockIdx.x) / groups / job.Hv;
    const int kh = head / (job.Hv / job.Hk);
    const int c = (group * 4 + wave) * 16 + row;
    const bool on = c < job.Dv;
    const int cc = on ? c : 0;
    const DeltaSpan span = delta_span(job, n);
    int first, count;
    delta_chunks(job, work, n, span, first, count);

    const int64_t matrix = (static_cast<int64_t>(n) * job.Hv + head) * job.Dk * job.Dv;
    f32x4 s[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int d = 16 * t + 4 * grp + r;
            s[t][r] = job.init && on && d < job.Dk ? job.init[matrix + static_cast<int64_t>(d) * job.Dv + c] : 0.f;
        }
    const Scalar *k = static_cast<const Scalar *>(job.k) + span.b * job.k_at[0] + kh * job.k_at[2];
    const Scalar *q = static_cast<const Scalar *>(job.q) + span.b * job.q_at[0] + kh * job.q_at[2];
    const Scalar *v = static_cast<const Scalar *>(job.v) + span.b * job.v_at[0] + head * job.v_at[2] + cc;
    Scalar *o = static_cast<Scalar *>(job.o) + (static_cast<int64_t>(span.b) * job.T * job.Hv + head) * job.Dv + cc;
    const int64_t o_step = static_cast<int64_t>(job.Hv) * job.Dv;
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};

    for (int i = 0; i < count; ++i) {
        const int64_t t0 = span.t0 + i * C;
        const int len = min(C, span.len - i * C);
        const int64_t record = static_cast<int64_t>(first + i) * job.Hv + head;
        __syncthreads();
        stage_rows(k + t0 * job.k_at[1], job.k_at[1], len, job.Dk, wide, ks, pitch);
        stage_rows(q + t0 * job.q_at[1], job.q_at[1], len, job.Dk, wide, qs, pitch);
        if (wave == 0) {
            const double gam = work.gamma[record * C + lane], end = work.gamma[record * C + C - 1];
            grow[lane] = expf(static_cast<float>(gam));
            left[lane] = expf(static_cast<float>(end - gam));
            beta_s[lane] = lane < len ? load_code(job.beta, job.beta_dtype, span.b * job.beta_at[0] +
                                                  (t0 + lane) * job.beta_at[1] + head * job.beta_at[2]) : 0.f;
        }
        f32x4 e[4], g[4], qo[4];
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int t = 16 * m + 4 * grp + r;
                e[m][r] = t < len && on ? load_f32(v + (t0 + t) * job.v_at[1]) : 0.f;
            }
        if (work.states && on) {
            float *keep = work.states + record * job.Dk * job.Dv + c;
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int d = 16 * t + 4 * grp + r;
                    if (d < job.Dk)
                        keep[static_cast<int64_t>(d) * job.Dv] = s[t][r];
                }
        }
        __syncthreads();
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            g[m] = qo[m] = zero;
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                g[m] = mfma4(load4(ks + (16 * m + row) * pitch + 16 * t + 4 * grp), s[t], g[m]);
                qo[m] = mfma4(load4(qs + (16 * m + row) * pitch + 16 * t + 4 * grp), s[t], qo[m]);
            }
        }
        const float *y = work.y + record * C * C, *p = work.p + record * C * C;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const f32x4 gr = load4(grow + 16 * m + 4 * grp);
            g[m] = e[m] - gr * g[m];
            qo[m] = job.scale * gr * qo[m];
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            e[m] = zero;
#pragma unroll
            for (int j = 0; j <= m; ++j)
                e[m] = mfma4(load4(y + (16 * m + row) * C + 16 * j + 4 * grp), g[j], e[m]);
        }
        if (work.e && on) {
            float *keep = work.e + record * C * job.Dv + c;
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    keep[static_cast<int64_t>(16 * m + 4 * grp + r) * job.Dv] = e[m][r];
        }
#pragma unroll
        for (int m = 0; m < 4; ++m)
            e[m] = e[m] * load4(beta_s + 16 * m + 4 * grp);  // now u
#pragma unroll
        for (int m = 0; m < 4; ++m) {
#pragma unroll
            for (int j = 0; j <= m; ++j)
                qo[m] = mfma4(load4(p + (16 * m + row) * C + 16 * j + 4 * grp), e[j], qo[m]);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int t = 16 * m + 4 * grp + r;
                if (t < len && on)
                    store_f32(o + (t0 + t) * o_step, qo[m][r]);
            }
        }
        const float total = grow[C - 1];
#pragma unroll
        for (int m = 0; m < 4; ++m)
            e[m] = e[m] * load4(left + 16 * m + 4 * grp);
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            s[t] = s[t] * total;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                s[t] = mfma4(load4(ks + (16 * j + 4 * grp) * pitch + 16 * t + row, pitch), e[j], s[t]);
        }
    }
    if (on) {
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int d = 16 * t + 4 * grp + r;
                if (d < job.Dk)
                    job.state[matrix + static_cast<int64_t>(d) * job.Dv + c] = s[t][r];
            }
        if (!job.cu)  // tokens that do not count
            for (int t = span.len + grp; t < job.T; t += 4)
                store_f32(o + t * o_step, 0.f);
    }
}

int padded(int Dk) { return Dk <= 32 ? 32 : Dk <= 64 ? 64 : Dk <= 96 ? 96 : Dk <= 128 ? 128 : Dk <= 160 ? 160 : 256; }

template<typename Scalar>
hipError_t prepare_typed(const DeltaJob &job, const DeltaWork &work, bool backward, hipStream_t stream) {
    const int wide = padded(job.Dk);
    const size_t bytes = (2 * kDeltaChunk * (wide + 4) + kDeltaChunk * (kDeltaChunk + 4)) * sizeof(float);
    hipLaunchKernelGGL(prepare_kernel<Scalar>, dim3(work.chunks, job.Hv), dim3(256), bytes, stream, job, work, wide,
                       backward);
    return hipGetLastError();
}

template<typename Scalar>
hipError_t chain_typed(const DeltaJob &job, const DeltaWork &work, hipStream_t stream, const char **why) {
    const int wide = padded(job.Dk), groups = (job.Dv + 63) / 64;
    const int64_t blocks = static_cast<int64_t>(job.N) * job.Hv * groups;
    if (blocks > 0x7fffffff) {
        *why = "delta rule: too many state columns for one launch";
        return hipErrorInvalidValue;
    }
    const size_t bytes = 2 * kDeltaChunk * (wide + 4) * sizeof(float);
#define RAMNET_CHAIN(DT)                                                                                        \
    if (wide == 16 * DT)                                                                                        \
        hipLaunchKernelGGL((chain_kernel<Scalar, DT>), dim3(static_cast<unsigned>(blocks)), dim3(256), bytes,   \
                           stream, job, work, groups)
    RAMNET_CHAIN(2);
    RAMNET_CHAIN(4);
    RAMNET_CHAIN(6);
    RAMNET_CHAIN(8);
    RAMNET_CHAIN(10);
    RAMNET_CHAIN(16);
#undef RAMNET_CHAIN
    return hipGetLastError();
}

}  // namespace

bool delta_is_recurrent(const DeltaJob &job) { return job.T <= 32; }

namespace {

// Consecutive buffers, each at a multiple of 256 bytes.
struct Carver {
    char *base;
    int64_t size = 0;
    template<typename T>
    T *take(int64_t count) {
        T *p = base ? reinterpret_cast<T *>(base + size) : nullptr;
        size += (count * static_cast<int64_t>(sizeof(T)) + 255) / 256 * 256;
        return p;
    }
};

// A packed sequence adds at most 63 / 64 of a chunk.
void count_chunks(const DeltaJob &job, bool packed, DeltaWork *work) {
    work->per_row = (job.T + kDeltaChunk - 1) / kDeltaChunk;
    work->chunks = packed ? work->per_row + job.N : job.N * work->per_row;
}

}  // namespace

int64_t delta_layout(const DeltaJob &job, bool packed, bool backward, char *base, DeltaWork *work) {
    count_chunks(job, packed, work);
    Carver carve{base};
    const int64_t records = static_cast<int64_t>(work->chunks) * job.Hv, square = kDeltaChunk * kDeltaChunk;
    work->offsets = packed ? carve.take<int32_t>(job.N + 1) : nullptr;
    work->gamma = carve.take<double>(records * kDeltaChunk);
    work->y = carve.take<float>(records * square);
    work->p = carve.take<float>(records * square);
    if (backward) {
        work->bl = carve.take<float>(records * square);
        work->x = carve.take<float>(records * kDeltaChunk * job.Dv);
        work->dstate = carve.take<float>(records * job.Dk * job.Dv);
    }
    return carve.size;
}

int64_t delta_kept(const DeltaJob &job, bool packed, char *base, DeltaWork *work) {
    count_chunks(job, packed, work);
    Carver carve{base};
    const int64_t records = static_cast<int64_t>(work->chunks) * job.Hv;
    work->e = carve.take<float>(records * kDeltaChunk * job.Dv);
    work->states = carve.take<float>(records * job.Dk * job.Dv);
    return carve.size;
}

hipError_t launch_delta_prepare(const DeltaJob &job, const DeltaWork &work, bool backward, hipStream_t stream,
                                const char **why) {
    if (work.offsets) {
        hipLaunchKernelGGL(offsets_kernel, dim3(1), dim3(1024), 0, stream, job, work);
        if (const hipError_t err = hipGetLastError())
            return err;
    }
    switch (job.dtype) {
        case kF32: return prepare_typed<float>(job, work, backward, stream);
        case kF16: return prepare_typed<_Float16>(job, work, backward, stream);
        case kBF16: return prepare_typed<bf16_t>(job, work, backward, stream);
        default: *why = "delta rule: unsupported dtype"; return hipErrorInvalidValue;
    }
}

hipError_t launch_delta_chain(const DeltaJob &job, const DeltaWork &work, hipStream_t stream, const char **why) {
    switch (job.dtype) {
        case kF32: return chain_typed<float>(job, work, stream, why);
        case kF16: return chain_typed<_Float16>(job, work, stream, why);
        case kBF16: return chain_typed<bf16_t>(job, work, stream, why);
        default: *why = "delta rule: unsupported dtype"; return hipErrorInvalidValue;
    }
}

}  // namespace ramnet
