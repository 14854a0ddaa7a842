// Gated delta rule, token by token: decode steps and short prompts.
//
// A block holds 32 columns of one head's state in registers (columns of S do
// not meet: each has its own u and o). Rows lie over row groups of threads, four
// columns to a thread: 16-byte accesses at an element's alignment, but for a
// row's last columns. A head's blocks share cache lines where its rows are no whole
// lines, so they run on one compute die (41 rows of 8 heads, 156 x 186: 24.6 us, 34.9
// in the blocks' own order; 64 rows of 16 heads, 128 x 127: 30.6 and 48.3).
// A token costs one reduction over rows: with S the state before it,
//     S_new^T q = e^g S^T q + (k.q) u,
// so S^T k, S^T q and k.q are summed together, within a wave by lane swaps and
// over the four waves through LDS, in a fixed order. The next token's inputs
// are on their way meanwhile.
//
// A decode step is bound by reading and writing the state once: one token of 64
// rows, 16 heads of 128 x 128 moves 134 MB in 24 us (5.5 TB/s, a large copy's
// rate). Several tokens add their latency: six of 32 rows take 22 us a call, 27
// with shuffles for the sums. More blocks at a time by fewer registers (80 and 64
// of the 90) spill: 24.6 and 45 us.
#include "delta_chunk.hpp"
#include "ramnet_kernels.hpp"

namespace ramnet {

namespace {

constexpr int kSlice = 32;    // columns of a block
constexpr int kThreads = 256;

constexpr int kVec = 4;       // columns of a thread

struct alignas(4) Four {
    float x[kVec];
};

template<typename Scalar, int R>
struct Token {
    uint32_t k[R], q[R];
    uint32_t v[kVec];
    float g, beta;
};

// a and b, each summed over the two halves of the wave (or of each 32 lanes): a
// in the first of the two, b in the second. No LDS is in it, as in a shuffle.
__device__ __forceinline__ float fold32(float a, float b) {
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(x[0]) + __uint_as_float(x[1]);
}
__device__ __forceinline__ float fold16(float a, float b) {
    const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(x[0]) + __uint_as_float(x[1]);
}
// Each lane's and that of the lane 8 further in its row of 16.
__device__ __forceinline__ float fold8(float a) {
    return a + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(a), 0x128, 0xF, 0xF, false));
}

// EVEN: Dv is a multiple of 4 (no parts of a piece: 90 registers instead of 98).
template<typename Scalar, int R, bool EVEN>
__global__ __launch_bounds__(kThreads) void recurrent_kernel(const DeltaJob job, int slices) {
    constexpr int CL = kSlice / kVec, RG = kThreads / CL;  // column lanes, row groups
    __shared__ __align__(16) float part[2][kThreads / kWave][2][kSlice];  // [k, q]
    __shared__ float part_kq[2][kThreads / kWave];
    const int tid = static_cast<int>(threadIdx.x), wave = tid / kWave;
    const int cl = tid % CL, rg = tid / CL;
    int slice, line;
    split_block(static_cast<int>(blockIdx.x), slices, job.N * job.Hv, slice, line);
    const int head = line % job.Hv, n = line / job.Hv;
    const int c = slice * kSlice + cl * kVec, width = EVEN ? (c < job.Dv ? kVec : 0) : min(kVec, job.Dv - c);
    const bool on = width > 0;
    const DeltaSpan span = delta_span(job, n);
    const int kh = head / (job.Hv / job.Hk);

    const Scalar *q = static_cast<const Scalar *>(job.q) + span.b * job.q_at[0] + kh * job.q_at[2];
    const Scalar *k = static_cast<const Scalar *>(job.k) + span.b * job.k_at[0] + kh * job.k_at[2];
    const Scalar *v = static_cast<const Scalar *>(job.v) + span.b * job.v_at[0] + head * job.v_at[2] + (on ? c : 0);
    const int64_t g0 = span.b * job.g_at[0] + head * job.g_at[2];
    const int64_t b0 = span.b * job.beta_at[0] + head * job.beta_at[2];
    Scalar *o = static_cast<Scalar *>(job.o) + (static_cast<int64_t>(span.b) * job.T * job.Hv + head) * job.Dv + c;
    const int64_t o_step = static_cast<int64_t>(job.Hv) * job.Dv;
    const int64_t matrix = (static_cast<int64_t>(n) * job.Hv + head) * job.Dk * job.Dv;

    float s[R][kVec];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int r = rg + RG * i;
        const float *from = job.init + matrix + static_cast<int64_t>(r) * job.Dv + c;
        const int have = r < job.Dk && job.init ? width : 0;
        Four w{};
        if (EVEN ? have > 0 : have == kVec) {
            w = *reinterpret_cast<const Four *>(from);
        } else if (!EVEN) {
#pragma unroll
            for (int e = 0; e < kVec; ++e)
                w.x[e] = e < have ? from[e] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < kVec; ++e)
            s[i][e] = w.x[e];
    }

    auto fetch = [&](int t, Token<Scalar, R> &x) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int r = rg + RG * i;
            x.k[i] = r < job.Dk ? load_bits(k + t * job.k_at[1] + r) : 0u;
            x.q[i] = r < job.Dk ? load_bits(q + t * job.q_at[1] + r) : 0u;
        }
#pragma unroll
        for (int e = 0; e < kVec; ++e)
            x.v[e] = load_bits(v + t * job.v_at[1] + ((EVEN ? on : e < width) ? e : 0));
        x.g = load_code(job.g, job.g_dtype, g0 + t * job.g_at[1]);
        x.beta = load_code(job.beta, job.beta_dtype, b0 + t * job.beta_at[1]);
    };

    Token<Scalar, R> now, next;
    if (span.len > 0)
        fetch(span.t0, now);
    for (int i = 0; i < span.len; ++i) {
        const int t = span.t0 + i, buf = i & 1;
        if (i + 1 < span.len)
            fetch(t + 1, next);
        float sk[kVec] = {}, sq[kVec] = {}, kq = 0.f, kr[R];
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const float qr = bits_f32<Scalar>(now.q[j]);
            kr[j] = bits_f32<Scalar>(now.k[j]);
            kq = fmaf(kr[j], qr, kq);
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                sk[e] = fmaf(kr[j], s[j][e], sk[e]);
                sq[e] = fmaf(qr, s[j][e], sq[e]);
            }
        }
        const int lane = tid % kWave;
        const float x = fold8(fold16(fold32(sk[0], sq[0]), fold32(sk[1], sq[1])));
        const float y = fold8(fold16(fold32(sk[2], sq[2]), fold32(sk[3], sq[3])));
        if (lane % 16 < CL) {  // rows of 16 lanes: columns e and e + 2 of k, e = 0, 1; then of q
            float *to = &part[buf][wave][lane / 32][cl * kVec + lane / 16 % 2];
            to[0] = x, to[2] = y;
        }
        kq = fold8(kq);
        kq = fold16(kq, kq);
        kq = fold32(kq, kq);
        if (lane == 0)
            part_kq[buf][wave] = kq;
        __syncthreads();  // (the other buffer is written next: one barrier a token)
        kq = 0.f;
#pragma unroll
        for (int w = 0; w < kThreads / kWave; ++w)
            kq += part_kq[buf][w];
        const float alpha = expf(now.g);
        float out[kVec];
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
            float a = 0.f, b = 0.f;
#pragma unroll
            for (int w = 0; w < kThreads / kWave; ++w) {
                a += part[buf][w][0][cl * kVec + e];
                b += part[buf][w][1][cl * kVec + e];
            }
            const float u = now.beta * (bits_f32<Scalar>(now.v[e]) - alpha * a);
            out[e] = job.scale * (alpha * b + kq * u);
#pragma unroll
            for (int j = 0; j < R; ++j)
                s[j][e] = fmaf(kr[j], u, alpha * s[j][e]);
        }
        if (rg == 0 && on) {
#pragma unroll
            for (int e = 0; e < kVec; ++e)
                if (EVEN || e < width)
                    store_f32(o + t * o_step + e, out[e]);
        }
        now = next;
    }

    if (on) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int r = rg + RG * i;
            if (r >= job.Dk)
                continue;
            float *dst = job.state + matrix + static_cast<int64_t>(r) * job.Dv + c;
            if (EVEN || width == kVec) {
                *reinterpret_cast<Four *>(dst) = Four{s[i][0], s[i][1], s[i][2], s[i][3]};
            } else {
#pragma unroll
                for (int e = 0; e < kVec; ++e)
                    if (EVEN || e < width)
                        dst[e] = s[i][e];
            }
        }
        // tokens that do not count
        auto clear = [&](int from, int to) {
            for (int t = from + rg; t < to; t += RG)
#pragma unroll
                for (int e = 0; e < kVec; ++e)
                    if (EVEN || e < width)
                        store_f32(o + t * o_step + e, 0.f);
        };
        if (!job.cu)
            clear(span.len, job.T);
        else {
            if (n == 0)
                clear(0, span.t0);
            if (n == job.N - 1)
                clear(span.t0 + span.len, job.T);
        }
    }
}

__global__ __launch_bounds__(kThreads) void zero_kernel(uint16_t *p, int64_t count) {
    const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < count; i += step)
        p[i] = 0;
}

template<typename Scalar>
hipError_t launch_typed(const DeltaJob &job, hipStream_t stream, const char **why) {
    const int slices = (job.Dv + kSlice - 1) / kSlice;
    const int64_t blocks = static_cast<int64_t>(job.N) * job.Hv * slices;
    if (blocks > 0x7fffffff) {
        *why = "delta rule: too many state columns for one launch";
        return hipErrorInvalidValue;
    }
    const dim3 grid(static_cast<unsigned>(blocks));
    const int per = (job.Dk + 31) / 32;  // rows of a thread
#define RAMNET_DELTA(R)                                                                                             \
    if (per <= R) {                                                                                                 \
        if (job.Dv % kVec == 0)                                                                                     \
            hipLaunchKernelGGL((recurrent_kernel<Scalar, R, true>), grid, dim3(kThreads), 0, stream, job, slices);  \
        else                                                                                                        \
            hipLaunchKernelGGL((recurrent_kernel<Scalar, R, false>), grid, dim3(kThreads), 0, stream, job, slices); \
        return hipGetLastError();                                                                                   \
    }
    RAMNET_DELTA(2)
    RAMNET_DELTA(4)
    RAMNET_DELTA(8)
#undef RAMNET_DELTA
    *why = "delta rule: Dk must be at most 256";
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_delta_zero(void *p, int64_t bytes, hipStream_t stream) {
    if (bytes > 0) {
        const int64_t count = bytes / 2, blocks = (count + kThreads - 1) / kThreads;
        hipLaunchKernelGGL(zero_kernel, dim3(static_cast<unsigned>(blocks < 1024 ? blocks : 1024)), dim3(kThreads), 0, stream,
                           static_cast<uint16_t *>(p), count);
    }
    return hipGetLastError();
}

hipError_t launch_delta_recurrent(const DeltaJob &job, hipStream_t stream, const char **why) {
    switch (job.dtype) {
        case kF32: return launch_typed<float>(job, stream, why);
        case kF16: return launch_typed<_Float16>(job, stream, why);
        case kBF16: return launch_typed<bf16_t>(job, stream, why);
        default: *why = "delta rule: unsupported dtype"; return hipErrorInvalidValue;
    }
}

}  // namespace ramnet
