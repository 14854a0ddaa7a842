// Gated delta rule in chunks of 64 tokens: what the chunks' own tokens give
// (prepare), then the states from chunk to chunk (chain).
#include "delta_split.hpp"
#include "ramnet_kernels.hpp"

#include <algorithm>

namespace ramnet {

namespace {

// First chunk of each packed sequence, and the sequences by their lengths: one
// starts its whole walk when its block does, the longest had better be first
// (thirteen sequences of 12345 tokens: chain 125 us; in their own order half as long again).
// More than 1024 keep their order. One block. The sum of the lengths is at
// most T where the bounds are in order; elsewhere it is held to the records
// there are.
__global__ __launch_bounds__(1024) void offsets_kernel(const DeltaJob job, const DeltaWork work) {
    __shared__ int lens[1024];
    __shared__ int wave_sum[16];
    __shared__ int carry;
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave, wave = uniform(tid / kWave);
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
        if (job.N <= 1024)
            lens[tid] = n < job.N ? delta_span(job, n).len : 0;
        __syncthreads();
        if (n < job.N) {
            int rank = n;
            if (job.N <= 1024) {
                rank = 0;
                for (int m = 0; m < job.N; ++m)
                    rank += lens[m] > lens[tid] || (lens[m] == lens[tid] && m < n);
            }
            work.order[rank] = n;
        }
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

// The rows of one wave's tile of K (or Q) as matrix operands, 16 bytes of a
// row a lane and block; zeros past the last token and Dk.
template<typename Scalar, int DT>
struct TileRows {
    static constexpr int kPer = 16 / static_cast<int>(sizeof(Scalar)), kN = 16 * DT / (4 * kPer);
    u32x4 x[kN];

    __device__ __forceinline__ void load(const Scalar *src, int64_t step, int row, int grp, int len, int D, bool whole) {
#pragma unroll
        for (int b = 0; b < kN; ++b) {
            const int d = (4 * b + grp) * kPer;
            const Scalar *p = src + row * step + d;
            x[b] = u32x4{0u, 0u, 0u, 0u};
            if (row >= len || d >= D)
                continue;
            if (whole) {
                x[b] = *reinterpret_cast<const u32x4 *>(p);
            } else {
#pragma unroll
                for (int e = 0; e < kPer; ++e)
                    if (d + e < D)
                        x[b][e * sizeof(Scalar) / 4] |= load_bits(p + e) << (e * sizeof(Scalar) % 4 * 8);
            }
        }
    }
    // the largest of each row, in all lanes of it
    __device__ __forceinline__ float row_max() const {
        float m = 0.f;
#pragma unroll
        for (int b = 0; b < kN; ++b)
#pragma unroll
            for (int e = 0; e < kPer; ++e)
                m = fmaxf(m, fabsf(bits_f32<Scalar>(sizeof(Scalar) == 4 ? x[b][e] : (x[b][e / 2] >> (e % 2 * 16)) & 0xFFFFu)));
        return column_max(m);
    }
    // += this tile times the transpose of the rows at `other` (this lane's row)
    __device__ __forceinline__ f32x4 times(const Scalar *other, int grp, f32x4 acc) const {
#pragma unroll
        for (int b = 0; b < kN; ++b) {
            const u32x4 y = *reinterpret_cast<const u32x4 *>(other + (4 * b + grp) * kPer);
            if constexpr (sizeof(Scalar) == 4) {
                acc = mfma4(__builtin_bit_cast(f32x4, x[b]), __builtin_bit_cast(f32x4, y), acc);
            } else if constexpr (__is_same(Scalar, bf16_t)) {
                typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x[b]),
                                                              __builtin_bit_cast(bf16x8, y), acc, 0, 0, 0);
            } else {
                acc = mfma16(x[b], y, acc);
            }
        }
        return acc;
    }
};

// Sum of the lanes up to this one, in 64 bits (DPP moves: a shuffle goes
// through the LDS).
template<int CTRL, int ROWS>
__device__ __forceinline__ double moved(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<uint32_t>(u), CTRL, ROWS, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<uint32_t>(u >> 32), CTRL, ROWS, 0xF, false);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ double running_sum(double x) {
    x += moved<0x111, 0xF>(x);  // from 1, 2, 4 and 8 lanes before within rows of 16
    x += moved<0x112, 0xF>(x);
    x += moved<0x114, 0xF>(x);
    x += moved<0x118, 0xF>(x);
    x += moved<0x142, 0xA>(x);  // the sum of the row before, in the second and fourth
    return x + moved<0x143, 0xC>(x);  // and of the first half, in the second
}

// Y, P, gamma and the scales of one chunk and value head: wave w has the
// tokens of tile w. Latency from end to end, so as many blocks as fit: P's
// operands and then Y take the place of the keys. Eight rows of 4096 tokens, 16
// heads of 128 in bf16 (518 MB in and out): 127 us, 4.1 TB/s.
template<typename Scalar, int DT>
__global__ __launch_bounds__(256, 4) void prepare_kernel(const DeltaJob job, const DeltaWork work, bool backward) {
    constexpr int C = kDeltaChunk, NP = C + 4, wide = 16 * DT, pitch = wide + 16 / static_cast<int>(sizeof(Scalar));
    constexpr int kSquare = C * NP, kPitchH = C + 8, kHalf = C * kPitchH;
    extern __shared__ __align__(16) float lds[];
    float *nm = lds, *ys = nm + kSquare;
    Scalar *ks = reinterpret_cast<Scalar *>(ys);
    uint16_t *ph = reinterpret_cast<uint16_t *>(ys);
    __shared__ double gam[C];
    __shared__ float beta_s[C], sk_s[C], sq_s[C], p_max[4];
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave, wave = uniform(tid / kWave);
    const int row = lane & 15, grp = lane >> 4;
    const int chunk = blockIdx.x, head = blockIdx.y, kh = head / (job.Hv / job.Hk);
    const DeltaPlace at = delta_place(job, work, chunk);
    if (at.len == 0) {
        // a record of no sequence: the tokens that no sequence covers have output 0
        if (at.n < 0 && !backward) {
            Scalar *o = static_cast<Scalar *>(job.o) + static_cast<int64_t>(head) * job.Dv;
            delta_outside(job, work, chunk, [&](int from, int to) {
                for (int64_t t = from + wave; t < to; t += 4)
                    for (int c = lane; c < job.Dv; c += kWave)
                        store_f32(o + t * job.Hv * job.Dv + c, 0.f);
            });
        }
        return;
    }
    const int64_t record = static_cast<int64_t>(chunk) * job.Hv + head;
    float g = 0.f, beta = 0.f;
    if (wave == 0 && lane < at.len) {
        const int64_t t = at.t0 + lane;
        g = load_code(job.g, job.g_dtype, at.b * job.g_at[0] + t * job.g_at[1] + head * job.g_at[2]);
        beta = load_code(job.beta, job.beta_dtype, at.b * job.beta_at[0] + t * job.beta_at[1] + head * job.beta_at[2]);
    }
    const bool whole = rows_whole<Scalar>(job);
    TileRows<Scalar, DT> kt, qt;
    kt.load(static_cast<const Scalar *>(job.k) + at.b * job.k_at[0] + at.t0 * job.k_at[1] + kh * job.k_at[2], job.k_at[1],
            16 * wave + row, grp, at.len, job.Dk, whole);
    qt.load(static_cast<const Scalar *>(job.q) + at.b * job.q_at[0] + at.t0 * job.q_at[1] + kh * job.q_at[2], job.q_at[1],
            16 * wave + row, grp, at.len, job.Dk, whole);
    if (wave == 0) {
        const double x = running_sum(static_cast<double>(delta_decay(g)) * kLog2e);
        gam[lane] = x;
        beta_s[lane] = beta;
        work.gamma[record * C + lane] = x;
    }
#pragma unroll
    for (int b = 0; b < kt.kN; ++b)
        *reinterpret_cast<u32x4 *>(ks + (16 * wave + row) * pitch + (4 * b + grp) * kt.kPer) = kt.x[b];
    // the tokens' scales: fp16 inputs are multiplied as they are
    {
        float sk = 1.f, sq = 1.f, inverse;
        if constexpr (!__is_same(Scalar, _Float16))
            sk = scale_of(kt.row_max(), inverse), sq = scale_of(qt.row_max(), inverse);
        if (grp == 0)
            sk_s[16 * wave + row] = sk, sq_s[16 * wave + row] = sq;
    }
    __syncthreads();

    // K K^T and Q K^T, lower tiles; P stays in registers
    float *p_out = backward ? work.p + record * C * C : nullptr, *bl_out = backward ? work.bl + record * C * C : nullptr;
    f32x4 p[4];
    float largest = 0.f;
#pragma unroll
    for (int tj = 0; tj < 4; ++tj) {
        p[tj] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (tj > wave)
            continue;
        const int j = 16 * tj + row;
        const f32x4 a = kt.times(ks + j * pitch, grp, f32x4{0.f, 0.f, 0.f, 0.f});
        p[tj] = qt.times(ks + j * pitch, grp, p[tj]);
        const double gj = gam[j];
        const float bj = beta_s[j];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = 16 * wave + 4 * grp + r;
            const float decay = i >= j ? decay_of(gam[i] - gj) : 0.f;
            const float pij = i >= j ? job.scale * p[tj][r] * decay : 0.f, aij = i > j ? a[r] * decay : 0.f;
            p[tj][r] = backward ? pij : pij * bj;
            largest = fmaxf(largest, fabsf(p[tj][r]));
            nm[i * NP + j] = aij * bj;
            if (backward)
                p_out[i * C + j] = pij, bl_out[i * C + j] = aij;
        }
    }
#pragma unroll
    for (int m = 1; m < 16; m <<= 1)
        largest = fmaxf(largest, __shfl_xor(largest, m));
    largest = column_max(largest);
    if (lane == 0)
        p_max[wave] = largest;
    __syncthreads();

    // P (backward: its transpose) as fp16 parts, then as operands to memory. One
    // scale for all of it: both parts are exact to 2^-39 of the largest.
    float p_inverse;
    const float scale_p = scale_of(fmaxf(fmaxf(p_max[0], p_max[1]), fmaxf(p_max[2], p_max[3])), p_inverse);
#pragma unroll
    for (int tj = 0; tj < 4; ++tj) {
        const int j = 16 * tj + row;
        if (tj > (wave | 1))
            continue;  // (no operand reaches there)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = 16 * wave + 4 * grp + r;
            const _Float16 hi = static_cast<_Float16>(p[tj][r] * scale_p);
            uint16_t *to = ph + (backward ? j * kPitchH + operand_at(i) : i * kPitchH + operand_at(j));
            *to = __builtin_bit_cast(uint16_t, hi);
            to[kHalf] = __builtin_bit_cast(uint16_t, static_cast<_Float16>(fmaf(p[tj][r], scale_p, -static_cast<float>(hi))));
        }
    }
    __syncthreads();
    for (int i = wave; i < 2 * kFrags; i += 4) {
        const int part = i >= kFrags, f = i - part * kFrags;
        int tile, block;
        frag_place(f, backward, tile, block);
        const u32x4 x = *reinterpret_cast<const u32x4 *>(ph + part * kHalf + (16 * tile + row) * kPitchH + 32 * block + 8 * grp);
        *reinterpret_cast<u32x4 *>(work.p_frags + record * 2 * kFragWords + part * kFragWords + (f * kWave + lane) * 4) = x;
    }
    // inverse of the unit lower triangular N: 16-blocks by substitution (lane = column),
    // then pairs of blocks: low part -Yb Nba Ya
    float x[16];
    {
        const float *block = nm + 16 * wave * NP + 16 * wave;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (i % 4 == 0)
                __builtin_amdgcn_sched_barrier(0);  // (four rows at a time: registers)
            f32x4 n[4];
#pragma unroll
            for (int j = 0; j < i; j += 4)
                n[j / 4] = load4(block + i * NP + j);
            float sum = i == row ? 1.f : 0.f;
#pragma unroll
            for (int j = 0; j < i; ++j)
                sum = fmaf(-n[j / 4][j % 4], x[j], sum);
            x[i] = sum;
        }
    }
    __syncthreads();
    for (int i = tid; i < kSquare / 4; i += 256)
        reinterpret_cast<f32x4 *>(ys)[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    __syncthreads();
    if (grp == 0)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            ys[(16 * wave + i) * NP + 16 * wave + row] = x[i];
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
    {
        // wave: row tile wave / 2, column tile wave % 2 of the low 32 x 32
        const int c = 16 * (wave & 1), i = 32 + 16 * (wave >> 1);
        f32x4 t[2], low = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            t[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int m = 0; m < 2; ++m)
                t[h] = mfma4(load4(nm + (32 + 16 * h + row) * NP + 16 * m + 4 * grp),
                             load4(ys + (16 * m + 4 * grp) * NP + c + row, NP), t[h]);
        }
#pragma unroll
        for (int m = 0; m < 2; ++m)
            low = mfma4(load4(ys + (i + row) * NP + 32 + 16 * m + 4 * grp), t[m], low);
#pragma unroll
        for (int r = 0; r < 4; ++r)
            ys[(i + 4 * grp + r) * NP + c + row] = -low[r];
    }
    __syncthreads();

    // the scale of Y, and the vectors
    float y_inverse, scale_y;
    {
        float largest = 0.f;
        for (int i = tid; i < kSquare / 4; i += 256) {
            const f32x4 v = reinterpret_cast<const f32x4 *>(ys)[i];
            largest = fmaxf(fmaxf(largest, fmaxf(fabsf(v[0]), fabsf(v[1]))), fmaxf(fabsf(v[2]), fabsf(v[3])));
        }
#pragma unroll
        for (int m = 1; m < 16; m <<= 1)
            largest = fmaxf(largest, __shfl_xor(largest, m));
        largest = column_max(largest);
        if (lane == 0)
            p_max[wave] = largest;
        __syncthreads();
        scale_y = scale_of(fmaxf(fmaxf(p_max[0], p_max[1]), fmaxf(p_max[2], p_max[3])), y_inverse);
        float *vec = work.vec + record * kVecs * C;
        if (wave == 0) {
            const float sk = sk_s[lane], sq = sq_s[lane], b = beta_s[lane];
            const float grow = decay_of(gam[lane]), left = decay_of(gam[C - 1] - gam[lane]);
            vec[kVecSk * C + lane] = sk;
            vec[kVecSq * C + lane] = sq;
            vec[kVecGrowK * C + lane] = grow / sk;
            vec[kVecGrowQ * C + lane] = job.scale * grow / sq;
            vec[kVecLeftK * C + lane] = (backward ? left : left * b) / sk;
            vec[kVecBeta * C + lane] = b;
            vec[kVecTotal * C + lane] = decay_of(gam[C - 1]);
            vec[kVecInv * C + lane] = lane == 0 ? y_inverse : p_inverse;
        }
    }
    for (int f = wave; f < kFrags; f += 4) {
        int tile, block;
        frag_place(f, backward, tile, block);
        const int a = 16 * tile + row, b = 32 * block + 4 * grp;
        f32x4 z[2];
        if (backward)
            z[0] = load4(ys + b * NP + a, NP), z[1] = load4(ys + (b + 16) * NP + a, NP);
        else
            z[0] = load4(ys + a * NP + b), z[1] = load4(ys + a * NP + b + 16);
        u32x4 hi, lo;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            uint32_t h, l;
            split2(z[w / 2][w % 2 * 2], z[w / 2][w % 2 * 2 + 1], scale_y, h, l);
            hi[w] = h, lo[w] = l;
        }
        uint32_t *out = work.y + record * 2 * kFragWords + (f * kWave + lane) * 4;
        *reinterpret_cast<u32x4 *>(out) = hi;
        *reinterpret_cast<u32x4 *>(out + kFragWords) = lo;
    }
}

// The states from chunk to chunk. Columns of S do not meet: each of the first
// four waves keeps 16 of them in registers and needs no other wave's results.
// The other four bring the next chunk's K and Q to LDS as matrix operands.
//
// A row's chunks can be cut into segments that run side by side: the states
// are linear in the state before. A first launch (MAP) runs the segments but
// the last from zeros and, with no values, from each unit vector: the second
// gives the matrix that a segment multiplies the state before it with.
// join_kernel puts the states at the segments' ends together, and the chain
// proper starts each segment from there.
//
// What binds a chunk is the latency of products that depend on one another: eight
// rows of 4096 tokens, 16 heads of 128 x 128 in bf16, take 259 us at 3.0 TB/s, the
// matrix units 27% and the LDS 31% busy.
//
// DT: Dk in tiles of 16; PIECES: fp16 parts of q and k.
template<typename Scalar, int DT, int PIECES, int BUFS, bool MAP>
__global__ __launch_bounds__(512, 2) void chain_kernel(const DeltaJob job, const DeltaWork work, int groups) {
    extern __shared__ __align__(16) float lds_base[];
    using Lds = ChunkLds<DT, PIECES, false>;
    constexpr int C = kDeltaChunk, BT = DT / 2;
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave, wave = uniform(tid / kWave);
    const int row = lane & 15, grp = lane >> 4;
    const int parts = MAP ? work.parts - 1 : work.parts;
    int group, item;
    split_block(static_cast<int>(blockIdx.x), groups, job.N * job.Hv * parts, group, item);
    const int part = item % parts, line = item / parts;
    const int head = line % job.Hv, n = delta_line(work, line / job.Hv);
    const int kh = head / (job.Hv / job.Hk);
    const int tiles = (job.Dv + 15) / 16;
    if (MAP && part == 0 && group * 4 >= tiles)
        return;  // (the first segment starts from the row's own state)
    DeltaSpan span = delta_span(job, n);
    const int row_end = span.len;
    int first, count;
    delta_chunks(job, work, n, span, first, count);
    const int segments = delta_segments(work, count);
    if (part >= segments || (MAP && part + 1 == segments))
        return;
    if (segments > 1) {
        const int from = part * work.part_chunks;
        first += from;
        count = min(count - from, work.part_chunks);
        span.t0 += from * C, span.len -= from * C;
    }
    auto buffer = [&](int i) {
        return Lds{reinterpret_cast<uint16_t *>(reinterpret_cast<char *>(lds_base) + (BUFS == 2 ? (i & 1) * Lds::kBytes : 0))};
    };

    if (wave >= 4) {
        const int at = tid - 256;
        const Scalar *k = static_cast<const Scalar *>(job.k) + span.b * job.k_at[0] + kh * job.k_at[2];
        const Scalar *q = static_cast<const Scalar *>(job.q) + span.b * job.q_at[0] + kh * job.q_at[2];
        Stager<Scalar, DT, PIECES, false> stager;
        // the loads' latency comes first: the chain is in its products of K and Q then, which
        // the stores to LDS would be in the way of (a chunk more in registers, stored
        // as soon as a buffer is free: a quarter longer for eight 4096-token prompts)
        auto bring = [&](auto wide) {
            auto load = [&](int i) {
                const int64_t t0 = span.t0 + i * C;
                stager.template load<decltype(wide)::value, !MAP>(
                    k + t0 * job.k_at[1], job.k_at[1], q + t0 * job.q_at[1], job.q_at[1], min(C, span.len - i * C), job.Dk,
                    work.vec + (static_cast<int64_t>(first + i) * job.Hv + head) * kVecs * C, at);
            };
            if (count > 0) {
                load(0);
                stager.template store<!MAP>(buffer(0), at);
            }
            __syncthreads();
            for (int i = 0; i < count; ++i) {
                load(min(i + 1, count - 1));
                if constexpr (BUFS == 1)
                    __syncthreads();  // chunk i is done with
                stager.template store<!MAP>(buffer(i + 1), at);
                __syncthreads();
            }
        };
        if (rows_whole<Scalar>(job))
            bring(std::true_type{});
        else
            bring(std::false_type{});
        return;
    }

    const int tile = group * 4 + wave;
    const bool is_map = MAP && tile >= tiles;
    const int c = (is_map ? tile - tiles : tile) * 16 + row;
    const int64_t matrix = (static_cast<int64_t>(n) * job.Hv + head) * job.Dk * job.Dv;
    const int64_t piece = static_cast<int64_t>(line) * work.parts + part;  // of the segments' buffers
    const Columns<float> state(job.Dv, job.Dv, grp, c), kept(delta_row(job.Dv), delta_row(job.Dv), grp, c);
    f32x4 s[DT];
    if (is_map) {
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                s[t][r] = 16 * t + 4 * grp + r == c && c < job.Dk ? 1.f : 0.f;
    } else {
        // A row that is cut has its first state twice: the last segment may write where it
        // came from (in place) before the first one has started, so it reads a copy, in the
        // last segment's place.
        float *const copy = work.ends + (piece - part + work.parts - 1) * job.Dk * job.Dv;
        const float *init = part == 0 ? !job.init ? nullptr : !MAP && segments > 1 ? copy : job.init + matrix
                            : MAP     ? nullptr
                                      : work.ends + (piece - 1) * job.Dk * job.Dv;
        const auto from = state.rows(init, init ? job.Dk : 0);
        state.each<DT>([&](int t, int r, int at) { s[t][r] = __uint_as_float(buffer_bits<float>(from, at)); });
        if (MAP && init) {
            const auto to = state.rows(copy, job.Dk);
            state.each<DT>([&](int t, int r, int at) { buffer_store<float>(s[t][r], to, at); });
        }
    }
    const Scalar *v = static_cast<const Scalar *>(job.v) + span.b * job.v_at[0] + head * job.v_at[2] +
                      span.t0 * job.v_at[1];
    const int64_t o_step = static_cast<int64_t>(job.Hv) * job.Dv;
    Scalar *o = static_cast<Scalar *>(job.o) + (static_cast<int64_t>(span.b) * job.T + span.t0) * o_step +
                static_cast<int64_t>(head) * job.Dv;
    const Columns<Scalar> v_cols(job.v_at[1], job.Dv, grp, c), o_cols(o_step, job.Dv, grp, c);
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    uint32_t v_bits[16];
    auto load_v = [&](int i) {
        const auto from = v_cols.rows(v + static_cast<int64_t>(i) * C * job.v_at[1], is_map ? 0 : min(C, span.len - i * C));
        v_cols.template each<4>([&](int m, int r, int at) { v_bits[4 * m + r] = buffer_bits<Scalar>(from, at); });
    };
    // the next chunk's operands are asked for as soon as this one's have been used
    u32x4 y_hi[kFrags], y_lo[kFrags], p_hi[kFrags];
    auto load_y = [&](int i) {
        const int64_t record = static_cast<int64_t>(first + i) * job.Hv + head;
        const u32x4 *yf = reinterpret_cast<const u32x4 *>(work.y + record * 2 * kFragWords);
#pragma unroll
        for (int f = 0; f < kFrags; ++f)
            y_hi[f] = yf[f * kWave + lane], y_lo[f] = yf[(kFrags + f) * kWave + lane];
    };
    auto load_p = [&](int i, int part, u32x4 (&p)[kFrags]) {
        const int64_t record = static_cast<int64_t>(first + i) * job.Hv + head;
        const u32x4 *pf = reinterpret_cast<const u32x4 *>(work.p_frags + (record * 2 + part) * kFragWords);
#pragma unroll
        for (int f = 0; f < kFrags; ++f)
            p[f] = pf[f * kWave + lane];
    };
    if (count > 0) {
        load_v(0);
        load_y(0);
        if constexpr (!MAP) {
            load_p(0, 0, p_hi);
            arrived(p_hi);
        }
        arrived(y_hi);
        arrived(y_lo);
        arrived(v_bits);
    }
    arrived(s);
    __syncthreads();

    for (int i = 0; i < count; ++i) {
        const int64_t record = static_cast<int64_t>(first + i) * job.Hv + head;
        const Lds lds = buffer(i);
        const float *vec = lds.vec();
        const float total = vec[kVecTotal * C];
        if (!MAP && work.states) {
            const auto to = kept.rows(work.states + record * job.Dk * delta_row(job.Dv), job.Dk);
            kept.each<DT>([&](int t, int r, int at) { buffer_store<float>(s[t][r], to, at); });
        }

        f32x4 g[4], qo[4];
        float s_inverse;
        {
            Operand<DT> so;
            so.set(s);
            s_inverse = so.inverse;
#pragma unroll
            for (int m = 0; m < 4; ++m)
                g[m] = qo[m] = zero;
            // steps: of each block of 32 rows of S, K's parts and then Q's
            constexpr int kEach = MAP ? PIECES : 2 * PIECES;
            pipelined<BT * kEach, 4>(
                [&](auto step, u32x4(&f)[4]) {
                    constexpr int at = decltype(step)::value, block = at / kEach, part = at % kEach;
                    const uint16_t *from = part < PIECES ? lds.k(part) : lds.q(part - PIECES);
#pragma unroll
                    for (int m = 0; m < 4; ++m)
                        f[m] = lds.row_frag(from, m, block, lane);
                },
                [&](auto step, const u32x4(&f)[4]) {
                    constexpr int at = decltype(step)::value, block = at / kEach, part = at % kEach;
                    constexpr bool is_k = part < PIECES;
#pragma unroll
                    for (int m = 0; m < 4; ++m) {
                        f32x4 &to = is_k ? g[m] : qo[m];
                        to = mfma16(f[m], so.hi[block], to);
                    }
                    if constexpr (part % PIECES == 0)
#pragma unroll
                        for (int m = 0; m < 4; ++m) {
                            f32x4 &to = is_k ? g[m] : qo[m];
                            to = mfma16(f[m], so.lo[block], to);
                        }
                });
        }
        // P's second part comes now, in the registers of the first products' operands (asked
        // for a chunk ahead like its first one it makes the loop spill: eight 4096-token
        // prompts take 477 us a call, 368 so)
        u32x4 p_lo[kFrags];
        if constexpr (!MAP)
            load_p(i, 1, p_lo);
        // what the state gives o, and v - S^T k but for the chunk's own tokens
        f32x4 e[4];
        float e_inverse;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const f32x4 gr = load4(vec + kVecGrowK * C + 16 * m + 4 * grp) * s_inverse;
            qo[m] = qo[m] * (load4(vec + kVecGrowQ * C + 16 * m + 4 * grp) * s_inverse);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                g[m][r] = fmaf(-gr[r], g[m][r], bits_f32<Scalar>(v_bits[4 * m + r]));
        }
        const int then = min(i + 1, count - 1);  // (the last chunk's once more rather than a branch)
        load_v(then);
        {
            Operand<4> ro;
            ro.set(g);
#pragma unroll
            for (int m = 0; m < 4; ++m)
                e[m] = zero;
            triangle<false>(y_hi, y_lo, ro.hi, ro.lo, e);
            e_inverse = vec[kVecInv * C] * ro.inverse;
            load_y(then);
        }
        // (e without its scale, which is taken into those of the operands made of it)
        if (!MAP && work.e) {
            const auto to = kept.rows(work.e + record * C * delta_row(job.Dv), C);
            kept.each<4>([&](int m, int r, int at) { buffer_store<float>(e[m][r] * e_inverse, to, at); });
        }
        if constexpr (!MAP) {
            Operand<4> eo;
            eo.set(e);
            f32x4 x[4];
#pragma unroll
            for (int m = 0; m < 4; ++m)
                x[m] = zero;
            triangle<false>(p_hi, p_lo, eo.hi, eo.lo, x);
            const float x_inverse = vec[kVecInv * C + 1] * eo.inverse * e_inverse;
#pragma unroll
            for (int m = 0; m < 4; ++m)
                qo[m] = qo[m] + x[m] * x_inverse;
            load_p(then, 0, p_hi);  // (before the stores: what waits for it does not wait for them)
            const auto to = o_cols.rows(o + static_cast<int64_t>(i) * C * o_step, min(C, span.len - i * C));
            o_cols.template each<4>([&](int m, int r, int at) { buffer_store<Scalar>(qo[m][r], to, at); });
        }
#pragma unroll
        for (int m = 0; m < 4; ++m)
            e[m] = e[m] * load4(vec + kVecLeftK * C + 16 * m + 4 * grp);
        Operand<4> wo;
        wo.set(e);
        wo.inverse *= e_inverse;
        // steps: a part of two tiles of S, the update of the two before beside it
        f32x4 x[2][2];
        auto update = [&](int pair, const f32x4(&y)[2]) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    s[2 * pair + h][r] = fmaf(y[h][r], wo.inverse, total * s[2 * pair + h][r]);
        };
        pipelined<DT / 2 * PIECES, 4>(
            [&](auto step, u32x4(&f)[4]) {
                constexpr int at = decltype(step)::value, pair = at / PIECES;
#pragma unroll
                for (int n = 0; n < 4; ++n)
                    f[n] = lds.col_frag(lds.kt(at % PIECES), 2 * pair + n / 2, n % 2, lane);
            },
            [&](auto step, const u32x4(&f)[4]) {
                constexpr int at = decltype(step)::value, pair = at / PIECES, part = at % PIECES;
                f32x4(&y)[2] = x[pair % 2];
                if constexpr (part == 0)
                    y[0] = y[1] = zero;
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        y[h] = mfma16(f[2 * h + b], wo.hi[b], y[h]);
                if constexpr (part == 0)
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            y[h] = mfma16(f[2 * h + b], wo.lo[b], y[h]);
                if constexpr (part == PIECES - 1 && pair > 0)
                    update(pair - 1, x[(pair - 1) % 2]);
            });
        update(DT / 2 - 1, x[(DT / 2 - 1) % 2]);
        __syncthreads();
        if constexpr (BUFS == 1)
            __syncthreads();  // chunk i + 1 is there
    }
    if (is_map) {
        if (tile < tiles + DT) {
            constexpr int wide = 16 * DT;
            const Columns<float> map(wide, wide, grp, c);
            const auto to = map.rows(work.maps + piece * wide * wide, wide);
            map.each<DT>([&](int t, int r, int at) { buffer_store<float>(s[t][r], to, at); });
        }
        return;
    }
    if (!MAP && part + 1 < segments)
        return;
    const auto to = state.rows(MAP ? work.ends + piece * job.Dk * job.Dv : job.state + matrix, job.Dk);
    state.each<DT>([&](int t, int r, int at) { buffer_store<float>(s[t][r], to, at); });
    if (!MAP && !job.cu && c < job.Dv)  // tokens that do not count
        for (int64_t t = row_end + grp; t < job.T; t += 4)
            store_f32(o + (t - (row_end - span.len)) * o_step + c, 0.f);
}

// The states at the ends of a row's segments: what the segment adds, and its
// map times the state before. One block per row, head and 16 columns, a wave a
// tile of Dk: few small products one after the other, in fp32 instructions (16
// segments of 8 heads, 128 x 128: 36 us).
// BACK: the ends lie from the last segment on, and the maps apply transposed.
template<int DT, bool BACK>
__global__ __launch_bounds__(kWave *DT) void join_kernel(const DeltaJob job, const DeltaWork work, int groups) {
    constexpr int wide = 16 * DT;
    __shared__ __align__(16) float s[2][16][wide + 4];  // columns of the state before
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave, wave = uniform(tid / kWave);
    const int row = lane & 15, grp = lane >> 4;
    const int group = static_cast<int>(blockIdx.x) % groups, line = static_cast<int>(blockIdx.x) / groups;
    const int c = group * 16 + row, d = 16 * wave + 4 * grp;
    const int n = delta_line(work, line / job.Hv);
    int first, count;
    delta_chunks(job, work, n, delta_span(job, n), first, count);
    const int segments = delta_segments(work, count);
    if (segments <= 2)
        return;  // (the first segment's end is whole)
    const int64_t piece = static_cast<int64_t>(line) * work.parts, size = static_cast<int64_t>(job.Dk) * job.Dv;
    const Columns<float> state(job.Dv, job.Dv, grp, c);
    auto ends = [&](int i) { return work.ends + (piece + i) * size + static_cast<int64_t>(16 * wave) * job.Dv; };
    const int rows = job.Dk - 16 * wave;  // (of this tile and those after it)
    auto load = [&](int i) {
        f32x4 x;
        const auto from = state.rows(ends(i), rows);
        state.each<1>([&](int, int r, int at) { x[r] = __uint_as_float(buffer_bits<float>(from, at)); });
        return x;
    };
    *reinterpret_cast<f32x4 *>(&s[0][row][d]) = load(0);
    // maps come two steps ahead of their use: a step is shorter than a load
    f32x4 next[2], map[2][DT];
    auto load_step = [&](int i, f32x4 &x, f32x4 (&m)[DT]) {
        if (i + 1 >= segments)
            return;
        x = load(i);
        const float *from = work.maps + (piece + (BACK ? segments - 1 - i : i)) * wide * wide;
#pragma unroll
        for (int t = 0; t < DT; ++t)
            m[t] = BACK ? load4(from + (16 * t + 4 * grp) * wide + 16 * wave + row, wide)
                        : load4(from + (16 * wave + row) * wide + 4 * grp + 16 * t);
    };
    load_step(1, next[1], map[1]);
    load_step(2, next[0], map[0]);
    arrived(next);
    arrived(map[0]);
    arrived(map[1]);
    __syncthreads();
    auto step = [&](int i, f32x4 &x, f32x4 (&m)[DT]) {
        f32x4 y = {0.f, 0.f, 0.f, 0.f};  // (two sums: half the chain)
#pragma unroll
        for (int t = 0; t < DT; t += 2) {
            x = mfma4(m[t], load4(&s[(i + 1) & 1][row][16 * t + 4 * grp]), x);
            y = mfma4(m[t + 1], load4(&s[(i + 1) & 1][row][16 * t + 16 + 4 * grp]), y);
        }
        x = x + y;
        const auto to = state.rows(ends(i), rows);
        state.each<1>([&](int, int r, int at) { buffer_store<float>(x[r], to, at); });
        *reinterpret_cast<f32x4 *>(&s[i & 1][row][d]) = x;
        load_step(i + 2, x, m);
        __syncthreads();
    };
    for (int i = 1; i + 1 < segments; i += 2) {
        step(i, next[1], map[1]);
        if (i + 2 < segments)
            step(i + 1, next[0], map[0]);
    }
}

template<typename Scalar>
hipError_t prepare_typed(const DeltaJob &job, const DeltaWork &work, bool backward, hipStream_t stream) {
    const int wide = delta_padded(job.Dk);
    const size_t rows = kDeltaChunk * (wide * sizeof(Scalar) + 16), square = kDeltaChunk * (kDeltaChunk + 4) * sizeof(float);
    const size_t parts = 2 * kDeltaChunk * (kDeltaChunk + 8) * 2;  // of P, in bytes
#define RAMNET_PREPARE(DT)                                                                                    \
    if (wide == 16 * DT)                                                                                      \
        hipLaunchKernelGGL((prepare_kernel<Scalar, DT>), dim3(work.chunks, job.Hv), dim3(256),                \
                           square + std::max({rows, square, parts}), stream, job, work, backward)
    RAMNET_PREPARE(2);
    RAMNET_PREPARE(4);
    RAMNET_PREPARE(6);
    RAMNET_PREPARE(8);
    RAMNET_PREPARE(10);
    if constexpr (sizeof(Scalar) < 4)  // (wider fp32 heads walk their tokens)
        RAMNET_PREPARE(16);
#undef RAMNET_PREPARE
    return hipGetLastError();
}

template<typename Scalar, int DT>
constexpr bool kChainFits = ChunkLds<DT, sizeof(Scalar) == 4 ? 2 : 1, false>::kBytes <= kLdsBytes;

template<typename Scalar, int DT>
hipError_t chain_launch(const DeltaJob &job, const DeltaWork &work, hipStream_t stream, const char **why) {
    constexpr int PIECES = sizeof(Scalar) == 4 ? 2 : 1;
    constexpr int bytes = ChunkLds<DT, PIECES, false>::kBytes;
    constexpr int BUFS = 2 * bytes <= kLdsBytes ? 2 : 1;  // (128 x 128 in bf16, eight 4096-token prompts: a fifth longer with one)
    const int tiles = (job.Dv + 15) / 16, groups = (tiles + 3) / 4, map_groups = (tiles + DT + 3) / 4;
    const int64_t lines = static_cast<int64_t>(job.N) * job.Hv;
    if (lines * work.parts * map_groups > 0x7fffffff || lines * tiles > 0x7fffffff) {
        *why = "delta rule: too many state columns for one launch";
        return hipErrorInvalidValue;
    }
    auto blocks = [&](int64_t n) { return dim3(static_cast<unsigned>(n)); };
    if (work.parts > 1) {
        hipLaunchKernelGGL((chain_kernel<Scalar, DT, PIECES, BUFS, true>), blocks(lines * (work.parts - 1) * map_groups),
                           dim3(512), BUFS * bytes, stream, job, work, map_groups);
        if (const hipError_t err = hipGetLastError())
            return err;
        if (const hipError_t err = launch_delta_join(job, work, false, stream))
            return err;
    }
    hipLaunchKernelGGL((chain_kernel<Scalar, DT, PIECES, BUFS, false>), blocks(lines * work.parts * groups), dim3(512),
                       BUFS * bytes, stream, job, work, groups);
    return hipGetLastError();
}

template<typename Scalar>
hipError_t chain_typed(const DeltaJob &job, const DeltaWork &work, hipStream_t stream, const char **why) {
    const int wide = delta_padded(job.Dk);
#define RAMNET_CHAIN(DT)                           \
    if constexpr (kChainFits<Scalar, DT>)          \
        if (wide == 16 * DT)                       \
    return chain_launch<Scalar, DT>(job, work, stream, why)
    RAMNET_CHAIN(2);
    RAMNET_CHAIN(4);
    RAMNET_CHAIN(6);
    RAMNET_CHAIN(8);
    RAMNET_CHAIN(10);
    RAMNET_CHAIN(16);
#undef RAMNET_CHAIN
    return hipErrorInvalidValue;
}

}  // namespace

// Short calls, and those whose chunks (two fp16 parts of each fp32 key and
// query) do not fit the LDS or whose matrices are out of reach. A chunk costs the
// same however few its tokens: with 128 x 128 heads in bf16, 8 heads, 32 rows of 16
// heads and 64 rows of them take 20, 48 and 78 us in chunks, and token by token 15, 35
// and 60 with 8 tokens, 17, 47 and 83 with 12, 22, 59 and 105 with 16.
bool delta_is_recurrent(const DeltaJob &job) {
    return job.T <= 8 || (job.dtype == kF32 && delta_padded(job.Dk) > 160) || !delta_within_reach(job);
}

bool delta_trains(const DeltaJob &job) {
    // (64 tokens of dq and dk, too, are within reach)
    return !(job.dtype == kF32 && delta_padded(job.Dk) > 160) && delta_within_reach(job) &&
           static_cast<int64_t>(job.Hk) * job.Dk < kDeltaReach / (4 * kDeltaChunk);
}

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

// Segments of a row: what costs least, in times of a chunk of the chain. A pass
// walks a segment's chunks (and starts, about two) once for every 256 blocks of 64
// columns; the first pass, 0.6 of the time, has the columns of the maps too; the
// join takes 0.6 a segment. One row of 32768 tokens, 8 heads of 128 x 128 (16
// blocks): 1.59 ms in one segment, 0.36 ms in 16. 4096 tokens: 16 blocks 210 us in
// one segment, 85 in 8, 95 in 16; 64 blocks 228 in one, 177 in 4; 128 blocks 272
// in one, 249 in 2.
// Packed rows may be one long one or all alike: segments are sized as for one, and
// a row is cut where it has more than two.
void count_parts(const DeltaJob &job, bool packed, DeltaWork *work) {
    constexpr int kUnits = 256, kMost = 64, kLeast = 4;
    const int64_t columns = static_cast<int64_t>(job.Hv) * ((job.Dv + 63) / 64);
    work->parts = 1, work->part_chunks = work->uncut = work->per_row;
    if (columns * job.N > kUnits / 2)
        return;
    const int64_t blocks = packed ? columns : columns * job.N;
    const int64_t map_blocks = blocks / ((job.Dv + 63) / 64) * ((delta_padded(job.Dk) + job.Dv + 63) / 64);
    float least = static_cast<float>(work->per_row + 2);
    for (int parts = 2; parts <= std::min(work->per_row / kLeast, kMost); ++parts) {
        const int chunks = (work->per_row + parts - 1) / parts;
        const int64_t first = (blocks + (parts - 2) * map_blocks + kUnits - 1) / kUnits;
        const int64_t second = (blocks * parts + kUnits - 1) / kUnits;
        const float cost = static_cast<float>(chunks + 2) * (0.6f * static_cast<float>(first) + static_cast<float>(second)) +
                           0.6f * static_cast<float>(parts - 2) + 2.f;
        if (cost < least)
            least = cost, work->part_chunks = chunks, work->parts = (work->per_row + chunks - 1) / chunks;
    }
    work->uncut = packed ? 2 * work->part_chunks : work->part_chunks;
}

int64_t map_floats(const DeltaJob &job, const DeltaWork &work) {
    const int64_t wide = delta_padded(job.Dk);
    return static_cast<int64_t>(job.N) * job.Hv * work.parts * wide * wide;
}

}  // namespace

int64_t delta_layout(const DeltaJob &job, bool packed, bool backward, char *base, DeltaWork *work) {
    count_chunks(job, packed, work);
    count_parts(job, packed, work);
    Carver carve{base};
    const int64_t records = static_cast<int64_t>(work->chunks) * job.Hv, square = kDeltaChunk * kDeltaChunk;
    work->offsets = packed ? carve.take<int32_t>(job.N + 1) : nullptr;
    work->order = packed ? carve.take<int32_t>(job.N) : nullptr;
    work->gamma = carve.take<double>(records * kDeltaChunk);
    work->vec = carve.take<float>(records * kVecs * kDeltaChunk);
    work->y = carve.take<uint32_t>(records * 2 * kFragWords);
    work->p_frags = carve.take<uint32_t>(records * 2 * kFragWords);
    if (work->parts > 1) {
        work->ends = carve.take<float>(static_cast<int64_t>(job.N) * job.Hv * work->parts * job.Dk * job.Dv);
        float *maps = backward ? nullptr : carve.take<float>(map_floats(job, *work));
        if (!work->maps)  // (else with what is kept)
            work->maps = maps;
    }
    if (backward) {
        work->p = carve.take<float>(records * square);
        work->bl = carve.take<float>(records * square);
        work->x = carve.take<float>(records * kDeltaChunk * delta_row(job.Dv));
        work->dstate = carve.take<float>(records * job.Dk * delta_row(job.Dv));
    }
    return carve.size;
}

int64_t delta_kept(const DeltaJob &job, bool packed, char *base, DeltaWork *work) {
    if (!delta_trains(job))
        return -1;
    count_chunks(job, packed, work);
    Carver carve{base};
    const int64_t records = static_cast<int64_t>(work->chunks) * job.Hv;
    work->e = carve.take<float>(records * kDeltaChunk * delta_row(job.Dv));
    work->states = carve.take<float>(records * job.Dk * delta_row(job.Dv));
    count_parts(job, packed, work);
    if (work->parts > 1)
        work->maps = carve.take<float>(map_floats(job, *work));
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

hipError_t launch_delta_join(const DeltaJob &job, const DeltaWork &work, bool backward, hipStream_t stream) {
    const int wide = delta_padded(job.Dk), tiles = (job.Dv + 15) / 16;
    const dim3 grid(static_cast<unsigned>(job.N * job.Hv * tiles));
    if (work.parts <= 2)  // (the first segment's end is whole)
        return hipGetLastError();
#define RAMNET_JOIN(DT)                                                                                                \
    if (wide == 16 * DT) {                                                                                             \
        if (backward)                                                                                                  \
            hipLaunchKernelGGL((join_kernel<DT, true>), grid, dim3(kWave * DT), 0, stream, job, work, tiles);          \
        else                                                                                                           \
            hipLaunchKernelGGL((join_kernel<DT, false>), grid, dim3(kWave * DT), 0, stream, job, work, tiles);         \
    }
    RAMNET_JOIN(2)
    RAMNET_JOIN(4)
    RAMNET_JOIN(6)
    RAMNET_JOIN(8)
    RAMNET_JOIN(10)
    RAMNET_JOIN(16)
#undef RAMNET_JOIN
    return hipGetLastError();
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
