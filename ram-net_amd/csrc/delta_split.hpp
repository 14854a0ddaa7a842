// fp32 products on 16-bit matrix instructions, for the gated delta rule.
//
// A value x, scaled by a power of two that brings the largest of its row or
// column to [2^14, 2^15), is hi + lo in fp16: hi rounds it, lo what is left,
// together to 2^-23 of x or 2^-39 of the largest. A product of two such is
// hi hi + hi lo + lo hi (lo lo is below 2^-22 of it); one of an input that is
// itself of 16 bits takes two, its own value being hi. bf16 inputs have 8
// significant bits and lie within fp16's once their token's largest is at
// 2^14: only elements below 2^-31 of it lose digits. fp32 matrix instructions
// run at 1/16 of the 16-bit rate, so three products are five times faster.
//
// A column of values or errors has one scale over a chunk's 64 tokens: a token's
// own are exact to 2^-24 down to 2^-15 of the column's largest there, to 2^-39 of
// that below. An infinity or a NaN reaches the chunk's other tokens, those before its
// own among them (zeros of a triangle times it): one in v, those of its column alone.
#pragma once

#include "delta_chunk.hpp"

namespace ramnet {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// The scale that brings m to [2^14, 2^15), and its inverse: powers of two.
__device__ __forceinline__ float scale_of(float m, float &inverse) {
    const uint32_t field = min(268u - ((__float_as_uint(m) >> 23) & 255u), 253u);
    inverse = __uint_as_float((254u - field) << 23);
    return __uint_as_float(field << 23);
}

// The largest over the four lanes that share a column (lanes 16 apart).
__device__ __forceinline__ float column_max(float m) {
    const uint32_t x = __float_as_uint(m);
    const auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    m = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const uint32_t y = __float_as_uint(m);
    const auto b = __builtin_amdgcn_permlane16_swap(y, y, false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Two values times a scale, each rounded once to fp16 (one instruction a value).
__device__ __forceinline__ uint32_t scaled_f16(float a, float b, float scale) {
    uint32_t h;
    asm("v_fma_mixlo_f16 %0, %1, %2, 0 op_sel_hi:[0,0,0]" : "=v"(h) : "v"(a), "v"(scale));
    asm("v_fma_mixhi_f16 %0, %1, %2, 0 op_sel_hi:[0,0,0]" : "+v"(h) : "v"(b), "v"(scale));
    return h;
}

// hi and lo of two values.
__device__ __forceinline__ void split2(float a, float b, float scale, uint32_t &hi, uint32_t &lo) {
    hi = scaled_f16(a, b, scale);
    uint32_t l;
    asm("v_fma_mixlo_f16 %0, %1, %2, -%3 op_sel_hi:[0,0,1]" : "=v"(l) : "v"(a), "v"(scale), "v"(hi));
    asm("v_fma_mixhi_f16 %0, %1, %2, -%3 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "+v"(l) : "v"(b), "v"(scale), "v"(hi));
    lo = l;
}

// N tiles of 16 rows (a multiple of 2) as B operands of 32 rows each. Rows go
// in the order a result tile holds them: position 8 g + j of a block is row
// 4 g + j of its first tile for j < 4, of its second one else; A operands are
// laid out to match.
template<int N>
struct Operand {
    u32x4 hi[N / 2], lo[N / 2];
    float inverse;  // of the column's scale

    __device__ __forceinline__ void set(const f32x4 (&x)[N]) {
        float m = 0.f;
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                m = fmaxf(m, fabsf(x[t][r]));
        const float scale = scale_of(column_max(m), inverse);
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
            for (int r = 0; r < 4; r += 2) {
                const int w = t % 2 * 2 + r / 2;
                uint32_t h, l;
                split2(x[t][r], x[t][r + 1], scale, h, l);
                hi[t / 2][w] = h, lo[t / 2][w] = l;
            }
    }
};

__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Position of element k within its row of an A operand: quads of a block of 32
// in the order above.
__device__ __forceinline__ int operand_at(int k) {
    const int quad = (k >> 2) & 7;
    return (k & ~31) | ((quad < 4 ? 2 * quad : 2 * quad - 7) << 2) | (k & 3);
}

// A window of rows in memory: loads past it give 0, stores past it are dropped.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t window(const void *base, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), 0, static_cast<int>(bytes), kBufWord3);
}

constexpr int kNowhere = kDeltaReach;  // past every window, with any row's offset on top

// A wave's 16 columns of a matrix whose rows are `step` elements apart (at
// least its width): rows 16 m + 4 (lane / 16) + r, in order of m and r.
template<typename T>
struct Columns {
    int lane, step;  // bytes: this lane's first element, and of a row
    int width;

    __device__ __forceinline__ Columns(int64_t row_step, int wide, int grp, int column)
        : step(static_cast<int>(row_step * static_cast<int64_t>(sizeof(T)))), width(wide * static_cast<int>(sizeof(T))) {
        lane = column < wide ? 4 * grp * step + column * static_cast<int>(sizeof(T)) : kNowhere;
    }
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t rows(const T *base, int count) const {
        return window(base, count > 0 ? static_cast<int64_t>(count - 1) * step + width : 0);
    }
    template<int TILES, typename F>
    __device__ __forceinline__ void each(F f) const {
        int at = lane;
        asm volatile("" : "+v"(at));  // (the rows' offsets are made here: kept over a loop they would fill the registers)
#pragma unroll
        for (int m = 0; m < TILES; ++m, at += 12 * step)
#pragma unroll
            for (int r = 0; r < 4; ++r, at += step)
                f(m, r, at);
    }
};

// The values have arrived. A loop that goes on with them, and asks for the next
// ones itself, would otherwise wait at its head for what it asked for last.
template<typename T, int N>
__device__ __forceinline__ void arrived(T (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i)
        asm volatile("" : "+v"(x[i]));
}

template<typename T>
__device__ __forceinline__ uint32_t buffer_bits(__amdgpu_buffer_rsrc_t from, int at) {
    if constexpr (sizeof(T) == 4)
        return __builtin_amdgcn_raw_buffer_load_b32(from, at, 0, 0);
    else
        return __builtin_amdgcn_raw_buffer_load_b16(from, at, 0, 0);
}

template<typename T>
__device__ __forceinline__ void buffer_store(float v, __amdgpu_buffer_rsrc_t to, int at) {
    if constexpr (sizeof(T) == 4)
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), to, at, 0, 0);
    else if constexpr (__is_same(T, bf16_t))
        __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, static_cast<__bf16>(v)), to, at, 0, 0);
    else
        __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, static_cast<_Float16>(v)), to, at, 0, 0);
}

// What prepare leaves per record, 64 values each, for the chain kernels: K and
// Q are scaled by sk and sq a token, Y and P by sy and sp as a whole.
enum : int {
    kVecSk, kVecSq,
    kVecGrowK,   // e^gamma / sk
    kVecGrowQ,   // scale e^gamma / sq
    kVecLeftK,   // e^(gamma_C - gamma) / sk (forward: times beta)
    kVecBeta,
    kVecTotal,   // e^gamma_C (GrowK of token 63 times its sk is not: a key of zeros has sk = 2^126)
    kVecInv,     // 1 / sy and then 1 / sp
    kVecs
};
static_assert(kVecs * kDeltaChunk == 512);  // two for each of a group's 256 threads (Stager)
enum : int { kFrags = 6, kFragWords = kFrags * kWave * 4 };  // operands of 16 x 32 of a triangular 64 x 64

// The row tile and block of 32 of fragment f.
__device__ __forceinline__ void frag_place(int f, bool upper, int &tile, int &block) {
    if (upper)
        tile = f < 4 ? f / 2 : f - 2, block = f < 4 ? f % 2 : 1;
    else
        tile = f < 2 ? f : 2 + (f - 2) / 2, block = f < 2 ? 0 : (f - 2) % 2;
}

// The K and Q of a chunk as A operands in LDS, PIECES fp16 parts of each:
//   k, q  [64 tokens][wide]   contraction over Dk
//   kt    [wide][64 tokens]   contraction over the tokens (and qt, backward)
// A row's pieces of 16 bytes lie in another order, by fours, in each 16 tokens: the
// tokens that 16 lanes store at a time, four apart, would else share four banks.
template<int DT, int PIECES, bool QT>
struct ChunkLds {
    static constexpr int kWide = 16 * DT, kPitch = kWide + 8, kPitchT = kDeltaChunk + 8;
    static constexpr int kRows = kDeltaChunk * kPitch, kCols = kWide * kPitchT;  // in halves
    static constexpr int kHalves = PIECES * (kRows + kCols + (QT ? kCols : kRows));
    static constexpr int kBytes = kHalves * 2 + kVecs * kDeltaChunk * 4;
    uint16_t *base;

    __device__ __forceinline__ uint16_t *k(int piece) const { return base + piece * kRows; }
    __device__ __forceinline__ uint16_t *kt(int piece) const { return base + PIECES * kRows + piece * kCols; }
    __device__ __forceinline__ uint16_t *q(int piece) const { return base + PIECES * (kRows + kCols) + piece * kRows; }
    __device__ __forceinline__ uint16_t *qt(int piece) const { return base + PIECES * (kRows + kCols) + piece * kCols; }
    __device__ __forceinline__ float *vec() const { return reinterpret_cast<float *>(base + kHalves); }

    __device__ __forceinline__ u32x4 row_frag(const uint16_t *m, int tile, int block, int lane) const {
        return *reinterpret_cast<const u32x4 *>(m + (16 * tile + (lane & 15)) * kPitch + 32 * block + 8 * (lane >> 4 ^ (tile & 3)));
    }
    __device__ __forceinline__ u32x4 col_frag(const uint16_t *m, int tile, int block, int lane) const {
        return *reinterpret_cast<const u32x4 *>(m + (16 * tile + (lane & 15)) * kPitchT + 32 * block + 8 * (lane >> 4));
    }
};

// Four tokens by eight elements of K or Q, from memory to LDS. A group of four
// waves takes a chunk's pieces in turn; loads of a chunk can be under way
// while the one before is worked on.
template<typename Scalar, int DT, int PIECES, bool QT>
struct Stager {
    using Lds = ChunkLds<DT, PIECES, QT>;
    static constexpr int kItems = (16 * (Lds::kWide / 8) + 255) / 256;  // of a thread
    static constexpr int kWords = sizeof(Scalar) * 8 / 4;
    uint32_t raw[2][kItems][4][kWords];
    f32x4 scales[2];  // of this thread's four tokens
    float vecs[2];

    // WIDE: in pieces of 16 bytes
    template<bool WIDE>
    __device__ __forceinline__ void load_one(const Scalar *src, int64_t step, int len, int Dk, int tid,
                                             uint32_t (&to)[kItems][4][kWords]) {
        constexpr int size = static_cast<int>(sizeof(Scalar));
        const int pitch = static_cast<int>(step) * size;
        const auto rows = window(src, len > 0 ? static_cast<int64_t>(len - 1) * pitch + Dk * size : 0);
#pragma unroll
        for (int n = 0; n < kItems; ++n) {
            const int item = tid + 256 * n, quad = item % 16, d = item / 16 * 8;
            const int first = d < Dk ? 4 * quad * pitch + d * size : kNowhere;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int at = first + e * pitch;
                if constexpr (WIDE) {
#pragma unroll
                    for (int w = 0; w < kWords; w += 4) {
                        const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(rows, at + 4 * w, 0, 0);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            to[n][e][w + i] = x[i];
                    }
                } else {
                    uint32_t x[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        x[i] = buffer_bits<Scalar>(rows, d + i < Dk ? at + i * size : kNowhere);
#pragma unroll
                    for (int i = 0; i < kWords; ++i)
                        to[n][e][i] = size == 4 ? x[i] : x[(2 * i) % 8] | x[(2 * i + 1) % 8] << 16;
                }
            }
        }
    }

    template<bool WIDE, bool Q>
    __device__ __forceinline__ void load(const Scalar *k, int64_t k_step, const Scalar *q, int64_t q_step, int len, int Dk,
                                         const float *vec, int tid) {
        vecs[0] = vec[tid], vecs[1] = vec[tid + 256];
        scales[0] = load4(vec + kVecSk * kDeltaChunk + tid % 16 * 4);
        scales[1] = load4(vec + kVecSq * kDeltaChunk + tid % 16 * 4);
        load_one<WIDE>(k, k_step, len, Dk, tid, raw[0]);
        if constexpr (Q)
            load_one<WIDE>(q, q_step, len, Dk, tid, raw[1]);
    }

    static __device__ __forceinline__ float value(const uint32_t (&w)[kWords], int i) {
        if constexpr (sizeof(Scalar) == 4)
            return __uint_as_float(w[i]);
        else
            return bits_f32<Scalar>((w[i / 2] >> (i % 2 * 16)) & 0xFFFFu);
    }

    // rows: into [64][wide]; cols: into [wide][64]; either may be null
    static __device__ __forceinline__ void store_one(const uint32_t (&from)[kItems][4][kWords], f32x4 s, int tid,
                                                     uint16_t *rows, uint16_t *cols) {
#pragma unroll
        for (int n = 0; n < kItems; ++n) {
            const int item = tid + 256 * n, quad = item % 16, d = item / 16 * 8;
            if (d >= Lds::kWide)
                continue;
            uint32_t h[PIECES][4][4];  // [token][pair of elements]
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    if constexpr (PIECES == 2)
                        split2(value(from[n][e], i), value(from[n][e], i + 1), s[e], h[0][e][i / 2], h[1][e][i / 2]);
                    else if constexpr (__is_same(Scalar, _Float16))
                        h[0][e][i / 2] = from[n][e][i / 2];  // as it is
                    else
                        h[0][e][i / 2] = scaled_f16(value(from[n][e], i), value(from[n][e], i + 1), s[e]);
                }
#pragma unroll
            for (int p = 0; p < PIECES; ++p) {
                if (rows)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint16_t *to = rows + p * Lds::kRows + (4 * quad + e) * Lds::kPitch;
                        *reinterpret_cast<u32x2 *>(to + (operand_at(d) ^ quad / 4 * 8)) = u32x2{h[p][e][0], h[p][e][1]};
                        *reinterpret_cast<u32x2 *>(to + (operand_at(d + 4) ^ quad / 4 * 8)) = u32x2{h[p][e][2], h[p][e][3]};
                    }
                if (cols)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        // element i of the four tokens
                        const uint32_t sel = i % 2 ? 0x07060302u : 0x05040100u;
                        u32x2 x;
                        x[0] = __builtin_amdgcn_perm(h[p][1][i / 2], h[p][0][i / 2], sel);
                        x[1] = __builtin_amdgcn_perm(h[p][3][i / 2], h[p][2][i / 2], sel);
                        *reinterpret_cast<u32x2 *>(cols + p * Lds::kCols + (d + i) * Lds::kPitchT +
                                                   operand_at(4 * quad)) = x;
                    }
            }
        }
    }

    template<bool Q>
    __device__ __forceinline__ void store(const Lds &lds, int tid) const {
        lds.vec()[tid] = vecs[0], lds.vec()[tid + 256] = vecs[1];
        store_one(raw[0], scales[0], tid, lds.k(0), lds.kt(0));
        if constexpr (Q)
            store_one(raw[1], scales[1], tid, QT ? nullptr : lds.q(0), QT ? lds.qt(0) : nullptr);
    }
};

// Products whose A operands come from LDS: a step's are read two steps before
// their use, so that the matrix unit does not wait for the LDS (left to itself the
// compiler keeps one or two reads under way). read(step, operands), use(step,
// operands).
template<int STEPS, int EACH, int STEP, typename Read, typename Use>
__device__ __forceinline__ void pipelined_step(u32x4 (&f)[3][EACH], Read read, Use use) {
    if constexpr (STEP < STEPS) {
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (STEP + 2 < STEPS)
            read(std::integral_constant<int, STEP + 2>{}, f[(STEP + 2) % 3]);
        use(std::integral_constant<int, STEP>{}, f[STEP % 3]);
        pipelined_step<STEPS, EACH, STEP + 1>(f, read, use);
    }
}

template<int STEPS, int EACH, typename Read, typename Use>
__device__ __forceinline__ void pipelined(Read read, Use use) {
    u32x4 f[3][EACH];
    read(std::integral_constant<int, 0>{}, f[0]);
    if constexpr (STEPS > 1)
        read(std::integral_constant<int, 1>{}, f[1]);
    pipelined_step<STEPS, EACH, 0>(f, read, use);
    __builtin_amdgcn_sched_barrier(0);
}

// A lower (forward) or upper triangular 64 x 64 of fragments times an operand:
// e += hi hi + hi lo + lo hi, the four row tiles' sums in turn. LO_B: whether the
// operand has a second part.
template<bool UPPER, bool LO_B = true>
__device__ __forceinline__ void triangle(const u32x4 (&hi)[kFrags], const u32x4 (&lo)[kFrags], const u32x4 (&b_hi)[2],
                                         const u32x4 (&b_lo)[2], f32x4 (&e)[4]) {
#pragma unroll
    for (int kind = 0; kind < 3; ++kind)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                if (UPPER ? b < m / 2 : b > m / 2)
                    continue;
                const int f = UPPER ? (m < 2 ? m * 2 + b : m + 2) : (m < 2 ? m : 2 + (m - 2) * 2 + b);
                if (kind == 0)
                    e[m] = mfma16(hi[f], b_hi[b], e[m]);
                else if (kind == 1 && LO_B)
                    e[m] = mfma16(hi[f], b_lo[b], e[m]);
                else if (kind == 2)
                    e[m] = mfma16(lo[f], b_hi[b], e[m]);
            }
}

// The segments' ends put together (work.parts > 1); backward: from the last
// segment on, with the maps transposed.
hipError_t launch_delta_join(const DeltaJob &job, const DeltaWork &work, bool backward, hipStream_t stream);

}  // namespace ramnet
