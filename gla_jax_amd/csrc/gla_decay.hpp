// Building blocks of the kernels for linear attention with one decay a head (gfx950):
//       S_t = exp(a_t) S_{t-1} + k_t v_t^T,   o_t = S_t^T q_t,   a_t one number a head and token.
//
// A workgroup walks the chunks of one (batch, head) pair (or of a segment of it) with the state in the accumulators of its
// matrix instructions.  With L_i the sum of a up to and with token i of the chunk,
//       o_i = sum_{j<=i} e^{L_i - L_j} (q_i.k_j) v_j + e^{L_i} S^T q_i,     S' = e^{L_C} S + sum_j e^{L_C - L_j} k_j v_j^T.
// The decay being one number, a pair's weight multiplies a finished product, so no operand of a score is rescaled and no
// weight is formed against an anchor: each is the exponential of its own pair's sum.  The sums are formed in 64 bits and
// subtracted there (64 additions a chunk), so a token with a hard reset (a = -inf) does not cost its neighbours precision.
//
// Operand layouts (lane l = 16c + r of a wave).  A 16 x 16 x 32 product takes from each lane row (or column) r of an operand and
// 8 of its 32 contracted values, the same ones for both operands: in order (8c .. 8c+7), or as a 16 x 16 accumulator holds
// its rows, in two halves (4c .. 4c+3 and 16+4c .. 16+4c+3), which makes two accumulators above each other an operand with
// no exchange between lanes.
#pragma once

#include "gla_chunk_common.hpp"

namespace gla {

template <typename T> struct DecayChunk;                       // tokens of a chunk
template <> struct DecayChunk<__bf16> { static constexpr int C = 64; };
template <> struct DecayChunk<float> { static constexpr int C = 32; };

// What the kernels take of an array of rows [B,T,heads,features]: strides in elements, features side by side.
struct DecayRows {
    const void *p;
    int64_t sb, st, sh;
};

// LDS rows carry 32 bytes of padding: 16 rows' 16-byte reads fall into different banks eight by eight, and the four rows of
// a transposing read as well.
template <typename T> constexpr int lds_stride(int features) { return features + 32 / (int)sizeof(T); }

// Per-lane offsets into an LDS tile of rows.
template <typename T> struct DecayLane {
    int row;        // row r, contraction over features in order:            r*S + 8c
    int row2;       // the same in two halves:                               r*S + 4c   (and 16 further)
    int col;        // feature r of a group of 16, contraction over rows in order
    __device__ __forceinline__ DecayLane(int stride)
    {
        const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
        row = r * stride + 8 * c;
        row2 = r * stride + 4 * c;
        if constexpr (sizeof(T) == 2) col = (8 * c + (r >> 2)) * stride + 4 * (r & 3);
        else col = 8 * c * stride + r;
    }
};
__device__ __forceinline__ bf16x8 lds_two_halves(const __bf16 *p)
{
    return __builtin_shufflevector(*reinterpret_cast<const bf16x4 *>(p), *reinterpret_cast<const bf16x4 *>(p + 16), 0, 1, 2, 3,
                                   4, 5, 6, 7);
}
__device__ __forceinline__ f32x8 lds_two_halves(const float *p)
{
    const f32x4 a = *reinterpret_cast<const f32x4 *>(p), b = *reinterpret_cast<const f32x4 *>(p + 16);
    f32x8 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) { r.v[e] = a[e]; r.v[4 + e] = b[e]; }
    return r;
}
// 32 rows of 16 features, the features as the operand's rows
__device__ __forceinline__ bf16x8 lds_columns(const __bf16 *p, int stride) { return lds_tr4x2(p, 4 * stride); }
__device__ __forceinline__ f32x8 lds_columns(const float *p, int stride)
{
    f32x8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r.v[e] = p[e * stride];
    return r;
}

// A float operand as N bf16 ones whose sum it is: 1 rounds it (2^-9 of a value), 2 leaves 2^-17, 3 leaves 2^-25, which is
// what a float holds.  float data take it as it is.
template <typename T, int N> struct Split;
template <int N> struct Split<__bf16, N> {
    bf16x8 part[N];
    __device__ __forceinline__ explicit Split(const float (&x)[8])
    {
        float rest[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) rest[e] = x[e];
#pragma unroll
        for (int i = 0; i < N; ++i) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                part[i][e] = (__bf16)rest[e];
                if (i + 1 < N) rest[e] -= (float)part[i][e];
            }
        }
    }
    // the small parts first
    __device__ __forceinline__ f32x4 left(bf16x8 b, f32x4 c) const
    {
#pragma unroll
        for (int i = N - 1; i >= 0; --i) c = mma_d(part[i], b, c);
        return c;
    }
    __device__ __forceinline__ f32x4 right(bf16x8 a, f32x4 c) const
    {
#pragma unroll
        for (int i = N - 1; i >= 0; --i) c = mma_d(a, part[i], c);
        return c;
    }
};
template <int N> struct Split<float, N> {
    f32x8 whole;
    __device__ __forceinline__ explicit Split(const float (&x)[8])
    {
#pragma unroll
        for (int e = 0; e < 8; ++e) whole.v[e] = x[e];
    }
    __device__ __forceinline__ f32x4 left(const f32x8 &b, f32x4 c) const { return mma_d(whole, b, c); }
    __device__ __forceinline__ f32x4 right(const f32x8 &a, f32x4 c) const { return mma_d(a, whole, c); }
};
__device__ __forceinline__ void two_tiles(f32x4 a, f32x4 b, float (&x)[8])
{
#pragma unroll
    for (int e = 0; e < 4; ++e) { x[e] = a[e]; x[4 + e] = b[e]; }
}

__device__ __forceinline__ double shfl_up_f64(double x, int by)
{
    return __hiloint2double(__shfl_up(__double2hiint(x), by, 64), __shfl_up(__double2loint(x), by, 64));
}

// The chunk's gates, by one wave: lane i holds token i's log decay (0 past the end).  Sums in powers of two.
// A gate below 2^-100000 counts as that (so -inf - (-inf) does not arise); a NaN stays one.
template <int C> struct ChunkGates {
    double sum[C];          // L_i
    float from_start[C];    // 2^{L_i}
    float to_end[C];        // 2^{L_C - L_i}
    float whole;            // 2^{L_C}
};
template <int C> __device__ __forceinline__ double chunk_gates(ChunkGates<C> &g, float a)
{
    const int lane = threadIdx.x & 63;
    double x = (double)a * 1.4426950408889634074;
    x = x < -1e5 ? -1e5 : x;
    if (lane >= C) x = 0.0;
#pragma unroll
    for (int by = 1; by < C; by *= 2) {
        const double other = shfl_up_f64(x, by);
        if (lane >= by) x += other;
    }
    const double all = __hiloint2double(__shfl(__double2hiint(x), C - 1, 64), __shfl(__double2loint(x), C - 1, 64));
    if (lane < C) {
        g.sum[lane] = x;
        g.from_start[lane] = fast_exp2((float)x);
        g.to_end[lane] = fast_exp2((float)(all - x));
        if (lane == 0) g.whole = fast_exp2((float)all);
    }
    return all;
}

// Rows of a chunk on their way from memory to LDS: `NT` threads hold C x F values in registers.
template <typename T, int C, int F, int NT> struct RowsInFlight {
    typedef typename FragTypes<T>::d8 d8;
    static constexpr int kPieces = C * F / 8, kPer = (kPieces + NT - 1) / NT;
    d8 x[kPer];
    // rows t0 .. t0+C-1 of `rows` (at the pair's first row), zeros from token `len` and from feature `features` on
    __device__ __forceinline__ void load(const T *rows, int64_t st, int64_t t0, int64_t len, int features)
    {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int at = threadIdx.x + i * NT, row = at / (F / 8), col = 8 * (at % (F / 8));
            x[i] = d8{};
            if (at < kPieces && t0 + row < len && col < features) x[i] = ld8(rows + (t0 + row) * st + col);
        }
    }
    __device__ __forceinline__ void store(T *tile, int stride) const
    {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int at = threadIdx.x + i * NT, row = at / (F / 8), col = 8 * (at % (F / 8));
            if (at < kPieces) st8(tile + row * stride + col, x[i]);
        }
    }
};

// Tile number n of the lower triangle of 16 x 16 tiles, counted by rows.
__device__ __forceinline__ void triangle(int n, int &ti, int &tj)
{
    ti = n < 1 ? 0 : n < 3 ? 1 : n < 6 ? 2 : 3;
    tj = n - ti * (ti + 1) / 2;
}

// The segments that sequences run as, when there are too few pairs to fill the GPU: `chunks` each but the last.
struct DecayPlan {
    int64_t chunks;     // chunks of a sequence
    int64_t per;        // chunks of a segment
    int64_t segments;
};

struct DecaySizes {
    int64_t B, T, H, HK, DK, DV;
};

// The states that enter the segments, from what every segment adds: `pass` says which way (see the kernels).  Launches the
// pass and the scan over the segments; `states` receives [B*H, segments, slabs][a slab in accumulator order] floats.
enum DecayPass { kDecayForward = 0, kDecayStates = 1, kDecayCotangents = 2 };
int decay_entering_states(void *stream, DecayPass pass, const DecaySizes &n, const DecayPlan &plan, gla_dtype dtype,
                          gla_dtype hidden_dtype, const void *hidden, const DecayRows &gates, const DecayRows &keys,
                          const DecayRows &values, const int32_t *lengths, float *states, float *decays);
__host__ __device__ inline int64_t decay_key_width(int64_t DK) { return DK <= 64 ? 64 : DK <= 128 ? 128 : 256; }     // features that a workgroup holds
inline int64_t decay_value_slab(int64_t DV) { return DV <= 64 ? 64 : 128; }
inline int64_t decay_slabs(int64_t DV) { return (DV + decay_value_slab(DV) - 1) / decay_value_slab(DV); }


int decay_forward(void *stream, const DecaySizes &n, const DecayPlan &plan, gla_dtype dtype, gla_dtype hidden_dtype,
                  const void *hidden_init, const DecayRows &gates, const DecayRows &keys, const DecayRows &values,
                  const DecayRows &queries, const int32_t *lengths, void *hidden_final, void *out, float *kept, float *entering,
                  float *decays);

// Results that several workgroups add to (the heads that share a key head; key and value features in slabs of 128) are
// written as floats in so many parts and summed in order.
struct DecayParts {
    int rows, values, gates;
    float *dquery, *dkey, *dvalue, *dgate;
    double *gate_sums;
};
int decay_backward(void *stream, const DecaySizes &n, const DecayPlan &plan, gla_dtype dtype, gla_dtype hidden_dtype,
                   const DecayRows &gates, const DecayRows &keys, const DecayRows &values, const DecayRows &queries,
                   const DecayRows &dout, const int32_t *lengths, const float *kept, const void *dhidden_final, bool constant_gates,
                   void *dhidden_init, float *dlog_decay, void *dvalue, void *dkey, void *dquery, float *entering, float *decays,
                   const DecayParts &parts);

}  // namespace gla
