// Building blocks of linear attention by the gated delta rule (gfx950):
//       S_t = (1 - b_t k_t k_t^T) e^{a_t} S_{t-1} + b_t k_t v_t^T,   o_t = S_t^T q_t,   a_t and b_t one number a head and token.
//
// In chunks of C tokens, with L_i the sum of a up to and with token i of a chunk and S the state before it, what the tokens write is
// the solution of a triangular system whose matrix does not depend on the state:
//       M_ij = e^{L_i - L_j} k_i.k_j for j < i,   r_i = v_i - e^{L_i} S^T k_i,   x = (1 + M b)^{-1} r,   u_i = b_i x_i
//       o_i = e^{L_i} S^T q_i + sum_{j<=i} P_ij u_j,   P_ij = e^{L_i - L_j} q_i.k_j,     S' = e^{L_C} S + sum_j e^{L_C - L_j} k_j u_j^T.
// So the work is in two kinds of kernels.  delta_prepare_kernel, all chunks at once, forms the inverses and the scores.  The walks go
// through a sequence's chunks with the state in the accumulators of their matrix instructions, and need nothing but products.
//
// A workgroup walks with 16 or 32 value columns of the state: four waves each hold a quarter of the features and make, of a chunk's products, 16
// tokens; three times a chunk they hand each other operands through LDS: the state, r, and u.  Four more bring keys, queries and values and do what
// the next state does not wait for.  The inverses and scores come from memory as delta_prepare_kernel's lanes held them.  All of it is requested two chunks
// ahead.  Where there are few sequences their columns are spread over the compute units, and long ones go in segments.
//
// What bounds the walks (128 x 128 features): the chain of a chunk.  Its three exchanges with their products take 2300 cycles where nothing is loaded
// (1.0 us); with a chunk's 80 KB, of which every column's workgroup needs all, 1.6 us for 16 columns where few workgroups run and 2.0 where they
// fill the GPU, 2.5 to 3.2 for 32.  Of that the matrix cores work 17 %, LDS and the path from the caches 40 % each.
//
// Precision.  Keys, queries and values are 16-bit numbers as they come.  What a 32-bit result (states, gradients of the gates) depends on
// and is formed in between enters a product as bf16 parts (Split): the state, the inverse, r, u and the scores of the backward walk in three, 2^-25 of a
// value.  (The state where keys meet it in two, 2^-18: walks 4 to 8 % shorter, and a gradient of beta off by more than 1e-6 of its norm where
// short sequences start from large states.)  What only 16-bit results depend on is in two, 2^-18, so that nothing but a result's own rounding is seen in it:
// the state that queries read, u and the scores of out, dv, the cotangents of states and the scores of dkey and dquery.  (With the scores of out and the cotangents
// of states rounded to 16 bits once, out and dkey were off by 2.3e-3 of their norm where their own rounding is 1.7e-3; 16 prompts of 0 to 1337 tokens took 164 us
// instead of 168, a training step of B4 T4096 H6 D128 455 instead of 493.)  float data take the matrix cores' float products.
//
// Operand layouts: gla_decay.hpp.  Rows of the state are the features pi(t, m) of gla_chunk_common.hpp, so that two accumulators above each
// other (tiles 2p and 2p + 1) are features 32p + 8c .. + 7: an operand of the contraction with keys in their natural order.
#pragma once

#include "gla_decay.hpp"
#include "gla_delta_places.hpp"

namespace gla {

template <typename T> struct DeltaChunk {
    static constexpr int C = DecayChunk<T>::C, CT = C / 16, CS = C / 32;
    static constexpr int kParts = sizeof(T) == 2 ? 3 : 1;      // of an operand that is a 32-bit number
    static constexpr int kFew = sizeof(T) == 2 ? 2 : 1;        // of one that only a 16-bit result depends on
    // steps of 32 tokens of a triangle's rows of tiles, 512 values each: lower ones have step ks <= t / 2, upper ones ks >= t / 2
    static constexpr int kSteps = CS == 1 ? CT : 6;
    static constexpr int lower(int t, int ks) { return t < 2 ? t : 2 * t - 2 + ks; }
    static constexpr int upper(int t, int ks) { return CS == 1 ? t : t < 2 ? 2 * t + ks : t + 2; }
    static constexpr int kGates = 4 * C;                        // floats of a chunk: e^{L_i}, e^{L_C - L_i}, b_i, and e^{L_C} in the last
};

// Where the prepared operands of a call lie.
struct DeltaPrepared {
    void *inverse;      // [pairs, chunks][steps][parts][64][8]
    void *scores;       // [pairs, chunks][steps][parts: few forward, all for the backward walk][64][8]
    float *gates;       // [pairs, chunks][kGates]
};

struct DeltaArgs {
    DecaySizes n;
    int64_t chunks, pairs;
    DecayRows gates, betas, keys, values, queries, dout;
    const int32_t *lengths;
    bool by_length;                 // walks: longest sequences first (at most 64)
    DeltaPrepared to;
    const void *hidden;             // hidden_init; backward: dhidden_final
    int hidden_dtype;
    void *hidden_out;               // hidden_final; dhidden_init
    void *out;
    // what the forward pass leaves for the backward, floats in the order of accumulators, four features or tokens of a column together: of
    // each pair the states before its chunks and at its end, [chunks + 1][DV / 16][tiles of features][4][16][4], and x,
    // [chunks][DV / 16][C / 16][4][16][4]
    float *kept;
    // what the backward walk leaves for the gradients: the cotangents of u in the order of x, those of the states behind the chunks
    // in the states' order, eight features of a column in T, part after part (kFew), and <state, its cotangent> there, [pairs, chunks][columns / 16][4]
    float *du;
    void *dstates;
    float *dots;
    // A long walk in segments of chunks at once (segments > 1): of each but the last, in the walk's order, what it leaves of a start from zero (of the
    // first, of hidden) and of a basis, [pairs, segments - 1][DV + DK][DK] floats; and the states that the others start from, [pairs, segments - 1][DV][DK].
    int segments, segment_chunks;
    float *summary, *starts;
    void *dvalue, *dkey, *dquery;   // dkey, dquery: in their own type, or (more than one part) floats [part][...]
    float *dgate, *dbeta;
    int row_parts;
};
inline __host__ __device__ int64_t delta_state_floats(const DecaySizes &n) { return 16 * delta_state_tiles(n.DK) * n.DV; }
inline __host__ __device__ int64_t delta_states_floats(const DecaySizes &n, int64_t chunks) { return (chunks + 1) * delta_state_floats(n); }
inline __host__ __device__ int64_t delta_written_floats(const DecaySizes &n, int64_t chunks, int C) { return chunks * C * n.DV; }

// Features pi(t, r) as the operand's rows, rows 32 * ks .. as the contracted index, in two halves: LdsTile::columns with another
// order of the features.
template <int F> __device__ __forceinline__ bf16x8 feature_columns(const __bf16 *p, int ks, int t)
{
    const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4, row = 4 * c + (r >> 2);
    const unsigned at = (2 * row * F + (((r & 3) ^ LdsTile<__bf16, F>::permuted(row)) << 4)) ^ (64 * (t >> 1) + 8 * (t & 1));
    return lds_tr4x2(at_bytes(p + 32 * ks * F, at), 16 * F);
}
template <int F> __device__ __forceinline__ f32x8 feature_columns(const float *p, int ks, int t)
{
    constexpr int kRow = LdsTile<float, F>::kRow;
    const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
    p += (32 * ks + 4 * c) * kRow + 32 * (t >> 1) + 8 * (r >> 2) + 4 * (t & 1) + (r & 3);
    f32x8 x;
#pragma unroll
    for (int e = 0; e < 8; ++e) x.v[e] = p[((e & 3) + 16 * (e >> 2)) * kRow];
    return x;
}

// A product of two operands in N parts each, without the products below 2^-9N of it; the small ones first.
template <typename D8, int N> __device__ __forceinline__ f32x4 mma_parts(const D8 (&a)[N], const D8 (&b)[N], f32x4 c)
{
#pragma unroll
    for (int s = N - 1; s >= 0; --s)
#pragma unroll
        for (int i = 0; i <= s; ++i) c = mma_d(a[i], b[s - i], c);
    return c;
}
// and of one in parts with one that is whole
template <typename D8, int N> __device__ __forceinline__ f32x4 mma_whole(const D8 &a, const D8 (&b)[N], f32x4 c)
{
#pragma unroll
    for (int i = N - 1; i >= 0; --i) c = mma_d(a, b[i], c);
    return c;
}
template <typename D8, int N> __device__ __forceinline__ f32x4 mma_whole(const D8 (&a)[N], const D8 &b, f32x4 c)
{
#pragma unroll
    for (int i = N - 1; i >= 0; --i) c = mma_d(a[i], b, c);
    return c;
}

// How many segments a walk is cut into.
int delta_segments(const DeltaArgs &a);
int delta_prepare(void *stream, const DeltaArgs &a, gla_dtype dtype, bool backward);
int delta_walk(void *stream, const DeltaArgs &a, gla_dtype dtype, bool backward);
int delta_gradients(void *stream, const DeltaArgs &a, gla_dtype dtype);
// dst <- the sum over the heads of a key head of parts [H / HK][B,T,HK,DK], in order
int delta_sum_heads(void *stream, const DecaySizes &n, gla_dtype dtype, const float *parts, void *dst);

}  // namespace gla
