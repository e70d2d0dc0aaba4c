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

constexpr int64_t kComputeUnits = 256;

template <typename T> struct DecayChunk;                       // tokens of a chunk
template <> struct DecayChunk<__bf16> { static constexpr int C = 64; };
template <> struct DecayChunk<float> { static constexpr int C = 32; };

// What the kernels take of an array of rows [B,T,heads,features]: strides in elements, features side by side.
struct DecayRows {
    const void *p;
    int64_t sb, st, sh;
};

// The same number, formed again from here on: what was derived from it before does not stay in registers.
__device__ __forceinline__ unsigned again(unsigned x)
{
    asm volatile("" : "+v"(x));
    return x;
}

__device__ __forceinline__ int again_uniform(int x)
{
    asm volatile("" : "+s"(x));
    return x;
}

// A pointer that all lanes share and a lane's place behind it in bytes: one register of a lane, where a 64-bit sum takes two.
template <typename P> __device__ __forceinline__ P *at_bytes(P *base, unsigned bytes)
{
    return reinterpret_cast<P *>(reinterpret_cast<std::conditional_t<std::is_const_v<P>, const char, char> *>(base) + bytes);
}

// A tile of rows in LDS, F features each, and the three ways in which a product takes it as an operand.
//
// 16-bit data lie without padding, the 16-byte pieces of a row permuted by the row's number: piece p of row i is at p ^ f(i).  No read has
// two lanes at a bank, as the counters say (256 bytes a cycle): 8-byte reads go by 32 lanes, i.e. 16 rows at one piece (halves) or 8 rows at
// a pair of pieces (columns); 16-byte reads by 16 lanes, of rows 0-3 and 12-15 at one piece and rows 4-11 at its neighbour.  So f takes
// every value once, neighbours of 8 rows get different pairs, and the values of rows 4-11 are whole pairs.  With rows padded by
// 16 or 32 bytes instead, one of the three had two lanes to a bank, and half of the forward pass's LDS cycles were conflicts.
// An exclusive or with the tile's or step's number and a constant number of rows makes every address from three numbers a
// lane.  `here` gives a copy whose addresses are formed where they are used: kept for a whole loop, they took 30 registers of the
// forward pass and 100 more were spilled.  float data keep rows padded by 16 bytes, with
// which three chunks of 128 x 128 features fit (forward pass of B16 T512 H16: 101 us; padded by 32 bytes, two of a chunk at a time, 110).
template <typename T, int F> struct LdsTile;
template <int F> struct LdsTile<__bf16, F> {
    static constexpr int kRow = F;
    unsigned at_rows, at_halves, at_columns;     // in bytes: what is left to add is a constant, which the instruction holds
    static __device__ __forceinline__ int permuted(int row)
    {
        const int upper = (row >> 3) & 1;
        return F >= 128 ? (((row & 7) ^ (upper << 2)) << 1) | upper : ((((row >> 1) & 3) ^ (upper << 1)) << 1) | upper;
    }
    __device__ __forceinline__ LdsTile()
    {
        const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4, row = 4 * c + (r >> 2);
        at_rows = 2 * r * F + ((c ^ permuted(r)) << 4);
        at_halves = 2 * r * F + (((c >> 1) ^ permuted(r)) << 4) + 8 * (c & 1);
        at_columns = 2 * row * F + ((((r & 3) >> 1) ^ permuted(row)) << 4) + 8 * (r & 1);
    }
    __device__ __forceinline__ LdsTile here() const
    {
        LdsTile t = *this;
        asm volatile("" : "+v"(t.at_rows), "+v"(t.at_halves), "+v"(t.at_columns));
        return t;
    }
    static __device__ __forceinline__ int piece(int row, int col) { return row * F + (((col >> 3) ^ permuted(row)) << 3); }
    // Volatile, or else the compiler joins the loads of one half for two tiles and moves every register of the operands to its place.
    static __device__ __forceinline__ bf16x4 half(const __bf16 *p)
    {
        return *(const volatile __attribute__((address_space(3))) bf16x4 *)p;
    }
    // rows 16 * t + r as the operand's rows, features 32 * ks .. as the contracted index, in order
    __device__ __forceinline__ bf16x8 rows(const __bf16 *p, int t, int ks) const { return ld8(at_bytes(p + 16 * t * F, at_rows ^ (64 * ks))); }
    // the same in two halves
    __device__ __forceinline__ bf16x8 halves(const __bf16 *p, int t, int ks) const
    {
        p += 16 * t * F;
        return __builtin_shufflevector(half(at_bytes(p, at_halves ^ (64 * ks))), half(at_bytes(p, at_halves ^ (64 * ks + 32))), 0, 1, 2, 3,
                                       4, 5, 6, 7);
    }
    // features 16 * t + r as the operand's rows, rows 32 * ks .. as the contracted index, in two halves
    __device__ __forceinline__ bf16x8 columns(const __bf16 *p, int ks, int t) const
    {
        return lds_tr4x2(at_bytes(p + 32 * ks * F, at_columns ^ (32 * t)), 16 * F);
    }
    // the place of features 16 * u + 4c .. of row 16 * t + r
    template <typename P> __device__ __forceinline__ P *four(P *p, int t, int u) const { return at_bytes(p + 16 * t * F, at_halves ^ (32 * u)); }
};
template <int F> struct LdsTile<float, F> {
    static constexpr int kRow = F + 4;
    int at_rows, at_halves, at_columns;
    __device__ __forceinline__ LdsTile()
    {
        const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
        at_rows = r * kRow + 8 * c;
        at_halves = r * kRow + 4 * c;
        at_columns = 4 * c * kRow + r;
    }
    __device__ __forceinline__ LdsTile here() const { return *this; }
    static __device__ __forceinline__ int piece(int row, int col) { return row * kRow + col; }
    __device__ __forceinline__ f32x8 rows(const float *p, int t, int ks) const { return ld8(p + 16 * t * kRow + at_rows + 32 * ks); }
    __device__ __forceinline__ f32x8 halves(const float *p, int t, int ks) const
    {
        p += 16 * t * kRow + at_halves + 32 * ks;
        const f32x4 a = *reinterpret_cast<const f32x4 *>(p), b = *reinterpret_cast<const f32x4 *>(p + 16);
        f32x8 r;
#pragma unroll
        for (int e = 0; e < 4; ++e) { r.v[e] = a[e]; r.v[4 + e] = b[e]; }
        return r;
    }
    __device__ __forceinline__ f32x8 columns(const float *p, int ks, int t) const
    {
        p += 32 * ks * kRow + at_columns + 16 * t;
        f32x8 r;
#pragma unroll
        for (int e = 0; e < 8; ++e) r.v[e] = p[((e & 3) + 16 * (e >> 2)) * kRow];
        return r;
    }
    template <typename P> __device__ __forceinline__ P *four(P *p, int t, int u) const { return p + (16 * t * kRow + at_halves + 16 * u); }
};

// A float operand as N bf16 ones whose sum it is: 1 rounds it (2^-9 of a value), 2 leaves 2^-17, 3 leaves 2^-25, which is
// what a float holds.  float data take it as it is.
template <typename T, int N> struct Split;
template <int N> struct Split<__bf16, N> {
    bf16x8 part[N];
    __device__ __forceinline__ explicit Split(const float (&x)[8])
    {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            f32x2 rest = {x[e], x[e + 1]};
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const bf16x2 p = __builtin_convertvector(rest, bf16x2);       // two at a time
                part[i][e] = p[0];
                part[i][e + 1] = p[1];
                if (i + 1 < N) {
                    const uint32_t bits = __builtin_bit_cast(uint32_t, p);
                    rest[0] -= __uint_as_float(bits << 16);
                    rest[1] -= __uint_as_float(bits & 0xffff0000u);
                }
            }
        }
    }
};
template <int N> struct Split<float, N> {
    f32x8 part[1];
    __device__ __forceinline__ explicit Split(const float (&x)[8])
    {
#pragma unroll
        for (int e = 0; e < 8; ++e) part[0].v[e] = x[e];
    }
};
// M products with the split operand on the left (right), the small parts first; products of one sum do not follow each other.
template <typename T, int N, typename D8, int M>
__device__ __forceinline__ void mma_left(const Split<T, N> &a, const D8 (&b)[M], f32x4 *c)
{
    constexpr int kParts = sizeof(a.part) / sizeof(a.part[0]);
#pragma unroll
    for (int i = kParts - 1; i >= 0; --i)
#pragma unroll
        for (int m = 0; m < M; ++m) c[m] = mma_d(a.part[i], b[m], c[m]);
}
template <typename T, int N, typename D8, int M>
__device__ __forceinline__ void mma_right(const D8 (&a)[M], const Split<T, N> &b, f32x4 *c)
{
    constexpr int kParts = sizeof(b.part) / sizeof(b.part[0]);
#pragma unroll
    for (int i = kParts - 1; i >= 0; --i)
#pragma unroll
        for (int m = 0; m < M; ++m) c[m] = mma_d(a[m], b.part[i], c[m]);
}
// A tile of scores: rows 16 * ta + 4c .. of one array against rows 16 * tb + r of another, over KS * 32 features.  Four steps' operands are
// read at a time, and two sums keep the products apart.
template <int KS, typename Tile, typename T>
__device__ __forceinline__ f32x4 tile_product(const Tile &l, const T *a, int ta, const T *b, int tb)
{
    typedef typename FragTypes<T>::d8 D8;
    constexpr int kAhead = sizeof(T) == 2 ? (KS < 4 ? KS : 4) : 1;
    f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int k0 = 0; k0 < KS; k0 += kAhead) {
        D8 x[kAhead], y[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            x[i] = l.rows(a, ta, k0 + i);
            y[i] = l.rows(b, tb, k0 + i);
        }
        if constexpr (kAhead > 1) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) s[(k0 + i) & 1] = mma_d(x[i], y[i], s[(k0 + i) & 1]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) s[0][e] += s[1][e];
    return s[0];
}
// Two tiles of scores behind each other as an operand, or (the second lies above the diagonal) one and zeros.
__device__ __forceinline__ bf16x8 two_score_tiles(const __bf16 *p, bool both)
{
    const bf16x4 zero = {};
    return __builtin_shufflevector(LdsTile<__bf16, 64>::half(p), both ? LdsTile<__bf16, 64>::half(p + 256) : zero, 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ __forceinline__ f32x8 two_score_tiles(const float *p, bool both)
{
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f}, a = *reinterpret_cast<const f32x4 *>(p), b = both ? *reinterpret_cast<const f32x4 *>(p + 256) : zero;
    f32x8 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) { r.v[e] = a[e]; r.v[4 + e] = b[e]; }
    return r;
}
__device__ __forceinline__ void two_tiles(f32x4 a, f32x4 b, float (&x)[8])
{
#pragma unroll
    for (int e = 0; e < 4; ++e) { x[e] = a[e]; x[4 + e] = b[e]; }
}

// Four results, rounded, until they are stored.
template <typename T> struct Packed4;
template <> struct Packed4<__bf16> { typedef bf16x4 t; };
template <> struct Packed4<float> { typedef f32x4 t; };
template <typename T> __device__ __forceinline__ typename Packed4<T>::t pack_results(f32x4 v)
{
    return __builtin_convertvector(v, typename Packed4<T>::t);
}

// The sum over the four lanes that have the same r, and over all lanes, without LDS.
__device__ __forceinline__ float sum_over_c(float x)
{
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}
__device__ __forceinline__ float sum_over_r(float x)
{
    x += dpp_f32<kDppQuadXor1>(x);
    x += dpp_f32<kDppQuadXor2>(x);
    x += dpp_f32<kDppRowHalfMirror>(x);
    x += dpp_f32<kDppRowMirror>(x);
    return x;
}

// Sums of a wave's 64-bit numbers up to each lane's, by moves inside rows of 16 lanes and from the rows before.
template <int CTRL, int ROWS> __device__ __forceinline__ double dpp_f64(double x)
{
    return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(x), CTRL, ROWS, 0xf, false),
                            __builtin_amdgcn_update_dpp(0, __double2loint(x), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ double prefix_sum_wave(double x)
{
    x += dpp_f64<0x111, 0xf>(x);      // row_shr:1
    x += dpp_f64<0x112, 0xf>(x);
    x += dpp_f64<0x114, 0xf>(x);
    x += dpp_f64<0x118, 0xf>(x);
    x += dpp_f64<0x142, 0xa>(x);      // row_bcast:15 into rows 1 and 3
    x += dpp_f64<0x143, 0xc>(x);      // row_bcast:31 into rows 2 and 3
    return x;
}

// The chunk's gates, by one wave, which has token i's log decay in lane i (0 past the end).  Sums in powers of two, formed in 64 bits
// and kept as a float and what it leaves, so that the difference of two is as exact as a float holds it.
// A gate below 2^-100000 counts as that (so -inf - (-inf) does not arise); a NaN stays one.
template <int C> struct ChunkGates {
    float sum[C], rest[C];  // L_i
    float from_start[C];    // 2^{L_i}
    float to_end[C];        // 2^{L_C - L_i}
    float whole, pad[3];    // 2^{L_C}
    // 2^{L_i - L_j}
    static __device__ __forceinline__ float weight(float si, float ri, float sj, float rj) { return fast_exp2((si - sj) + (ri - rj)); }
};
template <int C> __device__ __forceinline__ double chunk_gates(ChunkGates<C> &g, float a)
{
    const int lane = again(threadIdx.x) & 63;
    double x = (double)a * 1.4426950408889634074;
    x = x < -1e5 ? -1e5 : x;
    if (lane >= C) x = 0.0;
    x = prefix_sum_wave(x);
    const double all = __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(x), C - 1), __builtin_amdgcn_readlane(__double2loint(x), C - 1));
    if (lane < C) {
        const float s = (float)x;
        g.sum[lane] = s;
        g.rest[lane] = (float)(x - (double)s);
        g.from_start[lane] = fast_exp2(s);
        g.to_end[lane] = fast_exp2((float)(all - x));
        if (lane == 0) g.whole = fast_exp2((float)all);
    }
    return all;
}

// Rows of a chunk on their way from memory to LDS: `NT` threads hold C x F values in registers.  A thread's pieces lie a fixed number of
// rows apart; its place in a chunk is one number that stays, and a chunk is a pointer that all share.
template <typename T, int C, int F, int NT> struct RowsInFlight {
    typedef typename FragTypes<T>::d8 d8;
    static constexpr int kPieces = C * F / 8, kPer = (kPieces + NT - 1) / NT, kStep = NT / (F / 8);
    static_assert(NT % (F / 8) == 0, "");
    d8 x[kPer];
    // A thread's place: kept over a loop it would take registers, so it is formed again for every chunk, once for all arrays.
    static __device__ __forceinline__ unsigned here() { return again(threadIdx.x); }
    // The rows of a chunk that `rows` points at, the first of which exists and `there` in all.  No load is under a branch (a thread without
    // a piece reads one that exists, and `store` puts zeros in its place): with loads that may or may not have been issued the compiler
    // waits for every access to memory where it needs one of them.
    __device__ __forceinline__ void load(unsigned tid, const T *rows, int st, int there, int features)
    {
        const int row = tid / (F / 8), col = 8 * (tid % (F / 8)), from = col < features ? col : 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i)      // (rows lie less than 2^23 elements apart: 24-bit products, which take a quarter of the time)
            x[i] = ld8(at_bytes(rows, (__umul24(min(min(row + i * kStep, C - 1), there - 1), st) + from) * (unsigned)sizeof(T)));
    }
    __device__ __forceinline__ void store(unsigned tid, T *tile, int there, int features) const
    {
        const int row = tid / (F / 8), col = 8 * (tid % (F / 8)), first = LdsTile<T, F>::piece(row, col);
        auto place = [&](int i) {           // 16 rows further the order of the pieces is the same
            return tile + (kStep % 16 == 0 ? first + i * kStep * LdsTile<T, F>::kRow : LdsTile<T, F>::piece(row + i * kStep, col));
        };
        if (there >= C && features >= F) {
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (kPieces % NT == 0 || row + i * kStep < C) st8(place(i), x[i]);
        } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (kPieces % NT == 0 || row + i * kStep < C) st8(place(i), row + i * kStep < there && col < features ? x[i] : d8{});
        }
    }
};
// Waits for the wave's own accesses to memory, stores among them.  Put before a chunk's stores: the rows on their way have arrived by
// then, and the next chunk, which needs them, does not wait for the stores.
__device__ __forceinline__ void wait_for_memory() { __builtin_amdgcn_s_waitcnt(0x0f70); }

// Tile number n of the lower triangle of 16 x 16 tiles, counted by rows.
__device__ __forceinline__ void triangle(int n, int &ti, int &tj)
{
    ti = n < 1 ? 0 : n < 3 ? 1 : n < 6 ? 2 : 3;
    tj = n - ti * (ti + 1) / 2;
}

// The segments that sequences run as: the first `longer` ones have a chunk more than the others, which have `each`.  (Divisions in 64 bits
// took a microsecond of every kernel's beginning.)
struct DecayPlan {
    int64_t chunks;     // of a sequence
    int64_t segments;
    int each, longer;
    DecayPlan() = default;
    DecayPlan(int64_t chunks, int64_t segments) : chunks(chunks), segments(segments), each((int)(chunks / segments)), longer((int)(chunks % segments)) {}
    __host__ __device__ int first(int segment) const { return segment * each + (segment < longer ? segment : longer); }
    // the segment in which a sequence of so many chunks ends: behind it there is nothing to do
    __host__ __device__ int tail(int live) const
    {
        const unsigned last = live - 1, those = longer * (each + 1);
        return live <= 0 ? 0 : last < those ? last / (unsigned)(each + 1) : longer + (last - those) / (unsigned)each;
    }
};

struct DecaySizes {
    int64_t B, T, H, HK, DK, DV;
};

// The pair (batch, head), as b * H + h, of workgroup x: heads that share their keys go to the same one of the 8 dies, to which
// workgroups are dealt in turn, so that its cache reads them once.
__device__ __forceinline__ unsigned pair_of(unsigned x, const DecaySizes &n)
{
    const unsigned group = (unsigned)n.H / (unsigned)n.HK, units = (unsigned)n.B * (unsigned)n.HK, even = units / 8 * 8;
    if (group == 1) return x;
    unsigned unit, member;
    if (x < even * group) {
        unit = 8 * (x / 8 / group) + x % 8;
        member = x / 8 % group;
    } else {
        unit = x / group;
        member = x % group;
    }
    return unit * group + member;
}

// The states that enter the segments, from what every segment adds, or (cotangents) the cotangents of those that leave them.  Launches the
// pass and the scan over the segments; `states` receives [B*H, segments, slabs][a slab in accumulator order] floats.
int decay_entering_states(void *stream, bool cotangents, const DecaySizes &n, const DecayPlan &plan, gla_dtype dtype,
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
