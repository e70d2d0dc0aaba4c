// The gated delta rule: the walks over the chunks, forward with the state and backward with its cotangent.
#include "gla_delta.hpp"

namespace gla {
namespace {

template <typename T, int N> struct Columns { typedef T t __attribute__((ext_vector_type(N))); };
template <typename T> struct Columns<T, 1> { typedef T t; };
template <typename T, int N> __device__ __forceinline__ float column_of(typename Columns<T, N>::t v, int q)
{
    if constexpr (N == 1) return (float)v;
    else return (float)v[q];
}

// What both walks share: a wave holds NC columns a lane of one (batch, head) pair's state, TILES accumulators of 16 features (gla_delta.hpp) for
// each.  With two columns a lane they are neighbours, 2r and 2r + 1.
template <typename T, int DKP, int NC> struct Walk {
    typedef DeltaChunk<T> DC;
    typedef typename FragTypes<T>::d8 D8;
    typedef typename Columns<T, NC>::t Cols;
    static constexpr int C = DC::C, CT = DC::CT, CS = DC::CS, TILES = DKP / 16, KS = DKP / 32;
    int lane, r, c, DK, DV, T_, len, live, col0, col;
    unsigned pair;
    int64_t b, h, hk;
    bool mine;                                   // the lane's columns exist
    f32x4 S[NC][TILES];
    // true: there is nothing to do
    __device__ __forceinline__ bool place(const DeltaArgs &a)
    {
        lane = threadIdx.x & 63;
        r = lane & 15;
        c = lane >> 4;
        pair = blockIdx.x;
        col0 = ((int)blockIdx.y * (int)(blockDim.x >> 6) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * 16 * NC;
        DK = (int)a.n.DK;
        DV = (int)a.n.DV;
        if (pair >= (unsigned)a.pairs || col0 >= DV) return true;
        const unsigned H = (unsigned)a.n.H;
        b = pair / H;
        h = pair % H;
        hk = pair % H / (H / (unsigned)a.n.HK);
        col = col0 + (NC == 2 ? 2 * r : r);
        mine = col < DV;
        T_ = (int)a.n.T;
        len = a.lengths ? min(max(a.lengths[b], 0), T_) : T_;
        live = (len + C - 1) / C;
        return false;
    }
    __device__ __forceinline__ int feature(int t) const { return 32 * (t >> 1) + 8 * c + 4 * (t & 1); }      // of accumulator element 0
    __device__ __forceinline__ void load_state(const void *from, int dtype)
    {
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x[NC] = {};
                if (mine && feature(t) < DK) load_hidden<NC>(from, dtype, ((int64_t)pair * DK + feature(t) + e) * DV + col, x);
#pragma unroll
                for (int q = 0; q < NC; ++q) S[q][t][e] = x[q];
            }
    }
    __device__ __forceinline__ void store_state(void *to, int dtype) const
    {
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x[NC];
#pragma unroll
                for (int q = 0; q < NC; ++q) x[q] = S[q][t][e];
                if (mine && feature(t) < DK) store_hidden<NC>(to, dtype, ((int64_t)pair * DK + feature(t) + e) * DV + col, x);
            }
    }
    // rows of keys or queries, features as the contracted index in their order; rows behind the end read the last one
    __device__ __forceinline__ void load_rows(const DecayRows &x, int n, D8 (&to)[CT][KS]) const
    {
        const T *p = static_cast<const T *>(x.p) + b * x.sb + hk * x.sh;
#pragma unroll
        for (int ti = 0; ti < CT; ++ti) {
            const T *row = p + (int64_t)min(n * C + 16 * ti + r, len - 1) * x.st;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) to[ti][ks] = ld8(row + (32 * ks + 8 * c < DK ? 32 * ks + 8 * c : 0));
        }
    }
    __device__ __forceinline__ void load_columns(const void *from, const DeltaArgs &a, int n, D8 (&to)[TILES][CS]) const
    {
        const T *p = static_cast<const T *>(from) + ((b * a.n.HK + hk) * a.chunks + n) * (TILES * CS * 512) + lane * 8;
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int ks = 0; ks < CS; ++ks) to[t][ks] = ld8(p + (t * CS + ks) * 512);
    }
    template <int N> __device__ __forceinline__ void load_steps(const void *from, const DeltaArgs &a, int n, D8 (&to)[DC::kSteps][N]) const
    {
        const T *p = static_cast<const T *>(from) + ((int64_t)pair * a.chunks + n) * (DC::kSteps * N * 512) + lane * 8;
#pragma unroll
        for (int s = 0; s < DC::kSteps; ++s)
#pragma unroll
            for (int i = 0; i < N; ++i) to[s][i] = ld8(p + (s * N + i) * 512);
    }
    // the lane's columns of values or their cotangents, tokens 16ti + 4c + e
    __device__ __forceinline__ void load_values(const DecayRows &x, int n, Cols (&to)[CT][4]) const
    {
        const T *p = static_cast<const T *>(x.p) + b * x.sb + h * x.sh + (mine ? col : 0);
#pragma unroll
        for (int ti = 0; ti < CT; ++ti)
#pragma unroll
            for (int e = 0; e < 4; ++e) to[ti][e] = *reinterpret_cast<const Cols *>(p + (int64_t)min(n * C + 16 * ti + 4 * c + e, len - 1) * x.st);
    }
    __device__ __forceinline__ const float *gates(const DeltaArgs &a, int n) const { return a.to.gates + ((int64_t)pair * a.chunks + n) * DC::kGates; }
    // u, x or their cotangents: four tokens of a column
    __device__ __forceinline__ int64_t written(const DeltaArgs &a, int n, int ti, int q) const
    {
        return (((int64_t)n * (DV >> 4) + ((col + q) >> 4)) * CT + ti) * 256 + (c * 16 + ((col + q) & 15)) * 4;
    }
};

// Forward.  An operand's registers are filled for the next chunk as soon as this chunk's products have taken it.
template <typename T, int DKP, int NC, bool KEEP>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1))) void delta_walk_kernel(const DeltaArgs a)
{
    typedef Walk<T, DKP, NC> W;
    typedef typename W::DC DC;
    typedef typename W::D8 D8;
    constexpr int C = W::C, CT = W::CT, CS = W::CS, KS = W::KS, TILES = W::TILES, kParts = DC::kParts, kAll = sizeof(T) == 2 ? 3 : 1;
    W w;
    if (w.place(a)) return;
    const int r = w.r, c = w.c;
    w.load_state(a.hidden, a.hidden_dtype);
    float *kept = KEEP ? a.kept + w.pair * (delta_states_floats(a.n, a.chunks) + delta_written_floats(a.n, a.chunks, C)) : nullptr;
    float *xs = KEEP ? kept + delta_states_floats(a.n, a.chunks) : nullptr;
    auto keep = [&](int n) {
#pragma unroll
        for (int q = 0; q < NC; ++q)
#pragma unroll
            for (int t = 0; t < TILES; ++t)
                if (w.mine && w.feature(t) < w.DK)
                    *reinterpret_cast<f32x4 *>(kept + ((int64_t)n * w.DV + w.col + q) * w.DK + w.feature(t)) = w.S[q][t];
    };
    D8 K[CT][KS], Q[CT][KS], KT[TILES][CS], Z[DC::kSteps][kParts], P[DC::kSteps][1];
    typename W::Cols V[CT][4];
    T *out = static_cast<T *>(a.out) + (w.b * w.T_ * a.n.H + w.h) * w.DV + w.col0;
    const int64_t row = a.n.H * w.DV;
    const int at = 4 * NC * c;                   // the lane's values of a row of out
    const bool there = w.col0 + at < w.DV;
    if (w.live > 0) {
        w.load_rows(a.keys, 0, K);
        w.load_rows(a.queries, 0, Q);
        w.load_values(a.values, 0, V);
        w.load_steps(a.to.inverse, a, 0, Z);
        w.load_steps(a.to.scores, a, 0, P);
        w.load_columns(a.to.keys, a, 0, KT);
    }
    for (int n = 0; n < w.live; ++n) {
        const int next = min(n + 1, w.live - 1);
        const float *gate = w.gates(a, n);
        f32x4 start[CT], end[CT], beta[CT];
        float at_start[CT];
#pragma unroll
        for (int ti = 0; ti < CT; ++ti) {
            start[ti] = *reinterpret_cast<const f32x4 *>(gate + 16 * ti + 4 * c);
            end[ti] = *reinterpret_cast<const f32x4 *>(gate + C + 16 * ti + 4 * c);
            beta[ti] = *reinterpret_cast<const f32x4 *>(gate + 2 * C + 16 * ti + 4 * c);
            at_start[ti] = gate[16 * ti + r];
        }
        const float whole = gate[3 * C];
        if constexpr (KEEP) keep(n);
        f32x4 x[NC][CT], o[NC][CT];
#pragma unroll
        for (int q = 0; q < NC; ++q)
#pragma unroll
            for (int ti = 0; ti < CT; ++ti) x[q][ti] = o[q][ti] = f32x4{0.f, 0.f, 0.f, 0.f};
        // S^T k, and S^T q the other way round
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int q = 0; q < NC; ++q) {
                float s[8];
                two_tiles(w.S[q][2 * ks], w.S[q][2 * ks + 1], s);
                const Split<T, kParts> op(s);
#pragma unroll
                for (int ti = 0; ti < CT; ++ti) {
                    x[q][ti] = mma_whole(K[ti][ks], op.part, x[q][ti]);
                    o[q][ti] = mma_d(op.part[0], Q[ti][ks], o[q][ti]);
                }
            }
        w.load_rows(a.keys, next, K);
        w.load_rows(a.queries, next, Q);
#pragma unroll
        for (int q = 0; q < NC; ++q) {
            D8 op[CS][kParts];
#pragma unroll
            for (int ks = 0; ks < CS; ++ks) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int ti = 2 * ks + (i >> 2), e = i & 3;
                    const float value = w.mine && n * C + 16 * ti + 4 * c + e < w.len ? column_of<T, NC>(V[ti][e], q) : 0.f;
                    v[i] = value - start[ti][e] * x[q][ti][e];
                }
                const Split<T, kParts> split(v);
#pragma unroll
                for (int i = 0; i < kParts; ++i) op[ks][i] = split.part[i];
            }
#pragma unroll
            for (int ti = 0; ti < CT; ++ti) {
                x[q][ti] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks <= ti / 2; ++ks) x[q][ti] = mma_parts(Z[DC::lower(ti, ks)], op[ks], x[q][ti]);
            }
        }
        w.load_values(a.values, next, V);
        w.load_steps(a.to.inverse, a, next, Z);
        if constexpr (KEEP) {
#pragma unroll
            for (int q = 0; q < NC; ++q)
#pragma unroll
                for (int ti = 0; ti < CT; ++ti)
                    if (w.mine) *reinterpret_cast<f32x4 *>(xs + w.written(a, n, ti, q)) = x[q][ti];
        }
        // u
#pragma unroll
        for (int q = 0; q < NC; ++q)
#pragma unroll
            for (int ti = 0; ti < CT; ++ti)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[q][ti][e] *= beta[ti][e];
#pragma unroll
        for (int q = 0; q < NC; ++q) {
#pragma unroll
            for (int ti = 0; ti < CT; ++ti)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[q][ti][e] *= at_start[ti];
#pragma unroll
            for (int ks = 0; ks < CS; ++ks) {
                float u[8];
                two_tiles(x[q][2 * ks], x[q][2 * ks + 1], u);
                const Split<T, 1> op(u);
#pragma unroll
                for (int ti = 2 * ks; ti < CT; ++ti) o[q][ti] = mma_d(op.part[0], P[DC::lower(ti, ks)][0], o[q][ti]);
            }
        }
        w.load_steps(a.to.scores, a, next, P);
        // the state behind the chunk
#pragma unroll
        for (int q = 0; q < NC; ++q) {
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) w.S[q][t][e] *= whole;
#pragma unroll
            for (int ks = 0; ks < CS; ++ks) {
                float u[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) u[i] = x[q][2 * ks + (i >> 2)][i & 3] * end[2 * ks + (i >> 2)][i & 3];
                const Split<T, kAll> op(u);
#pragma unroll
                for (int t = 0; t < TILES; ++t) w.S[q][t] = mma_whole(KT[t][ks], op.part, w.S[q][t]);
            }
        }
        w.load_columns(a.to.keys, a, next, KT);
#pragma unroll
        for (int ti = 0; ti < CT; ++ti) {
            const int token = n * C + 16 * ti + r;
            float v[4 * NC];
#pragma unroll
            for (int i = 0; i < 4 * NC; ++i) v[i] = token < w.len ? o[i % NC][ti][i / NC] : 0.f;
            if (there && token < w.T_) store_vec<T, 4 * NC>(out + token * row + at, v);
        }
    }
    // rows past the end of a shorter sequence
    for (int token = w.live * C + r; token < w.T_; token += 16) {
        const float zero[4 * NC] = {};
        if (there) store_vec<T, 4 * NC>(out + token * row + at, zero);
    }
    if constexpr (KEEP) keep(w.live);
    w.store_state(a.hidden_out, a.hidden_dtype);
}

// Backward, from the last chunk to the first.  With dS the cotangent of the state behind a chunk and du that of u from what reads u,
//       du_j = sum_{i>=j} P_ij do_i + e^{L_C - L_j} dS^T k_j,   du <- (1 + b M)^{-T} du,   dv = dr = b du,
//       dS  <- e^{L_C} dS + sum_i e^{L_i} (q_i do_i^T - k_i dv_i^T).
template <typename T, int DKP, int NC>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1))) void delta_walk_back_kernel(const DeltaArgs a)
{
    typedef Walk<T, DKP, NC> W;
    typedef typename W::DC DC;
    typedef typename W::D8 D8;
    constexpr int C = W::C, CT = W::CT, CS = W::CS, KS = W::KS, TILES = W::TILES, kParts = DC::kParts, kAll = sizeof(T) == 2 ? 3 : 1;
    W w;
    if (w.place(a)) return;
    const int c = w.c;
    w.load_state(a.hidden, a.hidden_dtype);
    const float *kept = a.kept + w.pair * (delta_states_floats(a.n, a.chunks) + delta_written_floats(a.n, a.chunks, C));
    float *dus = a.du + w.pair * delta_written_floats(a.n, a.chunks, C);
    T *dstates = static_cast<T *>(a.dstates) + w.pair * a.chunks * a.n.DK * a.n.DV;
    D8 K[CT][KS], KT[TILES][CS], QT[TILES][CS], Z[DC::kSteps][kParts], P[DC::kSteps][kParts];
    typename W::Cols O[CT][4];
    f32x4 S[NC][TILES];
    auto load_kept = [&](int n) {
#pragma unroll
        for (int q = 0; q < NC; ++q)
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                S[q][t] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (w.mine && w.feature(t) < w.DK)
                    S[q][t] = *reinterpret_cast<const f32x4 *>(kept + ((int64_t)n * w.DV + w.col + q) * w.DK + w.feature(t));
            }
    };
    if (w.live > 0) {
        const int n = w.live - 1;
        w.load_rows(a.keys, n, K);
        w.load_steps(a.to.scores, a, n, P);
        w.load_values(a.dout, n, O);
        w.load_steps(a.to.inverse, a, n, Z);
        w.load_columns(a.to.queries, a, n, QT);
        w.load_columns(a.to.keys, a, n, KT);
        load_kept(n + 1);
    }
    for (int n = w.live - 1; n >= 0; --n) {
        const int next = max(n - 1, 0);
        const float *gate = w.gates(a, n);
        f32x4 start[CT], end[CT], beta[CT];
#pragma unroll
        for (int ti = 0; ti < CT; ++ti) {
            start[ti] = *reinterpret_cast<const f32x4 *>(gate + 16 * ti + 4 * c);
            end[ti] = *reinterpret_cast<const f32x4 *>(gate + C + 16 * ti + 4 * c);
            beta[ti] = *reinterpret_cast<const f32x4 *>(gate + 2 * C + 16 * ti + 4 * c);
        }
        const float whole = gate[3 * C];
        // the cotangent of the state behind the chunk, for the gradients; its product with that state
        float dot = 0.f;
#pragma unroll
        for (int q = 0; q < NC; ++q)
#pragma unroll
            for (int t = 0; t < TILES; t += 2) {
                float s[8];
                two_tiles(w.S[q][t], w.S[q][t + 1], s);
                if (w.mine && w.feature(t) < w.DK)
                    store_vec<T, 8>(dstates + ((int64_t)n * w.DV + w.col + q) * w.DK + w.feature(t), s);
#pragma unroll
                for (int e = 0; e < 4; ++e) dot += s[e] * S[q][t][e] + s[4 + e] * S[q][t + 1][e];
            }
        load_kept(n);
        dot = sum_over_c(sum_over_r(dot));
        if (w.lane == 0) a.dots[((int64_t)w.pair * a.chunks + n) * a.dot_slabs + w.col0 / (16 * NC)] = dot;

        f32x4 du[NC][CT];
#pragma unroll
        for (int q = 0; q < NC; ++q)
#pragma unroll
            for (int ti = 0; ti < CT; ++ti) du[q][ti] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int q = 0; q < NC; ++q) {
                float s[8];
                two_tiles(w.S[q][2 * ks], w.S[q][2 * ks + 1], s);
                const Split<T, kAll> op(s);
#pragma unroll
                for (int ti = 0; ti < CT; ++ti) du[q][ti] = mma_whole(K[ti][ks], op.part, du[q][ti]);
            }
        w.load_rows(a.keys, next, K);
        float dout[NC][CS][8];                   // tokens in the order of an operand
#pragma unroll
        for (int q = 0; q < NC; ++q)
#pragma unroll
            for (int ks = 0; ks < CS; ++ks)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int ti = 2 * ks + (i >> 2), e = i & 3;
                    dout[q][ks][i] = w.mine && n * C + 16 * ti + 4 * c + e < w.len ? column_of<T, NC>(O[ti][e], q) : 0.f;
                }
        w.load_values(a.dout, next, O);
#pragma unroll
        for (int q = 0; q < NC; ++q) {
            D8 op[CS][kParts];
#pragma unroll
            for (int ti = 0; ti < CT; ++ti)
#pragma unroll
                for (int e = 0; e < 4; ++e) du[q][ti][e] *= end[ti][e];
#pragma unroll
            for (int ks = 0; ks < CS; ++ks) {
                const Split<T, 1> o(dout[q][ks]);
#pragma unroll
                for (int tj = 0; tj < CT; ++tj)
                    if (ks >= tj / 2) du[q][tj] = mma_whole(P[DC::upper(tj, ks)], o.part[0], du[q][tj]);
            }
#pragma unroll
            for (int ks = 0; ks < CS; ++ks) {
                float u[8];
                two_tiles(du[q][2 * ks], du[q][2 * ks + 1], u);
                const Split<T, kParts> split(u);
#pragma unroll
                for (int i = 0; i < kParts; ++i) op[ks][i] = split.part[i];
            }
#pragma unroll
            for (int tj = 0; tj < CT; ++tj) {
                du[q][tj] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = tj / 2; ks < CS; ++ks) du[q][tj] = mma_parts(Z[DC::upper(tj, ks)], op[ks], du[q][tj]);
                if (w.mine) *reinterpret_cast<f32x4 *>(dus + w.written(a, n, tj, q)) = du[q][tj];
            }
        }
        w.load_steps(a.to.scores, a, next, P);
        w.load_steps(a.to.inverse, a, next, Z);
#pragma unroll
        for (int q = 0; q < NC; ++q) {
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) w.S[q][t][e] *= whole;
#pragma unroll
            for (int ks = 0; ks < CS; ++ks) {
                float o[8], v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int ti = 2 * ks + (i >> 2), e = i & 3;
                    o[i] = start[ti][e] * dout[q][ks][i];
                    v[i] = -start[ti][e] * (beta[ti][e] * du[q][ti][e]);
                }
                const Split<T, kAll> from_out(o), from_value(v);
#pragma unroll
                for (int t = 0; t < TILES; ++t) {
                    w.S[q][t] = mma_whole(QT[t][ks], from_out.part, w.S[q][t]);
                    w.S[q][t] = mma_whole(KT[t][ks], from_value.part, w.S[q][t]);
                }
            }
        }
        w.load_columns(a.to.queries, a, next, QT);
        w.load_columns(a.to.keys, a, next, KT);
    }
    w.store_state(a.hidden_out, a.hidden_dtype);
}

template <typename T, int DKP, int NC> int launch_walk(hipStream_t stream, const DeltaArgs &a, bool backward)
{
    const int slabs = (int)((a.n.DV + 16 * NC - 1) / (16 * NC));
    // a compute unit takes four waves; where they all fit, each has one of its own.  A pair's columns share a die, to which workgroups are dealt in turn
    const int waves = a.pairs * slabs <= kComputeUnits ? 1 : slabs < 4 ? slabs : 4;
    const dim3 grid((unsigned)((a.pairs + 7) / 8 * 8), (slabs + waves - 1) / waves);
    if (backward) delta_walk_back_kernel<T, DKP, NC><<<grid, 64 * waves, 0, stream>>>(a);
    else if (a.kept) delta_walk_kernel<T, DKP, NC, true><<<grid, 64 * waves, 0, stream>>>(a);
    else delta_walk_kernel<T, DKP, NC, false><<<grid, 64 * waves, 0, stream>>>(a);
    return launch_status();
}
template <typename T> int dispatch_walk(hipStream_t stream, const DeltaArgs &a, bool backward)
{
    const bool two = delta_wave_columns(a.n) == 32;
    if (a.n.DK <= 64) return two ? launch_walk<T, 64, 2>(stream, a, backward) : launch_walk<T, 64, 1>(stream, a, backward);
    return two ? launch_walk<T, 128, 2>(stream, a, backward) : launch_walk<T, 128, 1>(stream, a, backward);
}

}  // namespace

// Value columns of a wave: 32 share the operands' way from memory, 16 make twice the waves.
int64_t delta_wave_columns(const DecaySizes &n)
{
    return n.DV > 16 && n.B * n.H * ((n.DV + 15) / 16) > 4 * kComputeUnits ? 32 : 16;
}

int delta_walk(void *stream, const DeltaArgs &a, gla_dtype dtype, bool backward)
{
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == GLA_BF16 ? dispatch_walk<__bf16>(s, a, backward) : dispatch_walk<float>(s, a, backward);
}

}  // namespace gla
