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

// What both walks share.  A workgroup of kWaves waves holds NG times 16 value columns of one (batch, head) pair's state; wave w its features
// 16 PER w .. as PER accumulators for each 16 columns, and of a chunk the tokens 16w .. (where there are so many).  Two groups of columns next to
// each other share 32: a lane's are 2r and 2r + 1, so that it reads two values and writes eight results at a time.
template <typename T, int DKP, int NG> struct Walk {
    typedef DeltaChunk<T> DC;
    typedef typename FragTypes<T>::d8 D8;
    typedef typename Packed4<T>::t Four;
    static constexpr int kWaves = 4, C = DC::C, CT = DC::CT, CS = DC::CS, TILES = DKP / 16, KS = DKP / 32, PER = TILES / kWaves;
    static constexpr int NC = NG > 1 ? 2 : 1;            // columns of a lane that lie next to each other
    typedef typename Columns<T, NC>::t Cols;
    int tid, w, lane, r, c, DK, DV, T_, len, live, col0;
    unsigned pair;
    int64_t b, h, hk;
    f32x4 S[NG][PER];
    // true: there is nothing to do
    __device__ __forceinline__ bool place(const DeltaArgs &a)
    {
        tid = threadIdx.x;
        w = __builtin_amdgcn_readfirstlane(tid >> 6);
        lane = tid & 63;
        r = lane & 15;
        c = lane >> 4;
        pair = blockIdx.x;
        col0 = (int)blockIdx.y * 16 * NG;
        DK = (int)a.n.DK;
        DV = (int)a.n.DV;
        if (pair >= (unsigned)a.pairs) return true;
        const unsigned H = (unsigned)a.n.H;
        b = pair / H;
        h = pair % H;
        hk = pair % H / (H / (unsigned)a.n.HK);
        T_ = (int)a.n.T;
        len = a.lengths ? min(max(a.lengths[b], 0), T_) : T_;
        live = (len + C - 1) / C;
        return false;
    }
    __device__ __forceinline__ int column(int g) const { return col0 + (NC == 2 ? 32 * (g >> 1) + 2 * r + (g & 1) : r); }
    __device__ __forceinline__ bool mine(int g) const { return column(g) < DV; }
    __device__ __forceinline__ int feature(int p) const      // of accumulator element 0
    {
        const int t = w * PER + p;
        return 32 * (t >> 1) + 8 * c + 4 * (t & 1);
    }
    __device__ __forceinline__ void load_state(const void *from, int dtype)
    {
#pragma unroll
        for (int g = 0; g < NG; g += NC)
#pragma unroll
            for (int p = 0; p < PER; ++p)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float x[NC] = {};
                    if (mine(g) && feature(p) < DK) load_hidden<NC>(from, dtype, ((int64_t)pair * DK + feature(p) + e) * DV + column(g), x);
#pragma unroll
                    for (int q = 0; q < NC; ++q) S[g + q][p][e] = x[q];
                }
    }
    __device__ __forceinline__ void store_state(void *to, int dtype) const
    {
#pragma unroll
        for (int g = 0; g < NG; g += NC)
#pragma unroll
            for (int p = 0; p < PER; ++p)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float x[NC];
#pragma unroll
                    for (int q = 0; q < NC; ++q) x[q] = S[g + q][p][e];
                    if (mine(g) && feature(p) < DK) store_hidden<NC>(to, dtype, ((int64_t)pair * DK + feature(p) + e) * DV + column(g), x);
                }
    }
    // the wave's tokens of keys or queries, features as the contracted index in their order; tokens behind the end read the last one
    __device__ __forceinline__ void load_rows(const DecayRows &x, int n, D8 (&to)[KS]) const
    {
        const T *row = static_cast<const T *>(x.p) + b * x.sb + hk * x.sh + (int64_t)min(n * C + 16 * w + r, len - 1) * x.st;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) to[ks] = ld8(row + (32 * ks + 8 * c < DK ? 32 * ks + 8 * c : 0));
    }
    // the wave's features of keys or queries, tokens as the contracted index
    __device__ __forceinline__ void load_features(const void *from, const DeltaArgs &a, int n, D8 (&to)[PER][CS]) const
    {
        const T *p = static_cast<const T *>(from) + ((b * a.n.HK + hk) * a.chunks + n) * (TILES * CS * 512) + w * PER * CS * 512 + lane * 8;
#pragma unroll
        for (int t = 0; t < PER; ++t)
#pragma unroll
            for (int ks = 0; ks < CS; ++ks) to[t][ks] = ld8(p + (t * CS + ks) * 512);
    }
    // the wave's tokens of a lower (upper) triangle: steps 0 .. w / 2 (w / 2 ..), the last one twice where there is one alone
    template <bool UPPER, int N> __device__ __forceinline__ void load_steps(const void *from, const DeltaArgs &a, int n, D8 (&to)[CS][N]) const
    {
        const T *p = static_cast<const T *>(from) + ((int64_t)pair * a.chunks + n) * (DC::kSteps * N * 512) + lane * 8;
#pragma unroll
        for (int ks = 0; ks < CS; ++ks) {
            const int t = CS == 1 ? min(w, CT - 1) : w, step = UPPER ? DC::upper(t, max(ks, t / 2)) : DC::lower(t, min(ks, t / 2));
#pragma unroll
            for (int i = 0; i < N; ++i) to[ks][i] = ld8(p + (step * N + i) * 512);
        }
    }
    // the lane's columns of values or their cotangents, tokens 16w + 4c + e
    __device__ __forceinline__ void load_values(const DecayRows &x, int n, Cols (&to)[NG / NC][4]) const
    {
        const T *p = static_cast<const T *>(x.p) + b * x.sb + h * x.sh;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const T *row = p + (int64_t)min(n * C + 16 * w + 4 * c + e, len - 1) * x.st;
#pragma unroll
            for (int g = 0; g < NG; g += NC) to[g / NC][e] = *reinterpret_cast<const Cols *>(row + (mine(g) ? column(g) : 0));
        }
    }
    __device__ __forceinline__ float value(const Cols (&v)[NG / NC][4], int n, int g, int e) const
    {
        return mine(g) && n * C + 16 * w + 4 * c + e < len ? column_of<T, NC>(v[g / NC][e], g % NC) : 0.f;
    }
    // e^{L_i}, e^{L_C - L_i} and b_i of the wave's tokens
    struct Gates {
        f32x4 start, end, beta;
        float at_start, whole;                   // of token r
    };
    __device__ __forceinline__ void load_gates(const DeltaArgs &a, int n, Gates &to) const
    {
        const float *gate = a.to.gates + ((int64_t)pair * a.chunks + n) * DC::kGates;
        const int t = 16 * min(w, CT - 1);
        to.start = *reinterpret_cast<const f32x4 *>(gate + t + 4 * c);
        to.end = *reinterpret_cast<const f32x4 *>(gate + C + t + 4 * c);
        to.beta = *reinterpret_cast<const f32x4 *>(gate + 2 * C + t + 4 * c);
        to.at_start = gate[t + r];
        to.whole = gate[3 * C];
    }
    // x or the cotangents of u: the four tokens of a column
    __device__ __forceinline__ int64_t written(int n, int g) const
    {
        return (((int64_t)n * (DV >> 4) + (column(g) >> 4)) * CT + w) * 256 + (c * 16 + (column(g) & 15)) * 4;
    }
    // ---- operands in LDS: [group][step][part][lane][8], a wave's accumulators being half of a step ----
    template <int STEPS, int N> static __device__ __forceinline__ void put(T *to, int g, int t, int lane, f32x4 v)
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const Four f = pack_results<T>(v);
            *reinterpret_cast<Four *>(to + (((g * STEPS + (t >> 1)) * N + i) * 64 + lane) * 8 + 4 * (t & 1)) = f;
            if (i + 1 < N)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] -= (float)f[e];
        }
    }
    template <int STEPS, int N, int M> static __device__ __forceinline__ void get(const T *from, int g, int step, int lane, D8 (&to)[M])
    {
#pragma unroll
        for (int i = 0; i < M; ++i) to[i] = ld8(from + (((g * STEPS + step) * N + i) * 64 + lane) * 8);
    }
    template <int N> __device__ __forceinline__ void put_state(T *to) const
    {
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int p = 0; p < PER; ++p) put<KS, N>(to, g, w * PER + p, lane, S[g][p]);
    }
};

// Forward.  An operand's registers are filled for the next chunk as soon as this chunk's products have taken it.
template <typename T, int DKP, int NG, bool KEEP>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void delta_walk_kernel(const DeltaArgs a)
{
    typedef Walk<T, DKP, NG> W;
    typedef typename W::DC DC;
    typedef typename W::D8 D8;
    constexpr int C = W::C, CT = W::CT, CS = W::CS, KS = W::KS, PER = W::PER, NC = W::NC, kParts = DC::kParts, kFew = DC::kFew;
    extern __shared__ char smem[];
    T *sS = reinterpret_cast<T *>(smem), *sR = sS + NG * KS * kFew * 512, *sU = sR + NG * CS * kParts * 512, *sO = sU + NG * CS * kParts * 512;
    W w;
    if (w.place(a)) return;
    const int r = w.r, c = w.c, lane = w.lane;
    const bool tokens = w.w < CT;
    w.load_state(a.hidden, a.hidden_dtype);
    float *kept = KEEP ? a.kept + w.pair * (delta_states_floats(a.n, a.chunks) + delta_written_floats(a.n, a.chunks, C)) : nullptr;
    float *xs = KEEP ? kept + delta_states_floats(a.n, a.chunks) : nullptr;
    auto keep = [&](int n) {
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int p = 0; p < PER; ++p)
                if (w.mine(g) && w.feature(p) < w.DK)
                    *reinterpret_cast<f32x4 *>(kept + ((int64_t)n * w.DV + w.column(g)) * w.DK + w.feature(p)) = w.S[g][p];
    };
    D8 K[KS], Q[KS], KT[PER][CS], Z[CS][kParts], P[CS][1];
    typename W::Cols V[NG / NC][4];
    typename W::Gates next_gates;
    T *out = static_cast<T *>(a.out) + (w.b * w.T_ * a.n.H + w.h) * w.DV;
    const int64_t row = a.n.H * w.DV;
    auto store = [&](int token, auto values) {   // the lane's columns of a token, 4 NC of each NC groups
#pragma unroll
        for (int g = 0; g < NG; g += NC) {
            const int at = w.col0 + 16 * g + 4 * NC * c;
            float v[4 * NC];
#pragma unroll
            for (int i = 0; i < 4 * NC; ++i) v[i] = values(g + i % NC, i / NC);
            if (at < w.DV && token < w.T_) store_vec<T, 4 * NC>(out + token * row + at, v);
        }
    };
    if (w.live > 0) {
        w.load_gates(a, 0, next_gates);
        w.load_rows(a.keys, 0, K);
        w.load_rows(a.queries, 0, Q);
        w.load_values(a.values, 0, V);
        w.template load_steps<false>(a.to.inverse, a, 0, Z);
        w.template load_steps<false>(a.to.scores, a, 0, P);
        w.load_features(a.to.keys, a, 0, KT);
    }
    w.template put_state<kFew>(sS);
    for (int n = 0; n < w.live; ++n) {
        const int next = min(n + 1, w.live - 1);
        const typename W::Gates gate = next_gates;
        w.load_gates(a, next, next_gates);
        if constexpr (KEEP) keep(n);
        f32x4 x[NG], o[NG];
        lds_barrier();                           // the state's operands are there
        if (tokens) {
            // S^T k, and S^T q the other way round
#pragma unroll
            for (int g = 0; g < NG; ++g) x[g] = o[g] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    D8 s[kFew];
                    W::template get<KS, kFew>(sS, g, ks, lane, s);
                    x[g] = mma_whole(K[ks], s, x[g]);
                    o[g] = mma_whole(s, Q[ks], o[g]);
                }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[g][e] = w.value(V, n, g, e) - gate.start[e] * x[g][e];
                W::template put<CS, kParts>(sR, g, w.w, lane, x[g]);
            }
            w.load_rows(a.keys, next, K);
            w.load_rows(a.queries, next, Q);
            w.load_values(a.values, next, V);
        }
        lds_barrier();                           // r
        if (tokens) {
#pragma unroll
            for (int g = 0; g < NG; ++g) x[g] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < CS; ++ks)
                if (ks <= w.w / 2)
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        D8 v[kParts];
                        W::template get<CS, kParts>(sR, g, ks, lane, v);
                        x[g] = mma_parts(Z[ks], v, x[g]);
                    }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                f32x4 u, weighted;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    u[e] = gate.beta[e] * x[g][e];
                    weighted[e] = gate.end[e] * u[e];
                }
                W::template put<CS, kParts>(sU, g, w.w, lane, weighted);
                W::template put<CS, 1>(sO, g, w.w, lane, u);
                if constexpr (KEEP)
                    if (w.mine(g)) *reinterpret_cast<f32x4 *>(xs + w.written(n, g)) = x[g];
            }
            w.template load_steps<false>(a.to.inverse, a, next, Z);
        }
        lds_barrier();                           // u
        // the state behind the chunk
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int p = 0; p < PER; ++p)
#pragma unroll
                for (int e = 0; e < 4; ++e) w.S[g][p][e] *= gate.whole;
#pragma unroll
        for (int ks = 0; ks < CS; ++ks)
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                D8 u[kParts];
                W::template get<CS, kParts>(sU, g, ks, lane, u);
#pragma unroll
                for (int p = 0; p < PER; ++p) w.S[g][p] = mma_whole(KT[p][ks], u, w.S[g][p]);
            }
        w.load_features(a.to.keys, a, next, KT);
        w.template put_state<kFew>(sS);
        if (tokens) {
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[g][e] *= gate.at_start;
#pragma unroll
            for (int ks = 0; ks < CS; ++ks)
                if (ks <= w.w / 2)
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        D8 u[1];
                        W::template get<CS, 1>(sO, g, ks, lane, u);
                        o[g] = mma_d(u[0], P[ks][0], o[g]);
                    }
            w.template load_steps<false>(a.to.scores, a, next, P);
            const int token = n * C + 16 * w.w + r;
            store(token, [&](int g, int e) { return token < w.len ? o[g][e] : 0.f; });
        }
    }
    // rows past the end of a shorter sequence
    for (int token = w.live * C + 16 * w.w + r; token < w.T_; token += 16 * W::kWaves) store(token, [](int, int) { return 0.f; });
    if constexpr (KEEP) keep(w.live);
    w.store_state(a.hidden_out, a.hidden_dtype);
}

// Backward, from the last chunk to the first.  With dS the cotangent of the state behind a chunk and du that of u from what reads u,
//       du_j = sum_{i>=j} P_ij do_i + e^{L_C - L_j} dS^T k_j,   du <- (1 + b M)^{-T} du,   dv = dr = b du,
//       dS  <- e^{L_C} dS + sum_i e^{L_i} (q_i do_i^T - k_i dv_i^T).
template <typename T, int DKP, int NG>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void delta_walk_back_kernel(const DeltaArgs a)
{
    typedef Walk<T, DKP, NG> W;
    typedef typename W::DC DC;
    typedef typename W::D8 D8;
    constexpr int C = W::C, CT = W::CT, CS = W::CS, KS = W::KS, PER = W::PER, NC = W::NC, kParts = DC::kParts;
    constexpr int kRows = NG * CS * kParts * 512;
    extern __shared__ char smem[];
    // the cotangents of the state, of u before the system is solved, of out and of r (the last two scaled), and of out as it is
    T *sS = reinterpret_cast<T *>(smem), *sU = sS + NG * KS * kParts * 512, *sO = sU + kRows, *sR = sO + kRows, *sD = sR + kRows;
    W w;
    if (w.place(a)) return;
    const int lane = w.lane;
    const bool tokens = w.w < CT;
    w.load_state(a.hidden, a.hidden_dtype);
    const float *kept = a.kept + w.pair * (delta_states_floats(a.n, a.chunks) + delta_written_floats(a.n, a.chunks, C));
    float *dus = a.du + w.pair * delta_written_floats(a.n, a.chunks, C);
    T *dstates = static_cast<T *>(a.dstates) + w.pair * a.chunks * a.n.DK * a.n.DV;
    D8 K[KS], KT[PER][CS], QT[PER][CS], Z[CS][kParts], P[CS][kParts];
    typename W::Cols O[NG / NC][4];
    typename W::Gates next_gates;
    f32x4 S[NG][PER];
    auto load_kept = [&](int n) {
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int p = 0; p < PER; ++p) {
                const bool is = w.mine(g) && w.feature(p) < w.DK;
                S[g][p] = *reinterpret_cast<const f32x4 *>(kept + ((int64_t)n * w.DV + (is ? w.column(g) : 0)) * w.DK + (is ? w.feature(p) : 0));
            }
    };
    if (w.live > 0) {
        const int n = w.live - 1;
        w.load_gates(a, n, next_gates);
        load_kept(n + 1);
        w.load_values(a.dout, n, O);
        w.load_rows(a.keys, n, K);
        w.template load_steps<true>(a.to.scores, a, n, P);
        w.template load_steps<true>(a.to.inverse, a, n, Z);
        w.load_features(a.to.queries, a, n, QT);
        w.load_features(a.to.keys, a, n, KT);
    }
    for (int n = w.live - 1; n >= 0; --n) {
        const int next = max(n - 1, 0);
        const typename W::Gates gate = next_gates;
        w.load_gates(a, next, next_gates);
        // the cotangent of the state behind the chunk, for the gradients; its product with that state
        w.template put_state<kParts>(sS);
        float *dots = a.dots + (((int64_t)w.pair * a.chunks + n) * (w.DV >> 4) + (w.col0 >> 4)) * 4 + w.w;
#pragma unroll
        for (int g = 0; g < NG; g += NC) {
            float dot = 0.f;
#pragma unroll
            for (int q = g; q < g + NC; ++q)
#pragma unroll
                for (int p = 0; p < PER; ++p)
                    if (w.mine(q) && w.feature(p) < w.DK) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) dot += w.S[q][p][e] * S[q][p][e];
                        *reinterpret_cast<typename W::Four *>(dstates + ((int64_t)n * w.DV + w.column(q)) * w.DK + w.feature(p)) = pack_results<T>(w.S[q][p]);
                    }
            dot = sum_over_c(sum_over_r(dot));
            if (lane == 0)
                for (int q = 0; q < NC; ++q)
                    if (w.col0 + 16 * (g + q) < w.DV) dots[4 * (g + q)] = q ? 0.f : dot;
        }
        load_kept(n);
        if (tokens) {
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                f32x4 o, scaled;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    o[e] = w.value(O, n, g, e);
                    scaled[e] = gate.start[e] * o[e];
                }
                W::template put<CS, 1>(sD, g, w.w, lane, o);
                W::template put<CS, kParts>(sO, g, w.w, lane, scaled);
            }
            w.load_values(a.dout, next, O);
        }
        lds_barrier();                           // dS and do
        f32x4 du[NG];
        if (tokens) {
#pragma unroll
            for (int g = 0; g < NG; ++g) du[g] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    D8 s[kParts];
                    W::template get<KS, kParts>(sS, g, ks, lane, s);
                    du[g] = mma_whole(K[ks], s, du[g]);
                }
            w.load_rows(a.keys, next, K);
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int e = 0; e < 4; ++e) du[g][e] *= gate.end[e];
#pragma unroll
            for (int ks = 0; ks < CS; ++ks)
                if (ks >= w.w / 2 || CS == 1)
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        D8 o[1];
                        W::template get<CS, 1>(sD, g, ks, lane, o);
                        du[g] = mma_whole(P[ks], o[0], du[g]);
                    }
            w.template load_steps<true>(a.to.scores, a, next, P);
#pragma unroll
            for (int g = 0; g < NG; ++g) W::template put<CS, kParts>(sU, g, w.w, lane, du[g]);
        }
        lds_barrier();                           // du
        if (tokens) {
#pragma unroll
            for (int g = 0; g < NG; ++g) du[g] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < CS; ++ks)
                if (ks >= w.w / 2 || CS == 1)
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        D8 u[kParts];
                        W::template get<CS, kParts>(sU, g, ks, lane, u);
                        du[g] = mma_parts(Z[ks], u, du[g]);
                    }
            w.template load_steps<true>(a.to.inverse, a, next, Z);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = -gate.start[e] * (gate.beta[e] * du[g][e]);
                W::template put<CS, kParts>(sR, g, w.w, lane, v);
                if (w.mine(g)) *reinterpret_cast<f32x4 *>(dus + w.written(n, g)) = du[g];
            }
        }
        lds_barrier();                           // dr
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int p = 0; p < PER; ++p)
#pragma unroll
                for (int e = 0; e < 4; ++e) w.S[g][p][e] *= gate.whole;
#pragma unroll
        for (int ks = 0; ks < CS; ++ks)
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                D8 o[kParts], v[kParts];
                W::template get<CS, kParts>(sO, g, ks, lane, o);
                W::template get<CS, kParts>(sR, g, ks, lane, v);
#pragma unroll
                for (int p = 0; p < PER; ++p) w.S[g][p] = mma_whole(QT[p][ks], o, w.S[g][p]);
#pragma unroll
                for (int p = 0; p < PER; ++p) w.S[g][p] = mma_whole(KT[p][ks], v, w.S[g][p]);
            }
        w.load_features(a.to.queries, a, next, QT);
        w.load_features(a.to.keys, a, next, KT);
        lds_barrier();                           // what the next chunk's operands take the place of is read
    }
    w.store_state(a.hidden_out, a.hidden_dtype);
}

template <typename T, int DKP, int NG> int launch_walk(hipStream_t stream, const DeltaArgs &a, bool backward)
{
    typedef Walk<T, DKP, NG> W;
    typedef DeltaChunk<T> DC;
    // the columns of a pair share a die, to which workgroups are dealt in turn
    const dim3 grid((unsigned)((a.pairs + 7) / 8 * 8), (unsigned)((a.n.DV + 16 * NG - 1) / (16 * NG)));
    constexpr size_t lds = sizeof(T) * 512 * NG * (W::KS * DC::kFew + W::CS * (2 * DC::kParts + 1));
    constexpr size_t lds_back = sizeof(T) * 512 * NG * (W::KS * DC::kParts + W::CS * (3 * DC::kParts + 1));
    static_assert(lds_back <= 160 * 1024, "");
    static LdsGrant grants[3];
    if (backward) {
        if (int e = allow_lds(grants[0], reinterpret_cast<const void *>(delta_walk_back_kernel<T, DKP, NG>), lds_back)) return e;
        delta_walk_back_kernel<T, DKP, NG><<<grid, 256, lds_back, stream>>>(a);
    } else if (a.kept) {
        if (int e = allow_lds(grants[1], reinterpret_cast<const void *>(delta_walk_kernel<T, DKP, NG, true>), lds)) return e;
        delta_walk_kernel<T, DKP, NG, true><<<grid, 256, lds, stream>>>(a);
    } else {
        if (int e = allow_lds(grants[2], reinterpret_cast<const void *>(delta_walk_kernel<T, DKP, NG, false>), lds)) return e;
        delta_walk_kernel<T, DKP, NG, false><<<grid, 256, lds, stream>>>(a);
    }
    return launch_status();
}
// Value columns of a workgroup: 64 share the operands' way from memory, 16 make four times the workgroups.
template <typename T, int DKP> int choose_walk(hipStream_t stream, const DeltaArgs &a, bool backward)
{
    const int64_t groups = a.pairs * ((a.n.DV + 15) / 16);
    if (a.n.DV > 32 && groups >= 8 * kComputeUnits) return launch_walk<T, DKP, 4>(stream, a, backward);
    if (a.n.DV > 16 && groups >= 4 * kComputeUnits) return launch_walk<T, DKP, 2>(stream, a, backward);
    return launch_walk<T, DKP, 1>(stream, a, backward);
}
template <typename T> int dispatch_walk(hipStream_t stream, const DeltaArgs &a, bool backward)
{
    return a.n.DK <= 64 ? choose_walk<T, 64>(stream, a, backward) : choose_walk<T, 128>(stream, a, backward);
}

}  // namespace

int delta_walk(void *stream, const DeltaArgs &a, gla_dtype dtype, bool backward)
{
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == GLA_BF16 ? dispatch_walk<__bf16>(s, a, backward) : dispatch_walk<float>(s, a, backward);
}

}  // namespace gla
