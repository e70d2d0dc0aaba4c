// The gated delta rule: the walks over the chunks, forward with the state and backward with its cotangent.
#include "gla_delta.hpp"

namespace gla {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <typename T, int N> struct Columns { typedef T t __attribute__((ext_vector_type(N))); };
template <typename T> struct Columns<T, 1> { typedef T t; };
template <typename T, int N> __device__ __forceinline__ float column_of(typename Columns<T, N>::t v, int q)
{
    if constexpr (N == 1) return (float)v;
    else return (float)v[q];
}

// Of packed results the values that they stand for, without the conversions done again.
__device__ __forceinline__ f32x4 unpack_results(bf16x4 v)
{
    const auto u = __builtin_bit_cast(u32x2, v);
    return {__uint_as_float(u[0] << 16), __uint_as_float(u[0] & 0xffff0000u), __uint_as_float(u[1] << 16), __uint_as_float(u[1] & 0xffff0000u)};
}
__device__ __forceinline__ f32x4 unpack_results(f32x4 v) { return v; }

// Rows of a chunk as the load instructions see them: what lies behind the last row reads as zero, and a lane keeps one 32-bit place for
// the whole walk.
constexpr unsigned kNowhere = 0x7fffff00u;       // (rows of a chunk take at most 2^30 bytes)
template <typename Cols> __device__ __forceinline__ Cols load_columns(__amdgpu_buffer_rsrc_t rows, unsigned at)
{
    if constexpr (sizeof(Cols) == 2) return __builtin_bit_cast(Cols, __builtin_amdgcn_raw_buffer_load_b16(rows, at, 0, 0));
    else if constexpr (sizeof(Cols) == 4) return __builtin_bit_cast(Cols, __builtin_amdgcn_raw_buffer_load_b32(rows, at, 0, 0));
    else return __builtin_bit_cast(Cols, __builtin_amdgcn_raw_buffer_load_b64(rows, at, 0, 0));
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
    // an array's rows: its first one, and a lane's place in a chunk's
    struct Rows {
        const T *p;
        int st;
        unsigned at[4];
    };
    // true: there is nothing to do
    __device__ __forceinline__ bool place(const DeltaArgs &a)
    {
        tid = threadIdx.x;
        w = __builtin_amdgcn_readfirstlane(tid >> 6);
        lane = tid & 63;
        r = lane & 15;
        c = lane >> 4;
        DK = (int)a.n.DK;
        DV = (int)a.n.DV;
        const unsigned groups = ((unsigned)DV + 16 * NG - 1) / (16 * NG), turn = blockIdx.x / 8;
        pair = turn / groups * 8 + blockIdx.x % 8;
        col0 = (int)(turn % groups) * 16 * NG;
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
        auto load = [&](auto *rows) {            // (every lane loads, so that no load waits for another)
            typedef std::remove_const_t<std::remove_pointer_t<decltype(rows)>> H;
#pragma unroll
            for (int g = 0; g < NG; g += NC)
#pragma unroll
                for (int p = 0; p < PER; ++p)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool is = mine(g) && feature(p) < DK;
                        float x[NC];
                        load_vec<H, NC>(rows + ((int64_t)pair * DK + (is ? feature(p) + e : 0)) * DV + (is ? column(g) : 0), x);
#pragma unroll
                        for (int q = 0; q < NC; ++q) S[g + q][p][e] = is ? x[q] : 0.f;
                    }
        };
        if (dtype == GLA_BF16) load(static_cast<const __bf16 *>(from));
        else load(static_cast<const float *>(from));
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
    // the wave's tokens of keys or queries, features as the contracted index in their order
    __device__ __forceinline__ void load_rows(const void *from, const DeltaArgs &a, int n, D8 (&to)[KS]) const
    {
        const T *p = static_cast<const T *>(from) + ((b * a.n.HK + hk) * a.chunks + n) * (CT * KS * 512) + min(w, CT - 1) * KS * 512;
        const unsigned at = lane * 8 * (unsigned)sizeof(T);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) to[ks] = ld8(at_bytes(p + ks * 512, at));
    }
    // the wave's features of keys or queries, tokens as the contracted index
    __device__ __forceinline__ void load_features(const void *from, const DeltaArgs &a, int n, D8 (&to)[PER][CS]) const
    {
        const T *p = static_cast<const T *>(from) + ((b * a.n.HK + hk) * a.chunks + n) * (TILES * CS * 512) + w * PER * CS * 512;
        const unsigned at = lane * 8 * (unsigned)sizeof(T);
#pragma unroll
        for (int t = 0; t < PER; ++t)
#pragma unroll
            for (int ks = 0; ks < CS; ++ks) to[t][ks] = ld8(at_bytes(p + (t * CS + ks) * 512, at));
    }
    // the wave's tokens of a lower (upper) triangle: steps 0 .. w / 2 (w / 2 ..), the last one twice where there is one alone
    template <bool UPPER, int N> __device__ __forceinline__ void load_steps(const void *from, const DeltaArgs &a, int n, D8 (&to)[CS][N]) const
    {
        const T *p = static_cast<const T *>(from) + ((int64_t)pair * a.chunks + n) * (DC::kSteps * N * 512);
        const unsigned at = lane * 8 * (unsigned)sizeof(T);
#pragma unroll
        for (int ks = 0; ks < CS; ++ks) {
            const int t = CS == 1 ? min(w, CT - 1) : w, step = UPPER ? DC::upper(t, max(ks, t / 2)) : DC::lower(t, min(ks, t / 2));
#pragma unroll
            for (int i = 0; i < N; ++i) to[ks][i] = ld8(at_bytes(p + (step * N + i) * 512, at));
        }
    }
    // the lane's columns of values or their cotangents, tokens 16w + 4c + e; columns behind the last are whatever is there, and stay by themselves
    __device__ __forceinline__ Rows value_rows(const DecayRows &x) const
    {
        Rows y{static_cast<const T *>(x.p) + b * x.sb + h * x.sh, (int)x.st, {}};
#pragma unroll
        for (int e = 0; e < 4; ++e) y.at[e] = (unsigned)((16 * min(w, CT - 1) + 4 * c + e) * y.st + column(0)) * (unsigned)sizeof(T);
        return y;
    }
    __device__ __forceinline__ void load_values(const Rows &x, int n, Cols (&to)[NG / NC][4]) const
    {
        // (at most 2^30 bytes)
        const auto rows = __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(x.p + (int64_t)n * C * x.st), 0,
                                                            ((min(C, len - n * C) - 1) * x.st + DV) * (int)sizeof(T), 0x00027000);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int g = 0; g < NG; g += NC) to[g / NC][e] = load_columns<Cols>(rows, x.at[e] + 16 * g * (unsigned)sizeof(T));
    }
    static __device__ __forceinline__ float value(const Cols (&v)[NG / NC][4], int g, int e) { return column_of<T, NC>(v[g / NC][e], g % NC); }
    // of the chunk's gates: e^{L_i} (0), e^{L_C - L_i} (1) or b_i (2) of the wave's tokens 4c .., e^{L_i} of token r, e^{L_C}
    __device__ __forceinline__ const float *gates(const DeltaArgs &a, int n) const { return a.to.gates + ((int64_t)pair * a.chunks + n) * DC::kGates; }
    __device__ __forceinline__ f32x4 gate(const DeltaArgs &a, int n, int kind) const
    {
        return *reinterpret_cast<const f32x4 *>(at_bytes(gates(a, n) + kind * C + 16 * min(w, CT - 1), 16u * c));
    }
    __device__ __forceinline__ float gate_r(const DeltaArgs &a, int n) const { return *at_bytes(gates(a, n) + 16 * min(w, CT - 1), 4u * r); }
    __device__ __forceinline__ float gate_whole(const DeltaArgs &a, int n) const { return *at_bytes(gates(a, n) + 3 * C, again(0)); }
    // x or the cotangents of u: the four tokens of a column
    __device__ __forceinline__ int64_t written(int n, int g) const
    {
        return (((int64_t)n * (DV >> 4) + (column(g) >> 4)) * CT + w) * 256 + (c * 16 + (column(g) & 15)) * 4;
    }
    // states: the four features of a column
    __device__ __forceinline__ int64_t state_place(int n, int g, int p) const
    {
        return (((int64_t)n * (DV >> 4) + (column(g) >> 4)) * delta_state_tiles(DK) + (w * PER + p)) * 256 + (c * 16 + (column(g) & 15)) * 4;
    }
    // ---- operands in LDS: [group][step][part][lane][8], a wave's accumulators being half of a step ----
    template <int STEPS, int N> static __device__ __forceinline__ void put(T *to, int g, int t, int lane, f32x4 v)
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const Four f = pack_results<T>(v);
            *reinterpret_cast<Four *>(to + (((g * STEPS + (t >> 1)) * N + i) * 64 + lane) * 8 + 4 * (t & 1)) = f;
            if (i + 1 < N) {
                const f32x4 taken = unpack_results(f);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] -= taken[e];
            }
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
    const bool tokens = CT == W::kWaves || w.w < CT;
    w.load_state(a.hidden, a.hidden_dtype);
    float *kept = KEEP ? a.kept + w.pair * (delta_states_floats(a.n, a.chunks) + delta_written_floats(a.n, a.chunks, C)) : nullptr;
    float *xs = KEEP ? kept + delta_states_floats(a.n, a.chunks) : nullptr;
    auto keep = [&](int n) {
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int p = 0; p < PER; ++p)
                if (w.mine(g) && w.feature(p) < w.DK)
                    *reinterpret_cast<f32x4 *>(kept + w.state_place(n, g, p)) = w.S[g][p];
    };
    D8 K[KS], Q[KS], KT[PER][CS], Z[CS][kParts], P[CS][1];
    typename W::Cols V[NG / NC][4];
    const typename W::Rows values = w.value_rows(a.values);
    f32x4 start, end, beta;
    float at_start, whole;
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
        w.load_rows(a.to.key_rows, a, 0, K);
        w.load_rows(a.to.query_rows, a, 0, Q);
        w.load_values(values, 0, V);
        start = w.gate(a, 0, 0);
        end = w.gate(a, 0, 1);
        beta = w.gate(a, 0, 2);
        whole = w.gate_whole(a, 0);
        at_start = w.gate_r(a, 0);
        w.template load_steps<false>(a.to.inverse, a, 0, Z);
        w.template load_steps<false>(a.to.scores, a, 0, P);
        w.load_features(a.to.keys, a, 0, KT);
    }
    w.template put_state<kFew>(sS);
    for (int n = 0; n < w.live; ++n) {
        const int next = min(n + 1, w.live - 1);
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
                for (int e = 0; e < 4; ++e) x[g][e] = W::value(V, g, e) - start[e] * x[g][e];
                W::template put<CS, kParts>(sR, g, w.w, lane, x[g]);
            }
        }
        w.load_rows(a.to.key_rows, a, next, K);
        w.load_rows(a.to.query_rows, a, next, Q);
        w.load_values(values, next, V);
        start = w.gate(a, next, 0);
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
                    u[e] = beta[e] * x[g][e];
                    weighted[e] = end[e] * u[e];
                }
                W::template put<CS, kParts>(sU, g, w.w, lane, weighted);
                W::template put<CS, kFew>(sO, g, w.w, lane, u);
                if constexpr (KEEP)
                    if (w.mine(g)) *reinterpret_cast<f32x4 *>(xs + w.written(n, g)) = x[g];
            }
        }
        w.template load_steps<false>(a.to.inverse, a, next, Z);
        end = w.gate(a, next, 1);
        beta = w.gate(a, next, 2);
        lds_barrier();                           // u
        // the state behind the chunk
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int p = 0; p < PER; ++p)
#pragma unroll
                for (int e = 0; e < 4; ++e) w.S[g][p][e] *= whole;
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
        whole = w.gate_whole(a, next);
        w.template put_state<kFew>(sS);
        if (tokens) {
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[g][e] *= at_start;
#pragma unroll
            for (int ks = 0; ks < CS; ++ks)
                if (ks <= w.w / 2)
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        D8 u[kFew];
                        W::template get<CS, kFew>(sO, g, ks, lane, u);
                        o[g] = mma_whole(u, P[ks][0], o[g]);
                    }
            const int token = n * C + 16 * w.w + r;
            store(token, [&](int g, int e) { return token < w.len ? o[g][e] : 0.f; });
        }
        w.template load_steps<false>(a.to.scores, a, next, P);
        at_start = w.gate_r(a, next);
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
    const bool tokens = CT == W::kWaves || w.w < CT;
    w.load_state(a.hidden, a.hidden_dtype);
    const float *kept = a.kept + w.pair * (delta_states_floats(a.n, a.chunks) + delta_written_floats(a.n, a.chunks, C));
    float *dus = a.du + w.pair * delta_written_floats(a.n, a.chunks, C);
    T *dstates = static_cast<T *>(a.dstates) + w.pair * a.chunks * delta_state_floats(a.n);
    D8 K[KS], KT[PER][CS], QT[PER][CS], Z[CS][kParts], P[CS][kParts];
    typename W::Cols O[NG / NC][4];
    const typename W::Rows douts = w.value_rows(a.dout);
    f32x4 start, end, beta;
    float whole;
    f32x4 S[NG][PER];
    auto load_kept = [&](int n) {
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int p = 0; p < PER; ++p) {
                const bool is = w.mine(g) && w.feature(p) < w.DK;
                S[g][p] = *reinterpret_cast<const f32x4 *>(kept + (is ? w.state_place(n, g, p) : 0));
            }
    };
    if (w.live > 0) {
        const int n = w.live - 1;
        load_kept(n + 1);
        w.load_values(douts, n, O);
        w.load_rows(a.to.key_rows, a, n, K);
        start = w.gate(a, n, 0);
        end = w.gate(a, n, 1);
        beta = w.gate(a, n, 2);
        whole = w.gate_whole(a, n);
        w.template load_steps<true>(a.to.scores, a, n, P);
        w.template load_steps<true>(a.to.inverse, a, n, Z);
        w.load_features(a.to.queries, a, n, QT);
        w.load_features(a.to.keys, a, n, KT);
    }
    for (int n = w.live - 1; n >= 0; --n) {
        const int next = max(n - 1, 0);
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
                        *reinterpret_cast<typename W::Four *>(dstates + w.state_place(n, q, p)) = pack_results<T>(w.S[q][p]);
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
                    o[e] = W::value(O, g, e);
                    scaled[e] = start[e] * o[e];
                }
                W::template put<CS, 1>(sD, g, w.w, lane, o);
                W::template put<CS, kParts>(sO, g, w.w, lane, scaled);
            }
        }
        w.load_values(douts, next, O);
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
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int e = 0; e < 4; ++e) du[g][e] *= end[e];
#pragma unroll
            for (int ks = 0; ks < CS; ++ks)
                if (ks >= w.w / 2 || CS == 1)
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        D8 o[1];
                        W::template get<CS, 1>(sD, g, ks, lane, o);
                        du[g] = mma_whole(P[ks], o[0], du[g]);
                    }
#pragma unroll
            for (int g = 0; g < NG; ++g) W::template put<CS, kParts>(sU, g, w.w, lane, du[g]);
        }
        w.load_rows(a.to.key_rows, a, next, K);
        w.template load_steps<true>(a.to.scores, a, next, P);
        end = w.gate(a, next, 1);
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
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = -start[e] * (beta[e] * du[g][e]);
                W::template put<CS, kParts>(sR, g, w.w, lane, v);
                if (w.mine(g)) *reinterpret_cast<f32x4 *>(dus + w.written(n, g)) = du[g];
            }
        }
        w.template load_steps<true>(a.to.inverse, a, next, Z);
        start = w.gate(a, next, 0);
        beta = w.gate(a, next, 2);
        lds_barrier();                           // dr
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int p = 0; p < PER; ++p)
#pragma unroll
                for (int e = 0; e < 4; ++e) w.S[g][p][e] *= whole;
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
        whole = w.gate_whole(a, next);
        lds_barrier();                           // what the next chunk's operands take the place of is read
    }
    w.store_state(a.hidden_out, a.hidden_dtype);
}

template <typename T, int DKP, int NG> int launch_walk(hipStream_t stream, const DeltaArgs &a, bool backward)
{
    typedef Walk<T, DKP, NG> W;
    typedef DeltaChunk<T> DC;
    // the columns of a pair start next to each other on one die (workgroups are dealt to the eight in turn) and share what they read in its cache
    const unsigned grid = (unsigned)((a.pairs + 7) / 8 * 8 * ((a.n.DV + 16 * NG - 1) / (16 * NG)));
    constexpr size_t lds = sizeof(T) * 512 * NG * (W::KS * DC::kFew + W::CS * (2 * DC::kParts + DC::kFew));
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
