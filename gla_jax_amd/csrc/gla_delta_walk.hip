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

// What both walks share.  A workgroup holds NG times 16 value columns of one (batch, head) pair's state in the accumulators of four waves, its
// walkers: wave w has features 16 PER w .. as PER accumulators for each 16 columns, and of a chunk the tokens 16w .. (where there are so
// many).  Four helpers, one beside each walker on its SIMD, do what the next state does not wait for: they answer the queries, or, in the backward
// walk, prepare what the cotangent of out adds and leave what the gradients need.  Two groups of columns next to each other share 32: a
// lane's are 2r and 2r + 1, so that it reads two values and writes eight results at a time.
template <typename T, int DKP, int NG> struct Walk {
    typedef DeltaChunk<T> DC;
    typedef typename FragTypes<T>::d8 D8;
    typedef typename Packed4<T>::t Four;
    static constexpr int kWaves = 4, C = DC::C, CT = DC::CT, CS = DC::CS, TILES = DKP / 16, KS = DKP / 32, PER = TILES / kWaves;
    static constexpr int NC = NG > 1 ? 2 : 1;            // columns of a lane that lie next to each other
    typedef typename Columns<T, NC>::t Cols;
    int w, lane, r, c, DK, DV, T_, len, live, col0;
    unsigned pair;
    int64_t b, h, hk;
    bool helper;
    // an array's rows: its first one, and a lane's place in a chunk's
    struct Rows {
        const T *p;
        int st;
        unsigned at[4];
    };
    // true: there is nothing to do
    __device__ __forceinline__ bool place(const DeltaArgs &a)
    {
        w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        helper = w >= kWaves;
        w &= kWaves - 1;
        lane = threadIdx.x & 63;
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
    __device__ __forceinline__ bool tokens() const { return CT == kWaves || w < CT; }
    __device__ __forceinline__ int column(int g) const { return col0 + (NC == 2 ? 32 * (g >> 1) + 2 * r + (g & 1) : r); }
    __device__ __forceinline__ bool mine(int g) const { return column(g) < DV; }
    __device__ __forceinline__ int feature(int p) const      // of accumulator element 0
    {
        const int t = w * PER + p;
        return 32 * (t >> 1) + 8 * c + 4 * (t & 1);
    }
    __device__ __forceinline__ void load_state(const void *from, int dtype, f32x4 (&S)[NG][PER]) const
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
    __device__ __forceinline__ void store_state(void *to, int dtype, const f32x4 (&S)[NG][PER]) const
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
    // a prepared array's chunk: for each pair, or for each key head
    template <int SIZE> __device__ __forceinline__ const T *of_pair(const void *from, const DeltaArgs &a, int n) const
    {
        return static_cast<const T *>(from) + ((int64_t)pair * a.chunks + n) * SIZE;
    }
    template <int SIZE> __device__ __forceinline__ const T *of_key_head(const void *from, const DeltaArgs &a, int n) const
    {
        return static_cast<const T *>(from) + ((b * a.n.HK + hk) * a.chunks + n) * SIZE;
    }
    __device__ __forceinline__ D8 load_operand(const T *p) const { return ld8(at_bytes(p, lane * 8 * (unsigned)sizeof(T))); }
    // the wave's tokens of keys or queries, features as the contracted index in their order, step ks
    __device__ __forceinline__ D8 load_row(const void *from, const DeltaArgs &a, int n, int ks) const
    {
        return load_operand(of_key_head<CT * KS * 512>(from, a, n) + (min(w, CT - 1) * KS + ks) * 512);
    }
    // the wave's features of keys or queries, tokens as the contracted index
    __device__ __forceinline__ void load_features(const void *from, const DeltaArgs &a, int n, D8 (&to)[PER][CS]) const
    {
        const T *p = of_key_head<TILES * CS * 512>(from, a, n) + w * PER * CS * 512;
#pragma unroll
        for (int t = 0; t < PER; ++t)
#pragma unroll
            for (int ks = 0; ks < CS; ++ks) to[t][ks] = load_operand(p + (t * CS + ks) * 512);
    }
    // the wave's tokens of a lower (upper) triangle: steps 0 .. w / 2 (w / 2 ..), the last one twice where there is one alone
    template <bool UPPER, int N> __device__ __forceinline__ void load_steps(const void *from, const DeltaArgs &a, int n, D8 (&to)[CS][N]) const
    {
        const T *p = of_pair<DC::kSteps * N * 512>(from, a, n);
#pragma unroll
        for (int ks = 0; ks < CS; ++ks) {
            const int t = CS == 1 ? min(w, CT - 1) : w, step = UPPER ? DC::upper(t, max(ks, t / 2)) : DC::lower(t, min(ks, t / 2));
#pragma unroll
            for (int i = 0; i < N; ++i) to[ks][i] = load_operand(p + (step * N + i) * 512);
        }
    }
    // is step ks on this side of the diagonal?
    template <bool UPPER> __device__ __forceinline__ bool step(int ks) const { return CS == 1 || (UPPER ? ks >= w / 2 : ks <= w / 2); }
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
    // states: the four features 4c .. of tile t, a column
    __device__ __forceinline__ int64_t state_place(int n, int g, int t) const
    {
        return (((int64_t)n * (DV >> 4) + (column(g) >> 4)) * delta_state_tiles(DK) + t) * 256 + (c * 16 + (column(g) & 15)) * 4;
    }
    // cotangents of states: the eight features 8c .. of tiles 2 ks and 2 ks + 1, a column
    __device__ __forceinline__ int64_t cotangent_place(int n, int g, int ks) const
    {
        return (((int64_t)n * (DV >> 4) + (column(g) >> 4)) * (delta_state_tiles(DK) / 2) + ks) * 512 + (c * 16 + (column(g) & 15)) * 8;
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
    template <int N> __device__ __forceinline__ void put_state(T *to, const f32x4 (&S)[NG][PER]) const
    {
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int p = 0; p < PER; ++p) put<KS, N>(to, g, w * PER + p, lane, S[g][p]);
    }
    // ---- the three products of a walker's chunk ----
    // K S: the small parts' sum apart, so that products need not wait for each other; keys are loaded again as soon as they are used
    template <int N> __device__ __forceinline__ void keys_times_state(const DeltaArgs &a, int next, const T *state, D8 (&K)[KS], f32x4 (&x)[NG]) const
    {
        f32x4 low[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) x[g] = low[g] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            if (tokens())
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    D8 s[N];
                    get<KS, N>(state, g, ks, lane, s);
#pragma unroll
                    for (int i = N - 1; i >= 0; --i) {
                        f32x4 &to = i ? low[g] : x[g];
                        to = mma_d(K[ks], s[i], to);
                    }
                }
            K[ks] = load_row(a.to.key_rows, a, next, ks);
        }
        if constexpr (N > 1)
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[g][e] += low[g][e];
    }
    template <bool UPPER> __device__ __forceinline__ void solve(const DeltaArgs &a, int next, const T *rows, D8 (&Z)[CS][DC::kParts], f32x4 (&x)[NG]) const
    {
        constexpr int N = DC::kParts;
        if (tokens()) {
            f32x4 sum[NG][N];
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int i = 0; i < N; ++i) sum[g][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < CS; ++ks)
                if (step<UPPER>(ks))
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        D8 v[N];
                        get<CS, N>(rows, g, ks, lane, v);
#pragma unroll
                        for (int i = 0; i < N; ++i)
#pragma unroll
                            for (int s = i; s < N; ++s) sum[g][s] = mma_d(Z[ks][i], v[s - i], sum[g][s]);
                    }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                x[g] = sum[g][N - 1];
#pragma unroll
                for (int i = N - 2; i >= 0; --i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[g][e] += sum[g][i][e];
            }
        }
        load_steps<UPPER>(a.to.inverse, a, next, Z);
    }
    __device__ __forceinline__ void add_keys(const DeltaArgs &a, int next, const T *written, D8 (&KT)[PER][CS], f32x4 (&S)[NG][PER]) const
    {
#pragma unroll
        for (int ks = 0; ks < CS; ++ks)
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                D8 u[DC::kParts];
                get<CS, DC::kParts>(written, g, ks, lane, u);
#pragma unroll
                for (int i = DC::kParts - 1; i >= 0; --i)
#pragma unroll
                    for (int p = 0; p < PER; ++p) S[g][p] = mma_d(KT[p][ks], u[i], S[g][p]);
            }
        load_features(a.to.keys, a, next, KT);
    }
};

// Forward.  Three times a chunk the waves wait for each other: for the state's operands, r and u.
template <typename T, int DKP, int NG, bool KEEP> __global__ __launch_bounds__(512) void delta_walk_kernel(const DeltaArgs a)
{
    typedef Walk<T, DKP, NG> W;
    typedef typename W::DC DC;
    typedef typename W::D8 D8;
    constexpr int C = W::C, CS = W::CS, KS = W::KS, PER = W::PER, NC = W::NC, kParts = DC::kParts, kFew = DC::kFew;
    extern __shared__ char smem[];
    T *sS = reinterpret_cast<T *>(smem), *sR = sS + NG * KS * kFew * 512, *sU = sR + NG * CS * kParts * 512, *sO = sU + NG * CS * kParts * 512;
    W w;
    if (w.place(a)) return;
    const int lane = w.lane, last = w.live - 1;
    if (w.helper) {
        const int64_t row = a.n.H * w.DV;
        const unsigned places = (unsigned)((16 * w.w + w.r) * row);
        T *out = static_cast<T *>(a.out) + (w.b * w.T_ * a.n.H + w.h) * w.DV;
        auto store = [&](int from, auto values) {    // the lane's columns of token `from` + 16w + r, 4 NC of each NC groups
            T *to = at_bytes(out + from * row, places * (unsigned)sizeof(T));
#pragma unroll
            for (int g = 0; g < NG; g += NC) {
                const int at = w.col0 + 16 * g + 4 * NC * w.c;
                float v[4 * NC];
#pragma unroll
                for (int i = 0; i < 4 * NC; ++i) v[i] = values(g + i % NC, i / NC);
                if (at < w.DV && from + 16 * w.w + w.r < w.T_) store_vec<T, 4 * NC>(to + at, v);
            }
        };
        D8 Q[KS], P[CS][1];
        float at_start;
        if (w.live > 0) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) Q[ks] = w.load_row(a.to.query_rows, a, 0, ks);
            w.template load_steps<false>(a.to.scores, a, 0, P);
            at_start = w.gate_r(a, 0);
        }
        for (int n = 0; n < w.live; ++n) {
            const int next = min(n + 1, last);
            f32x4 o[NG];
            lds_barrier();                       // the state's operands are there
#pragma unroll
            for (int g = 0; g < NG; ++g) o[g] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                if (w.tokens())
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        D8 s[kFew];
                        W::template get<KS, kFew>(sS, g, ks, lane, s);
                        o[g] = mma_whole(s, Q[ks], o[g]);
                    }
                Q[ks] = w.load_row(a.to.query_rows, a, next, ks);
            }
            lds_barrier();                       // r
            lds_barrier();                       // u
            if (w.tokens()) {
#pragma unroll
                for (int g = 0; g < NG; ++g)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[g][e] *= at_start;
#pragma unroll
                for (int ks = 0; ks < CS; ++ks)
                    if (w.template step<false>(ks))
#pragma unroll
                        for (int g = 0; g < NG; ++g) {
                            D8 u[kFew];
                            W::template get<CS, kFew>(sO, g, ks, lane, u);
                            o[g] = mma_whole(u, P[ks][0], o[g]);
                        }
                const bool is = n * C + 16 * w.w + w.r < w.len;
                store(n * C, [&](int g, int e) { return is ? o[g][e] : 0.f; });
            }
            w.template load_steps<false>(a.to.scores, a, next, P);
            at_start = w.gate_r(a, next);
        }
        // rows past the end of a shorter sequence
        for (int from = w.live * C; from < w.T_; from += 16 * W::kWaves) store(from, [](int, int) { return 0.f; });
        return;
    }
    f32x4 S[NG][PER];
    w.load_state(a.hidden, a.hidden_dtype, S);
    float *kept = KEEP ? a.kept + w.pair * (delta_states_floats(a.n, a.chunks) + delta_written_floats(a.n, a.chunks, C)) : nullptr;
    float *xs = KEEP ? kept + delta_states_floats(a.n, a.chunks) : nullptr;
    auto keep = [&](int n) {
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int p = 0; p < PER; ++p)
                if (w.mine(g) && w.feature(p) < w.DK) *reinterpret_cast<f32x4 *>(kept + w.state_place(n, g, w.w * PER + p)) = S[g][p];
    };
    D8 K[KS], KT[PER][CS], Z[CS][kParts];
    typename W::Cols V[NG / NC][4];
    const typename W::Rows values = w.value_rows(a.values);
    f32x4 start, end, beta;
    float whole;
    if (w.live > 0) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) K[ks] = w.load_row(a.to.key_rows, a, 0, ks);
        w.load_values(values, 0, V);
        start = w.gate(a, 0, 0);
        w.template load_steps<false>(a.to.inverse, a, 0, Z);
        end = w.gate(a, 0, 1);
        beta = w.gate(a, 0, 2);
        w.load_features(a.to.keys, a, 0, KT);
        whole = w.gate_whole(a, 0);
    }
    w.template put_state<kFew>(sS, S);
    for (int n = 0; n < w.live; ++n) {
        const int next = min(n + 1, last);
        if constexpr (KEEP) keep(n);
        f32x4 x[NG];
        lds_barrier();                           // the state's operands are there
        w.template keys_times_state<kFew>(a, next, sS, K, x);
        if (w.tokens())
#pragma unroll
            for (int g = 0; g < NG; ++g) {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[g][e] = W::value(V, g, e) - start[e] * x[g][e];
                W::template put<CS, kParts>(sR, g, w.w, lane, x[g]);
            }
        w.load_values(values, next, V);
        start = w.gate(a, next, 0);
        lds_barrier();                           // r
        w.template solve<false>(a, next, sR, Z, x);
        if (w.tokens())
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
        end = w.gate(a, next, 1);
        beta = w.gate(a, next, 2);
        lds_barrier();                           // u
        // the state behind the chunk
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int p = 0; p < PER; ++p)
#pragma unroll
                for (int e = 0; e < 4; ++e) S[g][p][e] *= whole;
        w.add_keys(a, next, sU, KT, S);
        whole = w.gate_whole(a, next);
        w.template put_state<kFew>(sS, S);
    }
    if constexpr (KEEP) keep(w.live);
    w.store_state(a.hidden_out, a.hidden_dtype, S);
}

// Backward, from the last chunk to the first.  With dS the cotangent of the state behind a chunk and du that of u from what reads u,
//       du_j = sum_{i>=j} P_ij do_i + e^{L_C - L_j} dS^T k_j,   du <- (1 + b M)^{-T} du,   dv = dr = b du,
//       dS  <- e^{L_C} dS + sum_i e^{L_i} (q_i do_i^T - k_i dv_i^T).
// The helpers make the first sum and sum_i e^{L_i} q_i do_i^T, a chunk ahead.
template <typename T, int DKP, int NG> __global__ __launch_bounds__(512) void delta_walk_back_kernel(const DeltaArgs a)
{
    typedef Walk<T, DKP, NG> W;
    typedef typename W::DC DC;
    typedef typename W::D8 D8;
    constexpr int C = W::C, CT = W::CT, CS = W::CS, KS = W::KS, PER = W::PER, TILES = W::TILES, NC = W::NC, kParts = DC::kParts;
    constexpr int kRows = NG * CS * kParts * 512;
    extern __shared__ char smem[];
    // the cotangents of the state, of u before the system is solved, of r and of out (scaled), of out as it is; the helpers' sums, in floats
    T *sS = reinterpret_cast<T *>(smem), *sU = sS + NG * KS * kParts * 512, *sR = sU + kRows, *sO = sR + kRows, *sD = sO + kRows;
    float *sWritten = reinterpret_cast<float *>(sD + NG * CS * 512), *sState = sWritten + NG * CT * 256;
    W w;
    if (w.place(a)) return;
    const int lane = w.lane;
    auto four = [&](float *p, int i) -> f32x4 & { return *reinterpret_cast<f32x4 *>(p + i * 256 + lane * 4); };
    if (w.helper) {
        if (w.live == 0) return;
        const float *kept = a.kept + w.pair * (delta_states_floats(a.n, a.chunks) + delta_written_floats(a.n, a.chunks, C));
        T *dstates = static_cast<T *>(a.dstates) + w.pair * a.chunks * delta_state_floats(a.n);
        const typename W::Rows douts = w.value_rows(a.dout);
        D8 QT[PER][CS], P[CS][kParts];
        typename W::Cols O[NG / NC][4];
        f32x4 start, S[NG][2], written[NG], state[NG][PER];
        const bool features = w.w < KS && 32 * w.w + 8 * w.c < w.DK;     // of a state: the eight 32w + 8c ..
        auto load_kept = [&](int n) {
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    S[g][t] = *reinterpret_cast<const f32x4 *>(kept + (features && w.mine(g) ? w.state_place(n, g, 2 * w.w + t) : 0));
        };
        auto put_out = [&](int next) {           // the cotangents of out of one chunk as operands; `next`: what is loaded then
            if (w.tokens())
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
            w.load_values(douts, next, O);
            start = w.gate(a, next, 0);
        };
        auto sums = [&](int next) {
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                written[g] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int p = 0; p < PER; ++p) state[g][p] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
            if (w.tokens())
#pragma unroll
                for (int ks = 0; ks < CS; ++ks)
                    if (w.template step<true>(ks))
#pragma unroll
                        for (int g = 0; g < NG; ++g) {
                            D8 o[1];
                            W::template get<CS, 1>(sD, g, ks, lane, o);
                            written[g] = mma_whole(P[ks], o[0], written[g]);
                        }
            w.template load_steps<true>(a.to.scores, a, next, P);
#pragma unroll
            for (int ks = 0; ks < CS; ++ks)
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    D8 o[kParts];
                    W::template get<CS, kParts>(sO, g, ks, lane, o);
#pragma unroll
                    for (int i = kParts - 1; i >= 0; --i)
#pragma unroll
                        for (int p = 0; p < PER; ++p) state[g][p] = mma_d(QT[p][ks], o[i], state[g][p]);
                }
            w.load_features(a.to.queries, a, next, QT);
        };
        auto hand_written = [&] {
            if (w.tokens())
#pragma unroll
                for (int g = 0; g < NG; ++g) four(sWritten, g * CT + w.w) = written[g];
        };
        const int n0 = w.live - 1;
        load_kept(n0 + 1);
        w.load_values(douts, n0, O);
        start = w.gate(a, n0, 0);
        w.template load_steps<true>(a.to.scores, a, n0, P);
        w.load_features(a.to.queries, a, n0, QT);
        put_out(max(n0 - 1, 0));
        lds_barrier();                           // the operands of the first chunk's sums
        sums(max(n0 - 1, 0));
        hand_written();
        for (int n = n0; n >= 0; --n) {
            const int next = max(n - 2, 0);
            lds_barrier();                       // dS, and what the helpers add to du
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int p = 0; p < PER; ++p) four(sState, g * TILES + w.w * PER + p) = state[g][p];
            put_out(next);
            // the cotangent of the state behind the chunk, for the gradients; its product with that state
            float *dots = a.dots + (((int64_t)w.pair * a.chunks + n) * (w.DV >> 4) + (w.col0 >> 4)) * 4 + w.w;
#pragma unroll
            for (int g = 0; g < NG; g += NC) {
                float dot = 0.f;
#pragma unroll
                for (int q = g; q < g + NC; ++q)
                    if (features && w.mine(q)) {
                        D8 parts[kParts];
                        W::template get<KS, kParts>(sS, q, w.w, lane, parts);
                        float d[8], x[8];
                        unpack8(parts[kParts - 1], d);
#pragma unroll
                        for (int i = kParts - 2; i >= 0; --i) {
                            unpack8(parts[i], x);
#pragma unroll
                            for (int e = 0; e < 8; ++e) d[e] += x[e];
                        }
#pragma unroll
                        for (int e = 0; e < 8; ++e) dot += d[e] * S[q][e >> 2][e & 3];
                        st8(dstates + w.cotangent_place(n, q, w.w), parts[0]);
                    }
                dot = sum_over_c(sum_over_r(dot));
                if (lane == 0)
                    for (int q = 0; q < NC; ++q)
                        if (w.col0 + 16 * (g + q) < w.DV) dots[4 * (g + q)] = q ? 0.f : dot;
            }
            load_kept(n);
            lds_barrier();                       // du
            sums(next);
            lds_barrier();                       // dr
            hand_written();
        }
        return;
    }
    f32x4 S[NG][PER];
    w.load_state(a.hidden, a.hidden_dtype, S);
    if (w.live > 0) {
        float *dus = a.du + w.pair * delta_written_floats(a.n, a.chunks, C);
        D8 K[KS], KT[PER][CS], Z[CS][kParts];
        const int n0 = w.live - 1;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) K[ks] = w.load_row(a.to.key_rows, a, n0, ks);
        f32x4 end = w.gate(a, n0, 1);
        w.template load_steps<true>(a.to.inverse, a, n0, Z);
        f32x4 start = w.gate(a, n0, 0), beta = w.gate(a, n0, 2);
        w.load_features(a.to.keys, a, n0, KT);
        float whole = w.gate_whole(a, n0);
        w.template put_state<kParts>(sS, S);
        lds_barrier();                           // (the helpers')
        for (int n = n0; n >= 0; --n) {
            const int next = max(n - 1, 0);
            f32x4 du[NG];
            lds_barrier();                       // dS, and what the helpers add to du
            w.template keys_times_state<kParts>(a, next, sS, K, du);
            if (w.tokens())
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const f32x4 scores = four(sWritten, g * CT + w.w);
#pragma unroll
                    for (int e = 0; e < 4; ++e) du[g][e] = end[e] * du[g][e] + scores[e];
                    W::template put<CS, kParts>(sU, g, w.w, lane, du[g]);
                }
            end = w.gate(a, next, 1);
            lds_barrier();                       // du
            w.template solve<true>(a, next, sU, Z, du);
            if (w.tokens())
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    f32x4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = -start[e] * (beta[e] * du[g][e]);
                    W::template put<CS, kParts>(sR, g, w.w, lane, v);
                    if (w.mine(g)) *reinterpret_cast<f32x4 *>(dus + w.written(n, g)) = du[g];
                }
            start = w.gate(a, next, 0);
            beta = w.gate(a, next, 2);
            lds_barrier();                       // dr
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int p = 0; p < PER; ++p) {
                    const f32x4 out = four(sState, g * TILES + w.w * PER + p);
#pragma unroll
                    for (int e = 0; e < 4; ++e) S[g][p][e] = S[g][p][e] * whole + out[e];
                }
            w.add_keys(a, next, sR, KT, S);
            whole = w.gate_whole(a, next);
            w.template put_state<kParts>(sS, S);
        }
    }
    w.store_state(a.hidden_out, a.hidden_dtype, S);
}

// bytes of shared memory
template <typename T, int DKP, int NG, bool BACK> constexpr size_t walk_lds()
{
    typedef Walk<T, DKP, NG> W;
    typedef DeltaChunk<T> DC;
    return BACK ? sizeof(T) * 512 * NG * (W::KS * DC::kParts + W::CS * (3 * DC::kParts + 1)) + sizeof(float) * 256 * NG * (W::CT + W::TILES)
                : sizeof(T) * 512 * NG * (W::KS * DC::kFew + W::CS * (2 * DC::kParts + DC::kFew));
}
template <typename T, int DKP, int NG, bool BACK> int launch_walk(hipStream_t stream, const DeltaArgs &a)
{
    // the columns of a pair start next to each other on one die (workgroups are dealt to the eight in turn) and share what they read in its cache
    const unsigned grid = (unsigned)((a.pairs + 7) / 8 * 8 * ((a.n.DV + 16 * NG - 1) / (16 * NG)));
    constexpr size_t lds = walk_lds<T, DKP, NG, BACK>();
    static_assert(lds <= 160 * 1024, "");
    static LdsGrant grants[2];
    auto launch = [&](LdsGrant &grant, auto *kernel) {
        if (int e = allow_lds(grant, reinterpret_cast<const void *>(kernel), lds)) return e;
        kernel<<<grid, 512, lds, stream>>>(a);
        return launch_status();
    };
    if constexpr (BACK) return launch(grants[0], delta_walk_back_kernel<T, DKP, NG>);
    else return a.kept ? launch(grants[0], delta_walk_kernel<T, DKP, NG, true>) : launch(grants[1], delta_walk_kernel<T, DKP, NG, false>);
}
// Value columns of a workgroup: 64 share the operands' way from memory, 16 make four times the workgroups.
template <typename T, int DKP, bool BACK> int choose_walk(hipStream_t stream, const DeltaArgs &a)
{
    const int64_t groups = a.pairs * ((a.n.DV + 15) / 16);
    if constexpr (walk_lds<T, DKP, 4, BACK>() <= 160 * 1024)
        if (a.n.DV > 32 && groups >= 8 * kComputeUnits) return launch_walk<T, DKP, 4, BACK>(stream, a);
    if (a.n.DV > 16 && groups >= 4 * kComputeUnits) return launch_walk<T, DKP, 2, BACK>(stream, a);
    return launch_walk<T, DKP, 1, BACK>(stream, a);
}
template <typename T, bool BACK> int dispatch_walk(hipStream_t stream, const DeltaArgs &a)
{
    return a.n.DK <= 64 ? choose_walk<T, 64, BACK>(stream, a) : choose_walk<T, 128, BACK>(stream, a);
}

}  // namespace

int delta_walk(void *stream, const DeltaArgs &a, gla_dtype dtype, bool backward)
{
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == GLA_BF16) return backward ? dispatch_walk<__bf16, true>(s, a) : dispatch_walk<__bf16, false>(s, a);
    return backward ? dispatch_walk<float, true>(s, a) : dispatch_walk<float, false>(s, a);
}

}  // namespace gla
