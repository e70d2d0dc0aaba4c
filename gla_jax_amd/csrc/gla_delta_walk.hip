// The gated delta rule: the walks over the chunks, forward with the state and backward with its cotangent.
#include "gla_delta.hpp"

namespace gla {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr unsigned kNowhere = 0x7fffff00u;       // a place behind any chunk's rows
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
    int order, segment, first, end;                      // the segment's chunks: first .. end - 1
    bool basis;                                          // the columns are not the state's, but a basis of it
    unsigned pair;
    int64_t b, h, hk;
    bool helper;
    // an array's rows: its first one, and a lane's place in a chunk's
    struct Rows {
        const T *p;
        int st;
        unsigned at[4];
    };
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t chunk_rows(const Rows &x, int n, int width) const      // (at most 2^30 bytes)
    {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(x.p + (int64_t)n * C * x.st), 0, ((min(C, len - n * C) - 1) * x.st + width) * (int)sizeof(T),
                                                 0x00027000);
    }
    // true: there is nothing to do
    template <bool SUMMARY, bool BACK> __device__ __forceinline__ bool place(const DeltaArgs &a)
    {
        w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        helper = w >= kWaves;
        w &= kWaves - 1;
        lane = threadIdx.x & 63;
        r = lane & 15;
        c = lane >> 4;
        DK = (int)a.n.DK;
        DV = (int)a.n.DV;
        const unsigned of_values = ((unsigned)DV + 16 * NG - 1) / (16 * NG), groups = of_values + (SUMMARY ? ((unsigned)DK + 16 * NG - 1) / (16 * NG) : 0);
        const unsigned turn = blockIdx.x / 8, units = (a.segments - (SUMMARY ? 1 : 0)) * groups, group = turn % units % groups;
        pair = turn / units * 8 + blockIdx.x % 8;
        order = turn % units / groups;
        segment = BACK ? a.segments - 1 - order : order;
        basis = group >= of_values;
        col0 = (int)(basis ? group - of_values : group) * 16 * NG;
        if (SUMMARY && basis && order == 0) return true;         // (the first one's start is known)
        if (pair >= (unsigned)a.pairs) return true;
        const unsigned H = (unsigned)a.n.H;
        b = pair / H;
        h = pair % H;
        hk = pair % H / (H / (unsigned)a.n.HK);
        T_ = (int)a.n.T;
        if (a.by_length) {
            // The b-th longest sequence instead (of equal ones the first): where workgroups wait for compute units, the long ones do not come last.
            // (16 prompts of 0 to 1337 tokens, 16 heads: 150 -> 139 us.)
            const int B = (int)a.n.B, mine = lane < B ? min(max(a.lengths[lane], 0), T_) : -1;
            int longer = 0;
            for (int i = 0; i < B; ++i) {
                const int other = __builtin_amdgcn_readlane(mine, i);
                longer += other > mine || (other == mine && i < lane);
            }
            b = __builtin_ctzll(__ballot(lane < B && longer == (int)b));
            len = __builtin_amdgcn_readlane(mine, (int)b);
            pair = (unsigned)b * H + (unsigned)h;
        } else {
            len = a.lengths ? min(max(a.lengths[b], 0), T_) : T_;
        }
        live = (len + C - 1) / C;
        first = min(segment * a.segment_chunks, live);
        end = segment + 1 < a.segments ? min(first + a.segment_chunks, live) : live;
        return false;
    }
    __device__ __forceinline__ bool tokens() const { return CT == kWaves || w < CT; }
    __device__ __forceinline__ int column(int g) const { return col0 + (NC == 2 ? 32 * (g >> 1) + 2 * r + (g & 1) : r); }
    __device__ __forceinline__ bool mine(int g) const { return column(g) < (basis ? DK : DV); }
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
    // The state that a segment starts from: zero or a basis for its summary, else what the segments before it leave.
    template <bool SUMMARY> __device__ __forceinline__ void start_state(const DeltaArgs &a, f32x4 (&S)[NG][PER]) const
    {
        if (order == 0 && !basis) return load_state(a.hidden, a.hidden_dtype, S);
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int p = 0; p < PER; ++p) {
                const bool is = mine(g) && feature(p) < DK;
                if constexpr (SUMMARY)
#pragma unroll
                    for (int e = 0; e < 4; ++e) S[g][p][e] = basis && feature(p) + e == column(g) ? 1.f : 0.f;
                else {
                    const float *from = a.starts + ((int64_t)pair * (a.segments - 1) + order - 1) * DV * DK;
                    const f32x4 x = *reinterpret_cast<const f32x4 *>(from + (is ? column(g) * DK + feature(p) : 0));
                    S[g][p] = is ? x : f32x4{0.f, 0.f, 0.f, 0.f};
                }
            }
    }
    template <bool SUMMARY> __device__ __forceinline__ void end_state(const DeltaArgs &a, const f32x4 (&S)[NG][PER]) const
    {
        if constexpr (SUMMARY) {
            float *to = a.summary + (((int64_t)pair * (a.segments - 1) + order) * (DV + DK) + (basis ? DV : 0)) * DK;
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int p = 0; p < PER; ++p)
                    if (mine(g) && feature(p) < DK) *reinterpret_cast<f32x4 *>(to + column(g) * DK + feature(p)) = S[g][p];
        } else if (order == a.segments - 1) {
            store_state(a.hidden_out, a.hidden_dtype, S);
        }
    }
    // a prepared array's chunk
    template <int SIZE> __device__ __forceinline__ const T *of_pair(const void *from, const DeltaArgs &a, int n) const
    {
        return static_cast<const T *>(from) + ((int64_t)pair * a.chunks + n) * SIZE;
    }
    __device__ __forceinline__ D8 load_operand(const T *p) const { return ld8(at_bytes(p, lane * 8 * (unsigned)sizeof(T))); }
    // the wave's tokens of keys or queries on their way from memory to a tile in LDS: 1 KB of neighbouring pieces a load
    static constexpr int kPieces = DKP * (int)sizeof(T) / 16, kPer = 16 / (int)sizeof(T), kAtOnce = 64 / kPieces, kLoads = 16 / kAtOnce;
    typedef u32x4 Stage[kLoads];
    __device__ __forceinline__ Rows key_rows(const DecayRows &x) const
    {
        Rows y{static_cast<const T *>(x.p) + b * x.sb + hk * x.sh, (int)x.st, {}};
        const int col = lane % kPieces * kPer;
        y.at[0] = col < DK ? (unsigned)((16 * min(w, CT - 1) + lane / kPieces) * y.st + col) * (unsigned)sizeof(T) : kNowhere;
        return y;
    }
    __device__ __forceinline__ void load_stage(const Rows &x, int n, Stage &to) const
    {
        const auto rows = chunk_rows(x, n, DK);
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
            to[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rows, x.at[0] + (unsigned)(i * kAtOnce * x.st) * (unsigned)sizeof(T), 0, 0));
    }
    __device__ __forceinline__ void put_stage(T *tile, const Stage &from) const
    {
        if (tokens())
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int col = lane % kPieces * kPer, at = LdsTile<T, DKP>::piece(16 * w + lane / kPieces + i * kAtOnce, col & ~7) + (col & 7);
                *reinterpret_cast<u32x4 *>(tile + at) = from[i];
            }
    }
    // the wave's tokens, features as the contracted index in their order
    __device__ __forceinline__ void get_rows(const T *tile, D8 (&to)[KS]) const
    {
        if (tokens())
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) to[ks] = LdsTile<T, DKP>().rows(tile, w, ks);
    }
    // the wave's features, tokens as the contracted index
    __device__ __forceinline__ void get_features(const T *tile, D8 (&to)[PER][CS]) const
    {
#pragma unroll
        for (int t = 0; t < PER; ++t)
#pragma unroll
            for (int ks = 0; ks < CS; ++ks) to[t][ks] = feature_columns<DKP>(tile, ks, w * PER + t);
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
        const auto rows = chunk_rows(x, n, DV);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int g = 0; g < NG; g += NC) to[g / NC][e] = load_columns<Cols>(rows, x.at[e] + 16 * g * (unsigned)sizeof(T));
    }
    static __device__ __forceinline__ float value(const Cols (&v)[NG / NC][4], int g, int e) { return column_of<T, NC>(v[g / NC][e], g % NC); }
    // A chunk's gates: e^{L_i} (0), e^{L_C - L_i} (1), b_i (2), and e^{L_C}.  Each helper brings a kind.
    __device__ __forceinline__ float load_gate(const DeltaArgs &a, int n) const
    {
        return *at_bytes(a.to.gates + ((int64_t)pair * a.chunks + n) * DC::kGates + w * C, 4u * (lane & (C - 1)));
    }
    __device__ __forceinline__ f32x4 load_start(const DeltaArgs &a, int n) const
    {
        return *reinterpret_cast<const f32x4 *>(at_bytes(a.to.gates + ((int64_t)pair * a.chunks + n) * DC::kGates + 16 * min(w, CT - 1), 16u * c));
    }
    __device__ __forceinline__ void put_gate(float *gates, float x) const
    {
        if (lane < C) gates[w * C + lane] = x;
    }
    __device__ __forceinline__ f32x4 gate(const float *gates, int kind) const
    {
        return *reinterpret_cast<const f32x4 *>(gates + kind * C + 16 * min(w, CT - 1) + 4 * c);
    }
    // What brings chunks into the die's cache before the loads above ask for them.  A compute unit has only so many requests on their way to
    // memory, and a chunk takes 80 KB.  The workgroups of a pair's columns want the same, so each helper touches a part, one value of each 128
    // bytes: keys, queries, inverse, scores (in this order, 64 lines a wave, as far as there are waves), and of its own columns the values.
    // (Training step of B4 T4096 H6 D128 on data that no cache holds: walks 142 and 153 us without, 129 and 148 with, while cotangents of states were left
    // in one part; on data in the last-level cache no difference, nor with 32 columns from the other half of the states' lines: 291 us back for B8 T2048 H16.
    // At 64 features, with half as much to bring, 59 us without and 62 with, and summaries 283 and 296: those do without.)
    static constexpr int kAhead = 6;
    struct Ahead {
        const char *p;
        int64_t step;                            // bytes from chunk to chunk
        int st, size;                            // of rows: their distance; or the bytes of a chunk
        unsigned at;
    };
    template <int SCORE_PARTS> __device__ __forceinline__ Ahead ahead(const DeltaArgs &a, const Rows &keys, const Rows &queries) const
    {
        constexpr int e = (int)sizeof(T), kLines = DKP * e / 128, kOfRows = C * kLines / 64, kInverse = DC::kSteps * DC::kParts * 512 * e,
                      kScores = DC::kSteps * SCORE_PARTS * 512 * e, kOfInverse = (kInverse + 8191) / 8192, kOfScores = (kScores + 8191) / 8192;
        int job = col0 / (16 * NG) * kWaves + w;
        if (job < 2 * kOfRows) {
            const Rows &x = job < kOfRows ? keys : queries;
            const int line = lane % kLines * 128;
            return {reinterpret_cast<const char *>(x.p), (int64_t)C * x.st * e, x.st, 0,
                    line < DK * e ? (unsigned)((job % kOfRows * (64 / kLines) + lane / kLines) * x.st * e + line) : kNowhere};
        }
        job -= 2 * kOfRows;
        const bool inverse = job < kOfInverse;
        const int size = inverse ? kInverse : kScores;
        if (!inverse) job -= kOfInverse;
        return {static_cast<const char *>(inverse ? a.to.inverse : a.to.scores) + (int64_t)pair * a.chunks * size, size, 0, size,
                inverse || job < kOfScores ? 8192u * job + 128u * lane : kNowhere};
    }
    __device__ __forceinline__ uint32_t touch(const Ahead &x, int n) const
    {
        const int size = x.size ? x.size : ((min(C, len - n * C) - 1) * x.st + DK) * (int)sizeof(T);
        const auto chunk = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(x.p + n * x.step), 0, size, 0x00027000);
        return __builtin_amdgcn_raw_buffer_load_b32(chunk, x.at, 0, 0);
    }
    __device__ __forceinline__ uint32_t touch_values(const Rows &x, int n) const
    {
        return __builtin_amdgcn_raw_buffer_load_b32(chunk_rows(x, n, DV), lane < 16 ? (unsigned)((16 * min(w, CT - 1) + r) * x.st + col0) * (unsigned)sizeof(T) : kNowhere,
                                                    0, 0);
    }
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
    // cotangents of states: the eight features 8c .. of tiles 2 ks and 2 ks + 1, a column, the first part
    __device__ __forceinline__ int64_t cotangent_place(int n, int g, int ks) const
    {
        return (((int64_t)n * (DV >> 4) + (column(g) >> 4)) * (delta_state_tiles(DK) / 2) + ks) * (DC::kFew * 512) + (c * 16 + (column(g) & 15)) * 8;
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
    // K S: the small parts' sum apart, so that products need not wait for each other
    template <int N> __device__ __forceinline__ void keys_times_state(const T *state, const D8 (&K)[KS], f32x4 (&x)[NG]) const
    {
        if (!tokens()) return;
        f32x4 low[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) x[g] = low[g] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
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
        if constexpr (N > 1)
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[g][e] += low[g][e];
    }
    template <bool UPPER> __device__ __forceinline__ void solve(const T *rows, const D8 (&Z)[CS][DC::kParts], f32x4 (&x)[NG]) const
    {
        constexpr int N = DC::kParts;
        if (!tokens()) return;
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
    __device__ __forceinline__ void add_keys(const T *written, const D8 (&KT)[PER][CS], f32x4 (&S)[NG][PER]) const
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
    }
};
// step(n, x, y) for n = 0 .. live - 1, x and y taking turns.  The compiler's waits for a load count the loads behind it, the fewest on any way
// there: so what was requested before the loop has to be there first, and the loop has no way out in its middle.
template <typename Set, typename F> __device__ __forceinline__ void in_turns(int live, Set &x, Set &y, F step)
{
    wait_for_memory();
    int n = 0;
    for (; n + 1 < live; n += 2) {
        step(n, x, y);
        step(n + 1, y, x);
    }
    if (n < live) step(n, x, y);
}
template <typename T, int DKP> constexpr int kTile = DeltaChunk<T>::C * LdsTile<T, DKP>::kRow;

// Forward.  Three times a chunk the waves wait for each other: for the state's operands, r and u.
template <typename T, int DKP, int NG, bool KEEP, bool SUMMARY> __global__ __launch_bounds__(512) void delta_walk_kernel(const DeltaArgs a)
{
    typedef Walk<T, DKP, NG> W;
    typedef typename W::DC DC;
    typedef typename W::D8 D8;
    constexpr int C = W::C, CT = W::CT, CS = W::CS, KS = W::KS, PER = W::PER, NC = W::NC, kParts = DC::kParts, kFew = DC::kFew;
    constexpr bool kTouch = DKP > 64 && !SUMMARY;
    extern __shared__ char smem[];
    // keys of two chunks and queries of one; the state, r, u (for the state, scaled) and u (for out); values, and gates of two chunks
    T *sK[2] = {reinterpret_cast<T *>(smem), reinterpret_cast<T *>(smem) + kTile<T, DKP>}, *sQ = sK[1] + kTile<T, DKP>, *sS = sQ + kTile<T, DKP>,
      *sR = sS + NG * KS * kParts * 512, *sU = sR + NG * CS * kParts * 512, *sO = sU + NG * CS * kParts * 512;
    float *sV = reinterpret_cast<float *>(sO + NG * CS * kFew * 512), *sG[2] = {sV + NG * CT * 256, sV + NG * CT * 256 + DC::kGates};
    W w;
    if (w.template place<SUMMARY, false>(a)) return;
    const int lane = w.lane, count = w.end - w.first, last = w.end - 1;
    auto four = [&](float *p, int i) -> f32x4 & { return *reinterpret_cast<f32x4 *>(p + i * 256 + lane * 4); };
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
        struct Set {
            typename W::Stage key, query;
            typename W::Cols V[NG / NC][4];
            float gate;
            D8 P[CS][kFew];
            uint32_t touched[2];
        } x, y;
        const typename W::Rows keys = w.key_rows(a.keys), queries = w.key_rows(a.queries), values = w.value_rows(a.values);
        D8 Q[KS];
        auto load_rows = [&](int step, Set &to) {
            const int n = min(w.first + step, last);
            w.load_stage(keys, n, to.key);
            if constexpr (!SUMMARY) w.load_stage(queries, n, to.query);
            w.load_values(values, n, to.V);
            to.gate = w.load_gate(a, n);
        };
        auto load_scores = [&](int step, Set &to) {
            if constexpr (!SUMMARY) w.template load_steps<false>(a.to.scores, a, min(w.first + step, last), to.P);
        };
        const typename W::Ahead ahead = w.template ahead<kFew>(a, keys, queries);
        auto touch = [&](int step, Set &to) {
            if constexpr (!kTouch) return;
            const int n = min(w.first + step, last);
            to.touched[0] = w.touch(ahead, n);
            to.touched[1] = w.touch_values(values, n);
        };
        auto put_rows = [&](int step, const Set &from) {
            w.put_stage(sK[step & 1], from.key);
            if constexpr (!SUMMARY) w.put_stage(sQ, from.query);
            if (w.tokens())
#pragma unroll
                for (int g = 0; g < NG; ++g)
                    four(sV, g * CT + w.w) = SUMMARY && w.basis ? f32x4{0.f, 0.f, 0.f, 0.f}
                                                                : f32x4{W::value(from.V, g, 0), W::value(from.V, g, 1), W::value(from.V, g, 2), W::value(from.V, g, 3)};
            w.put_gate(sG[step & 1], from.gate);
            if constexpr (!SUMMARY) w.get_rows(sQ, Q);       // (the wave's own)
        };
        if (count > 0) {
            load_rows(0, x);
            load_scores(0, x);
            load_rows(1, y);
            load_scores(1, y);
            put_rows(0, x);
            load_rows(2, x);
            touch(W::kAhead - 2, x);
            touch(W::kAhead - 1, y);
            lds_barrier();                       // the first rows
        }
        in_turns(count, x, y, [&](int step, Set &mine, Set &next) {
            f32x4 o[NG];
            lds_barrier();                       // the state's operands are there
#pragma unroll
            for (int g = 0; g < NG; ++g) o[g] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (!SUMMARY && w.tokens())
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        D8 s[kFew];
                        W::template get<KS, kParts>(sS, g, ks, lane, s);
                        o[g] = mma_whole(s, Q[ks], o[g]);
                    }
            lds_barrier();                       // r
            put_rows(step + 1, next);
            load_rows(step + 3, next);
            lds_barrier();                       // u
            if (!SUMMARY && w.tokens()) {
                const float start = sG[step & 1][16 * w.w + w.r];
#pragma unroll
                for (int g = 0; g < NG; ++g)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[g][e] *= start;
#pragma unroll
                for (int ks = 0; ks < CS; ++ks)
                    if (w.template step<false>(ks))
#pragma unroll
                        for (int g = 0; g < NG; ++g) {
                            D8 u[kFew];
                            W::template get<CS, kFew>(sO, g, ks, lane, u);
                            o[g] = mma_parts(u, mine.P[ks], o[g]);
                        }
                const int from = (w.first + step) * C;
                const bool is = from + 16 * w.w + w.r < w.len;
                store(from, [&](int g, int e) { return is ? o[g][e] : 0.f; });
            }
            load_scores(step + 2, mine);
            if constexpr (kTouch) asm volatile("" ::"v"(mine.touched[0]), "v"(mine.touched[1]));       // (asked for two chunks ago)
            touch(step + W::kAhead, mine);
        });
        // rows past the end of a shorter sequence
        if (!SUMMARY && w.segment == a.segments - 1)
            for (int from = w.live * C; from < w.T_; from += 16 * W::kWaves) store(from, [](int, int) { return 0.f; });
        return;
    }
    f32x4 S[NG][PER];
    w.template start_state<SUMMARY>(a, S);
    float *kept = KEEP ? a.kept + w.pair * (delta_states_floats(a.n, a.chunks) + delta_written_floats(a.n, a.chunks, C)) : nullptr;
    float *xs = KEEP ? kept + delta_states_floats(a.n, a.chunks) : nullptr;
    auto keep = [&](int n) {
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int p = 0; p < PER; ++p)
                if (w.mine(g) && w.feature(p) < w.DK) *reinterpret_cast<f32x4 *>(kept + w.state_place(n, g, w.w * PER + p)) = S[g][p];
    };
    struct Set {
        D8 Z[CS][kParts];
    } x, y;
    auto load = [&](int step, Set &to) { w.template load_steps<false>(a.to.inverse, a, min(w.first + step, last), to.Z); };
    D8 K[KS], KT[PER][CS];
    if (count > 0) {
        load(0, x);
        load(1, y);
        w.template put_state<kParts>(sS, S);
        lds_barrier();                           // the first rows
        w.get_rows(sK[0], K);
    }
    in_turns(count, x, y, [&](int step, Set &mine, Set &) {
        const int n = w.first + step;
        const float *gates = sG[step & 1];
        if constexpr (KEEP) keep(n);
        f32x4 v[NG];
        lds_barrier();                           // the state's operands are there
        w.template keys_times_state<kParts>(sS, K, v);
        if (w.tokens()) {
            const f32x4 start = w.gate(gates, 0);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const f32x4 value = four(sV, g * CT + w.w);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[g][e] = value[e] - start[e] * v[g][e];
                W::template put<CS, kParts>(sR, g, w.w, lane, v[g]);
            }
        }
        lds_barrier();                           // r
        w.template solve<false>(sR, mine.Z, v);
        if (w.tokens()) {
            const f32x4 end = w.gate(gates, 1), beta = w.gate(gates, 2);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                f32x4 u, weighted;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    u[e] = beta[e] * v[g][e];
                    weighted[e] = end[e] * u[e];
                }
                W::template put<CS, kParts>(sU, g, w.w, lane, weighted);
                if constexpr (!SUMMARY) W::template put<CS, kFew>(sO, g, w.w, lane, u);
                if constexpr (KEEP)
                    if (w.mine(g)) *reinterpret_cast<f32x4 *>(xs + w.written(n, g)) = v[g];
            }
        }
        w.get_features(sK[step & 1], KT);
        const float whole = gates[3 * C];
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int p = 0; p < PER; ++p)
#pragma unroll
                for (int e = 0; e < 4; ++e) S[g][p][e] *= whole;
        load(step + 2, mine);
        lds_barrier();                           // u
        w.add_keys(sU, KT, S);                   // the state behind the chunk
        w.get_rows(sK[(step + 1) & 1], K);
        w.template put_state<kParts>(sS, S);
    });
    if constexpr (KEEP)
        if (w.end == w.live && (count > 0 || w.segment == 0)) keep(w.live);
    w.template end_state<SUMMARY>(a, S);
}

// Backward, from the last chunk to the first.  With dS the cotangent of the state behind a chunk and du that of u from what reads u,
//       du_j = sum_{i>=j} P_ij do_i + e^{L_C - L_j} dS^T k_j,   du <- (1 + b M)^{-T} du,   dv = dr = b du,
//       dS  <- e^{L_C} dS + sum_i e^{L_i} (q_i do_i^T - k_i dv_i^T).
// The helpers make the first sum and sum_i e^{L_i} q_i do_i^T, a chunk ahead.
template <typename T, int DKP, int NG, bool SUMMARY> __global__ __launch_bounds__(512) void delta_walk_back_kernel(const DeltaArgs a)
{
    typedef Walk<T, DKP, NG> W;
    typedef typename W::DC DC;
    typedef typename W::D8 D8;
    constexpr int C = W::C, CT = W::CT, CS = W::CS, KS = W::KS, PER = W::PER, TILES = W::TILES, NC = W::NC, kParts = DC::kParts;
    constexpr int kRows = NG * CS * kParts * 512;
    constexpr bool kTouch = DKP > 64 && !SUMMARY;
    extern __shared__ char smem[];
    // keys of two chunks and queries of one; the cotangents of the state, of u before the system is solved, of r and of out (scaled), of out as
    // it is; the helpers' sums, in floats; gates of two chunks
    T *sK[2] = {reinterpret_cast<T *>(smem), reinterpret_cast<T *>(smem) + kTile<T, DKP>}, *sQ = sK[1] + kTile<T, DKP>, *sS = sQ + kTile<T, DKP>,
      *sU = sS + NG * KS * kParts * 512, *sR = sU + kRows, *sO = sR + kRows, *sD = sO + kRows;
    float *sWritten = reinterpret_cast<float *>(sD + NG * CS * 512), *sState = sWritten + NG * CT * 256;
    float *sG[2] = {sState + NG * TILES * 256, sState + NG * TILES * 256 + DC::kGates};
    W w;
    if (w.template place<SUMMARY, true>(a)) return;
    const int lane = w.lane, count = w.end - w.first;
    auto chunk_of = [&](int step) { return max(w.end - 1 - step, w.first); };
    auto four = [&](float *p, int i) -> f32x4 & { return *reinterpret_cast<f32x4 *>(p + i * 256 + lane * 4); };
    if (w.helper) {
        if (count == 0) return;
        const float *kept = a.kept + w.pair * (delta_states_floats(a.n, a.chunks) + delta_written_floats(a.n, a.chunks, C));
        T *dstates = static_cast<T *>(a.dstates) + w.pair * a.chunks * delta_state_floats(a.n) * DC::kFew;
        const typename W::Rows douts = w.value_rows(a.dout), keys = w.key_rows(a.keys), queries = w.key_rows(a.queries);
        const bool features = w.w < KS && 32 * w.w + 8 * w.c < w.DK;     // of a state: the eight 32w + 8c ..
        struct Set {
            typename W::Stage key, query;
            typename W::Cols O[NG / NC][4];
            float gate;
            f32x4 start, S[NG][2];                      // the state behind the chunk
            D8 P[CS][kParts];
            uint32_t touched[3];
        } x, y;
        const typename W::Ahead ahead = w.template ahead<kParts>(a, keys, queries);
        const int64_t state_floats = delta_state_floats(a.n);
        const unsigned touched_line = delta_touched_line(w.DK, w.col0, 16 * NG, w.w, lane);
        auto touch = [&](int step, Set &to) {
            if constexpr (!kTouch) return;
            const int n = chunk_of(step);
            to.touched[0] = w.touch(ahead, n);
            to.touched[1] = w.touch_values(douts, n);
            to.touched[2] = __builtin_amdgcn_raw_buffer_load_b32(
                __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(kept + (n + 1) * state_floats), 0, 4 * (int)state_floats, 0x00027000), touched_line, 0, 0);
        };
        auto load_rows = [&](int step, Set &to) {
            const int n = chunk_of(step);
            w.load_stage(keys, n, to.key);
            w.load_stage(queries, n, to.query);
            w.load_values(douts, n, to.O);
            to.gate = w.load_gate(a, n);
            to.start = w.load_start(a, n);
        };
        auto load_kept = [&](int step, Set &to) {
            if constexpr (SUMMARY) return;
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    to.S[g][t] = *reinterpret_cast<const f32x4 *>(kept + (features && w.mine(g) ? w.state_place(chunk_of(step) + 1, g, 2 * w.w + t) : 0));
        };
        auto load_scores = [&](int step, Set &to) { w.template load_steps<true>(a.to.scores, a, chunk_of(step), to.P); };
        auto put_rows = [&](int step, const Set &from) {
            w.put_stage(sK[step & 1], from.key);
            w.put_stage(sQ, from.query);
            w.put_gate(sG[step & 1], from.gate);
            if (w.tokens())
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    f32x4 o, scaled;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        o[e] = SUMMARY && w.basis ? 0.f : W::value(from.O, g, e);
                        scaled[e] = from.start[e] * o[e];
                    }
                    W::template put<CS, 1>(sD, g, w.w, lane, o);
                    W::template put<CS, kParts>(sO, g, w.w, lane, scaled);
                }
        };
        f32x4 written[NG], state[NG][PER];
        auto sums = [&](const Set &of) {
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
                            written[g] = mma_whole(of.P[ks], o[0], written[g]);
                        }
            D8 QT[PER][CS];
            w.get_features(sQ, QT);
            w.add_keys(sO, QT, state);
        };
        auto hand_written = [&] {
            if (w.tokens())
#pragma unroll
                for (int g = 0; g < NG; ++g) four(sWritten, g * CT + w.w) = written[g];
        };
        load_rows(0, x);
        load_scores(0, x);
        load_kept(0, x);
        load_rows(1, y);
        load_scores(1, y);
        load_kept(1, y);
        put_rows(0, x);
        load_rows(2, x);
        touch(W::kAhead - 2, x);
        touch(W::kAhead - 1, y);
        lds_barrier();                           // the first keys, and the operands of the first sums
        sums(x);
        load_scores(2, x);
        hand_written();
        in_turns(count, x, y, [&](int step, Set &mine, Set &next) {
            const int n = w.end - 1 - step;
            lds_barrier();                       // dS, and what the helpers add to du
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int p = 0; p < PER; ++p) four(sState, g * TILES + w.w * PER + p) = state[g][p];
            put_rows(step + 1, next);
            lds_barrier();                       // du
            sums(next);
            // the cotangent of the state behind the chunk, for the gradients; its product with that state
            if constexpr (!SUMMARY) {
            float *dots = a.dots + (((int64_t)w.pair * a.chunks + n) * (w.DV >> 4) + (w.col0 >> 4)) * 4 + w.w;
#pragma unroll
            for (int g = 0; g < NG; g += NC) {
                float dot = 0.f;
#pragma unroll
                for (int q = g; q < g + NC; ++q)
                    if (features && w.mine(q)) {
                        D8 parts[kParts];
                        W::template get<KS, kParts>(sS, q, w.w, lane, parts);
                        float d[8], z[8];
                        unpack8(parts[kParts - 1], d);
#pragma unroll
                        for (int i = kParts - 2; i >= 0; --i) {
                            unpack8(parts[i], z);
#pragma unroll
                            for (int e = 0; e < 8; ++e) d[e] += z[e];
                        }
#pragma unroll
                        for (int e = 0; e < 8; ++e) dot += d[e] * mine.S[q][e >> 2][e & 3];
#pragma unroll
                        for (int i = 0; i < DC::kFew; ++i) st8(dstates + w.cotangent_place(n, q, w.w) + i * 512, parts[i]);
                    }
                dot = sum_over_c(sum_over_r(dot));
                if (lane == 0)
                    for (int q = 0; q < NC; ++q)
                        if (w.col0 + 16 * (g + q) < w.DV) dots[4 * (g + q)] = q ? 0.f : dot;
            }
            }
            lds_barrier();                       // dr
            hand_written();
            load_kept(step + 2, mine);
            load_rows(step + 3, next);
            load_scores(step + 3, next);
            if constexpr (kTouch) asm volatile("" ::"v"(mine.touched[0]), "v"(mine.touched[1]), "v"(mine.touched[2]));
            touch(step + W::kAhead, mine);
        });
        return;
    }
    f32x4 S[NG][PER];
    w.template start_state<SUMMARY>(a, S);
    if (count > 0) {
        float *dus = a.du + w.pair * delta_written_floats(a.n, a.chunks, C);
        struct Set {
            D8 Z[CS][kParts];
        } x, y;
        auto load = [&](int step, Set &to) { w.template load_steps<true>(a.to.inverse, a, chunk_of(step), to.Z); };
        load(0, x);
        load(1, y);
        D8 K[KS], KT[PER][CS];
        w.template put_state<kParts>(sS, S);
        lds_barrier();                           // the first keys
        w.get_rows(sK[0], K);
        in_turns(count, x, y, [&](int step, Set &mine, Set &) {
            const int n = w.end - 1 - step;
            const float *gates = sG[step & 1];
            f32x4 du[NG];
            lds_barrier();                       // dS, and what the helpers add to du
            w.template keys_times_state<kParts>(sS, K, du);
            if (w.tokens()) {
                const f32x4 end = w.gate(gates, 1);
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const f32x4 scores = four(sWritten, g * CT + w.w);
#pragma unroll
                    for (int e = 0; e < 4; ++e) du[g][e] = end[e] * du[g][e] + scores[e];
                    W::template put<CS, kParts>(sU, g, w.w, lane, du[g]);
                }
            }
            lds_barrier();                       // du
            w.template solve<true>(sU, mine.Z, du);
            if (w.tokens()) {
                const f32x4 start = w.gate(gates, 0), beta = w.gate(gates, 2);
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    f32x4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = -start[e] * (beta[e] * du[g][e]);
                    W::template put<CS, kParts>(sR, g, w.w, lane, v);
                    if (!SUMMARY && w.mine(g)) *reinterpret_cast<f32x4 *>(dus + w.written(n, g)) = du[g];
                }
            }
            w.get_features(sK[step & 1], KT);
            const float whole = gates[3 * C];
            load(step + 2, mine);
            lds_barrier();                       // dr
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int p = 0; p < PER; ++p) {
                    const f32x4 out = four(sState, g * TILES + w.w * PER + p);
#pragma unroll
                    for (int e = 0; e < 4; ++e) S[g][p][e] = S[g][p][e] * whole + out[e];
                }
            w.add_keys(sR, KT, S);
            w.get_rows(sK[(step + 1) & 1], K);
            w.template put_state<kParts>(sS, S);
        });
    }
    w.template end_state<SUMMARY>(a, S);
}

// From the segments' summaries the states that they start from: of the first, what it leaves; of each other, with A the basis' way through it,
//       S' = A S + what it leaves of a start from zero,
// in float products, a column of 16 values a workgroup.  Wave w makes features 32w .. of S', whose tiles are the next product's operand by way of LDS.
__global__ __launch_bounds__(256) void delta_join_kernel(const DeltaArgs a)
{
    constexpr int kRow = 128 + 4;
    __shared__ float state[2][16 * kRow];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
    const int DK = (int)a.n.DK, DV = (int)a.n.DV, column = 16 * (int)blockIdx.y + r;
    const int64_t pair = blockIdx.x, size = (int64_t)(DV + DK) * DK;
    const float *summary = a.summary + pair * (a.segments - 1) * size;
    float *starts = a.starts + pair * (a.segments - 1) * DV * DK;
    f32x4 S[2];
    for (int order = 0; order + 1 < a.segments; ++order, summary += size, starts += (int64_t)DV * DK) {
        const float *before = state[order & 1];
        float *behind = state[(order + 1) & 1];
        f32x4 A[2][8];
#pragma unroll
        for (int t = 0; t < 2; ++t) {            // (places behind the last feature are the first one's again, and go nowhere)
            const int tile = 32 * w + 16 * t < DK ? 32 * w + 16 * t : 0;
            S[t] = *reinterpret_cast<const f32x4 *>(summary + (int64_t)column * DK + tile + 4 * c);
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) A[t][k][e] = order ? summary[(int64_t)(DV + (16 * k < DK ? 16 * k : 0) + 4 * c + e) * DK + tile + r] : 0.f;
        }
        if (order)
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (16 * k < DK) {
                    const f32x4 s = *reinterpret_cast<const f32x4 *>(before + r * kRow + 16 * k + 4 * c);
#pragma unroll
                    for (int t = 0; t < 2; ++t) S[t] = mma_t(A[t][k], s, S[t]);
                }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int f = 32 * w + 16 * t + 4 * c;
            if (f >= DK) continue;
            *reinterpret_cast<f32x4 *>(starts + (int64_t)column * DK + f) = S[t];
            *reinterpret_cast<f32x4 *>(behind + r * kRow + f) = S[t];
        }
        __syncthreads();
    }
}

// bytes of shared memory
template <typename T, int DKP, int NG, bool BACK> constexpr size_t walk_lds()
{
    typedef Walk<T, DKP, NG> W;
    typedef DeltaChunk<T> DC;
    constexpr size_t tiles = sizeof(T) * 3 * kTile<T, DKP>;
    return tiles + sizeof(float) * 2 * DC::kGates +
           (BACK ? sizeof(T) * 512 * NG * (W::KS * DC::kParts + W::CS * (3 * DC::kParts + 1)) + sizeof(float) * 256 * NG * (W::CT + W::TILES)
                         : sizeof(T) * 512 * NG * (W::KS * DC::kParts + W::CS * (2 * DC::kParts + DC::kFew)) + sizeof(float) * 256 * NG * W::CT);
}
template <typename T, int DKP, int NG, bool BACK> int launch_walk(hipStream_t stream, const DeltaArgs &a, bool summary)
{
    // the columns of a pair start next to each other on one die (workgroups are dealt to the eight in turn) and share what they read in its cache
    const int64_t groups = (a.n.DV + 16 * NG - 1) / (16 * NG) + (summary ? (a.n.DK + 16 * NG - 1) / (16 * NG) : 0);
    const unsigned grid = (unsigned)((a.pairs + 7) / 8 * 8 * groups * (a.segments - (summary ? 1 : 0)));
    constexpr size_t lds = walk_lds<T, DKP, NG, BACK>();
    static_assert(lds <= 160 * 1024, "");
    static LdsGrant grants[3];
    DeltaArgs of_launch = a;
    of_launch.by_length = a.lengths && a.n.B > 1 && a.n.B <= 64 && grid > kComputeUnits;
    auto launch = [&](LdsGrant &grant, auto *kernel) {
        if (int e = allow_lds(grant, reinterpret_cast<const void *>(kernel), lds)) return e;
        kernel<<<grid, 512, lds, stream>>>(of_launch);
        return launch_status();
    };
    if constexpr (BACK) {
        return summary ? launch(grants[0], delta_walk_back_kernel<T, DKP, NG, true>) : launch(grants[1], delta_walk_back_kernel<T, DKP, NG, false>);
    } else {
        if (summary) return launch(grants[0], delta_walk_kernel<T, DKP, NG, false, true>);
        return a.kept ? launch(grants[1], delta_walk_kernel<T, DKP, NG, true, false>) : launch(grants[2], delta_walk_kernel<T, DKP, NG, false, false>);
    }
}
// Value columns of a workgroup: 32 share the operands' way from memory, 16 make twice the workgroups.
template <typename T, int DKP, bool BACK> int choose_walk(hipStream_t stream, const DeltaArgs &a)
{
    const int64_t groups = a.pairs * ((a.n.DV + 15) / 16);
    if (a.segments > 1) {
        if (int e = launch_walk<T, DKP, 2, BACK>(stream, a, true)) return e;
        delta_join_kernel<<<dim3((unsigned)a.pairs, (unsigned)((a.n.DV + 15) / 16)), 256, 0, stream>>>(a);
        if (int e = launch_status()) return e;
        return launch_walk<T, DKP, 2, BACK>(stream, a, false);
    }
    if (a.n.DV > 16 && groups > kComputeUnits) return launch_walk<T, DKP, 2, BACK>(stream, a, false);
    return launch_walk<T, DKP, 1, BACK>(stream, a, false);
}
template <typename T, bool BACK> int dispatch_walk(hipStream_t stream, const DeltaArgs &a)
{
    return a.n.DK <= 64 ? choose_walk<T, 64, BACK>(stream, a) : choose_walk<T, 128, BACK>(stream, a);
}

}  // namespace

// Segments are worth their summaries (a walk for the values and one for the basis) where one walk leaves compute units idle.  The number with the
// least time by what was measured at 128 x 128 features: 1.6 us a chunk for a workgroup of 16 columns, 2.45 for one of 32, 2.1 in a summary, 1.5 a
// step of the join, and 12 for the two launches more and their beginnings.
// (B1 T32768 H8: 803 us in one piece, 8 segments 280 + 20 + 164.)  Elsewhere it takes the costs for the same, and the padded T for every length; whole calls in us as it
// chooses, and in one piece:
//       bf16: 64 x 64, T32768 H8 207, 684;  T16384 H16 187, 372;  64 x 128, T8192 H8 100, 154;  training 64 x 64, T8192 H8 250, 435;  128 x 128, B2 T8192 H8 241, 243
//       float32: 64 x 64, T8192 H8 122, 336;  training H4 313, 771;  128 x 128, T8192 H4 346, 602;  T4096 H8 181, 312
// 16 value columns stay in one piece: segments walk with 32.
int delta_segments(const DeltaArgs &a)
{
    const int64_t of_pair = (a.n.DV + 31) / 32, wide = a.pairs * of_pair, basis = a.pairs * ((a.n.DK + 31) / 32);
    auto rounds = [](int64_t groups) { return (double)((groups + kComputeUnits - 1) / kComputeUnits); };
    int best = 1;
    double least = a.pairs * ((a.n.DV + 15) / 16) <= kComputeUnits ? 1.6 * a.chunks : 2.45 * a.chunks * rounds(wide);
    for (int64_t n = 2; a.n.DV > 16 && n <= 64 && 8 * n <= a.chunks && n * wide <= kComputeUnits; ++n) {
        const double time = (a.chunks + n - 1) / n * (2.45 + 2.1 * rounds((n - 1) * (wide + basis))) + 1.5 * n + 12.0;
        if (time < least) {
            least = time;
            best = (int)n;
        }
    }
    return best;
}

int delta_walk(void *stream, const DeltaArgs &a, gla_dtype dtype, bool backward)
{
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == GLA_BF16) return backward ? dispatch_walk<__bf16, true>(s, a) : dispatch_walk<__bf16, false>(s, a);
    return backward ? dispatch_walk<float, true>(s, a) : dispatch_walk<float, false>(s, a);
}

}  // namespace gla
