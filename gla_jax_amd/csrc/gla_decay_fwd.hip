// Linear attention with one decay a head: the forward pass, and the passes that give every segment of a sequence the state
// (or the state's cotangent) that enters it.
#include "gla_decay.hpp"

namespace gla {
namespace {

struct ForwardArgs {
    DecaySizes n;
    DecayPlan plan;
    DecayRows gates, keys, values, queries;     // cotangents: `keys` are the queries, `values` the cotangents of out
    const int32_t *lengths;
    const void *hidden;                          // hidden_init; cotangents: dhidden_final
    int hidden_dtype;
    void *hidden_final, *out;
    float *kept;                                 // the state before every chunk, [B,H,chunks,DK,DV], or NULL
    float *entering, *decays;                    // see decay_entering_states
};

// The state before chunk n, which the gradients need: tiles of 16 x 16 as a wave of decay_gradient_kernel takes them, lane 16c + r key
// feature r and value features 4c .. 4c+3.  (Four bytes a lane in the order of the rows, without the exchange between lanes, took 56 us of the
// forward pass instead of 52 at B4 T4096 H6 D128, and 88 instead of 84 of the gradients.)
template <int DKP, int TILES = DKP / 16>
__device__ __forceinline__ void keep_states(const ForwardArgs &a, const f32x4 (&S)[TILES], int64_t bh, int64_t n, int column, bool mine)
{
    const int tiles = (int)a.n.DV / 16, dk = again_uniform(mine ? (int)a.n.DK : 0);
    float *to = a.kept + ((bh * a.plan.chunks + n) * (a.n.DK / 16) * tiles + column / 16) * 256;
    const unsigned lane = again(threadIdx.x) & 63, at = ((lane & 12) << 2) + ((lane >> 2) & 12) + (lane & 3);
#pragma unroll
    for (int t = 0; t < TILES; ++t)
        if (16 * t < dk) {
            float x[4] = {S[t][0], S[t][1], S[t][2], S[t][3]};
            quad_transpose(x);
            *reinterpret_cast<f32x4 *>(at_bytes(to + (size_t)(t * tiles) * 256, 4 * sizeof(float) * at)) = f32x4{x[0], x[1], x[2], x[3]};
        }
}

// One workgroup: a (batch, head) pair's segment and 16 * NW value features; wave w holds the columns 16w .. 16w+15 of the
// state, TILES accumulators of 16 key features each.  Scores are formed transposed, so that a lane holds four neighbouring
// keys of one query, and kept in `T`: their one rounding adds as much as that of out itself.  The state is an operand in `T`
// too where it meets the queries; what it accumulates comes from values scaled in 32 bits and handed over in three parts,
// since hidden_final is a 32-bit result.  Half of a chunk's cycles are the vector instructions' (a wave's 520, 16 of them conversions of S and
// 120 the split of the values); two workgroups a compute unit fill the rest.
template <typename T, int DKP, int NW>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(DKP == 256 ? 2 : DKP == 128 && NW == 4 ? 3 : 4))) void decay_pass_kernel(const ForwardArgs a)
{
    constexpr int C = DecayChunk<T>::C, NT = NW * 64, DVS = 16 * NW, TILES = DKP / 16, KS = DKP / 32, CS = C / 32, CT = C / 16;
    typedef typename FragTypes<T>::d8 D8;
    typedef LdsTile<T, DKP> TileX;
    typedef LdsTile<T, DVS> TileY;
    typedef LdsTile<T, C> TileP;
    extern __shared__ char smem[];
    T *sX = reinterpret_cast<T *>(smem), *sY = sX + C * TileX::kRow, *sQ = sY + C * TileY::kRow, *sP = sQ + C * TileX::kRow;
    ChunkGates<C> *gates = reinterpret_cast<ChunkGates<C> *>(reinterpret_cast<char *>(sP + C * TileP::kRow));

    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, r = lane & 15, c = lane >> 4;
    const unsigned H = (unsigned)a.n.H, pair = pair_of(blockIdx.x, a.n);
    const int64_t bh = pair, b = pair / H, h = pair % H, hk = pair % H / (H / (unsigned)a.n.HK);
    const int dv0 = blockIdx.y * DVS, DK = (int)a.n.DK, DV = (int)a.n.DV;
    const int T_ = (int)a.n.T, len = a.lengths ? min(max(a.lengths[b], 0), T_) : T_;
    const int seg = blockIdx.z, tail = a.plan.tail((len + C - 1) / C);
    const int first = a.plan.first(seg), last = a.plan.first(seg + 1), live = min(last, (len + C - 1) / C);
    const T *X = static_cast<const T *>(a.keys.p) + b * a.keys.sb + hk * a.keys.sh;
    const T *Y = static_cast<const T *>(a.values.p) + b * a.values.sb + h * a.values.sh + dv0;
    const T *Q = static_cast<const T *>(a.queries.p) + b * a.queries.sb + hk * a.queries.sh;
    const float *G = static_cast<const float *>(a.gates.p) + b * a.gates.sb + h * a.gates.sh;
    const bool mine = dv0 + 16 * w < DV;         // the wave's columns exist
    const TileX tx;
    const TileY ty;
    const TileP tp;

    // ---- the state that enters ----
    const unsigned hidden_at = (4 * c + (r & 3)) * DV + dv0 + 16 * w + (r & ~3);      // of tile 0, four columns a lane
    f32x4 S[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) S[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (seg == 0) {
#pragma unroll
        for (int t = 0; t < TILES; ++t)
            if (mine && 16 * t < DK) {
                float x[4];
                load_hidden<4>(a.hidden, a.hidden_dtype, bh * DK * DV + (hidden_at + 16 * t * DV), x);
                quad_transpose(x);
                S[t] = f32x4{x[0], x[1], x[2], x[3]};
            }
    } else if (seg <= tail) {
        const int64_t slab = ((bh * a.plan.segments + seg - 1) * gridDim.y + blockIdx.y) * (int64_t)(DKP * DVS);
        const f32x4 *from = reinterpret_cast<const f32x4 *>(a.entering + slab) + w * TILES * 64 + lane;
#pragma unroll
        for (int t = 0; t < TILES; ++t) S[t] = from[t * 64];
    }

    RowsInFlight<T, C, DKP, NT> x, q;
    RowsInFlight<T, C, DVS, NT> y;
    const int x_st = (int)a.keys.st, y_st = (int)a.values.st, q_st = (int)a.queries.st;
    float g = 0.f;
    auto fetch_gates = [&](int n) {              // by the wave that makes the chunk's gates
        g = w == NW - 1 && lane < C && n * C + lane < len ? G[(int64_t)(n * C + lane) * a.gates.st] : 0.f;
    };
    auto fetch = [&](int n) {                    // the rows that the pointers have come to
        const int left = len - n * C;
        const unsigned at = x.here();
        x.load(at, X, x_st, left, DK);
        y.load(at, Y, y_st, left, DV - dv0);
        q.load(at, Q, q_st, left, DK);
        X += (int64_t)C * x_st;
        Y += (int64_t)C * y_st;
        Q += (int64_t)C * q_st;
    };
    // the upper tiles that a step of 32 keys takes along with the diagonal's
    for (int i = tid; i < C * TileP::kRow; i += NT) sP[i] = (T)0.f;
    const int count = max(live - first, 0);
    int n = first;
    if (count > 0) {
        X += (int64_t)n * C * a.keys.st;
        Y += (int64_t)n * C * a.values.st;
        Q += (int64_t)n * C * a.queries.st;
        fetch_gates(n);
        fetch(n);
        if (w == NW - 1) chunk_gates<C>(gates[0], g);
        if (count > 1) fetch_gates(n + 1);
    }
    for (int i = 0; i < count; ++i, ++n) {
        const ChunkGates<C> &gate = gates[i & 1];
        lds_barrier();                            // the last chunk's tiles are read
        const unsigned at = x.here();
        x.store(at, sX, len - n * C, DK);
        y.store(at, sY, len - n * C, DV - dv0);
        q.store(at, sQ, len - n * C, DK);
        lds_barrier();
        if (i + 1 < count) fetch(n + 1);

        {
            // scores, transposed: lane (r, c) has keys 4c .. 4c+3 of tile tj for query r of tile ti
            const TileX LX = tx.here();
            const TileP LP = tp.here();
#pragma unroll 1
            for (int n16 = w; n16 < CT * (CT + 1) / 2; n16 += NW) {
                int ti, tj;
                triangle(n16, ti, tj);
                const int qi = 16 * ti + r, kj = 16 * tj + 4 * c;
                const float at = gate.sum[qi], at_rest = gate.rest[qi];
                const f32x4 to = *reinterpret_cast<const f32x4 *>(gate.sum + kj), to_rest = *reinterpret_cast<const f32x4 *>(gate.rest + kj);
                f32x4 s = tile_product<KS>(LX, sX, tj, sQ, ti);
                float p[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float weight = ChunkGates<C>::weight(at, at_rest, to[e], to_rest[e]);
                    p[e] = kj + e <= qi ? s[e] * weight : 0.f;
                }
                store_vec<T, 4>(LP.four(sP, ti, tj), p);
            }
        }
        // the next chunk's gates, by a wave that has one score tile less than the first ones
        if (w == NW - 1 && i + 1 < count) {
            chunk_gates<C>(gates[(i + 1) & 1], g);
            if (i + 2 < count) fetch_gates(n + 2);
        }

        D8 yc[CS];                                // the wave's value columns, tokens as the contracted index
#pragma unroll
        for (int ks = 0; ks < CS; ++ks) yc[ks] = ty.columns(sY, ks, w);

        typename Packed4<T>::t result[CT];
        {
            // the state's part, while the other waves finish their scores
            const TileX LX = tx.here();
            f32x4 o[CT];
#pragma unroll
            for (int ti = 0; ti < CT; ++ti) o[ti] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                float s[8];
                two_tiles(S[2 * ks], S[2 * ks + 1], s);
                const Split<T, 1> op(s);
#pragma unroll
                for (int ti = 0; ti < CT; ti += 2) {
                    const D8 x[2] = {LX.halves(sQ, ti, ks), LX.halves(sQ, ti + 1, ks)};
                    mma_left(op, x, o + ti);
                }
                __builtin_amdgcn_sched_barrier(0);     // a step's operands at a time: all of them at once do not fit the registers
            }
#pragma unroll
            for (int ti = 0; ti < CT; ++ti) {
                const float scale = gate.from_start[16 * ti + r];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[ti][e] *= scale;
            }
            lds_barrier();                        // the scores are there
#pragma unroll
            for (int ti = 0; ti < CT; ++ti) {
#pragma unroll
                for (int ks = 0; ks <= ti / 2; ++ks) o[ti] = mma_d(yc[ks], tp.halves(sP, ti, ks), o[ti]);
                result[ti] = pack_results<T>(o[ti]);
            }
        }
        if (a.kept) keep_states<DKP>(a, S, bh, n, dv0 + 16 * w, mine);
        // ---- the chunk's own contribution ----
        const TileX LX = tx.here();
        const float whole = gate.whole;
        const float *weight = gate.to_end;
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[t][e] *= whole;
#pragma unroll
        for (int ks = 0; ks < CS; ++ks) {
            float v[8], by[8];
            unpack8(yc[ks], v);
            two_tiles(*reinterpret_cast<const f32x4 *>(weight + 32 * ks + 4 * c), *reinterpret_cast<const f32x4 *>(weight + 32 * ks + 16 + 4 * c), by);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= by[e];
            const Split<T, 3> op(v);
#pragma unroll
            for (int t = 0; t < TILES; t += 2) {
                const D8 k[2] = {LX.columns(sX, ks, t), LX.columns(sX, ks, t + 1)};
                mma_right(k, op, S + t);
                if (t % 4 == 2) __builtin_amdgcn_sched_barrier(0);
            }
        }
        {
            wait_for_memory();
            T *out = static_cast<T *>(a.out) + ((b * a.n.T + n * C) * a.n.H + h) * DV + dv0 + 16 * w;
            const unsigned row = (unsigned)a.n.H * DV, at = (again(r) * row + 4 * c) * (unsigned)sizeof(T);
#pragma unroll
            for (int ti = 0; ti < CT; ++ti)
                if (mine && n * C + 16 * ti + r < T_)
                    *reinterpret_cast<typename Packed4<T>::t *>(at_bytes(out + (size_t)(16 * ti * row), at)) = result[ti];
        }
    }
    // rows past the end of a shorter sequence
    for (int m = max(live, first); m < last; ++m)
        for (int i = tid; i < C * DVS / 8; i += NT) {
            const int t = m * C + i / (DVS / 8), col = dv0 + 8 * (i % (DVS / 8));
            if (t < T_ && col < DV) st8(static_cast<T *>(a.out) + ((b * a.n.T + t) * a.n.H + h) * DV + col, D8{});
        }
    if (seg == tail) {
        const unsigned at = again(hidden_at);
#pragma unroll
        for (int t = 0; t < TILES; ++t)
            if (mine && 16 * t < DK) {
                float s[4] = {S[t][0], S[t][1], S[t][2], S[t][3]};
                quad_transpose(s);
                store_hidden<4>(a.hidden_final, a.hidden_dtype, bh * DK * DV + (at + 16 * t * DV), s);
            }
    }
}

// The forward pass for up to 128 key features: the work of decay_pass_kernel, by two kinds of waves.  The first NW carry the state, 16
// value columns each, and make out.  The others bring the chunk after the next one from memory to LDS and form the next one's scores
// meanwhile: three chunks' rows and two chunks' scores in LDS, and one barrier a chunk.  A chunk takes 6400 cycles so, where one kind of
// waves with three barriers took 9800; of the 6400 a SIMD issues vector and matrix instructions in 3800.  B1 T32768 H8 D128: 64 us for
// 268 MB, 4.2 TB/s, of the 5.2 that a copy reaches.
template <typename T, int DKP, int NW>
__global__ __launch_bounds__(NW * 128) __attribute__((amdgpu_waves_per_eu(DKP == 128 && NW == 4 ? 2 : 4))) void decay_forward_kernel(const ForwardArgs a)
{
    constexpr int C = DecayChunk<T>::C, NT = NW * 64, DVS = 16 * NW, TILES = DKP / 16, KS = DKP / 32, CS = C / 32, CT = C / 16;
    typedef typename FragTypes<T>::d8 D8;
    typedef LdsTile<T, DKP> TileX;
    typedef LdsTile<T, DVS> TileY;
    constexpr int kX = C * TileX::kRow, kY = C * TileY::kRow, kChunk = 2 * kX + kY, kScores = CT * (CT + 1) / 2 * 256;
    extern __shared__ char smem[];
    // chunk i at kChunk * (i % 3); a tile of scores as the lanes of a wave hold it, tiles in the order of `triangle`
    T *sX = reinterpret_cast<T *>(smem), *sQ = sX + kX, *sY = sQ + kX, *sP = sX + 3 * kChunk;
    ChunkGates<C> *gates = reinterpret_cast<ChunkGates<C> *>(sP + 2 * kScores);

    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, r = lane & 15, c = lane >> 4;
    const unsigned H = (unsigned)a.n.H, pair = pair_of(blockIdx.x, a.n);
    const int64_t bh = pair, b = pair / H, h = pair % H, hk = pair % H / (H / (unsigned)a.n.HK);
    const int dv0 = blockIdx.y * DVS, DK = (int)a.n.DK, DV = (int)a.n.DV;
    const int T_ = (int)a.n.T, len = a.lengths ? min(max(a.lengths[b], 0), T_) : T_;
    const int seg = blockIdx.z, tail = a.plan.tail((len + C - 1) / C);
    const int first = a.plan.first(seg), last = a.plan.first(seg + 1), live = min(last, (len + C - 1) / C);
    const int count = max(live - first, 0);
    const TileX tx;
    const TileY ty;

    if (w < NW) {
        const bool mine = dv0 + 16 * w < DV;         // the wave's columns exist
        const unsigned hidden_at = (4 * c + (r & 3)) * DV + dv0 + 16 * w + (r & ~3);      // of tile 0, four columns a lane
        f32x4 S[TILES];
#pragma unroll
        for (int t = 0; t < TILES; ++t) S[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (seg == 0) {
#pragma unroll
            for (int t = 0; t < TILES; ++t)
                if (mine && 16 * t < DK) {
                    float x[4];
                    load_hidden<4>(a.hidden, a.hidden_dtype, bh * DK * DV + (hidden_at + 16 * t * DV), x);
                    quad_transpose(x);
                    S[t] = f32x4{x[0], x[1], x[2], x[3]};
                }
        } else if (seg <= tail) {
            const int64_t slab = ((bh * a.plan.segments + seg - 1) * gridDim.y + blockIdx.y) * (int64_t)(DKP * DVS);
            const f32x4 *from = reinterpret_cast<const f32x4 *>(a.entering + slab) + w * TILES * 64 + lane;
#pragma unroll
            for (int t = 0; t < TILES; ++t) S[t] = from[t * 64];
        }
        if (count > 0) {
            lds_barrier();
            lds_barrier();                        // the first chunk's scores are there
        }
        int place = 0;                            // i % 3
        for (int i = 0; i < count; ++i, place = place == 2 ? 0 : place + 1) {
            const int n = first + i, chunk = place * kChunk;
            const ChunkGates<C> &gate = gates[place];
            D8 yc[CS];                            // the wave's value columns, tokens as the contracted index
            f32x4 o[CT];
            {
                const TileX LX = tx.here();
#pragma unroll
                for (int ti = 0; ti < CT; ++ti) o[ti] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    float s[8];
                    two_tiles(S[2 * ks], S[2 * ks + 1], s);
                    const Split<T, 1> op(s);
#pragma unroll
                    for (int ti = 0; ti < CT; ti += 2) {
                        const D8 x[2] = {LX.halves(sQ + chunk, ti, ks), LX.halves(sQ + chunk, ti + 1, ks)};
                        mma_left(op, x, o + ti);
                    }
                }
#pragma unroll
                for (int ks = 0; ks < CS; ++ks) yc[ks] = ty.columns(sY + chunk, ks, w);
#pragma unroll
                for (int ti = 0; ti < CT; ++ti) {
                    const float scale = gate.from_start[16 * ti + r];
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[ti][e] *= scale;
                }
            }
            T *out = static_cast<T *>(a.out) + ((b * a.n.T + n * C) * a.n.H + h) * DV + dv0 + 16 * w;
            const unsigned row = (unsigned)a.n.H * DV, at = (again(r) * row + 4 * c) * (unsigned)sizeof(T);
#pragma unroll
            for (int ti = 0; ti < CT; ++ti) {
#pragma unroll
                for (int ks = 0; ks <= ti / 2; ++ks) {
                    const T *p = sP + (i & 1) * kScores + (ti * (ti + 1) / 2 + 2 * ks) * 256 + 4 * lane;
                    o[ti] = mma_d(yc[ks], two_score_tiles(p, 2 * ks + 1 <= ti), o[ti]);
                }
                if (mine && n * C + 16 * ti + r < T_)
                    *reinterpret_cast<typename Packed4<T>::t *>(at_bytes(out + (size_t)(16 * ti * row), at)) = pack_results<T>(o[ti]);
            }
            if (a.kept) keep_states<DKP>(a, S, bh, n, dv0 + 16 * w, mine);
            // ---- the chunk's own contribution ----
            const TileX LX = tx.here();
            const float whole = gate.whole;
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) S[t][e] *= whole;
#pragma unroll
            for (int ks = 0; ks < CS; ++ks) {
                float v[8], by[8];
                unpack8(yc[ks], v);
                two_tiles(*reinterpret_cast<const f32x4 *>(gate.to_end + 32 * ks + 4 * c), *reinterpret_cast<const f32x4 *>(gate.to_end + 32 * ks + 16 + 4 * c), by);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] *= by[e];
                const Split<T, 3> op(v);
#pragma unroll
                for (int t = 0; t < TILES; t += 2) {
                    const D8 k[2] = {LX.columns(sX + chunk, ks, t), LX.columns(sX + chunk, ks, t + 1)};
                    mma_right(k, op, S + t);
                    if (t % 4 == 2) __builtin_amdgcn_sched_barrier(0);
                }
            }
            lds_barrier();                        // the chunk is read, the next one's scores and the rows of the one after are there
        }
        if (seg == tail) {
            const unsigned at = again(hidden_at);
#pragma unroll
            for (int t = 0; t < TILES; ++t)
                if (mine && 16 * t < DK) {
                    float s[4] = {S[t][0], S[t][1], S[t][2], S[t][3]};
                    quad_transpose(s);
                    store_hidden<4>(a.hidden_final, a.hidden_dtype, bh * DK * DV + (at + 16 * t * DV), s);
                }
        }
    } else if (count > 0) {
        const int wb = w - NW;
        const T *X = static_cast<const T *>(a.keys.p) + b * a.keys.sb + hk * a.keys.sh + (int64_t)first * C * a.keys.st;
        const T *Y = static_cast<const T *>(a.values.p) + b * a.values.sb + h * a.values.sh + dv0 + (int64_t)first * C * a.values.st;
        const T *Q = static_cast<const T *>(a.queries.p) + b * a.queries.sb + hk * a.queries.sh + (int64_t)first * C * a.queries.st;
        const float *G = static_cast<const float *>(a.gates.p) + b * a.gates.sb + h * a.gates.sh;
        RowsInFlight<T, C, DKP, NT> x, q;
        RowsInFlight<T, C, DVS, NT> y;
        const int x_st = (int)a.keys.st, y_st = (int)a.values.st, q_st = (int)a.queries.st;
        float g = 0.f;
        auto fetch_gates = [&](int n) {              // by the wave that makes the chunk's gates
            g = wb == NW - 1 && lane < C && n * C + lane < len ? G[(int64_t)(n * C + lane) * a.gates.st] : 0.f;
        };
        auto fetch = [&](int n) {                    // the rows that the pointers have come to
            const int left = len - n * C;
            const unsigned at = x.here() - NT;
            x.load(at, X, x_st, left, DK);
            q.load(at, Q, q_st, left, DK);
            y.load(at, Y, y_st, left, DV - dv0);
            X += (int64_t)C * x_st;
            Y += (int64_t)C * y_st;
            Q += (int64_t)C * q_st;
        };
        // chunk i and its gates to their place
        auto stage = [&](int i, int place) {
            const int n = first + i, chunk = place * kChunk, left = len - n * C;
            const unsigned at = x.here() - NT;
            if (wb == NW - 1) chunk_gates<C>(gates[place], g);
            x.store(at, sX + chunk, left, DK);
            q.store(at, sQ + chunk, left, DK);
            y.store(at, sY + chunk, left, DV - dv0);
        };
        // chunk i on its way
        auto bring = [&](int i) {
            if (i >= count) return;
            fetch_gates(first + i);
            fetch(first + i);
        };
        auto scores = [&](int i, int place) {
            // transposed: lane (r, c) has keys 4c .. 4c+3 of tile tj for query r of tile ti
            const int chunk = place * kChunk;
            const ChunkGates<C> &gate = gates[place];
            const TileX LX = tx.here();
#pragma unroll 1
            for (int n16 = wb; n16 < CT * (CT + 1) / 2; n16 += NW) {
                int ti, tj;
                triangle(n16, ti, tj);
                const int qi = 16 * ti + r, kj = 16 * tj + 4 * c;
                const float at = gate.sum[qi], at_rest = gate.rest[qi];
                const f32x4 to = *reinterpret_cast<const f32x4 *>(gate.sum + kj), to_rest = *reinterpret_cast<const f32x4 *>(gate.rest + kj);
                f32x4 s = tile_product<KS>(LX, sX + chunk, tj, sQ + chunk, ti);
                float p[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float weight = ChunkGates<C>::weight(at, at_rest, to[e], to_rest[e]);
                    p[e] = kj + e <= qi ? s[e] * weight : 0.f;
                }
                store_vec<T, 4>(sP + (i & 1) * kScores + n16 * 256 + 4 * lane, p);
            }
        };
        bring(0);
        stage(0, 0);
        bring(1);
        lds_barrier();
        scores(0, 0);
        if (count > 1) stage(1, 1);
        bring(2);
        lds_barrier();
        int next = 1, after = 2;
        for (int i = 0; i < count; ++i) {
            if (i + 2 < count) stage(i + 2, after);
            if (i + 1 < count) scores(i + 1, next);
            // (issuing these loads takes 2000 cycles, for which the scores would have to wait: B16 T1337 H16 DK64 DV128 64 us instead of 74)
            bring(i + 3);
            lds_barrier();
            next = after;
            after = after == 2 ? 0 : after + 1;
        }
    }
    // rows past the end of a shorter sequence
    for (int m = max(live, first); m < last; ++m)
        for (int i = tid; i < C * DVS / 8; i += 2 * NT) {
            const int t = m * C + i / (DVS / 8), col = dv0 + 8 * (i % (DVS / 8));
            if (t < T_ && col < DV) st8(static_cast<T *>(a.out) + ((b * a.n.T + t) * a.n.H + h) * DV + col, D8{});
        }
}

// What a segment adds to the state that leaves it (cotangents: the chunks in reverse, queries for keys and cotangents of out for values),
// and how much of the state that entered it is left.  Two chunks' rows in LDS, one barrier a chunk; rows are on their way for two
// chunks, since a chunk takes less time than memory does.  A wave of its own makes the gates: 600 of a chunk's 4400 cycles, for which the
// others had to wait.  B1 T32768 H8 D128: 41 us for 130 MB, 3.2 TB/s: two waves a SIMD, whose vector and matrix instructions overlap little.
template <typename T, int DKP, int NW, bool kReverse>
__global__ __launch_bounds__(NW * 64 + 64) __attribute__((amdgpu_waves_per_eu(DKP == 256 && NW == 4 ? 2 : 3))) void decay_states_kernel(const ForwardArgs a)
{
    constexpr int C = DecayChunk<T>::C, NT = NW * 64, DVS = 16 * NW, TILES = DKP / 16, CS = C / 32;
    typedef typename FragTypes<T>::d8 D8;
    typedef LdsTile<T, DKP> TileX;
    typedef LdsTile<T, DVS> TileY;
    constexpr int kX = C * TileX::kRow, kChunk = kX + C * TileY::kRow;
    extern __shared__ char smem[];
    T *sX = reinterpret_cast<T *>(smem), *sY = sX + kX;
    ChunkGates<C> *gates = reinterpret_cast<ChunkGates<C> *>(sX + 2 * kChunk);

    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, r = lane & 15, c = lane >> 4;
    const unsigned H = (unsigned)a.n.H, pair = pair_of(blockIdx.x, a.n);
    const int64_t bh = pair, b = pair / H, h = pair % H, hk = pair % H / (H / (unsigned)a.n.HK);
    const int dv0 = blockIdx.y * DVS, DK = (int)a.n.DK, DV = (int)a.n.DV;
    const int T_ = (int)a.n.T, len = a.lengths ? min(max(a.lengths[b], 0), T_) : T_;
    const int order = blockIdx.z, tail = a.plan.tail((len + C - 1) / C), seg = kReverse ? tail - order : order;
    if (kReverse ? seg <= 0 : seg >= tail) return;      // no segment that it would be handed to
    const int first = a.plan.first(seg), live = min(a.plan.first(seg + 1), (len + C - 1) / C);
    const int count = live - first, step = kReverse ? -1 : 1, start = kReverse ? live - 1 : first;
    const T *X = static_cast<const T *>(a.keys.p) + b * a.keys.sb + hk * a.keys.sh + (int64_t)start * C * a.keys.st;
    const T *Y = static_cast<const T *>(a.values.p) + b * a.values.sb + h * a.values.sh + dv0 + (int64_t)start * C * a.values.st;
    const float *G = static_cast<const float *>(a.gates.p) + b * a.gates.sb + h * a.gates.sh;
    const TileX tx;
    const TileY ty;

    if (w == NW) {
        auto gate = [&](int i) {
            const int n = start + i * step;
            return i < count && lane < C && lane < len - n * C ? G[(int64_t)(n * C + lane) * a.gates.st] : 0.f;
        };
        float even = gate(0), odd = gate(1);
        double total = chunk_gates<C>(gates[0], even);
        even = gate(2);
        lds_barrier();
        for (int i = 0; i < count; ++i) {
            if (i + 1 < count) total += chunk_gates<C>(gates[(i + 1) & 1], odd);
            odd = even;
            even = gate(i + 3);
            lds_barrier();
        }
        if (blockIdx.y == 0 && lane == 0) a.decays[bh * a.plan.segments + order] = fast_exp2((float)total);
        return;
    }

    // key features 16t + 4c .., value feature 16w + r
    f32x4 S[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) S[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (order == 0) {
        const bool mine = dv0 + 16 * w < DV;
        const unsigned at = (4 * c + (r & 3)) * DV + dv0 + 16 * w + (r & ~3);      // four columns a lane
#pragma unroll
        for (int t = 0; t < TILES; ++t)
            if (mine && 16 * t < DK) {
                float x[4];
                load_hidden<4>(a.hidden, a.hidden_dtype, bh * DK * DV + (at + 16 * t * DV), x);
                quad_transpose(x);
                S[t] = f32x4{x[0], x[1], x[2], x[3]};
            }
    }

    struct Flight {
        RowsInFlight<T, C, DKP, NT> x;
        RowsInFlight<T, C, DVS, NT> y;
    } even, odd;
    const int x_st = (int)a.keys.st, y_st = (int)a.values.st;
    auto fetch = [&](Flight &f, int i) {         // chunk i, which the pointers have come to
        if (i >= count) return;
        const int n = start + i * step, left = len - n * C;
        const unsigned at = f.x.here();
        f.x.load(at, X, x_st, left, DK);
        f.y.load(at, Y, y_st, left, DV - dv0);
        X += (int64_t)(step * C) * x_st;
        Y += (int64_t)(step * C) * y_st;
    };
    auto stage = [&](Flight &f, int i) {         // to its place
        if (i >= count) return;
        const int left = len - (start + i * step) * C, chunk = (i & 1) * kChunk;
        const unsigned at = f.x.here();
        f.x.store(at, sX + chunk, left, DK);
        f.y.store(at, sY + chunk, left, DV - dv0);
    };
    auto add = [&](int i) {
        const ChunkGates<C> &gate = gates[i & 1];
        const int chunk = (i & 1) * kChunk;
        const TileX LX = tx.here();
        const float whole = gate.whole;
        const float *weight = kReverse ? gate.from_start : gate.to_end;
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[t][e] *= whole;
#pragma unroll
        for (int ks = 0; ks < CS; ++ks) {
            float v[8], by[8];
            unpack8(ty.columns(sY + chunk, ks, w), v);
            two_tiles(*reinterpret_cast<const f32x4 *>(weight + 32 * ks + 4 * c), *reinterpret_cast<const f32x4 *>(weight + 32 * ks + 16 + 4 * c), by);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= by[e];
            const Split<T, 3> op(v);
#pragma unroll
            for (int t = 0; t < TILES; t += 2) {
                const D8 k[2] = {LX.columns(sX + chunk, ks, t), LX.columns(sX + chunk, ks, t + 1)};
                mma_right(k, op, S + t);
                if (t % 4 == 2) __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    auto advance = [&](Flight &f, int i) {       // chunk i; the next one, which f holds, to its place
        stage(f, i + 1);
        fetch(f, i + 3);
        add(i);
        lds_barrier();
    };
    fetch(even, 0);
    fetch(odd, 1);
    stage(even, 0);
    fetch(even, 2);
    lds_barrier();
    for (int i = 0; i < count; i += 2) {
        advance(odd, i);
        if (i + 1 < count) advance(even, i + 1);
    }
    f32x4 *to = reinterpret_cast<f32x4 *>(a.entering + ((bh * a.plan.segments + order) * gridDim.y + blockIdx.y) * (int64_t)(DKP * DVS)) + w * TILES * 64 + lane;
#pragma unroll
    for (int t = 0; t < TILES; ++t) to[t * 64] = S[t];
}

// The states that enter segments 2, 3, ... from what each segment adds, in place: slot s holds the state after segment s (of cotangents,
// after the s-th from the sequence's end).
// One value a thread, all slots one after the other: for all that the compiler knows a store may change the next slot, so every load waits for the store
// before it.  A chain of as many memory latencies as there are segments bounds it (B1 T32768 H8 D128, 32 segments: 12.5 us for 31 MB, of
// which a copy of as much takes 6).
__global__ __launch_bounds__(256) void decay_scan_kernel(float *__restrict__ entering, const float *__restrict__ decays,
                                                         const int32_t *__restrict__ lengths, DecaySizes n, DecayPlan plan, int C,
                                                         int64_t count)
{
    const int64_t at = blockIdx.x * (int64_t)256 + threadIdx.x, bh = blockIdx.y, segments = plan.segments;
    if (at >= count) return;
    const int T = (int)n.T, len = lengths ? min(max(lengths[blockIdx.y / (unsigned)n.H], 0), T) : T, tail = plan.tail((len + C - 1) / C);
    float *p = entering + bh * segments * count + at;
    const float *d = decays + bh * segments;
    float s = p[0];
    for (int64_t i = 1; i < tail; ++i) {
        s = d[i] * s + p[i * count];
        p[i * count] = s;
    }
}

template <typename T, int DKP, int NW, bool kReverse> int launch_states(hipStream_t stream, const ForwardArgs &a)
{
    static LdsGrant grant;
    constexpr int C = DecayChunk<T>::C;
    constexpr size_t lds = sizeof(T) * 2 * C * (LdsTile<T, DKP>::kRow + LdsTile<T, 16 * NW>::kRow) + 2 * sizeof(ChunkGates<C>);
    if (int e = allow_lds(grant, reinterpret_cast<const void *>(decay_states_kernel<T, DKP, NW, kReverse>), lds)) return e;
    const dim3 grid(a.n.B * a.n.H, decay_slabs(a.n.DV), a.plan.segments - 1);
    decay_states_kernel<T, DKP, NW, kReverse><<<grid, NW * 64 + 64, lds, stream>>>(a);
    return launch_status();
}
template <typename T, bool kReverse> int dispatch_states(hipStream_t stream, const ForwardArgs &a)
{
    const int64_t key = decay_key_width(a.n.DK);
    if (decay_value_slab(a.n.DV) == 64)
        return key == 64    ? launch_states<T, 64, 4, kReverse>(stream, a)
               : key == 128 ? launch_states<T, 128, 4, kReverse>(stream, a)
                            : launch_states<T, 256, 4, kReverse>(stream, a);
    return key == 64    ? launch_states<T, 64, 8, kReverse>(stream, a)
           : key == 128 ? launch_states<T, 128, 8, kReverse>(stream, a)
                        : launch_states<T, 256, 8, kReverse>(stream, a);
}

// One workgroup of decay_forward_kernel is the fastest that a compute unit can be kept busy with (B16 T1024 H16 D128, 256 workgroups:
// 72 us, decay_pass_kernel 91), but its LDS and registers leave no room for a second one; where there are more workgroups than compute units,
// two of decay_pass_kernel at a time do more (64 x 64 features, 512 workgroups: 72 us against 77; 128 x 128: 145 against 148).
template <typename T, int DKP, int NW> int launch_forward(hipStream_t stream, const ForwardArgs &a)
{
    constexpr int C = DecayChunk<T>::C;
    constexpr size_t lds = sizeof(T) * (3 * C * (2 * LdsTile<T, DKP>::kRow + LdsTile<T, 16 * NW>::kRow) + (C / 16) * (C / 16 + 1) * 256) +
                           3 * sizeof(ChunkGates<C>);
    const dim3 grid(a.n.B * a.n.H, decay_slabs(a.n.DV), a.plan.segments);
    if constexpr (DKP <= 128 && lds <= 160 * 1024) {
        if ((int64_t)grid.x * grid.y * grid.z <= kComputeUnits) {
            static LdsGrant grant;
            if (int e = allow_lds(grant, reinterpret_cast<const void *>(decay_forward_kernel<T, DKP, NW>), lds)) return e;
            decay_forward_kernel<T, DKP, NW><<<grid, NW * 128, lds, stream>>>(a);
            return launch_status();
        }
    }
    static LdsGrant grant;
    constexpr size_t pass_lds = sizeof(T) * C * (2 * LdsTile<T, DKP>::kRow + LdsTile<T, 16 * NW>::kRow + LdsTile<T, C>::kRow) + 2 * sizeof(ChunkGates<C>);
    if (int e = allow_lds(grant, reinterpret_cast<const void *>(decay_pass_kernel<T, DKP, NW>), pass_lds)) return e;
    decay_pass_kernel<T, DKP, NW><<<grid, NW * 64, pass_lds, stream>>>(a);
    return launch_status();
}
template <typename T> int dispatch_forward(hipStream_t stream, const ForwardArgs &a)
{
    const int64_t key = decay_key_width(a.n.DK);
    if (decay_value_slab(a.n.DV) == 64)
        return key == 64    ? launch_forward<T, 64, 4>(stream, a)
               : key == 128 ? launch_forward<T, 128, 4>(stream, a)
                            : launch_forward<T, 256, 4>(stream, a);
    return key == 64    ? launch_forward<T, 64, 8>(stream, a)
           : key == 128 ? launch_forward<T, 128, 8>(stream, a)
                        : launch_forward<T, 256, 8>(stream, a);
}
}  // namespace

int decay_entering_states(void *stream, bool cotangents, const DecaySizes &n, const DecayPlan &plan, gla_dtype dtype,
                          gla_dtype hidden_dtype, const void *hidden, const DecayRows &gates, const DecayRows &keys,
                          const DecayRows &values, const int32_t *lengths, float *states, float *decays)
{
    if (plan.segments < 2) return 0;
    ForwardArgs a{};
    a.n = n;
    a.plan = plan;
    a.gates = gates;
    a.keys = keys;
    a.values = values;
    a.lengths = lengths;
    a.hidden = hidden;
    a.hidden_dtype = hidden_dtype;
    a.entering = states;
    a.decays = decays;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    int e = dtype == GLA_BF16 ? (cotangents ? dispatch_states<__bf16, true>(s, a) : dispatch_states<__bf16, false>(s, a))
                              : (cotangents ? dispatch_states<float, true>(s, a) : dispatch_states<float, false>(s, a));
    if (e || plan.segments < 3) return e;
    const int64_t count = decay_slabs(n.DV) * decay_value_slab(n.DV) * decay_key_width(n.DK);
    decay_scan_kernel<<<dim3((count + 255) / 256, n.B * n.H), 256, 0, s>>>(states, decays, lengths, n, plan,
                                                                                 dtype == GLA_BF16 ? DecayChunk<__bf16>::C : DecayChunk<float>::C, count);
    return launch_status();
}

int decay_forward(void *stream, const DecaySizes &n, const DecayPlan &plan, gla_dtype dtype, gla_dtype hidden_dtype,
                  const void *hidden_init, const DecayRows &gates, const DecayRows &keys, const DecayRows &values,
                  const DecayRows &queries, const int32_t *lengths, void *hidden_final, void *out, float *kept, float *entering,
                  float *decays)
{
    int e = decay_entering_states(stream, false, n, plan, dtype, hidden_dtype, hidden_init, gates, keys, values, lengths,
                                  entering, decays);
    if (e) return e;
    ForwardArgs a{n, plan, gates, keys, values, queries, lengths, hidden_init, hidden_dtype, hidden_final, out, kept, entering, decays};
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == GLA_BF16 ? dispatch_forward<__bf16>(s, a) : dispatch_forward<float>(s, a);
}

}  // namespace gla
