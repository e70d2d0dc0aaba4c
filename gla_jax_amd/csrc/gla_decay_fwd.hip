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

// One workgroup: a (batch, head) pair's segment and 16 * NW value features; wave w holds the columns 16w .. 16w+15 of the
// state, TILES accumulators of 16 key features each.  Scores are formed transposed, so that a lane holds four neighbouring
// keys of one query, and kept in `T`: their one rounding adds as much as that of out itself.  The state is an operand in `T`
// too where it meets the queries; what it accumulates comes from values scaled in 32 bits and handed over in three parts,
// since hidden_final is a 32-bit result.
template <typename T, int DKP, int NW, DecayPass PASS>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(DKP == 256 ? 2 : DKP == 128 && NW == 4 ? 3 : 4))) void decay_pass_kernel(const ForwardArgs a)
{
    constexpr int C = DecayChunk<T>::C, NT = NW * 64, DVS = 16 * NW, TILES = DKP / 16, KS = DKP / 32, CS = C / 32, CT = C / 16;
    constexpr bool kOut = PASS == kDecayForward, kReverse = PASS == kDecayCotangents;
    typedef typename FragTypes<T>::d8 D8;
    typedef LdsTile<T, DKP> TileX;
    typedef LdsTile<T, DVS> TileY;
    typedef LdsTile<T, C> TileP;
    extern __shared__ char smem[];
    T *sX = reinterpret_cast<T *>(smem), *sY = sX + C * TileX::kRow, *sQ = sY + C * TileY::kRow, *sP = sQ + (kOut ? C * TileX::kRow : 0);
    ChunkGates<C> *gates = reinterpret_cast<ChunkGates<C> *>(reinterpret_cast<char *>(sP + (kOut ? C * TileP::kRow : 0)));

    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, r = lane & 15, c = lane >> 4;
    const int64_t bh = pair_of(blockIdx.x, a.n), b = bh / a.n.H, h = bh % a.n.H, hk = h / (a.n.H / a.n.HK);
    const int dv0 = blockIdx.y * DVS, DK = (int)a.n.DK, DV = (int)a.n.DV;
    const int64_t order = blockIdx.z, seg = kReverse ? a.plan.segments - 1 - order : order;
    const int T_ = (int)a.n.T, len = a.lengths ? min(max(a.lengths[b], 0), T_) : T_;
    const int first = (int)a.plan.first(seg), last = (int)a.plan.first(seg + 1), live = min(last, (len + C - 1) / C);
    const T *X = static_cast<const T *>(a.keys.p) + b * a.keys.sb + hk * a.keys.sh;
    const T *Y = static_cast<const T *>(a.values.p) + b * a.values.sb + h * a.values.sh + dv0;
    const T *Q = kOut ? static_cast<const T *>(a.queries.p) + b * a.queries.sb + hk * a.queries.sh : nullptr;
    const float *G = static_cast<const float *>(a.gates.p) + b * a.gates.sb + h * a.gates.sh;
    const bool mine = dv0 + 16 * w < DV;         // the wave's columns exist
    const TileX tx;
    const TileY ty;
    const TileP tp;
    const int64_t slab = (bh * a.plan.segments * gridDim.y + blockIdx.y) * (int64_t)(DKP * DVS);
    const int64_t seg_step = (int64_t)gridDim.y * (DKP * DVS);

    // ---- the state that enters ----
    const unsigned hidden_at = (4 * c + (r & 3)) * DV + dv0 + 16 * w + (r & ~3);      // of tile 0, four columns a lane
    f32x4 S[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) S[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (order == 0) {
#pragma unroll
        for (int t = 0; t < TILES; ++t)
            if (mine && 16 * t < DK) {
                float x[4];
                load_hidden<4>(a.hidden, a.hidden_dtype, bh * DK * DV + (hidden_at + 16 * t * DV), x);
                quad_transpose(x);
                S[t] = f32x4{x[0], x[1], x[2], x[3]};
            }
    } else if (kOut) {
        const f32x4 *from = reinterpret_cast<const f32x4 *>(a.entering + slab + (order - 1) * seg_step) + w * TILES * 64 + lane;
#pragma unroll
        for (int t = 0; t < TILES; ++t) S[t] = from[t * 64];
    }

    RowsInFlight<T, C, DKP, NT> x, q;
    RowsInFlight<T, C, DVS, NT> y;
    const int x_st = (int)a.keys.st, y_st = (int)a.values.st, q_st = kOut ? (int)a.queries.st : 0;
    float g = 0.f;
    auto fetch_gates = [&](int n) {              // by the wave that makes the chunk's gates
        g = w == NW - 1 && lane < C && n * C + lane < len ? G[(int64_t)(n * C + lane) * a.gates.st] : 0.f;
    };
    auto fetch = [&](int n) {                    // the rows that the pointers have come to
        const int left = len - n * C;
        x.load(X, x_st, left, DK);
        y.load(Y, y_st, left, DV - dv0);
        if constexpr (kOut) q.load(Q, q_st, left, DK);
        X += (int64_t)(kReverse ? -C : C) * x_st;
        Y += (int64_t)(kReverse ? -C : C) * y_st;
        if constexpr (kOut) Q += (int64_t)C * q_st;
    };
    if constexpr (kOut) {
        // the upper tiles that a step of 32 keys takes along with the diagonal's
        for (int i = tid; i < C * TileP::kRow; i += NT) sP[i] = (T)0.f;
    }
    double total = 0.0;
    const int count = max(live - first, 0), step = kReverse ? -1 : 1;
    int n = kReverse ? live - 1 : first;
    if (count > 0) {
        X += (int64_t)n * C * a.keys.st;
        Y += (int64_t)n * C * a.values.st;
        if (kOut) Q += (int64_t)n * C * a.queries.st;
        fetch_gates(n);
        fetch(n);
        if (w == NW - 1) total += chunk_gates<C>(gates[0], g);
        if (count > 1) fetch_gates(n + step);
    }
    for (int i = 0; i < count; ++i, n += step) {
        const ChunkGates<C> &gate = gates[i & 1];
        lds_barrier();                            // the last chunk's tiles are read
        x.store(sX, len - n * C, DK);
        y.store(sY, len - n * C, DV - dv0);
        if constexpr (kOut) q.store(sQ, len - n * C, DK);
        lds_barrier();
        if (i + 1 < count) fetch(n + step);

        if constexpr (kOut) {
            // scores, transposed: lane (r, c) has keys 4c .. 4c+3 of tile tj for query r of tile ti
            const TileX LX = tx.here();
            const TileP LP = tp.here();
#pragma unroll 1
            for (int n16 = w; n16 < CT * (CT + 1) / 2; n16 += NW) {
                int ti, tj;
                triangle(n16, ti, tj);
                f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) s = mma_d(LX.rows(sX, tj, ks), LX.rows(sQ, ti, ks), s);
                const int qi = 16 * ti + r, kj = 16 * tj + 4 * c;
                const float at = gate.sum[qi], at_rest = gate.rest[qi];
                const f32x4 to = *reinterpret_cast<const f32x4 *>(gate.sum + kj), to_rest = *reinterpret_cast<const f32x4 *>(gate.rest + kj);
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
            total += chunk_gates<C>(gates[(i + 1) & 1], g);
            if (i + 2 < count) fetch_gates(n + 2 * step);
        }

        D8 yc[CS];                                // the wave's value columns, tokens as the contracted index
#pragma unroll
        for (int ks = 0; ks < CS; ++ks) yc[ks] = ty.columns(sY, ks, w);

        typename Packed4<T>::t result[CT];
        if constexpr (kOut) {
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
        if (kOut && a.kept) {
            // (four bytes a lane, 64 side by side: moving the values between lanes for wider stores costs more than it saves)
            float *to = a.kept + ((bh * a.plan.chunks + n) * DK * DV + dv0 + 16 * w);
            const unsigned at = (4 * c * DV + again(r)) * 4;
            const int dk = again_uniform(mine ? DK : 0);
#pragma unroll
            for (int t = 0; t < TILES; ++t)
                if (16 * t < dk)
#pragma unroll
                    for (int e = 0; e < 4; ++e) *at_bytes(to + (size_t)((16 * t + e) * DV), at) = S[t][e];
        }

        // ---- the chunk's own contribution ----
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
        if constexpr (kOut) {
            wait_for_memory();
            T *out = static_cast<T *>(a.out) + ((b * a.n.T + n * C) * a.n.H + h) * DV + dv0 + 16 * w;
            const unsigned row = (unsigned)a.n.H * DV, at = (again(r) * row + 4 * c) * (unsigned)sizeof(T);
#pragma unroll
            for (int ti = 0; ti < CT; ++ti)
                if (mine && n * C + 16 * ti + r < T_)
                    *reinterpret_cast<typename Packed4<T>::t *>(at_bytes(out + (size_t)(16 * ti * row), at)) = result[ti];
        }
    }

    if constexpr (kOut) {
        // rows past the end of a shorter sequence
        for (int m = max(live, first); m < last; ++m)
            for (int i = tid; i < C * DVS / 8; i += NT) {
                const int t = m * C + i / (DVS / 8), col = dv0 + 8 * (i % (DVS / 8));
                if (t < T_ && col < DV) st8(static_cast<T *>(a.out) + ((b * a.n.T + t) * a.n.H + h) * DV + col, D8{});
            }
        if (seg == a.plan.segments - 1) {
            const unsigned at = again(hidden_at);
#pragma unroll
            for (int t = 0; t < TILES; ++t)
                if (mine && 16 * t < DK) {
                    float s[4] = {S[t][0], S[t][1], S[t][2], S[t][3]};
                    quad_transpose(s);
                    store_hidden<4>(a.hidden_final, a.hidden_dtype, bh * DK * DV + (at + 16 * t * DV), s);
                }
        }
    } else {
        f32x4 *to = reinterpret_cast<f32x4 *>(a.entering + slab + order * seg_step) + w * TILES * 64 + lane;
#pragma unroll
        for (int t = 0; t < TILES; ++t) to[t * 64] = S[t];
        if (blockIdx.y == 0 && tid == NT - 1) a.decays[bh * a.plan.segments + order] = fast_exp2((float)total);
    }
}

// The states that enter segments 2, 3, ... from what each segment adds, in place: slot s holds the state after segment s.
// One value a thread: four would make wider accesses of it, but B1 T32768 H8 D128 then has 128 workgroups (20 us).
__global__ __launch_bounds__(256) void decay_scan_kernel(float *__restrict__ entering, const float *__restrict__ decays,
                                                         int64_t segments, int64_t count)
{
    const int64_t at = blockIdx.x * (int64_t)256 + threadIdx.x, bh = blockIdx.y;
    if (at >= count) return;
    float *p = entering + bh * segments * count + at;
    const float *d = decays + bh * segments;
    float s = p[0];
#pragma unroll 16
    for (int64_t i = 1; i + 1 < segments; ++i) {
        s = d[i] * s + p[i * count];
        p[i * count] = s;
    }
}

template <typename T, int DKP, int NW, DecayPass PASS> int launch_pass(hipStream_t stream, const ForwardArgs &a)
{
    static LdsGrant grant;
    constexpr int C = DecayChunk<T>::C;
    constexpr size_t lds = sizeof(T) * (C * LdsTile<T, DKP>::kRow * (PASS == kDecayForward ? 2 : 1) + C * LdsTile<T, 16 * NW>::kRow +
                                        (PASS == kDecayForward ? C * LdsTile<T, C>::kRow : 0)) +
                           2 * sizeof(ChunkGates<C>);
    if (int e = allow_lds(grant, reinterpret_cast<const void *>(decay_pass_kernel<T, DKP, NW, PASS>), lds)) return e;
    const dim3 grid(a.n.B * a.n.H, decay_slabs(a.n.DV), PASS == kDecayForward ? a.plan.segments : a.plan.segments - 1);
    decay_pass_kernel<T, DKP, NW, PASS><<<grid, NW * 64, lds, stream>>>(a);
    return launch_status();
}
template <typename T, DecayPass PASS> int dispatch_pass(hipStream_t stream, const ForwardArgs &a)
{
    const int64_t key = decay_key_width(a.n.DK);
    if (decay_value_slab(a.n.DV) == 64)
        return key == 64    ? launch_pass<T, 64, 4, PASS>(stream, a)
               : key == 128 ? launch_pass<T, 128, 4, PASS>(stream, a)
                            : launch_pass<T, 256, 4, PASS>(stream, a);
    return key == 64    ? launch_pass<T, 64, 8, PASS>(stream, a)
           : key == 128 ? launch_pass<T, 128, 8, PASS>(stream, a)
                        : launch_pass<T, 256, 8, PASS>(stream, a);
}

}  // namespace

int decay_entering_states(void *stream, DecayPass pass, const DecaySizes &n, const DecayPlan &plan, gla_dtype dtype,
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
    int e = dtype == GLA_BF16 ? (pass == kDecayStates ? dispatch_pass<__bf16, kDecayStates>(s, a) : dispatch_pass<__bf16, kDecayCotangents>(s, a))
                              : (pass == kDecayStates ? dispatch_pass<float, kDecayStates>(s, a) : dispatch_pass<float, kDecayCotangents>(s, a));
    if (e || plan.segments < 3) return e;
    const int64_t count = decay_slabs(n.DV) * decay_value_slab(n.DV) * decay_key_width(n.DK);
    decay_scan_kernel<<<dim3((count + 255) / 256, n.B * n.H), 256, 0, s>>>(states, decays, plan.segments, count);
    return launch_status();
}

int decay_forward(void *stream, const DecaySizes &n, const DecayPlan &plan, gla_dtype dtype, gla_dtype hidden_dtype,
                  const void *hidden_init, const DecayRows &gates, const DecayRows &keys, const DecayRows &values,
                  const DecayRows &queries, const int32_t *lengths, void *hidden_final, void *out, float *kept, float *entering,
                  float *decays)
{
    int e = decay_entering_states(stream, kDecayStates, n, plan, dtype, hidden_dtype, hidden_init, gates, keys, values, lengths,
                                  entering, decays);
    if (e) return e;
    ForwardArgs a{n, plan, gates, keys, values, queries, lengths, hidden_init, hidden_dtype, hidden_final, out, kept, entering, decays};
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == GLA_BF16 ? dispatch_pass<__bf16, kDecayForward>(s, a) : dispatch_pass<float, kDecayForward>(s, a);
}

}  // namespace gla
