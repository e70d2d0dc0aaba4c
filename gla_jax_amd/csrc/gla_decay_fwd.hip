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
__global__ __launch_bounds__(NW * 64) void decay_pass_kernel(const ForwardArgs a)
{
    constexpr int C = DecayChunk<T>::C, NT = NW * 64, DVS = 16 * NW, TILES = DKP / 16, KS = DKP / 32, CS = C / 32, CT = C / 16;
    constexpr int SX = lds_stride<T>(DKP), SY = lds_stride<T>(DVS), SP = lds_stride<T>(C);
    constexpr bool kOut = PASS == kDecayForward, kReverse = PASS == kDecayCotangents;
    typedef typename FragTypes<T>::d8 D8;
    extern __shared__ char smem[];
    T *sX = reinterpret_cast<T *>(smem), *sY = sX + C * SX, *sQ = sY + C * SY, *sP = sQ + (kOut ? C * SX : 0);
    ChunkGates<C> &gate = *reinterpret_cast<ChunkGates<C> *>(reinterpret_cast<char *>(sP + (kOut ? C * SP : 0)));

    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, r = lane & 15, c = lane >> 4;
    const int64_t bh = blockIdx.x, b = bh / a.n.H, h = bh % a.n.H, hk = h / (a.n.H / a.n.HK);
    const int dv0 = blockIdx.y * DVS, DK = (int)a.n.DK, DV = (int)a.n.DV;
    const int64_t order = blockIdx.z, seg = kReverse ? a.plan.segments - 1 - order : order;
    const int64_t len = a.lengths ? min(max((int64_t)a.lengths[b], (int64_t)0), a.n.T) : a.n.T;
    const int64_t first = seg * a.plan.per, last = min(first + a.plan.per, a.plan.chunks), live = min(last, (len + C - 1) / C);
    const T *X = static_cast<const T *>(a.keys.p) + b * a.keys.sb + hk * a.keys.sh;
    const T *Y = static_cast<const T *>(a.values.p) + b * a.values.sb + h * a.values.sh + dv0;
    const T *Q = kOut ? static_cast<const T *>(a.queries.p) + b * a.queries.sb + hk * a.queries.sh : nullptr;
    const float *G = static_cast<const float *>(a.gates.p) + b * a.gates.sb + h * a.gates.sh;
    const bool mine = dv0 + 16 * w < DV;         // the wave's columns exist
    const DecayLane<T> LX(SX), LY(SY), LP(SP);
    const int64_t slab = (bh * a.plan.segments * gridDim.y + blockIdx.y) * (int64_t)(DKP * DVS);
    const int64_t seg_step = (int64_t)gridDim.y * (DKP * DVS);

    // ---- the state that enters ----
    f32x4 S[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) S[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (order == 0) {
#pragma unroll
        for (int t = 0; t < TILES; ++t)
            if (mine && 16 * t < DK) {
                float x[4];
                load_hidden<4>(a.hidden, a.hidden_dtype, (bh * DK + 16 * t + 4 * c + (r & 3)) * DV + dv0 + 16 * w + (r & ~3), x);
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
    float g = 0.f;
    auto fetch = [&](int64_t n) {
        x.load(X, a.keys.st, n * C, len, DK);
        y.load(Y, a.values.st, n * C, len, DV - dv0);
        if constexpr (kOut) q.load(Q, a.queries.st, n * C, len, DK);
        g = w == 0 && lane < C && n * C + lane < len ? G[(n * C + lane) * a.gates.st] : 0.f;
    };
    if constexpr (kOut) {
        // the upper tiles that a step of 32 keys takes along with the diagonal's
        for (int i = tid; i < C * SP; i += NT) sP[i] = (T)0.f;
    }
    double total = 0.0;
    const int64_t count = max(live - first, (int64_t)0);
    if (count > 0) fetch(kReverse ? live - 1 : first);
    for (int64_t i = 0; i < count; ++i) {
        const int64_t n = kReverse ? live - 1 - i : first + i;
        lds_barrier();                            // the last chunk's tiles are read
        x.store(sX, SX);
        y.store(sY, SY);
        if constexpr (kOut) q.store(sQ, SX);
        if (w == 0) total += chunk_gates<C>(gate, g);
        lds_barrier();
        if (i + 1 < count) fetch(kReverse ? n - 1 : n + 1);

        if (kOut && a.kept) {
            float *to = a.kept + (bh * a.plan.chunks + n) * DK * DV;
#pragma unroll
            for (int t = 0; t < TILES; ++t)
                if (mine && 16 * t < DK) {
                    float s[4] = {S[t][0], S[t][1], S[t][2], S[t][3]};
                    quad_transpose(s);
                    store_vec<float, 4>(to + (16 * t + 4 * c + (r & 3)) * DV + dv0 + 16 * w + (r & ~3), s);
                }
        }

        D8 yc[CS];                                // the wave's value columns, tokens as the contracted index
#pragma unroll
        for (int ks = 0; ks < CS; ++ks) yc[ks] = lds_columns(sY + 32 * ks * SY + 16 * w + LY.col, SY);

        if constexpr (kOut) {
            // scores, transposed: lane (r, c) has keys 4c .. 4c+3 of tile tj for query r of tile ti
            for (int n16 = w; n16 < CT * (CT + 1) / 2; n16 += NW) {
                int ti, tj;
                triangle(n16, ti, tj);
                f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
                    s = mma_d(ld8(sX + 16 * tj * SX + LX.row + 32 * ks), ld8(sQ + 16 * ti * SX + LX.row + 32 * ks), s);
                const int qi = 16 * ti + r, kj = 16 * tj + 4 * c;
                const double at = gate.sum[qi];
                float p[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float weight = fast_exp2((float)(at - gate.sum[kj + e]));
                    p[e] = kj + e <= qi ? s[e] * weight : 0.f;
                }
                store_vec<T, 4>(sP + qi * SP + kj, p);
            }
            // the state's part, while the other waves finish their scores
            f32x4 o[CT];
#pragma unroll
            for (int ti = 0; ti < CT; ++ti) o[ti] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                float s[8];
                two_tiles(S[2 * ks], S[2 * ks + 1], s);
                const Split<T, 1> op(s);
#pragma unroll
                for (int ti = 0; ti < CT; ++ti) o[ti] = op.left(lds_two_halves(sQ + 16 * ti * SX + LX.row2 + 32 * ks), o[ti]);
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
                for (int ks = 0; ks <= ti / 2; ++ks) o[ti] = mma_d(yc[ks], ld8(sP + 16 * ti * SP + LP.row + 32 * ks), o[ti]);
                const int64_t t = n * C + 16 * ti + r;
                if (mine && t < a.n.T) {
                    const float v[4] = {o[ti][0], o[ti][1], o[ti][2], o[ti][3]};
                    store_vec<T, 4>(static_cast<T *>(a.out) + ((b * a.n.T + t) * a.n.H + h) * DV + dv0 + 16 * w + 4 * c, v);
                }
            }
        }

        // ---- the chunk's own contribution ----
        const float whole = gate.whole;
        const float *weight = kReverse ? gate.from_start : gate.to_end;
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[t][e] *= whole;
#pragma unroll
        for (int ks = 0; ks < CS; ++ks) {
            float v[8];
            unpack8(yc[ks], v);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= weight[32 * ks + 8 * c + e];
            const Split<T, 3> op(v);
#pragma unroll
            for (int t = 0; t < TILES; ++t) S[t] = op.right(lds_columns(sX + 32 * ks * SX + 16 * t + LX.col, SX), S[t]);
        }
    }

    if constexpr (kOut) {
        // rows past the end of a shorter sequence
        for (int64_t n = max(live, first); n < last; ++n)
            for (int i = tid; i < C * DVS / 8; i += NT) {
                const int64_t t = n * C + i / (DVS / 8);
                const int col = dv0 + 8 * (i % (DVS / 8));
                if (t < a.n.T && col < DV) st8(static_cast<T *>(a.out) + ((b * a.n.T + t) * a.n.H + h) * DV + col, D8{});
            }
        if (seg == a.plan.segments - 1) {
#pragma unroll
            for (int t = 0; t < TILES; ++t)
                if (mine && 16 * t < DK) {
                    float s[4] = {S[t][0], S[t][1], S[t][2], S[t][3]};
                    quad_transpose(s);
                    store_hidden<4>(a.hidden_final, a.hidden_dtype,
                                    (bh * DK + 16 * t + 4 * c + (r & 3)) * DV + dv0 + 16 * w + (r & ~3), s);
                }
        }
    } else {
        f32x4 *to = reinterpret_cast<f32x4 *>(a.entering + slab + order * seg_step) + w * TILES * 64 + lane;
#pragma unroll
        for (int t = 0; t < TILES; ++t) to[t * 64] = S[t];
        if (blockIdx.y == 0 && tid == 0) a.decays[bh * a.plan.segments + order] = fast_exp2((float)total);
    }
}

// The states that enter segments 2, 3, ... from what each segment adds, in place: slot s holds the state after segment s.
__global__ __launch_bounds__(256) void decay_scan_kernel(float *__restrict__ entering, const float *__restrict__ decays,
                                                         int64_t segments, int64_t quads)
{
    const int64_t at = blockIdx.x * (int64_t)256 + threadIdx.x, bh = blockIdx.y;
    if (at >= quads) return;
    f32x4 *p = reinterpret_cast<f32x4 *>(entering) + bh * segments * quads + at;
    const float *d = decays + bh * segments;
    f32x4 s = p[0];
#pragma unroll 8
    for (int64_t i = 1; i + 1 < segments; ++i) {
        const f32x4 add = p[i * quads];
        const float by = d[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] = by * s[e] + add[e];
        p[i * quads] = s;
    }
}

template <typename T, int DKP, int NW, DecayPass PASS> int launch_pass(hipStream_t stream, const ForwardArgs &a)
{
    static LdsGrant grant;
    constexpr int C = DecayChunk<T>::C;
    constexpr size_t lds = sizeof(T) * (C * lds_stride<T>(DKP) * (PASS == kDecayForward ? 2 : 1) + C * lds_stride<T>(16 * NW) +
                                        (PASS == kDecayForward ? C * lds_stride<T>(C) : 0)) +
                           sizeof(ChunkGates<C>);
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
    const int64_t quads = decay_slabs(n.DV) * decay_value_slab(n.DV) * decay_key_width(n.DK) / 4;
    decay_scan_kernel<<<dim3((quads + 255) / 256, n.B * n.H), 256, 0, s>>>(states, decays, plan.segments, quads);
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
