// Linear attention with one decay a head: the gradients.
//
// With dS the cotangent of the state that leaves a chunk (from what follows it), P_ij = e^{L_i - L_j} q_i.k_j and
// D_ij = e^{L_i - L_j} do_i.v_j for j <= i,
//       dq_i = sum_j D_ij k_j + e^{L_i} S do_i               u_i = e^{L_i} q_i.(S do_i)
//       dk_j = sum_i D_ij q_i + e^{L_C - L_j} dS v_j         w_j = e^{L_C - L_j} k_j.(dS v_j)
//       dv_j = sum_i P_ij do_i + e^{L_C - L_j} dS^T k_j
//       dS  <- e^{L_C} dS + sum_i e^{L_i} q_i do_i^T
// The gradient of a_t is the sum of what passes from before t to t or later: e^{L_C} <S, dS> over the chunk, w_j for j < t,
// u_i for i >= t, and P_ij (do_i.v_j) for j < t <= i, which is the sum over i >= t of that matrix's row sums less its column
// sums.  All of it is the chunk's own, so no difference runs over a whole sequence: that takes the state before every chunk,
// which the forward pass leaves in 32 bits.
#include "gla_decay.hpp"

namespace gla {
namespace {

struct BackwardArgs {
    DecaySizes n;
    DecayPlan plan;
    DecayRows gates, keys, values, queries, dout;
    const int32_t *lengths;
    const float *kept;                           // states before the chunks
    const void *dhidden_final;
    int hidden_dtype;
    const float *entering;
    void *dhidden_init;
    // results: in their own type, or (more than one part) floats [part][...]
    void *dvalue, *dkey, *dquery;
    float *dgate;                                // [part][B,T,H], or NULL
    double *dgate_sums;                          // [part][H][B][segments] where the gates are one constant a head, or NULL
    int row_parts, value_parts;                  // of dquery and dkey; of dvalue
};

// Results, at the first row of the chunk that is worked on.
struct Result {
    char *p;
    unsigned row;                                // bytes from one token to the next
    bool parts;                                  // floats, to be summed
    // four values of row 16t + r, 4c features behind the pointer
    template <typename V> __device__ __forceinline__ void put(int t, unsigned r, unsigned c, V v) const
    {
        *reinterpret_cast<V *>(at_bytes(p + (size_t)(16 * t * row), r * row + (unsigned)sizeof(V) * c)) = v;
    }
    template <typename T> __device__ __forceinline__ void put_as(int t, unsigned r, unsigned c, f32x4 v) const
    {
        if (parts) put(t, r, c, v);
        else put(t, r, c, pack_results<T>(v));
    }
};

// One workgroup: a segment of a (batch, head) pair, DKW key and DVW value features.  Its first waves make dq and dv: wave w of key
// features 16w .. 16w+15, with its columns of S, and of value features 16w .. 16w+15.  The others make dk and carry dS: its columns of
// key features lie in the accumulators with value features as rows, an operand of dk as they are; the first waves take dS from LDS, for
// <S, dS> and for dv, which contracts it over the other index, rounded to `T` as any operand of a 16-bit result.  (A second copy of dS by value columns cost 32
// registers and as many products as the first; all of it on 8 waves of twice the registers left a SIMD two waves, whose
// matrix, vector and LDS phases then followed each other: 135 us against 95 of 16 at B4 T4096 H6 D128.)
// S and dS enter what the gates' gradient is formed from in three parts, i.e. as the 32-bit numbers that they are.
//
// B4 T4096 H6 D128: 82 us for 288 MB (rows and states read once, gradients written), 3.5 TB/s; a compute unit holds one workgroup by its LDS, and
// 12 of a chunk's 21 thousand cycles are the last phase (dq and dv beside dk and dS), whose instructions alone issue in 8.
template <typename T, int DKW, int DVW>
__global__ __launch_bounds__(((DKW > DVW ? DKW : DVW) + DKW) * 4) void decay_gradient_kernel(const BackwardArgs a)
{
    constexpr int KT = DKW / 16, VT = DVW / 16, KK = DKW / 32, VK = DVW / 32, NA = KT > VT ? KT : VT, NW = NA + KT, NT = NW * 64;
    constexpr int C = DecayChunk<T>::C, CT = C / 16, CS = C / 32;
    typedef typename FragTypes<T>::d8 D8;
    typedef LdsTile<T, DKW> TileK;
    typedef LdsTile<T, DVW> TileV;
    typedef LdsTile<T, C> TileP;
    extern __shared__ char smem[];
    T *sQ = reinterpret_cast<T *>(smem), *sK = sQ + C * TileK::kRow, *sV = sK + C * TileK::kRow, *sO = sV + C * TileV::kRow,
      *sP = sO + C * TileV::kRow, *sD = sP + C * TileP::kRow;
    float *sS = reinterpret_cast<float *>(sD + C * TileP::kRow);
    ChunkGates<C> *gates = reinterpret_cast<ChunkGates<C> *>(sS + DKW * DVW);
    // what the gates' gradient is formed from, of a chunk and of the one before
    struct Sums {
        float row[CT][C];                        // row sums of one column of tiles
        float col[CT][C];                        // column sums of one row of tiles
        float u[KT][C], w[KT][C];
        float x[16];
    };
    Sums *sums = reinterpret_cast<Sums *>(gates + 2);
    double *sGate = reinterpret_cast<double *>(sums + 2);     // the gates' gradients so far, by token of the chunk

    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, r = lane & 15, c = lane >> 4;
    const unsigned H = (unsigned)a.n.H, pair = pair_of(blockIdx.x, a.n);
    const int64_t bh = pair, b = pair / H, h = pair % H, group = H / (unsigned)a.n.HK, hk = pair % H / (unsigned)group;
    const int DK = (int)a.n.DK, DV = (int)a.n.DV, vslabs = (DV + DVW - 1) / DVW;
    const int ks0 = blockIdx.y / vslabs, vs0 = blockIdx.y % vslabs, dk0 = ks0 * DKW, dv0 = vs0 * DVW;
    const int T_ = (int)a.n.T, len = a.lengths ? min(max(a.lengths[b], 0), T_) : T_;
    // from the segment in which the sequence ends down to the first; then those behind it, where only zeros are to be written
    const int order = blockIdx.z, tail = a.plan.tail((len + C - 1) / C),
              seg = tail - order + (order <= tail ? 0 : (int)a.plan.segments);
    const int first = a.plan.first(seg), last = a.plan.first(seg + 1), live = min(last, (len + C - 1) / C);
    const T *K = static_cast<const T *>(a.keys.p) + b * a.keys.sb + hk * a.keys.sh + dk0;
    const T *Q = static_cast<const T *>(a.queries.p) + b * a.queries.sb + hk * a.queries.sh + dk0;
    const T *V = static_cast<const T *>(a.values.p) + b * a.values.sb + h * a.values.sh + dv0;
    const T *O = static_cast<const T *>(a.dout.p) + b * a.dout.sb + h * a.dout.sh + dv0;
    const float *G = static_cast<const float *>(a.gates.p) + b * a.gates.sb + h * a.gates.sh;
    const bool second = w >= NA;                 // dk and dS, or else dq and dv
    const int wk = second ? w - NA : w;          // the wave's key features are 16 wk ..
    const bool has_keys = wk < KT, key_wave = has_keys && dk0 + 16 * wk < DK, value_wave = !second && w < VT && dv0 + 16 * w < DV;
    const TileK tk;
    const TileV tv;
    const TileP tp;

    // dq of the first waves or dk of the others, and dv
    auto result = [&](void *array, int parts, int64_t part, int64_t heads_features, int64_t at) {
        const unsigned size = parts > 1 ? 4 : sizeof(T);
        const int64_t row = (part * a.n.B + b) * a.n.T + (int64_t)(live - 1) * C;
        return Result{static_cast<char *>(array) + (row * heads_features + at) * size, (unsigned)heads_features * size, parts > 1};
    };
    Result qk = result(second ? a.dkey : a.dquery, a.row_parts, vs0 * group + h % group, a.n.HK * DK, hk * DK + dk0 + 16 * wk);
    Result dv = result(a.dvalue, a.value_parts, ks0, a.n.H * DV, h * DV + dv0 + 16 * w);
    const float *kept = a.kept + (((bh * a.plan.chunks + live - 1) * (DK / 16) + (key_wave ? dk0 / 16 + wk : 0)) * (DV / 16) + dv0 / 16) * 256;
    const int64_t kept_step = (int64_t)DK * DV;

    // ---- the cotangent that enters: key feature r of the wave's, value features 16t + 4c .. ----
    f32x4 state[VT];                             // dS, which stays; of the first waves S, a chunk's after the other
#pragma unroll
    for (int t = 0; t < VT; ++t) state[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (order == 0) {
#pragma unroll
        for (int t = 0; t < VT; ++t)
            if (second && key_wave && dv0 + 16 * t < DV) {
                float x[4];
                load_hidden<4>(a.dhidden_final, a.hidden_dtype, (bh * DK + dk0 + 16 * wk + r) * DV + dv0 + 16 * t + 4 * c, x);
                state[t] = f32x4{x[0], x[1], x[2], x[3]};
            }
    } else if (seg <= tail) {
        const int tiles = (int)decay_key_width(DK) / 16;
        const float *from = a.entering + ((bh * a.plan.segments + order - 1) * vslabs + vs0) * (int64_t)(tiles * 16 * DVW);
#pragma unroll
        for (int t = 0; t < VT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (second) state[t][e] = from[((t * tiles + dk0 / 16 + wk) * 64 + (r >> 2) * 16 + 4 * c + e) * 4 + (r & 3)];
    }

    RowsInFlight<T, C, DKW, NT> fk, fq;
    RowsInFlight<T, C, DVW, NT> fv, fo;
    const int k_st = (int)a.keys.st, q_st = (int)a.queries.st, v_st = (int)a.values.st, o_st = (int)a.dout.st;
    float g = 0.f;
    auto fetch_gates = [&](int n) {              // by the wave that makes the chunk's gates
        const int lane = again(tid) & 63;
        g = w == NW - 1 && lane < C && n * C + lane < len ? G[(int64_t)(n * C + lane) * a.gates.st] : 0.f;
    };
    auto fetch = [&](int n) {                    // the rows that the pointers have come to
        const int left = len - n * C;
        const unsigned at = fk.here();
        fk.load(at, K, k_st, left, DK - dk0);
        fq.load(at, Q, q_st, left, DK - dk0);
        fv.load(at, V, v_st, left, DV - dv0);
        fo.load(at, O, o_st, left, DV - dv0);
        K -= (int64_t)C * k_st;
        Q -= (int64_t)C * q_st;
        V -= (int64_t)C * v_st;
        O -= (int64_t)C * o_st;
    };

    if (tid < 64) sGate[tid] = 0.0;
    // The gates' gradient of chunk n, by one wave, from the sums that the others left.
    auto gates_gradient = [&](int n, const Sums &s) {
        const int lane = (int)again(tid) & 63;
        float u = 0.f, ww = 0.f;
        if (lane < C) {
#pragma unroll
            for (int i = 0; i < KT; ++i) { u += s.u[i][lane]; ww += s.w[i][lane]; }
#pragma unroll
            for (int i = 0; i < CT; ++i) {
                u += i <= lane / 16 ? s.row[i][lane] : 0.f;
                u -= i >= lane / 16 ? s.col[i][lane] : 0.f;
            }
        }
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < KT; ++i) x += s.x[i];
        float before = __shfl_up(ww, 1, 64);
        if (lane == 0) before = 0.f;
#pragma unroll
        for (int by = 1; by < C; by *= 2) {
            const float lower = __shfl_up(before, by, 64), upper = __shfl_down(u, by, 64);
            if (lane >= by) before += lower;
            if (lane + by < 64) u += upper;
        }
        const int t = n * C + lane;
        const float d = t < len ? x + before + u : 0.f;
        if (lane < C && t < T_) {
            if (a.dgate) a.dgate[((blockIdx.y * a.n.B + b) * a.n.T + t) * a.n.H + h] = d;
            sGate[lane] += d;
        }
    };

    for (int i = tid; i < C * TileP::kRow; i += NT) sP[i] = sD[i] = (T)0.f;      // the tiles above the diagonal that products take along
    // key feature r of the wave's, value features 16 t + 4c .. of the state that `from` points at (or others, where these do not exist)
    auto state_tile = [&](const float *from, int t) {
        return *reinterpret_cast<const f32x4 *>(at_bytes(from + (16 * t < DV - dv0 ? 256 * t : 0), (again(tid) & 63) * 16));
    };
    // dS in LDS, tiles of 16 key and 16 value features as the waves hold them.  The places of 16 lanes are permuted by the lanes' row, so that
    // reads along key features, too, have no two lanes at a bank.
    auto dS_tile = [&](int tk, int t) {
        const unsigned lane = again(tid) & 63, c = lane >> 4;
        return sS + (tk * VT + t) * 256 + (lane ^ c) * 4;
    };
    // key features 32 ks + 4c .. and 32 ks + 16 + 4c .. of value feature 16 t + r
    auto dS_columns = [&](int ks, int t, float (&x)[8]) {
        const unsigned lane = again(tid) & 63, r = lane & 15, c = lane >> 4, row = r >> 2;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = sS[((2 * ks + e / 4) * VT + t) * 256 + (16 * row + 4 * c + ((e & 3) ^ row)) * 4 + (r & 3)];
    };
    const int sums_wave = NW - 2;
    const int count = max(live - first, 0);
    int n = live - 1;
    if (count > 0) {
        K += (int64_t)n * C * a.keys.st;
        Q += (int64_t)n * C * a.queries.st;
        V += (int64_t)n * C * a.values.st;
        O += (int64_t)n * C * a.dout.st;
        fetch_gates(n);
        fetch(n);
        if (!second) {
#pragma unroll
            for (int t = 0; t < VT; ++t) state[t] = state_tile(kept, t);
        }
        if (w == NW - 1) chunk_gates<C>(gates[0], g);
        if (count > 1) fetch_gates(n - 1);
    }
    for (int i = 0; i < count; ++i, --n) {
        const ChunkGates<C> &gate = gates[i & 1];
        Sums &sum = sums[i & 1];
        lds_barrier();                            // the last chunk's tiles are read, its sums written
        const unsigned at = fk.here();
        fk.store(at, sK, len - n * C, DK - dk0);
        fq.store(at, sQ, len - n * C, DK - dk0);
        fv.store(at, sV, len - n * C, DV - dv0);
        fo.store(at, sO, len - n * C, DV - dv0);
        if (second) {                             // dS for the first waves
            float *p = dS_tile(wk, 0);
#pragma unroll
            for (int t = 0; t < VT; ++t) *reinterpret_cast<f32x4 *>(p + t * 256) = state[t];
        }
        lds_barrier();
        const float whole = gate.whole;
        if (!second && has_keys) {                // <S, dS>
            float x = 0.f;
            const float *p = dS_tile(w, 0);
#pragma unroll
            for (int t = 0; t < VT; ++t) {
                const f32x4 d = *reinterpret_cast<const f32x4 *>(p + t * 256);
#pragma unroll
                for (int e = 0; e < 4; ++e) x += d[e] * state[t][e];         // (where S is another's, dS is zero)
            }
            x = sum_over_c(sum_over_r(x));
            if (lane == 0) sum.x[wk] = whole * x;
        }
        if (i + 1 < count) fetch(n - 1);

        // ---- scores, transposed: lane (r, c) has keys 4c .. 4c+3 of tile tj for query r of tile ti ----
        {
            const TileK LK = tk.here();
            const TileV LV = tv.here();
            const TileP LP = tp.here();
            // (a lane's place formed again in every phase: spilled, it would be read behind the rows that are on their way)
            const int r = again(tid) & 15, c = (again(tid) >> 4) & 3;
#pragma unroll 1
            for (int n16 = w; n16 < CT * (CT + 1) / 2; n16 += NW) {
                int ti, tj;
                triangle(n16, ti, tj);
                f32x4 s = {0.f, 0.f, 0.f, 0.f}, d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < KK; ++ks) s = mma_d(LK.rows(sK, tj, ks), LK.rows(sQ, ti, ks), s);
#pragma unroll
                for (int ks = 0; ks < VK; ++ks) d = mma_d(LV.rows(sV, tj, ks), LV.rows(sO, ti, ks), d);
                const int qi = 16 * ti + r, kj = 16 * tj + 4 * c;
                const float at = gate.sum[qi], at_rest = gate.rest[qi];
                const f32x4 to = *reinterpret_cast<const f32x4 *>(gate.sum + kj), to_rest = *reinterpret_cast<const f32x4 *>(gate.rest + kj);
                float p[4], dd[4], row = 0.f, col[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float weight = ChunkGates<C>::weight(at, at_rest, to[e], to_rest[e]);
                    p[e] = s[e] * weight;
                    dd[e] = d[e] * weight;
                    col[e] = p[e] * d[e];
                }
                if (ti == tj)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!(kj + e <= qi)) p[e] = dd[e] = col[e] = 0.f;
                row = (col[0] + col[1]) + (col[2] + col[3]);
                store_vec<T, 4>(LP.four(sP, ti, tj), p);
                store_vec<T, 4>(LP.four(sD, ti, tj), dd);
                row = sum_over_c(row);
                if (c == 0) sum.row[tj][qi] = row;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    col[e] = sum_over_r(col[e]);
                }
                if (r == 0) store_vec<float, 4>(sum.col[ti] + kj, col);
            }
        }
        // beside the scores, by waves that have a tile less than the first ones or none: the last chunk's gradient of the gates, and
        // the next chunk's gates
        if (w == sums_wave && i > 0) gates_gradient(n + 1, sums[(i + 1) & 1]);
        if (w == NW - 1 && i + 1 < count) {
            chunk_gates<C>(gates[(i + 1) & 1], g);
            if (i + 2 < count) fetch_gates(n - 2);
        }
        lds_barrier();

        const unsigned row = again(tid) & 15, col = (again(tid) >> 4) & 3;
        const int left = T_ - n * C - (int)row;      // rows 16 t that exist
        f32x4 o[CT];
#pragma unroll
        for (int ti = 0; ti < CT; ++ti) o[ti] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (!second && has_keys) {
            // ---- dq ----
            {
                const TileV LV = tv.here();
                const float *next = i + 1 < count ? kept - kept_step : kept;
#pragma unroll
                for (int ks = 0; ks < VK; ++ks) {
                    float s[8];
                    two_tiles(state[2 * ks], state[2 * ks + 1], s);
                    const Split<T, 3> op(s);
                    // the next chunk's, as soon as these are used
                    state[2 * ks] = state_tile(next, 2 * ks);
                    state[2 * ks + 1] = state_tile(next, 2 * ks + 1);
#pragma unroll
                    for (int ti = 0; ti < CT; ti += 2) {
                        const D8 x[2] = {LV.halves(sO, ti, ks), LV.halves(sO, ti + 1, ks)};
                        mma_left(op, x, o + ti);
                    }
                    __builtin_amdgcn_sched_barrier(0);      // a step's operands at a time
                }
            }
            const TileK LK = tk.here();
            const TileP LP = tp.here();
            D8 kc[CS];
#pragma unroll
            for (int ks = 0; ks < CS; ++ks) kc[ks] = LK.columns(sK, ks, w);
            wait_for_memory();
#pragma unroll
            for (int ti = 0; ti < CT; ++ti) {
                const float scale = gate.from_start[16 * ti + row];
                float qv[4], u = 0.f;
                load_vec<T, 4>(LK.four(sQ, ti, w), qv);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    o[ti][e] *= scale;
                    u += qv[e] * o[ti][e];
                }
                u = sum_over_c(u);
                if (col == 0) sum.u[w][16 * ti + row] = u;
#pragma unroll
                for (int ks = 0; ks <= ti / 2; ++ks) o[ti] = mma_d(kc[ks], LP.halves(sD, ti, ks), o[ti]);
                if (key_wave && 16 * ti < left) qk.put_as<T>(ti, row, col, o[ti]);
                o[ti] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
        }
        if (second) {
            // ---- dk ----
            {
                const TileV LV = tv.here();
#pragma unroll
                for (int ks = 0; ks < VK; ++ks) {
                    float s[8];
                    two_tiles(state[2 * ks], state[2 * ks + 1], s);
                    const Split<T, 3> op(s);
#pragma unroll
                    for (int tj = 0; tj < CT; tj += 2) {
                        const D8 x[2] = {LV.halves(sV, tj, ks), LV.halves(sV, tj + 1, ks)};
                        mma_left(op, x, o + tj);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            const TileK LK = tk.here();
            D8 qc[CS];
#pragma unroll
            for (int ks = 0; ks < CS; ++ks) qc[ks] = LK.columns(sQ, ks, wk);
            wait_for_memory();
            {
                const TileP LP = tp.here();
#pragma unroll
                for (int tj = 0; tj < CT; ++tj) {
                    const float scale = gate.to_end[16 * tj + row];
                    float kv[4], ww = 0.f;
                    load_vec<T, 4>(LK.four(sK, tj, wk), kv);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        o[tj][e] *= scale;
                        ww += kv[e] * o[tj][e];
                    }
                    ww = sum_over_c(ww);
                    if (col == 0) sum.w[wk][16 * tj + row] = ww;
#pragma unroll
                    for (int ks = tj / 2; ks < CS; ++ks) o[tj] = mma_d(qc[ks], LP.columns(sD, ks, tj), o[tj]);
                    if (key_wave && 16 * tj < left) qk.put_as<T>(tj, row, col, o[tj]);
                }
            }
            // ---- dS: dhidden_init and the gates' gradient come from it ----
            const TileV LV = tv.here();
#pragma unroll
            for (int t = 0; t < VT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) state[t][e] *= whole;
#pragma unroll
            for (int ks = 0; ks < CS; ++ks) {
                float v[8], by[8];
                unpack8(qc[ks], v);
                two_tiles(*reinterpret_cast<const f32x4 *>(gate.from_start + 32 * ks + 4 * col),
                          *reinterpret_cast<const f32x4 *>(gate.from_start + 32 * ks + 16 + 4 * col), by);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] *= by[e];
                const Split<T, 3> op(v);
#pragma unroll
                for (int t = 0; t < VT; t += 2) {
                    const D8 x[2] = {LV.columns(sO, ks, t), LV.columns(sO, ks, t + 1)};
                    mma_right(x, op, state + t);
                    if (t % 4 == 2) __builtin_amdgcn_sched_barrier(0);
                }
            }
        } else if (w < VT) {
            // ---- dv ----
            const TileV LV = tv.here();
            const TileK LK = tk.here();
#pragma unroll
            for (int ks = 0; ks < KK; ++ks) {
                float d[8];
                dS_columns(ks, w, d);
                const D8 op = Split<T, 1>(d).part[0];
#pragma unroll
                for (int tj = 0; tj < CT; ++tj) o[tj] = mma_d(op, LK.halves(sK, tj, ks), o[tj]);
            }
            const TileP LP = tp.here();
            D8 oc[CS];
#pragma unroll
            for (int ks = 0; ks < CS; ++ks) oc[ks] = LV.columns(sO, ks, w);
#pragma unroll
            for (int tj = 0; tj < CT; ++tj) {
                const float scale = gate.to_end[16 * tj + row];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[tj][e] *= scale;
#pragma unroll
                for (int ks = tj / 2; ks < CS; ++ks) o[tj] = mma_d(oc[ks], LP.columns(sP, ks, tj), o[tj]);
                if (value_wave && 16 * tj < left) dv.put_as<T>(tj, row, col, o[tj]);
            }
        }
        qk.p -= (int64_t)C * qk.row;
        dv.p -= (int64_t)C * dv.row;
        kept -= kept_step;
    }
    lds_barrier();
    if (w == sums_wave) {
        if (count > 0) gates_gradient(first, sums[(count - 1) & 1]);
        if (a.dgate_sums) {
            double x = sGate[lane];
#pragma unroll
            for (int m = 1; m < 64; m *= 2) x += __hiloint2double(__shfl_xor(__double2hiint(x), m, 64), __shfl_xor(__double2loint(x), m, 64));
            if (lane == 0) a.dgate_sums[((blockIdx.y * a.n.H + h) * a.n.B + b) * a.plan.segments + order] = x;
        }
    }
    // rows past the end of a shorter sequence, each wave its features
    if (live < last) {
        const int from = max(live, first);
        qk.p += (int64_t)(from - live + 1 + count) * C * qk.row;
        dv.p += (int64_t)(from - live + 1 + count) * C * dv.row;
        for (int m = from; m < last; ++m) {
            const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = 0; t < CT; ++t) {
                const bool there = m * C + 16 * t + r < T_;
                if (key_wave && there) qk.put_as<T>(t, r, c, zero);
                if (value_wave && there) dv.put_as<T>(t, r, c, zero);
            }
            if (a.dgate && w == 0 && lane < C && m * C + lane < T_)
                a.dgate[((blockIdx.y * a.n.B + b) * a.n.T + m * C + lane) * a.n.H + h] = 0.f;
            qk.p += (int64_t)C * qk.row;
            dv.p += (int64_t)C * dv.row;
        }
    }
    if (seg == 0) {
#pragma unroll
        for (int t = 0; t < VT; ++t)
            if (second && key_wave && dv0 + 16 * t < DV) {
                const float x[4] = {state[t][0], state[t][1], state[t][2], state[t][3]};
                store_hidden<4>(a.dhidden_init, a.hidden_dtype, (bh * DK + dk0 + 16 * wk + r) * DV + dv0 + 16 * t + 4 * c, x);
            }
    }
}

// An array as the sum of `parts` arrays of n floats behind each other, rounded once; all of a call's in one launch.
struct PartSum {
    const float *src;
    void *dst;
    int64_t n;
    int parts;
    bool floats;                                 // dst is float, else T
};
struct PartSums {
    PartSum of[4];
    int count;
};
template <typename T> __device__ void sum_parts_of(const float *__restrict__ src, int parts, int64_t n, T *__restrict__ dst)
{
    // Rows come in multiples of 16 features, so their parts all begin on 16 bytes; those of dlog_decay, B T H floats each, need not.
    const bool fours = n % 4 == 0;
    for (int64_t i = 4 * (blockIdx.x * (int64_t)256 + threadIdx.x); i < n; i += 1024 * (int64_t)gridDim.x) {
        if (fours) {
            float s[4] = {0.f, 0.f, 0.f, 0.f}, x[4];
            for (int p = 0; p < parts; ++p) {
                load_vec<float, 4>(src + p * n + i, x);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[e] += x[e];
            }
            store_vec<T, 4>(dst + i, s);
        } else {
            for (int64_t j = i; j < min(i + 4, n); ++j) {
                float s = 0.f;
                for (int p = 0; p < parts; ++p) s += src[p * n + j];
                Elem<T>::store(dst + j, s);
            }
        }
    }
}
template <typename T> __global__ __launch_bounds__(256) void decay_sum_parts_kernel(const PartSums a)
{
    const PartSum &s = a.of[blockIdx.y];
    if (s.floats) sum_parts_of(s.src, s.parts, s.n, static_cast<float *>(s.dst));
    else sum_parts_of(s.src, s.parts, s.n, static_cast<T *>(s.dst));
}

// The gradient of one constant a head: the sum over parts, batch and segments, by one wave a head.
__global__ __launch_bounds__(64) void decay_sum_gates_kernel(const double *__restrict__ sums, int parts, int64_t H, int64_t n, float *__restrict__ dst)
{
    const int64_t h = blockIdx.x;
    double x = 0.0;
    for (int p = 0; p < parts; ++p)
        for (int64_t i = threadIdx.x; i < n; i += 64) x += sums[(p * H + h) * n + i];
#pragma unroll
    for (int m = 1; m < 64; m *= 2) x += __hiloint2double(__shfl_xor(__double2hiint(x), m, 64), __shfl_xor(__double2loint(x), m, 64));
    if (threadIdx.x == 0) dst[h] = (float)x;
}

template <typename T, int DKW, int DVW> int launch_gradient(hipStream_t stream, const BackwardArgs &a)
{
    static LdsGrant grant;
    constexpr int C = DecayChunk<T>::C, CT = C / 16, KT = DKW / 16;
    constexpr size_t lds = sizeof(T) * (2 * C * LdsTile<T, DKW>::kRow + 2 * C * LdsTile<T, DVW>::kRow + 2 * C * LdsTile<T, C>::kRow) +
                           sizeof(float) * DKW * DVW +
                           2 * sizeof(ChunkGates<C>) + sizeof(float) * 2 * (2 * CT * C + 2 * KT * C + 16) + sizeof(double) * 64;
    static_assert(lds <= 160 * 1024, "");
    if (int e = allow_lds(grant, reinterpret_cast<const void *>(decay_gradient_kernel<T, DKW, DVW>), lds)) return e;
    const dim3 grid(a.n.B * a.n.H, ((a.n.DK + DKW - 1) / DKW) * ((a.n.DV + DVW - 1) / DVW), a.plan.segments);
    decay_gradient_kernel<T, DKW, DVW><<<grid, ((DKW > DVW ? DKW : DVW) + DKW) * 4, lds, stream>>>(a);
    return launch_status();
}
template <typename T> int dispatch_gradient(hipStream_t stream, const BackwardArgs &a)
{
    if (a.n.DK <= 64) return a.n.DV <= 64 ? launch_gradient<T, 64, 64>(stream, a) : launch_gradient<T, 64, 128>(stream, a);
    return a.n.DV <= 64 ? launch_gradient<T, 128, 64>(stream, a) : launch_gradient<T, 128, 128>(stream, a);
}

}  // namespace

int decay_backward(void *stream, const DecaySizes &n, const DecayPlan &plan, gla_dtype dtype, gla_dtype hidden_dtype,
                   const DecayRows &gates, const DecayRows &keys, const DecayRows &values, const DecayRows &queries,
                   const DecayRows &dout, const int32_t *lengths, const float *kept, const void *dhidden_final, bool constant_gates,
                   void *dhidden_init, float *dlog_decay, void *dvalue, void *dkey, void *dquery, float *entering, float *decays,
                   const DecayParts &parts)
{
    int e = decay_entering_states(stream, true, n, plan, dtype, hidden_dtype, dhidden_final, gates, queries, dout,
                                  lengths, entering, decays);
    if (e) return e;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    BackwardArgs a{};
    a.n = n;
    a.plan = plan;
    a.gates = gates;
    a.keys = keys;
    a.values = values;
    a.queries = queries;
    a.dout = dout;
    a.lengths = lengths;
    a.kept = kept;
    a.dhidden_final = dhidden_final;
    a.hidden_dtype = hidden_dtype;
    a.entering = entering;
    a.dhidden_init = dhidden_init;
    a.row_parts = parts.rows;
    a.value_parts = parts.values;
    a.dquery = parts.rows > 1 ? parts.dquery : dquery;
    a.dkey = parts.rows > 1 ? parts.dkey : dkey;
    a.dvalue = parts.values > 1 ? parts.dvalue : dvalue;
    a.dgate = constant_gates ? nullptr : parts.gates > 1 ? parts.dgate : dlog_decay;
    a.dgate_sums = constant_gates ? parts.gate_sums : nullptr;
    e = dtype == GLA_BF16 ? dispatch_gradient<__bf16>(s, a) : dispatch_gradient<float>(s, a);
    const int64_t nk = n.B * n.T * n.HK * n.DK, nv = n.B * n.T * n.H * n.DV;
    PartSums sums{};
    int64_t most = 0;
    auto sum = [&](const float *src, int count, int64_t m, void *dst, bool floats) {
        if (count < 2 || m < 1) return;
        sums.of[sums.count++] = PartSum{src, dst, m, count, floats};
        most = most < m ? m : most;
    };
    sum(parts.dquery, parts.rows, nk, dquery, false);
    sum(parts.dkey, parts.rows, nk, dkey, false);
    sum(parts.dvalue, parts.values, nv, dvalue, false);
    if (!constant_gates) sum(parts.dgate, parts.gates, n.B * n.T * n.H, dlog_decay, true);
    if (!e && sums.count) {
        const int64_t blocks = (most + 1023) / 1024;
        const dim3 grid((unsigned)(blocks < 4096 ? blocks : 4096), sums.count);
        if (dtype == GLA_BF16) decay_sum_parts_kernel<__bf16><<<grid, 256, 0, s>>>(sums);
        else decay_sum_parts_kernel<float><<<grid, 256, 0, s>>>(sums);
        e = launch_status();
    }
    if (!e && constant_gates) {
        decay_sum_gates_kernel<<<n.H, 64, 0, s>>>(parts.gate_sums, parts.gates, n.H, n.B * plan.segments, dlog_decay);
        e = launch_status();
    }
    return e;
}

}  // namespace gla
