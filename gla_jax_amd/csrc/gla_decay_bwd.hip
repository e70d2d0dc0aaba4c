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

// One workgroup: a segment of a (batch, head) pair, DKW key and DVW value features.  Wave w owns key features 16w .. 16w+15
// for dq, dk and value features 16w .. 16w+15 for dv; dS is held twice, since it is contracted over either index: `by_value`
// has the wave's value columns with key rows, `by_key` the wave's key columns with value rows, each an operand as it lies.
// S and dS enter what the gates' gradient is formed from in three parts, i.e. as the 32-bit numbers that they are.
template <typename T, int DKW, int DVW>
__global__ __launch_bounds__((DKW > DVW ? DKW : DVW) * 4) void decay_gradient_kernel(const BackwardArgs a)
{
    constexpr int NW = (DKW > DVW ? DKW : DVW) / 16, NT = NW * 64, KT = DKW / 16, VT = DVW / 16, KK = DKW / 32, VK = DVW / 32;
    constexpr int C = DecayChunk<T>::C, CT = C / 16, CS = C / 32;
    constexpr int SK = lds_stride<T>(DKW), SV = lds_stride<T>(DVW), SP = lds_stride<T>(C);
    typedef typename FragTypes<T>::d8 D8;
    extern __shared__ char smem[];
    T *sQ = reinterpret_cast<T *>(smem), *sK = sQ + C * SK, *sV = sK + C * SK, *sO = sV + C * SV, *sP = sO + C * SV,
      *sD = sP + C * SP;
    ChunkGates<C> &gate = *reinterpret_cast<ChunkGates<C> *>(reinterpret_cast<char *>(sD + C * SP));
    float *sRow = reinterpret_cast<float *>(&gate + 1);       // [CT][C] row sums of one column of tiles
    float *sCol = sRow + CT * C;                              // [CT][C] column sums of one row of tiles
    float *sU = sCol + CT * C, *sW = sU + KT * C, *sX = sW + KT * C;

    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, r = lane & 15, c = lane >> 4;
    const int64_t bh = blockIdx.x, b = bh / a.n.H, h = bh % a.n.H, group = a.n.H / a.n.HK, hk = h / group;
    const int DK = (int)a.n.DK, DV = (int)a.n.DV, vslabs = (DV + DVW - 1) / DVW;
    const int ks0 = blockIdx.y / vslabs, vs0 = blockIdx.y % vslabs, dk0 = ks0 * DKW, dv0 = vs0 * DVW;
    const int64_t order = blockIdx.z, seg = a.plan.segments - 1 - order;
    const int64_t len = a.lengths ? min(max((int64_t)a.lengths[b], (int64_t)0), a.n.T) : a.n.T;
    const int64_t first = seg * a.plan.per, last = min(first + a.plan.per, a.plan.chunks), live = min(last, (len + C - 1) / C);
    const T *K = static_cast<const T *>(a.keys.p) + b * a.keys.sb + hk * a.keys.sh + dk0;
    const T *Q = static_cast<const T *>(a.queries.p) + b * a.queries.sb + hk * a.queries.sh + dk0;
    const T *V = static_cast<const T *>(a.values.p) + b * a.values.sb + h * a.values.sh + dv0;
    const T *O = static_cast<const T *>(a.dout.p) + b * a.dout.sb + h * a.dout.sh + dv0;
    const float *G = static_cast<const float *>(a.gates.p) + b * a.gates.sb + h * a.gates.sh;
    const bool key_wave = w < KT && dk0 + 16 * w < DK, value_wave = w < VT && dv0 + 16 * w < DV;
    const DecayLane<T> LK(SK), LV(SV), LP(SP);
    const int64_t part_qk = vs0 * group + h % group;
    const int64_t row_qk = hk * DK + dk0 + 16 * w + 4 * c, rows_qk = a.n.HK * DK;       // within a token's row
    const int64_t row_v = h * DV + dv0 + 16 * w + 4 * c, rows_v = a.n.H * DV;

    auto put = [&](void *to, bool parts, int64_t part, int64_t t, int64_t width, int64_t at, const float (&x)[4]) {
        const int64_t i = (b * a.n.T + t) * width + at;
        if (parts) store_vec<float, 4>(static_cast<float *>(to) + part * a.n.B * a.n.T * width + i, x);
        else store_vec<T, 4>(static_cast<T *>(to) + i, x);
    };

    // ---- the cotangent that enters, in both forms ----
    f32x4 by_value[KT], by_key[VT];
#pragma unroll
    for (int t = 0; t < KT; ++t) by_value[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < VT; ++t) by_key[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (order == 0) {
        const int64_t base = bh * DK * DV;
#pragma unroll
        for (int t = 0; t < KT; ++t)
            if (value_wave && dk0 + 16 * t < DK) {
                float x[4];
                load_hidden<4>(a.dhidden_final, a.hidden_dtype,
                               base + (int64_t)(dk0 + 16 * t + 4 * c + (r & 3)) * DV + dv0 + 16 * w + (r & ~3), x);
                quad_transpose(x);
                by_value[t] = f32x4{x[0], x[1], x[2], x[3]};
            }
#pragma unroll
        for (int t = 0; t < VT; ++t)
            if (key_wave && dv0 + 16 * t < DV) {
                float x[4];
                load_hidden<4>(a.dhidden_final, a.hidden_dtype, base + (int64_t)(dk0 + 16 * w + r) * DV + dv0 + 16 * t + 4 * c, x);
                by_key[t] = f32x4{x[0], x[1], x[2], x[3]};
            }
    } else {
        const int tiles = (int)decay_key_width(DK) / 16;
        const float *from = a.entering + ((bh * a.plan.segments + order - 1) * vslabs + vs0) * (int64_t)(tiles * 16 * DVW);
#pragma unroll
        for (int t = 0; t < KT; ++t)
            if (w < VT) by_value[t] = reinterpret_cast<const f32x4 *>(from)[(w * tiles + dk0 / 16 + t) * 64 + lane];
#pragma unroll
        for (int t = 0; t < VT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (w < KT) by_key[t][e] = from[((t * tiles + dk0 / 16 + w) * 64 + (r >> 2) * 16 + 4 * c + e) * 4 + (r & 3)];
    }

    RowsInFlight<T, C, DKW, NT> fk, fq;
    RowsInFlight<T, C, DVW, NT> fv, fo;
    float g = 0.f;
    auto fetch = [&](int64_t n) {
        fk.load(K, a.keys.st, n * C, len, DK - dk0);
        fq.load(Q, a.queries.st, n * C, len, DK - dk0);
        fv.load(V, a.values.st, n * C, len, DV - dv0);
        fo.load(O, a.dout.st, n * C, len, DV - dv0);
        g = w == 0 && lane < C && n * C + lane < len ? G[(n * C + lane) * a.gates.st] : 0.f;
    };

    double gate_sum = 0.0;
    // The gates' gradient of chunk n, by one wave, from the sums that the others left.
    auto gates_gradient = [&](int64_t n) {
        float u = 0.f, ww = 0.f;
        if (lane < C) {
#pragma unroll
            for (int i = 0; i < KT; ++i) { u += sU[i * C + lane]; ww += sW[i * C + lane]; }
            for (int i = 0; i <= lane / 16; ++i) u += sRow[i * C + lane];
            for (int i = lane / 16; i < CT; ++i) u -= sCol[i * C + lane];
        }
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < KT; ++i) x += sX[i];
        float before = __shfl_up(ww, 1, 64);
        if (lane == 0) before = 0.f;
#pragma unroll
        for (int by = 1; by < C; by *= 2) {
            const float lower = __shfl_up(before, by, 64), upper = __shfl_down(u, by, 64);
            if (lane >= by) before += lower;
            if (lane + by < 64) u += upper;
        }
        const int64_t t = n * C + lane;
        const float d = t < len ? x + before + u : 0.f;
        if (lane < C && t < a.n.T) {
            if (a.dgate) a.dgate[(((int64_t)blockIdx.y * a.n.B + b) * a.n.T + t) * a.n.H + h] = d;
            gate_sum += d;
        }
    };

    for (int i = tid; i < C * SP; i += NT) sP[i] = sD[i] = (T)0.f;      // the tiles above the diagonal that products take along
    const int gates_wave = NW - 1;
    const int64_t count = max(live - first, (int64_t)0);
    if (count > 0) fetch(live - 1);
    for (int64_t i = 0; i < count; ++i) {
        const int64_t n = live - 1 - i;
        lds_barrier();                            // the last chunk's tiles are read, its sums written
        fk.store(sK, SK);
        fq.store(sQ, SK);
        fv.store(sV, SV);
        fo.store(sO, SV);
        if (w == 0) chunk_gates<C>(gate, g);
        if (w == gates_wave && i > 0) gates_gradient(n + 1);
        lds_barrier();
        // the state before the chunk: key feature r of the wave's, value features in halves
        f32x4 S[VT];
#pragma unroll
        for (int t = 0; t < VT; ++t) {
            S[t] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (key_wave && dv0 + 16 * t < DV)
                S[t] = *reinterpret_cast<const f32x4 *>(a.kept + ((bh * a.plan.chunks + n) * DK + dk0 + 16 * w + r) * DV + dv0 +
                                                        16 * t + 4 * c);
        }
        if (i + 1 < count) fetch(n - 1);

        // ---- scores, transposed: lane (r, c) has keys 4c .. 4c+3 of tile tj for query r of tile ti ----
        for (int n16 = w; n16 < CT * (CT + 1) / 2; n16 += NW) {
            int ti, tj;
            triangle(n16, ti, tj);
            f32x4 s = {0.f, 0.f, 0.f, 0.f}, d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KK; ++ks)
                s = mma_d(ld8(sK + 16 * tj * SK + LK.row + 32 * ks), ld8(sQ + 16 * ti * SK + LK.row + 32 * ks), s);
#pragma unroll
            for (int ks = 0; ks < VK; ++ks)
                d = mma_d(ld8(sV + 16 * tj * SV + LV.row + 32 * ks), ld8(sO + 16 * ti * SV + LV.row + 32 * ks), d);
            const int qi = 16 * ti + r, kj = 16 * tj + 4 * c;
            const double at = gate.sum[qi];
            float p[4], dd[4], row = 0.f, col[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float weight = fast_exp2((float)(at - gate.sum[kj + e]));
                p[e] = kj + e <= qi ? s[e] * weight : 0.f;
                dd[e] = kj + e <= qi ? d[e] * weight : 0.f;
                col[e] = p[e] * d[e];
                if (!(kj + e <= qi)) col[e] = 0.f;
                row += col[e];
            }
            store_vec<T, 4>(sP + qi * SP + kj, p);
            store_vec<T, 4>(sD + qi * SP + kj, dd);
            row = reduce_over_cgroups(row);
            if (c == 0) sRow[tj * C + qi] = row;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x = col[e];
                x += dpp_f32<kDppQuadXor1>(x);
                x += dpp_f32<kDppQuadXor2>(x);
                x += dpp_f32<kDppRowHalfMirror>(x);
                x += dpp_f32<kDppRowMirror>(x);
                if (r == 0) sCol[ti * C + kj + e] = x;
            }
        }
        lds_barrier();

        const float whole = gate.whole;
        D8 qc[CS], kc[CS];
        if (w < KT) {
#pragma unroll
            for (int ks = 0; ks < CS; ++ks) {
                qc[ks] = lds_columns(sQ + 32 * ks * SK + 16 * w + LK.col, SK);
                kc[ks] = lds_columns(sK + 32 * ks * SK + 16 * w + LK.col, SK);
            }
            f32x4 o[CT];
            // ---- dq ----
            float x = 0.f;
#pragma unroll
            for (int t = 0; t < VT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) x += S[t][e] * by_key[t][e];
#pragma unroll
            for (int m = 1; m < 64; m *= 2) x += shfl_xor_f32(x, m);
            if (lane == 0) sX[w] = whole * x;
#pragma unroll
            for (int ti = 0; ti < CT; ++ti) o[ti] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < VK; ++ks) {
                float s[8];
                two_tiles(S[2 * ks], S[2 * ks + 1], s);
                const Split<T, 3> op(s);
#pragma unroll
                for (int ti = 0; ti < CT; ++ti) o[ti] = op.left(lds_two_halves(sO + 16 * ti * SV + LV.row2 + 32 * ks), o[ti]);
            }
#pragma unroll
            for (int ti = 0; ti < CT; ++ti) {
                const float scale = gate.from_start[16 * ti + r];
                float qv[4], u = 0.f;
                load_vec<T, 4>(sQ + (16 * ti + r) * SK + 16 * w + 4 * c, qv);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    o[ti][e] *= scale;
                    u += qv[e] * o[ti][e];
                }
                u = reduce_over_cgroups(u);
                if (c == 0) sU[w * C + 16 * ti + r] = u;
#pragma unroll
                for (int ks = 0; ks <= ti / 2; ++ks) o[ti] = mma_d(kc[ks], ld8(sD + 16 * ti * SP + LP.row + 32 * ks), o[ti]);
                const int64_t t = n * C + 16 * ti + r;
                const float v[4] = {o[ti][0], o[ti][1], o[ti][2], o[ti][3]};
                if (key_wave && t < a.n.T) put(a.dquery, a.row_parts > 1, part_qk, t, rows_qk, row_qk, v);
            }
            // ---- dk ----
#pragma unroll
            for (int tj = 0; tj < CT; ++tj) o[tj] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < VK; ++ks) {
                float s[8];
                two_tiles(by_key[2 * ks], by_key[2 * ks + 1], s);
                const Split<T, 3> op(s);
#pragma unroll
                for (int tj = 0; tj < CT; ++tj) o[tj] = op.left(lds_two_halves(sV + 16 * tj * SV + LV.row2 + 32 * ks), o[tj]);
            }
#pragma unroll
            for (int tj = 0; tj < CT; ++tj) {
                const float scale = gate.to_end[16 * tj + r];
                float kv[4], ww = 0.f;
                load_vec<T, 4>(sK + (16 * tj + r) * SK + 16 * w + 4 * c, kv);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    o[tj][e] *= scale;
                    ww += kv[e] * o[tj][e];
                }
                ww = reduce_over_cgroups(ww);
                if (c == 0) sW[w * C + 16 * tj + r] = ww;
#pragma unroll
                for (int ks = tj / 2; ks < CS; ++ks) o[tj] = mma_d(qc[ks], lds_columns(sD + 32 * ks * SP + 16 * tj + LP.col, SP), o[tj]);
                const int64_t t = n * C + 16 * tj + r;
                const float v[4] = {o[tj][0], o[tj][1], o[tj][2], o[tj][3]};
                if (key_wave && t < a.n.T) put(a.dkey, a.row_parts > 1, part_qk, t, rows_qk, row_qk, v);
            }
        }
        if (w < VT) {
            D8 oc[CS];
#pragma unroll
            for (int ks = 0; ks < CS; ++ks) oc[ks] = lds_columns(sO + 32 * ks * SV + 16 * w + LV.col, SV);
            // ---- dv ----
            f32x4 o[CT];
#pragma unroll
            for (int tj = 0; tj < CT; ++tj) o[tj] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KK; ++ks) {
                float s[8];
                two_tiles(by_value[2 * ks], by_value[2 * ks + 1], s);
                const Split<T, 1> op(s);
#pragma unroll
                for (int tj = 0; tj < CT; ++tj) o[tj] = op.left(lds_two_halves(sK + 16 * tj * SK + LK.row2 + 32 * ks), o[tj]);
            }
#pragma unroll
            for (int tj = 0; tj < CT; ++tj) {
                const float scale = gate.to_end[16 * tj + r];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[tj][e] *= scale;
#pragma unroll
                for (int ks = tj / 2; ks < CS; ++ks) o[tj] = mma_d(oc[ks], lds_columns(sP + 32 * ks * SP + 16 * tj + LP.col, SP), o[tj]);
                const int64_t t = n * C + 16 * tj + r;
                const float v[4] = {o[tj][0], o[tj][1], o[tj][2], o[tj][3]};
                if (value_wave && t < a.n.T) put(a.dvalue, a.value_parts > 1, ks0, t, rows_v, row_v, v);
            }
            // ---- dS by value columns: two parts, as its only use is as an operand of dv ----
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) by_value[t][e] *= whole;
#pragma unroll
            for (int ks = 0; ks < CS; ++ks) {
                float v[8];
                unpack8(oc[ks], v);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] *= gate.from_start[32 * ks + 8 * c + e];
                const Split<T, 2> op(v);
#pragma unroll
                for (int t = 0; t < KT; ++t) by_value[t] = op.right(lds_columns(sQ + 32 * ks * SK + 16 * t + LK.col, SK), by_value[t]);
            }
        }
        if (w < KT) {
            // ---- dS by key columns: dhidden_init and the gates' gradient come from it ----
#pragma unroll
            for (int t = 0; t < VT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) by_key[t][e] *= whole;
#pragma unroll
            for (int ks = 0; ks < CS; ++ks) {
                float v[8];
                unpack8(qc[ks], v);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] *= gate.from_start[32 * ks + 8 * c + e];
                const Split<T, 3> op(v);
#pragma unroll
                for (int t = 0; t < VT; ++t) by_key[t] = op.right(lds_columns(sO + 32 * ks * SV + 16 * t + LV.col, SV), by_key[t]);
            }
        }
    }
    lds_barrier();
    if (w == gates_wave) {
        if (count > 0) gates_gradient(first);
        if (a.dgate_sums) {
            double x = gate_sum;
#pragma unroll
            for (int m = 1; m < 64; m *= 2) x += __hiloint2double(__shfl_xor(__double2hiint(x), m, 64), __shfl_xor(__double2loint(x), m, 64));
            if (lane == 0) a.dgate_sums[((blockIdx.y * a.n.H + h) * a.n.B + b) * a.plan.segments + order] = x;
        }
    }
    // rows past the end of a shorter sequence
    for (int64_t t = max(live, first) * C + tid / 16; t < min(last * C, a.n.T); t += NT / 16) {
        const float zero[4] = {0.f, 0.f, 0.f, 0.f};
        for (int col = 4 * (tid % 16); col < DKW && dk0 + col < DK; col += 64) {
            put(a.dquery, a.row_parts > 1, part_qk, t, rows_qk, hk * DK + dk0 + col, zero);
            put(a.dkey, a.row_parts > 1, part_qk, t, rows_qk, hk * DK + dk0 + col, zero);
        }
        for (int col = 4 * (tid % 16); col < DVW && dv0 + col < DV; col += 64)
            put(a.dvalue, a.value_parts > 1, ks0, t, rows_v, h * DV + dv0 + col, zero);
        if (a.dgate && tid % 16 == 0) a.dgate[(((int64_t)blockIdx.y * a.n.B + b) * a.n.T + t) * a.n.H + h] = 0.f;
    }
    if (seg == 0) {
#pragma unroll
        for (int t = 0; t < VT; ++t)
            if (key_wave && dv0 + 16 * t < DV) {
                const float x[4] = {by_key[t][0], by_key[t][1], by_key[t][2], by_key[t][3]};
                store_hidden<4>(a.dhidden_init, a.hidden_dtype, (bh * DK + dk0 + 16 * w + r) * DV + dv0 + 16 * t + 4 * c, x);
            }
    }
}

// dst = the sum of `parts` arrays of n floats behind each other, rounded once.
template <typename T> __global__ __launch_bounds__(256) void decay_sum_parts_kernel(const float *__restrict__ src, int parts, int64_t n, T *__restrict__ dst)
{
    for (int64_t i = 4 * (blockIdx.x * (int64_t)256 + threadIdx.x); i < n; i += 1024 * (int64_t)gridDim.x) {
        if (i + 4 <= n) {
            float s[4] = {0.f, 0.f, 0.f, 0.f}, x[4];
            for (int p = 0; p < parts; ++p) {
                load_vec<float, 2>(src + p * n + i, reinterpret_cast<float (&)[2]>(x[0]));
                load_vec<float, 2>(src + p * n + i + 2, reinterpret_cast<float (&)[2]>(x[2]));
#pragma unroll
                for (int e = 0; e < 4; ++e) s[e] += x[e];
            }
            store_vec<T, 4>(dst + i, s);
        } else {
            for (int64_t j = i; j < n; ++j) {
                float s = 0.f;
                for (int p = 0; p < parts; ++p) s += src[p * n + j];
                Elem<T>::store(dst + j, s);
            }
        }
    }
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
    constexpr size_t lds = sizeof(T) * (2 * C * lds_stride<T>(DKW) + 2 * C * lds_stride<T>(DVW) + 2 * C * lds_stride<T>(C)) +
                           sizeof(ChunkGates<C>) + sizeof(float) * (2 * CT * C + 2 * KT * C + KT);
    if (int e = allow_lds(grant, reinterpret_cast<const void *>(decay_gradient_kernel<T, DKW, DVW>), lds)) return e;
    const dim3 grid(a.n.B * a.n.H, ((a.n.DK + DKW - 1) / DKW) * ((a.n.DV + DVW - 1) / DVW), a.plan.segments);
    decay_gradient_kernel<T, DKW, DVW><<<grid, (DKW > DVW ? DKW : DVW) * 4, lds, stream>>>(a);
    return launch_status();
}
template <typename T> int dispatch_gradient(hipStream_t stream, const BackwardArgs &a)
{
    if (a.n.DK <= 64) return a.n.DV <= 64 ? launch_gradient<T, 64, 64>(stream, a) : launch_gradient<T, 64, 128>(stream, a);
    return a.n.DV <= 64 ? launch_gradient<T, 128, 64>(stream, a) : launch_gradient<T, 128, 128>(stream, a);
}

template <typename T> int sum_parts(hipStream_t stream, const float *src, int parts, int64_t n, void *dst)
{
    const int64_t blocks = (n + 1023) / 1024;
    decay_sum_parts_kernel<T><<<(unsigned)(blocks < 4096 ? blocks : 4096), 256, 0, stream>>>(src, parts, n, static_cast<T *>(dst));
    return launch_status();
}

}  // namespace

int decay_backward(void *stream, const DecaySizes &n, const DecayPlan &plan, gla_dtype dtype, gla_dtype hidden_dtype,
                   const DecayRows &gates, const DecayRows &keys, const DecayRows &values, const DecayRows &queries,
                   const DecayRows &dout, const int32_t *lengths, const float *kept, const void *dhidden_final, bool constant_gates,
                   void *dhidden_init, float *dlog_decay, void *dvalue, void *dkey, void *dquery, float *entering, float *decays,
                   const DecayParts &parts)
{
    int e = decay_entering_states(stream, kDecayCotangents, n, plan, dtype, hidden_dtype, dhidden_final, gates, queries, dout,
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
    auto sum = [&](const float *src, int count, int64_t m, void *dst) {
        if (!e && m) e = dtype == GLA_BF16 ? sum_parts<__bf16>(s, src, count, m, dst) : sum_parts<float>(s, src, count, m, dst);
    };
    if (parts.rows > 1) {
        sum(parts.dquery, parts.rows, nk, dquery);
        sum(parts.dkey, parts.rows, nk, dkey);
    }
    if (parts.values > 1) sum(parts.dvalue, parts.values, nv, dvalue);
    if (!e && !constant_gates && parts.gates > 1 && n.T) e = sum_parts<float>(s, parts.dgate, parts.gates, n.B * n.T * n.H, dlog_decay);
    if (!e && constant_gates) {
        decay_sum_gates_kernel<<<n.H, 64, 0, s>>>(parts.gate_sums, parts.gates, n.H, n.B * plan.segments, dlog_decay);
        e = launch_status();
    }
    return e;
}

}  // namespace gla
