// The gated delta rule: the gradients of a chunk, all chunks at once, behind the backward walk.
//
// With S the state before a chunk, S' the one behind it, dS' its cotangent, u = b x, dv = b du and
//       D_ij = e^{L_i - L_j} do_i.u_j for j <= i,   E_ij = e^{L_i - L_j} dv_i.u_j for j < i,
//       dq_i = e^{L_i} S do_i + sum_j D_ij k_j
//       dk_j = -e^{L_j} S dv_j + e^{L_C - L_j} dS' u_j + sum_i D_ij q_i - sum_i (E + E^T)_ij k_i
//       db_i = x_i.du_i
// For the gradient of a_t: what is read at i carries e^{L_i} and what is written at j carries e^{-L_j}, and of all that multiplies the
// state, u_j.du_j (written) and dv_i.(v_i - x_i) (read) leave dv.v:
//       da_t = <S', dS'> + sum_{i>=t} (o_i.do_i - v_i.dv_i)    over the chunk's tokens i,
// with o_i.do_i = sum_j P_ij (do_i.u_j) + e^{L_i} q_i.(S do_i).  The first term starts the sum anew at every chunk, so no difference runs over a
// whole sequence.  (Off by 5e-7 of its norm; the chunked form differentiated step by step in 32-bit operations is off by 3e-7.)
#include "gla_delta.hpp"

namespace gla {
namespace {

constexpr int kSlice = 64;                       // value features at a time

template <typename T, int F> __device__ __forceinline__ int place_in(int row, int col) { return LdsTile<T, F>::piece(row, col & ~7) + (col & 7); }

// values of the states' place in LDS
template <typename T, int DKP> constexpr int state_place()
{
    typedef DeltaChunk<T> DC;
    constexpr int states = (DC::kParts + DC::kFew) * kSlice * LdsTile<T, DKP>::kRow, scores = 2 * DC::C * (DC::kFew * LdsTile<T, DC::C>::kRow + LdsTile<T, DKP>::kRow);
    return states > scores ? states : scores;
}

// 175 us for the 1536 chunks of B4 T4096 H6 D128, 87 for the 1056 of B2 T2050 H16 64x128: 537 MB and 3.1 TB/s at 128 x 128, of which the states before the
// chunks are 100 (32 bits), their cotangents 100 (in two parts; in one, 154 and 85 us), what was written and its cotangents 50 each, and registers that do not fit 30
// each way.  LDS and registers leave one workgroup a compute unit, whose phases (a slice's rows arrive, its products, the scores) do not overlap; chunk after
// chunk in one workgroup, the next one's first rows on their way, it needs 90 to 180 registers more than there are.
// One workgroup: a chunk of a (batch, head) pair; a wave makes 16 key features of dq and dk, at 64 features of every second tile of tokens.
template <typename T, int DKP> __global__ __launch_bounds__(512) void delta_gradient_kernel(const DeltaArgs a)
{
    typedef DeltaChunk<T> DC;
    constexpr int C = DC::C, CT = DC::CT, CS = DC::CS, KS = DKP / 32, NW = 8, NT = 64 * NW, VS = kSlice / 32, kParts = DC::kParts, kFew = DC::kFew;
    constexpr int kTriangle = CT * (CT + 1) / 2, kUnits = (2 * kTriangle + NW - 1) / NW, kShare = NW / CT;
    constexpr int FT = DKP / 16, SHARES = NW / FT, OWN = CT / SHARES;      // tiles of features; waves to each; its tiles of tokens
    typedef typename FragTypes<T>::d8 D8;
    typedef typename Packed4<T>::t Four;
    typedef LdsTile<T, DKP> TileK;
    typedef LdsTile<T, kSlice> TileO;
    typedef LdsTile<T, C> TileU;
    constexpr int kK = C * TileK::kRow, kS = kSlice * TileK::kRow, kU = kSlice * TileU::kRow, kP = C * TileU::kRow;
    extern __shared__ char smem[];
    // the scores, keys and queries take the states' place
    T *sS = reinterpret_cast<T *>(smem), *sD = sS + kParts * kS, *sO = sS + state_place<T, DKP>(), *sU = sO + C * TileO::kRow, *sX = sU + kParts * kU,
      *sP = sS, *sE = sP + kFew * kP, *sK = sE + kFew * kP, *sQ = sK + kK;
    ChunkGates<C> *gate = reinterpret_cast<ChunkGates<C> *>(sX + kFew * kU);
    struct Sums {
        float beta[C];
        float pairs[CT][C];                      // row sums of P (do.u), one column of tiles each
        float state[FT][C];                      // e^{L_i} q_i.(S do_i), 16 features each
        float db[kShare][C], vdv[kShare][C];
    };
    Sums &sums = *reinterpret_cast<Sums *>(gate + 1);

    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, r = lane & 15, c = lane >> 4;
    const int wf = w % FT, wt = w / FT;          // the wave's features 16 wf .. and tiles of tokens wt + SHARES t
    const unsigned H = (unsigned)a.n.H, group = H / (unsigned)a.n.HK, rest = blockIdx.x / H, chunks = (unsigned)a.chunks;
    const int64_t h = blockIdx.x % H, n = rest % chunks, b = rest / chunks, hk = blockIdx.x % H / group, pair = b * H + h;
    const int T_ = (int)a.n.T, len = a.lengths ? min(max(a.lengths[b], 0), T_) : T_, first = (int)n * C, there = len - first;
    const int DK = (int)a.n.DK, DV = (int)a.n.DV;
    const bool parts = a.row_parts > 1;
    const int64_t key_row = a.n.HK * DK, key_at = (((parts ? blockIdx.x % H % group : 0) * a.n.B + b) * T_ + first) * key_row + hk * DK;
    T *dV = static_cast<T *>(a.dvalue) + ((b * T_ + first) * H + h) * DV;
    auto put_keys = [&](void *array, int ti, f32x4 v) {       // four features of a token
        const int64_t at = key_at + (16 * ti + r) * key_row + 16 * wf + 4 * c;
        if (16 * wf >= DK || first + 16 * ti + r >= T_) return;
        if (parts) *reinterpret_cast<f32x4 *>(static_cast<float *>(array) + at) = v;
        else *reinterpret_cast<Four *>(static_cast<T *>(array) + at) = pack_results<T>(v);
    };
    const int64_t gate_at = (b * T_ + first + lane) * H + h;
    if (there <= 0) {                            // behind the end: zeros
        for (int ti = wt; ti < CT; ti += SHARES) {
            put_keys(a.dquery, ti, f32x4{0.f, 0.f, 0.f, 0.f});
            put_keys(a.dkey, ti, f32x4{0.f, 0.f, 0.f, 0.f});
        }
        for (int i = tid; i < C * (DV / 4); i += NT)
            if (first + i / (DV / 4) < T_) *reinterpret_cast<Four *>(dV + (int64_t)(i / (DV / 4)) * H * DV + 4 * (i % (DV / 4))) = Four{};
        if (w == 0 && lane < C && first + lane < T_) a.dgate[gate_at] = a.dbeta[gate_at] = 0.f;
        return;
    }
    const T *V = static_cast<const T *>(a.values.p) + b * a.values.sb + h * a.values.sh + first * a.values.st;
    const T *O = static_cast<const T *>(a.dout.p) + b * a.dout.sb + h * a.dout.sh + first * a.dout.st;
    const float *G = static_cast<const float *>(a.gates.p) + b * a.gates.sb + h * a.gates.sh + first * a.gates.st;
    const int64_t floats = delta_written_floats(a.n, a.chunks, C), state = delta_state_floats(a.n);
    const float *kept = a.kept + pair * (delta_states_floats(a.n, a.chunks) + floats), *xs = kept + delta_states_floats(a.n, a.chunks) + n * C * DV;
    const float *dus = a.du + pair * floats + n * C * DV;
    const T *dS = static_cast<const T *>(a.dstates) + (pair * chunks + n) * state * kFew;
    kept += n * state;
    // A slice of values on its way: no load is under a branch, for then each waits for the one before, and the next slice's are issued before the
    // products of one.  (One after the other they took 25000 of a chunk's 46000 cycles at 128 x 128 features.)
    constexpr int kStates = kSlice / 16 * KS / NW, kTiles = kSlice / 16 / kShare;
    static_assert(kSlice / 16 * KS % NW == 0 && kSlice / 16 % kShare == 0, "");
    RowsInFlight<T, C, kSlice, NT> o;
    f32x4 low[kStates], high[kStates], written[kTiles], dwritten[kTiles];
    D8 dstate[kStates][kFew];
    T value[kTiles][4];
    const int own = w % CT, token = 16 * own + 4 * c;       // of what was written
    auto load_slice = [&](int dv0) {
        o.load(tid, O + dv0, (int)a.dout.st, there, DV - dv0);
#pragma unroll
        for (int i = 0; i < kStates; ++i) {
            const int m = (w + i * NW) / KS, ks = (w + i * NW) % KS;
            const unsigned from = dv0 + 16 * m < DV && 32 * ks < DK ? (((dv0 >> 4) + m) * (delta_state_tiles(DK) / 2) + ks) * 512 : 0;
            low[i] = *reinterpret_cast<const f32x4 *>(kept + from + lane * 4);
            high[i] = *reinterpret_cast<const f32x4 *>(kept + from + 256 + lane * 4);
#pragma unroll
            for (int p = 0; p < kFew; ++p) dstate[i][p] = ld8(dS + from * kFew + p * 512 + lane * 8);
        }
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
            const int m = w / CT + i * kShare, at = dv0 + 16 * m < DV ? dv0 + 16 * m : 0;
            const unsigned from = (at / 16 * CT + own) * 256 + lane * 4;
            written[i] = *reinterpret_cast<const f32x4 *>(xs + from);
            dwritten[i] = *reinterpret_cast<const f32x4 *>(dus + from);
#pragma unroll
            for (int e = 0; e < 4; ++e) value[i][e] = V[(int64_t)min(token + e, there - 1) * a.values.st + at + r];
        }
    };
    RowsInFlight<T, C, DKP, NT> key, query;
    load_slice(0);
    float log_decay = 0.f;
    {
        if (w == 0) {
            log_decay = lane < C && lane < there ? G[lane * a.gates.st] : 0.f;
            chunk_gates<C>(*gate, log_decay);
        }
        if (w == 1 && lane < C) sums.beta[lane] = a.to.gates[(pair * chunks + n) * DC::kGates + 2 * C + lane];
    }
    const TileK tk;
    const TileO to;
    const TileU tu;
    f32x4 score[kUnits], fromO[OWN], fromX[OWN], fromU[OWN];
    float db[4] = {}, vdv[4] = {};               // of the tokens 16 (w % CT) + 4c + e
#pragma unroll
    for (int m = 0; m < kUnits; ++m) score[m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < OWN; ++t) fromO[t] = fromX[t] = fromU[t] = f32x4{0.f, 0.f, 0.f, 0.f};

    for (int dv0 = 0; dv0 < DV; dv0 += kSlice) {
        lds_barrier();                           // beta is there; the last slice's tiles are read
#pragma unroll
        for (int i = 0; i < kStates; ++i) {      // eight features of a value feature a lane
            const int m = (w + i * NW) / KS, ks = (w + i * NW) % KS, col = 32 * ks + 8 * c, at = TileK::piece(16 * m + r, col);
            const bool is = dv0 + 16 * m < DV && col < DK;
            float x[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = is ? low[i][e] : 0.f, x[4 + e] = is ? high[i][e] : 0.f;
            const Split<T, kParts> split(x);
#pragma unroll
            for (int p = 0; p < kParts; ++p) st8(sS + p * kS + at, split.part[p]);
#pragma unroll
            for (int p = 0; p < kFew; ++p) st8(sD + p * kS + at, is ? dstate[i][p] : D8{});
        }
        const f32x4 beta = *reinterpret_cast<const f32x4 *>(sums.beta + token);
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
            const int m = w / CT + i * kShare, at = place_in<T, C>(16 * m + r, token);
            const bool is = dv0 + 16 * m < DV;
            f32x4 u, dx;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = is ? written[i][e] : 0.f, du = is ? dwritten[i][e] : 0.f, v = is && token + e < there ? (float)value[i][e] : 0.f;
                u[e] = beta[e] * x;
                dx[e] = beta[e] * du;
                db[e] += x * du;
                vdv[e] += v * dx[e];
            }
#pragma unroll
            for (int p = 0; p < kFew; ++p) {
                const Four f = pack_results<T>(dx);
                *reinterpret_cast<Four *>(sX + p * kU + at) = f;
#pragma unroll
                for (int e = 0; e < 4; ++e) dx[e] -= (float)f[e];
            }
#pragma unroll
            for (int p = 0; p < kParts; ++p) {
                const Four f = pack_results<T>(u);
                *reinterpret_cast<Four *>(sU + p * kU + at) = f;
#pragma unroll
                for (int e = 0; e < 4; ++e) u[e] -= (float)f[e];
            }
        }
        o.store(tid, sO, there, DV - dv0);
        if (dv0 + kSlice < DV) {
            load_slice(dv0 + kSlice);
        } else {
            key.load(tid, static_cast<const T *>(a.keys.p) + b * a.keys.sb + hk * a.keys.sh + first * a.keys.st, (int)a.keys.st, there, DK);
            query.load(tid, static_cast<const T *>(a.queries.p) + b * a.queries.sb + hk * a.queries.sh + first * a.queries.st, (int)a.queries.st, there, DK);
        }
        lds_barrier();
        // dv, a token's 4 values twice
        for (int unit = w; unit < CT * VS; unit += NW) {
            const int ti = unit / VS, ks = unit % VS, token = 16 * ti + r, value = dv0 + 32 * ks + 4 * c;
            const D8 x = tu.columns(sX, ks, ti);
            float v[8];
            unpack8(x, v);
            T *row = dV + (int64_t)token * H * DV;
            if (first + token < T_) {
                const float low[4] = {v[0], v[1], v[2], v[3]}, high[4] = {v[4], v[5], v[6], v[7]};
                if (value < DV) store_vec<T, 4>(row + value, low);
                if (value + 16 < DV) store_vec<T, 4>(row + value + 16, high);
            }
        }
#pragma unroll
        for (int m = 0; m < kUnits; ++m) {
            const int unit = w + m * NW;
            if (unit >= 2 * kTriangle) break;
            int ti, tj;
            triangle(unit < kTriangle ? unit : unit - kTriangle, ti, tj);
#pragma unroll
            for (int ks = 0; ks < VS; ++ks) {
                if (unit < kTriangle) {
                    const D8 o = to.halves(sO, ti, ks);
#pragma unroll
                    for (int p = kParts - 1; p >= 0; --p) score[m] = mma_d(tu.columns(sU + p * kU, ks, tj), o, score[m]);
                } else {
                    D8 x[kFew], u[kFew];
#pragma unroll
                    for (int p = 0; p < kFew; ++p) {
                        x[p] = tu.columns(sX + p * kU, ks, ti);
                        u[p] = tu.columns(sU + p * kU, ks, tj);
                    }
                    score[m] = mma_parts(u, x, score[m]);
                }
            }
        }
#pragma unroll
        for (int ks = 0; ks < VS; ++ks) {
            D8 s[kParts];
#pragma unroll
            for (int p = 0; p < kParts; ++p) s[p] = tk.columns(sS + p * kS, ks, wf);
#pragma unroll
            for (int t = 0; t < OWN; ++t) {
                const int ti = wt + SHARES * t;
                fromO[t] = mma_whole(s, to.halves(sO, ti, ks), fromO[t]);
                D8 x[kFew], few[kFew];
#pragma unroll
                for (int p = 0; p < kFew; ++p) {
                    x[p] = tu.columns(sX + p * kU, ks, ti);
                    few[p] = s[p];
                }
                fromX[t] = mma_parts(few, x, fromX[t]);
            }
        }
        // (in a loop of its own, without the states' parts beside: 175 us, together 181)
#pragma unroll
        for (int ks = 0; ks < VS; ++ks) {
            D8 d[kFew];
#pragma unroll
            for (int p = 0; p < kFew; ++p) d[p] = tk.columns(sD + p * kS, ks, wf);
#pragma unroll
            for (int t = 0; t < OWN; ++t) {
                const int ti = wt + SHARES * t;
                D8 u[kFew];
#pragma unroll
                for (int p = 0; p < kFew; ++p) u[p] = tu.columns(sU + p * kU, ks, ti);
                fromU[t] = mma_parts(d, u, fromU[t]);
            }
        }
    }
    lds_barrier();                               // the states are read
    key.store(tid, sK, there, DK);
    query.store(tid, sQ, there, DK);
    if (w < CT / 2 * kFew) *reinterpret_cast<Four *>(tu.four(sP + w % kFew * kP, w / kFew * 2, w / kFew * 2 + 1)) = Four{};      // the tiles above the diagonal that operands reach into
    lds_barrier();
#pragma unroll
    for (int m = 0; m < kUnits; ++m) {
        const int unit = w + m * NW;
        if (unit >= 2 * kTriangle) break;
        int ti, tj;
        triangle(unit < kTriangle ? unit : unit - kTriangle, ti, tj);
        const int i = 16 * ti + r, j = 16 * tj + 4 * c;
        f32x4 weight;
#pragma unroll
        for (int e = 0; e < 4; ++e) weight[e] = ChunkGates<C>::weight(gate->sum[i], gate->rest[i], gate->sum[j + e], gate->rest[j + e]);
        if (unit < kTriangle) {
            const f32x4 qk = tile_product<KS>(tk, sK, tj, sQ, ti);
            float sum = 0.f;
            f32x4 d;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                d[e] = j + e <= i ? weight[e] * score[m][e] : 0.f;
                sum += j + e <= i ? qk[e] * d[e] : 0.f;
            }
            sum = sum_over_c(sum);
            if (c == 0) sums.pairs[tj][i] = sum;
#pragma unroll
            for (int p = 0; p < kFew; ++p) {
                const Four f = pack_results<T>(d);
                *reinterpret_cast<Four *>(tu.four(sP + p * kP, ti, tj)) = f;
#pragma unroll
                for (int e = 0; e < 4; ++e) d[e] -= (float)f[e];
            }
        } else {
            f32x4 d;
#pragma unroll
            for (int e = 0; e < 4; ++e) d[e] = j + e < i ? -weight[e] * score[m][e] : 0.f;
#pragma unroll
            for (int p = 0; p < kFew; ++p) {
                const Four f = pack_results<T>(d);
                *reinterpret_cast<Four *>(tu.four(sE + p * kP, ti, tj)) = f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (j + e < i) sE[p * kP + place_in<T, C>(j + e, i)] = f[e];
                    d[e] -= (float)f[e];
                }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < OWN; ++t) {
        const int ti = wt + SHARES * t;
        const float start = gate->from_start[16 * ti + r], end = gate->to_end[16 * ti + r];
        const Four q = *reinterpret_cast<const Four *>(tk.four(sQ, ti, wf));
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            fromO[t][e] *= start;
            sum += fromO[t][e] * (float)q[e];
            fromX[t][e] = end * fromU[t][e] - start * fromX[t][e];
        }
        sum = sum_over_c(sum);
        if (c == 0) sums.state[wf][16 * ti + r] = sum;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        db[e] = sum_over_r(db[e]);
        vdv[e] = sum_over_r(vdv[e]);
        if (r == 0) {
            sums.db[w / CT][16 * (w % CT) + 4 * c + e] = db[e];
            sums.vdv[w / CT][16 * (w % CT) + 4 * c + e] = vdv[e];
        }
    }
    lds_barrier();
    if (w == 0) {
        double x = 0.0;
        float beta = 0.f;
        if (lane < C) {
            for (int tj = 0; tj <= lane / 16; ++tj) x += sums.pairs[tj][lane];
            for (int i = 0; i < FT; ++i) x += sums.state[i][lane];
            for (int i = 0; i < kShare; ++i) {
                x -= sums.vdv[i][lane];
                beta += sums.db[i][lane];
            }
            if (lane >= there) x = 0.0;
        }
        double behind = 0.0;
        for (int i = 0; i < DV / 4; ++i) behind += a.dots[(pair * chunks + n) * (DV / 4) + i];
        const double before = prefix_sum_wave(x), all = __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(before), 63),
                                                                         __builtin_amdgcn_readlane(__double2loint(before), 63));
        if (lane < C && first + lane < T_) {
            // (a gate that forgets all has no gradient: the sum says so but for its rounding)
            a.dgate[gate_at] = lane < there && log_decay != -INFINITY ? (float)(behind + (all - before + x)) : 0.f;
            a.dbeta[gate_at] = lane < there ? beta : 0.f;
        }
    }
    D8 kc[CS], qc[CS];
#pragma unroll
    for (int ks = 0; ks < CS; ++ks) {
        kc[ks] = tk.columns(sK, ks, wf);
        qc[ks] = tk.columns(sQ, ks, wf);
    }
#pragma unroll
    for (int t = 0; t < OWN; ++t) {
        const int ti = wt + SHARES * t;
#pragma unroll
        for (int ks = 0; ks < CS; ++ks) {
#pragma unroll
            for (int p = kFew - 1; p >= 0; --p) {
                if (ks <= ti / 2) fromO[t] = mma_d(kc[ks], tu.halves(sP + p * kP, ti, ks), fromO[t]);
                if (ks >= ti / 2) fromX[t] = mma_d(qc[ks], tu.columns(sP + p * kP, ks, ti), fromX[t]);
                fromX[t] = mma_d(kc[ks], tu.halves(sE + p * kP, ti, ks), fromX[t]);
            }
        }
        put_keys(a.dquery, ti, fromO[t]);
        put_keys(a.dkey, ti, fromX[t]);
    }
}

// Gradients of heads that share a key head, summed in order.
template <typename T> __global__ __launch_bounds__(256) void delta_sum_heads_kernel(const float *__restrict__ src, int parts, int64_t n, T *__restrict__ dst)
{
    for (int64_t i = 4 * (blockIdx.x * (int64_t)256 + threadIdx.x); i < n; i += 1024 * (int64_t)gridDim.x) {
        float s[4] = {0.f, 0.f, 0.f, 0.f}, x[4];
        for (int p = 0; p < parts; ++p) {
            load_vec<float, 4>(src + p * n + i, x);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += x[e];
        }
        store_vec<T, 4>(dst + i, s);
    }
}

template <typename T, int DKP> int launch_gradient(hipStream_t stream, const DeltaArgs &a)
{
    typedef DeltaChunk<T> DC;
    static LdsGrant grant;
    constexpr int C = DC::C, NW = 8, kParts = DC::kParts;
    constexpr size_t lds = sizeof(T) * (state_place<T, DKP>() + C * LdsTile<T, kSlice>::kRow + (kParts + DC::kFew) * kSlice * LdsTile<T, C>::kRow) +
                           sizeof(ChunkGates<C>) + sizeof(float) * C * (1 + DC::CT + DKP / 16 + 2 * (NW / DC::CT));
    static_assert(lds <= 160 * 1024 && NW % DC::CT == 0, "");
    if (int e = allow_lds(grant, reinterpret_cast<const void *>(delta_gradient_kernel<T, DKP>), lds)) return e;
    delta_gradient_kernel<T, DKP><<<a.pairs * a.chunks, 64 * NW, lds, stream>>>(a);
    return launch_status();
}

}  // namespace

int delta_gradients(void *stream, const DeltaArgs &a, gla_dtype dtype)
{
    if (a.chunks == 0) return 0;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == GLA_BF16) return a.n.DK <= 64 ? launch_gradient<__bf16, 64>(s, a) : launch_gradient<__bf16, 128>(s, a);
    return a.n.DK <= 64 ? launch_gradient<float, 64>(s, a) : launch_gradient<float, 128>(s, a);
}

int delta_sum_heads(void *stream, const DecaySizes &n, gla_dtype dtype, const float *parts, void *dst)
{
    const int64_t count = n.B * n.T * n.HK * n.DK, blocks = (count + 1023) / 1024;
    const dim3 grid((unsigned)(blocks < 4096 ? blocks : 4096));
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == GLA_BF16) delta_sum_heads_kernel<__bf16><<<grid, 256, 0, s>>>(parts, (int)(n.H / n.HK), count, static_cast<__bf16 *>(dst));
    else delta_sum_heads_kernel<float><<<grid, 256, 0, s>>>(parts, (int)(n.H / n.HK), count, static_cast<float *>(dst));
    return launch_status();
}

}  // namespace gla
