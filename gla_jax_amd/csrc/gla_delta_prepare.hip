// The gated delta rule: what the walks multiply by, of all chunks at once.
#include "gla_delta.hpp"

namespace gla {
namespace {

// One workgroup: a chunk of a (batch, head) pair.  Forward it leaves (1 + M b)^{-1} and P with rows i as the operands' rows, backward
// the transposes of (1 + b M)^{-1} and P, with rows j.
//
// The inverse, in 32 bits throughout: each wave solves for one block of 16 rows on the diagonal by substitution, a column a lane, and then
// goes down (forward, for the transposed matrix: up) its own column of blocks, X_ij = -X_ii sum_k N_ik X_kj, by float products whose accumulators are
// the next product's operands as they are.  The waves wait for each other once.
//
// 27 us for the 1536 chunks of B4 T4096 H6 D128 (101 MB, 3.7 TB/s), 58 for the 4096 of B1 T32768 H8, 6.9 for one.  A workgroup takes 19000 cycles, of which it
// waits 8000 for its rows, makes scores for 3000 and solves for 5500, each a chain of dependent steps; three of them share a compute unit.
template <typename T, int DKP, bool BACK> __global__ __launch_bounds__(256) void delta_prepare_kernel(const DeltaArgs a)
{
    typedef DeltaChunk<T> DC;
    constexpr int C = DC::C, CT = DC::CT, KS = DKP / 32, NW = 4, NT = 256, kTriangle = CT * (CT + 1) / 2;
    constexpr int kRow = C + 4, kBlock = 16 * 20, kParts = DC::kParts, kScoreParts = BACK ? kParts : DC::kFew;
    typedef typename FragTypes<T>::d8 D8;
    typedef typename Packed4<T>::t Four;
    typedef LdsTile<T, DKP> Tile;
    extern __shared__ char smem[];
    T *sK = reinterpret_cast<T *>(smem), *sQ = sK + C * Tile::kRow;
    float *sN = reinterpret_cast<float *>(sQ + C * Tile::kRow), *sB = sN + C * kRow, *sX = reinterpret_cast<float *>(sQ);      // (behind the scores the queries are not needed)
    static_assert(CT * kBlock * sizeof(float) <= C * Tile::kRow * sizeof(T), "");
    ChunkGates<C> *gate = reinterpret_cast<ChunkGates<C> *>(sB + C);

    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, r = lane & 15, c = lane >> 4;
    const unsigned H = (unsigned)a.n.H, group = H / (unsigned)a.n.HK, rest = blockIdx.x / H, chunks = (unsigned)a.chunks;
    const int64_t h = blockIdx.x % H, n = rest % chunks, b = rest / chunks, hk = blockIdx.x % H / group;
    const int T_ = (int)a.n.T, len = a.lengths ? min(max(a.lengths[b], 0), T_) : T_, first = (int)n * C, there = len - first;
    if (there <= 0) return;
    const int DK = (int)a.n.DK;
    {
        RowsInFlight<T, C, DKP, NT> x, q;
        const unsigned at = tid;
        x.load(at, static_cast<const T *>(a.keys.p) + b * a.keys.sb + hk * a.keys.sh + first * a.keys.st, (int)a.keys.st, there, DK);
        q.load(at, static_cast<const T *>(a.queries.p) + b * a.queries.sb + hk * a.queries.sh + first * a.queries.st, (int)a.queries.st, there, DK);
        if (w == NW - 1) {
            const float *G = static_cast<const float *>(a.gates.p) + b * a.gates.sb + h * a.gates.sh;
            chunk_gates<C>(*gate, lane < C && lane < there ? G[(first + lane) * a.gates.st] : 0.f);
        } else if (w == NW - 2 && lane < C) {
            const float *B = static_cast<const float *>(a.betas.p) + b * a.betas.sb + h * a.betas.sh;
            sB[lane] = lane < there ? B[(first + lane) * a.betas.st] : 0.f;
        }
        x.store(at, sK, there, DK);
        q.store(at, sQ, there, DK);
    }
    lds_barrier();
    const int64_t pair = b * H + h, pc = pair * chunks + n;
    T *inverse = static_cast<T *>(a.to.inverse) + pc * (DC::kSteps * kParts * 512);
    T *scores = static_cast<T *>(a.to.scores) + pc * (DC::kSteps * kScoreParts * 512);
    // four values of a tile behind the operand's rows 16t .., contracted tokens 16u ..
    auto put = [&](T *to, auto parts, int t, int u, f32x4 v) {
        constexpr int N = decltype(parts)::value;
        const int step = BACK ? DC::upper(t, u >> 1) : DC::lower(t, u >> 1);
#pragma unroll
        for (int p = 0; p < N; ++p) {
            const Four f = pack_results<T>(v);
            *reinterpret_cast<Four *>(to + ((step * N + p) * 64 + lane) * 8 + 4 * (u & 1)) = f;
            if (t == u && (t & 1) == (BACK ? 1 : 0))     // the other half of the step lies on the other side of the diagonal
                *reinterpret_cast<Four *>(to + ((step * N + p) * 64 + lane) * 8 + 4 * (BACK ? 0 : 1)) = Four{};
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] -= (float)f[e];
        }
    };
    // M and P tile by tile, both at a time: they have one operand and their weights in common.  Forward four neighbouring j of one i a lane,
    // backward four i of one j.
    const Tile tile;
#pragma unroll
    for (int m = 0; m < (kTriangle + NW - 1) / NW; ++m) {
        const int unit = w + m * NW;
        if (unit >= kTriangle) break;
        int ti, tj;
        triangle(unit, ti, tj);
        const Tile L = tile.here();
        f32x4 kk = {0.f, 0.f, 0.f, 0.f}, qk = kk;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const D8 kj = L.rows(sK, tj, ks), ki = L.rows(sK, ti, ks), qi = L.rows(sQ, ti, ks);
            kk = BACK ? mma_d(ki, kj, kk) : mma_d(kj, ki, kk);
            qk = BACK ? mma_d(qi, kj, qk) : mma_d(kj, qi, qk);
        }
        const int i0 = 16 * ti + (BACK ? 4 * c : r), j0 = 16 * tj + (BACK ? r : 4 * c), one = BACK ? j0 : i0, four = BACK ? i0 : j0;
        const float sum1 = gate->sum[one], rest1 = gate->rest[one];
        const f32x4 sum4 = *reinterpret_cast<const f32x4 *>(gate->sum + four), rest4 = *reinterpret_cast<const f32x4 *>(gate->rest + four),
                    beta4 = *reinterpret_cast<const f32x4 *>(sB + four);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = BACK ? i0 + e : i0, j = BACK ? j0 : j0 + e;
            const float weight = BACK ? ChunkGates<C>::weight(sum4[e], rest4[e], sum1, rest1) : ChunkGates<C>::weight(sum1, rest1, sum4[e], rest4[e]);
            // (the gate that N takes is b_j forward and b_i backward: of the four in both cases)
            sN[(four + e) * kRow + one] = j < i ? kk[e] * weight * beta4[e] : 0.f;
            qk[e] = j <= i ? qk[e] * weight : 0.f;
        }
        if (BACK) put(scores, std::integral_constant<int, kScoreParts>{}, tj, ti, qk);
        else put(scores, std::integral_constant<int, kScoreParts>{}, ti, tj, qk);
    }
    if (tid < C) {
        float *to = a.to.gates + pc * DC::kGates;
        to[tid] = gate->from_start[tid];
        to[C + tid] = gate->to_end[tid];
        to[2 * C + tid] = sB[tid];
        if (tid == 0) to[3 * C] = gate->whole;
    }
    lds_barrier();

    // sN holds N (backward) or its transpose (forward), what lies on the other side of its diagonal blocks zero or not read
    f32x4 X[CT];
    if (w < CT) {
        float x[16];
        f32x4 rows[16][4];                       // (of the triangle: all on their way at once)
        const float *D = sN + 16 * w * kRow + 16 * w;
#pragma unroll
        for (int m = 0; m < 16; ++m) {
            const int i = BACK ? m : 15 - m;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (BACK ? 4 * j < i : 4 * j + 3 > i) rows[i][j] = *reinterpret_cast<const f32x4 *>(D + i * kRow + 4 * j);
        }
#pragma unroll
        for (int m = 0; m < 16; ++m) {
            const int i = BACK ? m : 15 - m;
            float s = i == r ? 1.f : 0.f;
#pragma unroll
            for (int k = 0; k < m; ++k) {        // the newest last
                const int j = BACK ? k : 15 - k;
                s -= rows[i][j >> 2][j & 3] * x[j];
            }
            x[i] = s;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            X[0][e] = c == 0 ? x[e] : c == 1 ? x[4 + e] : c == 2 ? x[8 + e] : x[12 + e];
            sX[w * kBlock + (4 * c + e) * 20 + r] = X[0][e];
        }
    }
    lds_barrier();
    if (w >= CT) return;
    constexpr auto kAll = std::integral_constant<int, kParts>{};
    put(inverse, kAll, w, w, X[0]);
#pragma unroll
    for (int s = 1; s < CT; ++s) {
        const int i = BACK ? w + s : w - s;
        if (i < 0 || i >= CT) break;
        f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < s; ++k) {
            const int kb = BACK ? w + k : w - k;
            y = mma_t(*reinterpret_cast<const f32x4 *>(sN + (16 * i + r) * kRow + 16 * kb + 4 * c), X[k], y);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = -y[e];
        X[s] = mma_t(*reinterpret_cast<const f32x4 *>(sX + i * kBlock + r * 20 + 4 * c), y, f32x4{0.f, 0.f, 0.f, 0.f});
        put(inverse, kAll, w, i, X[s]);
    }
}

template <typename T, int DKP, bool BACK> int launch_prepare(hipStream_t stream, const DeltaArgs &a)
{
    typedef DeltaChunk<T> DC;
    constexpr size_t lds = sizeof(T) * 2 * DC::C * LdsTile<T, DKP>::kRow +
                           sizeof(float) * (DC::C * (DC::C + 4) + DC::C) + sizeof(ChunkGates<DC::C>);
    static_assert(lds <= 64 * 1024, "");
    delta_prepare_kernel<T, DKP, BACK><<<a.pairs * a.chunks, 256, lds, stream>>>(a);
    return launch_status();
}
template <typename T, bool BACK> int dispatch_prepare(hipStream_t stream, const DeltaArgs &a)
{
    return a.n.DK <= 64 ? launch_prepare<T, 64, BACK>(stream, a) : launch_prepare<T, 128, BACK>(stream, a);
}

}  // namespace

int delta_prepare(void *stream, const DeltaArgs &a, gla_dtype dtype, bool backward)
{
    if (a.chunks == 0) return 0;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == GLA_BF16) return backward ? dispatch_prepare<__bf16, true>(s, a) : dispatch_prepare<__bf16, false>(s, a);
    return backward ? dispatch_prepare<float, true>(s, a) : dispatch_prepare<float, false>(s, a);
}

}  // namespace gla
