// Linear attention with one decay a head, and by the gated delta rule, one token for each row of a batch: the states lie in a pool and are
// updated where they lie.  Bound by reading and writing every state once.
//
// A wave takes 32 value columns of one state: a lane holds a piece of 16 bytes of each of DKP / (rows side by side) rows, all
// of them requested before the first is used.  A lane's rows follow each other, so that it reads its keys and queries in
// whole pieces; the lanes that hold the same columns are summed at the end.  Nothing goes through LDS.  128 rows of 16 heads of 128 x 128
// float states, none idle: 51.4 us for 270 MB, 5.25 TB/s.
//
// The delta rule writes b (v - S^T k) instead of v, S being decayed already: one more sum over the key features, of what the registers hold.
#include "gla_common.hpp"

namespace gla {
namespace {

// Indices of 4 or 8 bytes.
struct Indices {
    const void *p;
    int wide;
    __device__ __forceinline__ int64_t at(int64_t i) const
    {
        return wide ? static_cast<const int64_t *>(p)[i] : (int64_t) static_cast<const int32_t *>(p)[i];
    }
};

struct StepArgs {
    int64_t pool, B, H, HK, DK, DV, beams;
    void *states;
    const float *log_decay, *beta;               // beta: NULL where all of the value is written
    int64_t gates_b, gates_h, beta_b, beta_h;
    const void *value, *key, *query;
    int64_t value_b, value_h, key_b, key_h, query_b, query_h;
    Indices slots, parents;
    void *out;
};

// The pool's row of batch row i: i itself, or what `slots` says; -1 where that is none.
__device__ __forceinline__ int64_t slot_of(const StepArgs &a, int64_t i)
{
    const int64_t s = a.slots.p ? a.slots.at(i) : i;
    return s >= 0 && s < a.pool ? s : -1;
}

template <typename T, typename HT, int DKP, bool DELTA> struct StepState {
    static constexpr int VEC = 16 / sizeof(HT), LPR = 32 / VEC, SIDE = 64 / LPR, PER = DKP / SIDE;
    typedef HT Piece __attribute__((ext_vector_type(VEC)));
    typedef T Four __attribute__((ext_vector_type(4)));
    Piece x[PER];
    Four k[PER / 4], q[PER / 4], v[VEC / 4];
    float log_decay, beta;
    // The token's rows, before the state: it takes longer, and in the beams' case it is not yet known where it lies.  No load is under a
    // condition, after which memory would be waited for; what does not exist reads what does, and counts as zero later.
    __device__ __forceinline__ void load_rows(const T *key, const T *query, const T *value, const float *gate, const float *rate, int DK,
                                              int DV, int row0, int col)
    {
#pragma unroll
        for (int i = 0; i < PER; i += 4) {
            const int at = row0 + i < DK ? row0 + i : 0;
            k[i / 4] = *reinterpret_cast<const Four *>(key + at);
            q[i / 4] = *reinterpret_cast<const Four *>(query + at);
        }
#pragma unroll
        for (int e = 0; e < VEC; e += 4) v[e / 4] = *reinterpret_cast<const Four *>(value + (col < DV ? col : 0) + e);
        log_decay = *gate;
        if constexpr (DELTA) beta = *rate;
    }
    __device__ __forceinline__ void load(const HT *state, int DK, int DV, int row0, int col)
    {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            x[i] = Piece{};
            if (row0 + i < DK && col < DV) x[i] = *reinterpret_cast<const Piece *>(state + (int64_t)(row0 + i) * DV + col);
        }
    }
    // over the lanes that hold the same columns
    static __device__ __forceinline__ void sum_rows(float (&o)[VEC])
    {
#pragma unroll
        for (int m = LPR; m < 64; m *= 2)
#pragma unroll
            for (int e = 0; e < VEC; ++e) o[e] += shfl_xor_f32(o[e], m);
    }
    // The token's update, and its output for the lane's columns (zeros outside): the sum runs over the key features in 32 bits
    // from the state before it is rounded.
    __device__ __forceinline__ void step(HT *state, T *out, int DK, int DV, int row0, int col)
    {
        const float decay = expf(log_decay);
        float vv[VEC], o[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            vv[e] = (float)v[e / 4][e % 4];
            o[e] = 0.f;
        }
        if constexpr (DELTA) {
            // what the state answers the key with
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const float ki = row0 + i < DK ? (float)k[i / 4][i % 4] : 0.f;
#pragma unroll
                for (int e = 0; e < VEC; ++e) o[e] += ki * (decay * (float)x[i][e]);
            }
            sum_rows(o);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                vv[e] = beta * (vv[e] - o[e]);
                o[e] = 0.f;
            }
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            // (4 divides DK: four rows exist or do not)
            const float ki = row0 + i < DK ? (float)k[i / 4][i % 4] : 0.f, qi = row0 + i < DK ? (float)q[i / 4][i % 4] : 0.f;
            float s[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                s[e] = decay * (float)x[i][e] + ki * vv[e];
                o[e] += qi * s[e];
            }
            if (row0 + i < DK && col < DV) store_vec<HT, VEC>(state + (int64_t)(row0 + i) * DV + col, s);
        }
        sum_rows(o);
        if ((threadIdx.x & 63) < LPR && col < DV) store_vec<T, VEC>(out + col, o);
    }
};

template <typename T, typename HT, int DKP, bool DELTA>
__global__ __launch_bounds__(256) void decay_step_kernel(const StepArgs a)
{
    typedef StepState<T, HT, DKP, DELTA> State;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const unsigned H = (unsigned)a.H;
    const int64_t b = blockIdx.x / H, h = blockIdx.x % H, hk = blockIdx.x % H / (H / (unsigned)a.HK);
    const int DK = (int)a.DK, DV = (int)a.DV, col = 32 * (blockIdx.y * waves + w) + State::VEC * (lane % State::LPR),
              row0 = State::PER * (lane / State::LPR);
    State s;
    s.load_rows(static_cast<const T *>(a.key) + b * a.key_b + hk * a.key_h, static_cast<const T *>(a.query) + b * a.query_b + hk * a.query_h,
                static_cast<const T *>(a.value) + b * a.value_b + h * a.value_h, a.log_decay + b * a.gates_b + h * a.gates_h,
                a.beta + b * a.beta_b + h * a.beta_h, DK, DV, row0, col);
    const int64_t slot = slot_of(a, b);
    T *out = static_cast<T *>(a.out) + (b * a.H + h) * DV;
    if (slot < 0) {                               // a row without a state
        const float zero[State::VEC] = {};
        if (lane < State::LPR && col < DV) store_vec<T, State::VEC>(out + col, zero);
        return;
    }
    HT *state = static_cast<HT *>(a.states) + (slot * a.H + h) * DK * DV;
    s.load(state, DK, DV, row0, col);
    s.step(state, out, DK, DV, row0, col);
}

// The waves that hold their part of a state in registers: 16 of 128 registers, 8 of 256.
constexpr int waves_of_beams(int DK) { return DK <= 128 ? 16 : 8; }

// The same for a group of beams, each from the state of the beam that it continues: a wave a beam, all of a group in one
// workgroup, which has read every state (of these columns) before it writes the first.  16 groups of 8 beams, 16 heads of 64 x 64 bfloat16:
// 7.7 us for 35 MB, 4.5 TB/s.
template <typename T, typename HT, int DKP, bool DELTA>
__global__ __launch_bounds__(64 * waves_of_beams(DKP)) void decay_step_beams_kernel(const StepArgs a)
{
    typedef StepState<T, HT, DKP, DELTA> State;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const unsigned H = (unsigned)a.H;
    const int64_t group = blockIdx.x / H, h = blockIdx.x % H, hk = blockIdx.x % H / (H / (unsigned)a.HK), b = group * a.beams + w;
    const int DK = (int)a.DK, DV = (int)a.DV, col = 32 * blockIdx.y + State::VEC * (lane % State::LPR),
              row0 = State::PER * (lane / State::LPR);
    State s;
    s.load_rows(static_cast<const T *>(a.key) + b * a.key_b + hk * a.key_h, static_cast<const T *>(a.query) + b * a.query_b + hk * a.query_h,
                static_cast<const T *>(a.value) + b * a.value_b + h * a.value_h, a.log_decay + b * a.gates_b + h * a.gates_h,
                a.beta + b * a.beta_b + h * a.beta_h, DK, DV, row0, col);
    const int64_t parent = a.parents.at(b), source = parent >= 0 && parent < a.beams ? group * a.beams + parent : b;
    const int64_t slot = slot_of(a, b);
    int64_t from = slot_of(a, source);
    if (from < 0) from = slot;
    T *out = static_cast<T *>(a.out) + (b * a.H + h) * DV;
    if (slot >= 0) s.load(static_cast<const HT *>(a.states) + (from * a.H + h) * DK * DV, DK, DV, row0, col);
    // the loads have to be back, not only issued, before another wave's stores may follow
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (slot < 0) {
        const float zero[State::VEC] = {};
        if (lane < State::LPR && col < DV) store_vec<T, State::VEC>(out + col, zero);
        return;
    }
    s.step(static_cast<HT *>(a.states) + (slot * a.H + h) * DK * DV, out, DK, DV, row0, col);
}

template <typename T, typename HT, int DKP, bool DELTA> int launch_step(hipStream_t stream, const StepArgs &a)
{
    const int64_t cols = (a.DV + 31) / 32;
    if (a.beams) {
        decay_step_beams_kernel<T, HT, DKP, DELTA><<<dim3(a.B / a.beams * a.H, cols), a.beams * 64, 0, stream>>>(a);
    } else {
        // Four waves side by side share the lines of a row (128 rows of 16 heads of 128 x 128: 51 us, each in a workgroup of its own 57); where there
        // are few, each has a compute unit of its own (4 rows: 4.3 us against 4.5; 16 rows take 8.0 either way).
        const int waves = a.B * a.H * cols >= 1024 ? (cols < 4 ? (int)cols : 4) : 1;
        decay_step_kernel<T, HT, DKP, DELTA><<<dim3(a.B * a.H, (cols + waves - 1) / waves), waves * 64, 0, stream>>>(a);
    }
    return launch_status();
}
template <typename T, typename HT, bool DELTA> int dispatch_step(hipStream_t stream, const StepArgs &a)
{
    return a.DK <= 64 ? launch_step<T, HT, 64, DELTA>(stream, a) : a.DK <= 128 ? launch_step<T, HT, 128, DELTA>(stream, a)
                                                                               : launch_step<T, HT, 256, DELTA>(stream, a);
}

// ---- states in another order ------------------------------------------------------------------
// states[w] <- states[parents[w]] in place, for every group of `beams` rows.  A thread takes one piece of a row's bytes of all
// the group's rows: it has read them all before it writes the first, and no other thread touches them.  A beam that continues
// itself moves nothing.  16 groups of 8 beams, 256 KB a beam: 8 us for the 67 MB that all of them are (they stay in the last-level cache).
struct ReorderArgs {
    int64_t pool, beams, pieces, blocks;       // pieces of a row; workgroups that share a row
    void *states;
    Indices parents, slots;
};
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <typename P, int WMAX> __global__ __launch_bounds__(256) void reorder_states_kernel(const ReorderArgs a)
{
    // lane w of every wave reads beam w's indices, all at once, and hands them round
    const int64_t group = blockIdx.x / a.blocks, at = blockIdx.x % a.blocks * 256 + threadIdx.x, first = group * a.beams;
    const int lane = threadIdx.x & 63;
    int64_t slot = -1, parent = lane;
    if (lane < a.beams) {
        parent = a.parents.at(first + lane);
        slot = a.slots.p ? a.slots.at(first + lane) : first + lane;
    }
    if (slot < 0 || slot >= a.pool) slot = -1;
    const int source = parent >= 0 && parent < a.beams ? (int)parent : lane, low = (int)slot, high = (int)(slot >> 32);
    // (no thread leaves before: what a lane hands round it has to have formed)
    const bool mine = at < a.pieces;
    P *states = static_cast<P *>(a.states);
    auto row = [&](int w) {
        return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane(high, w) << 32 | (uint32_t)__builtin_amdgcn_readlane(low, w));
    };
    // every load is issued before the first store; a beam that moves nothing has its wave read one piece of the pool's beginning
    P x[WMAX];
    int64_t to[WMAX];
#pragma unroll
    for (int w = 0; w < WMAX; ++w) {
        const int from = __builtin_amdgcn_readlane(source, w);
        const int64_t s = row(from), d = row(w);
        const bool moves = w < a.beams && from != w && s >= 0 && d >= 0;
        to[w] = moves ? d : -1;
        x[w] = states[moves && mine ? s * a.pieces + at : 0];
    }
#pragma unroll
    for (int w = 0; w < WMAX; ++w)
        if (mine && to[w] >= 0) states[to[w] * a.pieces + at] = x[w];
}
template <typename P> int launch_reorder(hipStream_t stream, const ReorderArgs &a, int64_t groups)
{
    const dim3 grid(a.blocks * groups);
    if (a.beams <= 4) reorder_states_kernel<P, 4><<<grid, 256, 0, stream>>>(a);
    else if (a.beams <= 16) reorder_states_kernel<P, 16><<<grid, 256, 0, stream>>>(a);
    else if constexpr (sizeof(P) < 16) reorder_states_kernel<P, 64><<<grid, 256, 0, stream>>>(a);
    else return GLA_ERR_SHAPE;                   // (64 pieces of 16 bytes a thread do not fit its registers: the caller takes smaller ones)
    return launch_status();
}

int64_t bytes_of(gla_dtype d) { return d == GLA_BF16 ? 2 : 4; }
bool dtype_ok(gla_dtype d) { return d == GLA_F32 || d == GLA_BF16; }

}  // namespace
}  // namespace gla

using namespace gla;

extern "C" int gla_reorder_states(void *stream, int64_t pool, int64_t groups, int64_t beams, int64_t row_bytes, int wide_indices,
                                  const void *parents, const void *slots, void *states)
{
    if (!parents || !states) return GLA_ERR_NULL;
    if (pool < 1 || groups < 1 || beams < 1 || beams > GLA_MOST_BEAMS || row_bytes < 1) return GLA_ERR_SHAPE;
    if (!slots && groups * beams > pool) return GLA_ERR_SHAPE;
    const uintptr_t index = wide_indices ? 7 : 3;
    if ((reinterpret_cast<uintptr_t>(parents) & index) || (reinterpret_cast<uintptr_t>(slots) & index)) return GLA_ERR_ALIGN;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const uintptr_t place = reinterpret_cast<uintptr_t>(states) | (uintptr_t)row_bytes;
    ReorderArgs a{pool, beams, 0, 0, states, {parents, wide_indices}, {slots, wide_indices}};
    // 16 bytes of up to 16 rows in a thread's registers, 4 bytes of more
    const int64_t piece = place % 16 == 0 && beams <= 16 ? 16 : place % 4 == 0 ? 4 : 1;
    a.pieces = row_bytes / piece;
    a.blocks = (a.pieces + 255) / 256;
    if (a.blocks >= ((int64_t)1 << 31) || groups >= ((int64_t)1 << 31) || a.blocks * groups >= ((int64_t)1 << 31)) return GLA_ERR_SHAPE;
    return piece == 16 ? launch_reorder<u32x4>(s, a, groups) : piece == 4 ? launch_reorder<uint32_t>(s, a, groups) : launch_reorder<uint8_t>(s, a, groups);
}

namespace gla {
namespace {

// Strides: batch and head strides of log_decay, beta (delta), value, key and query.
template <bool DELTA>
int step(void *stream, int64_t pool, int64_t B, int64_t H, int64_t HK, int64_t DK, int64_t DV, int64_t beams, gla_dtype dtype,
         gla_dtype state_dtype, int wide_indices, const int64_t *strides, const float *log_decay, const float *beta, const void *value,
         const void *key, const void *query, const void *slots, const void *parents, void *states, void *out)
{
    if (!log_decay || (DELTA && !beta) || !value || !key || !query || !states || !out || (beams > 0 && !parents)) return GLA_ERR_NULL;
    if (pool < 1 || B < 1 || H < 1 || HK < 1 || DK < 1 || DV < 1 || beams < 0 || H % HK || DK % 16 || DV % 16 || DK > 256 || DV > 256)
        return GLA_ERR_SHAPE;
    if (B * H >= ((int64_t)1 << 31) || (!slots && B > pool) || (beams > 0 && (B % beams || beams > GLA_MOST_BEAMS))) return GLA_ERR_SHAPE;
    if (!dtype_ok(dtype) || !dtype_ok(state_dtype)) return GLA_ERR_DTYPE;
    StepArgs a{pool, B, H, HK, DK, DV, beams, states, log_decay, beta, H, 1, H, 1, value, key, query,
               H * DV, DV, HK * DK, DK, HK * DK, DK, {slots, wide_indices}, {parents, wide_indices}, out};
    if (strides) {
        int64_t *all[10] = {&a.gates_b, &a.gates_h, &a.beta_b, &a.beta_h, &a.value_b, &a.value_h, &a.key_b, &a.key_h, &a.query_b, &a.query_h};
        for (int i = 0, from = 0; i < 10; ++i)
            if (DELTA || (i != 2 && i != 3)) *all[i] = strides[from++];
    }
    const int64_t piece = 16 / bytes_of(dtype);
    for (int64_t x : {a.value_b, a.value_h, a.key_b, a.key_h, a.query_b, a.query_h})
        if (x % piece) return GLA_ERR_ALIGN;
    for (const void *x : {value, key, query, static_cast<const void *>(states), static_cast<const void *>(out)})
        if (!aligned16(x)) return GLA_ERR_ALIGN;
    const uintptr_t index = wide_indices ? 7 : 3;
    if ((reinterpret_cast<uintptr_t>(slots) & index) || (reinterpret_cast<uintptr_t>(parents) & index) ||
        (reinterpret_cast<uintptr_t>(log_decay) & 3) || (reinterpret_cast<uintptr_t>(beta) & 3))
        return GLA_ERR_ALIGN;
    if (beams > waves_of_beams((int)DK)) {
        // more beams than a workgroup has waves for take the reordering as a pass of its own, in pieces of 4 bytes (128 rows of 16 heads of 64 x 64
        // bfloat16: 25 us in searches of 32 beams, 8.4 of 16)
        const int rc = gla_reorder_states(stream, pool, B / beams, beams, H * DK * DV * bytes_of(state_dtype), wide_indices, parents,
                                          slots, states);
        if (rc) return rc;
        a.beams = 0;
    }
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == GLA_BF16) return state_dtype == GLA_BF16 ? dispatch_step<__bf16, __bf16, DELTA>(s, a) : dispatch_step<__bf16, float, DELTA>(s, a);
    return state_dtype == GLA_BF16 ? dispatch_step<float, __bf16, DELTA>(s, a) : dispatch_step<float, float, DELTA>(s, a);
}

}  // namespace
}  // namespace gla

extern "C" int gla_decay_step(void *stream, int64_t pool, int64_t B, int64_t H, int64_t HK, int64_t DK, int64_t DV, int64_t beams,
                              gla_dtype dtype, gla_dtype state_dtype, int wide_indices, const int64_t *strides, const float *log_decay,
                              const void *value, const void *key, const void *query, const void *slots, const void *parents,
                              void *states, void *out)
{
    return step<false>(stream, pool, B, H, HK, DK, DV, beams, dtype, state_dtype, wide_indices, strides, log_decay, nullptr, value, key, query,
                       slots, parents, states, out);
}

extern "C" int gla_delta_step(void *stream, int64_t pool, int64_t B, int64_t H, int64_t HK, int64_t DK, int64_t DV, int64_t beams,
                              gla_dtype dtype, gla_dtype state_dtype, int wide_indices, const int64_t *strides, const float *log_decay,
                              const float *beta, const void *value, const void *key, const void *query, const void *slots,
                              const void *parents, void *states, void *out)
{
    return step<true>(stream, pool, B, H, HK, DK, DV, beams, dtype, state_dtype, wide_indices, strides, log_decay, beta, value, key, query,
                      slots, parents, states, out);
}
