// Beam search's selection: the best continuations of a search's beams over the vocabulary.
//
// A candidate's score is its beam's score plus log softmax of its logit.  Within a beam the order is that of the logits, so the
// logits are read once: every workgroup takes a stretch of a row, leaves its largest value, its sum of exponentials and its
// `num` largest logits; a workgroup a search then joins the sums, scores what is left and takes the best `num` of all beams.
// Everything compared is one 64-bit key, the value above and the inverted place below: keys are unique and equal values come in
// the order of their places.  Bound by reading the logits.
#include "gla_common.hpp"

namespace gla {
namespace {

typedef unsigned long long u64;

// Floats as unsigned numbers of the same order; -inf is 0x007fffff, so 0 is below every value.
__device__ __forceinline__ uint32_t ordered(float x)
{
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o)
{
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ u64 key_of(float x, uint32_t place)
{
    return ((u64)ordered(x + 0.f) << 32) | (uint32_t)~place;      // (-0 + 0 is 0: the two are equal)
}
__device__ __forceinline__ u64 shfl_xor_u64(u64 x, int m)
{
    return ((u64)(uint32_t)__shfl_xor((int)(x >> 32), m, 64) << 32) | (uint32_t)__shfl_xor((int)x, m, 64);
}
__device__ __forceinline__ u64 wave_max(u64 x)
{
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
        const u64 y = shfl_xor_u64(x, m);
        x = x > y ? x : y;
    }
    return x;
}

constexpr int kThreads = 256, kWaves = kThreads / 64;

struct SelectArgs {
    int64_t groups, beams, vocab, row;           // row: elements from a beam's logits to the next one's
    int num, per;                                // candidates in all; of a beam: min(num, vocab)
    int64_t splits;
    const void *logits;
    const float *scores;
    const uint8_t *finished;
    int64_t eos;
    float *most, *sums;                          // [rows][splits]
    u64 *kept;                                   // [rows][splits][per]
    float *out_scores;
    int64_t *out_parents, *out_tokens;
};

// The block's largest key, in every thread; `slots` has kWaves places of LDS.
__device__ __forceinline__ u64 block_max(u64 x, u64 *slots)
{
    x = wave_max(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = x;
    __syncthreads();
    u64 best = slots[0];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) best = slots[i] > best ? slots[i] : best;
    return best;
}

// EACH values a thread, in pieces of VEC side by side.  VEC = 1 takes rows that do not begin on 16 bytes.
template <typename T, int EACH, int VEC>
__global__ __launch_bounds__(kThreads) void beam_stretch_kernel(const SelectArgs a)
{
    __shared__ u64 slots[kWaves];
    __shared__ float parts[kWaves];
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.y, split = blockIdx.x, first = split * (kThreads * EACH);
    if (a.finished && a.finished[row]) return;   // its one candidate is made later
    const T *x = static_cast<const T *>(a.logits) + row * a.row;
    u64 key[EACH];
    float v[EACH];
#pragma unroll
    for (int i = 0; i < EACH; i += VEC) {
        const int64_t at = first + (int64_t)(i / VEC) * (kThreads * VEC) + tid * VEC;
        float t[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) t[e] = 0.f;
        if (VEC > 1 ? at < a.vocab : at < a.vocab) load_vec<T, VEC>(x + at, t);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            v[i + e] = t[e] != t[e] ? -INFINITY : t[e];
            key[i + e] = at < a.vocab ? key_of(v[i + e], (uint32_t)(at + e)) : 0;
            if (at >= a.vocab) v[i + e] = -INFINITY;
        }
    }
    u64 best = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) best = key[i] > best ? key[i] : best;
    u64 top = block_max(best, slots);
    const float most = value_of((uint32_t)(top >> 32));
    // the sum in two levels: a thread's, then the threads' in a fixed order
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < EACH; ++i) sum += most == -INFINITY ? 0.f : fast_exp2((v[i] - most) * kLog2e);
#pragma unroll
    for (int m = 1; m < 64; m *= 2) sum += shfl_xor_f32(sum, m);
    if ((tid & 63) == 0) parts[tid >> 6] = sum;
    u64 *kept = a.kept + (row * a.splits + split) * a.per;
    for (int n = 0; n < a.per; ++n) {
        if (tid == 0) kept[n] = top;
        if (n + 1 == a.per) break;
        if (best == top && top) {
            u64 next = 0;
#pragma unroll
            for (int i = 0; i < EACH; ++i) next = key[i] < top && key[i] > next ? key[i] : next;
            best = next;
        }
        top = block_max(best, slots);
    }
    __syncthreads();
    if (tid == 0) {
        float s = parts[0];
#pragma unroll
        for (int i = 1; i < kWaves; ++i) s += parts[i];
        a.most[row * a.splits + split] = most;
        a.sums[row * a.splits + split] = s;
    }
}

// One workgroup a search.
__global__ __launch_bounds__(kThreads) void beam_join_kernel(const SelectArgs a)
{
    __shared__ u64 slots[kWaves];
    __shared__ float lse[GLA_MOST_BEAMS];
    const int tid = threadIdx.x, lane = tid & 63;
    const int64_t group = blockIdx.x;
    for (int64_t w = tid >> 6; w < a.beams; w += kWaves) {
        const int64_t row = group * a.beams + w;
        if (a.finished && a.finished[row]) continue;
        float most = -INFINITY;
        for (int64_t i = lane; i < a.splits; i += 64) most = fmaxf(most, a.most[row * a.splits + i]);
#pragma unroll
        for (int m = 1; m < 64; m *= 2) most = fmaxf(most, shfl_xor_f32(most, m));
        float sum = 0.f;
        for (int64_t i = lane; i < a.splits; i += 64) {
            const float m = a.most[row * a.splits + i];
            if (m != -INFINITY) sum += a.sums[row * a.splits + i] * expf(m - most);
        }
#pragma unroll
        for (int m = 1; m < 64; m *= 2) sum += shfl_xor_f32(sum, m);
        if (lane == 0) lse[w] = most + logf(sum);
    }
    __syncthreads();
    const int64_t of_beam = a.splits * a.per, total = a.beams * of_beam;
    // candidate i as a key: its score above, its place among beams x vocabulary below
    auto candidate = [&](int64_t i) -> u64 {
        const int64_t w = i / of_beam, n = i % of_beam, row = group * a.beams + w;
        float score;
        uint32_t token;
        if (a.finished && a.finished[row]) {
            // the end again at the score that it has, and the others without a chance, in order
            if (n >= a.per) return 0;
            token = (uint32_t)(n == 0 ? a.eos : n <= a.eos ? n - 1 : n);
            score = n == 0 ? a.scores[row] : -INFINITY;
        } else {
            const u64 k = a.kept[row * of_beam + n];
            if (!k) return 0;
            token = ~(uint32_t)k;
            score = a.scores[row] + (value_of((uint32_t)(k >> 32)) - lse[w]);
        }
        if (score != score) score = -INFINITY;
        return key_of(score, (uint32_t)(w * a.vocab) + token);
    };
    u64 best = 0;
    for (int64_t i = tid; i < total; i += kThreads) {
        const u64 k = candidate(i);
        best = k > best ? k : best;
    }
    for (int n = 0; n < a.num; ++n) {
        const u64 top = block_max(best, slots);
        if (tid == 0) {
            const uint32_t place = ~(uint32_t)top;
            a.out_scores[group * a.num + n] = value_of((uint32_t)(top >> 32));
            a.out_parents[group * a.num + n] = place / a.vocab;
            a.out_tokens[group * a.num + n] = place % a.vocab;
        }
        if (best == top) {
            u64 next = 0;
            for (int64_t i = tid; i < total; i += kThreads) {
                const u64 k = candidate(i);
                next = k < top && k > next ? k : next;
            }
            best = next;
        }
    }
}

constexpr int kEach = 16;
int64_t splits_of(int64_t vocab) { return (vocab + kThreads * kEach - 1) / (kThreads * kEach); }
int64_t per_of(int64_t vocab, int64_t num) { return num < vocab ? num : vocab; }

bool sizes_ok(int64_t groups, int64_t beams, int64_t vocab, int64_t num)
{
    return groups >= 1 && beams >= 1 && beams <= GLA_MOST_BEAMS && vocab >= 1 && vocab < ((int64_t)1 << 31) / beams && num >= 1 &&
           num <= GLA_MOST_CANDIDATES && num <= beams * vocab && groups < ((int64_t)1 << 31) && groups * beams <= 65535;
}

}  // namespace
}  // namespace gla

using namespace gla;

extern "C" size_t gla_beam_select_workspace_bytes(int64_t groups, int64_t beams, int64_t vocab, int64_t num)
{
    if (!sizes_ok(groups, beams, vocab, num)) return 0;
    const int64_t stretches = groups * beams * splits_of(vocab);
    return (size_t)(stretches * (per_of(vocab, num) * 8 + 8));
}

extern "C" int gla_beam_select(void *stream, int64_t groups, int64_t beams, int64_t vocab, int64_t num, gla_dtype dtype, int64_t row,
                               const void *logits, const float *scores, const void *finished, int64_t eos, float *out_scores,
                               int64_t *out_parents, int64_t *out_tokens, void *workspace, size_t workspace_bytes)
{
    if (!logits || !scores || !out_scores || !out_parents || !out_tokens) return GLA_ERR_NULL;
    if (!sizes_ok(groups, beams, vocab, num) || row < vocab || (finished && (eos < 0 || eos >= vocab))) return GLA_ERR_SHAPE;
    if (dtype != GLA_F32 && dtype != GLA_BF16) return GLA_ERR_DTYPE;
    const size_t need = gla_beam_select_workspace_bytes(groups, beams, vocab, num);
    if (!workspace || workspace_bytes < need) return GLA_ERR_WORKSPACE;
    const int size = dtype == GLA_BF16 ? 2 : 4;
    if (!aligned16(workspace) || (reinterpret_cast<uintptr_t>(logits) % size) || (reinterpret_cast<uintptr_t>(scores) & 3) ||
        (reinterpret_cast<uintptr_t>(out_scores) & 3) || (reinterpret_cast<uintptr_t>(out_parents) & 7) ||
        (reinterpret_cast<uintptr_t>(out_tokens) & 7))
        return GLA_ERR_ALIGN;
    SelectArgs a{};
    a.groups = groups;
    a.beams = beams;
    a.vocab = vocab;
    a.row = row;
    a.num = (int)num;
    a.per = (int)per_of(vocab, num);
    a.splits = splits_of(vocab);
    a.logits = logits;
    a.scores = scores;
    a.finished = static_cast<const uint8_t *>(finished);
    a.eos = eos;
    const int64_t stretches = groups * beams * a.splits;
    a.kept = static_cast<u64 *>(workspace);
    a.most = reinterpret_cast<float *>(a.kept + stretches * a.per);
    a.sums = a.most + stretches;
    a.out_scores = out_scores;
    a.out_parents = out_parents;
    a.out_tokens = out_tokens;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const dim3 grid(a.splits, groups * beams);
    const bool pieces = aligned16(logits) && row * size % 16 == 0 && vocab * size % 16 == 0;
    if (dtype == GLA_BF16) {
        if (pieces) beam_stretch_kernel<__bf16, kEach, 8><<<grid, kThreads, 0, s>>>(a);
        else beam_stretch_kernel<__bf16, kEach, 1><<<grid, kThreads, 0, s>>>(a);
    } else {
        if (pieces) beam_stretch_kernel<float, kEach, 4><<<grid, kThreads, 0, s>>>(a);
        else beam_stretch_kernel<float, kEach, 1><<<grid, kThreads, 0, s>>>(a);
    }
    if (int e = launch_status()) return e;
    beam_join_kernel<<<groups, kThreads, 0, s>>>(a);
    return launch_status();
}
