// Beam search's selection: the best continuations of a search's beams over the vocabulary.
//
// A candidate's score is its beam's score plus log softmax of its logit.  Within a beam the order is that of the logits, so the
// logits are read once: every workgroup takes a stretch of a row, leaves its largest value, its sum of exponentials and its
// `num` largest logits; a workgroup a search then joins the sums, scores what is left and takes the best `num` of all beams.
// Everything compared is one 64-bit key, the value above and the inverted place below: keys are unique and equal values come in
// the order of their places.  16 searches of 8 beams over 131072 bfloat16 logits: 14.5 us for the stretches' 33.5 MB and 6.5 for the join, a chain of
// dependent steps.  All 1024 stretches are on the machine at once and in the same phase, first loads, then 64 exponentials a thread and the
// bound, so neither hides the other (2.3 TB/s).
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
// A logit; -inf where it is not a number.  The maximum of a signalling NaN and a number is a quiet NaN, only that of a quiet one the number, and the
// compiler takes every float that comes from a bfloat16 for quiet: so the first instruction is written out.  (A comparison instead cost a
// register too many where rows do not begin on 16 bytes: 16 searches of 8 beams over 131071 bfloat16 logits 32.3 us, this 29.9, and 30 with neither.)
__device__ __forceinline__ float number(float x)
{
    asm("v_max_f32 %0, %0, %0\n\tv_max_f32 %0, 0xff800000, %0" : "+v"(x));
    return x;
}
constexpr int kThreads = 256, kHeld = 4;

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

// The largest `num` of a workgroup's keys, in order, without a round for each.  Every thread names its own largest; in a wave the
// num-th of 64 such is a bound that num keys reach, and the highest of the waves' bounds still is one.  What reaches it is collected (of
// N keys a thread at most N * num a wave, keys being unique) and ranked by counting.  Comparing all names costs 64 steps, the collected
// ones a few more than num; taking the maximum num times took four times as long at num = 8.
template <int WAVES> struct SelectLds {
    u64 names[WAVES][64];
    u64 bound[WAVES];
    int count;
};
// The bound, in every thread (below 64: num keys are not there), and the largest key of all in `top`; num is at most 64.  Has the
// workgroup's threads meet twice.
template <int WAVES> __device__ __forceinline__ u64 select_bound(SelectLds<WAVES> &l, u64 best, int num, u64 &top)
{
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if (best == 0) best = 63 - lane;             // a thread without a key: a name below all keys, and no other thread's
    l.names[w][lane] = best;
    if (threadIdx.x == 0) l.count = 0;
    __syncthreads();
    int above = 0;
#pragma unroll 16
    for (int i = 0; i < 64; ++i) above += l.names[w][i] > best;
    if (above == num - 1) l.bound[w] = best;
    if (above == 0) l.names[w][0] = best;        // (each wave has read its own names: its lanes are in step)
    __syncthreads();
    u64 bound = l.bound[0];
    top = l.names[0][0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) {
        bound = l.bound[i] > bound ? l.bound[i] : bound;
        top = l.names[i][0] > top ? l.names[i][0] : top;
    }
    return bound;
}

// EACH values a thread, in pieces of 16 bytes, which rows that do not begin on 16 bytes read one by one: the sums come out the same.
template <typename T, int EACH, bool PIECES>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(PIECES ? 4 : 2))) void beam_stretch_kernel(const SelectArgs a)
{
    constexpr int kWaves = kThreads / 64, VEC = 16 / sizeof(T);
    __shared__ SelectLds<kWaves> lds;
    __shared__ float parts[kWaves];
    extern __shared__ u64 collected[];           // EACH * per of each wave
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.y, split = blockIdx.x, first = split * (kThreads * EACH);
    if (a.finished && a.finished[row]) return;   // its one candidate is made later
    const T *x = static_cast<const T *>(a.logits) + row * a.row + first;
    const int there = (int)min(a.vocab - first, (int64_t)(kThreads * EACH));
    // Every load is issued before the first is used, and none is under a condition (a wait for memory would follow each): what lies behind the
    // row's end reads its last values and counts as -inf.
    T raw[EACH];
#pragma unroll
    for (int i = 0; i < EACH; i += VEC) {
        const int at = (i / VEC) * (kThreads * VEC) + tid * VEC;
        if constexpr (PIECES) {
            typedef T Piece __attribute__((ext_vector_type(VEC)));
            const Piece t = *reinterpret_cast<const Piece *>(x + min(at, there - VEC));      // (VEC divides what is there)
#pragma unroll
            for (int e = 0; e < VEC; ++e) raw[i + e] = t[e];
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) raw[i + e] = x[min(at + e, there - 1)];
        }
    }
    float v[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) v[i] = number((float)raw[i]);
    if (there < kThreads * EACH)
#pragma unroll
        for (int i = 0; i < EACH; ++i)
            if ((i / VEC) * (kThreads * VEC) + tid * VEC + i % VEC >= there) v[i] = -INFINITY;
    auto place = [&](int i) { return (i / VEC) * (kThreads * VEC) + tid * VEC + i % VEC; };
    // of equal values the first: a thread's places ascend
    float most = v[0];
    int which = place(0);
#pragma unroll
    for (int i = 1; i < EACH; ++i)
        if (v[i] > most) {
            most = v[i];
            which = place(i);
        }
    u64 top;
    const u64 bound = select_bound<kWaves>(lds, tid * VEC < there ? key_of(most, (uint32_t)(first + which)) : 0, a.per, top);
    const float least = bound < 64 ? -INFINITY : value_of((uint32_t)(bound >> 32));
    most = value_of((uint32_t)(top >> 32));
    // The sum in two levels: a thread's, then the threads' in a fixed order.  What reaches the bound is marked beside it (few do, but where the stretch
    // has fewer than `per`) and read again: a branch for each value took a third of the kernel's instructions.
    float sum = 0.f;
    constexpr int kWord = EACH < 32 ? EACH : 32;
    uint32_t marks[EACH / kWord];
#pragma unroll
    for (int j = 0; j < EACH / kWord; ++j) {
        marks[j] = 0;
#pragma unroll
        for (int i = j * kWord; i < (j + 1) * kWord; ++i) {
            sum += most == -INFINITY ? 0.f : fast_exp2((v[i] - most) * kLog2e);
            marks[j] = 2 * marks[j] + (v[i] >= least);
        }
    }
#pragma unroll
    for (int j = 0; j < EACH / kWord; ++j)
        for (uint32_t left = marks[j]; left;) {
            const int bit = 31 - __clz((int)left), at = place((j + 1) * kWord - 1 - bit);
            left ^= 1u << bit;
            if (at >= there) continue;
            const u64 key = key_of(number((float)x[at]), (uint32_t)(first + at));
            if (key >= bound) collected[atomicAdd(&lds.count, 1)] = key;
        }
#pragma unroll
    for (int m = 1; m < 64; m *= 2) sum += shfl_xor_f32(sum, m);
    if ((tid & 63) == 0) parts[tid >> 6] = sum;
    __syncthreads();
    const int count = lds.count;
    u64 *kept = a.kept + (row * a.splits + split) * a.per;
    for (int i = tid; i < count; i += kThreads) {
        const u64 key = collected[i];
        int above = 0;
        for (int j = 0; j < count; ++j) above += collected[j] > key;
        if (above < a.per) kept[above] = key;
    }
    for (int i = count + tid; i < a.per; i += kThreads) kept[i] = 0;
    if (tid == 0) {
        float s = parts[0];
#pragma unroll
        for (int i = 1; i < kWaves; ++i) s += parts[i];
        a.most[row * a.splits + split] = most;
        a.sums[row * a.splits + split] = s;
    }
}

// One workgroup a search.  1024 threads hold 4096 candidates; up to 1024 take a quarter of them, whose waves need not share a SIMD's time where all
// compare names (1 search of 4 beams over 32000, both kernels: 8.9 us instead of 10.5; 32 of them 12.4 instead of 14.0; 8192 candidates with a quarter of them 38.8
// instead of 19.2).
template <int THREADS> __global__ __launch_bounds__(THREADS) void beam_join_kernel(const SelectArgs a)
{
    constexpr int kWaves = THREADS / 64, kRoom = 2048;
    __shared__ SelectLds<kWaves> lds;
    __shared__ u64 collected[kRoom];
    __shared__ float lse[GLA_MOST_BEAMS], beam_score[GLA_MOST_BEAMS];
    __shared__ int ended[GLA_MOST_BEAMS];
    const int tid = threadIdx.x, lane = tid & 63;
    const int64_t group = blockIdx.x;
    // What is read does not wait for what was read: the first candidates, the beams and the stretches' sums are all on their way at once.
    const unsigned of_beam = (unsigned)(a.splits * a.per), total = (unsigned)a.beams * of_beam;
    const u64 *kept = a.kept + group * total;
    u64 held[kHeld];
#pragma unroll
    for (int j = 0; j < kHeld; ++j) held[j] = tid + j * THREADS < total ? kept[tid + j * THREADS] : 0;
    if (tid < a.beams) {
        beam_score[tid] = a.scores[group * a.beams + tid];
        ended[tid] = a.finished && a.finished[group * a.beams + tid];
    }
    for (int w = tid >> 6; w < a.beams; w += kWaves) {
        const int64_t row = (group * a.beams + w) * a.splits;
        float most = -INFINITY, sum = 0.f;       // (of a beam that has ended, whatever lies there: not used)
        for (int i = lane; i < a.splits; i += 64) {
            const float m = a.most[row + i], s = a.sums[row + i], higher = fmaxf(most, m);
            if (higher != -INFINITY) {
                sum = sum * expf(most - higher) + s * expf(m - higher);
                most = higher;
            }
            if (m != m || s != s) sum = NAN;
        }
        float all = most;
#pragma unroll
        for (int m = 1; m < 64; m *= 2) all = fmaxf(all, shfl_xor_f32(all, m));
        sum = most == -INFINITY && sum == 0.f ? 0.f : sum * expf(most - all);
#pragma unroll
        for (int m = 1; m < 64; m *= 2) sum += shfl_xor_f32(sum, m);
        if (lane == 0) lse[w] = all + logf(sum);
    }
    __syncthreads();
    // candidate i as a key: its score above, its place among beams x vocabulary below
    auto candidate = [&](unsigned i, u64 k) -> u64 {
        const unsigned w = i / of_beam, n = i % of_beam;
        float score;
        uint32_t token;
        if (ended[w]) {
            // the end again at the score that it has, and the others without a chance, in order
            if (n >= (unsigned)a.per) return 0;
            token = (uint32_t)(n == 0 ? a.eos : n <= a.eos ? n - 1 : n);
            score = n == 0 ? beam_score[w] : -INFINITY;
        } else {
            if (!k) return 0;
            token = ~(uint32_t)k;
            score = beam_score[w] + (value_of((uint32_t)(k >> 32)) - lse[w]);
        }
        if (score != score) score = -INFINITY;
        return key_of(score, (uint32_t)(w * a.vocab) + token);
    };
    auto put = [&](int n, u64 key) {
        const uint32_t place = ~(uint32_t)key;
        a.out_scores[group * a.num + n] = value_of((uint32_t)(key >> 32));
        a.out_parents[group * a.num + n] = place / (uint32_t)a.vocab;
        a.out_tokens[group * a.num + n] = place % (uint32_t)a.vocab;
    };
    u64 best = 0;
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
        held[j] = tid + j * THREADS < total ? candidate(tid + j * THREADS, held[j]) : 0;
        best = held[j] > best ? held[j] : best;
    }
    for (unsigned i = tid + kHeld * THREADS; i < total; i += THREADS) {
        const u64 k = candidate(i, kept[i]);
        best = k > best ? k : best;
    }
    u64 top;
    const u64 bound = select_bound<kWaves>(lds, best, a.num, top);
    auto collect = [&](u64 k) {
        if (k < bound || k == 0) return;
        const int at = atomicAdd(&lds.count, 1);
        if (at < kRoom) collected[at] = k;
    };
#pragma unroll
    for (int j = 0; j < kHeld; ++j) collect(held[j]);
    for (unsigned i = tid + kHeld * THREADS; i < total; i += THREADS) collect(candidate(i, kept[i]));
    __syncthreads();
    const int count = lds.count;
    if (count <= kRoom) {
        for (int i = tid; i < count; i += THREADS) {
            const u64 key = collected[i];
            int above = 0;
            for (int j = 0; j < count; ++j) above += collected[j] > key;
            if (above < a.num) put(above, key);
        }
        return;
    }
    // more than there is room for (many candidates of few threads): one after the other, each round over all of them.  64 beams over 131072 tokens at
    // num = 64 get here with some 4300 of 32768, since the bound is the least of a wave's names then: 1190 us; num = 32 does not: 34 us for 32 beams.
    for (int n = 0; n < a.num; ++n) {
        u64 next = 0;
        for (unsigned i = tid; i < total; i += THREADS) {
            const u64 k = candidate(i, kept[i]);
            next = (n == 0 || k < top) && k > next ? k : next;
        }
        __syncthreads();
        select_bound<kWaves>(lds, next, 1, top);
        if (tid == 0) put(n, top);
    }
}

int64_t per_of(int64_t vocab, int64_t num) { return num < vocab ? num : vocab; }
// Values a thread: 16, and 64 where that still makes enough workgroups, or where 16 left a search's join more than its threads hold.
// Finding a stretch's bound takes as long as reading 50 values a thread: 16 searches of 8 beams over 131072 tokens take 25.6 us with 16 and 20.4 with 64,
// and one of 16 beams 19.2 (8192 candidates for the join) and 15.8; one of 4 over 32000 has 32 workgroups with 16 and 8 with 64: 8.9 and 11.3.
constexpr int kFew = 16, kMany = 64;
int64_t stretches(int64_t vocab, int each) { return (vocab + (int64_t)kThreads * each - 1) / ((int64_t)kThreads * each); }
int each_of(int64_t groups, int64_t beams, int64_t vocab, int64_t num)
{
    return groups * beams * vocab >= (int64_t)512 * kThreads * kMany || beams * stretches(vocab, kFew) * per_of(vocab, num) > kHeld * 1024 ? kMany : kFew;
}
int64_t splits_of(int64_t groups, int64_t beams, int64_t vocab, int64_t num) { return stretches(vocab, each_of(groups, beams, vocab, num)); }

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
    const int64_t stretches = groups * beams * splits_of(groups, beams, vocab, num);
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
    a.splits = splits_of(groups, beams, vocab, num);
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
    const bool many = each_of(groups, beams, vocab, num) == kMany;
    const auto kernel = dtype == GLA_BF16 ? pieces ? many ? beam_stretch_kernel<__bf16, kMany, true> : beam_stretch_kernel<__bf16, kFew, true>
                                                   : many ? beam_stretch_kernel<__bf16, kMany, false> : beam_stretch_kernel<__bf16, kFew, false>
                                          : pieces ? many ? beam_stretch_kernel<float, kMany, true> : beam_stretch_kernel<float, kFew, true>
                                                   : many ? beam_stretch_kernel<float, kMany, false> : beam_stretch_kernel<float, kFew, false>;
    const size_t room = (size_t)kThreads / 64 * each_of(groups, beams, vocab, num) * a.per * sizeof(u64);
    static LdsGrant grants[8];
    const size_t most = many ? (size_t)kThreads / 64 * kMany * GLA_MOST_CANDIDATES * sizeof(u64) : room;      // granted once, for any num
    if (int e = allow_lds(grants[(dtype == GLA_BF16) * 4 + pieces * 2 + many], reinterpret_cast<const void *>(kernel), most)) return e;
    kernel<<<grid, kThreads, room, s>>>(a);
    if (int e = launch_status()) return e;
    if (beams * a.splits * a.per <= kHeld * 256) beam_join_kernel<256><<<groups, 256, 0, s>>>(a);
    else beam_join_kernel<1024><<<groups, 1024, 0, s>>>(a);
    return launch_status();
}
