// Log probabilities of given tokens, the entropy of the distribution and its largest alternatives, and the logits' gradient.
//
// One workgroup takes a row of logits and reads it once: every thread keeps the largest value m that it has seen, the sum of e^{x - m} and of
// (x - m) e^{x - m}, rescaled where m grows, and the threads' three numbers are joined at the end:
//       log p_i = (x_i - m) - log s,    H = log s - t / s.
// Bound by the read: 4096 rows of 32000 in 16 bits 52 to 69 us (5.0 to 3.8 TB/s, by what the last-level cache holds of them); 500 rows of 131072 28 us (4.6
// TB/s), and 34 with 20 alternatives.  What comes near it are the exponentials (four issue slots of a value's eleven).
//
// The alternatives need no second pass over the row.  The threads are 64 groups, each with a largest value; the top-th largest of the 64
// is reached by `top` values at least, and whatever reaches it lies in the stretches of threads whose own largest value does: they alone are read
// again, by whole waves (24 threads at 20 alternatives of a row in no order: 64 ln(64 / 44)).  Equal values are common in 16 bits, and all of them are
// taken along; if they are more than there is room for, the row is searched once for each alternative.
#include "gla_common.hpp"

namespace gla {
namespace {

typedef unsigned long long u64;

constexpr int kMostTop = GLA_MOST_ALTERNATIVES;
constexpr int64_t kMostGroups = (int64_t)1 << 22;  // workgroups of a launch: it counts its threads in 32 bits
constexpr int kRoom = 1024;                      // threads, or values, that reach a bound

struct LogprobArgs {
    int64_t vocab, row;                          // row: elements from one row of logits to the next
    int top, wide;
    const void *logits, *tokens;
    float *given, *entropy, *stats, *near;       // stats: m and log s of each row, or NULL
    int64_t *index;
};
struct LogprobGradArgs {
    int64_t vocab, row, grad_row, segments;
    int wide;
    const void *logits, *tokens;
    const float *stats, *entropy, *dgiven, *dentropy;
    void *dlogits;
};

__device__ __forceinline__ int64_t token_at(const void *tokens, int wide, int64_t i)
{
    return wide ? static_cast<const int64_t *>(tokens)[i] : (int64_t) static_cast<const int32_t *>(tokens)[i];
}
// The value above and the inverted place below: of equal values the first is the largest key.  What is not a number counts as -inf.
__device__ __forceinline__ u64 key_of(float x, int64_t place)
{
    if (!(x == x)) x = -INFINITY;
    x += 0.f;                                    // (-0 + 0 is 0: the two are equal)
    const uint32_t u = __float_as_uint(x);
    return ((u64)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32) | (uint32_t)~(uint32_t)place;
}
__device__ __forceinline__ float value_of(u64 key)
{
    const uint32_t o = (uint32_t)(key >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

// A row as pieces of 16 bytes, and what lies before the first and behind the last.
template <typename T> struct RowPieces {
    static constexpr int VEC = 16 / sizeof(T);
    typedef T Piece __attribute__((ext_vector_type(VEC)));
    const T *x;
    int64_t head, pieces, behind, vocab;
    __device__ __forceinline__ RowPieces(const T *x, int64_t vocab) : x(x), vocab(vocab)
    {
        head = (int64_t)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int64_t)sizeof(T);
        if (head > vocab) head = vocab;
        pieces = (vocab - head) / VEC;
        behind = head + pieces * VEC;
    }
    __device__ __forceinline__ const Piece *at(int64_t p) const { return reinterpret_cast<const Piece *>(x + head) + p; }
    __device__ __forceinline__ int64_t place(int64_t p) const { return head + p * VEC; }
    // the place of loose value i, of `loose` many
    __device__ __forceinline__ int loose() const { return (int)(head + vocab - behind); }
    __device__ __forceinline__ int64_t loose_place(int i) const { return i < head ? i : behind + (i - head); }
};

// The running maximum and sums; all sums are of 32 bits.
struct Softmax {
    float most = -INFINITY, sum = 0.f, weighted = 0.f;
    __device__ __forceinline__ static float floor_of(float m) { return fmaxf(m, -3.4028235e38f); }
    // Rescaled for a maximum that is as high or higher.
    __device__ __forceinline__ void raise(float m)
    {
        const float by = floor_of(most) - floor_of(m), scale = fast_exp2(by * kLog2e);
        weighted = sum > 0.f ? scale * (weighted + fmaxf(by, -200.f) * sum) : sum;       // (nothing so far, or a sum that is not a number)
        sum *= scale;
        most = m;
    }
    // A value's place in the sums; -inf adds nothing to either, what is not a number makes both such.
    __device__ __forceinline__ static void add(float x, float least, float &sum, float &weighted)
    {
        const float d = x - least, e = fast_exp2(d * kLog2e);
        sum += e;
        weighted += fmaxf(d, -200.f) * e;
    }
    template <int N> __device__ __forceinline__ void take(const float (&v)[N])
    {
        float m = most;
#pragma unroll
        for (int i = 0; i < N; ++i) m = fmaxf(m, v[i]);
        raise(m);
        const float least = floor_of(m);
        float s[2] = {0.f, 0.f}, t[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < N; ++i) add(v[i], least, s[i & 1], t[i & 1]);
        sum += s[0] + s[1];
        weighted += t[0] + t[1];
    }
    __device__ __forceinline__ void join(float m, float s, float t)
    {
        const float all = fmaxf(most, m);
        raise(all);
        Softmax other{m, s, t};
        other.raise(all);
        sum += other.sum;
        weighted += other.weighted;
    }
};

template <typename T, int THREADS, bool TOP>
__global__ __launch_bounds__(THREADS) void token_logprobs_kernel(const LogprobArgs a)
{
    typedef RowPieces<T> Row;
    constexpr int VEC = Row::VEC, kWaves = THREADS / 64, U = 8;      // pieces that a thread has on their way
    __shared__ float parts[kWaves][3];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int64_t row = blockIdx.x, token = token_at(a.tokens, a.wide, row);
    if (token < 0 || token >= a.vocab) {         // a position that does not count: its logits are not read
        if (tid == 0) {
            a.given[row] = a.entropy[row] = 0.f;
            if (a.stats) a.stats[2 * row] = a.stats[2 * row + 1] = 0.f;
        }
        if (TOP && tid < a.top) {
            a.near[row * a.top + tid] = -INFINITY;
            a.index[row * a.top + tid] = -1;
        }
        return;
    }
    const Row x(static_cast<const T *>(a.logits) + row * a.row, a.vocab);
    const float given = tid == 0 ? (float)x.x[token] : 0.f;      // (on its way beside the row)
    Softmax mine;
    int64_t p = tid;
    auto chunk = [&](auto whole) {
        typename Row::Piece raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = *x.at(decltype(whole)::value || p + u * THREADS < x.pieces ? p + u * THREADS : x.pieces - 1);
        float v[U * VEC];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                v[u * VEC + e] = decltype(whole)::value || p + u * THREADS < x.pieces ? (float)raw[u][e] : -INFINITY;
        mine.take(v);
        p += U * THREADS;
    };
    while (p - tid + U * THREADS <= x.pieces) chunk(std::true_type{});
    if (p - tid < x.pieces) chunk(std::false_type{});
    if (tid < x.loose()) {
        const float v[1] = {(float)x.x[x.loose_place(tid)]};
        mine.take(v);
    }
    const float own_most = mine.most;
    {
        float all = mine.most;
#pragma unroll
        for (int m = 1; m < 64; m *= 2) all = fmaxf(all, shfl_xor_f32(all, m));
        mine.raise(all);
#pragma unroll
        for (int m = 1; m < 64; m *= 2) {
            mine.sum += shfl_xor_f32(mine.sum, m);
            mine.weighted += shfl_xor_f32(mine.weighted, m);
        }
        if (lane == 0) {
            parts[w][0] = all;
            parts[w][1] = mine.sum;
            parts[w][2] = mine.weighted;
        }
    }
    __syncthreads();
    Softmax joined{parts[0][0], parts[0][1], parts[0][2]};
#pragma unroll 1
    for (int i = 1; i < kWaves; ++i) joined.join(parts[i][0], parts[i][1], parts[i][2]);
    const float most = joined.most, log_sum = most == -INFINITY ? NAN : logf(joined.sum);
    if (tid == 0) {
        a.given[row] = (given - most) - log_sum;
        a.entropy[row] = log_sum - joined.weighted / joined.sum;
        if (a.stats) {
            a.stats[2 * row] = most;
            a.stats[2 * row + 1] = log_sum;
        }
    }
    if constexpr (TOP) {
        __shared__ float peaks[64];
        __shared__ u64 collected[kRoom];
        __shared__ int listed[THREADS];
        __shared__ int threads, values;
        __shared__ float bound_of_all;
        const int top = a.top;
        const bool numbers = joined.sum == joined.sum;       // (where one is none, the largest of the others may have been lost beside it)
        float peak = own_most;
#pragma unroll
        for (int m = 1; m < THREADS / 64; m *= 2) peak = fmaxf(peak, shfl_xor_f32(peak, m));
        if (tid % (THREADS / 64) == 0) peaks[tid / (THREADS / 64)] = peak;
        if (tid == 0) threads = values = 0;
        __syncthreads();
        if (w == 0) {
            const float mine_of_64 = peaks[lane];
            int above = 0;
#pragma unroll 16
            for (int i = 0; i < 64; ++i) {
                const float other = peaks[i];
                above += other > mine_of_64 || (other == mine_of_64 && i < lane);
            }
            if (above == top - 1) bound_of_all = mine_of_64;
        }
        __syncthreads();
        // where fewer than `top` of the 64 have anything above -inf: all that is above
        const float bound = fmaxf(bound_of_all, -3.4028235e38f);
        if (own_most >= bound) listed[atomicAdd(&threads, 1)] = tid;
        __syncthreads();
        const int threads_there = threads;
        auto collect = [&](float v, int64_t place) {
            if (!(v >= bound)) return;
            const int at = atomicAdd(&values, 1);
            if (at < kRoom) collected[at] = key_of(v, place);
        };
        // A wave reads the pieces of as many threads as it has lanes for.
        const int64_t each = (x.pieces + THREADS - 1) / THREADS;     // pieces of a thread, at most
        const int lanes = each > 32 ? 64 : each > 16 ? 32 : each > 8 ? 16 : each > 4 ? 8 : 4, side = 64 / lanes;
        for (int i = w * side + lane / lanes; i < threads_there; i += kWaves * side) {
            const int id = listed[i];
            for (int64_t q = id + (int64_t)(lane % lanes) * THREADS; q < x.pieces; q += (int64_t)lanes * THREADS) {
                const typename Row::Piece piece = *x.at(q);
#pragma unroll
                for (int e = 0; e < VEC; ++e) collect((float)piece[e], x.place(q) + e);
            }
        }
        if (tid < x.loose()) collect((float)x.x[x.loose_place(tid)], x.loose_place(tid));
        __syncthreads();
        const int count = values;
        float *near = a.near + row * top;
        int64_t *index = a.index + row * top;
        auto put = [&](int n, u64 key) {
            near[n] = (value_of(key) - most) - log_sum;
            index[n] = (uint32_t)~(uint32_t)key;
        };
        if (numbers && count <= kRoom) {
            for (int i = tid; i < count; i += THREADS) {
                const u64 key = collected[i];
                int over = 0;
                for (int j = 0; j < count; ++j) over += collected[j] > key;
                if (over < top) put(over, key);
            }
            // the rest are the first tokens of -inf, which lie among the first `top`, of all and more as are above
            if (w == 0 && count < top) {
                int found = count;
                for (int64_t i = lane; i - lane < a.vocab && found < top; i += 64) {
                    const bool is = i < a.vocab && !((float)x.x[i] >= bound);
                    const u64 all = __ballot(is);
                    const int n = found + __popcll(all & (((u64)1 << lane) - 1));
                    if (is && n < top) put(n, key_of(-INFINITY, i));
                    found += __popcll(all);
                }
            }
            return;
        }
        // more than there is room for (a row of equal values, or of few that are finite): one after the other, over the whole row
        u64 last = ~(u64)0;
        for (int n = 0; n < top; ++n) {
            u64 best = 0;
            for (int64_t i = tid; i < a.vocab; i += THREADS) {
                const u64 key = key_of((float)x.x[i], i);
                best = key < last && key > best ? key : best;
            }
#pragma unroll
            for (int m = 1; m < 64; m *= 2) {
                const u64 other = ((u64)(uint32_t)__shfl_xor((int)(best >> 32), m, 64) << 32) | (uint32_t)__shfl_xor((int)best, m, 64);
                best = other > best ? other : best;
            }
            __syncthreads();
            if (lane == 0) collected[w] = best;
            __syncthreads();
            last = collected[0];
#pragma unroll 1
            for (int i = 1; i < kWaves; ++i) last = collected[i] > last ? collected[i] : last;
            if (tid == 0) put(n, last);
        }
    }
}

// The logits' gradient: with g and h the cotangents of log p_token and of H,
//       dx_i = g ([i = token] - p_i) - h p_i (log p_i + H).
// A workgroup takes a segment of a row: one read, one write.  4096 rows of 32000 in 16 bits 80 us, 524 MB, the read partly from the last-level cache.
constexpr int kGradThreads = 256, kGradPieces = 4;
template <typename T> __global__ __launch_bounds__(kGradThreads) void token_logprobs_grad_kernel(const LogprobGradArgs a)
{
    typedef RowPieces<T> Row;
    constexpr int VEC = Row::VEC;
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x / a.segments, segment = blockIdx.x % a.segments, token = token_at(a.tokens, a.wide, row);
    // (rows of both arrays begin at the same place within 16 bytes)
    const Row x(static_cast<const T *>(a.logits) + row * a.row, a.vocab);
    T *to = static_cast<T *>(a.dlogits) + row * a.grad_row;
    const bool counts = token >= 0 && token < a.vocab;
    const float g = counts && a.dgiven ? a.dgiven[row] : 0.f, h = counts && a.dentropy ? a.dentropy[row] : 0.f;
    const float most = a.stats[2 * row], log_sum = a.stats[2 * row + 1], entropy = a.entropy[row];
    auto gradient = [&](float v) {
        const float log_p = (v - most) - log_sum, p = fast_exp2(log_p * kLog2e);
        // (a log p of -inf with a p of 0 adds nothing)
        return -p * (g + h * (fmaxf(log_p, -200.f) + entropy));
    };
    const int64_t first = segment * (kGradThreads * kGradPieces) + tid;
    if (!counts) {
#pragma unroll
        for (int u = 0; u < kGradPieces; ++u) {
            const int64_t p = first + u * kGradThreads;
            if (p < x.pieces) *reinterpret_cast<typename Row::Piece *>(to + x.place(p)) = typename Row::Piece{};
        }
        if (segment == 0 && tid < x.loose()) to[x.loose_place(tid)] = (T)0.f;
        return;
    }
    typename Row::Piece raw[kGradPieces];
#pragma unroll
    for (int u = 0; u < kGradPieces; ++u) {
        const int64_t p = first + u * kGradThreads;
        if (x.pieces > 0) raw[u] = *x.at(p < x.pieces ? p : x.pieces - 1);
    }
#pragma unroll
    for (int u = 0; u < kGradPieces; ++u) {
        const int64_t p = first + u * kGradThreads;
        if (p >= x.pieces) continue;
        float v[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = gradient((float)raw[u][e]);
        const int64_t at = token - x.place(p);
        if (at >= 0 && at < VEC)
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] += e == at ? g : 0.f;
        store_vec<T, VEC>(to + x.place(p), v);
    }
    if (segment == 0 && tid < x.loose()) {
        const int64_t i = x.loose_place(tid);
        Elem<T>::store(to + i, gradient((float)x.x[i]) + (i == token ? g : 0.f));
    }
}

bool sizes_ok(int64_t rows, int64_t vocab, int64_t top)
{
    return rows >= 0 && rows < ((int64_t)1 << 31) && vocab >= 1 && vocab < ((int64_t)1 << 31) && top >= 0 && top <= kMostTop && top <= vocab;
}

// 256 threads a row: 4096 rows of 32000 in 16 bits 52 us (512 threads 68, 1024 150), 777 rows of 50001 floats 35 (35, 39), one of 32000 floats 5.6 (5.3,
// 6.6).  512 where alternatives follow, whose stretches then have half the length: 500 rows of 131072 with 20 alternatives 39 us (256 threads
// 42, 1024 45), one of 131072 floats 15 (20, 16).  Neither looks at the length of a row, and a thread goes through eight whole pieces at its end: 8192 rows of 1000
// to 8000 take 37 to 40 us in 16 bits (the read alone 3 to 27), with 20 alternatives 144 to 151.  Rows so short that fewer than `top` of the 64 groups of threads hold
// a value (up to 1216 tokens in 16 bits at 20, 4032 at 64) hand over all that they have, or are searched once for each
// alternative: 8192 rows of 1000 with 20 683 us, of 4000 with 64 2020.  A row of 131072 floats has one compute unit.
template <typename T> int dispatch_logprobs(hipStream_t stream, const LogprobArgs &a, int64_t rows)
{
    if (a.top) token_logprobs_kernel<T, 512, true><<<rows, 512, 0, stream>>>(a);
    else token_logprobs_kernel<T, 256, false><<<rows, 256, 0, stream>>>(a);
    return launch_status();
}

}  // namespace
}  // namespace gla

using namespace gla;

extern "C" int gla_token_logprobs(void *stream, int64_t rows, int64_t vocab, int64_t top, gla_dtype dtype, int64_t row, int wide_indices,
                                  const void *logits, const void *tokens, float *logprobs, float *entropy, float *stats, float *top_logprobs,
                                  int64_t *top_tokens)
{
    if (!sizes_ok(rows, vocab, top) || (rows > 1 && row < vocab)) return GLA_ERR_SHAPE;
    if (rows == 0) return GLA_OK;
    if (!logits || !tokens || !logprobs || !entropy || (top && (!top_logprobs || !top_tokens))) return GLA_ERR_NULL;
    if (dtype != GLA_F32 && dtype != GLA_BF16) return GLA_ERR_DTYPE;
    const int64_t size = dtype == GLA_BF16 ? 2 : 4;
    if (reinterpret_cast<uintptr_t>(logits) % size || (reinterpret_cast<uintptr_t>(tokens) & (wide_indices ? 7 : 3)) ||
        (reinterpret_cast<uintptr_t>(top_tokens) & 7))
        return GLA_ERR_ALIGN;
    for (const float *x : {logprobs, entropy, stats, top_logprobs})
        if (reinterpret_cast<uintptr_t>(x) & 3) return GLA_ERR_ALIGN;
    LogprobArgs a{vocab, row, (int)top, wide_indices, logits, tokens, logprobs, entropy, stats, top_logprobs, top_tokens};
    const hipStream_t s = static_cast<hipStream_t>(stream);
    for (int64_t n = 0; n < rows; n += kMostGroups) {
        const int64_t some = rows - n < kMostGroups ? rows - n : kMostGroups;
        a.logits = static_cast<const char *>(logits) + n * row * size;
        a.tokens = static_cast<const char *>(tokens) + n * (wide_indices ? 8 : 4);
        a.given = logprobs + n;
        a.entropy = entropy + n;
        a.stats = stats ? stats + 2 * n : nullptr;
        a.near = top ? top_logprobs + n * top : nullptr;
        a.index = top ? top_tokens + n * top : nullptr;
        if (int e = dtype == GLA_BF16 ? dispatch_logprobs<__bf16>(s, a, some) : dispatch_logprobs<float>(s, a, some)) return e;
    }
    return GLA_OK;
}

extern "C" int gla_token_logprobs_bwd(void *stream, int64_t rows, int64_t vocab, gla_dtype dtype, int64_t row, int64_t grad_row,
                                      int wide_indices, const void *logits, const void *tokens, const float *stats, const float *entropy,
                                      const float *dlogprobs, const float *dentropy, void *dlogits)
{
    if (!sizes_ok(rows, vocab, 0) || (rows > 1 && (row < vocab || grad_row < vocab))) return GLA_ERR_SHAPE;
    if (rows == 0) return GLA_OK;
    if (!logits || !tokens || !stats || !entropy || !dlogits) return GLA_ERR_NULL;
    if (dtype != GLA_F32 && dtype != GLA_BF16) return GLA_ERR_DTYPE;
    const int64_t size = dtype == GLA_BF16 ? 2 : 4, pieces = vocab * size / 16;
    if (reinterpret_cast<uintptr_t>(logits) % size || (reinterpret_cast<uintptr_t>(tokens) & (wide_indices ? 7 : 3))) return GLA_ERR_ALIGN;
    // rows of both arrays have to begin at the same place within 16 bytes
    if (((reinterpret_cast<uintptr_t>(logits) - reinterpret_cast<uintptr_t>(dlogits)) & 15) || (rows > 1 && (row - grad_row) * size % 16))
        return GLA_ERR_ALIGN;
    for (const float *x : {stats, entropy, dlogprobs, dentropy})
        if (reinterpret_cast<uintptr_t>(x) & 3) return GLA_ERR_ALIGN;
    LogprobGradArgs a{vocab, row, grad_row, (pieces + kGradThreads * kGradPieces - 1) / (kGradThreads * kGradPieces), wide_indices, logits, tokens,
                      stats, entropy, dlogprobs, dentropy, dlogits};
    if (a.segments < 1) a.segments = 1;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t at_once = kMostGroups / a.segments;
    for (int64_t n = 0; n < rows; n += at_once) {
        const unsigned grid = (unsigned)((rows - n < at_once ? rows - n : at_once) * a.segments);
        a.logits = static_cast<const char *>(logits) + n * row * size;
        a.dlogits = static_cast<char *>(dlogits) + n * grad_row * size;
        a.tokens = static_cast<const char *>(tokens) + n * (wide_indices ? 8 : 4);
        a.stats = stats + 2 * n;
        a.entropy = entropy + n;
        a.dgiven = dlogprobs ? dlogprobs + n : nullptr;
        a.dentropy = dentropy ? dentropy + n : nullptr;
        if (dtype == GLA_BF16) token_logprobs_grad_kernel<__bf16><<<grid, kGradThreads, 0, s>>>(a);
        else token_logprobs_grad_kernel<float><<<grid, kGradThreads, 0, s>>>(a);
        if (int e = launch_status()) return e;
    }
    return GLA_OK;
}
