// Entry points of linear attention with one decay a head: argument checks, the split into segments, workspaces.
#include "gla_decay.hpp"

namespace gla {
namespace {

constexpr int64_t kMostFeatures = 256;
constexpr int64_t kMostRow = (int64_t)1 << 23;      // elements from one token to the next: a chunk's places are 32-bit numbers

int64_t pad256(int64_t x) { return (x + 255) & ~(int64_t)255; }

// Sequences run as segments side by side where that fills the GPU better: one workgroup walks a segment's chunks in order, so B1
// T32768 H8 D128 as whole sequences would use 8 of 256 compute units (16 segments: 178 us, 32: 115, 64: 133).  A compute unit takes one
// workgroup at a time here: two at once hardly do more together.  Weighed are, in the time of a chunk, the rounds that `slots` of them take, a
// workgroup's start, and what segments cost besides: the pass that finds the states entering them (`pass` of the work, on half of the rows)
// and a state for each to write, scan and read.  A whole number of rounds leaves no compute unit idle, so only the counts that just fill some are looked
// at; a segment has two chunks at least.  Ragged sequences count as half full, their longest segment as what the others wait for: B16 T1337
// H16 D128 of lengths 0 to 1337 takes 77 us whole; in two segments 103 by decay_pass_kernel, which 512 workgroups take, and 100 by
// decay_forward_kernel, made to take them; in four 121 and 122.
DecayPlan plan_segments(const DecaySizes &n, gla_dtype dtype, int64_t workgroups, int64_t slots, double pass, bool ragged)
{
    const int64_t C = dtype == GLA_BF16 ? DecayChunk<__bf16>::C : DecayChunk<float>::C;
    const int64_t chunks = (n.T + C - 1) / C;
    int64_t best = 1;
    const double work = (double)workgroups * chunks / slots;
    double least = 0.0;
    for (int64_t rounds = 0; rounds <= 4; ++rounds) {
        int64_t segments = rounds ? rounds * slots / workgroups : 1;
        if (segments > chunks / 2) segments = chunks / 2;
        if (rounds && segments < 2) continue;
        if (segments < 1) segments = 1;
        const int64_t longest = (chunks + segments - 1) / segments, taken = (workgroups * segments + slots - 1) / slots;
        // a state is written, scanned and read, the rows of a chunk are read: DK / 32 of them move as much
        const double states = 0.012 * n.DK;
        double cost = ragged ? 0.5 * work + longest + taken : taken * (longest + 1.0);
        if (segments > 1) cost += pass * (ragged ? 0.5 * work + longest : work) + taken + states * workgroups * segments / slots + 1.0;
        if (rounds == 0 || cost < least) {
            least = cost;
            best = segments;
        }
    }
    return DecayPlan(chunks, best);
}
DecayPlan forward_plan(const DecaySizes &n, gla_dtype dtype, bool ragged)
{
    return plan_segments(n, dtype, n.B * n.H * decay_slabs(n.DV), kComputeUnits, 0.6, ragged);
}
DecayPlan backward_plan(const DecaySizes &n, gla_dtype dtype, bool ragged)
{
    return plan_segments(n, dtype, n.B * n.H * decay_slabs(n.DV) * (n.DK > 128 ? 2 : 1), kComputeUnits, 0.2, ragged);
}

int64_t entering_bytes(const DecaySizes &n, const DecayPlan &p)
{
    if (p.segments < 2) return 0;
    return pad256(n.B * n.H * p.segments * decay_slabs(n.DV) * decay_value_slab(n.DV) * decay_key_width(n.DK) * 4) +
           pad256(n.B * n.H * p.segments * 4);
}
void split_entering(const DecaySizes &n, const DecayPlan &p, char *ws, float *&states, float *&decays)
{
    states = reinterpret_cast<float *>(ws);
    decays = reinterpret_cast<float *>(ws + pad256(n.B * n.H * p.segments * decay_slabs(n.DV) * decay_value_slab(n.DV) *
                                                   decay_key_width(n.DK) * 4));
}

DecayParts plan_parts(const DecaySizes &n)
{
    DecayParts p{};
    const int64_t ks = n.DK > 128 ? 2 : 1, vs = decay_slabs(n.DV);
    p.rows = (int)(vs * (n.H / n.HK));
    p.values = (int)ks;
    p.gates = (int)(ks * vs);
    return p;
}
// Assigns the parts' arrays behind `ws` (which may be NULL: for the size alone).
int64_t place_parts(const DecaySizes &n, const DecayPlan &plan, bool constant_gates, DecayParts &p, char *ws)
{
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        char *x = ws + at;
        at += pad256(bytes);
        return x;
    };
    if (p.rows > 1) {
        p.dquery = reinterpret_cast<float *>(take(p.rows * n.B * n.T * n.HK * n.DK * 4));
        p.dkey = reinterpret_cast<float *>(take(p.rows * n.B * n.T * n.HK * n.DK * 4));
    }
    if (p.values > 1) p.dvalue = reinterpret_cast<float *>(take(p.values * n.B * n.T * n.H * n.DV * 4));
    if (p.gates > 1 && !constant_gates) p.dgate = reinterpret_cast<float *>(take(p.gates * n.B * n.T * n.H * 4));
    if (constant_gates) p.gate_sums = reinterpret_cast<double *>(take(p.gates * n.H * n.B * plan.segments * 8));
    return at;
}

// The arrays' places: strides of log_decay, value, key, query in this order, batch, token and head each (in elements).
struct Places {
    DecayRows gates, values, keys, queries;
};
Places place(const DecaySizes &n, const int64_t *strides, const void *log_decay, const void *value, const void *key, const void *query)
{
    Places p{{log_decay, n.T * n.H, n.H, 1},
             {value, n.T * n.H * n.DV, n.H * n.DV, n.DV},
             {key, n.T * n.HK * n.DK, n.HK * n.DK, n.DK},
             {query, n.T * n.HK * n.DK, n.HK * n.DK, n.DK}};
    if (strides) {
        DecayRows *all[4] = {&p.gates, &p.values, &p.keys, &p.queries};
        for (int i = 0; i < 4; ++i) {
            all[i]->sb = strides[3 * i];
            all[i]->st = strides[3 * i + 1];
            all[i]->sh = strides[3 * i + 2];
        }
    }
    return p;
}
bool dtype_ok(gla_dtype d) { return d == GLA_F32 || d == GLA_BF16; }

bool rows_near(const DecayRows &r) { return r.st >= 0 && r.st < kMostRow; }

// Rows are read 16 bytes at a time.
bool rows_aligned(const DecayRows &r, gla_dtype dtype)
{
    const int64_t piece = dtype == GLA_BF16 ? 8 : 4;
    return aligned16(r.p) && r.sb % piece == 0 && r.st % piece == 0 && r.sh % piece == 0;
}

int check_sizes(const DecaySizes &n)
{
    const int64_t limit = (int64_t)1 << 30;
    if (n.B < 1 || n.T < 0 || n.H < 1 || n.HK < 1 || n.DK < 1 || n.DV < 1) return GLA_ERR_SHAPE;
    if (n.H % n.HK || n.DK % 16 || n.DV % 16 || n.DK > kMostFeatures || n.DV > kMostFeatures) return GLA_ERR_SHAPE;
    if (n.B >= limit || n.H >= limit || n.T >= limit || n.B * n.H >= limit) return GLA_ERR_SHAPE;
    if (n.H * n.DV >= kMostRow || n.HK * n.DK >= kMostRow) return GLA_ERR_SHAPE;
    return GLA_OK;
}
int64_t kept_bytes(const DecaySizes &n, gla_dtype dtype)
{
    const int64_t C = dtype == GLA_BF16 ? DecayChunk<__bf16>::C : DecayChunk<float>::C;
    return n.B * n.H * ((n.T + C - 1) / C) * n.DK * n.DV * 4;
}

}  // namespace
}  // namespace gla

using namespace gla;

extern "C" size_t gla_decay_states_bytes(int64_t B, int64_t T, int64_t H, int64_t HK, int64_t DK, int64_t DV, gla_dtype dtype)
{
    const DecaySizes n{B, T, H, HK, DK, DV};
    if (check_sizes(n) || !dtype_ok(dtype)) return 0;
    return (size_t)kept_bytes(n, dtype);
}

extern "C" size_t gla_decay_fwd_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t HK, int64_t DK, int64_t DV, gla_dtype dtype,
                                                int ragged)
{
    const DecaySizes n{B, T, H, HK, DK, DV};
    if (check_sizes(n) || !dtype_ok(dtype)) return 0;
    return (size_t)entering_bytes(n, forward_plan(n, dtype, ragged != 0));
}

extern "C" size_t gla_decay_bwd_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t HK, int64_t DK, int64_t DV, gla_dtype dtype,
                                                int constant_decay, int ragged)
{
    const DecaySizes n{B, T, H, HK, DK, DV};
    if (check_sizes(n) || !dtype_ok(dtype)) return 0;
    const DecayPlan plan = backward_plan(n, dtype, ragged != 0);
    DecayParts parts = plan_parts(n);
    return (size_t)(entering_bytes(n, plan) + place_parts(n, plan, constant_decay != 0, parts, nullptr));
}

extern "C" int gla_decay_fwd(void *stream, int64_t B, int64_t T, int64_t H, int64_t HK, int64_t DK, int64_t DV, gla_dtype dtype,
                             gla_dtype hidden_dtype, const int64_t *strides, const void *hidden_init, const float *log_decay,
                             const void *value, const void *key, const void *query, const int32_t *lengths, void *hidden_final,
                             void *out, void *states, void *workspace, size_t workspace_bytes)
{
    const DecaySizes n{B, T, H, HK, DK, DV};
    if (!hidden_init || !hidden_final || (T > 0 && (!log_decay || !value || !key || !query || !out))) return GLA_ERR_NULL;
    if (int e = check_sizes(n)) return e;
    if (!dtype_ok(dtype) || !dtype_ok(hidden_dtype)) return GLA_ERR_DTYPE;
    const Places p = place(n, strides, log_decay, value, key, query);
    if (!aligned16(hidden_init) || !aligned16(hidden_final) || !aligned16(out) || !aligned16(states) ||
        !rows_aligned(p.values, dtype) || !rows_aligned(p.keys, dtype) || !rows_aligned(p.queries, dtype) ||
        (reinterpret_cast<uintptr_t>(log_decay) & 3) || (reinterpret_cast<uintptr_t>(lengths) & 3))
        return GLA_ERR_ALIGN;
    if (!rows_near(p.values) || !rows_near(p.keys) || !rows_near(p.queries)) return GLA_ERR_SHAPE;
    const DecayPlan plan = forward_plan(n, dtype, lengths != nullptr);
    const int64_t need = entering_bytes(n, plan);
    if (need && (!workspace || (int64_t)workspace_bytes < need)) return GLA_ERR_WORKSPACE;
    if (need && !aligned16(workspace)) return GLA_ERR_ALIGN;
    float *entering = nullptr, *decays = nullptr;
    if (need) split_entering(n, plan, static_cast<char *>(workspace), entering, decays);
    return decay_forward(stream, n, plan, dtype, hidden_dtype, hidden_init, p.gates, p.keys, p.values, p.queries, lengths,
                         hidden_final, out, static_cast<float *>(states), entering, decays);
}

extern "C" int gla_decay_bwd(void *stream, int64_t B, int64_t T, int64_t H, int64_t HK, int64_t DK, int64_t DV, gla_dtype dtype,
                             gla_dtype hidden_dtype, int constant_decay, const int64_t *strides, const float *log_decay,
                             const void *value, const void *key, const void *query, const int32_t *lengths, const void *states,
                             const void *dhidden_final, const void *dout, void *dhidden_init, float *dlog_decay, void *dvalue,
                             void *dkey, void *dquery, void *workspace, size_t workspace_bytes)
{
    const DecaySizes n{B, T, H, HK, DK, DV};
    if (!dhidden_final || !dhidden_init || (constant_decay && !dlog_decay) ||
        (T > 0 && (!log_decay || !value || !key || !query || !states || !dout || !dlog_decay || !dvalue || !dkey || !dquery)))
        return GLA_ERR_NULL;
    if (int e = check_sizes(n)) return e;
    if (!dtype_ok(dtype) || !dtype_ok(hidden_dtype)) return GLA_ERR_DTYPE;
    const Places p = place(n, strides, log_decay, value, key, query);
    const DecayRows cotangents{dout, T * H * DV, H * DV, DV};
    for (const void *x : {dhidden_final, static_cast<const void *>(dhidden_init), static_cast<const void *>(dvalue),
                          static_cast<const void *>(dkey), static_cast<const void *>(dquery), states, dout})
        if (!aligned16(x)) return GLA_ERR_ALIGN;
    if (!rows_aligned(p.values, dtype) || !rows_aligned(p.keys, dtype) || !rows_aligned(p.queries, dtype) ||
        !aligned16(dlog_decay) || (reinterpret_cast<uintptr_t>(log_decay) & 3) || (reinterpret_cast<uintptr_t>(lengths) & 3))
        return GLA_ERR_ALIGN;
    if (!rows_near(p.values) || !rows_near(p.keys) || !rows_near(p.queries)) return GLA_ERR_SHAPE;
    const DecayPlan plan = backward_plan(n, dtype, lengths != nullptr);
    DecayParts parts = plan_parts(n);
    const int64_t first = entering_bytes(n, plan), need = first + place_parts(n, plan, constant_decay != 0, parts, nullptr);
    if (need && (!workspace || (int64_t)workspace_bytes < need)) return GLA_ERR_WORKSPACE;
    if (need && !aligned16(workspace)) return GLA_ERR_ALIGN;
    float *entering = nullptr, *decays = nullptr;
    if (first) split_entering(n, plan, static_cast<char *>(workspace), entering, decays);
    place_parts(n, plan, constant_decay != 0, parts, static_cast<char *>(workspace) + first);
    return decay_backward(stream, n, plan, dtype, hidden_dtype, p.gates, p.keys, p.values, p.queries, cotangents, lengths,
                          static_cast<const float *>(states), dhidden_final, constant_decay != 0, dhidden_init, dlog_decay, dvalue,
                          dkey, dquery, entering, decays, parts);
}
