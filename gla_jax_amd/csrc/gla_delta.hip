// Entry points of the gated delta rule over whole sequences: argument checks, workspaces, launches.
#include "gla_delta.hpp"

namespace gla {
namespace {

constexpr int64_t kMostKeys = GLA_MOST_DELTA_KEYS, kMostValues = 256;
constexpr int64_t kMostRow = (int64_t)1 << 23;      // elements from one token to the next: a chunk's places are 32-bit numbers

int64_t pad256(int64_t x) { return (x + 255) & ~(int64_t)255; }
bool dtype_ok(gla_dtype d) { return d == GLA_F32 || d == GLA_BF16; }
int64_t bytes_of(gla_dtype d) { return d == GLA_BF16 ? 2 : 4; }
int64_t chunk_of(gla_dtype d) { return d == GLA_BF16 ? DeltaChunk<__bf16>::C : DeltaChunk<float>::C; }
int64_t chunks_of(const DecaySizes &n, gla_dtype d) { return (n.T + chunk_of(d) - 1) / chunk_of(d); }

int check_sizes(const DecaySizes &n, gla_dtype dtype)
{
    const int64_t limit = (int64_t)1 << 30;
    if (n.B < 1 || n.T < 0 || n.H < 1 || n.HK < 1 || n.DK < 1 || n.DV < 1) return GLA_ERR_SHAPE;
    if (n.H % n.HK || n.DK % 16 || n.DV % 16 || n.DK > kMostKeys || n.DV > kMostValues) return GLA_ERR_SHAPE;
    if (n.B >= limit || n.H >= limit || n.T >= limit || n.B * n.H >= limit) return GLA_ERR_SHAPE;
    if (n.H * n.DV >= kMostRow || n.HK * n.DK >= kMostRow) return GLA_ERR_SHAPE;
    if (!dtype_ok(dtype)) return GLA_ERR_DTYPE;
    // (workgroups of 512 threads, which a launch counts in 32 bits)
    const int64_t most = (int64_t)1 << 23, pairs = (n.B * n.H + 7) / 8 * 8;
    if (pairs * chunks_of(n, dtype) >= most || pairs * ((n.DV + 31) / 32) >= most) return GLA_ERR_SHAPE;
    return GLA_OK;
}

// Assigns the places of a call's scratch behind `ws` (which may be NULL: for the size alone); what the backward pass takes more of.
int64_t lay_out(DeltaArgs &a, gla_dtype dtype, bool backward, char *ws, float **dquery, float **dkey)
{
    const int64_t C = chunk_of(dtype), e = bytes_of(dtype), chunk_pairs = a.pairs * a.chunks;
    const int64_t parts = dtype == GLA_BF16 ? DeltaChunk<__bf16>::kParts : 1, few = dtype == GLA_BF16 ? DeltaChunk<__bf16>::kFew : 1;
    const int64_t steps = dtype == GLA_BF16 ? DeltaChunk<__bf16>::kSteps : DeltaChunk<float>::kSteps;
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        char *x = ws + at;
        at += pad256(bytes);
        return x;
    };
    a.to.inverse = take(chunk_pairs * steps * parts * 512 * e);
    a.to.scores = take(chunk_pairs * steps * (backward ? parts : few) * 512 * e);
    a.to.gates = reinterpret_cast<float *>(take(chunk_pairs * 4 * C * 4));
    a.summary = reinterpret_cast<float *>(take(a.pairs * (a.segments - 1) * (a.n.DV + a.n.DK) * a.n.DK * 4));
    a.starts = reinterpret_cast<float *>(take(a.pairs * (a.segments - 1) * a.n.DV * a.n.DK * 4));
    if (!backward) return at;
    a.du = reinterpret_cast<float *>(take(a.pairs * delta_written_floats(a.n, a.chunks, (int)C) * 4));
    a.dstates = take(chunk_pairs * delta_state_floats(a.n) * few * e);
    a.dots = reinterpret_cast<float *>(take(chunk_pairs * (a.n.DV / 16) * 4 * 4));
    a.row_parts = (int)(a.n.H / a.n.HK);
    if (a.row_parts > 1) {
        const int64_t rows = a.row_parts * a.n.B * a.n.T * a.n.HK * a.n.DK * 4;
        *dquery = reinterpret_cast<float *>(take(rows));
        *dkey = reinterpret_cast<float *>(take(rows));
    }
    return at;
}
DeltaArgs sizes_of(const DecaySizes &n, gla_dtype dtype)
{
    DeltaArgs a{};
    a.n = n;
    a.chunks = chunks_of(n, dtype);
    a.pairs = n.B * n.H;
    a.segments = 1;
    a.segment_chunks = (int)a.chunks;
    if (a.chunks) {
        a.segment_chunks = (int)((a.chunks + delta_segments(a) - 1) / delta_segments(a));
        a.segments = (int)((a.chunks + a.segment_chunks - 1) / a.segment_chunks);
    }
    return a;
}
int64_t workspace_bytes(const DecaySizes &n, gla_dtype dtype, bool backward)
{
    DeltaArgs a = sizes_of(n, dtype);
    float *dquery, *dkey;
    return a.chunks ? lay_out(a, dtype, backward, nullptr, &dquery, &dkey) : 0;
}

// The arrays' places: strides of log_decay, beta, value, key, query in this order, batch, token and head each (in elements).
int place(DeltaArgs &a, gla_dtype dtype, const int64_t *strides, const void *log_decay, const void *beta, const void *value, const void *key,
          const void *query)
{
    const DecaySizes &n = a.n;
    a.gates = {log_decay, n.T * n.H, n.H, 1};
    a.betas = {beta, n.T * n.H, n.H, 1};
    a.values = {value, n.T * n.H * n.DV, n.H * n.DV, n.DV};
    a.keys = {key, n.T * n.HK * n.DK, n.HK * n.DK, n.DK};
    a.queries = {query, n.T * n.HK * n.DK, n.HK * n.DK, n.DK};
    DecayRows *all[5] = {&a.gates, &a.betas, &a.values, &a.keys, &a.queries};
    for (int i = 0; strides && i < 5; ++i) {
        all[i]->sb = strides[3 * i];
        all[i]->st = strides[3 * i + 1];
        all[i]->sh = strides[3 * i + 2];
    }
    if ((reinterpret_cast<uintptr_t>(log_decay) & 3) || (reinterpret_cast<uintptr_t>(beta) & 3)) return GLA_ERR_ALIGN;
    const int64_t piece = 16 / bytes_of(dtype);
    for (int i = 2; i < 5; ++i) {
        if (!aligned16(all[i]->p) || all[i]->sb % piece || all[i]->st % piece || all[i]->sh % piece) return GLA_ERR_ALIGN;
        if (all[i]->st < 0 || all[i]->st >= kMostRow) return GLA_ERR_SHAPE;
    }
    return GLA_OK;
}

}  // namespace
}  // namespace gla

using namespace gla;

extern "C" size_t gla_delta_states_bytes(int64_t B, int64_t T, int64_t H, int64_t HK, int64_t DK, int64_t DV, gla_dtype dtype)
{
    const DecaySizes n{B, T, H, HK, DK, DV};
    if (check_sizes(n, dtype)) return 0;
    const int64_t chunks = chunks_of(n, dtype);
    return (size_t)(B * H * (delta_states_floats(n, chunks) + delta_written_floats(n, chunks, (int)chunk_of(dtype))) * 4);
}

extern "C" size_t gla_delta_fwd_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t HK, int64_t DK, int64_t DV, gla_dtype dtype)
{
    const DecaySizes n{B, T, H, HK, DK, DV};
    return check_sizes(n, dtype) ? 0 : (size_t)workspace_bytes(n, dtype, false);
}

extern "C" size_t gla_delta_bwd_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t HK, int64_t DK, int64_t DV, gla_dtype dtype)
{
    const DecaySizes n{B, T, H, HK, DK, DV};
    return check_sizes(n, dtype) ? 0 : (size_t)workspace_bytes(n, dtype, true);
}

extern "C" int gla_delta_fwd(void *stream, int64_t B, int64_t T, int64_t H, int64_t HK, int64_t DK, int64_t DV, gla_dtype dtype,
                             gla_dtype hidden_dtype, const int64_t *strides, const void *hidden_init, const float *log_decay,
                             const float *beta, const void *value, const void *key, const void *query, const int32_t *lengths,
                             void *hidden_final, void *out, void *states, void *workspace, size_t workspace_bytes_)
{
    const DecaySizes n{B, T, H, HK, DK, DV};
    if (!hidden_init || !hidden_final || (T > 0 && (!log_decay || !beta || !value || !key || !query || !out))) return GLA_ERR_NULL;
    if (int e = check_sizes(n, dtype)) return e;
    if (!dtype_ok(hidden_dtype)) return GLA_ERR_DTYPE;
    DeltaArgs a = sizes_of(n, dtype);
    if (int e = place(a, dtype, strides, log_decay, beta, value, key, query)) return e;
    if (!aligned16(hidden_init) || !aligned16(hidden_final) || !aligned16(out) || !aligned16(states) || (reinterpret_cast<uintptr_t>(lengths) & 3))
        return GLA_ERR_ALIGN;
    const int64_t need = workspace_bytes(n, dtype, false);
    if (need && (!workspace || (int64_t)workspace_bytes_ < need)) return GLA_ERR_WORKSPACE;
    if (need && !aligned16(workspace)) return GLA_ERR_ALIGN;
    float *dquery, *dkey;
    if (need) lay_out(a, dtype, false, static_cast<char *>(workspace), &dquery, &dkey);
    a.lengths = lengths;
    a.hidden = hidden_init;
    a.hidden_dtype = hidden_dtype;
    a.hidden_out = hidden_final;
    a.out = out;
    a.kept = static_cast<float *>(states);
    if (int e = delta_prepare(stream, a, dtype, false)) return e;
    return delta_walk(stream, a, dtype, false);
}

extern "C" int gla_delta_bwd(void *stream, int64_t B, int64_t T, int64_t H, int64_t HK, int64_t DK, int64_t DV, gla_dtype dtype,
                             gla_dtype hidden_dtype, const int64_t *strides, const float *log_decay, const float *beta, const void *value,
                             const void *key, const void *query, const int32_t *lengths, const void *states, const void *dhidden_final,
                             const void *dout, void *dhidden_init, float *dlog_decay, float *dbeta, void *dvalue, void *dkey, void *dquery,
                             void *workspace, size_t workspace_bytes_)
{
    const DecaySizes n{B, T, H, HK, DK, DV};
    if (!dhidden_final || !dhidden_init || (T > 0 && (!log_decay || !beta || !value || !key || !query || !states || !dout || !dlog_decay ||
                                                      !dbeta || !dvalue || !dkey || !dquery)))
        return GLA_ERR_NULL;
    if (int e = check_sizes(n, dtype)) return e;
    if (!dtype_ok(hidden_dtype)) return GLA_ERR_DTYPE;
    DeltaArgs a = sizes_of(n, dtype);
    if (int e = place(a, dtype, strides, log_decay, beta, value, key, query)) return e;
    for (const void *x : {dhidden_final, static_cast<const void *>(dhidden_init), static_cast<const void *>(dvalue),
                          static_cast<const void *>(dkey), static_cast<const void *>(dquery), states, dout})
        if (!aligned16(x)) return GLA_ERR_ALIGN;
    if ((reinterpret_cast<uintptr_t>(dlog_decay) & 3) || (reinterpret_cast<uintptr_t>(dbeta) & 3) || (reinterpret_cast<uintptr_t>(lengths) & 3))
        return GLA_ERR_ALIGN;
    const int64_t need = workspace_bytes(n, dtype, true);
    if (need && (!workspace || (int64_t)workspace_bytes_ < need)) return GLA_ERR_WORKSPACE;
    if (need && !aligned16(workspace)) return GLA_ERR_ALIGN;
    float *dquery_parts = nullptr, *dkey_parts = nullptr;
    if (need) lay_out(a, dtype, true, static_cast<char *>(workspace), &dquery_parts, &dkey_parts);
    a.dout = {dout, T * H * DV, H * DV, DV};
    a.lengths = lengths;
    a.hidden = dhidden_final;
    a.hidden_dtype = hidden_dtype;
    a.hidden_out = dhidden_init;
    a.kept = static_cast<float *>(const_cast<void *>(states));
    a.dvalue = dvalue;
    a.dkey = a.row_parts > 1 ? dkey_parts : dkey;
    a.dquery = a.row_parts > 1 ? dquery_parts : dquery;
    a.dgate = dlog_decay;
    a.dbeta = dbeta;
    if (int e = delta_prepare(stream, a, dtype, true)) return e;
    if (int e = delta_walk(stream, a, dtype, true)) return e;
    if (int e = delta_gradients(stream, a, dtype)) return e;
    if (a.chunks == 0 || a.row_parts == 1) return GLA_OK;
    if (int e = delta_sum_heads(stream, n, dtype, dquery_parts, dquery)) return e;
    return delta_sum_heads(stream, n, dtype, dkey_parts, dkey);
}
