// Attention's entry points: checks, the split of long axes, the order of the passes
// (attention_kernels.h).
#include "attention_kernels.h"

namespace gefen {
namespace attn {

extern template int launch_width<float>(Pass, const Params&, hipStream_t);
extern template int launch_width<f16_t>(Pass, const Params&, hipStream_t);
extern template int launch_width<bf16_t>(Pass, const Params&, hipStream_t);
extern template int launch_range<f16_t>(const Params&, hipStream_t);

int launch_type(int dtype, Pass pass, const Params& a, hipStream_t st) {
    if (dtype == GEFEN_F32) return launch_width<float>(pass, a, st);
    if (dtype == GEFEN_F16) return launch_width<f16_t>(pass, a, st);
    return launch_width<bf16_t>(pass, a, st);
}

int64_t stat_count(const gefen_attention_task& t) { return t.batch * t.queries * t.heads; }
int64_t round16(int64_t floats) { return (floats + 3) / 4 * 4; }
int64_t out_count(Pass pass, const gefen_attention_task& t) {
    return t.batch * t.width * (pass == kKeysPass ? t.keys * t.kv_heads : t.queries * t.heads);
}

// Into how many parts a workgroup's tiles are split.  Few workgroups leave the chip idle: one
// query of 16 sequences over 8192 keys, 128 of them, took 263 us whole, 100 us in 4 parts with the
// join and 107 in 8; 195 workgroups of 16 tiles took 31.5 us whole and 32.2 in 2 parts, so there
// have to be three; those of dK and dV, which differ in length, took 78 us whole and 61 in 2.
// `slots` is what the chip holds of heads above 64, a workgroup a CU in float32 and two in 16 bits;
// narrower heads, of which it holds up to twice as many, are split for the same number.
// Packed sequences of uneven length make as many as the chip holds wait for the longest one's keys
// (11 sequences of 16384 tokens, 2048 workgroups: 1360 us whole, 1115 us in 4 parts with the join;
// one sequence of 8192: 1570 and 1590).  A part has four tiles at least, for its sums go through
// memory: of the whole axis, and where sequences are split for their lengths of their mean one (64
// sequences of 128 tokens, 8 heads of 128: dK and dV 46 us whole, 184 in 4 parts with the join; one
// of 8192 beside 1024 of 8, 32 / 8 heads: 1530 us whole and 1620).
int parts_of(Pass pass, const gefen_attention_task& t) {
    const bool keys = pass == kKeysPass;
    const int64_t slots = t.dtype == GEFEN_F32 ? 256 : 512, group = t.heads / t.kv_heads;
    const int64_t cols = keys ? t.keys : t.queries * group;
    const int64_t tiles = keys ? group * ((t.queries + BN - 1) / BN) : (t.keys + BN - 1) / BN;
    const int64_t wgs = t.batch * t.kv_heads * ((cols + kCols - 1) / kCols) * (keys ? 2 : 1);
    if (wgs == 0 || tiles == 0) return 1;
    int64_t parts = slots / wgs;
    if (!keys && parts < 3) parts = 1;
    if (keys && t.offsets && t.sequences > 1 && wgs < 8 * slots && parts < 4) {
        const int64_t mean = (t.queries + t.sequences - 1) / t.sequences;
        parts = std::max(parts, std::min((int64_t)4, group * ((mean + BN - 1) / BN) / 4));
    }
    parts = parts < tiles / 4 ? parts : tiles / 4;
    return (int)(parts < 1 ? 1 : parts > 32 ? 32 : parts);
}
// Floats of the parts' results and (forward) lse.
int64_t partial_count(Pass pass, const gefen_attention_task& t) {
    const int parts = parts_of(pass, t);
    if (parts == 1) return 0;
    return parts * (round16(out_count(pass, t)) * (pass == kKeysPass ? 2 : 1) +
                    (pass == kForwardPass ? round16(stat_count(t)) : 0));
}
void set_parts(Pass pass, const gefen_attention_task& t, float* memory, Params* a) {
    a->parts = parts_of(pass, t);
    a->partial = memory;
    a->partial_stride = round16(out_count(pass, t));
    a->partial_lse = memory + a->parts * a->partial_stride;
    a->stats = round16(stat_count(t));
}

// Workgroups along x that every pass can launch: HIP takes fewer than 2^32 work items there.
// Split work (parts_of) has a few thousand, and what doubles or multiplies a grid is along y and z.
constexpr int64_t kMostBlocks = (((int64_t)1 << 32) - 1) / kThreads;

// Checks what does not depend on the direction.
int check_task(const gefen_attention_task* t) {
    if (!t) return fail_inval("attention: no task");
    if (!valid_dtype(t->dtype)) return fail_inval("attention: unknown dtype %d", t->dtype);
    if (t->batch < 0 || t->queries < 0 || t->keys < 0 || t->heads < 1 || t->kv_heads < 1)
        return fail_inval("attention: sizes must not be negative, and there is a head at least");
    if (t->heads % t->kv_heads) return fail_inval("attention: heads must be a multiple of kv_heads");
    if (t->width < 1 || t->width > GEFEN_ATTENTION_MAX_WIDTH)
        return fail_inval("attention: width must be 1 to %d, got %lld", GEFEN_ATTENTION_MAX_WIDTH, (long long)t->width);
    const int64_t most = (int64_t)1 << 30;
    if (t->batch > most || t->queries > most || t->keys > most || t->heads > 65536)
        return fail_inval("attention: sizes out of range");
    const int64_t group = t->heads / t->kv_heads, pairs = t->batch * t->kv_heads;
    if (t->queries * group > most || pairs > most || pairs * ((t->queries * group + kCols - 1) / kCols) > kMostBlocks ||
        pairs * ((t->keys + kCols - 1) / kCols) > kMostBlocks)
        return fail_inval("attention: sizes out of range: batch * kv_heads times the blocks of %d keys, or of "
                          "queries * heads / kv_heads, must stay below 2^24",
                          kCols);
    if (!(t->scale >= 0.0) || !isfinite(t->scale)) return fail_inval("attention: scale must be finite and not negative");
    if (t->offsets && (t->batch != 1 || t->queries != t->keys || t->sequences < 0 || t->sequences > most))
        return fail_inval("attention: packed sequences are one batch of as many queries as keys");
    if (t->offsets && t->key_lengths) return fail_inval("attention: either offsets or key_lengths");
    if (t->key_lengths && !aligned(t->key_lengths, t->lengths_int64 ? 8 : 4))
        return fail_inval("attention: key_lengths must be aligned");
    if (t->offsets && !aligned(t->offsets, t->offsets_int64 ? 8 : 4))
        return fail_inval("attention: offsets must be aligned");
    return GEFEN_OK;
}
int check_tensor(const gefen_attention_task& t, const void* p, int64_t numel, const char* name) {
    if (numel && !p) return fail_inval("attention: %s is missing", name);
    if (!aligned(p, dtype_size(t.dtype))) return fail_inval("attention: %s must be aligned to its elements", name);
    return GEFEN_OK;
}
int check_floats(const void* p, const char* name) {
    if (!p || !aligned(p, 4)) return fail_inval("attention: %s must be aligned float32 memory", name);
    return GEFEN_OK;
}

Params params_of(const gefen_attention_task& t) {
    Params a{};
    auto view = [](const void* p, const int64_t* s) { return View{const_cast<void*>(p), s[0], s[1], s[2]}; };
    auto dense = [&](void* p, int64_t rows, int64_t heads) {
        return View{p, rows * heads * t.width, heads * t.width, t.width};
    };
    a.q = view(t.query, t.query_strides);
    a.k = view(t.key, t.key_strides);
    a.v = view(t.value, t.value_strides);
    a.go = view(t.grad_out, t.grad_out_strides);
    a.o = dense(t.out, t.queries, t.heads);
    a.gq = dense(t.grad_query, t.queries, t.heads);
    a.gk = dense(t.grad_key, t.keys, t.kv_heads);
    a.gv = dense(t.grad_value, t.keys, t.kv_heads);
    a.lse = t.lse;
    a.key_lengths = t.key_lengths;
    a.offsets = t.offsets;
    a.lengths64 = t.lengths_int64;
    a.offsets64 = t.offsets_int64;
    a.sequences = (int32_t)t.sequences;
    a.batch = (int32_t)t.batch;
    a.queries = (int32_t)t.queries;
    a.keys = (int32_t)t.keys;
    a.kv_heads = (int32_t)t.kv_heads;
    a.group = (int32_t)(t.heads / t.kv_heads);
    a.width = (int32_t)t.width;
    a.causal = t.causal;
    a.rows = a.queries * a.group;
    // 2^(31 + s) / group rounded up, s = ceil(log2 group): exact quotients below 2^31
    int s = 0;
    while ((1 << s) < a.group) ++s;
    a.div_shift = 31 + s;
    a.div_mul = (uint32_t)((((uint64_t)1 << a.div_shift) + a.group - 1) / a.group);
    a.scale = (float)t.scale;
    a.c = (float)(t.scale * 1.4426950408889634);
    return a;
}

}  // namespace attn
}  // namespace gefen

using namespace gefen;
using namespace gefen::attn;

namespace {
int check_workspace(const void* workspace, size_t bytes, size_t need) {
    if (need && (!workspace || !aligned(workspace, 16) || bytes < need))
        return fail_inval("attention: workspace too small, missing or not aligned to 16 bytes");
    return GEFEN_OK;
}
}  // namespace

extern "C" size_t gefen_attention_forward_workspace_size(const gefen_attention_task* task) {
    if (check_task(task) != GEFEN_OK) return 0;
    return (size_t)partial_count(kForwardPass, *task) * 4;
}

extern "C" int gefen_attention_forward(const gefen_attention_task* task, void* workspace, size_t workspace_bytes,
                                       gefen_stream_t stream) {
    if (int rc = check_task(task)) return rc;
    const gefen_attention_task& t = *task;
    const int64_t nq = out_count(kForwardPass, t), nk = out_count(kKeysPass, t);
    if (int rc = check_tensor(t, t.query, nq, "query")) return rc;
    if (int rc = check_tensor(t, t.key, nk, "key")) return rc;
    if (int rc = check_tensor(t, t.value, nk, "value")) return rc;
    if (int rc = check_tensor(t, t.out, nq, "out")) return rc;
    if (t.lse && !aligned(t.lse, 4)) return fail_inval("attention: lse must be aligned float32 memory");
    if (int rc = check_workspace(workspace, workspace_bytes, gefen_attention_forward_workspace_size(task))) return rc;
    if (nq == 0) return GEFEN_OK;
    Params a = params_of(t);
    set_parts(kForwardPass, t, static_cast<float*>(workspace), &a);
    return launch_type(t.dtype, kForwardPass, a, static_cast<hipStream_t>(stream));
}

extern "C" size_t gefen_attention_backward_workspace_size(const gefen_attention_task* task) {
    if (check_task(task) != GEFEN_OK) return 0;
    const int64_t range = task->dtype == GEFEN_F16 ? 2 * task->batch * task->kv_heads * kRangeParts : 0;
    const int64_t q = partial_count(kQueriesPass, *task), k = partial_count(kKeysPass, *task);
    return (size_t)(round16(stat_count(*task)) + round16(range) + (q > k ? q : k) + 4) * 4;
}

extern "C" int gefen_attention_backward(const gefen_attention_task* task, void* workspace, size_t workspace_bytes,
                                        gefen_stream_t stream) {
    if (int rc = check_task(task)) return rc;
    const gefen_attention_task& t = *task;
    const int64_t nq = out_count(kForwardPass, t), nk = out_count(kKeysPass, t);
    if (int rc = check_tensor(t, t.query, nq, "query")) return rc;
    if (int rc = check_tensor(t, t.key, nk, "key")) return rc;
    if (int rc = check_tensor(t, t.value, nk, "value")) return rc;
    if (int rc = check_tensor(t, t.out, nq, "out")) return rc;
    if (int rc = check_tensor(t, t.grad_out, nq, "grad_out")) return rc;
    if (int rc = check_tensor(t, t.grad_query, nq, "grad_query")) return rc;
    const bool key_grads = t.grad_key || t.grad_value;
    if (int rc = check_tensor(t, t.grad_key, key_grads ? nk : 0, "grad_key")) return rc;
    if (int rc = check_tensor(t, t.grad_value, key_grads ? nk : 0, "grad_value")) return rc;
    if (nq)
        if (int rc = check_floats(t.lse, "lse")) return rc;
    if (int rc = check_workspace(workspace, workspace_bytes, gefen_attention_backward_workspace_size(task))) return rc;
    Params a = params_of(t);
    a.delta = static_cast<float*>(workspace);
    a.range = a.delta + round16(stat_count(t));
    // the two passes follow each other: their parts share the memory behind
    float* const parts = a.range + (t.dtype == GEFEN_F16 ? round16(2 * t.batch * t.kv_heads * kRangeParts) : 0);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (t.dtype == GEFEN_F16 && nq && nk) {
        if (int rc = launch_range<f16_t>(a, st)) return rc;
    }
    if (nq) {
        set_parts(kQueriesPass, t, parts, &a);
        if (int rc = launch_type(t.dtype, kQueriesPass, a, st)) return rc;
    }
    if (nk && key_grads) {
        set_parts(kKeysPass, t, parts, &a);
        if (int rc = launch_type(t.dtype, kKeysPass, a, st)) return rc;
    }
    return GEFEN_OK;
}
