// Attention of new tokens over a paged cache that also adds up, for every cached token, what the last `window` of them give it:
//     mass'[r, h, t] = decay mass[r, h, t] + sum over (token, head) rows of 2^(s_row(t) - lse_row)
// The attention writes the rows' denominators down, a second kernel sums the weights by keys: bf16 in ktk_prefill_umma.cu and
// ktk_prefill_mass_umma.cu, fp32 in ktk_prefill_mass_f32.cu.
#include "ktk_prefill_mass.cuh"

using namespace ktk;

namespace {
size_t up(size_t bytes) { return (bytes + 255) / 256 * 256; }
size_t lse_bytes(const ktk_shape* s, int64_t total_new) {
    return up((size_t)total_new * s->num_kv_heads * s->group_size * (s->dtype == KTK_F32 ? sizeof(float) : 16));
}
}  // namespace

extern "C" size_t ktk_prefill_mass_workspace_bytes(const ktk_shape* shape, int64_t total_new_tokens, int32_t max_new_tokens,
                                                   int64_t max_pages_per_seq, int64_t total_pages, int32_t window) {
    if (check_shape(shape, "ktk_prefill_mass_workspace_bytes") != KTK_OK || shape->batch == 0 || total_new_tokens <= 0 ||
        max_new_tokens < 1 || max_pages_per_seq < 1)
        return 0;
    if (max_new_tokens > total_new_tokens) max_new_tokens = (int32_t)total_new_tokens;
    const size_t behind = shape->dtype == KTK_F32 ? 0 : mass_plan(shape, max_new_tokens, max_pages_per_seq, total_pages, window).partial * sizeof(float);
    return lse_bytes(shape, total_new_tokens) + up(behind);
}

extern "C" int ktk_prefill_attention_mass(const void* q, const int32_t* q_indptr, int64_t total_new_tokens,
                                          int32_t max_new_tokens, const void* kv_cache, const int32_t* kv_indices,
                                          const int32_t* kv_indptr, const int32_t* kv_last_page_len, const ktk_view* view_in,
                                          int64_t max_pages_per_seq, int64_t total_pages, int32_t window, float sm_scale,
                                          const ktk_mass* mass, void* o, void* workspace, size_t workspace_bytes,
                                          const ktk_shape* s, int32_t* status, void* stream) {
    const char* who = "ktk_prefill_attention_mass";
    int rc = check_shape(s, who);
    if (rc == KTK_OK) rc = check_view(view_in, who);
    if (rc != KTK_OK) return rc;
    if (s->batch == 0 || total_new_tokens == 0) return KTK_OK;
    if ((rc = check_mass(mass, who)) != KTK_OK || (rc = check_aligned({q, kv_cache, o, workspace}, who)) != KTK_OK ||
        (rc = check_apart(mass->in, mass->out, (size_t)mass->rows * s->num_kv_heads * mass->stride * sizeof(float), who, "mass")) != KTK_OK)
        return rc;
    if (!(sm_scale >= 1e-30f && sm_scale - sm_scale == 0.0f)) {          // denominators are divided by it
        set_error("%s: sm_scale %g: finite, at least 1e-30", who, (double)sm_scale);
        return KTK_ERR_ARG;
    }
    if (total_new_tokens < 0 || max_new_tokens < 1 || window < 0 || max_pages_per_seq < 1) {
        set_error("%s: total_new_tokens %lld, max_new_tokens %d, window %d, max_pages_per_seq %lld", who,
                  (long long)total_new_tokens, max_new_tokens, window, (long long)max_pages_per_seq);
        return KTK_ERR_ARG;
    }
    if (max_new_tokens > total_new_tokens) max_new_tokens = (int32_t)total_new_tokens;
    const View view = make_view(view_in);
    if (view.page_count) total_pages = -1;
    const size_t need = ktk_prefill_mass_workspace_bytes(s, total_new_tokens, max_new_tokens, max_pages_per_seq, total_pages, window);
    if (workspace == nullptr || workspace_bytes < need) {
        set_error("%s: workspace of %zu bytes needed, got %zu", who, need, workspace ? workspace_bytes : (size_t)0);
        return KTK_ERR_WORKSPACE;
    }
    if (max_pages_per_seq > kMassMaxPages) {
        set_error("%s: %lld pages per sequence, at most %d", who, (long long)max_pages_per_seq, kMassMaxPages);
        return KTK_ERR_TOO_LARGE;
    }
    if (!q || !q_indptr || !kv_cache || !kv_indices || !kv_indptr || !kv_last_page_len || !o) {
        set_error("%s: null pointer argument", who);
        return KTK_ERR_ARG;
    }
    // the attention may be done with a query when it writes its output, the weights are not
    const size_t bytes = (size_t)total_new_tokens * s->num_kv_heads * s->group_size * kHeadDim * (s->dtype == KTK_F32 ? 4 : 2);
    if ((uintptr_t)q < (uintptr_t)o + bytes && (uintptr_t)o < (uintptr_t)q + bytes) {
        set_error("%s: q and o overlap", who);
        return KTK_ERR_ARG;
    }
    void* lse = workspace;
    PrefillMassParams p{};
    p.q = q; p.o = o; p.cache = kv_cache; p.q_indptr = q_indptr; p.kv_indices = kv_indices; p.kv_indptr = kv_indptr;
    p.kv_last_page_len = kv_last_page_len; p.page_count = view.page_count; p.sink_tokens = view.sink_tokens;
    p.batch = s->batch; p.Hkv = s->num_kv_heads; p.G = s->group_size; p.num_pages = s->num_pages; p.total_new = total_new_tokens;
    p.max_new = max_new_tokens; p.max_pages = (int)max_pages_per_seq;
    p.scale_log2 = sm_scale * kLog2e; p.lse = lse; p.window = window; p.status = status;
    p.m.in = mass->in; p.m.out = mass->out; p.m.stride = mass->stride; p.m.rows = mass->rows;
    p.m.slot_index = view.slot_index; p.m.decay = mass->decay;
    cudaStream_t st = (cudaStream_t)stream;
    if (s->dtype == KTK_F32) return launch_prefill_mass_f32(p, st);
    rc = prefill_attention(who, q, q_indptr, total_new_tokens, max_new_tokens, kv_cache, kv_indices, kv_indptr, kv_last_page_len,
                           view_in, sm_scale, o, lse, max_pages_per_seq, nullptr, 0, KTK_VARIANT_AUTO, s, status, stream);
    if (rc != KTK_OK) return rc;
    const MassPlan plan = mass_plan(s, max_new_tokens, max_pages_per_seq, total_pages, window);
    p.splits = plan.splits;
    p.partial = (float*)((char*)workspace + lse_bytes(s, total_new_tokens));
    return launch_prefill_mass_umma(p, plan.groups, st);
}
