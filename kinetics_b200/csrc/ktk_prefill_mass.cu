// Attention of new tokens over a paged cache that also adds up, for every cached token, what the last `window` of them give it:
//     mass'[r, h, t] = decay mass[r, h, t] + sum over (token, head) rows of 2^(s_row(t) - lse_row)
// The attention itself is that of ktk_prefill.cu, which writes the rows' denominators down; the weights are then summed by keys: bf16
// in ktk_prefill_mass_umma.cu, fp32 here.
#include "ktk_prefill_mass.cuh"

namespace ktk {

constexpr int kPsKeys = 128;    // keys of a CTA, one per thread
constexpr int kPsRows = 32;     // rows of a stage

// One CTA per (sequence, kv head, 128 keys): a thread holds a key and walks the rows that see it.
__global__ void __launch_bounds__(kPsKeys)
prefill_mass_simt_kernel(const PrefillMassParams p, int chunks) {
    __shared__ __align__(16) float rows[kPsRows][kHeadDim];
    __shared__ float row_lse[kPsRows];
    wait_for_front();
    const int64_t unit = blockIdx.x / chunks;
    const int part = (int)(blockIdx.x % chunks), tid = threadIdx.x;
    const int b = (int)(unit / p.Hkv), h = (int)(unit % p.Hkv), G = p.G, Hq = p.Hkv * G;
    MassSequence s;
    if (!mass_sequence(p, b, part == 0 && h == 0, s)) return;
    const int t0 = part * kPsKeys, t = t0 + tid;
    if (t0 >= s.sp.total) return;
    float key[kHeadDim];
    bool on = t < s.sp.total;
    if (on) {
        int e, slot;
        page_of_pos(t, s.sp.first_fill, e, slot);
        const int64_t page = p.kv_indices[s.sp.start + e];
        if (page < 0 || page >= p.num_pages) {
            report(p.status, KTK_STATUS_BAD_PAGE);
            on = false;
        } else {
            const float* src = (const float*)p.cache + ((page * 2 * kPageSize + slot) * p.Hkv + h) * kHeadDim;
#pragma unroll
            for (int i = 0; i < kHeadDim; i += 8) load8(src + i, *reinterpret_cast<float(*)[8]>(key + i));
        }
    }
    if (!on) {
#pragma unroll
        for (int i = 0; i < kHeadDim; ++i) key[i] = 0.0f;
    }
    // tokens that are counted and see the chunk's first key
    const int tok0 = max(s.counted, t0 - s.base_pos);
    const int n_rows = (s.n_new - tok0) * G;
    float sum = 0.0f;
    for (int r0 = 0; r0 < n_rows; r0 += kPsRows) {
        const int n = n_rows - r0 < kPsRows ? n_rows - r0 : kPsRows;
        __syncthreads();
        for (int i = tid; i < n * (kHeadDim / 8); i += kPsKeys) {
            const int r = i / (kHeadDim / 8), c = i % (kHeadDim / 8), tok = tok0 + (r0 + r) / G, g = (r0 + r) % G;
            float f[8];
            load8((const float*)p.q + ((int64_t)(s.q0 + tok) * Hq + h * G + g) * kHeadDim + c * 8, f);
#pragma unroll
            for (int k = 0; k < 8; ++k) rows[r][c * 8 + k] = f[k];
        }
        if (tid < n) row_lse[tid] = ((const float*)p.lse)[(int64_t)(s.q0 + tok0 + (r0 + tid) / G) * Hq + h * G + (r0 + tid) % G];
        __syncthreads();
        for (int r = 0; r < n; ++r) {
            float dot[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < kHeadDim; i += 4) {
                const float4 v = *reinterpret_cast<const float4*>(&rows[r][i]);
                dot[0] = fmaf(v.x, key[i], dot[0]);
                dot[1] = fmaf(v.y, key[i + 1], dot[1]);
                dot[2] = fmaf(v.z, key[i + 2], dot[2]);
                dot[3] = fmaf(v.w, key[i + 3], dot[3]);
            }
            const float x = (dot[0] + dot[1]) + (dot[2] + dot[3]);
            if (t <= s.base_pos + tok0 + (r0 + r) / G) sum += exp2f(x * p.scale_log2 + row_lse[r]);
        }
    }
    if (on) {
        const int64_t at = ((int64_t)s.row * p.Hkv + h) * p.m.stride + t;
        p.m.out[at] = t >= s.base_pos ? sum : fmaf(p.m.decay, p.m.in[at], sum);
    }
}

}  // namespace ktk

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
    const size_t behind = shape->dtype == KTK_F32
                              ? ktk_prefill_workspace_bytes(total_new_tokens, shape->dtype, KTK_VARIANT_AUTO)
                              : mass_plan(shape, max_new_tokens, max_pages_per_seq, total_pages, window).partial * sizeof(float);
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
    if (!(sm_scale != 0.0f && sm_scale - sm_scale == 0.0f)) {
        set_error("%s: sm_scale %g: finite, and not 0", who, (double)sm_scale);
        return KTK_ERR_ARG;
    }
    if (total_new_tokens < 0 || max_new_tokens < 1 || window < 0 || max_pages_per_seq < 1) {
        set_error("%s: total_new_tokens %lld, max_new_tokens %d, window %d, max_pages_per_seq %lld", who,
                  (long long)total_new_tokens, max_new_tokens, window, (long long)max_pages_per_seq);
        return KTK_ERR_ARG;
    }
    const View view = make_view(view_in);
    if (view.page_count) total_pages = -1;
    const size_t need = ktk_prefill_mass_workspace_bytes(s, total_new_tokens, max_new_tokens, max_pages_per_seq, total_pages, window);
    if (workspace == nullptr || workspace_bytes < need) {
        set_error("%s: workspace of %zu bytes needed, got %zu", who, need, workspace ? workspace_bytes : (size_t)0);
        return KTK_ERR_WORKSPACE;
    }
    const int64_t chunks = (max_pages_per_seq * kPageSize + kPsKeys - 1) / kPsKeys, ctas = chunks * s->batch * s->num_kv_heads;
    if (max_pages_per_seq > (1 << 27) || ctas > 2147483647LL) {
        set_error("%s: batch * num_kv_heads * max_pages_per_seq exceeds the grid limit", who);
        return KTK_ERR_TOO_LARGE;
    }
    void* lse = workspace;
    char* behind = (char*)workspace + lse_bytes(s, total_new_tokens);
    rc = prefill_attention(who, q, q_indptr, total_new_tokens, max_new_tokens, kv_cache, kv_indices, kv_indptr, kv_last_page_len,
                           view_in, sm_scale, o, lse, behind, need - lse_bytes(s, total_new_tokens), KTK_VARIANT_AUTO, s, status, stream);
    if (rc != KTK_OK) return rc;
    PrefillMassParams p{};
    p.q = q; p.cache = kv_cache; p.q_indptr = q_indptr; p.kv_indices = kv_indices; p.kv_indptr = kv_indptr;
    p.kv_last_page_len = kv_last_page_len; p.page_count = view.page_count; p.sink_tokens = view.sink_tokens;
    p.batch = s->batch; p.Hkv = s->num_kv_heads; p.G = s->group_size; p.num_pages = s->num_pages; p.total_new = total_new_tokens;
    p.scale_log2 = sm_scale * kLog2e; p.lse = lse; p.window = window; p.status = status;
    p.m.in = mass->in; p.m.out = mass->out; p.m.stride = mass->stride; p.m.rows = mass->rows;
    p.m.slot_index = view.slot_index; p.m.decay = mass->decay;
    cudaStream_t st = (cudaStream_t)stream;
    if (s->dtype == KTK_BF16) {
        const MassPlan plan = mass_plan(s, max_new_tokens, max_pages_per_seq, total_pages, window);
        p.splits = plan.splits;
        p.partial = (float*)behind;
        return launch_prefill_mass_umma(p, plan.groups, st);
    }
    KTK_CUDA_TRY(launch_behind(false, prefill_mass_simt_kernel, (unsigned)ctas, kPsKeys, 0, st, p, (int)chunks), who);
    return KTK_OK;
}
