// Attention of new tokens over a paged cache that also adds up, for every cached token, what the last `window` of them give it:
//     mass'[r, h, t] = decay mass[r, h, t] + sum over (token, head) rows of 2^(s_row(t) - lse_row)
// The attention itself is that of ktk_prefill.cu, which writes the rows' denominators down; the weights are then summed by keys.
#include "ktk_decode_mma.cuh"

namespace ktk {

struct PrefillMassParams {
    const void* q;
    const void* cache;
    const int32_t* q_indptr;
    const int32_t* kv_indices;
    const int32_t* kv_indptr;
    const int32_t* kv_last_page_len;
    const int32_t* page_count;
    int sink_tokens;
    int batch, Hkv, G;
    int64_t num_pages;
    float scale_log2;
    const float* lse;           // [total_new, Hq]
    int window;
    int32_t* status;
    MassParams m;
};

constexpr int kPmKeys = 128;    // keys of a CTA, one per thread
constexpr int kPmRows = 32;     // rows of a stage

// What the CTA's sequence is, and where it lies in the mass array; false: nothing to do
struct MassSequence {
    SeqPages sp;
    int q0, n_new, base_pos, row;
};
__device__ __forceinline__ bool mass_sequence(const PrefillMassParams& p, int b, bool first, MassSequence& s) {
    s.q0 = p.q_indptr[b];
    s.n_new = p.q_indptr[b + 1] - s.q0;
    if (s.n_new <= 0) return false;
    s.sp = seq_pages(p.kv_indptr, p.page_count, p.kv_last_page_len, p.sink_tokens, b);
    s.base_pos = s.sp.total - s.n_new;
    s.row = p.m.slot_index ? p.m.slot_index[b] : b;
    if (s.sp.bad || s.base_pos < 0 || s.row < 0 || s.row >= p.m.rows || s.sp.total > p.m.stride) {
        if (first && threadIdx.x == 0) report(p.status, KTK_STATUS_BAD_TABLE);
        return false;
    }
    return true;
}

// One CTA per (sequence, kv head, 128 keys): a thread holds a key and walks the rows that see it.
template <typename T>
__global__ void __launch_bounds__(kPmKeys)
prefill_mass_simt_kernel(const PrefillMassParams p, int chunks) {
    __shared__ __align__(16) float rows[kPmRows][kHeadDim];
    __shared__ float row_lse[kPmRows];
    wait_for_front();
    const int64_t unit = blockIdx.x / chunks;
    const int part = (int)(blockIdx.x % chunks), tid = threadIdx.x;
    const int b = (int)(unit / p.Hkv), h = (int)(unit % p.Hkv), G = p.G, Hq = p.Hkv * G;
    MassSequence s;
    if (!mass_sequence(p, b, part == 0 && h == 0, s)) return;
    const int t0 = part * kPmKeys, t = t0 + tid;
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
            const T* src = (const T*)p.cache + ((page * 2 * kPageSize + slot) * p.Hkv + h) * kHeadDim;
#pragma unroll
            for (int i = 0; i < kHeadDim; i += 8) load8(src + i, *reinterpret_cast<float(*)[8]>(key + i));
        }
    }
    if (!on) {
#pragma unroll
        for (int i = 0; i < kHeadDim; ++i) key[i] = 0.0f;
    }
    // tokens that are counted and see the chunk's first key
    int tok0 = p.window > 0 && p.window < s.n_new ? s.n_new - p.window : 0;
    if (t0 - s.base_pos > tok0) tok0 = t0 - s.base_pos;
    const int n_rows = (s.n_new - tok0) * G;
    float sum = 0.0f;
    for (int r0 = 0; r0 < n_rows; r0 += kPmRows) {
        const int n = n_rows - r0 < kPmRows ? n_rows - r0 : kPmRows;
        __syncthreads();
        for (int i = tid; i < n * (kHeadDim / 8); i += kPmKeys) {
            const int r = i / (kHeadDim / 8), c = i % (kHeadDim / 8), tok = tok0 + (r0 + r) / G, g = (r0 + r) % G;
            float f[8];
            load8((const T*)p.q + ((int64_t)(s.q0 + tok) * Hq + h * G + g) * kHeadDim + c * 8, f);
#pragma unroll
            for (int k = 0; k < 8; ++k) rows[r][c * 8 + k] = f[k];
        }
        if (tid < n) row_lse[tid] = p.lse[(int64_t)(s.q0 + tok0 + (r0 + tid) / G) * Hq + h * G + (r0 + tid) % G];
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
            if (t <= s.base_pos + tok0 + (r0 + r) / G) sum += exp2f(x * p.scale_log2 - row_lse[r]);
        }
    }
    if (on) {
        const int64_t at = ((int64_t)s.row * p.Hkv + h) * p.m.stride + t;
        p.m.out[at] = t >= s.base_pos ? sum : fmaf(p.m.decay, p.m.in[at], sum);
    }
}

}  // namespace ktk

using namespace ktk;

static size_t lse_bytes(const ktk_shape* s, int64_t total_new) {
    return ((size_t)total_new * s->num_kv_heads * s->group_size * sizeof(float) + 255) / 256 * 256;
}

extern "C" size_t ktk_prefill_mass_workspace_bytes(const ktk_shape* shape, int64_t total_new_tokens) {
    if (check_shape(shape, "ktk_prefill_mass_workspace_bytes") != KTK_OK || total_new_tokens <= 0) return 0;
    return lse_bytes(shape, total_new_tokens) + ktk_prefill_workspace_bytes(total_new_tokens, shape->dtype, KTK_VARIANT_AUTO);
}

extern "C" int ktk_prefill_attention_mass(const void* q, const int32_t* q_indptr, int64_t total_new_tokens,
                                          int32_t max_new_tokens, const void* kv_cache, const int32_t* kv_indices,
                                          const int32_t* kv_indptr, const int32_t* kv_last_page_len, const ktk_view* view_in,
                                          int64_t max_tokens, int32_t window, float sm_scale, const ktk_mass* mass, void* o,
                                          void* workspace, size_t workspace_bytes, const ktk_shape* s, int32_t* status,
                                          void* stream) {
    const char* who = "ktk_prefill_attention_mass";
    int rc = check_shape(s, who);
    if (rc == KTK_OK) rc = check_view(view_in, who);
    if (rc != KTK_OK) return rc;
    if (s->batch == 0 || total_new_tokens == 0) return KTK_OK;
    if ((rc = check_mass(mass, who)) != KTK_OK || (rc = check_aligned({q, kv_cache, o, workspace}, who)) != KTK_OK ||
        (rc = check_apart(mass->in, mass->out, (size_t)mass->rows * s->num_kv_heads * mass->stride * sizeof(float), who, "mass")) != KTK_OK)
        return rc;
    if (total_new_tokens < 0 || window < 0 || max_tokens < 1) {
        set_error("%s: total_new_tokens %lld, window %d, max_tokens %lld", who, (long long)total_new_tokens, window, (long long)max_tokens);
        return KTK_ERR_ARG;
    }
    const size_t need = ktk_prefill_mass_workspace_bytes(s, total_new_tokens);
    if (workspace == nullptr || workspace_bytes < need) {
        set_error("%s: workspace of %zu bytes needed, got %zu", who, need, workspace ? workspace_bytes : (size_t)0);
        return KTK_ERR_WORKSPACE;
    }
    if (max_tokens > mass->stride) max_tokens = mass->stride;          // longer sequences are reported
    const int64_t chunks = (max_tokens + kPmKeys - 1) / kPmKeys, ctas = chunks * s->batch * s->num_kv_heads;
    if (ctas > 2147483647LL) {
        set_error("%s: batch * num_kv_heads * max_tokens exceeds the grid limit", who);
        return KTK_ERR_TOO_LARGE;
    }
    float* lse = (float*)workspace;
    const size_t behind = lse_bytes(s, total_new_tokens);
    rc = prefill_attention(who, q, q_indptr, total_new_tokens, max_new_tokens, kv_cache, kv_indices, kv_indptr, kv_last_page_len,
                           view_in, sm_scale, o, lse, (char*)workspace + behind, workspace_bytes - behind, KTK_VARIANT_AUTO, s,
                           status, stream);
    if (rc != KTK_OK) return rc;
    const View view = make_view(view_in);
    PrefillMassParams p;
    p.q = q; p.cache = kv_cache; p.q_indptr = q_indptr; p.kv_indices = kv_indices; p.kv_indptr = kv_indptr;
    p.kv_last_page_len = kv_last_page_len; p.page_count = view.page_count; p.sink_tokens = view.sink_tokens;
    p.batch = s->batch; p.Hkv = s->num_kv_heads; p.G = s->group_size; p.num_pages = s->num_pages;
    p.scale_log2 = sm_scale * kLog2e; p.lse = lse; p.window = window; p.status = status;
    p.m = MassParams{};
    p.m.in = mass->in; p.m.out = mass->out; p.m.stride = mass->stride; p.m.rows = mass->rows;
    p.m.slot_index = view.slot_index; p.m.decay = mass->decay;
    const auto kernel = s->dtype == KTK_F32 ? prefill_mass_simt_kernel<float> : prefill_mass_simt_kernel<__nv_bfloat16>;
    KTK_CUDA_TRY(launch_behind(false, kernel, (unsigned)ctas, kPmKeys, 0, (cudaStream_t)stream, p, (int)chunks), who);
    return KTK_OK;
}
