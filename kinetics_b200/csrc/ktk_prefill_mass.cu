// Attention of new tokens over a paged cache that also adds up, for every cached token, what the last `window` of them give it:
//     mass'[r, h, t] = decay mass[r, h, t] + sum over (token, head) rows of 2^(s_row(t) - lse_row)
// The attention itself is that of ktk_prefill.cu, which writes the rows' denominators down; the weights are then summed by keys: bf16
// in ktk_prefill_mass_umma.cu, fp32 here.
#include "ktk_prefill_mass.cuh"

namespace ktk {

constexpr int kPsKeys = 64, kPsRows = 64;     // keys of a CTA, rows of a tile
constexpr int kPsThreads = 256;               // 16 x 16, four keys and four rows each
constexpr int kPsDims = 32;                   // dimensions of a stage
constexpr int kPsLd = kPsKeys + 4;            // floats between dimensions in shared memory (16-byte aligned, writes spread over banks)

// One CTA per (sequence, kv head, 64 keys): tiles of 64 rows against its keys, 32 dimensions at a time through shared memory
// ([dimension][key or row]), four by four products in registers.  FMA-bound: 4096 cycles per tile and SM.
__global__ void __launch_bounds__(kPsThreads)
prefill_mass_simt_kernel(const PrefillMassParams p, int chunks) {
    __shared__ __align__(16) float keys[kPsDims][kPsLd], rows[kPsDims][kPsLd];
    __shared__ float row_lse[kPsRows], sums[16][kPsKeys];
    wait_for_front();
    const int64_t unit = blockIdx.x / chunks;
    const int part = (int)(blockIdx.x % chunks), tid = threadIdx.x, tk = tid % 16, tr = tid / 16;
    const int b = (int)(unit / p.Hkv), h = (int)(unit % p.Hkv), G = p.G, Hq = p.Hkv * G;
    MassSequence s;
    if (!mass_sequence(p, b, part == 0 && h == 0, s)) return;
    const int t0 = part * kPsKeys;
    if (t0 >= s.sp.total) return;
    // a thread brings a quarter of a key's and of a row's dimensions of a stage: 8 floats
    const int mine = tid / 4, quarter = tid % 4 * 8;
    const float* key = nullptr;
    if (t0 + mine < s.sp.total) {
        int e, slot;
        page_of_pos(t0 + mine, s.sp.first_fill, e, slot);
        const int64_t page = p.kv_indices[s.sp.start + e];
        if (page < 0 || page >= p.num_pages) report(p.status, KTK_STATUS_BAD_PAGE);
        else key = (const float*)p.cache + ((page * 2 * kPageSize + slot) * p.Hkv + h) * kHeadDim;
    }
    // tokens that are counted and see the chunk's first key
    const int tok0 = max(s.counted, t0 - s.base_pos), n_rows = (s.n_new - tok0) * G;
    float sum[4] = {};
    for (int r0 = 0; r0 < n_rows; r0 += kPsRows) {
        const int r = r0 + mine;
        const float* row = r < n_rows ? (const float*)p.q + ((int64_t)(s.q0 + tok0 + r / G) * Hq + h * G + r % G) * kHeadDim : nullptr;
        float dot[4][4] = {};                     // [row][key]
        for (int d0 = 0; d0 < kHeadDim; d0 += kPsDims) {
            float kv[8] = {}, qv[8] = {};
            if (key) load8(key + d0 + quarter, kv);
            if (row) load8(row + d0 + quarter, qv);
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                keys[quarter + i][mine] = kv[i];
                rows[quarter + i][mine] = qv[i];
            }
            if (d0 == 0 && tid < kPsRows)
                row_lse[tid] = r0 + tid < n_rows ? ((const float*)p.lse)[(int64_t)(s.q0 + tok0 + (r0 + tid) / G) * Hq + h * G + (r0 + tid) % G] : 0.0f;
            __syncthreads();
#pragma unroll
            for (int d = 0; d < kPsDims; ++d) {
                const float4 k4 = *reinterpret_cast<const float4*>(&keys[d][tk * 4]), q4 = *reinterpret_cast<const float4*>(&rows[d][tr * 4]);
                const float k[4] = {k4.x, k4.y, k4.z, k4.w}, q[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) dot[i][j] = fmaf(q[i], k[j], dot[i][j]);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = r0 + tr * 4 + i, sees = at < n_rows ? s.base_pos + tok0 + at / G : -1;
            const float lse = row_lse[tr * 4 + i];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (t0 + tk * 4 + j <= sees) sum[j] += exp2f(fmaf(dot[i][j], p.scale_log2, lse));
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[tr][tk * 4 + j] = sum[j];
    __syncthreads();
    if (tid < kPsKeys && t0 + tid < s.sp.total) {
        const int t = t0 + tid;
        float total = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) total += sums[i][tid];
        const int64_t at = ((int64_t)s.row * p.Hkv + h) * p.m.stride + t;
        p.m.out[at] = t >= s.base_pos ? total : fmaf(p.m.decay, p.m.in[at], total);
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
    KTK_CUDA_TRY(launch_behind(false, prefill_mass_simt_kernel, (unsigned)ctas, kPsThreads, 0, st, p, (int)chunks), who);
    return KTK_OK;
}
