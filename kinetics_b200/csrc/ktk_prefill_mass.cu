// Attention of new tokens over a paged cache that also adds up, for every cached token, what the last `window` of them give it:
//     mass'[r, h, t] = decay mass[r, h, t] + sum over (token, head) rows of 2^(s_row(t) - lse_row)
// The attention itself is that of ktk_prefill.cu, which writes the rows' denominators down; the weights are then summed by keys: bf16
// in ktk_prefill_mass_umma.cu, fp32 here.
#include <cooperative_groups.h>

#include "ktk_prefill_mass.cuh"

namespace ktk {

constexpr int kPsKeys = 32, kPsRows = 64;     // keys of a CTA, rows of a tile
constexpr int kPsThreads = 128;               // 8 x 16, four keys and four rows each
constexpr int kPsLd = kHeadDim + 4;           // floats between keys or rows in shared memory: eight of them lie in different banks
constexpr int kPsSmem = (kPsKeys + 2 * kPsRows) * kPsLd * 4;

// One CTA per (sequence, kv head, 32 keys), its keys and two tiles of 64 rows in shared memory: a tile is multiplied, four by four
// products in a thread's registers, while the next one comes.  Bound by shared memory: 32 cycles per dimension and tile.  Stages of 32
// dimensions instead of whole tiles were bound by the loads' latency, 2 us each.
// Where that leaves SMs idle, a cluster of CTAs takes the tiles in turn and its first one adds the sums.
__global__ void __launch_bounds__(kPsThreads)
prefill_mass_simt_kernel(const PrefillMassParams p, int chunks, int cluster) {
    extern __shared__ __align__(16) float ps_smem[];
    __shared__ float sums[kPsThreads / 8][kPsKeys], totals[kPsKeys];
    float* keys = ps_smem;                        // [key][kPsLd], then [tile][row][kPsLd]
    wait_for_front();
    const int64_t item = blockIdx.x / cluster, unit = item / chunks;
    const int part = (int)(item % chunks), rank = (int)(blockIdx.x % cluster), tid = threadIdx.x, tk = tid % 8, tr = tid / 8;
    const int b = (int)(unit / p.Hkv), h = (int)(unit % p.Hkv), G = p.G, Hq = p.Hkv * G, shift = 31 - __clz(G);    // 1, 2, 4 or 8
    MassSequence s;
    if (!mass_sequence(p, b, part == 0 && h == 0 && rank == 0, s)) return;      // the same for the cluster
    const int t0 = part * kPsKeys;
    if (t0 >= s.sp.total) return;
    // tokens that are counted and see the chunk's first key
    const int tok0 = max(s.counted, t0 - s.base_pos), n_rows = (s.n_new - tok0) * G;
    const auto row_of = [&](int r) { return (int64_t)(s.q0 + tok0 + (r >> shift)) * Hq + h * G + (r & (G - 1)); };
    // a warp brings a key or a row at a time, 16 bytes a lane; places without one get zeros
    const int warp = tid / 32, lane = tid % 32;
    for (int k = warp; k < kPsKeys; k += kPsThreads / 32) {
        const float* src = nullptr;
        if (t0 + k < s.sp.total) {
            int e, slot;
            page_of_pos(t0 + k, s.sp.first_fill, e, slot);
            const int64_t page = p.kv_indices[s.sp.start + e];
            if (page < 0 || page >= p.num_pages) report(p.status, KTK_STATUS_BAD_PAGE);
            else src = (const float*)p.cache + ((page * 2 * kPageSize + slot) * p.Hkv + h) * kHeadDim;
        }
        cp_async16(smem_u32(keys + k * kPsLd + lane * 4), src ? src + lane * 4 : (const float*)p.cache, src ? 16 : 0);
    }
    const auto load_rows = [&](int r0, int tile) {
        float* rows = keys + (kPsKeys + tile * kPsRows) * kPsLd;
        for (int r = warp; r < kPsRows; r += kPsThreads / 32) {
            const bool on = r0 + r < n_rows;
            cp_async16(smem_u32(rows + r * kPsLd + lane * 4), (const float*)p.q + (on ? row_of(r0 + r) * kHeadDim + lane * 4 : 0), on ? 16 : 0);
        }
        cp_async_commit();
    };
    load_rows(rank * kPsRows, 0);
    float sum[4] = {};
    for (int r0 = rank * kPsRows, tile = 0; r0 < n_rows; r0 += cluster * kPsRows, tile ^= 1) {
        if (r0 + cluster * kPsRows < n_rows) load_rows(r0 + cluster * kPsRows, tile ^ 1);
        else cp_async_commit();
        int sees[4];
        float lse[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = r0 + tr + 16 * i;
            sees[i] = r < n_rows ? s.base_pos + tok0 + (r >> shift) : -1;
            lse[i] = r < n_rows ? ((const float*)p.lse)[row_of(r)] : 0.0f;
        }
        cp_async_wait<1>();
        __syncthreads();
        const float* rows = keys + (kPsKeys + tile * kPsRows) * kPsLd;
        float dot[4][4] = {};                     // [row tr + 16 i][key tk + 8 j]
#pragma unroll 4
        for (int d = 0; d < kHeadDim; d += 4) {
            float4 k[4], q[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) k[j] = *reinterpret_cast<const float4*>(keys + (tk + 8 * j) * kPsLd + d);
#pragma unroll
            for (int i = 0; i < 4; ++i) q[i] = *reinterpret_cast<const float4*>(rows + (tr + 16 * i) * kPsLd + d);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    dot[i][j] = fmaf(q[i].x, k[j].x, dot[i][j]);
                    dot[i][j] = fmaf(q[i].y, k[j].y, dot[i][j]);
                    dot[i][j] = fmaf(q[i].z, k[j].z, dot[i][j]);
                    dot[i][j] = fmaf(q[i].w, k[j].w, dot[i][j]);
                }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (t0 + tk + 8 * j <= sees[i]) sum[j] += exp2f(fmaf(dot[i][j], p.scale_log2, lse[i]));
        __syncthreads();                          // the tile is free
    }
    cp_async_wait<0>();
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[tr][tk + 8 * j] = sum[j];
    __syncthreads();
    float total = 0.0f;
    if (tid < kPsKeys) {
#pragma unroll
        for (int i = 0; i < kPsThreads / 8; ++i) total += sums[i][tid];
        totals[tid] = total;
    }
    if (cluster > 1) {
        auto cl = cooperative_groups::this_cluster();
        cl.sync();
        if (rank == 0 && tid < kPsKeys)
            for (int i = 1; i < cluster; ++i) total += *cl.map_shared_rank(&totals[tid], i);
        cl.sync();                                // the others stay until theirs are read
    }
    if (rank == 0 && tid < kPsKeys && t0 + tid < s.sp.total) {
        const int t = t0 + tid;
        const int64_t at = ((int64_t)s.row * p.Hkv + h) * p.m.stride + t;
        p.m.out[at] = t >= s.base_pos ? total : fmaf(p.m.decay, p.m.in[at], total);
    }
}

static int launch_prefill_mass_simt(const PrefillMassParams& p, int64_t ctas, int chunks, int max_new, cudaStream_t st) {
    const char* who = "ktk_prefill_attention_mass";
    const int64_t rows = (int64_t)(p.window > 0 && p.window < max_new ? p.window : max_new) * p.G;
    int cluster = 1;
    while (cluster < 8 && ctas * cluster <= sm_count() && rows > (int64_t)kPsRows * cluster) cluster *= 2;
    KTK_CUDA_TRY(cudaFuncSetAttribute(prefill_mass_simt_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPsSmem), who);
    KTK_CUDA_TRY(launch_cluster(false, prefill_mass_simt_kernel, (unsigned)(ctas * cluster), kPsThreads, kPsSmem, cluster, st, p, chunks, cluster),
                 who);
    return KTK_OK;
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
    if (!(sm_scale >= 1e-30f && sm_scale - sm_scale == 0.0f)) {          // denominators are divided by it
        set_error("%s: sm_scale %g: finite, at least 1e-30", who, (double)sm_scale);
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
    if (max_pages_per_seq > kMassMaxPages || ctas > 2147483647LL / 8) {
        set_error("%s: batch * num_kv_heads * max_pages_per_seq exceeds the grid limit", who);
        return KTK_ERR_TOO_LARGE;
    }
    void* lse = workspace;
    char* behind = (char*)workspace + lse_bytes(s, total_new_tokens);
    rc = prefill_attention(who, q, q_indptr, total_new_tokens, max_new_tokens, kv_cache, kv_indices, kv_indptr, kv_last_page_len,
                           view_in, sm_scale, o, lse, max_pages_per_seq, behind, need - lse_bytes(s, total_new_tokens), KTK_VARIANT_AUTO, s, status, stream);
    if (rc != KTK_OK) return rc;
    PrefillMassParams p{};
    p.q = q; p.cache = kv_cache; p.q_indptr = q_indptr; p.kv_indices = kv_indices; p.kv_indptr = kv_indptr;
    p.kv_last_page_len = kv_last_page_len; p.page_count = view.page_count; p.sink_tokens = view.sink_tokens;
    p.batch = s->batch; p.Hkv = s->num_kv_heads; p.G = s->group_size; p.num_pages = s->num_pages; p.total_new = total_new_tokens;
    p.max_new = max_new_tokens; p.max_pages = (int)max_pages_per_seq;
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
    return launch_prefill_mass_simt(p, ctas, (int)chunks, max_new_tokens, st);
}
